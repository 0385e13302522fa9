// The paged cache in 8 bits: its layout, and the code of a block's keys or values.
//
// A full block of one head holds its keys as int8 codes [page, D] and its values transposed, codes
// [D, page], each with one scale (a code stands for code * scale). A sequence's last block, not
// full yet, lies in 16 bits in the sequence's open block, k_tail [page, D] and v_tail [D, page];
// its page's scales are 0 until it is full. So a code depends on its block's 16-bit numbers alone,
// never on how many calls wrote them, and the latest keys are exact. (A block that its sequence is
// cut back into after it was full is the exception: its earlier numbers are those that the codes
// stand for, rounded to 16 bits.) Transposed values give attention's second product its operand (16
// slots of a channel) as it lies in memory.
#pragma once

#include "kv_common.h"

namespace rt {

struct KvInt8 {
  int8_t *k_codes, *v_codes;   // [P, Hkv, page, D], [P, Hkv, D, page]
  float *k_scales, *v_scales;  // [P, Hkv]; 0: not full
  void *k_tail, *v_tail;       // [B, Hkv, page, D], [B, Hkv, D, page]
};

// Codes of one block: code = 127 x / top to the nearest even, top its largest finite magnitude
// (floored at kKvTopFloor). 127 x is exact (18 bits at most), and q + r (y - q top) with q = y r is
// the quotient of y = 127 x rounded to nearest (kv_code_value's comment), so a tie between two
// codes is seen as one. Adding 1.5 2^23 rounds it to a whole number, whose byte is the last one of
// the sum. `odd` blocks: infinities become +-127, NaN 0; a top above 2^100, whose reciprocal may
// lose bits, comes in scaled by 2^-64 with its numbers.
struct BlockCode {
  float top, r, shrink;
  bool odd;
  __device__ BlockCode(float most, bool not_finite) {
    odd = not_finite || most > 0x1p100f;
    shrink = most > 0x1p100f ? 0x1p-64f : 1.0f;
    top = most * shrink;
    r = 1.0f / top;
  }
  template <bool ODD>
  __device__ uint32_t word(float x) const {  // the code is its last byte
#pragma clang fp contract(off)
    float y = x * 127.0f;
    if constexpr (ODD) {
      y = fminf(fmaxf(x * shrink, -top), top) * 127.0f;
      y = x == x ? y : 0.0f;
    }
    const float q = y * r;
    return __builtin_bit_cast(uint32_t,
                              __builtin_fmaf(__builtin_fmaf(-q, top, y), r, q) + 12582912.0f);
  }
  template <bool ODD>
  __device__ int four(float a, float b, float c, float d) const {
    const uint32_t ab = __builtin_amdgcn_perm(word<ODD>(b), word<ODD>(a), 0x0c0c0400u);
    const uint32_t cd = __builtin_amdgcn_perm(word<ODD>(d), word<ODD>(c), 0x0c0c0400u);
    return static_cast<int>(ab | cd << 16);
  }
};
// A number's part in `top`.
__device__ inline float finite_size(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;
}

// Numbers of 16 bits two at a time, as whole numbers: their magnitudes order like the bits below
// the sign, and they themselves like two's complement once negative ones have these bits flipped.
typedef unsigned short v2u16 __attribute__((ext_vector_type(2)));
typedef short v2i16 __attribute__((ext_vector_type(2)));
__device__ inline v2u16 max_magnitude(v2u16 most, uint32_t x) {
  return __builtin_elementwise_max(most, __builtin_bit_cast(v2u16, x & 0x7fff7fffu));
}
__device__ inline v2i16 ordered(uint32_t x) {  // (its own inverse)
  const v2i16 v = __builtin_bit_cast(v2i16, x);
  const uint32_t flip = __builtin_bit_cast(uint32_t, v >> 15) & 0x7fff7fffu;
  return __builtin_bit_cast(v2i16, x ^ flip);
}
template <class E>
inline constexpr int kInfinityBits = 0x7f80;  // from here on: not finite
template <>
inline constexpr int kInfinityBits<_Float16> = 0x7c00;
template <class E>
__device__ inline float from_bits(int bits) {
  const unsigned short b = static_cast<unsigned short>(bits);
  return static_cast<float>(__builtin_bit_cast(E, b));
}

// Host: the checks of an 8-bit cache's pointers.
inline int kv_check_int8(const KvInt8& c, int64_t B, int64_t P) {
  RT_CHECK_ARG(P == 0 || (c.k_codes && c.v_codes && c.k_scales && c.v_scales), "null cache");
  RT_CHECK_ARG(B == 0 || (c.k_tail && c.v_tail), "null open blocks");
  RT_CHECK_ARG(kv_rows_aligned(c.k_codes, 0, 0) && kv_rows_aligned(c.v_codes, 0, 0) &&
                   kv_rows_aligned(c.k_tail, 0, 0) && kv_rows_aligned(c.v_tail, 0, 0),
               "the cache must start on 16 bytes");
  return kOk;
}

}  // namespace rt
