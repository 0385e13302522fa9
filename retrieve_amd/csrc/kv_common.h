// What the paged-cache kernels (kv_append, kv_select, kv_attention) share: the element types, a
// token's place in the cache, and the int8 row code.
#pragma once

#include "rt_common.h"

namespace rt {

// The types of queries, keys and values (the `dtype` of the C ABI).
enum KvType : int { kKvBf16 = 0, kKvF16 = 1 };

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v8f __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));

template <class E>
struct Kv;
template <>
struct Kv<__bf16> {
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
};
template <>
struct Kv<_Float16> {
  typedef _Float16 V8 __attribute__((ext_vector_type(8)));
};

// The packed tokens' places and the sequences' page tables.
struct KvTokens {
  const int32_t* positions;   // [T]
  const int32_t* seq_ids;     // [T], rows of the page table
  const int32_t* page_table;  // [B, max_pages], physical pages; outside [0, P): absent
  int32_t B, max_pages, P;
  int32_t shift;  // log2 of the page's tokens
};

// A token's position, last block and page-table row. A position or sequence outside the table
// makes it a padding token: `last` is -1 and nothing is read or written for it.
struct KvPlace {
  int32_t pos, last;
  const int32_t* row;
};

__device__ inline KvPlace kv_place(const KvTokens& k, int64_t t) {
  KvPlace p{k.positions[t], -1, k.page_table};
  const int32_t s = k.seq_ids[t];
  if (p.pos < 0 || s < 0 || s >= k.B || (p.pos >> k.shift) >= k.max_pages) return p;
  p.last = p.pos >> k.shift;
  p.row += static_cast<int64_t>(s) * k.max_pages;
  return p;
}

// The physical page of a block of a token's sequence, -1 where it has none.
__device__ inline int32_t kv_page(const KvTokens& k, const KvPlace& p, int32_t block) {
  const int32_t page = p.row[block];
  return page >= 0 && page < k.P ? page : -1;
}

// One code of an int8 row whose largest magnitude is `top` (floored at kKvTopFloor): the quotient
// rounded to fp32, times 127, to the nearest even. Always in [-127, 127], NaN included.
constexpr float kKvTopFloor = 1e-8f;
__device__ inline int kv_code(float x, float top) {
#pragma clang fp contract(off)
  const float v = rintf(x / top * 127.0f);
  return static_cast<int>(fminf(fmaxf(v, -127.0f), 127.0f));
}

// The same code by a reciprocal r = 1 / top (rounded to nearest): q = x r, then q + r (x - q top)
// is the quotient rounded to nearest wherever |x| <= top, top is normal and its significand is not
// all ones (Markstein's theorem; queries of 16 bits have neither), in 3 instructions instead of
// about ten. For a top above 2^100, whose reciprocal may lose bits, x and top come in scaled by
// 2^-64; for an infinite one (r = 0) as 1, since 0 times the infinity would not be a number.
__device__ inline float kv_code_value(float x, float top, float r) {
#pragma clang fp contract(off)
  const float q = x * r;
  const float quotient = __builtin_fmaf(__builtin_fmaf(-q, top, x), r, q);
  return fmaxf(rintf(quotient * 127.0f), -127.0f);  // (NaN: -127)
}

// Eight wait states behind matrix products, before x is read. The compiler counts them itself
// within a block, but not where a branch comes between a product and its first use: the path that
// takes the branch then reads the old registers.
template <class V, int N>
__device__ inline void settle(V (&x)[N]) {
  if constexpr (N == 1) {
    asm volatile("s_nop 7" : "+v"(x[0]));
  } else if constexpr (N == 2) {
    asm volatile("s_nop 7" : "+v"(x[0]), "+v"(x[1]));
  } else if constexpr (N == 4) {
    asm volatile("s_nop 7" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
  } else {
    static_assert(N == 8, "1, 2, 4 or 8 results");
    asm volatile("s_nop 7"
                 : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]),
                   "+v"(x[6]), "+v"(x[7]));
  }
}

// Host: the checks every entry point makes of the shared arguments.
inline int kv_check(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype, int64_t B,
                    int64_t max_pages, int64_t P, int64_t page) {
  RT_CHECK_ARG(T >= 0 && T <= INT32_MAX, "tokens must be in [0, 2^31), got %lld",
               static_cast<long long>(T));
  RT_CHECK_ARG(Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hq <= 1024,
               "query heads (%lld, at most 1024) must be a multiple of key/value heads (%lld)",
               static_cast<long long>(Hq), static_cast<long long>(Hkv));
  RT_CHECK_ARG(B >= 0 && max_pages >= 0 && P >= 0 && B <= INT32_MAX && max_pages <= INT32_MAX &&
                   P <= INT32_MAX,
               "the page table's and the cache's sizes must be in [0, 2^31)");
  RT_CHECK_ARG(page == 16 || page == 32 || page == 64 || page == 128,
               "a page holds 16, 32, 64 or 128 tokens, got %lld", static_cast<long long>(page));
  if (dtype != kKvBf16 && dtype != kKvF16) {
    set_error("dtype must be 0 (bf16) or 1 (fp16), got %d", dtype);
    return kInvalidType;
  }
  if (D != 64 && D != 96 && D != 128 && D != 192 && D != 256) {
    set_error("heads have 64, 96, 128, 192 or 256 channels, got %lld", static_cast<long long>(D));
    return kInvalidType;
  }
  return kOk;
}

inline int32_t kv_shift(int64_t page) { return 31 - __builtin_clz(static_cast<uint32_t>(page)); }

// Host: a [T, H, D] operand's strides (elements) keep every row on 16 bytes.
inline bool kv_rows_aligned(const void* p, int64_t token_stride, int64_t head_stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && token_stride % 8 == 0 && head_stride % 8 == 0;
}

// Calls f with the element type and the channels as a compile-time number.
template <class F>
int kv_dispatch(int dtype, int64_t D, F&& f) {
  auto by_d = [&](auto e) {
    using E = decltype(e);
    switch (D) {
      case 64: return f(E{}, std::integral_constant<int, 64>{});
      case 96: return f(E{}, std::integral_constant<int, 96>{});
      case 128: return f(E{}, std::integral_constant<int, 128>{});
      case 192: return f(E{}, std::integral_constant<int, 192>{});
      default: return f(E{}, std::integral_constant<int, 256>{});
    }
  };
  return dtype == kKvBf16 ? by_d(__bf16{}) : by_d(_Float16{});
}

}  // namespace rt
