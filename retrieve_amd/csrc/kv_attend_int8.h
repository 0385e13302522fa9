// Softmax attention of each token over chosen blocks of the 8-bit paged cache (kv_int8.h).
//
// out = sum_j w_j v_j / sum_j w_j with w_j = exp(x_j), x_j = scale q . k_j over the listed blocks'
// keys at positions up to the token's; keys and values of full blocks are codes times one scale a
// block and head, those of the token's own open block 16-bit numbers.
//
// Codes meet the matrix cores as fp16: a byte u = code + 128 with eight zero bits above it is the
// subnormal u 2^-24, which they take exactly, so 4 codes cost 3 instructions (1024 + u, less 1152,
// would be 5). The 128 too many are taken off as 128 sum(q) where the first product starts and as
// 128 sum(p), an operand of constant codes, behind the second. bf16 queries become fp16 as well: a
// row is scaled by a power of two so that its largest magnitude is in [2^14, 2^15), where fp16
// holds every 8-bit significand down to 2^-17; what is lost is below 2^-39 of the row's largest.
// The row's power of two and the scale's come back as one whole exponent, applied to the block's
// scale times the scale's significand: infinite only beside scores that are far, or next to 0.
//
// The scale of a block's keys multiplies the scores; that of its values, s_v, goes into the
// exponent: with t = x log2 e + log2 s_v and m the running maximum of t, p = 2^(t - m) is the
// weight that the second product wants (codes stand for s_v each), and p / s_v what the sum of
// weights wants. So neither product is rescaled from block to block. Beside codes p is rounded to
// fp16 (2^-11, and held 2^7 times as large as the maximum says: it reaches 2^15, its step below
// 2^-14 is 2^-31 of the largest weight) whatever the queries' type; beside the open block, whose
// values are of the queries' type, to that (bf16: 2^-8). The sum takes it unrounded. The maximum is
// raised only where a score passes it by 8 (in powers of two), so most steps exchange nothing
// between lanes. A score and its maximum meet in one fused multiply-add: past 2^23 that leaves the
// rounded maximum by whole powers of two, so rows of such scores are `far`, and taken again key by
// key (AloneSums).
//
// A wave holds columns, 16 query heads a tile: heads of one token, or heads of several tokens that
// share a key/value head. It takes 64 keys a step, four subtiles of 16 slots, lane group g (lanes
// 16 g to 16 g + 15) having subtile g:
//   S^T [keys x columns] = K Q^T: four products of 16 keys, row m of product j being slot 4 j +
//     m % 4 of subtile m / 4, so that lane group g gets slots 4 j .. 4 j + 3 of its own subtile: 16
//     neighbouring slots over the four products;
//   O^T [channels x columns] += V^T P^T: the weights are where the first product left them, and the
//     operand V^T is 16 bytes of a channel (values lie transposed).
// A lane's column is one head in both products: maxima, sums and rescaling stay in the lane.
//
// An operand's neighbouring lanes hold different rows (keys, channels). Loaded like that, every
// lane's 16 bytes are an access of their own (56 of 64 lanes' counted; prompts of 2053 tokens were
// bound by that, 210 us). So memory is read in its own order, 1 KiB a load, straight to the wave's
// own LDS, and the operands from there: the next step's keys as soon as this one's are read, its
// values likewise. 16-byte chunks are permuted by the row where they are loaded, so that those of
// one read lie in different banks.
//
// Single tokens are bound by memory: 64 of them over 64 blocks of 64 keys (8 heads of 128 channels,
// 526 MB of codes) take 93 us, 5.6 TB/s; about 15 us of that are the start (lists, pages and scales
// are looked up one after the other before the first codes) and the end, the rest runs at 6.7 TB/s.
// Prompts are bound by the vector instructions (59 % of the time, a third of them makes codes into
// fp16 and a third is the softmax) and by the waits between operands and products: 2053 tokens over
// 16 blocks each take 153 us. 8 tokens share a pass there; 4, whose codes are widened for one tile
// of columns, take 169.
#pragma once

#include <type_traits>

#include "kv_attend.h"
#include "kv_int8.h"
#include "lds_load.h"

namespace rt {

struct AttendInt8Args : AttendBase {
  KvInt8 cache;
  float size;  // scale = size * 2^power, size in [0.5, 1)
  int32_t power;
};

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef int v2i __attribute__((ext_vector_type(2)));

__device__ inline v4f mma16(v8h a, v8h b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline v4f mma16(Kv<__bf16>::V8 a, Kv<__bf16>::V8 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight codes (two words), plus 128, as fp16 in units of 2^-24.
constexpr int kCodeBits = 24;
constexpr float kCodeUnit = 0x1p-24f;
__device__ inline v8h codes_to_half(int lo, int hi) {
  const uint32_t a = static_cast<uint32_t>(lo) ^ 0x80808080u;
  const uint32_t b = static_cast<uint32_t>(hi) ^ 0x80808080u;
  union {
    uint32_t u[4];
    v8h v;
  } x;
  x.u[0] = __builtin_amdgcn_perm(0u, a, 0x0c010c00u);  // (0x0c: a zero byte)
  x.u[1] = __builtin_amdgcn_perm(0u, a, 0x0c030c02u);
  x.u[2] = __builtin_amdgcn_perm(0u, b, 0x0c010c00u);
  x.u[3] = __builtin_amdgcn_perm(0u, b, 0x0c030c02u);
  return x.v;
}
__device__ inline v8h codes_of_128() {
  union {
    uint32_t u[4];
    v8h v;
  } x = {{0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u}};
  return x.v;
}

// A lane's 16 bytes at `from` straight to lds + 16 lane. STREAM: of rows that are read once (not
// kept in L2 before others).
template <bool STREAM>
__device__ inline void load_to_lds(const int8_t* from, char* lds) {
  auto* g = (const __attribute__((address_space(1))) void*)(from);
  auto* l = (__attribute__((address_space(3))) void*)(lds);
  if constexpr (STREAM) {
    __builtin_amdgcn_global_load_lds(g, l, 16, 0, kNontemporal);
  } else {
    __builtin_amdgcn_global_load_lds(g, l, 16, 0, 0);
  }
}

// N reads of 16 bytes from LDS, STEP bytes apart, waited for. As instructions of the compiler's
// they would wait for every load to LDS under way (it cannot tell the places apart); here the
// caller has waited for the ones that count.
__device__ inline uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)(p)));
}
template <int STEP, int N>
__device__ inline void read_lds(uint32_t at, v4i (&x)[N]) {
  static_assert(N == 2 || N == 4, "reads of a block");
  static_assert((N - 1) * STEP < 65536, "offsets");
  if constexpr (N == 4) {
    asm volatile(
        "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:%5\n\tds_read_b128 %2, %4 offset:%6\n\t"
        "ds_read_b128 %3, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
        : "v"(at), "i"(STEP), "i"(2 * STEP), "i"(3 * STEP)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1])
        : "v"(at), "i"(STEP)
        : "memory");
  }
}
// Four of 8 bytes.
template <int STEP>
__device__ inline void read_lds_halves(uint32_t at, v2i (&x)[4]) {
  asm volatile(
      "ds_read_b64 %0, %4\n\tds_read_b64 %1, %4 offset:%5\n\tds_read_b64 %2, %4 offset:%6\n\t"
      "ds_read_b64 %3, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
      : "v"(at), "i"(STEP), "i"(2 * STEP), "i"(3 * STEP)
      : "memory");
}

// Where 16-byte chunk c of a staged row of keys (of 64) lies in the row: rows that a read takes
// together (4 j + m % 4 of subtile m / 4, m the lane) have it in different banks.
template <int D>
__device__ inline int key_chunk(int row, int c) {
  const int b0 = row & 1, b1 = (row >> 1) & 1, s0 = (row >> 4) & 1, s1 = (row >> 5) & 1;
  if constexpr (D == 256) return c ^ (b0 | b1 << 1 | s0 << 2 | s1 << 3);
  if constexpr (D == 128) return c ^ (b1 | s0 << 1 | (s1 ^ b0) << 2);
  return c < D / 64 * 4 ? c ^ (s0 | (s1 ^ b1) << 1) : c;
}
// Staged values: pages of 64 slots and more: channels of four chunks, one a subtile; pages of 32:
// page by page, channels of two; pages of 16: subtile by subtile, channels of one.
template <int D, int SHIFT>
__device__ inline int value_offset(int channel, int sub) {
  if constexpr (SHIFT >= 6) {
    const int b1 = (channel >> 1) & 1, b2 = (channel >> 2) & 1, b3 = (channel >> 3) & 1;
    return 64 * channel + 16 * (sub ^ (b2 | (b3 ^ b1) << 1));
  } else if constexpr (SHIFT == 5) {
    return 32 * D * (sub >> 1) + 32 * channel + 16 * ((sub ^ (channel >> 3)) & 1);
  } else {
    return 16 * D * sub + 16 * channel;
  }
}

// The largest of 16 numbers (NaN passed over) in 8 instructions; fmaxf would first quiet each,
// which costs as many again. For results that have settled.
__device__ inline float max3(float a, float b, float c) {
  float x;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(x) : "v"(a), "v"(b), "v"(c));
  return x;
}
__device__ inline float most_of(const v4f (&x)[4]) {
  const float a = max3(x[0][0], x[0][1], x[0][2]), b = max3(x[0][3], x[1][0], x[1][1]);
  const float c = max3(x[1][2], x[1][3], x[2][0]), d = max3(x[2][1], x[2][2], x[2][3]);
  const float e = max3(x[3][0], x[3][1], x[3][2]);
  return max3(max3(a, b, c), max3(d, e, x[3][3]), a);
}

// What a lane knows of its subtile (16 slots), 64 of them being looked up at a time.
struct Subtile {
  int32_t page, at;  // physical page; first slot * 32 + keys (0: none)
  uint32_t who;      // the tokens whose lists hold it
  float ks, lift, inv;  // the keys' scale times a.size; the values' one's logarithm and inverse
  __device__ void clear() {
    page = 0;
    at = 0;
    who = 0u;
    ks = inv = 1.0f;
    lift = 0.0f;
  }
  // Its page's scales, and what is kept of them; false: the page has no codes.
  __device__ void scales(const AttendInt8Args& a, int head, float (&scale)[2]) const {
    const int64_t row = static_cast<int64_t>(page) * a.Hkv + head;
    scale[0] = a.cache.k_scales[row];
    scale[1] = a.cache.v_scales[row];
  }
  __device__ bool take(const AttendInt8Args& a, const float (&scale)[2]) {
    if (!(scale[0] > 0.0f)) return false;
    ks = scale[0] * a.size;
    lift = __builtin_amdgcn_logf(scale[1]);
    inv = 1.0f / scale[1];
    return true;
  }
};
// A step's four subtiles (subtiles 4 i to 4 i + 3), of which this lane has the scores of one.
struct Step {
  int i;
  int32_t page, at;
  uint32_t who;
  float ks, lift, inv;
};

__device__ inline float lane_value(float x, int lane) {
  return __builtin_bit_cast(float,
                            __builtin_amdgcn_readlane(__builtin_bit_cast(int32_t, x), lane));
}

// A wave's queries, accumulators and sums: CT tiles of 16 columns, lane % 16 of each tile this
// lane's. acc: channel 16 i + 4 (lane / 16) + r, in units of kCodeUnit and with 128 sum(p) too
// much, which is in `over`; m: the maximum of t less kLift, l: this lane's share of the sum.
template <class E, int D, int SHIFT, int CT>
struct Int8Wave {
  using V8 = typename Kv<E>::V8;
  static constexpr int DT = D / 16, KS = D / 32;  // channel tiles, steps of 32 channels
  static constexpr int KL = D / 64;               // 16-byte loads of a key a lane
  static constexpr bool HALF = D % 64 != 0;       // and one of 8 bytes
  static constexpr float kLift = 7.0f;            // maximum - m
  static constexpr float kFar = 0x1p23f;
  static constexpr float kLeast = 1.17549435e-38f, kMost = 3.402823466e38f;  // (normal, finite)
  v4f acc[CT][DT], over[CT];
  float m[CT], l[CT];
  bool far;  // a score was past kFar, in some column: the sums are of no use
  // Two tiles' queries stay in LDS: in registers they would spill others beside the next step's
  // keys and values.
  static constexpr bool kQueriesInLds = CT > 1;
  v8h qf[kQueriesInLds ? 1 : KS];
  const v8h* q_lds;  // [CT][KS][64]
  int power[CT];    // a score is multiplied by its block's ks * 2^power
  float start[CT];  // -128 sum(q), in units of kCodeUnit
  bool odd[CT];     // the column's query is not finite
  static constexpr int LOADS = D / 16;  // of 64 keys' codes, of their values': 1 KiB each
  static constexpr int STAGE = 64 * D;  // bytes of a step's keys in the wave's LDS; its values too

  __device__ void clear() {
    far = false;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[c][i] = v4f{0.f, 0.f, 0.f, 0.f};
      over[c] = v4f{0.f, 0.f, 0.f, 0.f};
      m[c] = -3.402823466e38f;
      l[c] = 0.0f;
    }
  }
  // The first of a lane group's eight channels in step s of the first product.
  __device__ static int channel(int s, int grp) {
    return s < 2 * KL ? 64 * (s >> 1) + 16 * grp + 8 * (s & 1) : 64 * KL + 8 * grp;
  }
  // This lane's column of a tile is query head `head` of token t (its first row where it is not
  // `real`).
  __device__ static void fetch_q(const AttendInt8Args& a, int64_t t, int64_t head, bool real,
                                 V8 (&x)[KS]) {
    const E* q = static_cast<const E*>(a.q) + (real ? t * a.q_st + head * a.q_sh : 0);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      x[s] = *reinterpret_cast<const V8*>(q + channel(s, lane_id() >> 4));
    }
  }
  // The fetched queries as tile c's (zeros where they are not `real`).
  __device__ void take_q(const AttendInt8Args& a, int c, const V8 (&x)[KS], bool real,
                         v8h* lds = nullptr) {
    float most = 0.0f, none = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = static_cast<float>(x[s][e]);
        most = fmaxf(most, fabsf(f));
        none = fmaf(f, 0.0f, none);  // (not a number beside an infinity or a NaN)
      }
    }
#pragma unroll
    for (int i = 16; i < kWave; i <<= 1) {
      most = fmaxf(most, __shfl_xor(most, i));
      none += __shfl_xor(none, i);
    }
    odd[c] = real && !(none == 0.0f);
    real = real && !odd[c];
    int up = 0;
    if constexpr (!std::is_same<E, _Float16>::value) {
      if (real && most > 0.0f) up = 15 - __builtin_amdgcn_frexp_expf(most);
    }
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      v8h y;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = real ? ldexpf(static_cast<float>(a.minus ? -x[s][e] : x[s][e]), up) : 0.0f;
        y[e] = static_cast<_Float16>(f);
        sum += static_cast<float>(y[e]);
      }
      if constexpr (kQueriesInLds) {
        lds[(c * KS + s) * kWave + lane_id()] = y;
      } else {
        qf[s] = y;
      }
    }
#pragma unroll
    for (int i = 16; i < kWave; i <<= 1) sum += __shfl_xor(sum, i);
    start[c] = sum * (-128.0f * kCodeUnit);
    power[c] = a.power - up + kCodeBits;
  }

  // The step of quad i. Its page is one where pages hold 64 slots or more.
  __device__ static Step step_of(const Subtile& s, int i) {
    Step x;
    x.i = i;
    const int own = 4 * i + (lane_id() >> 4);
    x.at = __shfl(s.at, own);
    if constexpr (SHIFT >= 6) {
      x.page = __builtin_amdgcn_readlane(s.page, 4 * i);
      x.who = __builtin_amdgcn_readlane(static_cast<int32_t>(s.who), 4 * i);
      x.ks = lane_value(s.ks, 4 * i);
      x.lift = lane_value(s.lift, 4 * i);
      x.inv = lane_value(s.inv, 4 * i);
    } else {
      x.page = __shfl(s.page, own);
      x.who = __shfl(s.who, own);
      x.ks = __shfl(s.ks, own);
      x.lift = __shfl(s.lift, own);
      x.inv = __shfl(s.inv, own);
    }
    return x;
  }
  // A step's keys to LDS: 64 rows, chunks permuted (key_chunk). STREAM: rows that are read once.
  template <bool STREAM>
  __device__ static void load_k(const AttendInt8Args& a, const Subtile& s, int head, int quad,
                                char* lds) {
    const auto rows = [&](int32_t page, int32_t at) {
      return a.cache.k_codes +
             (((static_cast<int64_t>(page) * a.Hkv + head) << SHIFT) + (at >> 5)) * D;
    };
    const auto of = [&](int sub) {  // the same in every lane
      return rows(__builtin_amdgcn_readlane(s.page, 4 * quad + sub),
                  __builtin_amdgcn_readlane(s.at, 4 * quad + sub));
    };
    const int8_t* first = of(0);
#pragma unroll
    for (int x = 0; x < LOADS; ++x) {
      const int at = x * kWave + lane_id(), row = at / (D / 16), c = at % (D / 16);
      const int in = row * D + 16 * key_chunk<D>(row, c);
      if constexpr (SHIFT >= 6) {
        buffer_load_lds<16, STREAM>(first, 64 * D, in, lds + x * 1024);
      } else if constexpr (D % 64 == 0) {
        constexpr int EACH = D / 64;  // loads of a subtile
        if (x > 0 && x % EACH == 0) first = of(x / EACH);
        buffer_load_lds<16, STREAM>(first, 16 * D, in - x / EACH * (16 * D), lds + x * 1024);
      } else {
        const int from = 4 * quad + (row >> 4);
        const int8_t* const mine = rows(__shfl(s.page, from), __shfl(s.at, from));
        load_to_lds<STREAM>(mine + (in - (row >> 4) * (16 * D)),
                            lds + x * 1024);
      }
    }
  }
  // A step's values to LDS, as value_offset has them.
  template <bool STREAM>
  __device__ static void load_v(const AttendInt8Args& a, const Subtile& s, int head, int quad,
                                char* lds) {
    const auto page = [&](int32_t p) {
      return a.cache.v_codes + (((static_cast<int64_t>(p) * a.Hkv + head) * D) << SHIFT);
    };
    const auto of = [&](int sub) {
      return page(__builtin_amdgcn_readlane(s.page, 4 * quad + sub));
    };
    const int8_t* first = of(0);
    if constexpr (SHIFT >= 6) first += __builtin_amdgcn_readlane(s.at, 4 * quad) >> 5;
#pragma unroll
    for (int x = 0; x < LOADS; ++x) {
      const int at = x * kWave + lane_id();
      if constexpr (SHIFT >= 6) {
        const int channel = at >> 2, in = value_offset<D, SHIFT>(channel, at & 3) - 64 * channel;
        // (of a channel of 128 slots another step takes the rest of the line)
        buffer_load_lds<16, STREAM && SHIFT == 6>(first, D << SHIFT, (channel << SHIFT) + in,
                                                  lds + x * 1024);
      } else if constexpr (SHIFT == 5) {
        constexpr int EACH = LOADS / 2;  // loads of a page
        if (x == EACH) first = of(2);
        const int in = at - x / EACH * (2 * D), channel = in >> 1;
        buffer_load_lds<16, STREAM>(first, D << SHIFT, value_offset<D, SHIFT>(channel, in & 1),
                                    lds + x * 1024);
      } else if constexpr (D % 64 == 0) {
        constexpr int EACH = D / 64;
        if (x > 0 && x % EACH == 0) first = of(x / EACH);
        buffer_load_lds<16, STREAM>(first, D << SHIFT, 16 * (at - x / EACH * D), lds + x * 1024);
      } else {
        const int sub = at / D;
        load_to_lds<STREAM>(page(__shfl(s.page, 4 * quad + sub)) + 16 * (at - sub * D),
                            lds + x * 1024);
      }
    }
  }
  // The weights of tile c's scores (slot 4 j + r of this lane's subtile): the maximum raised, the
  // sum extended. f multiplies the scores, lift is the logarithm of what the values stand for, inv
  // its inverse. A column has the subtile's first n keys (`some` lane's n is not 16, or its scores
  // may not be numbers), or none of them where it does not count.
  template <class P>
  __device__ void weigh(int c, v4f (&sc)[4], float f, float lift, float inv, bool counts, int n,
                        bool some, P (&p)[2]) {
    settle(sc);
    if (some) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[j][r] = counts && 4 * j + r < n ? sc[j][r] : -INFINITY;
      }
    }
    // (a score of -inf stays that, one of 0 too; another whose factor was infinite is far: scores
    // in units of the codes are 0 or 2^-48 at least)
    f = fminf(fmaxf(f, kLeast), kMost);
    if (!counts) lift = -INFINITY;
    const float high = fmaf(most_of(sc), f, lift);
    if (__any(high - m[c] > 8.0f + kLift)) {
      far |= __any(fabsf(high) > kFar && high != -INFINITY) != 0;
      float next = fmaxf(high, __shfl_xor(high, 16));
      next = fmaxf(next, __shfl_xor(next, 32));
      next = fmaxf(next - kLift, m[c]);
      const float keep = __builtin_amdgcn_exp2f(m[c] - next);
      m[c] = next;
      l[c] *= keep;
      over[c] *= keep;
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[c][i] *= keep;
    }
    const float less = lift - m[c];
    float sum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        e[r] = __builtin_amdgcn_exp2f(fmaf(sc[j][r], f, less));
        p[j / 2][4 * (j % 2) + r] =
            static_cast<std::remove_reference_t<decltype(p[0][0])>>(e[r]);
      }
      sum[j] = (e[0] + e[1]) + (e[2] + e[3]);
    }
    l[c] = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), inv, l[c]);
  }
  // One step on what load_k and load_v have under way to `keys` and `values`; `fetch_k` and
  // `fetch_v` start the next one's loads there (`more`) as soon as this one's operands are read.
  // counts, n: of each tile's column in this lane's subtile; `some`: a lane's n is not 16.
  template <class FK, class FV>
  __device__ void step(const char* keys, const char* values, const Step& s,
                       const bool (&counts)[CT], const int (&n)[CT], bool some, bool more,
                       FK&& fetch_k, FV&& fetch_v) {
    const int col = lane_id() & 15, grp = lane_id() >> 4;
    wait_vmcnt<LOADS>();  // (the values' loads are later)
    v4f sc[CT][4];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[c][j] = v4f{start[c], start[c], start[c], start[c]};
    }
    const int row = 16 * (col >> 2) + (col & 3);
    const uint32_t k_at = lds_address(keys) + row * D;
    const uint32_t q_at = kQueriesInLds ? lds_address(q_lds) + 16 * lane_id() : 0;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      v8h q[CT][2];
      if constexpr (kQueriesInLds) {
        static_assert(CT == 2, "two tiles");
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          v4i x[2];
          read_lds<16 * kWave>(q_at + (c * KS + 2 * i) * 16 * kWave, x);
          q[c][0] = __builtin_bit_cast(v8h, x[0]);
          q[c][1] = __builtin_bit_cast(v8h, x[1]);
        }
      } else {
        q[0][0] = qf[2 * i];
        q[0][1] = qf[2 * i + 1];
      }
      v4i k[4];
      read_lds<4 * D>(k_at + 16 * key_chunk<D>(row, 4 * i + grp), k);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v8h x = codes_to_half(k[j][0], k[j][1]), y = codes_to_half(k[j][2], k[j][3]);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          sc[c][j] = mma16(x, q[c][0], sc[c][j]);
          sc[c][j] = mma16(y, q[c][1], sc[c][j]);
        }
      }
    }
    if constexpr (HALF) {
      v8h q[CT];
      if constexpr (kQueriesInLds) {
        v4i x[2];
        read_lds<KS * 16 * kWave>(q_at + 2 * KL * 16 * kWave, x);
#pragma unroll
        for (int c = 0; c < CT; ++c) q[c] = __builtin_bit_cast(v8h, x[c]);
      } else {
        q[0] = qf[2 * KL];
      }
      v2i k[4];
      read_lds_halves<4 * D>(k_at + 64 * KL + 8 * grp, k);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v8h x = codes_to_half(k[j][0], k[j][1]);
#pragma unroll
        for (int c = 0; c < CT; ++c) sc[c][j] = mma16(x, q[c], sc[c][j]);
      }
    }
    if (more) {
      fetch_k();
      wait_vmcnt<LOADS>();
    } else {
      wait_vmcnt<0>();
    }
    v8h p[CT][2];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      // (a tile none of whose columns counts the step: weights of 0, without their exponentials)
      p[c][0] = p[c][1] = v8h{};
      if (CT > 1 && !__any(counts[c])) continue;
      weigh(c, sc[c], ldexpf(s.ks, power[c]), s.lift, s.inv, counts[c], n[c], some, p[c]);
    }
    constexpr int ROW = SHIFT >= 6 ? 64 : SHIFT == 5 ? 32 : 16;  // bytes of a staged channel
    const uint32_t v_at = lds_address(values) + value_offset<D, SHIFT>(col, grp);
    const auto add = [&](int i, const v4i& v) {
      const v8h x = codes_to_half(v[0], v[1]), y = codes_to_half(v[2], v[3]);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        acc[c][i] = mma16(x, p[c][0], acc[c][i]);
        acc[c][i] = mma16(y, p[c][1], acc[c][i]);
      }
    };
#pragma unroll
    for (int i = 0; i + 4 <= DT; i += 4) {
      v4i v[4];
      read_lds<16 * ROW>(v_at + 16 * i * ROW, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) add(i + j, v[j]);
    }
    if constexpr (DT % 4 != 0) {
      v4i v[2];
      read_lds<16 * ROW>(v_at + 16 * (DT - 2) * ROW, v);
#pragma unroll
      for (int j = 0; j < 2; ++j) add(DT - 2 + j, v[j]);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      over[c] = mma16(codes_of_128(), p[c][0], over[c]);
      over[c] = mma16(codes_of_128(), p[c][1], over[c]);
    }
    if (more) fetch_v();
  }
  // One step of tile c over a sequence's open block: 16-bit rows, in their own type. This lane's
  // subtile begins at slot `first`, its column (head hq of token t) has n keys of it; n_most, the
  // most of any column. Once a list at most, so the queries are read again. Values that are not
  // finite would reach the columns that do not have them (0 times infinity): where there are any,
  // each token's sums are taken alone.
  __device__ void open_step(const AttendInt8Args& a, int c, int64_t seq, int head, int64_t t,
                            int64_t hq, bool real, int first, int n, int n_most, int tokens,
                            int tok) {
    const int grp = lane_id() >> 4, col = lane_id() & 15;
    const int64_t open = ((seq * a.Hkv + head) << SHIFT) * D;
    real = real && !odd[c];
    const E* q = static_cast<const E*>(a.q) + (real ? t * a.q_st + hq * a.q_sh : 0) + 8 * grp;
    v4f sc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) sc[j] = v4f{0.f, 0.f, 0.f, 0.f};
    const int k_slot = __shfl(first, 16 * (col >> 2));  // (first slot of the keys' subtile)
    const E* k = static_cast<const E*>(a.cache.k_tail) + open + (k_slot + (col & 3)) * D + 8 * grp;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      V8 x = *reinterpret_cast<const V8*>(q + 32 * s);
      if (!real) x = V8{};
      if (a.minus) x = -x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sc[j] = mma16(*reinterpret_cast<const V8*>(k + 4 * j * D + 32 * s), x, sc[j]);
      }
    }
    V8 p[2];
    weigh(c, sc, a.scale, 0.0f, 1.0f, n > 0, n, true, p);
    const E* v = static_cast<const E*>(a.cache.v_tail) + open + (col << SHIFT) + first;
    float none = 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const V8 x = reinterpret_cast<const V8*>(v + ((16 * i) << SHIFT))[h];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (8 * h + e < n_most) none = fmaf(static_cast<float>(x[e]), 0.0f, none);
        }
      }
    }
    const bool alone = __any(!(none == 0.0f));
    for (int one = 0; one < (alone ? tokens : 1); ++one) {
      const bool mine = !alone || tok == one;
      int most = n_most;
      if (alone) {  // the keys of this token in each lane's subtile
        most = mine ? n : 0;
        for (int i = 1; i < 16; i <<= 1) most = max(most, __shfl_xor(most, i));
      }
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        v4f sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          V8 x = reinterpret_cast<const V8*>(v + ((16 * i) << SHIFT))[h];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (8 * h + e >= most) x[e] = static_cast<E>(0.0f);  // (slots that hold anything)
          }
          sum = mma16(x, p[h], sum);
        }
        v4f all[1] = {sum};
        settle(all);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[c][i][r] = mine ? fmaf(all[0][r], kCodeUnit, acc[c][i][r]) : acc[c][i][r];
        }
      }
    }
  }
  // The sums in their own units; a column whose query is not finite is not a number.
  __device__ void finish() {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      l[c] += __shfl_xor(l[c], 16);
      l[c] += __shfl_xor(l[c], 32);
      if (odd[c] && l[c] != 0.0f) l[c] = NAN;
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[c][i] = (acc[c][i] - over[c]) * (1.0f / kCodeUnit);
    }
  }
};

// Waves a SIMD that the registers leave room for: as many as the workgroups' LDS does (512 D bytes
// and up to 20 KiB each of a CU's 160 KiB), but for what would spill then: two tiles of 64 channels
// over pages of 16 and 32, the split form (0 tiles) and two tiles of 96, one of 96 over pages of 16.
constexpr int attend_int8_waves(int D, int shift, int tiles) {
  if (D > 128) return 1;
  return (D <= 64 && shift >= 6) || (D <= 96 && shift >= 5 && tiles == 1) ? 3 : 2;
}

// The sums of one query head of one token over a wave's share of its list (units of 64 keys part,
// part + parts, ...), key by key, for rows of far scores: it spares registers, not time. A score is
// summed in 64 bits and rounded once, so equal ones are equal whatever their blocks' scales; the
// maximum is of the scores alone, and weights times a value's scale stay in fp32. Channel d of the
// sums is in acc[d / 64] of lane d % 64.
template <class E, int D, int SHIFT>
struct AloneSums {
  using V8 = typename Kv<E>::V8;
  static constexpr int R = (D + kWave - 1) / kWave;
  float m, l, acc[R];

  __device__ void run(const AttendInt8Args& a, int64_t t, int head, int64_t hq, int part,
                      int parts) {
    m = -3.402823466e38f;
    l = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = 0.0f;
    const KvPlace place = kv_place(a.tok, t);
    if (place.last < 0) return;
    const int lane = lane_id();
    const int64_t seq = a.tok.seq_ids[t], open = ((seq * a.Hkv + head) << SHIFT) * D;
    const int32_t* list = a.blocks + (t * a.Hkv + head) * a.count;
    const E* q = static_cast<const E*>(a.q) + t * a.q_st + hq * a.q_sh;
    const E* k_tail = static_cast<const E*>(a.cache.k_tail) + open;
    const E* v_tail = static_cast<const E*>(a.cache.v_tail) + open;
    const double scale = a.minus ? -static_cast<double>(a.scale) : a.scale;
    const int64_t keys = static_cast<int64_t>(a.count) << SHIFT;
#pragma unroll 1
    for (int64_t first = int64_t{part} * 64; first < keys; first += int64_t{parts} * 64) {
      const int64_t key = first + lane;
      const int32_t slot = static_cast<int32_t>(key) & ((1 << SHIFT) - 1);
      int32_t page = -1;  // -1: no key; past the cache's: the open block
      float x = -INFINITY, vs = 0.0f;
      if (key < keys) {
        const int32_t block = list[key >> SHIFT];
        if (block >= 0 && block <= place.last && slot <= place.pos - (block << SHIFT)) {
          page = kv_page(a.tok, place, block);
        }
        if (page >= 0) {
          const int64_t row = static_cast<int64_t>(page) * a.Hkv + head;
          const float ks = a.cache.k_scales[row];
          if (ks > 0.0f) {
            vs = a.cache.v_scales[row];
          } else {
            page = block == place.last ? a.tok.P : -1;
          }
          if (page >= 0) {
            const int8_t* codes = a.cache.k_codes + ((row << SHIFT) + slot) * D;
            double sum = 0.0, none = 0.0;
#pragma unroll 1
            for (int d = 0; d < D; d += 8) {
              const V8 f = *reinterpret_cast<const V8*>(q + d);
              V8 k{};
              v2i c{};
              if (ks > 0.0f) {
                c = *reinterpret_cast<const v2i*>(codes + d);
              } else {
                k = *reinterpret_cast<const V8*>(k_tail + slot * D + d);
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const double of = static_cast<double>(static_cast<float>(f[e]));
                const float code = static_cast<int8_t>(c[e >> 2] >> (8 * (e & 3)));
                sum = __builtin_fma(of, ks > 0.0f ? code : static_cast<float>(k[e]), sum);
                none = __builtin_fma(of, 0.0, none);
              }
            }
            // (a query that is not finite: not a number, whatever the key)
            x = static_cast<float>((sum + none) * (ks > 0.0f ? ks : 1.0f) * scale);
          }
        }
      }
      float top = x;
#pragma unroll
      for (int i = 1; i < kWave; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
      const float next = fmaxf(m, top), keep = __builtin_amdgcn_exp2f(m - next);
      const float w = page < 0 ? 0.0f : __builtin_amdgcn_exp2f(x - next);
      float sum = w;
#pragma unroll
      for (int i = 1; i < kWave; i <<= 1) sum += __shfl_xor(sum, i);
      m = next;
      l = l * keep + sum;
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r] *= keep;
#pragma unroll 1
      for (uint64_t left = __ballot(page >= 0); left != 0; left &= left - 1) {
        const int at = __builtin_ctzll(left);
        const int32_t pg = __builtin_amdgcn_readlane(page, at);
        const int32_t sl = __builtin_amdgcn_readlane(slot, at);
        const float wj = lane_value(w, at), sj = lane_value(vs, at);
        const int8_t* codes = a.cache.v_codes +
                              (((static_cast<int64_t>(pg) * a.Hkv + head) * D) << SHIFT) + sl;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int d = r * kWave + lane;
          if (d < D) {
            const float v = pg < a.tok.P ? static_cast<float>(codes[d << SHIFT]) * sj
                                         : static_cast<float>(v_tail[(d << SHIFT) + sl]);
            acc[r] = fmaf(wj, v, acc[r]);
          }
        }
      }
    }
  }
};

// The kernel's arguments, read where they are used: what a path that is seldom taken reads would
// otherwise be held in registers from the start.
__device__ inline const AttendInt8Args& late_args() {
  auto* p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttendInt8Args*)(p);
}

// Single tokens, and few rows: the workgroup's waves (and `parts` workgroups) share a row's list in
// units of 64 keys.
template <class E, int D, int SHIFT>
struct SplitWave : Int8Wave<E, D, SHIFT, 1> {
  using Base = Int8Wave<E, D, SHIFT, 1>;
  // Chunk `chunk` of this wave's units of 64 keys (units part, part + parts, ...): a subtile a
  // lane, those with keys in codes (`full`) and in the open block. False: past the list's end.
  __device__ static bool fetch(const AttendInt8Args& a, const int32_t* list, const KvPlace& place,
                               int head, int part, int parts, int chunk, Subtile& s,
                               uint64_t& full, uint64_t& open) {
    const int64_t first = (part + static_cast<int64_t>(parts) * 16 * chunk) * 64;
    if (first >= static_cast<int64_t>(a.count) << SHIFT) return false;
    const int64_t unit = part + static_cast<int64_t>(parts) * (16 * chunk + (lane_id() >> 2));
    const int64_t key = unit * 64 + 16 * (lane_id() & 3);
    const int64_t entry = key >> SHIFT;
    s.clear();
    bool is_open = false;
    if (entry < a.count) {
      const int32_t block = list[entry];
      if (block >= 0 && block <= place.last) {
        const int32_t p = kv_page(a.tok, place, block);
        const int32_t slot = static_cast<int32_t>(key) & ((1 << SHIFT) - 1);
        const int32_t n = place.pos - (block << SHIFT) - slot + 1;
        if (p >= 0 && n > 0) {
          s.page = p;
          float scale[2];
          s.scales(a, head, scale);
          is_open = !s.take(a, scale);
          // (a block before the token's own that has no codes was never filled)
          if (!is_open || block == place.last) {
            s.at = slot * 32 + (n < 16 ? n : 16);
          }
        }
      }
    }
    full = __ballot(s.at != 0 && !is_open);
    open = __ballot(s.at != 0 && is_open);
    return true;
  }
  // The sums of a wave's share taken again, a column at a time, by way of `lds` (16 rows of D) and
  // `ml`, which are the wave's own and free.
  __device__ void alone(const AttendInt8Args& a, int64_t t, int head, int tile, int part, int parts,
                        float* lds, float (&ml)[16][2]) {
    const int lane = lane_id(), col = lane & 15, grp = lane >> 4;
    const int heads = a.G - tile * 16 < 16 ? a.G - tile * 16 : 16;
    AloneSums<E, D, SHIFT> sums;
#pragma unroll 1
    for (int g = 0; g < 16; ++g) {
      if (g < heads) {
        sums.run(a, t, head, static_cast<int64_t>(head) * a.G + tile * 16 + g, part, parts);
      }
#pragma unroll
      for (int r = 0; r < sums.R; ++r) {
        const int d = r * kWave + lane;
        if (d < D) lds[g * D + d] = g < heads ? sums.acc[r] : 0.0f;
      }
      if (lane == 0) {
        ml[g][0] = g < heads ? sums.m : -3.402823466e38f;
        ml[g][1] = g < heads ? sums.l : 0.0f;
      }
    }
    wave_sync_memory();
    this->m[0] = ml[col][0];
    this->l[0] = ml[col][1];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      this->acc[0][i] = *reinterpret_cast<const v4f*>(lds + col * D + 16 * i + 4 * grp);
    }
    wave_sync_memory();
  }
  // `stream`: others do not read these blocks.
  __device__ void run(const AttendInt8Args& a, int64_t t, int head, int tile, int part, int parts,
                      bool stream, char* keys, char* values) {
    this->clear();
    const int g = tile * 16 + (lane_id() & 15), grp = lane_id() >> 4;
    const int64_t hq = head * a.G + g;
    const KvPlace place = kv_place(a.tok, t);
    this->odd[0] = false;
    if (place.last < 0) return;
    const int32_t* list = a.blocks + (t * a.Hkv + head) * a.count;
    {
      typename Kv<E>::V8 q[D / 32];
      Base::fetch_q(a, t, hq, g < a.G, q);
      this->take_q(a, 0, q, g < a.G);
    }
    Subtile s;
    uint64_t full, open;
    for (int chunk = 0; fetch(a, list, place, head, part, parts, chunk, s, full, open); ++chunk) {
      const uint64_t all = full;
      Step then;
      bool counts = false, late_counts = false, more = full != 0;
      auto next = [&] {
        const int i = __builtin_ctzll(full) >> 2;
        full &= ~(uint64_t{15} << (4 * i));
        then = this->step_of(s, i);
        late_counts = (all >> (4 * i + grp)) & 1;
      };
      auto load_k = [&] {
        if (stream) {
          this->template load_k<true>(a, s, head, then.i, keys);
        } else {
          this->template load_k<false>(a, s, head, then.i, keys);
        }
      };
      auto load_v = [&] {
        if (stream) {
          this->template load_v<true>(a, s, head, then.i, values);
        } else {
          this->template load_v<false>(a, s, head, then.i, values);
        }
      };
      if (more) {
        next();
        load_k();
        load_v();
      }
      while (more) {
        const Step now = then;
        counts = late_counts;
        more = full != 0;
        if (more) next();
        const int n[1] = {now.at & 31};
        const bool c[1] = {counts};
        this->step(keys, values, now, c, n, __any(n[0] != 16), more, load_k, load_v);
      }
      while (open != 0) {
        const int i = __builtin_ctzll(open) >> 2, own = 4 * i + grp;
        const int32_t at = __shfl(s.at, own);
        const bool here = (open >> own) & 1;
        open &= ~(uint64_t{15} << (4 * i));
        const int n = here ? at & 31 : 0;
        this->open_step(a, 0, a.tok.seq_ids[t], head, t, hq, g < a.G, here ? at >> 5 : 0, n, n, 1,
                        0);
      }
    }
  }
};

template <class E, int D, int SHIFT>
__global__ void __launch_bounds__(kAttendWaves* kWave, attend_int8_waves(D, SHIFT, 0))
    kv_attend_int8_split_kernel(AttendInt8Args a) {
  __shared__ __attribute__((aligned(16))) char lds[kAttendWaves][64 * D];  // keys, then sums
  __shared__ __attribute__((aligned(16))) char values[kAttendWaves][64 * D];
  __shared__ float ml[kAttendWaves][16][2];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int part = blockIdx.x % a.parts;
  const int64_t row = blockIdx.x / a.parts;  // (token, key/value head, tile)
  const int tile = static_cast<int>(row % a.tiles);
  const int head = static_cast<int>(row / a.tiles % a.Hkv);
  const int64_t t = row / a.tiles / a.Hkv;
  SplitWave<E, D, SHIFT> w;
  // (neighbours of one sequence choose mostly the same blocks: these stay in L2)
  const int32_t seq = a.tok.seq_ids[t];
  const bool beside = (t > 0 && a.tok.seq_ids[t - 1] == seq) ||
                      (t + 1 < a.T && a.tok.seq_ids[t + 1] == seq);
  const int first = part * kAttendWaves + wave, parts = a.parts * kAttendWaves;
  w.run(a, t, head, tile, first, parts, !beside, lds[wave], values[wave]);
  if (__builtin_expect(w.far, 0)) {
    w.alone(late_args(), t, head, tile, first, parts, reinterpret_cast<float*>(values[wave]),
            ml[wave]);
  } else {
    w.finish();
  }
  join_waves<E, D>(a, w.acc[0], w.m[0], w.l[0], t, head, tile, row, part, lds, ml);
}

// Prompts: a workgroup holds the heads of several neighbouring tokens (CT tiles of 16 columns,
// floor(16 / G) tokens each) and passes once over all the blocks that any of them lists, each
// column counting its own: neighbours mostly choose alike, so a block's codes are loaded and
// widened once for them. Its waves take the steps in turn, each with all the columns, and join
// their sums.
//
// The lists are joined by physical page in a hash table in LDS: of a page's entries the first (by
// token, then place) stands for all and holds the tokens' bits; the pages are taken in the order of
// these, so the sums' order depends on the lists alone.
constexpr int kJoinEntries = 512;  // of a workgroup's lists
constexpr int kJoinTable = 2 * kJoinEntries;

template <int D, int CT>
struct JoinInt8Lds {
  union {
    struct {
      int32_t page[kJoinTable];
      uint32_t who[kJoinTable];
      uint32_t first[kJoinTable];
    };
    char keys[kAttendWaves][64 * D];  // then sums
  };
  char values[kAttendWaves][64 * D];
  v8h q[CT > 1 ? CT * (D / 32) * kWave : 1];
  int32_t list[kJoinEntries];
  uint32_t list_who[kJoinEntries];
  int32_t counts[kAttendWaves];
  float ml[kAttendWaves][16][2];
  float column[CT][16][3];  // power, start, odd
};

// The pages of tokens t0 .. t0 + tokens - 1: how many.
template <class Lds>
__device__ inline int join_lists(const AttendInt8Args& a, int64_t t0, int tokens, int head,
                                 Lds& lds) {
  constexpr int THREADS = kAttendWaves * kWave, EACH = kJoinEntries / THREADS;
  const int lane = lane_id(), wave = threadIdx.x / kWave, entries = tokens * a.count;
  int table = 64;
  while (table < 2 * entries) table <<= 1;
  for (int i = threadIdx.x; i < table; i += THREADS) {
    lds.page[i] = -1;
    lds.who[i] = 0u;
    lds.first[i] = ~0u;
  }
  __syncthreads();
  int slot[EACH];
  int32_t page[EACH];
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    const int e = (wave * EACH + r) * kWave + lane;
    page[r] = -1;
    slot[r] = 0;
    if (e < entries) {
      const int tok = e / a.count;
      const KvPlace p = kv_place(a.tok, t0 + tok);
      const int32_t b = a.blocks[((t0 + tok) * a.Hkv + head) * a.count + e % a.count];
      if (b >= 0 && b <= p.last) page[r] = kv_page(a.tok, p, b);
      if (page[r] >= 0) {
        int s = static_cast<int>((static_cast<uint32_t>(page[r]) * 0x9E3779B1u) >> 16) &
                (table - 1);
        for (;;) {  // (at most half full: a free place or the page's own is met)
          const int32_t old = atomicCAS(&lds.page[s], -1, page[r]);
          if (old == -1 || old == page[r]) break;
          s = (s + 1) & (table - 1);
        }
        slot[r] = s;
        atomicOr(&lds.who[s], 1u << tok);
        atomicMin(&lds.first[s], static_cast<uint32_t>(e));
      }
    }
  }
  __syncthreads();
  bool first[EACH];
  int mine = 0;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    const uint32_t e = (wave * EACH + r) * kWave + lane;
    first[r] = page[r] >= 0 && lds.first[slot[r]] == e;
    mine += __popcll(__ballot(first[r]));
  }
  if (lane == 0) lds.counts[wave] = mine;
  __syncthreads();
  int listed = 0, to = 0;
#pragma unroll
  for (int w = 0; w < kAttendWaves; ++w) {
    to += w < wave ? lds.counts[w] : 0;
    listed += lds.counts[w];
  }
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    const uint64_t m = __ballot(first[r]);
    if (first[r]) {
      const int at = to + __popcll(m & ((uint64_t{1} << lane) - 1));
      lds.list[at] = page[r];
      lds.list_who[at] = lds.who[slot[r]];
    }
    to += __popcll(m);
  }
  __syncthreads();  // (the table's place is free)
  return __builtin_amdgcn_readfirstlane(listed);
}

template <class E, int D, int SHIFT, int CT>
__global__ void __launch_bounds__(kAttendWaves* kWave, attend_int8_waves(D, SHIFT, CT))
    kv_attend_int8_joined_kernel(AttendInt8Args a) {
  __shared__ __attribute__((aligned(16))) JoinInt8Lds<D, CT> lds;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = lane_id(), col = lane & 15, grp = lane >> 4;
  const int head = blockIdx.x % a.Hkv;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / a.Hkv) * a.joined;
  const int tokens = a.T - t0 < a.joined ? static_cast<int>(a.T - t0) : a.joined;
  const int listed = join_lists(a, t0, tokens, head, lds);
  const int each = 16 / a.G;  // tokens of a tile
  Int8Wave<E, D, SHIFT, CT> w;
  using V8 = typename Kv<E>::V8;
  w.clear();
  w.q_lds = lds.q;
  bool real[CT];
  int tok[CT], own_keys[CT];
  int32_t own[CT];  // the token's own page, which ends after own_keys
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    tok[c] = c * each + col / a.G;
    real[c] = col / a.G < each && tok[c] < tokens;
    if (!real[c]) tok[c] = 0;
    const KvPlace p = kv_place(a.tok, t0 + tok[c]);
    own[c] = real[c] && p.last >= 0 ? kv_page(a.tok, p, p.last) : -1;
    own_keys[c] = (p.pos & ((1 << SHIFT) - 1)) + 1;
    if constexpr (CT == 1) {
      V8 x[D / 32];
      w.fetch_q(a, t0 + tok[c], head * a.G + col % a.G, real[c], x);
      w.take_q(a, c, x, real[c]);
    }
  }
  if constexpr (CT > 1) {  // a wave a tile, for all
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      if (wave != c) continue;
      V8 x[D / 32];
      w.fetch_q(a, t0 + tok[c], head * a.G + col % a.G, real[c], x);
      w.take_q(a, c, x, real[c], lds.q);
      if (grp == 0) {
        lds.column[c][col][0] = static_cast<float>(w.power[c]);
        lds.column[c][col][1] = w.start[c];
        lds.column[c][col][2] = w.odd[c] ? 1.0f : 0.0f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      w.power[c] = static_cast<int>(lds.column[c][col][0]);
      w.start[c] = lds.column[c][col][1];
      w.odd[c] = lds.column[c][col][2] != 0.0f;
    }
  }
  constexpr int PER = 1 << (SHIFT - 4);  // subtiles of a page
  // Chunks of 16 steps, the waves in turn: lane l has subtile l % 4 of this wave's step l / 4.
  const int steps = (listed * PER + 3) / 4;
  for (int base = wave; base < steps; base += 16 * kAttendWaves) {
    Subtile s;
    s.clear();
    const int i = 4 * (base + kAttendWaves * (lane >> 2)) + (lane & 3);
    bool is_open = false;
    if (i < listed * PER) {
      s.page = lds.list[i / PER];
      s.who = lds.list_who[i / PER];
      s.at = i % PER * 16 * 32 + 16;
      float scale[2];
      s.scales(a, head, scale);
      is_open = !s.take(a, scale);
    }
    // (open pages are their tokens' own or were never filled)
    uint64_t full = __ballot(s.at != 0 && !is_open), open = __ballot(s.at != 0 && is_open);
    const int32_t open_who = is_open ? static_cast<int32_t>(s.who) : 0;
    if (is_open) s.who = 0u;
    Step then;
    bool counts[CT], some = false, more = full != 0;
    int n[CT];
    auto next = [&] {
      const int q = __builtin_ctzll(full) >> 2;
      full &= ~(uint64_t{15} << (4 * q));
      then = w.step_of(s, q);
    };
    // whether each column counts the step's subtile of this lane, and how many of its keys
    auto keys = [&](const Step& x) {
      bool part = false;
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        counts[c] = real[c] && ((x.who >> tok[c]) & 1u) != 0;
        n[c] = 16;
        if (counts[c] && x.page == own[c]) {
          const int left = own_keys[c] - (x.at >> 5);
          n[c] = left < 16 ? left : 16;
          part |= left < 16;
        }
      }
      some = __any(part);
    };
    if (more) {
      next();
      w.template load_k<false>(a, s, head, then.i, lds.keys[wave]);
      w.template load_v<false>(a, s, head, then.i, lds.values[wave]);
    }
    while (more) {
      const Step now = then;
      more = full != 0;
      if (more) next();
      keys(now);
      w.step(lds.keys[wave], lds.values[wave], now, counts, n, some, more,
             [&] { w.template load_k<false>(a, s, head, then.i, lds.keys[wave]); },
             [&] { w.template load_v<false>(a, s, head, then.i, lds.values[wave]); });
    }
    while (open != 0) {  // one page at a time: its sequence's open block
      const int from = __builtin_ctzll(open), q = from >> 2;
      const int32_t page = __builtin_amdgcn_readlane(s.page, from);
      const uint32_t who = __builtin_amdgcn_readlane(open_who, from);
      const int at = 4 * q + grp;
      const int32_t at_page = __shfl(s.page, at), at_slot = __shfl(s.at, at) >> 5;
      const bool here = ((open >> at) & 1) && at_page == page;
      const int first = here ? at_slot : 0;
      open &= ~(__ballot(s.page == page) & (uint64_t{15} << (4 * q)));
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const bool mine = real[c] && own[c] == page && ((who >> tok[c]) & 1u) != 0;
        const int left = own_keys[c] - first, keys_here = mine && here && left > 0 ? left : 0;
        const int nc = keys_here < 16 ? keys_here : 16;
        int most = nc;
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) most = max(most, __shfl_xor(most, x));
        const uint64_t any = __ballot(mine);
        if (any == 0) continue;
        const int one = __builtin_amdgcn_readlane(tok[c], __builtin_ctzll(any));
        w.open_step(a, c, a.tok.seq_ids[t0 + one], head, t0 + tok[c], head * a.G + col % a.G,
                    real[c], first, nc, most, tokens, tok[c]);
      }
    }
  }
  if (lane == 0) lds.counts[wave] = w.far ? 1 : 0;
  __syncthreads();  // (the stages are free)
  int far = 0;
#pragma unroll
  for (int i = 0; i < kAttendWaves; ++i) far |= lds.counts[i];
  if (__builtin_expect(__builtin_amdgcn_readfirstlane(far) != 0, 0)) {  // (the rows one by one)
    const AttendInt8Args& a = late_args();
#pragma unroll 1
    for (int i = wave; i < tokens * a.G; i += kAttendWaves) {
      const int64_t t = t0 + i / a.G, hq = static_cast<int64_t>(head) * a.G + i % a.G;
      AloneSums<E, D, SHIFT> sums;
      sums.run(a, t, head, hq, 0, 1);
      const float inv = inverse_sum(sums.l);
      E* out = static_cast<E*>(a.out) + (t * a.Hq + hq) * D;
#pragma unroll
      for (int r = 0; r < sums.R; ++r) {
        const int d = r * kWave + lane;
        if (d < D) out[d] = static_cast<E>(sums.acc[r] * inv);
      }
      if (lane == 0) a.lse[t * a.Hq + hq] = log_sum(sums.m, sums.l);
    }
    return;
  }
  w.finish();
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    if (c > 0 && c * each >= tokens) continue;
    if (c > 0) __syncthreads();
    join_columns<E, D>(w.acc[c], w.m[c], w.l[c], wave, lds.keys, lds.ml, each * a.G,
                       [&](int g, int ch, float m, float l, v4f sum) {
      typedef E V4 __attribute__((ext_vector_type(4)));
      const int of = c * each + g / a.G;
      if (of >= tokens) return;
      const int64_t row = (t0 + of) * a.Hq + head * a.G + g % a.G;
      const float inv = inverse_sum(l);
      V4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = static_cast<E>(sum[e] * inv);
      *reinterpret_cast<V4*>(static_cast<E*>(a.out) + row * D + ch) = x;
      if (ch == 0) a.lse[row] = log_sum(m, l);
    });
  }
}

// How a call is spread: `parts` workgroups a row; 0: `joined` tokens a workgroup, in
// `tiles` of 16 columns.
struct AttendInt8Plan {
  int64_t rows;
  int32_t tiles, parts, joined;
};

template <class E, int D, int SHIFT>
int attend_int8_launch(const AttendInt8Args& a, const AttendInt8Plan& plan, hipStream_t s) {
  const dim3 threads(kAttendWaves * kWave);
  if (plan.parts == 0) {
    const dim3 grid(static_cast<unsigned>(cdiv(a.T, plan.joined) * a.Hkv));
    if (plan.tiles == 2) {
      kv_attend_int8_joined_kernel<E, D, SHIFT, 2><<<grid, threads, 0, s>>>(a);
    } else {
      kv_attend_int8_joined_kernel<E, D, SHIFT, 1><<<grid, threads, 0, s>>>(a);
    }
  } else {
    const dim3 grid(static_cast<unsigned>(plan.rows * plan.parts));
    kv_attend_int8_split_kernel<E, D, SHIFT><<<grid, threads, 0, s>>>(a);
    if (plan.parts > 1) {
      kv_join_kernel<E, D><<<dim3(static_cast<unsigned>(a.T * a.Hq)), dim3(D / 4), 0, s>>>(a);
    }
  }
  RT_CHECK_HIP(hipGetLastError());
  return kOk;
}

template <class E, int SHIFT>
int attend_int8_dims(int64_t D, const AttendInt8Args& a, const AttendInt8Plan& p, hipStream_t s) {
  switch (D) {
    case 64: return attend_int8_launch<E, 64, SHIFT>(a, p, s);
    case 96: return attend_int8_launch<E, 96, SHIFT>(a, p, s);
    case 128: return attend_int8_launch<E, 128, SHIFT>(a, p, s);
    case 192: return attend_int8_launch<E, 192, SHIFT>(a, p, s);
    default: return attend_int8_launch<E, 256, SHIFT>(a, p, s);
  }
}

// The kernels of a type over pages of 16 and 32, of 64 and 128 slots: a file each.
int attend_int8_bf16_16(int64_t, const AttendInt8Args&, const AttendInt8Plan&, hipStream_t);
int attend_int8_bf16_64(int64_t, const AttendInt8Args&, const AttendInt8Plan&, hipStream_t);
int attend_int8_f16_16(int64_t, const AttendInt8Args&, const AttendInt8Plan&, hipStream_t);
int attend_int8_f16_64(int64_t, const AttendInt8Args&, const AttendInt8Plan&, hipStream_t);

}  // namespace rt
