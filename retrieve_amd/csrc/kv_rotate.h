// The rotary position, and the norm before it, of one row's chunks of 8 channels: what the paged
// cache's appending kernels apply to queries and keys on their way.
//
// Norm: y = x r w with r = 1 / sqrt(mean(x^2) + eps). The sum runs in 64 bits (where the squares of
// 16-bit numbers are exact), r is rounded once to fp32 and each of the two products once more.
// Every kernel of the 8-bit cache adds in one order (Pair's), so a block's codes do not depend on
// how its tokens were split over calls. The 16-bit append's rows and bounds add in two orders:
// their sums may differ in the last of 53 bits, which the rounding to 24 almost never shows (where
// it does, a bound may be a key's neighbour in 16 bits).
//
// Rotation: with (c, s) the table's cosine and sine of the token's position, a pair of channels
// (a, b) becomes (a c - b s, b c + a s), every product and sum rounded once to fp32 (no fused
// multiply-add), then to 16 bits. Between the norm and the rotation nothing is rounded to 16 bits.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "kv_common.h"

namespace rt {

// Weights of a head's channels, null for no norm; `wide`: fp32, else of the rows' type.
struct HeadNorm {
  const void* weight;
  bool wide;
};

struct TurnArgs {
  const float* cos_sin;  // [table_len, rot], rot / 2 cosines then rot / 2 sines
  int32_t table_len, rot;
  HeadNorm norm[2];  // of queries, of keys
  double eps;
};

// How channel i meets its partner: halves of the rotated part with every half on whole chunks,
// the same with other halves, or neighbouring channels.
enum RotMode : int { kRotHalf = 0, kRotHalfOdd = 1, kRotPairs = 2 };

__device__ inline float rot_first(float a, float b, float c, float s) {
#pragma clang fp contract(off)
  return a * c - b * s;
}
__device__ inline float rot_second(float b, float a, float c, float s) {
#pragma clang fp contract(off)
  return b * c + a * s;
}

// The cosines and sines of a chunk's channels at a position (1, 0 past the rotated part);
// neighbours that turn together share theirs.
template <int MODE>
struct Turn {
  static constexpr int N = MODE == kRotPairs ? 4 : 8;
  float c[N], s[N];
  __device__ float cos(int e) const { return c[MODE == kRotPairs ? e >> 1 : e]; }
  __device__ float sin(int e) const { return s[MODE == kRotPairs ? e >> 1 : e]; }
  __device__ void load(const TurnArgs& a, int32_t pos, int chunk) {
    const int half = a.rot >> 1;
    const float* row = a.cos_sin + static_cast<int64_t>(pos) * a.rot;
    if ((MODE == kRotHalf || (MODE == kRotPairs && a.rot % 8 == 0)) && 8 * chunk < a.rot) {
      const int j = MODE == kRotPairs ? 4 * chunk : 8 * chunk < half ? 8 * chunk : 8 * chunk - half;
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const v4f cv = *reinterpret_cast<const v4f*>(row + j + e);
        const v4f sv = *reinterpret_cast<const v4f*>(row + half + j + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          c[e + i] = cv[i];
          s[e + i] = sv[i];
        }
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int i = MODE == kRotPairs ? 8 * chunk + 2 * e : 8 * chunk + e;
      const int j = MODE == kRotPairs ? i >> 1 : i < half ? i : i - half;
      c[e] = i < a.rot ? row[j] : 1.0f;
      s[e] = i < a.rot ? row[half + j] : 0.0f;
    }
  }
};

// The weights of a chunk's channels (1 where there are none).
template <class E>
struct Weights {
  float w[8];
  __device__ void load(const HeadNorm& n, int chunk) {
    if (n.weight == nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.0f;
    } else if (n.wide) {
      const v4f* p = static_cast<const v4f*>(n.weight) + 2 * chunk;
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = p[e >> 2][e & 3];
    } else {
      const typename Kv<E>::V8 x = static_cast<const typename Kv<E>::V8*>(n.weight)[chunk];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = static_cast<float>(x[e]);
    }
  }
  __device__ static float at(const HeadNorm& n, int i) {
    return n.weight == nullptr ? 1.0f
           : n.wide            ? static_cast<const float*>(n.weight)[i]
                               : static_cast<float>(static_cast<const E*>(n.weight)[i]);
  }
};

// r of a row of D channels that C neighbouring lanes of a wave hold, N chunks a lane; this is lane
// `part` of them. C is 1 or 3 times a power of two, and the first of them starts on that power.
template <class E, int D, int C, int N>
__device__ inline float row_scale(const typename Kv<E>::V8 (&x)[N], int part, double eps) {
  constexpr int P = C & -C;
  static_assert(C == P || C == 3 * P, "lanes of a row");
  double sum = 0.0;
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double f = static_cast<double>(static_cast<float>(x[n][e]));
      sum = __builtin_fma(f, f, sum);
    }
  }
#pragma unroll
  for (int i = 1; i < P; i <<= 1) sum += __shfl_xor(sum, i);
  if constexpr (C == 3 * P) {
    const int base = lane_id() - part;
    sum = (__shfl(sum, base) + __shfl(sum, base + P)) + __shfl(sum, base + 2 * P);
  }
  // 1 / sqrt by two Newton steps on the instruction's 23 bits (a division and a root in 64 bits
  // take 45 instructions); infinite and 0 (of 0 and of an infinity) as it gives them.
  const double mean = sum * (1.0 / D) + eps;
  double y = __builtin_amdgcn_rsq(mean);
  if (y > 0.0 && y < INFINITY) {
#pragma unroll
    for (int i = 0; i < 2; ++i) y = __builtin_fma(0.5 * y, __builtin_fma(-mean * y, y, 1.0), y);
  }
  return static_cast<float>(y);
}

// Chunk `chunk` of a row, read as x, after the norm (r and the chunk's weights; NORM only) and the
// rotation.
template <class E, int MODE, bool NORM>
__device__ inline typename Kv<E>::V8 turned_chunk(const E* row, typename Kv<E>::V8 x, int chunk,
                                                  const Turn<MODE>& t, const TurnArgs& a,
                                                  const HeadNorm& norm, float r,
                                                  const Weights<E>& w) {
  using V8 = typename Kv<E>::V8;
  if (!NORM && 8 * chunk >= a.rot) return x;
  float own[8], other[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    own[e] = static_cast<float>(x[e]);
    if (NORM) own[e] = own[e] * r * w.w[e];
  }
  V8 out;
  if (NORM && 8 * chunk >= a.rot) {
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = static_cast<E>(own[e]);
    return out;
  }
  const int half = a.rot >> 1;
  if (MODE == kRotPairs) {
#pragma unroll
    for (int e = 0; e < 8; ++e) other[e] = own[e ^ 1];
  } else if (MODE == kRotHalf) {
    const int at = 8 * chunk < half ? 8 * chunk + half : 8 * chunk - half;
    const V8 y = *reinterpret_cast<const V8*>(row + at);
    Weights<E> v;
    if (NORM) v.load(norm, at / 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      other[e] = static_cast<float>(y[e]);
      if (NORM) other[e] = other[e] * r * v.w[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = 8 * chunk + e, at = i < half ? i + half : i - half;
      other[e] = i < a.rot ? static_cast<float>(row[at]) : 0.0f;
      if (NORM && i < a.rot) other[e] = other[e] * r * Weights<E>::at(norm, at);
    }
  }
  if (MODE == kRotPairs && 8 * chunk + 8 <= a.rot) {  // (the whole chunk turns)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      out[e] = static_cast<E>(rot_first(own[e], own[e + 1], t.cos(e), t.sin(e)));
      out[e + 1] = static_cast<E>(rot_second(own[e + 1], own[e], t.cos(e), t.sin(e)));
    }
    return out;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = 8 * chunk + e;
    const bool first = MODE == kRotPairs ? (e & 1) == 0 : i < half;
    const float z = first ? rot_first(own[e], other[e], t.cos(e), t.sin(e))
                          : rot_second(own[e], other[e], t.cos(e), t.sin(e));
    out[e] = i < a.rot ? static_cast<E>(z) : NORM ? static_cast<E>(own[e]) : x[e];
  }
  return out;
}

// A lane's two chunks of a row, what turns them and the norms' weights. Split halves: partners in
// the rotated part, neighbours' distance apart in the rest; otherwise the same place in either half
// of the row.
template <class E, int D, int MODE, bool NORM>
struct Pair {
  using V8 = typename Kv<E>::V8;
  static constexpr int C = D / 16;
  int part, chunk[2];
  Turn<MODE> turn[MODE == kRotHalf ? 1 : 2];
  bool turned;  // split halves: in the rotated part
  Weights<E> weights[NORM ? 2 : 1][2];  // of queries, of keys

  Pair() = default;
  __device__ Pair(const TurnArgs& a, int lane) {
    const int r = a.rot / 16;
    part = lane;
    turned = lane < r;
    if (MODE == kRotHalf) {
      chunk[0] = turned ? lane : lane + r;
      chunk[1] = turned ? lane + r : lane + C;
    } else {
      chunk[0] = lane;
      chunk[1] = lane + C;
    }
  }
  __device__ void load(const TurnArgs& a, int32_t pos) {
    load_turn(a, pos);
    load_weights(a, 0);
    load_weights(a, 1);
  }
  __device__ void load_turn(const TurnArgs& a, int32_t pos) {
    if (a.rot > 0) {
      turn[0].load(a, pos, chunk[0]);
      if constexpr (MODE != kRotHalf) turn[1].load(a, pos, chunk[1]);
    }
  }
  __device__ void load_weights(const TurnArgs& a, int kind) {
    if constexpr (NORM) {
#pragma unroll
      for (int j = 0; j < 2; ++j) weights[kind][j].load(a.norm[kind], chunk[j]);
    }
  }
  // x: the two chunks as read, of a query (kind 0) or a key (1); `row` for partners elsewhere
  __device__ void apply(const E* row, const TurnArgs& a, int kind, V8 (&x)[2]) const {
    float r = 1.0f;
    if constexpr (NORM) {
      r = row_scale<E, D, C>(x, part, a.eps);
      if ((kind ? a.norm[1] : a.norm[0]).weight == nullptr) r = 1.0f;
    }
    if constexpr (MODE == kRotHalf) {
      if (!NORM && !turned) return;
      float f[8], s[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = static_cast<float>(x[0][e]);
        s[e] = static_cast<float>(x[1][e]);
        if constexpr (NORM) {
          f[e] = f[e] * r * (kind ? weights[1][0].w[e] : weights[0][0].w[e]);
          s[e] = s[e] * r * (kind ? weights[1][1].w[e] : weights[0][1].w[e]);
        }
      }
      if (turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[0][e] = static_cast<E>(rot_first(f[e], s[e], turn[0].c[e], turn[0].s[e]));
          x[1][e] = static_cast<E>(rot_second(s[e], f[e], turn[0].c[e], turn[0].s[e]));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[0][e] = static_cast<E>(f[e]);
          x[1][e] = static_cast<E>(s[e]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        Weights<E> w;
        if constexpr (NORM) {
#pragma unroll
          for (int e = 0; e < 8; ++e) w.w[e] = kind ? weights[1][i].w[e] : weights[0][i].w[e];
        }
        x[i] = turned_chunk<E, MODE, NORM>(row, x[i], chunk[i], turn[i], a,
                                           kind ? a.norm[1] : a.norm[0], r, w);
      }
    }
  }
};

// Host: the checks of the table and the weights (of their pointers where there are tokens).
inline int kv_check_turn(int64_t T, int64_t D, const float* cos_sin, int64_t table_len, int64_t rot,
                         const void* q_weight, const void* k_weight, double eps) {
  RT_CHECK_ARG(rot >= 0 && rot % 2 == 0 && rot <= D, "the rotated part must be even, at most %lld",
               static_cast<long long>(D));
  RT_CHECK_ARG(table_len >= 0 && table_len <= INT32_MAX, "the rotary table has too many rows");
  RT_CHECK_ARG(eps >= 0.0 && eps <= 1.7e308, "eps must be finite and not negative, got %g", eps);
  if (T == 0) return kOk;
  RT_CHECK_ARG(rot == 0 || table_len == 0 || cos_sin, "null pointer");
  for (const void* p : {static_cast<const void*>(cos_sin), q_weight, k_weight}) {
    RT_CHECK_ARG(reinterpret_cast<uintptr_t>(p) % 16 == 0,
                 "the rotary table and the norms' weights must start on 16 bytes");
  }
  return kOk;
}
inline TurnArgs kv_turn_args(const float* cos_sin, int64_t table_len, int64_t rot,
                             const void* q_weight, const void* k_weight, int wide, double eps) {
  return {cos_sin, static_cast<int32_t>(table_len), static_cast<int32_t>(rot),
          {{q_weight, wide != 0}, {k_weight, wide != 0}}, eps};
}

// Calls f with the rotation's layout and whether heads are normed as compile-time numbers.
template <class F>
int kv_turn_dispatch(int64_t rot, bool interleaved, bool norm, F&& f) {
  auto by_mode = [&](auto n) {
    if (interleaved) return f(std::integral_constant<int, kRotPairs>{}, n);
    return rot % 16 == 0 ? f(std::integral_constant<int, kRotHalf>{}, n)
                         : f(std::integral_constant<int, kRotHalfOdd>{}, n);
  };
  return norm ? by_mode(std::true_type{}) : by_mode(std::false_type{});
}

}  // namespace rt
