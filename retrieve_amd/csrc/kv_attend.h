// What attention over a paged cache in 16 and in 8 bits shares: the arguments of a call, and the
// join of a row's parts.
#pragma once

#include "kv_common.h"

namespace rt {

constexpr int kAttendWaves = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttendBase {
  const void* q;
  int64_t q_st, q_sh;
  int64_t T;
  int32_t Hq, Hkv, G, tiles;  // G query heads a key/value head, in tiles of 16
  const int32_t* blocks;  // [T, Hkv, count]
  int32_t count;
  KvTokens tok;
  float scale;      // its magnitude (above 0) times log2 e; the queries carry its sign
  bool minus;
  int32_t parts;    // workgroups that share a row
  int32_t joined;   // tokens a wave takes together
  void* out;        // [T, Hq, D]
  float* lse;       // [T, Hq]
  float* part_out;  // [rows, parts, 16, D], sums of weights times values
  float* part_ml;   // [rows, parts, 16, 2], maxima (powers of two) and sums
};

// 1 / l; 0 for a row without a key; NaN stays.
__device__ inline float inverse_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
__device__ inline float log_sum(float m, float l) {
  return l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

// The sums of the workgroup's waves over the same columns, joined at the largest maximum: f(column,
// first of four channels, maximum, sum of weights, sums). acc: channel 16 i + 4 (lane / 16) + r of
// column lane % 16; `columns` of them count.
template <class E, int D, class F>
__device__ inline void join_columns(const v4f (&acc)[D / 16], float m_wave, float l_wave, int wave,
                                    char (&lds)[kAttendWaves][64 * D],
                                    float (&ml)[kAttendWaves][16][2], int columns, F&& f) {
  // the sums as fp32 rows of a column, 16-byte chunks permuted by the column (bank conflicts)
  const int col = lane_id() & 15, grp = lane_id() >> 4;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    *reinterpret_cast<v4f*>(lds[wave] + col * (D * 4) + (((4 * i + grp) ^ (col & 7)) << 4)) =
        acc[i];
  }
  if (grp == 0) {
    ml[wave][col][0] = m_wave;
    ml[wave][col][1] = l_wave;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < columns * (D / 4); i += kAttendWaves * kWave) {
    const int g = i / (D / 4), c = i % (D / 4);
    float m = ml[0][g][0];
#pragma unroll
    for (int j = 1; j < kAttendWaves; ++j) m = fmaxf(m, ml[j][g][0]);
    float l = 0.0f;
    v4f sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kAttendWaves; ++j) {
      const float x = __builtin_amdgcn_exp2f(ml[j][g][0] - m);
      l += x * ml[j][g][1];
      sum += x * *reinterpret_cast<const v4f*>(lds[j] + g * (D * 4) + ((c ^ (g & 7)) << 4));
    }
    f(g, 4 * c, m, l, sum);
  }
}

// A row's sums of the workgroup's waves: to the outputs where one workgroup has the whole row, else
// to the row's parts.
template <class E, int D>
__device__ inline void join_waves(const AttendBase& a, const v4f (&acc)[D / 16], float m_wave,
                                  float l_wave, int64_t t, int head, int tile, int64_t row,
                                  int part, char (&lds)[kAttendWaves][64 * D],
                                  float (&ml)[kAttendWaves][16][2]) {
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int heads = a.G - tile * 16 < 16 ? a.G - tile * 16 : 16;
  join_columns<E, D>(acc, m_wave, l_wave, wave, lds, ml, heads,
                     [&](int g, int ch, float m, float l, v4f sum) {
    if (a.parts == 1) {
      typedef E V4 __attribute__((ext_vector_type(4)));
      const int64_t r = t * a.Hq + head * a.G + tile * 16 + g;
      const float inv = inverse_sum(l);
      V4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = static_cast<E>(sum[e] * inv);
      *reinterpret_cast<V4*>(static_cast<E*>(a.out) + r * D + ch) = x;
      if (ch == 0) a.lse[r] = log_sum(m, l);
    } else {
      const int64_t r = (row * a.parts + part) * 16 + g;
      *reinterpret_cast<v4f*>(a.part_out + r * D + ch) = sum;
      if (ch == 0) {
        a.part_ml[2 * r] = m;
        a.part_ml[2 * r + 1] = l;
      }
    }
  });
}

// The parts of a row joined at their largest maximum, in order: a thread has 4 channels of a head.
template <class E, int D>
__global__ void __launch_bounds__(D / 4) kv_join_kernel(AttendBase a) {
  typedef E V4 __attribute__((ext_vector_type(4)));
  const int64_t r = blockIdx.x;  // (token, query head)
  const int64_t t = r / a.Hq;
  const int hq = static_cast<int>(r % a.Hq), head = hq / a.G, g = hq % a.G;
  const int64_t row = (t * a.Hkv + head) * a.tiles + g / 16;
  const int64_t first = row * a.parts * 16 + g % 16;
  float m = a.part_ml[2 * first];
#pragma unroll 8
  for (int p = 1; p < a.parts; ++p) m = fmaxf(m, a.part_ml[2 * (first + 16 * p)]);
  float l = 0.0f;
  v4f sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int p = 0; p < a.parts; ++p) {
    const int64_t at = first + 16 * p;
    const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * at] - m);
    l += f * a.part_ml[2 * at + 1];
    sum += f * *reinterpret_cast<const v4f*>(a.part_out + at * D + 4 * threadIdx.x);
  }
  const float inv = inverse_sum(l);
  V4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = static_cast<E>(sum[e] * inv);
  *reinterpret_cast<V4*>(static_cast<E*>(a.out) + r * D + 4 * threadIdx.x) = x;
  if (threadIdx.x == 0) a.lse[r] = log_sum(m, l);
}

}  // namespace rt
