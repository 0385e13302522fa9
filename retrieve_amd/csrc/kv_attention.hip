// Softmax attention of each token over the blocks chosen for it and its key/value head.
//
// out = sum_j exp(x_j - m) v_j / l over the keys j of the listed blocks at positions up to the
// token's, with x_j = scale q . k_j, m their maximum and l the sum of the weights, kept running
// over one pass; lse = m + log l. Rows without a key: 0 and -inf.
//
// A wave holds up to 16 query heads of one key/value head (the heads that share it: its keys and
// values are read once for all of them) and takes 32 keys a step:
//   S^T [keys x heads] = K Q^T   K's rows straight from memory in the operand's layout (a lane has
//                                16 bytes of one key), Q^T in registers throughout;
//   O^T [channels x heads] += V^T P^T   the weights are where the first product left them (lane l:
//                                head l % 16, keys 4 (l / 16) + r of each 16), so P^T needs no
//                                exchange; V is staged through the wave's own LDS, swizzled, and
//                                read transposed (ds_read_tr: 4 keys of one channel a lane).
// A lane's column is one head in both products: maxima, sums and rescaling stay in the lane. The
// maximum is raised only where a score passes it by 8 (in powers of two: weights reach 256 at
// most, far inside both types), so most steps do not touch the accumulators or exchange lanes. A
// score and its maximum meet in one fused multiply-add; of scores past 2^23, where that would
// differ from the rounded maximum by whole powers of two, each is rounded first (`far`).
// Weights are rounded to the values' 16 bits for the matrix cores (l sums them unrounded):
// relative 2^-9 / 2^-12 a weight, the size of the output's own rounding (against 64 bits the
// outputs are off by 2.3e-3 / 2.9e-4 of their size, by 1.7e-3 / 2.1e-4 with weights of 32 bits).
// fp16's step is absolute below 2^-14, so its weights are held 2^5 times as large (m is 5 below the
// maximum; they reach 2^13): at most 2^-30 of the row's largest weight a key, half an output's
// rounding over 2^17 keys.
//
// Memory: a wave keeps the next step's keys and values in flight (registers) while it works on
// this one. Slots past the token's position are read but replaced: scores by -inf, values by 0.
// Single tokens are bound by the cache's bytes: 64 sequences of lists of 64 blocks, 64 keys of 128
// channels a block, 8 key/value heads take 158 us (6.6 TB/s). Prompts read most blocks from L2 and
// are bound by the steps' instructions (2053 tokens of 32 heads over 16 blocks: 136 us).
#include <cmath>
#include <type_traits>

#include "../../include/retrieve_amd.h"
#include "kv_attend.h"
#include "lds_load.h"

namespace rt {

struct AttendArgs : AttendBase {
  const void *k_cache, *v_cache;
};

template <class E>
struct AttendOp;
template <>
struct AttendOp<__bf16> {
  using V8 = Kv<__bf16>::V8;
  typedef __bf16 V4 __attribute__((ext_vector_type(4)));
  __device__ static v4f mma(V8 a, V8 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static V4 read_tr(const char* lds) {
    typedef __attribute__((address_space(3))) V4 LdsV4;
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LdsV4*)lds);
  }
};
template <>
struct AttendOp<_Float16> {
  using V8 = Kv<_Float16>::V8;
  typedef _Float16 V4 __attribute__((ext_vector_type(4)));
  __device__ static v4f mma(V8 a, V8 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ static V4 read_tr(const char* lds) {
    typedef __fp16 Raw __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) Raw LdsRaw;
    return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((LdsRaw*)lds));
  }
};

// The staged values: 32 rows of D channels; the 32-byte granules of a row are permuted by the row
// so that the 16 rows a transposed read takes at one channel lie in different banks.
template <int D>
__device__ inline int granule_swizzle(int row) {
  return D % 128 == 0 ? row & 7 : D % 64 == 0 ? (row >> 1) & 3 : (row >> 2) & 1;
}

// A step's two tiles of 16 keys: their first rows in the caches and how many keys count.
struct Tiles {
  int64_t row[2];
  int n[2];
};

// The tiles of one wave: of a row's list in units of 64 keys, units part, part + parts, ... A chunk
// of 16 units is looked up at a time, one tile a lane; steps (two neighbouring tiles) without keys
// are left out.
struct TileList {
  const int32_t* list;
  KvPlace place;
  int32_t head, part, parts, chunk;
  uint64_t left;  // tiles of this chunk with keys to come
  int32_t page, at;  // this lane's: physical page, first slot * 32 + keys

  __device__ void fetch(const AttendArgs& a) {
    const int64_t unit = part + static_cast<int64_t>(parts) * (16 * chunk + (lane_id() >> 2));
    const int64_t key = unit * 64 + 16 * (lane_id() & 3);
    const int64_t entry = key >> a.tok.shift;
    page = 0;
    at = 0;
    if (entry < a.count) {
      const int32_t block = list[entry];
      if (block >= 0 && block <= place.last) {
        const int32_t p = kv_page(a.tok, place, block);
        const int32_t slot = static_cast<int32_t>(key) & ((1 << a.tok.shift) - 1);
        const int32_t n = place.pos - (block << a.tok.shift) - slot + 1;
        if (p >= 0 && n > 0) {
          page = p;
          at = slot * 32 + (n < 16 ? n : 16);
        }
      }
    }
    left = __ballot(at != 0);
  }
  __device__ bool next(const AttendArgs& a, Tiles& s) {
    while (left == 0) {
      ++chunk;
      const int64_t first = (part + static_cast<int64_t>(parts) * 16 * chunk) * 64;
      if (first >= static_cast<int64_t>(a.count) << a.tok.shift) return false;
      fetch(a);
    }
    const int i = __builtin_ctzll(left) & ~1;
    left &= ~(uint64_t{3} << i);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int32_t p = __builtin_amdgcn_readlane(page, i + j);
      const int32_t x = __builtin_amdgcn_readlane(at, i + j);
      s.row[j] = ((static_cast<int64_t>(p) * a.Hkv + head) << a.tok.shift) + (x >> 5);
      s.n[j] = x & 31;
    }
    return true;
  }
};

// Sixteen bytes of a cache; STREAM: of rows that are read once (not kept in L2 before others: 64
// sequences of 64 blocks 168 us, 187 with ordinary loads; 400 tokens of prompts, split, which share
// blocks, 157 us streamed and 121 with ordinary loads).
template <bool STREAM, class V>
__device__ inline V load_row(const V* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  return *p;
}

// A wave's accumulators (channel 16 i + 4 (lane / 16) + r of column lane % 16), the columns' maxima
// (less kLift) and this lane's share of their sums; its queries and the step in flight.
template <class E, int D>
struct AttendWave {
  using Op = AttendOp<E>;
  using V8 = typename Op::V8;
  static constexpr int KS = D / 32, DT = D / 16, VL = D / 16;  // VL: 16-byte loads of V a lane
  static constexpr float kLift = std::is_same<E, _Float16>::value ? 5.0f : 0.0f;  // maximum - m
  static constexpr float kFar = 0x1p23f;
  v4f acc[DT];
  float m, l;
  bool far;  // a maximum has been past kFar, in some column
  V8 qf[KS], kf[2][KS], vf[VL];

  __device__ void clear() {
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
    m = -3.402823466e38f;
    l = 0.0f;
    far = false;
  }
  // This lane's column is query head `head` of token t (zeros where it is not `real`).
  __device__ void load_q(const AttendArgs& a, int64_t t, int64_t head, bool real) {
    const E* q = static_cast<const E*>(a.q) + (real ? t * a.q_st + head * a.q_sh : 0) +
                 8 * (lane_id() >> 4);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const V8 x = *reinterpret_cast<const V8*>(q + 32 * s);
      qf[s] = real ? (a.minus ? -x : x) : V8{};
    }
  }
  template <bool STREAM>
  __device__ void load_k(const AttendArgs& a, const Tiles& s) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const E* base = static_cast<const E*>(a.k_cache) + s.row[j] * D;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        kf[j][i] = load_row<STREAM>(reinterpret_cast<const V8*>(
            base + ((lane_id() & 15) * D + 8 * (lane_id() >> 4) + 32 * i)));
      }
    }
  }
  template <bool STREAM>
  __device__ void load_v(const AttendArgs& a, const Tiles& s) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const E* base = static_cast<const E*>(a.v_cache) + s.row[j] * D;
#pragma unroll
      for (int i = 0; i < VL / 2; ++i) {
        vf[j * (VL / 2) + i] =
            load_row<STREAM>(reinterpret_cast<const V8*>(base + (i * 64 + lane_id()) * 8));
      }
    }
  }
  // One step on what load_k and load_v brought; `fetch_k` and `fetch_v` start the next one's loads
  // as soon as the registers are free. A column's keys count up to n[j] in tile j; V's rows from
  // rows[j] on are read as zeros (slots that may never have been written).
  template <class FK, class FV>
  __device__ void step(const AttendArgs& a, char* lds, bool whole, const int (&n)[2],
                       const int (&rows)[2], FK&& fetch_k, FV&& fetch_v) {
    const int lane = lane_id();
    v4f sc[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sc[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; ++i) sc[j] = Op::mma(kf[j][i], qf[i], sc[j]);
    }
    fetch_k();
    if (rows[0] < 16 || rows[1] < 16) {
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int row = ((i % (VL / 2)) * 64 + lane) / (D / 8);
        if (row >= rows[i / (VL / 2)]) vf[i] = V8{};
      }
    }
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int at = i * 64 + lane, row = at / (D / 8), c = at % (D / 8);
      *reinterpret_cast<V8*>(lds + row * (D * 2) + (((c >> 1) ^ granule_swizzle<D>(row)) << 5) +
                             (c & 1) * 16) = vf[i];
    }
    fetch_v();
    V8 p[1];
    weigh<false>(a.scale, sc, whole, n, p);
    asm volatile("" ::: "memory");  // (the staged rows are read by other lanes of this wave)
    add(lds, p);
    asm volatile("" ::: "memory");
  }
  __device__ static float rounded(float x, float scale) {
#pragma clang fp contract(off)
    return x * scale;
  }
  // The weights of the scores of N tiles (key 4 (lane / 16) + r of tile j at 4 (j % 2) + r of p[j /
  // 2]), rounded for the second product; the maximum raised and the sum extended. A column counts
  // the first n[j] keys of tile j (all where `whole`). ALONE: far scores make the sums no
  // numbers (the caller takes such rows alone).
  template <bool ALONE, int N>
  __device__ void weigh(float scale, v4f (&sc)[N], bool whole, const int (&n)[N],
                        V8 (&p)[N / 2]) {
    settle(sc);
    if (!whole) {
      const int at = 4 * (lane_id() >> 4);
#pragma unroll
      for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[j][r] = at + r < n[j] ? sc[j][r] : -INFINITY;
      }
    }
    float top[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      top[j] = fmaxf(fmaxf(sc[j][0], sc[j][1]), fmaxf(sc[j][2], sc[j][3]));
    }
#pragma unroll
    for (int j = 1; j < N; ++j) top[0] = fmaxf(top[0], top[j]);
    const float high = top[0] * scale;
    if (__any(high - m > 8.0f + kLift)) {
      const bool is_far = __any(fabsf(high) > kFar && high != -INFINITY);
      if (ALONE) {
        if (is_far) acc[0][0] = NAN;
      } else {
        far |= is_far;
      }
      float next = fmaxf(high, __shfl_xor(high, 16));
      next = fmaxf(next, __shfl_xor(next, 32));
      next = fmaxf(next - kLift, m);
      const float keep = __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= keep;
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] *= keep;
    }
    float sum[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float t[4], e[4];
      if (!ALONE && far) {  // (rounded first, as the maximum is)
#pragma unroll
        for (int r = 0; r < 4; ++r) t[r] = rounded(sc[j][r], scale) - m;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) t[r] = fmaf(sc[j][r], scale, -m);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        e[r] = __builtin_amdgcn_exp2f(t[r]);
        p[j / 2][4 * (j % 2) + r] = static_cast<E>(e[r]);
      }
      sum[j] = (e[0] + e[1]) + (e[2] + e[3]);
    }
#pragma unroll
    for (int j = 0; j < N; j += 2) l += sum[j] + sum[j + 1];
  }
  // The second product: 32 N staged rows of values, swizzled by granules.
  template <int N>
  __device__ void add(const char* lds, const V8 (&p)[N]) {
    const int col = lane_id() & 15, grp = lane_id() >> 4;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
#pragma unroll
      for (int h = 0; h < N; ++h) {
        typename Op::V4 x[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = 16 * j + 4 * grp + (col >> 2);
          x[j] = Op::read_tr(lds + (32 * h + row) * (D * 2) +
                             ((i ^ granule_swizzle<D>(row)) << 5) + (col & 3) * 8);
        }
        const V8 v = {x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
        acc[i] = Op::mma(v, p[h], acc[i]);
      }
    }
  }
  __device__ void join_sums() {
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
  }

  // One token's heads (tile `tile` of the group) over part of its list.
  template <bool STREAM>
  __device__ void run(const AttendArgs& a, int64_t t, int head, int tile, int part, int parts,
                      char* lds) {
    clear();
    TileList tiles;
    tiles.place = kv_place(a.tok, t);
    if (tiles.place.last < 0) return;
    tiles.list = a.blocks + (t * a.Hkv + head) * a.count;
    tiles.head = head;
    tiles.part = part;
    tiles.parts = parts;
    tiles.chunk = -1;
    tiles.left = 0;
    const int g = tile * 16 + (lane_id() & 15);
    load_q(a, t, head * a.G + g, g < a.G);
    Tiles now, then;
    bool more = tiles.next(a, then);
    if (more) {
      load_k<STREAM>(a, then);
      load_v<STREAM>(a, then);
    }
    while (more) {
      now = then;
      more = tiles.next(a, then);
      step(a, lds, now.n[0] == 16 && now.n[1] == 16, now.n, now.n,
           [&] { if (more) load_k<STREAM>(a, then); },
           [&] { if (more) load_v<STREAM>(a, then); });
    }
    join_sums();
  }
};

// This lane's column, query head `head` of token t, to the outputs.
template <class E, int D>
__device__ inline void emit(const AttendArgs& a, const AttendWave<E, D>& w, int64_t t, int head) {
  typedef E V4 __attribute__((ext_vector_type(4)));
  const int grp = lane_id() >> 4;
  const int64_t row = t * a.Hq + head;
  const float inv = inverse_sum(w.l);
  E* out = static_cast<E*>(a.out) + row * D + 4 * grp;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    V4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = static_cast<E>(w.acc[i][r] * inv);
    *reinterpret_cast<V4*>(out + 16 * i) = x;
  }
  if (grp == 0) a.lse[row] = log_sum(w.m, w.l);
}

// Many rows (from 4096, when the GPU holds no more waves): a wave a row, four neighbouring tokens
// of one head a workgroup (they mostly choose the same blocks). For groups of more than 8 heads,
// which fill the columns of a wave by themselves, and lists too long to be joined.
template <class E, int D>
__global__ void __launch_bounds__(kAttendWaves* kWave, D <= 128 ? 2 : 1)
    kv_attend_rows_kernel(AttendArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[kAttendWaves][64 * D];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int heads = a.Hkv * a.tiles;
  const int64_t t = static_cast<int64_t>(blockIdx.x / heads) * kAttendWaves + wave;
  if (t >= a.T) return;
  const int head = blockIdx.x % heads / a.tiles, tile = blockIdx.x % heads % a.tiles;
  AttendWave<E, D> w;
  w.template run<false>(a, t, head, tile, 0, 1, lds[wave]);
  const int g = tile * 16 + (lane_id() & 15);
  if (g < a.G) emit(a, w, t, head * a.G + g);
}

// One query head of one token by a wave, key by key (a lane scores one of 64, then sums its own
// channels): only for rows beside values that are not finite or of far scores, so it spares
// registers, not time.
template <class E, int D>
__device__ inline void attend_alone(const AttendArgs& a, int64_t t, int head, int hq, float* qs) {
  using V8 = typename Kv<E>::V8;
  constexpr int R = (D + kWave - 1) / kWave;
  const int lane = lane_id();
  const KvPlace p = kv_place(a.tok, t);
  const E* q = static_cast<const E*>(a.q) + t * a.q_st + hq * a.q_sh;
  // (a scale above 1 behind the product: a query may be large beside small keys)
  const float below = fminf(a.scale, 1.0f), above = fmaxf(a.scale, 1.0f);
  const float scale = a.minus ? -below : below;
  for (int d = lane; d < D; d += kWave) qs[d] = static_cast<float>(q[d]) * scale;
  asm volatile("" ::: "memory");
  const int size = 1 << a.tok.shift;
  float m = -3.402823466e38f, l = 0.0f, acc[R] = {};
  for (int i = 0; i < a.count; ++i) {
    const int32_t block = a.blocks[(t * a.Hkv + head) * a.count + i];
    if (block < 0 || block > p.last) continue;
    const int32_t page = kv_page(a.tok, p, block);
    if (page < 0) continue;
    const int64_t base = ((static_cast<int64_t>(page) * a.Hkv + head) << a.tok.shift) * D;
    const int keys = block == p.last ? (p.pos & (size - 1)) + 1 : size;
    for (int j0 = 0; j0 < keys; j0 += kWave) {
      const int j = j0 + lane;
      float x = -INFINITY;
      if (j < keys) {
        const E* k = static_cast<const E*>(a.k_cache) + base + j * D;
        x = 0.0f;
#pragma unroll 2
        for (int d = 0; d < D; d += 8) {
          const V8 kv = *reinterpret_cast<const V8*>(k + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) x = fmaf(static_cast<float>(kv[e]), qs[d + e], x);
        }
        x *= above;
      }
      float top = x;
      for (int s = 1; s < kWave; s <<= 1) top = fmaxf(top, __shfl_xor(top, s));
      const float next = fmaxf(m, top), keep = __builtin_amdgcn_exp2f(m - next);
      const float w = __builtin_amdgcn_exp2f(x - next);
      float sum = w;
      for (int s = 1; s < kWave; s <<= 1) sum += __shfl_xor(sum, s);
      l = l * keep + sum;
      m = next;
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r] *= keep;
      const int n = keys - j0 < kWave ? keys - j0 : kWave;
      for (int jj = 0; jj < n; ++jj) {
        const float wj = __shfl(w, jj);
        const E* v = static_cast<const E*>(a.v_cache) + base + (j0 + jj) * D;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int d = r * kWave + lane;
          if (d < D) acc[r] = fmaf(wj, static_cast<float>(v[d]), acc[r]);
        }
      }
    }
  }
  const float inv = inverse_sum(l);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int d = r * kWave + lane;
    if (d < D) static_cast<E*>(a.out)[(t * a.Hq + hq) * D + d] = static_cast<E>(acc[r] * inv);
  }
  if (lane == 0) a.lse[t * a.Hq + hq] = log_sum(m, l);
  asm volatile("" ::: "memory");
}

// Many tokens whose group has 8 heads or fewer: a wave holds the heads of several neighbouring
// tokens (columns that one token would leave empty), a workgroup four such waves, and passes once
// over all the blocks that any of their tokens lists, each column counting its own. Neighbours
// mostly choose alike, so a block is read once for them; a wave sits out the blocks that none
// of its tokens lists.
//
// The lists are joined by physical page in a hash table: of a page's entries the first (by token,
// then place) stands for all and holds the tokens' bits; they are taken in the order of their
// blocks, so it depends on the lists alone. Keys and values go straight to LDS, a step of 32 keys
// ahead of the one in work, each wave loading one of a step's four tiles; slots that no token has
// written read as zeros (past the buffer's range). A weight of 0 meets every other column's
// values: where those are not finite the sums are not either, and the wave's tokens are done
// again one by one.
//
// A step is bound by its chain of instructions (loads issued, two products, the weights, the next
// step's numbers: about 2,300 cycles for 32 keys of 128 channels), hidden by four workgroups a CU.
// Eight waves and 64 keys a step share more of the loads and have fewer barriers, but wait longer
// at each: a prompt of 8192 tokens takes 521 us instead of 464.
constexpr int kJoinWaves = 4;
constexpr int kJoinTiles = kJoinWaves / 2;  // of a step: a wave loads one of its K or V tiles
// Entries of a workgroup's lists: of the first, the table is no larger than the stages of 128
// channels; the second costs the narrower ones a workgroup a CU.
constexpr int kJoinMost = 512, kJoinMore = 1024;
constexpr int kJoinTokens = 8;   // tokens of a wave: their bits in a mask

template <int D, int MOST>
struct JoinLds {
  static constexpr int kTable = 2 * MOST;
  static constexpr int kTile = 16 * D * 2;  // bytes of 16 rows
  union {
    char stage[2][kJoinWaves][kTile];  // a step's K tiles, then its V tiles
    float q[kJoinWaves][D];            // attend_alone's
    struct {
      int32_t page[kTable];
      uint32_t tokens[kTable];
      uint32_t first[kTable], keys[kTable], part[kTable];
    };
  };
  int32_t list[MOST];  // pages
  uint32_t who[MOST];
  uint8_t keys_of[MOST];  // slots that hold keys, less 1; bit 7: some tokens count fewer
  int32_t counts[kJoinWaves];
};

// The 16-byte chunks of a staged key row are permuted by the row, so that the rows of one chunk
// lie in different banks.
template <int D>
__device__ inline int chunk_swizzle(int row) {
  return D % 64 == 0 ? row & 7 : (row >> 1) & 3;
}

template <class E, int D, int MOST>
__global__ void __launch_bounds__(kJoinWaves* kWave, D > 128 ? 2 : MOST > kJoinMost ? 3 : 4)
    kv_attend_joined_kernel(AttendArgs a) {
  using Wave = AttendWave<E, D>;
  using V8 = typename Wave::V8;
  using Lds = JoinLds<D, MOST>;
  constexpr int LOADS = D / 32;  // of a wave in a step
  __shared__ __attribute__((aligned(16))) Lds lds;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = lane_id(), col = lane & 15, grp = lane >> 4;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / a.Hkv) * kJoinWaves * a.joined;
  const int head = blockIdx.x % a.Hkv;
  const int most = kJoinWaves * a.joined;
  const int tokens = a.T - t0 < most ? static_cast<int>(a.T - t0) : most;
  const int size = 1 << a.tok.shift;

  // the union of the lists
  for (int i = threadIdx.x; i < Lds::kTable; i += kJoinWaves * kWave) {
    lds.page[i] = -1;
    lds.tokens[i] = 0u;
    lds.first[i] = ~0u;
    lds.keys[i] = 0u;
    lds.part[i] = 0u;
  }
  __syncthreads();
  constexpr int EACH = MOST / (kJoinWaves * kWave);
  int32_t page[EACH];
  uint32_t block[EACH];
  int slot[EACH], rank[EACH];
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    const int e = (wave * EACH + r) * kWave + lane;
    page[r] = -1;
    block[r] = 0u;
    slot[r] = 0;
    if (e >= tokens * a.count) continue;
    const int tok = e / a.count;
    const KvPlace p = kv_place(a.tok, t0 + tok);
    const int32_t b = a.blocks[((t0 + tok) * a.Hkv + head) * a.count + e % a.count];
    if (b < 0 || b > p.last) continue;
    page[r] = kv_page(a.tok, p, b);
    if (page[r] < 0) continue;
    block[r] = b;
    int s = static_cast<int>((static_cast<uint32_t>(page[r]) * 0x9E3779B1u) >> 16) &
            (Lds::kTable - 1);
    for (;;) {  // (at most half full: a free place or the page's own is met)
      const int32_t old = atomicCAS(&lds.page[s], -1, page[r]);
      if (old == -1 || old == page[r]) break;
      s = (s + 1) & (Lds::kTable - 1);
    }
    slot[r] = s;
    atomicOr(&lds.tokens[s], 1u << (tok / a.joined * kJoinTokens + tok % a.joined));
    atomicMin(&lds.first[s], static_cast<uint32_t>(e));
    const int slots = b == p.last ? (p.pos & (size - 1)) + 1 : size;
    atomicMax(&lds.keys[s], static_cast<uint32_t>(slots));
    if (slots < size) lds.part[s] = 1u;
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
  int listed = 0, at = 0;
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) {
    at += w < wave ? lds.counts[w] : 0;
    listed += lds.counts[w];
  }
  listed = __builtin_amdgcn_readfirstlane(listed);
  // by block: the workgroups of a head, which sweep the cache side by side, then meet in its L2
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    const uint64_t m = __ballot(first[r]);
    rank[r] = at + __popcll(m & ((uint64_t{1} << lane) - 1));
    if (first[r]) lds.first[rank[r]] = block[r];  // (the table's firsts have been read)
    at += __popcll(m);
  }
  if (threadIdx.x < 8) lds.first[listed + threadIdx.x] = ~0u;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    if (!first[r]) continue;
    int to = 0;
    for (int i = 0; i < listed; i += 8) {
      v4i b[2];
      b[0] = *reinterpret_cast<const v4i*>(&lds.first[i]);
      b[1] = *reinterpret_cast<const v4i*>(&lds.first[i + 4]);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const uint32_t o = static_cast<uint32_t>(b[x >> 2][x & 3]);
        to += o < block[r] || (o == block[r] && i + x < rank[r]) ? 1 : 0;
      }
    }
    lds.list[to] = page[r];
    lds.who[to] = lds.tokens[slot[r]];
    lds.keys_of[to] = static_cast<uint8_t>(lds.keys[slot[r]] - 1u + 128u * lds.part[slot[r]]);
  }

  // this lane's column: its token's own page ends after `own_keys`
  const int tok = col / a.G;
  const bool real = tok < a.joined && wave * a.joined + tok < tokens;
  const int64_t t = t0 + (real ? wave * a.joined + tok : 0);
  const int hq = head * a.G + col % a.G;
  int32_t own = -1, own_keys = 0;
  if (real) {
    const KvPlace p = kv_place(a.tok, t);
    if (p.last >= 0) own = kv_page(a.tok, p, p.last);
    own_keys = (p.pos & (size - 1)) + 1;
  }
  const int here = tokens - wave * a.joined;  // this wave's tokens, their bits for both tiles
  const uint32_t all =
      ((1u << (here < 0 ? 0 : here > a.joined ? a.joined : here)) - 1u) * 0x0101u;
  Wave w;
  w.clear();
  w.load_q(a, t, hq, real);
  __syncthreads();  // the list is whole, and the table's place free for the stages

  // A lane's 16-byte chunks of the tile that this wave loads.
  int offset[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int x = i * 64 + lane, row = x / (D / 8), c = x % (D / 8);
    const int from = wave < kJoinTiles ? c ^ chunk_swizzle<D>(row)
                              : (((c >> 1) ^ granule_swizzle<D>(row)) << 1) + (c & 1);
    offset[i] = row * (D * 2) + from * 16;
  }
  // Steps of two tiles of 16 keys. 64 at a time are worked out, one a lane: whose columns count
  // (the wave's tokens, a byte a tile; `part`: some not all of a page's slots), and what this wave
  // loads: its tile's first row and rows. Steps without keys are left out.
  const int total = listed << (a.tok.shift - 4);  // tiles
  int64_t my_row = 0;
  uint32_t my_who = 0u;
  int32_t my_rows = 0, base = -kWave;
  uint64_t left = 0;
  struct Step {
    int64_t row;   // to load
    int32_t rows;  // 32: `part`
    int32_t at;    // its first tile; `total`: there is none
    uint32_t who;
  };
  auto next = [&]() {
    Step s{0, 0, total, 0u};
    while (left == 0) {
      base += kWave;
      if (kJoinTiles * base >= total) return s;
      bool any = false, part = false;
      my_who = 0u;
#pragma unroll
      for (int j = 0; j < kJoinTiles; ++j) {
        const int i = kJoinTiles * (base + lane) + j, e = i < total ? i >> (a.tok.shift - 4) : 0;
        const int about = i < total ? lds.keys_of[e] : 0, from = (i << 4) & (size - 1);
        const int n = i < total ? (about & 127) + 1 - from : 0;
        any |= n > 0;
        part |= about >= 128;
        if (i < total) {
          my_who |= ((lds.who[e] >> (wave * kJoinTokens)) & 255u) << (8 * j);
        }
        if (j == wave % kJoinTiles) {
          my_row = ((static_cast<int64_t>(lds.list[e]) * a.Hkv + head) << a.tok.shift) + from;
          my_rows = n < 0 ? 0 : n > 16 ? 16 : n;
        }
      }
      my_rows += part ? 32 : 0;
      left = __ballot(any);
    }
    const int i = __builtin_ctzll(left);
    left &= left - 1;
    s.at = kJoinTiles * (base + i);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int32_t>(my_row), i);
    s.row = static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int32_t>(my_row >> 32), i))
                << 32 | lo;
    s.rows = __builtin_amdgcn_readlane(my_rows, i);
    s.who = __builtin_amdgcn_readlane(static_cast<int32_t>(my_who), i);
    return s;
  };
  const char* cache = static_cast<const char*>(wave < kJoinTiles ? a.k_cache : a.v_cache);
  auto issue = [&](const Step& s, char* stage) {
    const char* from = cache + s.row * (D * 2);
    const int bytes = (s.rows & 31) * (D * 2);
#pragma unroll
    for (int x = 0; x < LOADS; ++x) {
      buffer_load_lds<16, false>(from, bytes, offset[x],
                                 stage + wave * Lds::kTile + x * (kWave * 16));
    }
  };
  // One step from `use` while the next goes into `fill`. (The two stages differ: said by
  // `restrict`, else every read here would wait for the loads just started.)
  auto work = [&](char* __restrict fill, const char* __restrict use, const Step& late,
                  const Step& s) {
    if (late.at < total) issue(late, fill);
    v4f sc[kJoinTiles];
#pragma unroll
    for (int j = 0; j < kJoinTiles; ++j) sc[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
#pragma unroll
      for (int j = 0; j < kJoinTiles; ++j) {
        const V8 k = *reinterpret_cast<const V8*>(
            use + j * Lds::kTile + col * (D * 2) + (((grp + 4 * x) ^ chunk_swizzle<D>(col)) << 4));
        sc[j] = Wave::Op::mma(k, w.qf[x], sc[j]);
      }
    }
    const bool whole = s.rows < 32 && s.who == all;
    int n[kJoinTiles];
    if (!whole) {
#pragma unroll
      for (int j = 0; j < kJoinTiles; ++j) {
        const bool counts = ((s.who >> (8 * j + tok)) & 1u) != 0;
        n[j] = !real || counts ? 16 : 0;
        if (s.rows >= 32 && real && counts) {
          const int i = s.at + j;
          const int end = lds.list[i >> (a.tok.shift - 4)] == own ? own_keys : size;
          n[j] = end - ((i << 4) & (size - 1));
        }
      }
    }
    V8 p[kJoinTiles / 2];
    w.template weigh<true>(a.scale, sc, whole, n, p);
    w.add(use + kJoinTiles * Lds::kTile, p);
  };
  Step now = next();
  if (now.at < total) issue(now, lds.stage[0][0]);
  int get = 0;
  while (now.at < total) {
    Step late = next();
    wait_vmcnt<0>();
    tile_barrier();
    while (now.who == 0) {  // (nothing here for this wave's tokens)
      get ^= 1;
      now = late;
      if (now.at >= total) break;
      issue(now, lds.stage[get][0]);
      late = next();
      wait_vmcnt<0>();
      tile_barrier();
    }
    if (now.at >= total) break;
    work(lds.stage[get ^ 1][0], lds.stage[get][0], late, now);
    get ^= 1;
    now = late;
  }
  w.join_sums();
  __syncthreads();  // (the stages are free)
  float odd = 0.0f;  // 0 times every sum: not a number where one is not finite, or scores are far
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
#pragma unroll
    for (int r = 0; r < 4; ++r) odd = fmaf(w.acc[i][r], 0.0f, odd);
  }
  if (!__any(real && !(odd == 0.0f))) {
    if (real) emit(a, w, t, hq);
    return;
  }
  for (int i = 0; i < a.joined && wave * a.joined + i < tokens; ++i) {
    const int64_t one = t0 + wave * a.joined + i;
    for (int g = 0; g < a.G; ++g) attend_alone<E, D>(a, one, head, head * a.G + g, lds.q[wave]);
  }
}

// Few rows: the workgroup's waves (and `parts` workgroups) share a row's list; their sums are
// joined at the largest maximum, here where one workgroup has the whole row, else by
// kv_join_kernel.
template <class E, int D>
__global__ void __launch_bounds__(kAttendWaves* kWave, D <= 128 ? 2 : 1)
    kv_attend_split_kernel(AttendArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[kAttendWaves][64 * D];
  __shared__ float ml[kAttendWaves][16][2];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int part = blockIdx.x % a.parts;
  const int64_t row = blockIdx.x / a.parts;  // (token, key/value head, tile)
  const int tile = static_cast<int>(row % a.tiles);
  const int head = static_cast<int>(row / a.tiles % a.Hkv);
  const int64_t t = row / a.tiles / a.Hkv;
  AttendWave<E, D> w;
  // A token beside one of its own sequence chooses mostly its blocks: these stay in L2. Others'
  // rows are read once.
  const int32_t seq = a.tok.seq_ids[t];
  const bool beside = (t > 0 && a.tok.seq_ids[t - 1] == seq) ||
                      (t + 1 < a.T && a.tok.seq_ids[t + 1] == seq);
  const int first = part * kAttendWaves + wave, parts = a.parts * kAttendWaves;
  if (beside) {
    w.template run<false>(a, t, head, tile, first, parts, lds[wave]);
  } else {
    w.template run<true>(a, t, head, tile, first, parts, lds[wave]);
  }
  join_waves<E, D>(a, w.acc, w.m, w.l, t, head, tile, row, part, lds, ml);
}

// How a call of `seqs` sequences at most is spread: `parts` workgroups a row; 0: `joined` tokens a
// wave, or (0) a wave a row.
struct AttendPlan {
  int64_t rows;
  int32_t tiles, parts, joined;
  bool more;  // joined lists of up to kJoinMore entries
};

// Times in us are of lists of 16 blocks of 64 keys, 32 heads of 8 key/value heads.
inline AttendPlan attend_plan(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t seqs,
                              int64_t page, int64_t count) {
  AttendPlan p;
  const int64_t G = Hq / Hkv;
  p.tiles = static_cast<int32_t>(cdiv(G, 16));
  p.rows = T * Hkv * p.tiles;
  p.parts = 0;
  int64_t joined = 16 / (G < 16 ? G : 16);
  if (joined > kJoinTokens) joined = kJoinTokens;
  const int64_t entries = kJoinWaves * (count > 0 ? count : 1);
  // workgroups of the small table on the GPU (four a CU, two of the wide heads); the larger table
  // has one token a wave, or more workgroups than this
  const int64_t held = D <= 128 ? 1024 : 512;
  // Lists of which kJoinMost holds one token a wave: two of them by the larger table, where there
  // are more workgroups than the GPU holds and a block's work outweighs its entries' in the table
  // (1000 tokens of 10 heads of 128, 96 blocks of 32 keys: 382 for 488; of 20 heads of 64: 573 for
  // 519, but 551 for 650 with 70 blocks of 64). Lists of which it holds none: one, against a wave a
  // row (1000 tokens of 10 heads of 128, 200 blocks of 16: 747 for 1105; of 20 heads of 96: 1243
  // for 1103, but 1599 for 3035 with 160 blocks of 64).
  p.more = kJoinMost / entries < 1 ? D > 96 || page >= 64
                                   : kJoinMost / entries < 2 && (D > 64 || page >= 64) &&
                                         cdiv(T, kJoinWaves) * Hkv > held;
  const int64_t lists = (p.more ? kJoinMore : kJoinMost) / entries;
  if (joined > lists) joined = lists;
  // (one token a wave still shares a workgroup's loads: 460 tokens of 10 heads of 128, lists of 96
  // blocks of 32 keys, 260 us for 532 with a wave a row)
  p.joined = G <= 8 ? static_cast<int32_t>(joined) : 0;
  // A joined workgroup's time is its chain of steps, whether it has a CU for itself or shares it,
  // so while the GPU holds them all there are twice as many with half the tokens (and a shorter
  // union): 1024 tokens of 128 channels 103 for 127, 511 tokens 73 for 114.
  while (p.joined > 1 && cdiv(T, kJoinWaves * (p.joined / 2)) * Hkv <= held) p.joined /= 2;
  // Prompts are joined where the chain is shorter than the split form's reads of every row's blocks
  // (split and joined: 64 channels, 300 tokens 50 and 50, 400 tokens 63 and 52; 128 channels, 200
  // tokens 67 and 53; 256 channels, 100 tokens 100 and 99, 200 tokens 176 and 85). No more tokens
  // than sequences are taken for single tokens, which share nothing: 500 of 128 channels take 328
  // split and 365 joined, 2000 take 1246 and 1434.
  if (T > seqs && (p.joined > 0 ? p.rows * D >= 200 << 10 : p.rows >= 4096)) return p;
  // Workgroups of four waves for two on every CU, each wave with a unit of 64 keys at least. A
  // second launch that joins the parts costs 4 us, a row in one workgroup more: one token of 8
  // heads over 32 blocks of 64 keys takes 12 us in 8 parts a row, 23 in one workgroup of 8 waves.
  // (Rows whose parts are several are too few to be joined: the workspace does not depend on seqs.)
  const int64_t most = cdiv(count * page, 64 * kAttendWaves);
  const int64_t want = cdiv(512, p.rows > 0 ? p.rows : 1);
  p.parts = static_cast<int32_t>(want < most ? want : most);
  if (p.parts < 1) p.parts = 1;
  return p;
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_kv_attention_workspace(int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                            int64_t page, int64_t count) {
  if (Hkv < 1 || T < 1) return 0;
  const AttendPlan p = attend_plan(T, Hq, Hkv, D, 0, page, count);
  return p.parts > 1 ? static_cast<size_t>(p.rows) * p.parts * 16 * (D + 2) * sizeof(float) : 0;
}

extern "C" int rt_kv_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                               int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype,
                               const void* k_cache, const void* v_cache, int64_t P, int64_t page,
                               const int32_t* blocks, int64_t count, const int32_t* positions,
                               const int32_t* seq_ids, const int32_t* page_table, int64_t B,
                               int64_t max_pages, float scale, void* out, float* lse,
                               void* workspace, size_t workspace_bytes, rt_stream_t stream) {
  return rt_kv_attention_of(q, q_token_stride, q_head_stride, T, Hq, Hkv, D, dtype, k_cache,
                            v_cache, P, page, blocks, count, positions, seq_ids, page_table, B,
                            max_pages, scale, B, out, lse, workspace, workspace_bytes, stream);
}

extern "C" int rt_kv_attention_of(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                  int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype,
                                  const void* k_cache, const void* v_cache, int64_t P, int64_t page,
                                  const int32_t* blocks, int64_t count, const int32_t* positions,
                                  const int32_t* seq_ids, const int32_t* page_table, int64_t B,
                                  int64_t max_pages, float scale, int64_t sequences, void* out,
                                  float* lse, void* workspace, size_t workspace_bytes,
                                  rt_stream_t stream) {
  if (const int st = kv_check(T, Hq, Hkv, D, dtype, B, max_pages, P, page)) return st;
  RT_CHECK_ARG(count >= 0 && count <= (1 << 20), "count must be in [0, 2^20], got %lld",
               static_cast<long long>(count));
  if (T == 0) return kOk;
  RT_CHECK_ARG(q && positions && seq_ids && out && lse && (count == 0 || blocks), "null pointer");
  RT_CHECK_ARG(B * max_pages == 0 || page_table, "null page table");
  RT_CHECK_ARG(P == 0 || (k_cache && v_cache), "null cache");
  RT_CHECK_ARG(kv_rows_aligned(q, q_token_stride, q_head_stride) &&
                   kv_rows_aligned(k_cache, 0, 0) && kv_rows_aligned(v_cache, 0, 0) &&
                   kv_rows_aligned(out, 0, 0),
               "rows must start on 16 bytes");
  RT_CHECK_ARG(T * Hq <= INT32_MAX, "too many tokens");
  RT_CHECK_ARG(std::isfinite(scale * kLog2e), "the scale must be finite, got %g",
               static_cast<double>(scale));
  RT_CHECK_ARG(sequences >= 0, "sequences must not be negative, got %lld",
               static_cast<long long>(sequences));
  const size_t need = rt_kv_attention_workspace(T, Hq, Hkv, D, page, count);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
    set_error("workspace too small: %zu < %zu", workspace_bytes, need);
    return kWorkspaceTooSmall;
  }
  const AttendPlan plan = attend_plan(T, Hq, Hkv, D, sequences, page, count);
  AttendArgs a{};
  a.q = q, a.q_st = q_token_stride, a.q_sh = q_head_stride, a.T = T;
  a.Hq = static_cast<int32_t>(Hq), a.Hkv = static_cast<int32_t>(Hkv);
  a.G = a.Hq / a.Hkv, a.tiles = plan.tiles;
  a.k_cache = k_cache, a.v_cache = v_cache, a.blocks = blocks;
  a.count = static_cast<int32_t>(count);
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  // (a scale of 0 becomes the least number: the scores are 0 all the same, and -inf stays -inf)
  a.scale = fmaxf(fabsf(scale * kLog2e), 1.17549435e-38f), a.minus = scale < 0.0f;
  a.out = out, a.lse = lse, a.parts = plan.parts;
  a.joined = plan.joined;
  a.part_out = static_cast<float*>(workspace);
  a.part_ml = a.part_out + (plan.parts > 1 ? plan.rows * plan.parts * 16 * D : 0);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return kv_dispatch(dtype, D, [&](auto e, auto d) -> int {
    using E = decltype(e);
    constexpr int DD = decltype(d)::value;
    const dim3 threads(kAttendWaves * kWave);
    if (plan.parts == 0 && plan.joined > 0) {
      const int64_t grid = cdiv(T, kJoinWaves * plan.joined) * Hkv;
      const dim3 g(static_cast<unsigned>(grid)), b(kJoinWaves * kWave);
      if (plan.more) {
        kv_attend_joined_kernel<E, DD, kJoinMore><<<g, b, 0, s>>>(a);
      } else {
        kv_attend_joined_kernel<E, DD, kJoinMost><<<g, b, 0, s>>>(a);
      }
    } else if (plan.parts == 0) {
      const int64_t grid = cdiv(T, kAttendWaves) * Hkv * plan.tiles;
      kv_attend_rows_kernel<E, DD><<<dim3(static_cast<unsigned>(grid)), threads, 0, s>>>(a);
    } else {
      const int64_t grid = plan.rows * plan.parts;
      kv_attend_split_kernel<E, DD><<<dim3(static_cast<unsigned>(grid)), threads, 0, s>>>(a);
      if (plan.parts > 1) {
        kv_join_kernel<E, DD><<<dim3(static_cast<unsigned>(T * Hq)), dim3(DD / 4), 0, s>>>(a);
      }
    }
    RT_CHECK_HIP(hipGetLastError());
    return kOk;
  });
}
