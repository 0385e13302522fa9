// Appending to a paged key/value cache with the rotary position applied on the way, and the int8
// bounds of the blocks that become full.
//
// Rotation: with (c, s) the table's cosine and sine of the token's position, a pair of channels
// (a, b) becomes (a c - b s, b c + a s). Every product and sum is rounded once to fp32 (no fused
// multiply-add), then to the cache's 16 bits: the same bits whichever tile a token falls in, so
// a block's bounds do not depend on how its tokens were split over calls.
//
// Bounds of a full block: per channel lo and hi over its stored keys, mid = (lo + hi) / 2 and half
// = (hi - lo) / 2, the row [mid | half] as int8 codes of one scale. q . mid + |q| . half is then
// the most that any key of the block can score with q. Minimum and maximum do not depend on the
// order, so the codes are the same in any split.
//
// One launch. Some workgroups look for tokens that complete a block: the block's keys that are part
// of this call are rotated again from the input (no wait on the waves that store them), the
// earlier ones come from the cache. In the others a wave moves a token's rows (or some of them,
// where there are few tokens): a lane holds two 16-byte chunks of a row, which in the split layout
// are partners, with their cosines and sines, and walks over the heads, two rows in flight.
//
// Bound by memory: every row is read and written once. 32768 tokens of 32 rows of 256 channels take
// 229 to 234 us (4.8 TB/s, what a large copy reaches) with nontemporal loads and stores (when they
// were taken 238, 283 with ordinary stores; four rows in flight instead of two 250). A decode step
// is bound by its launch (3 us). With norms 9001 tokens of 48 rows of 128 channels take 54 us (47 at
// that rate), a decode step 4.
#include <type_traits>

#include "../../include/retrieve_amd.h"
#include "kv_rotate.h"

namespace rt {

constexpr int kAppendThreads = 256;

struct AppendArgs : TurnArgs {
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // token and head strides, elements
  int64_t T;
  int32_t Hq, Hkv;
  KvTokens tok;
  void *k_cache, *v_cache;
  int8_t* bounds;
  float* scales;
  void* q_out;
  int32_t row_parts;      // waves a token's rows are split over
  uint32_t bound_groups;  // workgroups that look for full blocks
  int32_t tile;           // tokens that one of them looks at
};

// Where a token's row goes: (page, head, slot), in elements.
template <int D>
__device__ inline int64_t cache_row(const AppendArgs& a, int32_t page, int head, int32_t pos) {
  const int64_t block = static_cast<int64_t>(page) * a.Hkv + head;
  return ((block << a.tok.shift) + (pos & ((1 << a.tok.shift) - 1))) * D;
}

template <class E, int D, int MODE, bool NORM>
__device__ inline void move_rows(const AppendArgs& a, int64_t unit) {
  using V8 = typename Kv<E>::V8;
  constexpr int C = D / 16, SLOTS = kWave / C, FLIGHT = 2;
  const int lane = lane_id() % C, slot = lane_id() / C;
  const int64_t t = unit / a.row_parts;
  if (t >= a.T || slot >= SLOTS) return;
  const KvPlace p = kv_place(a.tok, t);
  const int32_t page = p.last >= 0 ? kv_page(a.tok, p, p.last) : -1;
  const bool valid = page >= 0 && (a.rot == 0 || p.pos < a.table_len);
  Pair<E, D, MODE, NORM> pair(a, lane);
  if (valid) pair.load(a, p.pos);
  const int rows = a.Hq + 2 * a.Hkv, step = a.row_parts * SLOTS;
  const E* q = static_cast<const E*>(a.q) + t * a.q_st;
  const E* k = static_cast<const E*>(a.k) + t * a.k_st;
  const E* v = static_cast<const E*>(a.v) + t * a.v_st;
  E* to_q = static_cast<E*>(a.q_out) + t * a.Hq * D;
  const int64_t at = valid ? cache_row<D>(a, page, 0, p.pos) : 0;
  const int64_t head = static_cast<int64_t>(D) << a.tok.shift;  // from head to head of a page
  for (int r0 = static_cast<int>(unit % a.row_parts) * SLOTS + slot; r0 < rows;
       r0 += FLIGHT * step) {
    V8 x[FLIGHT][2];
    const E* from[FLIGHT];
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
      const int r = r0 + i * step;
      from[i] = r < a.Hq           ? q + r * a.q_sh
                : r < a.Hq + a.Hkv ? k + (r - a.Hq) * a.k_sh
                                   : v + (r - a.Hq - a.Hkv) * a.v_sh;
      x[i][0] = V8{};
      x[i][1] = V8{};
      if (valid && r < rows) {
        x[i][0] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(from[i]) + pair.chunk[0]);
        x[i][1] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(from[i]) + pair.chunk[1]);
      }
    }
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
      const int r = r0 + i * step;
      if (r >= rows || (r >= a.Hq && !valid)) continue;
      if (valid && r < a.Hq + a.Hkv && (NORM || a.rot > 0)) {
        pair.apply(from[i], a, r < a.Hq ? 0 : 1, x[i]);
      }
      E* to = r < a.Hq           ? to_q + r * D
              : r < a.Hq + a.Hkv ? static_cast<E*>(a.k_cache) + at + (r - a.Hq) * head
                                 : static_cast<E*>(a.v_cache) + at + (r - a.Hq - a.Hkv) * head;
      __builtin_nontemporal_store(x[i][0], reinterpret_cast<V8*>(to) + pair.chunk[0]);
      __builtin_nontemporal_store(x[i][1], reinterpret_cast<V8*>(to) + pair.chunk[1]);
    }
  }
}

template <class E, int D, int MODE, bool NORM>
__device__ inline void fill_bounds(const AppendArgs& a) {
  using V8 = typename Kv<E>::V8;
  // (a norm's lanes of a row are neighbours of one wave)
  constexpr int C = D / 8, WAVE_SLOTS = kWave / C;
  constexpr int SLOTS = NORM ? kAppendThreads / kWave * WAVE_SLOTS : kAppendThreads / C;
  __shared__ float lows[SLOTS][D], highs[SLOTS][D];
  __shared__ float tops[kAppendThreads / kWave];
  const int head = static_cast<int>(blockIdx.x % a.Hkv);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / a.Hkv) * a.tile;
  const int size = 1 << a.tok.shift;
  int chunk = threadIdx.x % C, slot = threadIdx.x / C;
  if constexpr (NORM) {
    chunk = lane_id() % C;
    slot = lane_id() / C < WAVE_SLOTS
               ? static_cast<int>(threadIdx.x / kWave) * WAVE_SLOTS + lane_id() / C
               : SLOTS;
  }
  const E* k = static_cast<const E*>(a.k) + head * a.k_sh;
  const HeadNorm& norm = a.norm[1];
  Weights<E> w;
  if (NORM) w.load(norm, chunk);
  // which of the tile's tokens complete a block: one a lane (the same in every wave)
  const int64_t mine = t0 + lane_id();
  bool full = false;
  if (lane_id() < a.tile && mine < a.T) {
    const KvPlace p = kv_place(a.tok, mine);
    full = p.last >= 0 && (p.pos & (size - 1)) == size - 1 && kv_page(a.tok, p, p.last) >= 0 &&
           (a.rot == 0 || p.pos < a.table_len);
  }
  for (uint64_t left = __ballot(full); left != 0; left &= left - 1) {
    const int64_t t = t0 + __builtin_ctzll(left);
    const KvPlace p = kv_place(a.tok, t);
    const int32_t page = kv_page(a.tok, p, p.last);
    const int32_t seq = a.tok.seq_ids[t];
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = INFINITY;
      hi[e] = -INFINITY;
    }
    if (slot < SLOTS) {
      for (int o = slot; o < size; o += SLOTS) {
        const int64_t from = t - (size - 1 - o);
        const int32_t pos = p.pos - (size - 1 - o);
        V8 x;
        if (from >= 0 && a.tok.positions[from] == pos && a.tok.seq_ids[from] == seq) {
          Turn<MODE> turn;
          if (a.rot > 0) turn.load(a, pos, chunk);
          const E* row = k + from * a.k_st;
          const V8 own[1] = {reinterpret_cast<const V8*>(row)[chunk]};
          float r = 1.0f;
          if (NORM && norm.weight) r = row_scale<E, D, C>(own, chunk, a.eps);
          x = turned_chunk<E, MODE, NORM>(row, own[0], chunk, turn, a, norm, r, w);
        } else {
          x = *reinterpret_cast<const V8*>(static_cast<const E*>(a.k_cache) +
                                           cache_row<D>(a, page, head, pos) + 8 * chunk);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          lo[e] = fminf(lo[e], static_cast<float>(x[e]));
          hi[e] = fmaxf(hi[e], static_cast<float>(x[e]));
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lows[slot][8 * chunk + e] = lo[e];
        highs[slot][8 * chunk + e] = hi[e];
      }
    }
    __syncthreads();
    const int d = threadIdx.x;
    float mid = 0.0f, half = 0.0f;
    if (d < D) {
      float l = lows[0][d], h = highs[0][d];
      for (int i = 1; i < SLOTS; ++i) {
        l = fminf(l, lows[i][d]);
        h = fmaxf(h, highs[i][d]);
      }
      mid = (l + h) * 0.5f;
      half = (h - l) * 0.5f;
    }
    float top = fmaxf(fabsf(mid), half);
    for (int x = 1; x < kWave; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    if (lane_id() == 0) tops[threadIdx.x / kWave] = top;
    __syncthreads();
    top = kKvTopFloor;
    for (int w = 0; w < kAppendThreads / kWave; ++w) top = fmaxf(top, tops[w]);
    const int64_t row = static_cast<int64_t>(page) * a.Hkv + head;
    if (d < D) {
      a.bounds[row * 2 * D + d] = static_cast<int8_t>(kv_code(mid, top));
      a.bounds[row * 2 * D + D + d] = static_cast<int8_t>(kv_code(half, top));
    }
    if (d == 0) a.scales[row] = top / 127.0f;
    __syncthreads();
  }
}

// Workgroups a CU that the registers have to leave room for (the rows in flight hide the memory:
// fp16 rows of 256, neighbours turned, 245 us with 5, 234 with 6).
constexpr int append_groups(int mode, bool norm) {
  if (mode == kRotHalfOdd) return norm ? 3 : 4;
  return norm ? 4 : mode == kRotPairs ? 6 : 5;
}

template <class E, int D, int MODE, bool NORM>
__global__ void __launch_bounds__(kAppendThreads, append_groups(MODE, NORM))
    kv_append_kernel(AppendArgs a) {
  if (blockIdx.x < a.bound_groups) {
    fill_bounds<E, D, MODE, NORM>(a);
  } else {
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    move_rows<E, D, MODE, NORM>(
        a, (blockIdx.x - a.bound_groups) * (kAppendThreads / kWave) + wave);
  }
}

}  // namespace rt

using namespace rt;

extern "C" int rt_kv_append(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                            const void* k, int64_t k_token_stride, int64_t k_head_stride,
                            const void* v, int64_t v_token_stride, int64_t v_head_stride, int64_t T,
                            int64_t Hq, int64_t Hkv, int64_t D, int dtype, const float* cos_sin,
                            int64_t table_len, int64_t rot, int interleaved,
                            const int32_t* positions, const int32_t* seq_ids,
                            const int32_t* page_table, int64_t B, int64_t max_pages, void* k_cache,
                            void* v_cache, int64_t P, int64_t page, int8_t* bounds,
                            float* bound_scales, void* q_out, rt_stream_t stream) {
  return rt_kv_append_norm(q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, v,
                           v_token_stride, v_head_stride, T, Hq, Hkv, D, dtype, nullptr, nullptr, 0,
                           0.0, cos_sin, table_len, rot, interleaved, positions, seq_ids, page_table,
                           B, max_pages, k_cache, v_cache, P, page, bounds, bound_scales, q_out,
                           stream);
}

extern "C" int rt_kv_append_norm(
    const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
    int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
    int64_t v_head_stride, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype,
    const void* q_weight, const void* k_weight, int wide_weights, double eps, const float* cos_sin,
    int64_t table_len, int64_t rot, int interleaved, const int32_t* positions,
    const int32_t* seq_ids, const int32_t* page_table, int64_t B, int64_t max_pages, void* k_cache,
    void* v_cache, int64_t P, int64_t page, int8_t* bounds, float* bound_scales, void* q_out,
    rt_stream_t stream) {
  if (const int st = kv_check(T, Hq, Hkv, D, dtype, B, max_pages, P, page)) return st;
  if (const int st = kv_check_turn(T, D, cos_sin, table_len, rot, q_weight, k_weight, eps)) {
    return st;
  }
  if (T == 0) return kOk;
  RT_CHECK_ARG(q && k && v && positions && seq_ids && q_out, "null pointer");
  RT_CHECK_ARG(B * max_pages == 0 || page_table, "null page table");
  RT_CHECK_ARG(P == 0 || (k_cache && v_cache && bounds && bound_scales), "null cache");
  RT_CHECK_ARG(kv_rows_aligned(q, q_token_stride, q_head_stride) &&
                   kv_rows_aligned(k, k_token_stride, k_head_stride) &&
                   kv_rows_aligned(v, v_token_stride, v_head_stride) &&
                   kv_rows_aligned(k_cache, 0, 0) && kv_rows_aligned(v_cache, 0, 0) &&
                   kv_rows_aligned(q_out, 0, 0),
               "rows must start on 16 bytes");
  AppendArgs a{};
  a.q = q, a.k = k, a.v = v;
  a.q_st = q_token_stride, a.q_sh = q_head_stride;
  a.k_st = k_token_stride, a.k_sh = k_head_stride;
  a.v_st = v_token_stride, a.v_sh = v_head_stride;
  a.T = T, a.Hq = static_cast<int32_t>(Hq), a.Hkv = static_cast<int32_t>(Hkv);
  static_cast<TurnArgs&>(a) = kv_turn_args(cos_sin, table_len, rot, q_weight, k_weight,
                                           wide_weights, eps);
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  a.k_cache = k_cache, a.v_cache = v_cache, a.bounds = bounds, a.scales = bound_scales;
  a.q_out = q_out;
  const int slots = static_cast<int>(kWave / (D / 16));
  const int64_t all = cdiv(Hq + 2 * Hkv, slots);
  // Few tokens: a token's rows over as many waves as have one each. Many: one wave a token.
  const int64_t parts = cdiv(4096, T);
  a.row_parts = static_cast<int32_t>(parts < all ? parts : all);
  // Few tokens may all complete a block in one step (sequences of one length): a workgroup for each
  // and every head, up to 1024 of them (more would cost their launch). In prompts one token in
  // `page` does: 64 tokens a workgroup.
  const int64_t tile = next_pow2(cdiv(T * Hkv, 1024));
  a.tile = static_cast<int32_t>(tile < 64 ? tile : 64);
  const int64_t bound_groups = cdiv(T, a.tile) * Hkv;
  const int64_t grid = bound_groups + cdiv(T * a.row_parts, kAppendThreads / kWave);
  RT_CHECK_ARG(grid <= INT32_MAX, "too many tokens");
  a.bound_groups = static_cast<uint32_t>(bound_groups);
  return kv_dispatch(dtype, D, [&](auto e, auto d) -> int {
    using E = decltype(e);
    constexpr int DD = decltype(d)::value;
    const bool normed = q_weight || k_weight;
    return kv_turn_dispatch(rot, interleaved, normed, [&](auto mode, auto norm) -> int {
      kv_append_kernel<E, DD, decltype(mode)::value, decltype(norm)::value>
          <<<dim3(static_cast<unsigned>(grid)), dim3(kAppendThreads), 0,
             static_cast<hipStream_t>(stream)>>>(a);
      RT_CHECK_HIP(hipGetLastError());
      return kOk;
    });
  });
}
