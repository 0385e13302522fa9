// Softmax attention of each token over the blocks chosen for it and its key/value head.
//
// out = sum_j exp(x_j - m) v_j / l over the keys j of the listed blocks at positions up to the token's,
// with x_j = scale q . k_j, m their maximum and l the sum of the weights, kept running over one
// pass (a new maximum rescales what is summed); lse = m + log l. Rows without a key: 0 and -inf.
#include <type_traits>

#include "../../include/retrieve_amd.h"
#include "kv_common.h"

namespace rt {

struct AttendArgs {
  const void* q;
  int64_t q_st, q_sh;
  int64_t T;
  int32_t Hq, Hkv;
  const void *k_cache, *v_cache;
  const int32_t* blocks;  // [T, Hkv, count]
  int32_t count;
  KvTokens tok;
  float scale;
  void* out;   // [T, Hq, D]
  float* lse;  // [T, Hq]
};

// One wave a token and query head; a lane scores one key of 64, then sums its own channels.
template <class E, int D>
__global__ void __launch_bounds__(kWave) kv_attention_kernel(AttendArgs a) {
  using V8 = typename Kv<E>::V8;
  constexpr int R = (D + kWave - 1) / kWave;
  __shared__ float qs[D];
  const int64_t t = blockIdx.x / a.Hq;
  const int hq = blockIdx.x % a.Hq, h = hq / (a.Hq / a.Hkv);
  const int lane = lane_id();
  const KvPlace p = kv_place(a.tok, t);
  const E* q = static_cast<const E*>(a.q) + t * a.q_st + hq * a.q_sh;
  for (int d = lane; d < D; d += kWave) qs[d] = static_cast<float>(q[d]) * a.scale;
  __syncthreads();
  const int size = 1 << a.tok.shift;
  const int32_t* list = a.blocks + (t * a.Hkv + h) * a.count;
  float m = -INFINITY, l = 0.0f, acc[R] = {};
  for (int i = 0; i < a.count; ++i) {
    const int32_t block = list[i];
    if (block < 0 || block > p.last) continue;
    const int32_t page = kv_page(a.tok, p, block);
    if (page < 0) continue;
    const int64_t base = ((static_cast<int64_t>(page) * a.Hkv + h) << a.tok.shift) * D;
    const int64_t first = static_cast<int64_t>(block) << a.tok.shift;
    const int keys = p.pos - first + 1 < size ? static_cast<int>(p.pos - first + 1) : size;
    for (int j0 = 0; j0 < keys; j0 += kWave) {
      const int j = j0 + lane;
      float x = -INFINITY;
      if (j < keys) {
        const E* k = static_cast<const E*>(a.k_cache) + base + static_cast<int64_t>(j) * D;
        x = 0.0f;
        for (int d = 0; d < D; d += 8) {
          const V8 kv = *reinterpret_cast<const V8*>(k + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) x = fmaf(static_cast<float>(kv[e]), qs[d + e], x);
        }
      }
      float top = x;
      for (int s = 1; s < kWave; s <<= 1) top = fmaxf(top, __shfl_xor(top, s));
      const float next = fmaxf(m, top);
      const float safe = next == -INFINITY ? 0.0f : next;
      const float w = __expf(x - safe), keep = __expf(m - safe);
      float sum = w;
      for (int s = 1; s < kWave; s <<= 1) sum += __shfl_xor(sum, s);
      l = l * keep + sum;
      m = next;
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r] *= keep;
      const int n = keys - j0 < kWave ? keys - j0 : kWave;
      for (int jj = 0; jj < n; ++jj) {
        const float wj = __shfl(w, jj);
        const E* v = static_cast<const E*>(a.v_cache) + base + static_cast<int64_t>(j0 + jj) * D;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int d = r * kWave + lane;
          if (d < D) acc[r] = fmaf(wj, static_cast<float>(v[d]), acc[r]);
        }
      }
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
  E* out = static_cast<E*>(a.out) + (t * a.Hq + hq) * D;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int d = r * kWave + lane;
    if (d < D) out[d] = static_cast<E>(acc[r] * inv);
  }
  if (lane == 0) a.lse[t * a.Hq + hq] = l > 0.0f || l != l ? m + logf(l) : -INFINITY;
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_kv_attention_workspace(int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                            int64_t page, int64_t count) {
  return 0;
}

extern "C" int rt_kv_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                               int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype,
                               const void* k_cache, const void* v_cache, int64_t P, int64_t page,
                               const int32_t* blocks, int64_t count, const int32_t* positions,
                               const int32_t* seq_ids, const int32_t* page_table, int64_t B,
                               int64_t max_pages, float scale, void* out, float* lse,
                               void* workspace, size_t workspace_bytes, rt_stream_t stream) {
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
  const size_t need = rt_kv_attention_workspace(T, Hq, Hkv, D, page, count);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
    set_error("workspace too small: %zu < %zu", workspace_bytes, need);
    return kWorkspaceTooSmall;
  }
  AttendArgs a{};
  a.q = q, a.q_st = q_token_stride, a.q_sh = q_head_stride, a.T = T;
  a.Hq = static_cast<int32_t>(Hq), a.Hkv = static_cast<int32_t>(Hkv);
  a.k_cache = k_cache, a.v_cache = v_cache, a.blocks = blocks;
  a.count = static_cast<int32_t>(count);
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  a.scale = scale, a.out = out, a.lse = lse;
  return kv_dispatch(dtype, D, [&](auto e, auto d) -> int {
    kv_attention_kernel<decltype(e), decltype(d)::value>
        <<<dim3(static_cast<unsigned>(T * Hq)), dim3(kWave), 0, static_cast<hipStream_t>(stream)>>>(
            a);
    RT_CHECK_HIP(hipGetLastError());
    return kOk;
  });
}
