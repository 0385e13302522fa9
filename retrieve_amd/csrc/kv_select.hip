// The best blocks of each token and key/value head, by the int8 bounds' score.
//
// A query head's row is quantised as the bounds are (codes c, scale s); block b's score with it is
// (c . mid_b + |c| . half_b) s times the block's scale, an upper bound on what any of its keys can
// score, and the group's score is the largest of its heads'. The sum is an int32 (at most
// 2 * 256 * 127^2 < 2^23, so exact as fp32 too); the two products are rounded once each, in this order,
// and rounding is monotone, so the largest over the heads is taken before the block's scale.
#include <type_traits>

#include "../../include/retrieve_amd.h"
#include "kv_common.h"

namespace rt {

constexpr int kSelectThreads = 256;

struct SelectArgs {
  const void* q;
  int64_t q_st, q_sh;
  int64_t T;
  int32_t Hq, Hkv;
  const int8_t* bounds;
  const float* scales;
  KvTokens tok;
  int32_t count, sink, recent;
  int32_t* out;    // [T, Hkv, count]
  uint32_t* keys;  // [T * Hkv, max_pages]
};

// The key of a candidate's score (0: not a candidate). A score that is not a number is the least.
__device__ inline uint32_t score_key(float s) {
  return key_of_f32(s == s ? s : -INFINITY);
}

template <class E, int D>
__global__ void __launch_bounds__(kSelectThreads) kv_score_kernel(SelectArgs a) {
  __shared__ __attribute__((aligned(16))) int8_t codes[2 * D];
  __shared__ float tops[kSelectThreads / kWave];
  const int64_t t = blockIdx.x / a.Hkv;
  const int h = blockIdx.x % a.Hkv;
  const KvPlace p = kv_place(a.tok, t);
  const int32_t end = p.last - a.recent + 1;  // candidates: [sink, end)
  if (end <= a.sink) return;
  uint32_t* keys = a.keys + static_cast<int64_t>(blockIdx.x) * a.tok.max_pages;
  const int G = a.Hq / a.Hkv;
  for (int g = 0; g < G; ++g) {
    const E* q = static_cast<const E*>(a.q) + t * a.q_st + (h * G + g) * a.q_sh;
    const int d = threadIdx.x;
    const float x = d < D ? static_cast<float>(q[d]) : 0.0f;
    float top = fabsf(x);
    for (int i = 1; i < kWave; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
    if (lane_id() == 0) tops[threadIdx.x / kWave] = top;
    __syncthreads();
    top = kKvTopFloor;
    for (int w = 0; w < kSelectThreads / kWave; ++w) top = fmaxf(top, tops[w]);
    if (d < D) {
      const int c = kv_code(x, top);
      codes[d] = static_cast<int8_t>(c);
      codes[D + d] = static_cast<int8_t>(c < 0 ? -c : c);
    }
    __syncthreads();
    const float scale = top / 127.0f;
    for (int32_t b = a.sink + threadIdx.x; b < end; b += kSelectThreads) {
      const int32_t page = kv_page(a.tok, p, b);
      const int64_t row = static_cast<int64_t>(page < 0 ? 0 : page) * a.Hkv + h;
      int dot = 0;
      if (page >= 0) {
        for (int i = 0; i < 2 * D; i += 4) {
          dot = __builtin_amdgcn_sdot4(*reinterpret_cast<const int*>(a.bounds + row * 2 * D + i),
                                       *reinterpret_cast<const int*>(codes + i), dot, false);
        }
      }
      const float s = static_cast<float>(dot) * scale;
      const float best = g == 0 ? s : fmaxf(s, __uint_as_float(keys[b]));
      keys[b] = g + 1 < G ? __float_as_uint(best)
                          : page < 0 ? 0u : score_key(best * a.scales[row]);
    }
    __syncthreads();
  }
}

// Keeps the forced blocks and the best `count - forced` candidates of one row: the bits of the
// last kept key from the top, then one pass in block order.
__global__ void __launch_bounds__(kSelectThreads) kv_keep_kernel(SelectArgs a) {
  __shared__ int part[kSelectThreads / kWave];
  const int64_t t = blockIdx.x / a.Hkv;
  const KvPlace p = kv_place(a.tok, t);
  const uint32_t* keys = a.keys + static_cast<int64_t>(blockIdx.x) * a.tok.max_pages;
  int32_t* out = a.out + static_cast<int64_t>(blockIdx.x) * a.count;
  const int32_t end = p.last - a.recent + 1;
  const int want = a.count - a.sink - a.recent;
  auto total = [&](auto pred) {
    int n = 0;
    for (int32_t b = a.sink + threadIdx.x; b < end; b += kSelectThreads) n += pred(keys[b]) ? 1 : 0;
    for (int i = 1; i < kWave; i <<= 1) n += __shfl_xor(n, i);
    __syncthreads();
    if (lane_id() == 0) part[threadIdx.x / kWave] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < kSelectThreads / kWave; ++w) n += part[w];
    return n;
  };
  // the largest key that at least `want` candidates reach (1 if fewer are candidates at all)
  uint32_t cut = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t probe = cut | (1u << bit);
    if (total([&](uint32_t k) { return k >= probe; }) >= want) cut = probe;
  }
  if (cut == 0) cut = 1;
  const int above = total([&](uint32_t k) { return k > cut; });
  int ties = want - above;  // of the cut's own key, the lowest blocks
  int at = 0;
  for (int32_t b0 = 0; b0 <= p.last; b0 += kSelectThreads) {
    const int32_t b = b0 + static_cast<int32_t>(threadIdx.x);
    const bool forced = b <= p.last && (b < a.sink || b >= end);
    const uint32_t key = b <= p.last && !forced ? keys[b] : 0u;
    auto before = [&](bool x, int& all) {  // set lanes before this one, and all of them
      const uint64_t m = __ballot(x);
      __syncthreads();
      if (lane_id() == 0) part[threadIdx.x / kWave] = __popcll(m);
      __syncthreads();
      int n = __popcll(m & ((uint64_t{1} << lane_id()) - 1));
      all = 0;
      for (int w = 0; w < kSelectThreads / kWave; ++w) {
        n += w < static_cast<int>(threadIdx.x / kWave) ? part[w] : 0;
        all += part[w];
      }
      return n;
    };
    int n_ties, n_kept;
    const int my_tie = before(key == cut, n_ties);
    const bool keep = forced || key > cut || (key == cut && my_tie < ties);
    ties -= n_ties < ties ? n_ties : ties;
    const int slot = at + before(keep, n_kept);
    if (keep) out[slot] = b;
    at += n_kept;
  }
  for (int i = at + threadIdx.x; i < a.count; i += kSelectThreads) out[i] = -1;
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_kv_select_workspace(int64_t T, int64_t Hkv, int64_t max_pages) {
  return static_cast<size_t>(T) * Hkv * max_pages * sizeof(uint32_t);
}

extern "C" int rt_kv_select(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t T,
                            int64_t Hq, int64_t Hkv, int64_t D, int dtype, const int8_t* bounds,
                            const float* bound_scales, int64_t P, int64_t page,
                            const int32_t* positions, const int32_t* seq_ids,
                            const int32_t* page_table, int64_t B, int64_t max_pages, int64_t count,
                            int64_t sink, int64_t recent, int32_t* out, void* workspace,
                            size_t workspace_bytes, rt_stream_t stream) {
  if (const int st = kv_check(T, Hq, Hkv, D, dtype, B, max_pages, P, page)) return st;
  RT_CHECK_ARG(count >= 1 && count <= 1024, "count must be in [1, 1024], got %lld",
               static_cast<long long>(count));
  RT_CHECK_ARG(sink >= 0 && recent >= 1 && sink + recent <= count,
               "sink >= 0 and recent >= 1 must fit in count");
  if (T == 0) return kOk;
  RT_CHECK_ARG(q && positions && seq_ids && out, "null pointer");
  RT_CHECK_ARG(B * max_pages == 0 || page_table, "null page table");
  RT_CHECK_ARG(P == 0 || (bounds && bound_scales), "null bounds");
  RT_CHECK_ARG(kv_rows_aligned(q, q_token_stride, q_head_stride) && kv_rows_aligned(bounds, 0, 0),
               "rows must start on 16 bytes");
  RT_CHECK_ARG(T * Hkv <= INT32_MAX, "too many tokens");
  const size_t need = rt_kv_select_workspace(T, Hkv, max_pages);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
    set_error("workspace too small: %zu < %zu", workspace_bytes, need);
    return kWorkspaceTooSmall;
  }
  SelectArgs a{};
  a.q = q, a.q_st = q_token_stride, a.q_sh = q_head_stride, a.T = T;
  a.Hq = static_cast<int32_t>(Hq), a.Hkv = static_cast<int32_t>(Hkv);
  a.bounds = bounds, a.scales = bound_scales;
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  a.count = static_cast<int32_t>(count), a.sink = static_cast<int32_t>(sink);
  a.recent = static_cast<int32_t>(recent), a.out = out, a.keys = static_cast<uint32_t*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 g(static_cast<unsigned>(T * Hkv)), b(kSelectThreads);
  return kv_dispatch(dtype, D, [&](auto e, auto d) -> int {
    kv_score_kernel<decltype(e), decltype(d)::value><<<g, b, 0, s>>>(a);
    kv_keep_kernel<<<g, b, 0, s>>>(a);
    RT_CHECK_HIP(hipGetLastError());
    return kOk;
  });
}
