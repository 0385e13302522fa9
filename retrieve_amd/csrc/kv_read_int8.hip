// Tokens of the 8-bit paged cache (kv_int8.h) read back in 16 bits: code times its block's scale,
// rounded once, or the open block's row as it is.
//
// A token's values lie a slot from a channel's row of slots, so 16 neighbouring slots are read
// together: a workgroup looks at 64 tokens of one head, finds the runs of tokens within 16 slots,
// and a wave takes a run: its keys row by row, its values 16 bytes of a channel a lane, turned
// through LDS. Bound by memory: a token's codes are read once, its 16 bits written once; 131001
// tokens of 8 heads of 128 channels take 174 us (4.63 TB/s; a large copy beside it 4.81). What that
// took: a run's loads all under way before the first is waited for, and stores of which
// neighbouring lanes write neighbouring bytes (201 us without both); nontemporal loads of the
// values were slower, since a run's 16 bytes of a channel are a part of a line. 2003 tokens of 14
// heads of 64 take 6 us.
#include "../../include/retrieve_amd.h"
#include "kv_int8.h"

namespace rt {

constexpr int kReadWaves = 4;

struct ReadArgs {
  int64_t T;
  int32_t Hkv;
  KvTokens tok;
  KvInt8 cache;
  void *k_out, *v_out;  // [T, Hkv, D]
};

// Eight codes as 16-bit numbers.
template <class E>
__device__ inline typename Kv<E>::V8 widen(int lo, int hi, float scale) {
  typename Kv<E>::V8 x;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int code = static_cast<int8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
    x[i] = static_cast<E>(static_cast<float>(code) * scale);
  }
  return x;
}

template <class E, int D>
__global__ void __launch_bounds__(kReadWaves* kWave) kv_read_int8_kernel(ReadArgs a) {
  using V8 = typename Kv<E>::V8;
  constexpr int C = D / 16, ROWS = kWave / C;  // a row's lanes; rows at once
  constexpr int KP = (16 + ROWS - 1) / ROWS, VP = (D + kWave - 1) / kWave;  // loads a lane
  __shared__ __attribute__((aligned(16))) E turned[kReadWaves][16][D];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = lane_id();
  const int head = static_cast<int>(blockIdx.x % a.Hkv);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / a.Hkv) * kWave;
  // a token a lane: its sequence, slot and page (-1: padding), and whether a run begins with it
  const int64_t mine = t0 + lane;
  const int size = 1 << a.tok.shift;
  int32_t page = -1, seq = -1, pos = -1;
  if (mine < a.T) {
    const KvPlace p = kv_place(a.tok, mine);
    pos = p.pos;
    seq = a.tok.seq_ids[mine];
    if (p.last >= 0) page = kv_page(a.tok, p, p.last);
  }
  const int32_t pos_before = __shfl_up(pos, 1), seq_before = __shfl_up(seq, 1);
  const int32_t page_before = __shfl_up(page, 1);
  const bool begins = mine < a.T && (lane == 0 || (pos & 15) == 0 || seq != seq_before ||
                                     static_cast<int64_t>(pos) != int64_t{pos_before} + 1 ||
                                     page != page_before || page < 0);
  const uint64_t runs = __ballot(begins);
  const int tokens = a.T - t0 < kWave ? static_cast<int>(a.T - t0) : kWave;
  int job = 0;
  for (uint64_t left = runs; left != 0; ++job) {
    const int at = __builtin_ctzll(left);
    left &= left - 1;
    if (job % kReadWaves != wave) continue;
    const int end = left != 0 ? __builtin_ctzll(left) : tokens, n = end - at;
    const int32_t pg = __builtin_amdgcn_readlane(page, at);
    const int32_t sq = __builtin_amdgcn_readlane(seq, at);
    const int slot = __builtin_amdgcn_readlane(pos, at) & (size - 1);
    const int64_t to = ((t0 + at) * a.Hkv + head) * D, step = static_cast<int64_t>(a.Hkv) * D;
    E* k_out = static_cast<E*>(a.k_out) + to;
    E* v_out = static_cast<E*>(a.v_out) + to;
    const int64_t row = static_cast<int64_t>(pg) * a.Hkv + head;
    const float ks = pg >= 0 ? a.cache.k_scales[row] : 0.0f;
    const float vs = pg >= 0 ? a.cache.v_scales[row] : 0.0f;
    const int64_t full = (row << a.tok.shift) * D;
    const int64_t open = ((static_cast<int64_t>(sq) * a.Hkv + head) << a.tok.shift) * D;
    const int c = lane % C, r0 = lane / C < ROWS ? lane / C : 16;
    // everything of the run under way at once: keys row by row, values 16 slots of a channel
    typedef int V2i __attribute__((ext_vector_type(2)));
    V2i kc[KP][2];  // (chunks c and c + C of 8 channels: neighbours store side by side)
    v4i vc[VP];
    V8 kt[KP][2], vt[VP][2];
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int r = r0 + i * ROWS;
      if (r >= n || pg < 0) continue;
      if (ks > 0.0f) {
        const V2i* from =
            reinterpret_cast<const V2i*>(a.cache.k_codes + full + (slot + r) * D);
        kc[i][0] = __builtin_nontemporal_load(from + c);
        kc[i][1] = __builtin_nontemporal_load(from + c + C);
      } else {
        const V8* from = reinterpret_cast<const V8*>(static_cast<const E*>(a.cache.k_tail) + open +
                                                     (slot + r) * D);
        kt[i][0] = from[c];
        kt[i][1] = from[c + C];
      }
    }
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const int d = lane + i * kWave;
      const int64_t from = (static_cast<int64_t>(d) << a.tok.shift) + (slot & ~15);
      if (d >= D || pg < 0) continue;
      if (vs > 0.0f) {
        // (the other runs of the block take the rest of the line: not streamed)
        vc[i] = *reinterpret_cast<const v4i*>(a.cache.v_codes + full + from);
      } else {
        const V8* tail = reinterpret_cast<const V8*>(static_cast<const E*>(a.cache.v_tail) + open +
                                                     from);
        vt[i][0] = tail[0];
        vt[i][1] = tail[1];
      }
    }
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int r = r0 + i * ROWS;
      if (r >= n) continue;
      V8 x[2] = {V8{}, V8{}};
      if (ks > 0.0f) {
        x[0] = widen<E>(kc[i][0][0], kc[i][0][1], ks);
        x[1] = widen<E>(kc[i][1][0], kc[i][1][1], ks);
      } else if (pg >= 0) {
        x[0] = kt[i][0];
        x[1] = kt[i][1];
      }
      V8* out = reinterpret_cast<V8*>(k_out + r * step);
      out[c] = x[0];
      out[c + C] = x[1];
    }
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const int d = lane + i * kWave;
      if (d >= D) continue;
      V8 x[2] = {V8{}, V8{}};
      if (vs > 0.0f) {
        x[0] = widen<E>(vc[i][0], vc[i][1], vs);
        x[1] = widen<E>(vc[i][2], vc[i][3], vs);
      } else if (pg >= 0) {
        x[0] = vt[i][0];
        x[1] = vt[i][1];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) turned[wave][e][d] = x[e >> 3][e & 7];
    }
    wave_sync_memory();
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int r = r0 + i * ROWS;
      if (r >= n) continue;
      const V8* from = reinterpret_cast<const V8*>(turned[wave][(slot & 15) + r]);
      V8* out = reinterpret_cast<V8*>(v_out + r * step);
      out[c] = from[c];
      out[c + C] = from[c + C];
    }
    wave_sync_memory();
  }
}

}  // namespace rt

using namespace rt;

extern "C" int rt_kv_read_int8(const int8_t* k_codes, const int8_t* v_codes, const float* k_scales,
                               const float* v_scales, const void* k_tail, const void* v_tail,
                               int64_t T, int64_t Hkv, int64_t D, int dtype, int64_t P,
                               int64_t page, const int32_t* positions, const int32_t* seq_ids,
                               const int32_t* page_table, int64_t B, int64_t max_pages, void* k_out,
                               void* v_out, rt_stream_t stream) {
  if (const int st = kv_check(T, Hkv, Hkv, D, dtype, B, max_pages, P, page)) return st;
  if (T == 0) return kOk;
  const KvInt8 cache{const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes),
                     const_cast<float*>(k_scales), const_cast<float*>(v_scales),
                     const_cast<void*>(k_tail), const_cast<void*>(v_tail)};
  if (const int st = kv_check_int8(cache, B, P)) return st;
  RT_CHECK_ARG(positions && seq_ids && k_out && v_out, "null pointer");
  RT_CHECK_ARG(B * max_pages == 0 || page_table, "null page table");
  RT_CHECK_ARG(kv_rows_aligned(k_out, 0, 0) && kv_rows_aligned(v_out, 0, 0),
               "rows must start on 16 bytes");
  const int64_t grid = cdiv(T, kWave) * Hkv;
  RT_CHECK_ARG(grid <= INT32_MAX, "too many tokens");
  ReadArgs a{};
  a.T = T, a.Hkv = static_cast<int32_t>(Hkv);
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  a.cache = cache, a.k_out = k_out, a.v_out = v_out;
  return kv_dispatch(dtype, D, [&](auto e, auto d) -> int {
    kv_read_int8_kernel<decltype(e), decltype(d)::value>
        <<<dim3(static_cast<unsigned>(grid)), dim3(kReadWaves * kWave), 0,
           static_cast<hipStream_t>(stream)>>>(a);
    RT_CHECK_HIP(hipGetLastError());
    return kOk;
  });
}
