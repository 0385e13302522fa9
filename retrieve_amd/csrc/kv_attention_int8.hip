// Attention over the 8-bit paged cache: the entry point, and how a call is spread over the GPU. The
// kernels: kv_attend_int8.h.
#include <cmath>

#include "../../include/retrieve_amd.h"
#include "kv_attend_int8.h"

namespace rt {

inline AttendInt8Plan attend_int8_plan(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t seqs,
                                       int64_t page, int64_t count) {
  AttendInt8Plan p;
  const int64_t G = Hq / Hkv;
  p.tiles = static_cast<int32_t>(cdiv(G, 16));
  p.rows = T * Hkv * p.tiles;
  p.parts = 0;
  // Prompts: as many neighbouring tokens a workgroup as two tiles of columns hold, the table of
  // their lists takes and leave two workgroups a CU. Two or more join their lists: over 1024 keys
  // of 8 heads of 128 channels 128 tokens take 25 us and 37 split, 256 30 and 59, 1024 97 and 209
  // (of 64 channels 128 tokens 17 and 21, of 256 73 and 120). One token a workgroup would take what
  // it takes split where the lists are short (64 tokens: 20 and 21), and longer where they are not.
  // Where most sequences have one token there is less to share: 256 tokens of 250 take 135 joined
  // and 125 split, of 128 sequences (64 blocks each) 280 and 253, of 64 (16 blocks) 63 and 89.
  int64_t joined = T > 2 * seqs && G <= 16 ? 2 * (16 / G) : 0;
  while (joined > 1 && (joined * count > kJoinEntries || cdiv(T, joined) * Hkv < 512)) joined /= 2;
  p.joined = static_cast<int32_t>(joined);
  if (joined > 1) {
    p.tiles = joined > 16 / G ? 2 : 1;
    return p;
  }
  // Workgroups of four waves for two on every CU, each wave with a unit of 64 keys at least.
  const int64_t most = cdiv(count * page, 64 * kAttendWaves);
  const int64_t want = cdiv(512, p.rows > 0 ? p.rows : 1);
  p.parts = static_cast<int32_t>(want < most ? want : most);
  if (p.parts < 1) p.parts = 1;
  return p;
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_kv_attention_int8_workspace(int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                                 int64_t page, int64_t count) {
  if (Hkv < 1 || T < 1) return 0;
  // (as many sequences as tokens: the lists are split, the only form that has parts to keep)
  const AttendInt8Plan p = attend_int8_plan(T, Hq, Hkv, D, T, page, count);
  return p.parts > 1 ? static_cast<size_t>(p.rows) * p.parts * 16 * (D + 2) * sizeof(float) : 0;
}

extern "C" int rt_kv_attention_int8(
    const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t T, int64_t Hq,
    int64_t Hkv, int64_t D, int dtype, const int8_t* k_codes, const int8_t* v_codes,
    const float* k_scales, const float* v_scales, const void* k_tail, const void* v_tail, int64_t P,
    int64_t page, const int32_t* blocks, int64_t count, const int32_t* positions,
    const int32_t* seq_ids, const int32_t* page_table, int64_t B, int64_t max_pages, float scale,
    int64_t sequences, void* out, float* lse, void* workspace, size_t workspace_bytes,
    rt_stream_t stream) {
  if (const int st = kv_check(T, Hq, Hkv, D, dtype, B, max_pages, P, page)) return st;
  RT_CHECK_ARG(count >= 0 && count <= (1 << 20), "count must be in [0, 2^20], got %lld",
               static_cast<long long>(count));
  RT_CHECK_ARG(std::isfinite(scale * kLog2e), "the scale must be finite, got %g",
               static_cast<double>(scale));
  RT_CHECK_ARG(sequences >= 0, "sequences must not be negative, got %lld",
               static_cast<long long>(sequences));
  if (T == 0) return kOk;
  RT_CHECK_ARG(q && positions && seq_ids && out && lse && (count == 0 || blocks), "null pointer");
  RT_CHECK_ARG(B * max_pages == 0 || page_table, "null page table");
  const KvInt8 cache{const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes),
                     const_cast<float*>(k_scales), const_cast<float*>(v_scales),
                     const_cast<void*>(k_tail), const_cast<void*>(v_tail)};
  if (const int st = kv_check_int8(cache, B, P)) return st;
  RT_CHECK_ARG(kv_rows_aligned(q, q_token_stride, q_head_stride) && kv_rows_aligned(out, 0, 0),
               "rows must start on 16 bytes");
  RT_CHECK_ARG(T * Hq <= INT32_MAX, "too many tokens");
  const size_t need = rt_kv_attention_int8_workspace(T, Hq, Hkv, D, page, count);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
    set_error("workspace too small: %zu < %zu", workspace_bytes, need);
    return kWorkspaceTooSmall;
  }
  const AttendInt8Plan plan = attend_int8_plan(T, Hq, Hkv, D, sequences, page, count);
  AttendInt8Args a{};
  a.q = q, a.q_st = q_token_stride, a.q_sh = q_head_stride, a.T = T;
  a.Hq = static_cast<int32_t>(Hq), a.Hkv = static_cast<int32_t>(Hkv);
  a.G = a.Hq / a.Hkv, a.tiles = plan.tiles;
  a.cache = cache, a.blocks = blocks;
  a.count = static_cast<int32_t>(count);
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  // (a scale of 0 becomes the least number: the scores are 0 all the same, and -inf stays -inf)
  a.scale = fmaxf(fabsf(scale * kLog2e), 1.17549435e-38f), a.minus = scale < 0.0f;
  a.size = std::frexp(a.scale, &a.power);
  a.out = out, a.lse = lse, a.parts = plan.parts;
  a.part_out = static_cast<float*>(workspace);
  a.part_ml = a.part_out + (plan.parts > 1 ? plan.rows * plan.parts * 16 * D : 0);
  a.joined = plan.joined;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool small = a.tok.shift < 6;
  if (dtype == kKvBf16) {
    return small ? attend_int8_bf16_16(D, a, plan, s) : attend_int8_bf16_64(D, a, plan, s);
  }
  return small ? attend_int8_f16_16(D, a, plan, s) : attend_int8_f16_64(D, a, plan, s);
}
