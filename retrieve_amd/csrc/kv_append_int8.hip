// Appending to the 8-bit paged cache: the entry point, and how a call is spread over the GPU. The
// kernels: kv_append_int8.h.
#include "../../include/retrieve_amd.h"
#include "kv_append_int8.h"

using namespace rt;

extern "C" int rt_kv_append_int8(
    const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
    int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
    int64_t v_head_stride, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype,
    const void* q_weight, const void* k_weight, int wide_weights, double eps, const float* cos_sin,
    int64_t table_len, int64_t rot, int interleaved, const int32_t* positions,
    const int32_t* seq_ids, const int32_t* page_table, int64_t B, int64_t max_pages,
    int8_t* k_codes, int8_t* v_codes, float* k_scales, float* v_scales, void* k_tail, void* v_tail,
    int64_t P, int64_t page, int8_t* bounds, float* bound_scales, void* q_out,
    rt_stream_t stream) {
  if (const int st = kv_check(T, Hq, Hkv, D, dtype, B, max_pages, P, page)) return st;
  if (const int st = kv_check_turn(T, D, cos_sin, table_len, rot, q_weight, k_weight, eps)) {
    return st;
  }
  if (T == 0) return kOk;
  const KvInt8 cache{k_codes, v_codes, k_scales, v_scales, k_tail, v_tail};
  if (const int st = kv_check_int8(cache, B, P)) return st;
  RT_CHECK_ARG(q && k && v && positions && seq_ids && q_out, "null pointer");
  RT_CHECK_ARG(B * max_pages == 0 || page_table, "null page table");
  RT_CHECK_ARG(P == 0 || (bounds && bound_scales), "null bounds");
  RT_CHECK_ARG(kv_rows_aligned(q, q_token_stride, q_head_stride) &&
                   kv_rows_aligned(k, k_token_stride, k_head_stride) &&
                   kv_rows_aligned(v, v_token_stride, v_head_stride) &&
                   kv_rows_aligned(q_out, 0, 0),
               "rows must start on 16 bytes");
  WriteArgs a{};
  static_cast<TurnArgs&>(a) = kv_turn_args(cos_sin, table_len, rot, q_weight, k_weight,
                                           wide_weights, eps);
  a.q = q, a.k = k, a.v = v;
  a.q_st = q_token_stride, a.q_sh = q_head_stride;
  a.k_st = k_token_stride, a.k_sh = k_head_stride;
  a.v_st = v_token_stride, a.v_sh = v_head_stride;
  a.T = T, a.Hq = static_cast<int32_t>(Hq), a.Hkv = static_cast<int32_t>(Hkv);
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  a.cache = cache, a.bounds = bounds, a.bound_scales = bound_scales;
  a.q_out = q_out;
  // Few tokens: a token's rows over as many waves as have one each. Many: one wave a token.
  const int64_t all = cdiv(Hq + 2 * Hkv, kWave / (D / 16)), parts = cdiv(4096, T);
  a.row_parts = static_cast<int32_t>(parts < all ? parts : all);
  // Few tokens may all complete a block in one step: a workgroup for each, every head and keys and
  // values, up to 1024 of them; in prompts 64 tokens a workgroup.
  const int64_t tile = next_pow2(cdiv(T * Hkv, 512));
  a.tile = static_cast<int32_t>(tile < 64 ? tile : 64);
  const int64_t fill_groups = cdiv(T, a.tile) * Hkv * 2;
  const int64_t grid = fill_groups + cdiv(T * a.row_parts, write_threads(D) / kWave);
  RT_CHECK_ARG(grid <= INT32_MAX, "too many tokens");
  a.fill_groups = static_cast<uint32_t>(fill_groups);
  // a block's codes of values; least and largest keys (32 numbers of 16 bits a thread)
  const int64_t codes = page * D, ends = write_threads(D) * 32 * 2;
  const unsigned lds = static_cast<unsigned>(codes > ends ? codes : ends);
  AppendInt8* const launch =
      dtype == kKvBf16 ? (D > 128 ? append_int8_bf16_256 : append_int8_bf16_128)
                       : (D > 128 ? append_int8_f16_256 : append_int8_f16_128);
  return launch(D, a, static_cast<unsigned>(grid), lds, interleaved != 0,
                static_cast<hipStream_t>(stream));
}
