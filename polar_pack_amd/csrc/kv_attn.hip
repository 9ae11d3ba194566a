// Attention of a call's tokens to the cache: how a call is dealt, the entry points, and the few-row kernel's 8-bit forms.
#include "kv_attn_split.h"

namespace pp {

// The row tile by the mean rows of a sequence and head (tokens x query heads a key head), in us on both sides,
// sequences of int8 codes of 16 query and 2 key heads of 128 unless said:
// * 16 or 32 rows at 24: 4 sequences of 4000 tokens 17.6 / 24.4, 64 of 8000 90 / 65.  From 17 rows on 32, which a
//   large batch reads its codes once for.
// * 32 rows or the many-row kernel's 128: at 48 rows 4 of 40,000 50 / 67, 64 of 2000 31 / 65, 200 of 1000 76 / 87; at
//   64, 4 of 4000 26.6 / 26.6, 64 of 8000 107 / 158 (8 query and key heads, e4m3, 64 of up to 500: 55 / 50); at 128,
//   75 / 72, 57 / 70 and 183 / 167.  To 64 rows 32.  At 256 values a head the two are even sooner: at 48, 4 of 4000 45 / 37,
//   64 of 2000 58 / 101, 24 of 4000 74 / 75; to 32 rows there.
// * 128 rows or 256, which 8 wavefronts share, at 128: 72 / 70, 167 / 152 (64 values a head, 8 key heads: 24 of 4000
//   100 / 105, 64 of 8000 469 / 409); 256 from 129 on, and never for more than 128 values, whose sums fill the registers.
// A batch of prompts and single tokens takes what its mean asks for: a prompt of 2000 and 60 single tokens of
// 1000-8000 125 (152 in tiles of 32), of 500 105 (57 in tiles of 32).
//
// Shares for a workgroup a CU, two of few rows with 64 values a head (kv_attn_split_kernel): one / two at 16 rows, 24
// sequences in a window of 2000 26 / 23, 64 of up to 8190 63 / 56, 4 of 40,000 36 / 37; at 32 rows 32 / 29, 83 / 68,
// 50 / 48; alike with e4m3 and pages of 16.  None for batches that one workgroup cannot count, and none for
// prompts of two row tiles a CU and more.  Cut / whole, 4 prompts: 256 row tiles 53 / 50, 384 117 / 68, 512 144 / 99,
// 1024 503 / 333; behind 4000 tokens each 128 115 / 144, 256 193 / 172, 320 246 / 288, 384 301 / 308, 448 363 / 328.
// What lies behind a prompt only the device knows; whole tiles never lose from 448 on.
//
// 4 bits, few rows, to 128 values a head: two workgroups a CU where there are as many row tiles as CUs, so that few are
// cut into many parts.  One / two, in us: 256 row tiles (128 sequences of 1000-8000, 2 key heads) 45.9 / 43.2, 512 (64 of
// 500-1000, 8) 33.1 / 30.7; 128 (16 of 8000-16,000, 8) 50.2 / 51.0, 64 (8 of 30-40,000) 63.8 / 64.6, 8 21.9 / 25.8.
static AttnPlan attn_plan(int64_t heads, int64_t D, int64_t block, int64_t width, int64_t batch, int64_t tokens,
                          int64_t q_heads, bool four) {
  const int64_t group = q_heads / heads, rows = (tokens * group + batch - 1) / batch, cus = device_cu_count();
  AttnPlan P;
  P.rows = rows <= 16 ? 16 : rows <= (D <= 192 ? 64 : 32) ? 32 : rows <= 128 || D > 128 ? 128 : 256;
  const int64_t row_tiles = tokens * group / P.rows + batch + 1;
  const bool two = P.rows <= 32 && (D == 64 || (four && P.rows == 16 && D == 128 && batch * heads >= cus));
  P.shares = ((two ? 2 : 1) * cus + heads - 1) / heads;
  const int64_t most = row_tiles * ((width * block + 255) / 256 + 1);       // of 4 tiles each
  if (P.shares > most) P.shares = most;
  if (batch > KV_DEAL_BATCH || (P.rows > 32 && tokens * q_heads / P.rows >= 2 * cus)) P.shares = 0;
  P.grid = P.shares ? P.shares : row_tiles;
  P.bytes = heads * P.shares * (2 * P.rows * (D + 4) * 4 + (int64_t)sizeof(ManyPart));
  P.counts = P.rows <= 32 ? heads * P.shares * 4 : 0;
  return P;
}

}  // namespace pp

using namespace pp;

// What a call over codes of this kind needs; nothing where the sizes are none.
static AttnPlan attn_sizes(int64_t heads, int64_t D, int64_t block, int64_t width, int64_t batch, int64_t tokens,
                           int64_t q_heads, bool four) {
  if (heads <= 0 || D <= 0 || block <= 0 || width <= 0 || batch <= 0 || tokens <= 0 || q_heads < heads) return AttnPlan{};
  return attn_plan(heads, D, block, width, batch, tokens, q_heads, four);
}

extern "C" int64_t pp_kv_attention_codes_workspace_size(int64_t codes, int64_t heads, int64_t head_dim, int64_t block,
                                                        int64_t table_width, int64_t batch, int64_t tokens, int64_t q_heads) {
  return attn_sizes(heads, head_dim, block, table_width, batch, tokens, q_heads, codes == PP_KV_E2M1).bytes;
}

extern "C" int64_t pp_kv_attention_codes_counts_size(int64_t codes, int64_t heads, int64_t head_dim, int64_t block,
                                                     int64_t table_width, int64_t batch, int64_t tokens, int64_t q_heads) {
  return attn_sizes(heads, head_dim, block, table_width, batch, tokens, q_heads, codes == PP_KV_E2M1).counts;
}

extern "C" int64_t pp_kv_attention_workspace_size(int64_t heads, int64_t head_dim, int64_t block, int64_t table_width,
                                                  int64_t batch, int64_t tokens, int64_t q_heads) {
  const int64_t eight = attn_sizes(heads, head_dim, block, table_width, batch, tokens, q_heads, false).bytes;
  const int64_t four = attn_sizes(heads, head_dim, block, table_width, batch, tokens, q_heads, true).bytes;
  return eight > four ? eight : four;
}

extern "C" int64_t pp_kv_attention_counts_size(int64_t heads, int64_t head_dim, int64_t block, int64_t table_width,
                                               int64_t batch, int64_t tokens, int64_t q_heads) {
  const int64_t eight = attn_sizes(heads, head_dim, block, table_width, batch, tokens, q_heads, false).counts;
  const int64_t four = attn_sizes(heads, head_dim, block, table_width, batch, tokens, q_heads, true).counts;
  return eight > four ? eight : four;
}

extern "C" int pp_kv_attention(const pp_kv_cache* cache, const void* q, int64_t q_st, int64_t q_sh, int64_t q_heads,
                               int dtype, int64_t tokens, const int32_t* table, int64_t table_ld, int64_t table_width,
                               const int32_t* lengths, const int32_t* cu, int64_t batch, int causal, int64_t window,
                               float scale, void* out, float* lse, void* workspace, int64_t workspace_size,
                               void* counts, int64_t counts_size, void* stream) {
  AttnArgs A;
  int rc = kv_check_cache(cache, &A.C);
  if (rc) return rc;
  rc = kv_check_seqs(A.C, table, table_ld, table_width, lengths, cu, batch, tokens, &A.S);
  if (rc) return rc;
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16, "pp_kv_attention: dtype %d is not PP_F16 or PP_BF16", dtype);
  PP_REQUIRE(q_heads > 0 && q_heads % A.C.heads == 0 && q_heads <= 65535,
             "pp_kv_attention: %lld query heads over %d heads", (long long)q_heads, A.C.heads);
  PP_REQUIRE(tokens * q_heads <= INT32_MAX, "pp_kv_attention: too many rows");
  PP_REQUIRE(window >= 0 && (causal || window == 0), "pp_kv_attention: a window needs causal attention");
  if (tokens == 0) return PP_OK;
  PP_REQUIRE(q && out, "pp_kv_attention: null queries or output");
  PP_REQUIRE(aligned(q, 2) && aligned(out, 16), "pp_kv_attention: queries or output are not aligned");
  const AttnPlan P = attn_plan(A.C.heads, cache->head_dim, A.C.block, table_width, batch, tokens, q_heads,
                               cache->codes == PP_KV_E2M1);
  PP_REQUIRE(P.bytes == 0 || (workspace && workspace_size >= P.bytes && aligned(workspace, 16)),
             "pp_kv_attention: workspace of %lld bytes at a 16-byte boundary needed", (long long)P.bytes);
  PP_REQUIRE(P.counts == 0 || (counts && counts_size >= P.counts && aligned(counts, 4)),
             "pp_kv_attention: %lld bytes of counts, zero, needed", (long long)P.counts);
  A.q = (const uint16_t*)q;
  A.q_st = q_st; A.q_sh = q_sh;
  A.q_vec = aligned(q, 16) && q_st % 8 == 0 && q_sh % 8 == 0;
  A.out = (uint16_t*)out;
  A.lse = lse;
  A.parts = (float*)workspace;
  A.q_heads = (int)q_heads;
  A.group = (int)q_heads / A.C.heads;
  A.window = (int)(window < INT32_MAX ? window : 0);
  A.causal = causal;
  A.shares = (int)P.shares;
  A.desc = P.shares ? (ManyPart*)(A.parts + A.C.heads * P.shares * 2 * P.rows * (cache->head_dim + 4)) : nullptr;
  A.counts = (uint32_t*)counts;
  PP_REQUIRE(P.grid <= INT32_MAX, "pp_kv_attention: too many rows");
  A.scale = scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
  const int D = cache->head_dim;
  if (P.rows > 32) return kv_attn_many(A, P, D, cache->codes, dtype, st);
  if (cache->codes == PP_KV_E2M1) return kv_attn_split4(A, P, D, dtype, st);
  if (cache->codes == PP_KV_INT8)
    return dtype == PP_F16 ? attn_width<PP_KV_INT8, IoF16>(A, P, D, st) : attn_width<PP_KV_INT8, IoBf16>(A, P, D, st);
  return dtype == PP_F16 ? attn_width<PP_KV_E4M3, IoF16>(A, P, D, st) : attn_width<PP_KV_E4M3, IoBf16>(A, P, D, st);
}
