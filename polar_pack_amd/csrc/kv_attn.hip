// Attention of a call's tokens to the 8-bit cache.
//
// Row (token, query head) with position p = lengths[b] - n_b + i sees the keys j of
// (p - window, p] (causal) or of [0, length):
//   s_j = scale * ks * sum_d q_d kcode_jd,   o_d = sum_j e^(s_j - m) vs vcode_jd / sum_j e^(s_j - m).
#include "kv_common.h"

namespace pp {

struct AttnArgs {
  KvCache C;
  KvSeqs S;
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* out;
  float* lse;
  int q_heads, group, window, causal;
  float scale;      // of the scores, times log2(e)
};

template <int CODES, typename IO, int D>
__global__ __launch_bounds__(64) void kv_attn_rows_kernel(const AttnArgs A) {
  using Q = KvCodes<CODES>;
  const KvCache& C = A.C;
  const KvSeqs& S = A.S;
  const int row = blockIdx.x, hq = blockIdx.y, h = hq / A.group, lane = threadIdx.x;
  __shared__ float qf[D], pw[64];
  int b = row;
  if (S.cu != nullptr) b = kv_find(S, row, 1, 1, 0);
  const int s0 = kv_start(S, b), n = kv_start(S, b + 1) - s0;
  int64_t len = 0, pos = -1;
  if (b < S.batch && n > 0) {
    len = S.lengths[b];
    pos = len - n + (row - s0);
    if (len > ((int64_t)S.width << C.shift)) len = (int64_t)S.width << C.shift;
  }
  const int64_t hi = pos < 0 ? 0 : A.causal ? (pos + 1 < len ? pos + 1 : len) : len;
  const int64_t lo = A.window && pos >= A.window ? pos - A.window + 1 : 0;
  for (int d = lane; d < D; d += 64) qf[d] = IO::get(A.q[row * A.q_st + hq * A.q_sh + d]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[D / 64] = {};
  for (int64_t t0 = lo & ~63; t0 < hi; t0 += 64) {
    const int64_t j = t0 + lane;
    float s = -INFINITY, vscale = 0.f;
    if (j >= lo && j < hi) {
      const int page = S.table[(int64_t)b * S.ld + (j >> C.shift)];
      if (page >= 0 && page < C.pages) {
        const int64_t ph = (int64_t)page * C.heads + h;
        const uint32_t* k = reinterpret_cast<const uint32_t*>(C.k + (ph * C.block + (j & (C.block - 1))) * D);
        float acc = 0.f;
        for (int w = 0; w < D / 4; ++w) {
          float f[4];
          Q::unpack(k[w], f);
          acc += f[0] * qf[4 * w] + f[1] * qf[4 * w + 1] + f[2] * qf[4 * w + 2] + f[3] * qf[4 * w + 3];
        }
        s = acc * C.ks[ph] * A.scale;
        vscale = C.vs[ph];
      }
    }
    float top = s;
    for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float mn = fmaxf(m, top);
    const float keep = mn == -INFINITY ? 1.f : exp2f(m - mn);
    const float p = s == -INFINITY ? 0.f : exp2f(s - mn);
    l = l * keep + p;
    m = mn;
    pw[lane] = p * vscale;
    __syncthreads();
    for (int x = 0; x < D / 64; ++x) {
      const int d = lane + 64 * x;
      float acc = o[x] * keep;
      for (int t = 0; t < 64; ++t) {
        const float w = pw[t];
        if (w == 0.f) continue;
        const int64_t jj = t0 + t;
        const int page = S.table[(int64_t)b * S.ld + (jj >> C.shift)];
        const uint8_t c = C.v[(((int64_t)page * C.heads + h) * D + d) * C.block + (jj & (C.block - 1))];
        float f[4];
        Q::unpack(c, f);
        acc += w * f[0];
      }
      o[x] = acc;
    }
    __syncthreads();
  }
  l = wave_sum(l);
  const int64_t at = (int64_t)row * A.q_heads + hq;
  for (int x = 0; x < D / 64; ++x) A.out[at * D + lane + 64 * x] = IO::put(l == 0.f ? 0.f : o[x] / l);
  if (A.lse && lane == 0) A.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace pp

using namespace pp;

extern "C" int64_t pp_kv_attention_workspace_size(const pp_kv_cache* cache, int64_t table_width, int64_t batch,
                                                  int64_t tokens, int64_t q_heads) {
  return 0;
}

extern "C" int pp_kv_attention(const pp_kv_cache* cache, const void* q, int64_t q_st, int64_t q_sh, int64_t q_heads,
                               int dtype, int64_t tokens, const int32_t* table, int64_t table_ld, int64_t table_width,
                               const int32_t* lengths, const int32_t* cu, int64_t batch, int causal, int64_t window,
                               float scale, void* out, float* lse, void* workspace, int64_t workspace_size,
                               void* stream) {
  AttnArgs A;
  int rc = kv_check_cache(cache, &A.C);
  if (rc) return rc;
  rc = kv_check_seqs(table, table_ld, table_width, lengths, cu, batch, tokens, &A.S);
  if (rc) return rc;
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16, "pp_kv_attention: dtype %d is not PP_F16 or PP_BF16", dtype);
  PP_REQUIRE(q_heads > 0 && q_heads % A.C.heads == 0 && q_heads <= 65535,
             "pp_kv_attention: %lld query heads over %d heads", (long long)q_heads, A.C.heads);
  PP_REQUIRE(window >= 0 && (causal || window == 0), "pp_kv_attention: a window needs causal attention");
  if (tokens == 0) return PP_OK;
  PP_REQUIRE(q && out, "pp_kv_attention: null queries or output");
  A.q = (const uint16_t*)q;
  A.q_st = q_st; A.q_sh = q_sh;
  A.out = (uint16_t*)out;
  A.lse = lse;
  A.q_heads = (int)q_heads;
  A.group = (int)q_heads / A.C.heads;
  A.window = (int)(window < INT32_MAX ? window : 0);
  A.causal = causal;
  A.scale = scale * 1.4426950408889634f;
  const dim3 grid((unsigned)tokens, (unsigned)q_heads);
  const bool i8 = cache->codes == PP_KV_INT8, h = dtype == PP_F16;
#define PP_ATTN(D)                                                                                          \
  (i8 ? (h ? kv_attn_rows_kernel<PP_KV_INT8, IoF16, D> : kv_attn_rows_kernel<PP_KV_INT8, IoBf16, D>)        \
      : (h ? kv_attn_rows_kernel<PP_KV_E4M3, IoF16, D> : kv_attn_rows_kernel<PP_KV_E4M3, IoBf16, D>))
  auto kern = cache->head_dim == 64 ? PP_ATTN(64) : cache->head_dim == 128 ? PP_ATTN(128)
              : cache->head_dim == 192 ? PP_ATTN(192) : PP_ATTN(256);
#undef PP_ATTN
  hipLaunchKernelGGL(kern, grid, dim3(64), 0, (hipStream_t)stream, A);
  PP_LAUNCH_CHECK();
  return PP_OK;
}
