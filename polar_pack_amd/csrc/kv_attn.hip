// Attention of a call's tokens to the 8-bit cache.
//
// Row (token, query head) with position p = lengths[b] - n_b + i sees the keys j of
// (p - window, p] (causal) or of [0, length):
//   s_j = scale * ks * sum_d q_d kcode_jd,   o_d = sum_j e^(s_j - m) vs vcode_jd / sum_j e^(s_j - m).
#include "kv_attn.h"

namespace pp {

// Few rows a sequence and head (single tokens, drafts).  A workgroup takes 16 * RT rows of one
// sequence and key/value head and a run of 64-token tiles, dealt to its 4 wavefronts in turn; runs of
// one row tile are joined by kv_attn_join_kernel.
//
// The codes go from memory to the matrix cores without LDS: S^T = K Q^T takes rows of K as they lie
// (16 bytes a lane), O^T = V^T P^T rows of the transposed V.  Which token is which row of a product is
// free, so S^T's rows are numbered such that the 16 scores a lane holds of a tile, tokens
// 16 g + 0..15 of lane group g = lane / 16, are the ones whose V codes its 16-byte load brings:
// row m of product t is token 16 (m / 4) + 4 t + m % 4, and P needs no exchange between lanes.
// Scales stay out of the codes: ks multiplies a lane's scores, log2 vs is added to the exponent,
// so that weights e^(s - m) vs are at most 2^14 in fp16 whatever the scales, and the sum of
// e^(s - m) takes them times 1 / vs.
template <int CODES, typename IO, int D, int RT, int NP>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void kv_attn_split_kernel(const AttnArgs A) {
  constexpr int J = D / 64, DT = D / 16, R = 16 * RT;
  const KvCache& C = A.C;
  const KvSeqs& S = A.S;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), m16 = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % A.splits, h = blockIdx.y;
  RowTile T;
  if (!kv_row_tile(A, blockIdx.x / A.splits, R, T)) return;
  int a, z;
  const int ns = kv_runs(A, T, split, a, z);
  if (split >= ns) return;
  const int shift = C.shift, bs = C.block;

  // this lane's rows: column m16 of row tile x
  f16x8 q[RT][J][2];
  float rf[RT];
  int lo[RT], hi[RT];
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int r = T.r0 + 16 * x + m16;
    const bool real = r < T.rows;
    const int i = real ? r / A.group : 0, gq = real ? r - i * A.group : 0;
    kv_visible(A, T, i, real, lo[x], hi[x]);
    rf[x] = load_q<IO, D>(A, T.s0 + i, h * A.group + gq, g, real, q[x]);
  }
  f32x4 o[RT][DT];
  float mx[RT], l[RT];
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    mx[x] = -INFINITY;
    l[x] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[x][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Tiles of this wavefront: a + wave, a + wave + 4, ...; lane e holds the table's entry e % NP of
  // tile e / NP of the next 64 / NP tiles.
  const int32_t* table = S.table + (int64_t)T.b * S.ld;
  int ids = 0;
  auto refill = [&](int tile) {
    const int64_t at = (((int64_t)tile + 4 * (lane / NP)) * 64 >> shift) + lane % NP;
    ids = at < S.width ? table[at] : -1;
    ids = ids < C.pages ? ids : -1;
  };
  u32x4 kc[4][J], vc[DT];
  float ks = 0.f, vs = 0.f, ks_n = 0.f, vs_n = 0.f;
  bool okv = false, ok_n = false;
  int64_t vbase_n = 0;
  const int km = NP == 1 ? 0 : (16 * (m16 >> 2)) >> shift, vm = NP == 1 ? 0 : (16 * g) >> shift;   // page of the tile
  auto page_of = [&](int step, int which) {
    int p = lane_read(ids, (step % (64 / NP)) * NP);
#pragma unroll
    for (int e = 1; e < NP; ++e) {
      const int pe = lane_read(ids, (step % (64 / NP)) * NP + e);
      p = which == e ? pe : p;
    }
    return p;
  };
  auto load_k = [&](int tile, int step) {
    int pk = page_of(step, km);
    pk = pk < 0 ? 0 : pk;
    const uint8_t* base = C.k + ((int64_t)pk * C.heads + h) * (bs * D);
    const int tok = (tile * 64 + 16 * (m16 >> 2)) & (bs - 1);
    const int off = (tok + (m16 & 3)) * D + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < J; ++j) kc[t][j] = *reinterpret_cast<const u32x4*>(base + off + 4 * t * D + 64 * j);
    const int pv = page_of(step, vm);
    ok_n = pv >= 0;
    const int64_t ph = (int64_t)(pv < 0 ? 0 : pv) * C.heads + h;
    ks_n = C.ks[ph];
    vs_n = C.vs[ph];
    vbase_n = ph * (bs * D);
  };
  auto load_v = [&](int tile) {
    const uint8_t* base = C.v + vbase_n + ((tile * 64 + 16 * g) & (bs - 1)) + m16 * bs;
#pragma unroll
    for (int d = 0; d < DT; ++d) vc[d] = *reinterpret_cast<const u32x4*>(base + d * 16 * bs);
  };

  int tile = a + wave, step = 0;
  if (tile < z) {
    refill(tile);
    load_k(tile, 0);
    load_v(tile);
  }
  for (; tile < z; tile += 4, ++step) {
    ks = ks_n; vs = vs_n; okv = ok_n;
    f32x4 s[RT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int x = 0; x < RT; ++x) s[x][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        f16x8 ka, kb;
        to_halves<CODES>(kc[t][j], ka, kb);
#pragma unroll
        for (int x = 0; x < RT; ++x) {
          s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q[x][j][0], s[x][t], 0, 0, 0);
          s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, q[x][j][1], s[x][t], 0, 0, 0);
        }
      }
    }
    const bool more = tile + 4 < z;
    if (more) {
      if ((step + 1) % (64 / NP) == 0) refill(tile + 4);
      load_k(tile + 4, step + 1);
    }
    // scores to weights
    const bool vbad = mag(vs) >= 0x7f800000u;                    // the values are NaN, the sum of weights is not
    const float vq = vbad ? 1.f : fmaxf(vs, KV_SCALE_MIN);
    const float lv = __builtin_amdgcn_logf(vq), iv = 1.0f / vq;
    const int t0 = tile * 64 + 16 * g;
    f16x8 p[RT][2];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      const float c = ks * rf[x];
      const bool edge = __any(!okv || t0 < lo[x] || t0 + 16 > hi[x]);
      float e[16], top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) e[4 * t + r] = s[x][t][r] * c + lv;
      if (edge) {
#pragma unroll
        for (int k = 0; k < 16; ++k) e[k] = okv && t0 + k >= lo[x] && t0 + k < hi[x] ? e[k] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) top = fmaxf(top, e[k]);
      top = max_groups(top);
      if (__any(top > mx[x])) {
        const float mn = fmaxf(mx[x], top);
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx[x] - mn);
        mx[x] = mn;
        l[x] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[x][d] *= f;
      }
      const float ref = (mx[x] == -INFINITY ? 0.f : mx[x]) - KV_P_LOG2;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        e[k] = __builtin_amdgcn_exp2f(e[k] - ref);
        sum += e[k];
        p[x][k / 8][k % 8] = (f16)e[k];
      }
      l[x] += sum * iv;
      if (__any(vbad)) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (vbad && okv && t0 + k >= lo[x] && t0 + k < hi[x]) p[x][k / 8][k % 8] = (f16)NAN;
      }
    }
    if (CODES == PP_KV_E4M3) {                   // codes past the length may be NaN
      const int seen = okv ? T.lim - t0 : 0;
      if (__any(seen < 16)) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int left = seen - 4 * w;
          const uint32_t keep = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
#pragma unroll
          for (int d = 0; d < DT; ++d) vc[d][w] &= keep;
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      f16x8 va, vb;
      to_halves<CODES>(vc[d], va, vb);
#pragma unroll
      for (int x = 0; x < RT; ++x) {
        o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[x][0], o[x][d], 0, 0, 0);
        o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb, p[x][1], o[x][d], 0, 0, 0);
      }
    }
    if (more) load_v(tile + 4);
  }

  // The 4 wavefronts' sums meet in LDS: halves of them add the other half's, twice.
  __shared__ float so[2][R][D + 4];
  __shared__ float sm[2][R], sl[2][R];
#pragma unroll
  for (int x = 0; x < RT; ++x) l[x] = sum_groups(l[x]);
#pragma unroll
  for (int half = 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int x = 0; x < RT; ++x) {
        const int r = 16 * x + m16, w = wave - half;
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&so[w][r][16 * d + 4 * g]) = o[x][d];
        if (g == 0) { sm[w][r] = mx[x]; sl[w][r] = l[x]; }
      }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int x = 0; x < RT; ++x) {
        const int r = 16 * x + m16;
        const float mo = sm[wave][r], mn = fmaxf(mx[x], mo);
        const float f = mx[x] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx[x] - mn);
        const float fo = mo == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mo - mn);
        mx[x] = mn;
        l[x] = l[x] * f + sl[wave][r] * fo;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[x][d] = o[x][d] * f + *reinterpret_cast<const f32x4*>(&so[wave][r][16 * d + 4 * g]) * fo;
      }
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int r = T.r0 + 16 * x + m16;
    if (r >= T.rows) continue;
    const int i = r / A.group;
    const int64_t at = (int64_t)(T.s0 + i) * A.q_heads + h * A.group + (r - i * A.group);
    if (ns == 1) {
      const float inv = kv_inverse(l[x]);
#pragma unroll
      for (int d = 0; d < DT; ++d)
        store4<IO>(A.out + at * D + 16 * d + 4 * g, o[x][d] * inv);
      if (A.lse && g == 0) A.lse[at] = kv_lse(mx[x], l[x]);
    } else {
      float* part = A.parts + (at * A.splits + split) * (D + 4);
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(part + 16 * d + 4 * g) = o[x][d];
      if (g == 0) {
        part[D] = mx[x];
        part[D + 1] = l[x];
      }
    }
  }
}

// One wavefront joins the runs of one row.
template <typename IO, int D>
__global__ __launch_bounds__(64) void kv_attn_join_kernel(const AttnArgs A, int R) {
  const int64_t at = blockIdx.x;
  const int token = (int)(at / A.q_heads), hq = (int)(at % A.q_heads), lane = threadIdx.x;
  RowTile T;
  kv_tile_of(A, token, hq % A.group, R, T);
  int a, z;
  const int ns = kv_runs(A, T, 0, a, z);
  if (ns <= 1) return;
  const float* part = A.parts + at * A.splits * (D + 4);
  float m = -INFINITY;
  for (int s = lane; s < ns; s += 64) m = fmaxf(m, part[s * (D + 4) + D]);
  for (int x = 32; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  float l = 0.f, o[D / 64] = {};
  for (int s = 0; s < ns; ++s) {
    const float* p = part + s * (D + 4);
    const float f = p[D] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(p[D] - m);
    l += p[D + 1] * f;
#pragma unroll
    for (int x = 0; x < D / 64; ++x) o[x] += p[64 * x + lane] * f;
  }
  const float inv = kv_inverse(l);
#pragma unroll
  for (int x = 0; x < D / 64; ++x) A.out[at * D + 64 * x + lane] = IO::put(o[x] * inv);
  if (A.lse && lane == 0) A.lse[at] = kv_lse(m, l);
}

struct AttnPlan {
  int rt;
  int64_t splits, bytes;
};

static AttnPlan attn_plan(const pp_kv_cache* c, int64_t width, int64_t batch, int64_t tokens, int64_t q_heads) {
  const int64_t rows = (tokens * (q_heads / c->heads) + batch - 1) / batch;      // a sequence and head, on average
  AttnPlan P;
  P.rt = rows > 16 ? 2 : 1;
  const int64_t items = batch * ((rows + 16 * P.rt - 1) / (16 * P.rt)) * c->heads;
  // two workgroups a CU; a run is at least 4 tiles
  const int64_t most = (width * c->block + 255) / 256;
  int64_t s = (2 * (int64_t)device_cu_count() + items - 1) / items;
  if (s > most) s = most;
  if (s < 1) s = 1;
  P.splits = s;
  P.bytes = s > 1 ? tokens * q_heads * s * (c->head_dim + 4) * 4 : 0;
  return P;
}

// Row tiles of R rows that the call may have: those of the sequences begin at floor(rows before / R) + b.
static int64_t attn_items(const AttnArgs& A, int R) {
  return A.S.cu ? (int64_t)A.S.tokens * A.group / R + A.S.batch + 1
                : (int64_t)A.S.batch * ((A.group + R - 1) / R);
}

template <int CODES, typename IO, int D>
static int attn_launch(const AttnArgs& A, const AttnPlan& P, hipStream_t st) {
  const dim3 grid((unsigned)(attn_items(A, 16 * P.rt) * P.splits), (unsigned)A.C.heads);
  auto pick = [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    auto kern = A.C.block >= 64 ? kv_attn_split_kernel<CODES, IO, D, RT, 1>
                : A.C.block == 32 ? kv_attn_split_kernel<CODES, IO, D, RT, 2> : kv_attn_split_kernel<CODES, IO, D, RT, 4>;
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, A);
  };
  if (P.rt == 1) pick(std::integral_constant<int, 1>());
  else pick(std::integral_constant<int, 2>());
  PP_LAUNCH_CHECK();
  if (P.splits > 1) {
    hipLaunchKernelGGL((kv_attn_join_kernel<IO, D>), dim3((unsigned)((int64_t)A.S.tokens * A.q_heads)), dim3(64), 0, st,
                       A, 16 * P.rt);
    PP_LAUNCH_CHECK();
  }
  return PP_OK;
}

template <int CODES, typename IO>
static int attn_width(const AttnArgs& A, const AttnPlan& P, int D, hipStream_t st) {
  switch (D) {
    case 64: return attn_launch<CODES, IO, 64>(A, P, st);
    case 128: return attn_launch<CODES, IO, 128>(A, P, st);
    case 192: return attn_launch<CODES, IO, 192>(A, P, st);
    default: return attn_launch<CODES, IO, 256>(A, P, st);
  }
}

}  // namespace pp

using namespace pp;

extern "C" int64_t pp_kv_attention_workspace_size(const pp_kv_cache* cache, int64_t table_width, int64_t batch,
                                                  int64_t tokens, int64_t q_heads) {
  KvCache c;
  if (kv_check_cache(cache, &c) || table_width <= 0 || batch <= 0 || tokens <= 0 || q_heads < cache->heads) return 0;
  return attn_plan(cache, table_width, batch, tokens, q_heads).bytes;
}

extern "C" int pp_kv_attention(const pp_kv_cache* cache, const void* q, int64_t q_st, int64_t q_sh, int64_t q_heads,
                               int dtype, int64_t tokens, const int32_t* table, int64_t table_ld, int64_t table_width,
                               const int32_t* lengths, const int32_t* cu, int64_t batch, int causal, int64_t window,
                               float scale, void* out, float* lse, void* workspace, int64_t workspace_size,
                               void* stream) {
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
  const AttnPlan P = attn_plan(cache, table_width, batch, tokens, q_heads);
  PP_REQUIRE(P.bytes == 0 || (workspace && workspace_size >= P.bytes && aligned(workspace, 16)),
             "pp_kv_attention: workspace of %lld bytes at a 16-byte boundary needed", (long long)P.bytes);
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
  A.splits = (int)P.splits;
  PP_REQUIRE(attn_items(A, 16 * P.rt) * P.splits <= INT32_MAX, "pp_kv_attention: too many rows");
  A.scale = scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
  const int D = cache->head_dim;
  if (cache->codes == PP_KV_INT8)
    return dtype == PP_F16 ? attn_width<PP_KV_INT8, IoF16>(A, P, D, st) : attn_width<PP_KV_INT8, IoBf16>(A, P, D, st);
  return dtype == PP_F16 ? attn_width<PP_KV_E4M3, IoF16>(A, P, D, st) : attn_width<PP_KV_E4M3, IoBf16>(A, P, D, st);
}
