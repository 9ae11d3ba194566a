// Writing keys and values into the cache, and reading them back: 8 bits, and the entry points.
#include "kv_append.h"
#include "kv_cache4.h"

namespace pp {

int kv_check_cache(const pp_kv_cache* c, KvCache* out) {
  PP_REQUIRE(c != nullptr, "kv cache: null");
  PP_REQUIRE(c->k && c->v && c->k_scale && c->v_scale, "kv cache: null codes or scales");
  PP_REQUIRE(c->pages > 0 && c->pages <= INT32_MAX, "kv cache: pages %lld", (long long)c->pages);
  PP_REQUIRE(c->heads > 0 && c->heads <= 65535, "kv cache: heads %d not in 1..65535", c->heads);
  PP_REQUIRE(c->block == 16 || c->block == 32 || c->block == 64 || c->block == 128,
             "kv cache: block %d is not 16, 32, 64 or 128", c->block);
  PP_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 192 || c->head_dim == 256,
             "kv cache: head_dim %d is not 64, 128, 192 or 256", c->head_dim);
  PP_REQUIRE(c->codes == PP_KV_INT8 || c->codes == PP_KV_E4M3 || c->codes == PP_KV_E2M1, "kv cache: codes %d", c->codes);
  PP_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16), "kv cache: codes are not 16-byte aligned");
  PP_REQUIRE(c->codes != PP_KV_E2M1 || (aligned(c->k_scale, 16) && aligned(c->v_scale, 16)),
             "kv cache: scales of 4-bit codes are not 16-byte aligned");
  *out = KvCache{(uint8_t*)c->k, (uint8_t*)c->v, (float*)c->k_scale, (float*)c->v_scale, c->pages, c->heads, c->block,
                 c->block == 16 ? 4 : c->block == 32 ? 5 : c->block == 64 ? 6 : 7};
  return PP_OK;
}

int kv_check_seqs(const KvCache& c, const int32_t* table, int64_t ld, int64_t width, const int32_t* lengths, const int32_t* cu,
                  int64_t batch, int64_t tokens, KvSeqs* out) {
  PP_REQUIRE(table && lengths, "kv: null block table or lengths");
  PP_REQUIRE(batch > 0 && batch <= (1 << 24), "kv: batch %lld not in 1..2^24", (long long)batch);
  PP_REQUIRE(tokens >= 0 && tokens <= (1 << 28), "kv: tokens %lld not in 0..2^28", (long long)tokens);
  PP_REQUIRE(width > 0 && width <= (1 << 30) >> c.shift, "kv: a block table of %lld pages holds no or over 2^30 tokens",
             (long long)width);
  PP_REQUIRE(ld >= width || batch == 1, "kv: block table rows of %lld overlap (stride %lld)", (long long)width,
             (long long)ld);
  PP_REQUIRE(cu != nullptr || tokens == batch, "kv: %lld tokens of %lld sequences need cu", (long long)tokens,
             (long long)batch);
  *out = KvSeqs{table, ld, lengths, cu, (int)width, (int)batch, (int)tokens};
  return PP_OK;
}

int append_check(const char* name, const pp_kv_cache* cache, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                 int64_t v_st, int64_t v_sh, int dtype, int64_t tokens, const int32_t* table, int64_t table_ld,
                 int64_t table_width, const int32_t* lengths, const int32_t* cu, int64_t batch, AppendArgs* A) {
  int rc = kv_check_cache(cache, &A->C);
  if (rc) return rc;
  rc = kv_check_seqs(A->C, table, table_ld, table_width, lengths, cu, batch, tokens, &A->S);
  if (rc) return rc;
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16, "%s: dtype %d is not PP_F16 or PP_BF16", name, dtype);
  if (tokens == 0) return PP_OK;
  PP_REQUIRE(k && v, "%s: null keys or values", name);
  PP_REQUIRE(aligned(k, 2) && aligned(v, 2), "%s: keys or values are not 2-byte aligned", name);
  A->x[0] = (const uint16_t*)k;
  A->x[1] = (const uint16_t*)v;
  A->st[0] = k_st; A->st[1] = v_st;
  A->sh[0] = k_sh; A->sh[1] = v_sh;
  A->vec = aligned(k, 16) && aligned(v, 16) && k_st % 8 == 0 && k_sh % 8 == 0 && v_st % 8 == 0 && v_sh % 8 == 0;
  return PP_OK;
}

template <int CODES, typename IO, int D>
__global__ __launch_bounds__(1024) void kv_append_kernel(const AppendArgs A) {
  const KvCache& C = A.C;
  Piece P;
  const Unit N = kv_unit(C);
  if (!kv_piece(C, A.S, N.item, C.shift, P) || P.page < 0) return;
  const int head = N.head, isv = N.isv;
  __shared__ uint32_t red[16];
  extern __shared__ uint32_t tile[];                   // V codes: [D][block / 4 + 1] words
  u32x4 x[4];
  const int tid = threadIdx.x;
  const uint32_t top = load_unit<D>(P, A.x[isv] + (int64_t)head * A.sh[isv], A.st[isv], A.vec, tid,
                                    tid < (C.block / 4) * (D / 8), x);
  append_page<CODES, D>(C, P, head, isv, top, [](uint32_t w) { return mag(IO::get((uint16_t)w)); }, red, tile, tid,
                        blockDim.x, true, [&](int i, int j) { return half_of<IO>(x[i], j); });
}

// Reading back: the same units, each output row written once; tokens that lie on no page, or past
// the last sequence, read zero.
template <int CODES, typename IO, int D>
__global__ __launch_bounds__(1024) void kv_read_kernel(const ReadArgs A) {
  using Q = KvCodes<CODES>;
  const KvCache& C = A.C;
  Piece P;
  const Unit N = kv_unit(C);
  if (!kv_piece(C, A.S, N.item, C.shift, P)) return;
  const int head = N.head, isv = N.isv;
  const int tid = threadIdx.x, nthr = blockDim.x;
  extern __shared__ uint32_t tile[];
  const bool none = P.page < 0;                        // read page 0, write zeros
  const int64_t ph = (int64_t)(none ? 0 : P.page) * C.heads + head, base = ph * (C.block * D);
  const float scale = none ? 0.f : (isv ? C.vs : C.ks)[ph];
  const int tg = tid / (D / 8), dg = tid % (D / 8);
  const bool mine = tid < (C.block / 4) * (D / 8);
  uint32_t w8[4][2];
  if (isv) {
    const u32x4* v = reinterpret_cast<const u32x4*>(C.v + base);
    const int ql = C.shift - 4, ld = C.block / 4 + 1;
    for (int w = tid; w < D << ql; w += nthr) {
      const u32x4 c = v[w];
      uint32_t* t = tile + (w >> ql) * ld + 4 * (w & ((1 << ql) - 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = c[i];
    }
    __syncthreads();
    if (!mine) return;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = tile[(8 * dg + 4 * j + i) * ld + tg];
      swap_bytes(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) w8[i][j] = c[i];
    }
  } else {
    if (!mine) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(C.k + base + (4 * tg + i) * D + 8 * dg);
      w8[i][0] = w[0];
      w8[i][1] = w[1];
    }
  }
  typedef typename IO::raw raw;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * tg + i;
    if (t < P.lo || t >= P.hi) continue;
    raw* o = reinterpret_cast<raw*>(A.out[isv]) + ((P.row0 + t) * C.heads + head) * D + 8 * dg;
    float x[8];
    Q::unpack(none ? 0u : w8[i][0], x);
    Q::unpack(none ? 0u : w8[i][1], x + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= scale;
    if constexpr (sizeof(raw) == 4) {
      reinterpret_cast<f32x4*>(o)[0] = f32x4{x[0], x[1], x[2], x[3]};
      reinterpret_cast<f32x4*>(o)[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
      *reinterpret_cast<u32x4*>(o) = u32x4{IO::put2(x[0], x[1]), IO::put2(x[2], x[3]), IO::put2(x[4], x[5]),
                                           IO::put2(x[6], x[7])};
    }
  }
}

}  // namespace pp

using namespace pp;

extern "C" int pp_kv_append(const pp_kv_cache* cache, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                            int64_t v_st, int64_t v_sh, int dtype, int64_t tokens, const int32_t* table,
                            int64_t table_ld, int64_t table_width, const int32_t* lengths, const int32_t* cu,
                            int64_t batch, void* stream) {
  AppendArgs A;
  const int rc = append_check("pp_kv_append", cache, k, k_st, k_sh, v, v_st, v_sh, dtype, tokens, table, table_ld,
                              table_width, lengths, cu, batch, &A);
  if (rc || tokens == 0) return rc;
  if (cache->codes == PP_KV_E2M1) return kv_append4(A, nullptr, nullptr, cache->head_dim, dtype, (hipStream_t)stream);
  const int64_t items = kv_pieces(A.S, A.C.shift);
  const dim3 wg(unit_threads(A.C.block, cache->head_dim));
  PP_REQUIRE(items * 2 * A.C.heads <= UINT32_MAX / wg.x, "pp_kv_append: too many tokens and sequences");
  const dim3 grid((unsigned)(items * 2 * A.C.heads));
  const unsigned lds = tile_bytes(A.C.block, cache->head_dim);
  return by_width(cache->head_dim, [&](auto d) -> int {
    constexpr int D = decltype(d)::value;
    const bool i8 = cache->codes == PP_KV_INT8, h = dtype == PP_F16;
    auto kern = i8 ? (h ? kv_append_kernel<PP_KV_INT8, IoF16, D> : kv_append_kernel<PP_KV_INT8, IoBf16, D>)
                   : (h ? kv_append_kernel<PP_KV_E4M3, IoF16, D> : kv_append_kernel<PP_KV_E4M3, IoBf16, D>);
    hipLaunchKernelGGL(kern, grid, wg, lds, (hipStream_t)stream, A);
    PP_LAUNCH_CHECK();
    return PP_OK;
  });
}

extern "C" int pp_kv_read(const pp_kv_cache* cache, const int32_t* table, int64_t table_ld, int64_t table_width,
                          const int32_t* lengths, const int32_t* cu, int64_t batch, int64_t tokens, int dtype,
                          void* k_out, void* v_out, void* stream) {
  ReadArgs A;
  int rc = kv_check_cache(cache, &A.C);
  if (rc) return rc;
  rc = kv_check_seqs(A.C, table, table_ld, table_width, lengths, cu, batch, tokens, &A.S);
  if (rc) return rc;
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16 || dtype == PP_F32, "pp_kv_read: dtype %d", dtype);
  if (tokens == 0) return PP_OK;
  PP_REQUIRE(k_out && v_out, "pp_kv_read: null outputs");
  PP_REQUIRE(aligned(k_out, 16) && aligned(v_out, 16), "pp_kv_read: outputs are not 16-byte aligned");
  A.out[0] = k_out;
  A.out[1] = v_out;
  if (cache->codes == PP_KV_E2M1) return kv_read4(A, cache->head_dim, dtype, (hipStream_t)stream);
  const int64_t items = kv_pieces(A.S, A.C.shift);
  const dim3 wg(unit_threads(A.C.block, cache->head_dim));
  PP_REQUIRE(items * 2 * A.C.heads <= UINT32_MAX / wg.x, "pp_kv_read: too many tokens and sequences");
  const dim3 grid((unsigned)(items * 2 * A.C.heads));
  const unsigned lds = tile_bytes(A.C.block, cache->head_dim);
  return by_width(cache->head_dim, [&](auto d) -> int {
    constexpr int D = decltype(d)::value;
    const bool i8 = cache->codes == PP_KV_INT8;
    auto kern = dtype == PP_F16    ? (i8 ? kv_read_kernel<PP_KV_INT8, IoF16, D> : kv_read_kernel<PP_KV_E4M3, IoF16, D>)
                : dtype == PP_BF16 ? (i8 ? kv_read_kernel<PP_KV_INT8, IoBf16, D> : kv_read_kernel<PP_KV_E4M3, IoBf16, D>)
                                   : (i8 ? kv_read_kernel<PP_KV_INT8, IoF32, D> : kv_read_kernel<PP_KV_E4M3, IoF32, D>);
    hipLaunchKernelGGL(kern, grid, wg, lds, (hipStream_t)stream, A);
    PP_LAUNCH_CHECK();
    return PP_OK;
  });
}
