// Queries and keys turned by their positions, keys and values written to the cache, in one launch: 8 bits and the
// entry point.
//
// What bounds it: the queries' way through memory, and instructions (63 % busy).  4 prompts of 2048 tokens, 16 query and
// 2 key heads of 128 in fp16, 81 MB: 21 us, 3.9 TB/s (34 with heads one after another and appends before all queries);
// single tokens of 4 sequences 7.8 us, as an append without rotation (7.4): the chain of lengths, pages, values and old scale.
#include "kv_cache4.h"
#include "rotate_keys.h"

namespace pp {

struct RotateArgs {
  AppendArgs A;
  Rot R;
  RotRows Q;
  int beside, chunks, threads;   // heads a workgroup, workgroups a page and side, threads a head
  Roles roles;
};

template <int CODES, typename IO, int D>
__global__ __launch_bounds__(D < 128 ? 512 : 4 * D, 4) void kv_rotate_append_kernel(const RotateArgs X) {
  unsigned index;
  if (!X.roles.appends(blockIdx.x, index)) {
    rotate_queries<IO, 1>(X.A.S, X.R, X.Q, index);
    return;
  }
  const AppendArgs& A = X.A;
  const KvCache& C = A.C;
  const uint32_t n = 2 * (uint32_t)X.chunks, item = index / n, r = index - item * n;
  const int isv = r >= (uint32_t)X.chunks, sub = uniform(threadIdx.x / X.threads), tid = threadIdx.x - sub * X.threads;
  const int head = (int)(isv ? r - X.chunks : r) * X.beside + sub;
  Piece P;
  if (!kv_piece(C, A.S, (int)item, C.shift, P) || P.page < 0) return;
  __shared__ uint32_t maxima[8][16];
  extern __shared__ __align__(16) uint32_t lds[];      // of keys the table, of values the codes
  const bool active = head < C.heads, mine = active && tid < (C.block / 4) * (D / 8);
  uint32_t* const red = maxima[sub];
  const uint16_t* src = A.x[isv] + (int64_t)min(head, C.heads - 1) * A.sh[isv];
  if (isv) {
    u32x4 x[4];
    const uint32_t top = load_unit<D>(P, src, A.st[1], A.vec, tid, mine, x);
    append_page<CODES, D>(C, P, head, 1, top, [](uint32_t w) { return mag(IO::get((uint16_t)w)); }, red,
                          lds + sub * D * (C.block / 4 + 1), tid, X.threads, active,
                          [&](int i, int j) { return half_of<IO>(x[i], j); });
    return;
  }
  Trig<float>* const tab = reinterpret_cast<Trig<float>*>(lds);
  rot_table(X.R, P, tab);
  __syncthreads();
  float x[4][8];
  uint32_t top = 0;
  load_turned<IO, float, D>(X.R, P, src, A.st[0], A.vec, tid, mine, tab, [&](int i, const float* v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[i][j] = v[j];
      top = max(top, mag(v[j]));
    }
  });
  append_page<CODES, D>(C, P, head, 0, top, [](uint32_t w) { return w; }, red, lds, tid, X.threads, active,
                        [&](int i, int j) { return x[i][j]; });
}

}  // namespace pp

using namespace pp;

extern "C" int pp_kv_rotate_append(const pp_kv_cache* cache, const void* q, int64_t q_st, int64_t q_sh, int64_t q_heads,
                                   void* q_out, const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
                                   int64_t v_sh, int dtype, int64_t tokens, const pp_rotary* rotary,
                                   const void* positions, int64_t pos_ld, int pos_type, const int32_t* table,
                                   int64_t table_ld, int64_t table_width, const int32_t* lengths, const int32_t* cu,
                                   int64_t batch, void* stream) {
  RotateArgs X;
  int rc = append_check("pp_kv_rotate_append", cache, k, k_st, k_sh, v, v_st, v_sh, dtype, tokens, table, table_ld,
                        table_width, lengths, cu, batch, &X.A);
  if (rc) return rc;
  const int D = cache->head_dim;
  rc = rot_check(rotary, positions, pos_ld, pos_type, tokens, D, false, &X.R);
  if (rc || tokens == 0) return rc;
  PP_REQUIRE(q_heads >= 0 && q_heads <= 65535, "pp_kv_rotate_append: %lld query heads", (long long)q_heads);
  X.Q = RotRows{q_heads ? q : nullptr, q_out, q_st, q_sh, q_heads * D, D, (int)tokens, (int)q_heads, D, 1, 0};
  if (X.Q.x) {
    PP_REQUIRE(q_out && aligned(q, 2) && aligned(q_out, 16), "pp_kv_rotate_append: queries or their output null or not aligned");
    X.Q.vec = aligned(q, 16) && q_st % 8 == 0 && q_sh % 8 == 0;
    const int64_t groups = rot_groups(tokens * rot_units(X.R.half, D), q_heads, 1024);
    X.Q.per = (int)((q_heads + groups - 1) / groups);
  }
  PP_REQUIRE(X.Q.x || q_heads == 0, "pp_kv_rotate_append: null queries");
  if (cache->codes == PP_KV_E2M1) return kv_append4(X.A, &X.R, &X.Q, D, dtype, (hipStream_t)stream);
  const KvCache& C = X.A.C;
  const int64_t items = kv_pieces(X.A.S, C.shift);
  X.threads = (int)unit_threads(C.block, D);
  X.beside = heads_beside(X.A.S, X.threads, C.heads);
  X.chunks = (C.heads + X.beside - 1) / X.beside;
  const dim3 wg(X.threads * X.beside);
  const int64_t units = items * 2 * X.chunks, blocks = units + query_blocks(X.R, X.Q, wg.x);
  PP_REQUIRE(blocks <= UINT32_MAX / wg.x, "pp_kv_rotate_append: too many tokens and sequences");
  X.roles = roles(units, blocks);
  // a piece of a call without cu is one token
  const unsigned table_bytes = (cu ? C.block : 1) * (unsigned)rot_stride(X.R) * (unsigned)sizeof(Trig<float>);
  const unsigned tiles = tile_bytes(C.block, D) * X.beside, lds = table_bytes > tiles ? table_bytes : tiles;
  return by_width(D, [&](auto d) -> int {
    constexpr int W = decltype(d)::value;
    const bool i8 = cache->codes == PP_KV_INT8, h = dtype == PP_F16;
    auto kern = i8 ? (h ? kv_rotate_append_kernel<PP_KV_INT8, IoF16, W> : kv_rotate_append_kernel<PP_KV_INT8, IoBf16, W>)
                   : (h ? kv_rotate_append_kernel<PP_KV_E4M3, IoF16, W> : kv_rotate_append_kernel<PP_KV_E4M3, IoBf16, W>);
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), wg, lds, (hipStream_t)stream, X);
    PP_LAUNCH_CHECK();
    return PP_OK;
  });
}
