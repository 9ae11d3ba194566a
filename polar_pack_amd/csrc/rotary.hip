// Rotary positions of rows of queries or keys.
#include "rotary.h"

namespace pp {

int rot_check(const pp_rotary* r, const void* positions, int64_t pos_ld, int pos_type, int64_t tokens, int64_t head_dim,
              bool needed, Rot* out) {
  PP_REQUIRE(r != nullptr && r->turns != nullptr, "rotary: null");
  PP_REQUIRE(r->rotary_dim >= 16 && r->rotary_dim % 16 == 0 && r->rotary_dim <= head_dim,
             "rotary: rotary_dim %d is not a multiple of 16 up to %lld", r->rotary_dim, (long long)head_dim);
  PP_REQUIRE(r->n_axes >= 1 && r->n_axes <= 255, "rotary: %d axes not in 1..255", r->n_axes);
  PP_REQUIRE(r->axes != nullptr || r->n_axes == 1, "rotary: null axes");
  PP_REQUIRE(r->pairs == PP_PAIRS_HALVES || r->pairs == PP_PAIRS_NEIGHBOURS, "rotary: pairs %d", r->pairs);
  PP_REQUIRE(positions != nullptr || !needed, "rotary: null positions");
  PP_REQUIRE(pos_type == PP_POS_I32 || pos_type == PP_POS_I64, "rotary: positions of type %d", pos_type);
  PP_REQUIRE(aligned(r->turns, 8) && aligned(positions, pos_type == PP_POS_I64 ? 8 : 4), "rotary: operands are not aligned");
  *out = Rot{r->turns, r->axes, positions, pos_ld, r->n_axes, r->rotary_dim / 2, r->pairs == PP_PAIRS_NEIGHBOURS,
             pos_type == PP_POS_I64, r->scaling};
  return PP_OK;
}

// What bounds it: memory.  16,200 tokens of 18 heads of 128 in bf16 with three axes (149 MB): 26.7 us, 5.6 TB/s, where a copy
// reaches 4.9; before a token's positions were read at once for all its frequencies 36.4.
template <typename IO>
__global__ __launch_bounds__(256) void rotate_kernel(const Rot R, const RotRows A) {
  const int token = blockIdx.x * blockDim.y + threadIdx.y;
  if (token < A.tokens) rotate_unit<IO, 1>(R, A, token, threadIdx.x, blockIdx.y, 0, false);
}

}  // namespace pp

using namespace pp;

extern "C" int pp_rotate(const void* x, int64_t x_st, int64_t x_sh, int dtype, int64_t tokens, int64_t heads,
                         int64_t head_dim, const pp_rotary* rotary, const void* positions, int64_t pos_ld, int pos_type,
                         void* out, int64_t o_st, int64_t o_sh, void* stream) {
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16 || dtype == PP_F32, "pp_rotate: dtype %d", dtype);
  PP_REQUIRE(tokens >= 0 && tokens <= (1 << 28), "pp_rotate: tokens %lld not in 0..2^28", (long long)tokens);
  PP_REQUIRE(heads >= 0 && heads <= 65535, "pp_rotate: heads %lld not in 0..65535", (long long)heads);
  PP_REQUIRE(head_dim >= 16 && head_dim % 8 == 0 && head_dim <= 512, "pp_rotate: head_dim %lld is not a multiple of 8 in 16..512",
             (long long)head_dim);
  if (tokens == 0 || heads == 0) return PP_OK;
  Rot R;
  const int rc = rot_check(rotary, positions, pos_ld, pos_type, tokens, head_dim, true, &R);
  if (rc) return rc;
  PP_REQUIRE(x && out, "pp_rotate: null rows");
  const int es = dtype == PP_F32 ? 4 : 2, per16 = 16 / es;
  PP_REQUIRE(aligned(x, es) && aligned(out, es), "pp_rotate: rows are not aligned to their type");
  RotRows A{x, out, x_st, x_sh, o_st, o_sh, (int)tokens, (int)heads, (int)head_dim, 1, 0};
  A.vec = aligned(x, 16) && aligned(out, 16) && x_st % per16 == 0 && x_sh % per16 == 0 && o_st % per16 == 0 && o_sh % per16 == 0;
  const int units = rot_units(R.half, A.D);
  const int64_t groups = rot_groups(tokens * units, heads, 512);
  A.per = (int)((heads + groups - 1) / groups);
  const dim3 wg(units, 256 / units), grid((unsigned)((tokens + wg.y - 1) / wg.y), (unsigned)((heads + A.per - 1) / A.per));
  auto kern = dtype == PP_F16 ? rotate_kernel<IoF16> : dtype == PP_BF16 ? rotate_kernel<IoBf16> : rotate_kernel<IoF32>;
  hipLaunchKernelGGL(kern, grid, wg, 0, (hipStream_t)stream, R, A);
  PP_LAUNCH_CHECK();
  return PP_OK;
}
