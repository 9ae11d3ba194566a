// The 4-bit cache: appending to it, as the values are or turned, and reading it back.
//
// A workgroup takes 32 tokens of a page (16 where a page is no longer) and a head, or several side by side, keys and values
// both: a value of either that is not finite marks the token in the scales of its keys.  Thread (tg, dg) holds tokens
// 4 tg .. 4 tg + 3 and values 8 dg .. 8 dg + 7, so the largest of a group of 32 meets over four neighbouring lanes.
// Turned keys are computed in 64 bits and rounded to odd, so that a code is the one nearest to the key whatever lies
// between: a step of 4 bits is wide, and a rounding before it would move one value in some 10^7 by a whole step.
//
// What bounds it: instructions beside memory.  16 ragged prompts (14,752 tokens), 8 key heads and 32 query heads of 128
// in bf16, 305 MB: 77 us, 4.0 TB/s with the vector units 49 % busy; the queries' rows alone would take 44, the keys and
// values alone 31 (not turned 18).  The keys' sines in 64 bits, once for four heads, and their rounding to odd are a third of the
// instructions.  64 single tokens 7.9 us, latency.  Reading back 17 us (58 MB written, 4.7 TB/s).
#include "kv_cache4.h"
#include "rotate_keys.h"

namespace pp {

constexpr int SHIFT4 = 5;
__host__ __device__ inline int shift4(const KvCache& C) { return C.shift < SHIFT4 ? C.shift : SHIFT4; }

struct Append4Args {
  AppendArgs A;
  Rot R;
  RotRows Q;
  int beside, chunks, threads;   // heads a workgroup, workgroups a piece, threads a head
  Roles roles;
};

// A number of 64 bits as a float, rounded to odd: what is compared or rounded again to fewer bits comes out as if
// it had been rounded once.
__device__ __forceinline__ float odd_float(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = (uint32_t)u, rest = lo & 0x1fffffffu;
  const uint64_t w = (u & 0xffffffffe0000000ull) | (rest ? 0x20000000u : 0u);
  return (float)__longlong_as_double((long long)w);
}
__device__ __forceinline__ float odd_float(float x) { return x; }

// Over the four lanes of a group.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));     // lane ^ 1
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));  // lane ^ 2
}

constexpr int ROW4 = 20;      // bytes of a row of V codes in LDS: 32 tokens, and 4 so that rows begin in other banks

// TURN: keys are turned (in 64 bits).
template <typename IO, int D, bool TURN>
__global__ __launch_bounds__(TURN ? 512 : 256, TURN ? 3 : 4) void kv_append4_kernel(const Append4Args X) {
  typedef std::conditional_t<TURN, double, float> real;
  unsigned index = blockIdx.x;
  if (TURN && !X.roles.appends(blockIdx.x, index)) {
    rotate_queries<IO, 2>(X.A.S, X.R, X.Q, index);
    return;
  }
  const AppendArgs& A = X.A;
  const KvCache& C = A.C;
  const int item = index / X.chunks, sub = TURN ? uniform(threadIdx.x / X.threads) : 0;
  const int tid = threadIdx.x - sub * X.threads, nthr = X.threads, head = (index - item * X.chunks) * X.beside + sub;
  const int shift = shift4(C);
  Piece P;
  if (!kv_piece(C, A.S, item, shift, P) || P.page < 0) return;
  __shared__ uint32_t bad[8];                            // tokens that are not finite, for each head
  extern __shared__ __align__(16) uint8_t lds[];         // V codes of each head, then the table
  uint8_t* const tile = lds + sub * (D * ROW4);
  const int tg = tid / (D / 8), dg = tid % (D / 8);
  const bool active = head < C.heads, mine = active && tid < (1 << shift) / 4 * (D / 8), leads = mine && dg % 4 == 0;
  if (tid == 0) bad[sub] = 0;
  Trig<real>* const tab = reinterpret_cast<Trig<real>*>(lds + X.beside * (D * ROW4));
  if constexpr (TURN) rot_table(X.R, P, tab);
  __syncthreads();
  uint32_t& flags = bad[sub];
  u32x4 xv[4];
  load_unit<D>(P, A.x[1] + (int64_t)min(head, C.heads - 1) * A.sh[1], A.st[1], A.vec, tid, mine, xv);
  uint32_t kw[4], kb[4], vb = 0, lost = 0;
  auto code_keys = [&](int i, const real* x) {
    float f[8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = odd_float(x[j]);
      top = max(top, mag(f[j]));
    }
    lost |= top >= 0x7f800000u ? 1u << i : 0u;
    const int e = scale4(quad_max(top));
    const float s = scale4_value(e);
    kb[i] = scale4_byte(e);
    kw[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0], f[1], s, 0);
    kw[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(kw[i], f[2], f[3], s, 1);
    kw[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(kw[i], f[4], f[5], s, 2);
    kw[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(kw[i], f[6], f[7], s, 3);
  };
  const uint16_t* const keys = A.x[0] + (int64_t)min(head, C.heads - 1) * A.sh[0];
  if constexpr (TURN) {
    load_turned<IO, real, D>(X.R, P, keys, A.st[0], A.vec, tid, mine, tab, code_keys);
  } else {
    u32x4 w[4];
    load_unit<D>(P, keys, A.st[0], A.vec, tid, mine, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      real x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = half_of<IO>(w[i], j);
      code_keys(i, x);
    }
  }
  float f[4][8];
  // a byte of V is two tokens of different scales: they are divided out first, exactly
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u16x2 big = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, xv[i][j] & 0x7fff7fffu));
    const uint32_t top = mag(IO::get((uint16_t)max((uint32_t)big[0], (uint32_t)big[1])));
    lost |= top >= 0x7f800000u ? 1u << i : 0u;
    const int e = scale4(quad_max(top));
    const float s = scale4_value(-e);
    vb |= scale4_byte(e) << (8 * i);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[i][j] = half_of<IO>(xv[i], j) * s;
  }
  if (mine) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0][j], f[1][j], 1.f, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2][j], f[3][j], 1.f, 1);
      *reinterpret_cast<uint16_t*>(tile + (8 * dg + j) * ROW4 + 2 * tg) = (uint16_t)w;
    }
    if (lost) atomicOr(&flags, lost << (4 * tg));
  }
  __syncthreads();
  if (!active) return;
  const uint32_t broken = flags;
  const int64_t ph = (int64_t)P.page * C.heads + head;
  if (mine) {
    const int64_t row = ph * C.block + P.from;
    uint8_t* const vs = scales_v(C) + (ph * (D / 32) + dg / 4) * C.block + P.from + 4 * tg;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * tg + i;
      if (t < P.lo || t >= P.hi) continue;
      *reinterpret_cast<uint32_t*>(C.k + (row + t) * (D / 2) + 4 * dg) = kw[i];
      if (leads) {
        scales_k(C)[(row + t) * (D / 32) + dg / 4] = (uint8_t)(broken >> t & 1 ? SCALE4_NAN : kb[i]);
        vs[i] = (uint8_t)(vb >> (8 * i));
      }
    }
  }
  uint8_t* const v = C.v + ph * (D / 2) * C.block + P.from / 2;
  const int row_bytes = C.block / 2;
  if (P.lo == 0 && P.hi == 32) {
    for (int d = tid; d < D; d += nthr) {
      const uint32_t* t = reinterpret_cast<const uint32_t*>(tile + d * ROW4);
      *reinterpret_cast<u32x4*>(v + d * row_bytes) = u32x4{t[0], t[1], t[2], t[3]};
    }
  } else {
    const int wl = shift - 3;                          // words of 8 tokens; other tokens' codes stay
    for (int w = tid; w < D << wl; w += nthr) {
      const int d = w >> wl, q = w & ((1 << wl) - 1), lo = max(P.lo - 8 * q, 0), hi = min(P.hi - 8 * q, 8);
      if (lo >= hi) continue;
      uint32_t* const at = reinterpret_cast<uint32_t*>(v + d * row_bytes) + q;
      const uint32_t out = *reinterpret_cast<const uint32_t*>(tile + d * ROW4 + 4 * q);
      const uint32_t mask = (hi - lo == 8 ? ~0u : (1u << (4 * (hi - lo))) - 1) << (4 * lo);
      *at = mask == ~0u ? out : (*at & ~mask) | (out & mask);
    }
  }
}

template <typename IO, int D>
__global__ __launch_bounds__(256) void kv_read4_kernel(const ReadArgs A) {
  const KvCache& C = A.C;
  Piece P;
  const Unit N = kv_unit(C);
  const int shift = shift4(C);
  if (!kv_piece(C, A.S, N.item, shift, P)) return;
  const int head = N.head, isv = N.isv, tid = threadIdx.x, nthr = blockDim.x;
  __shared__ __align__(16) uint8_t tile[D * ROW4];
  const bool none = P.page < 0;                          // read page 0, write zeros
  const int64_t ph = (int64_t)(none ? 0 : P.page) * C.heads + head, row = ph * C.block + (none ? 0 : P.from);
  const int tg = tid / (D / 8), dg = tid % (D / 8);
  const bool mine = tid < (1 << shift) / 4 * (D / 8);
  if (isv) {
    const uint8_t* v = C.v + ph * (D / 2) * C.block + (none ? 0 : P.from / 2);
    const int wl = shift - 3;
    for (int w = tid; w < D << wl; w += nthr) {
      const int d = w >> wl, q = w & ((1 << wl) - 1);
      *reinterpret_cast<uint32_t*>(tile + d * ROW4 + 4 * q) = reinterpret_cast<const uint32_t*>(v + d * (C.block / 2))[q];
    }
    __syncthreads();
  }
  if (!mine) return;
  float x[4][8];
  if (isv) {
    const uint32_t vb = *reinterpret_cast<const uint32_t*>(scales_v(C) + (ph * (D / 32) + dg / 4) * C.block +
                                                            (none ? 0 : P.from) + 4 * tg);
    float s[4] = {__builtin_amdgcn_cvt_f32_bf8(vb, 0), __builtin_amdgcn_cvt_f32_bf8(vb, 1),
                  __builtin_amdgcn_cvt_f32_bf8(vb, 2), __builtin_amdgcn_cvt_f32_bf8(vb, 3)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {                        // a token that was not finite is marked in its keys' scales
      const uint32_t mark = scales_k(C)[(row + 4 * tg + i) * (D / 32)];
      if ((mark & 0x7f) > 0x7c) s[i] = NAN;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w = *reinterpret_cast<const uint16_t*>(tile + (8 * dg + j) * ROW4 + 2 * tg);
      const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
      x[0][j] = a[0] * s[0];
      x[1][j] = a[1] * s[1];
      x[2][j] = b[0] * s[2];
      x[3][j] = b[1] * s[3];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(C.k + (row + 4 * tg + i) * (D / 2) + 4 * dg);
      const float s = __builtin_amdgcn_cvt_f32_bf8(scales_k(C)[(row + 4 * tg + i) * (D / 32) + dg / 4], 0);
      const f32x2 y[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1),
                          __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3)};
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = y[j / 2][j & 1] * s;
    }
  }
  typedef typename IO::raw raw;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * tg + i;
    if (t < P.lo || t >= P.hi) continue;
    raw* o = reinterpret_cast<raw*>(A.out[isv]) + ((P.row0 + t) * C.heads + head) * D + 8 * dg;
    if (none) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = 0.f;
    }
    store_row<IO>(o, true, x[i]);
  }
}

static unsigned threads4(const KvCache& C, int D) { return unit_threads(1 << shift4(C), D); }

int kv_append4(const AppendArgs& A, const Rot* rot, const RotRows* q, int D, int dtype, hipStream_t st) {
  const bool h = dtype == PP_F16;
  const int64_t items = kv_pieces(A.S, shift4(A.C));
  Append4Args X{A, rot ? *rot : Rot{}, q ? *q : RotRows{}, 1, 0, (int)threads4(A.C, D), Roles{}};
  if (rot) X.beside = heads_beside(A.S, X.threads, A.C.heads);
  X.chunks = (A.C.heads + X.beside - 1) / X.beside;
  const unsigned threads = X.threads * X.beside;
  const int64_t units = items * X.chunks, blocks = units + (rot ? query_blocks(X.R, X.Q, threads) : 0);
  PP_REQUIRE(blocks <= UINT32_MAX / threads, "kv append: too many tokens and sequences");
  X.roles = roles(units, blocks);
  const unsigned table = rot ? (A.S.cu ? 1u << shift4(A.C) : 1u) * (unsigned)rot_stride(*rot) * (unsigned)sizeof(Trig<double>) : 0;
  const unsigned lds = X.beside * (unsigned)(D * ROW4) + table;
  return by_width(D, [&](auto d) -> int {
    constexpr int W = decltype(d)::value;
    auto kern = rot ? (h ? kv_append4_kernel<IoF16, W, true> : kv_append4_kernel<IoBf16, W, true>)
                    : (h ? kv_append4_kernel<IoF16, W, false> : kv_append4_kernel<IoBf16, W, false>);
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(threads), lds, st, X);
    PP_LAUNCH_CHECK();
    return PP_OK;
  });
}

int kv_read4(const ReadArgs& A, int D, int dtype, hipStream_t st) {
  const int64_t items = kv_pieces(A.S, shift4(A.C));
  const unsigned threads = threads4(A.C, D);
  PP_REQUIRE(items * 2 * A.C.heads <= UINT32_MAX / threads, "pp_kv_read: too many tokens and sequences");
  return by_width(D, [&](auto d) -> int {
    constexpr int W = decltype(d)::value;
    auto kern = dtype == PP_F16 ? kv_read4_kernel<IoF16, W> : dtype == PP_BF16 ? kv_read4_kernel<IoBf16, W> : kv_read4_kernel<IoF32, W>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(items * 2 * A.C.heads)), dim3(threads), 0, st, A);
    PP_LAUNCH_CHECK();
    return PP_OK;
  });
}

}  // namespace pp
