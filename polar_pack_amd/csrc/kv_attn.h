// What the attention kernels of the 8-bit cache share: rows, what they see, runs of keys, queries.
#pragma once

#include "kv_common.h"

namespace pp {

// Weights e^(s - m) vs are kept up to 2^14 in fp16: the smallest that is not flushed is 2^-38 of the
// largest.
constexpr float KV_P_LOG2 = 14.f;

struct AttnArgs {
  KvCache C;
  KvSeqs S;
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* out;
  float* lse;
  float* parts;     // [token][query head][run][D + 4]: sums, maximum, sum of weights
  int q_heads, group, window, causal, splits, q_vec;
  float scale;      // of the scores, times log2(e)
};

// Rows r0 .. of sequence b's `rows` = tokens * group rows of a key/value head; row r is its token r / group.
struct RowTile {
  int b, s0, r0, rows;
  int pos0;       // position of the sequence's first token of the call
  int lim;        // keys [0, lim) exist
  int lo, hi;     // keys that any of the tile's rows sees
};

__device__ __forceinline__ void kv_visible(const AttnArgs& A, const RowTile& T, int i, bool real, int& lo, int& hi) {
  const int64_t pos = (int64_t)T.pos0 + i;
  lo = A.window && pos >= A.window ? (int)(pos - A.window + 1) : 0;
  hi = !real || pos < 0 ? 0 : A.causal && pos + 1 < T.lim ? (int)pos + 1 : T.lim;
}

// The tile of rows r0 .. r0 + R - 1; T.b and T.r0 are set.
__device__ __forceinline__ bool kv_tile_fill(const AttnArgs& A, int R, RowTile& T) {
  const KvSeqs& S = A.S;
  T.s0 = kv_start(S, T.b);
  const int n = kv_start(S, T.b + 1) - T.s0;
  T.rows = n * A.group;
  if (T.r0 >= T.rows) return false;
  T.lim = 0;
  T.pos0 = 0;
  if (T.b < S.batch) {
    const int len = S.lengths[T.b];
    T.pos0 = len < 0 ? -n : len - n;
    const int64_t cap = (int64_t)S.width << A.C.shift;
    T.lim = len < 0 ? 0 : len < cap ? len : (int)cap;
  }
  const int i0 = T.r0 / A.group, last = min(T.rows, T.r0 + R) - 1;
  int x;
  kv_visible(A, T, i0, true, T.lo, x);
  kv_visible(A, T, last / A.group, true, x, T.hi);
  if (!A.causal && T.lim > 0) T.hi = T.lim;
  return true;
}

// Work item `at` of the call: tiles of R rows, sequence after sequence.
__device__ __forceinline__ bool kv_row_tile(const AttnArgs& A, int at, int R, RowTile& T) {
  if (A.S.cu == nullptr) {
    const int per = (A.group + R - 1) / R;
    T.b = at / per;
    if (T.b >= A.S.batch) return false;
    T.r0 = (at - T.b * per) * R;
  } else {
    T.b = kv_find(A.S, at, A.group, R, 1);
    T.r0 = (at - kv_begin(A.S, T.b, A.group, R, 1)) * R;
  }
  T.b = uniform(T.b);
  return kv_tile_fill(A, R, T);
}

// The tile that holds query g of token `token`.
__device__ __forceinline__ void kv_tile_of(const AttnArgs& A, int token, int g, int R, RowTile& T) {
  T.b = A.S.cu == nullptr ? token : kv_find(A.S, token, 1, 1, 0);
  T.r0 = ((token - kv_start(A.S, T.b)) * A.group + g) / R * R;
  kv_tile_fill(A, R, T);
}

// Runs of 64-key tiles: how many a row tile has, and the tiles [a, z) of run `split`.
__device__ __forceinline__ int kv_runs(const AttnArgs& A, const RowTile& T, int split, int& a, int& z) {
  const int first = T.lo >> 6, end = T.hi > T.lo ? (T.hi + 63) >> 6 : first;
  const int tiles = end - first;
  int run = (tiles + A.splits - 1) / A.splits;
  run = run < 4 ? 4 : (run + 3) / 4 * 4;
  a = first + split * run;
  z = min(end, a + run);
  return tiles > run ? (tiles + run - 1) / run : 1;
}

__device__ __forceinline__ int lane_read(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Over the lanes l, l ^ 16, l ^ 32, l ^ 48, which hold the parts of one row.
__device__ __forceinline__ float max_groups(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 16 codes as two operands of 8 halves.
template <int CODES>
__device__ __forceinline__ void to_halves(u32x4 w, f16x8& a, f16x8& b) {
  f16x2 h[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) KvCodes<CODES>::halves(w[i], h[2 * i], h[2 * i + 1]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[2 * i] = h[i][0];
    a[2 * i + 1] = h[i][1];
    b[2 * i] = h[4 + i][0];
    b[2 * i + 1] = h[4 + i][1];
  }
}

// A row's query as the second operand of S^T = K Q^T: lane group g holds values 64 j + 16 g + 8 e + 0..7
// as q[j][e], scaled by a power of two so that the largest lies in [2^13, 2^14): bf16 queries of any
// size keep all their bits in fp16 (what is below 2^-37 of the largest loses some).  Returns the factor
// of the row's sums, score scale and power of two; NaN for a row that is not finite.
template <typename IO, int D>
__device__ __forceinline__ float load_q(const AttnArgs& A, int token, int hq, int g, bool real, f16x8 (*q)[2]) {
  float x[D / 64][2][8];
  uint32_t top = 0;
  const uint16_t* p = A.q + (int64_t)token * A.q_st + (int64_t)hq * A.q_sh + 16 * g;
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (real) {
        load8<IO>(p + 64 * j + 8 * e, A.q_vec, x[j][e]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[j][e][k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, mag(x[j][e][k]));
    }
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  const float t = __uint_as_float(top);
  const bool finite = top < 0x7f800000u;
  const int ex = top == 0 || !finite ? 0 : 14 - __builtin_amdgcn_frexp_expf(t);
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int k = 0; k < 8; ++k) q[j][e][k] = (f16)ldexpf(x[j][e][k], ex);
  return finite ? ldexpf(A.scale, -ex) : NAN;
}

// 1 / l, and 0 for a row that saw nothing; a NaN stays.
__device__ __forceinline__ float kv_inverse(float l) { return l == 0.f ? 0.f : 1.0f / l; }
__device__ __forceinline__ float kv_lse(float m, float l) {
  return l == 0.f ? -INFINITY : (m - KV_P_LOG2 + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

template <typename IO>
__device__ __forceinline__ void store4(uint16_t* p, f32x4 v) {
  u32x2 w;
  w[0] = (uint32_t)IO::put(v[0]) | (uint32_t)IO::put(v[1]) << 16;
  w[1] = (uint32_t)IO::put(v[2]) | (uint32_t)IO::put(v[3]) << 16;
  *reinterpret_cast<u32x2*>(p) = w;
}

}  // namespace pp
