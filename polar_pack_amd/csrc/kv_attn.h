// What the attention kernels of the 8-bit cache share: rows, what they see, runs of keys, queries.
#pragma once

#include "kv_common.h"

namespace pp {

// Weights are 2^(s - ref), s with log2 of vs in it, ref 14 below the largest s: up to 2^14 in fp16, the smallest that is
// not flushed 2^-38 of the largest.  Past 2^24 floats are so far apart that the 14 would round to 16, whose 2^16 fp16
// does not hold; ref is the largest s itself there.
constexpr float KV_P_LOG2 = 14.f;
__device__ __forceinline__ float kv_ref(float top) {
  const float ref = top - KV_P_LOG2;
  return top - ref > 15.f ? top : ref;
}

// A row tile of many rows whose keys several workgroups share: the parts, and the rows.
struct ManyPart {
  int runs, s0, r0, rows;
};

struct AttnArgs {
  KvCache C;
  KvSeqs S;
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* out;
  float* lse;
  float* parts;     // [head][workgroup][2][row][D + 4]: what a workgroup has of a row tile that it shares: sums of
                    // values, reference, sum of weights; 1: of the one that begins in it, 0: of one that began before
  ManyPart* desc;   // [head][workgroup] (many rows): the shared row tile that begins in it, runs 0: none
  uint32_t* counts; // [head][workgroup]: parts that are done of the row tile that begins in it; 0 before and after
  int q_heads, group, window, causal, q_vec;
  int shares;       // workgroups a key/value head, 0: one a row tile
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

// What the rows r0 .. r0 + R - 1 of a sequence see.
__device__ __forceinline__ void kv_tile_range(const AttnArgs& A, int R, RowTile& T) {
  const int i0 = T.r0 / A.group, last = min(T.rows, T.r0 + R) - 1;
  int x;
  kv_visible(A, T, i0, true, T.lo, x);
  kv_visible(A, T, last / A.group, true, x, T.hi);
  if (!A.causal && T.lim > 0) T.hi = T.lim;
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
  kv_tile_range(A, R, T);
  return true;
}

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return uniform(v);
}
__device__ __forceinline__ int wave_max(int v) { return -wave_min(-v); }

// Work item `at` of the call: tiles of R rows (a power of two), sequence after sequence.
__device__ __forceinline__ bool kv_row_tile(const AttnArgs& A, int at, int R, RowTile& T) {
  if (A.S.cu == nullptr) {
    const int per = (A.group + R - 1) / R;
    T.b = at / per;
    if (T.b >= A.S.batch) return false;
    T.r0 = (at - T.b * per) * R;
  } else {
    T.b = kv_find(A.S, at, A.group, __builtin_ctz(R), 1);
    T.r0 = (at - kv_begin(A.S, T.b, A.group, __builtin_ctz(R), 1)) * R;
  }
  T.b = uniform(T.b);
  return kv_tile_fill(A, R, T);
}

// Work item `at` with the row tiles that see the most keys first, so that the last workgroups to start are
// short ones: every sequence's last row tile, then every one's last but one.  More sequences
// than a wavefront has lanes come one after another.
__device__ __forceinline__ bool kv_row_tile_from_last(const AttnArgs& A, int at, int R, RowTile& T) {
  const KvSeqs& S = A.S;
  if (S.batch > 63) {
    const int items = (int)((int64_t)S.tokens * A.group / R) + S.batch + 1;
    return kv_row_tile(A, items - 1 - at, R, T);
  }
  const int b = threadIdx.x & 63;
  const int n = b <= S.batch ? kv_start(S, b + 1) - kv_start(S, b) : 0;
  const int tiles = n > 0 ? (n * A.group + R - 1) / R : 0;
  auto sum = [](int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return uniform(v);
  };
  int lo = 0, hi = wave_max(tiles);        // the round: the largest with sum of min(tiles, round) <= at
  if (at >= sum(tiles)) return false;
  int before = 0;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2, done = sum(min(tiles, mid));
    if (done <= at) {
      lo = mid;
      before = done;
    } else {
      hi = mid;
    }
  }
  uint64_t left = __ballot(tiles > lo);
  for (int skip = at - before; skip > 0; --skip) left &= left - 1;
  T.b = __builtin_ctzll(left);
  T.r0 = (__builtin_amdgcn_readlane(tiles, T.b) - 1 - lo) * R;
  return kv_tile_fill(A, R, T);
}

// How the few-row kernel deals a call: its tiles of 64 keys, row tile after row tile, cut into equal
// shares, one a workgroup, wherever that falls.  The lengths are on the device, so every workgroup
// counts the tiles itself and finds where its share begins: thread t of 256 looks at sequences 4t .. 4t + 3
// (of 512 at 2t, 2t + 1), then a sum and a scan over the workgroup.  A row tile that sees no key counts as one tile, the tokens
// past cu[batch] are sequence `batch`.  Going on to a row tile costs a workgroup about as much as KV_TURN
// tiles, so each begins with that many that hold no keys.
constexpr int KV_TURN = 16;
constexpr int KV_DEAL_BATCH = 1020;      // sequences that can be dealt; row tiles of more are not cut

struct Deal {
  int64_t at, end;    // tiles of the call that are this workgroup's and not done
  int share;          // tiles a workgroup
  int first, tiles;   // of each of the sequence's row tiles: key tile it begins at, tiles that hold keys
  int into;           // tile of the row tile that `at` is, KV_TURN the first that holds keys
};

// What sequence b's row tiles have to read, and its rows.
__device__ __forceinline__ int kv_sequence(const AttnArgs& A, int b, RowTile& T, int& first, int& tiles) {
  const KvSeqs& S = A.S;
  T.b = b;
  const int len = S.lengths[b < S.batch ? b : 0];              // beside the offsets, not after them
  T.s0 = kv_start(S, b);
  const int n = kv_start(S, b + 1) - T.s0;
  T.rows = n > 0 ? n * A.group : 0;
  T.pos0 = T.lim = first = 0;
  tiles = 1;
  if (n <= 0) return 0;
  if (b < S.batch) {
    const int64_t cap = (int64_t)S.width << A.C.shift;
    T.pos0 = len < 0 ? -n : len - n;
    T.lim = len < 0 ? 0 : len < cap ? len : (int)cap;
  }
  int lo, hi, x;
  kv_visible(A, T, 0, true, lo, x);
  kv_visible(A, T, n - 1, true, x, hi);
  if (!A.causal) hi = T.lim;
  first = lo >> 6;
  tiles = hi > lo ? ((hi + 63) >> 6) - first : 1;
  return n;
}

template <int THREADS>
__device__ __forceinline__ bool kv_deal(const AttnArgs& A, int R, RowTile& T, Deal& U) {
  __shared__ int64_t sums[THREADS / 64], from;
  __shared__ int found[7];
  constexpr int PER = 1024 / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t work[PER], total = 0;
  RowTile X[PER];
  int first[PER], tiles[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = PER * tid + k;
    work[k] = 0;
    if (b > A.S.batch) continue;
    kv_sequence(A, b, X[k], first[k], tiles[k]);
    work[k] = (int64_t)((X[k].rows + R - 1) / R) * (tiles[k] + KV_TURN);
    total += work[k];
  }
  int64_t upto = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t v = __shfl_up((long long)upto, o, 64);
    upto += lane >= o ? v : 0;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int64_t all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) all += sums[w];
  for (int w = 0; w < wave; ++w) upto += sums[w];
  const int64_t share = (all + A.shares - 1) / A.shares;
  U.share = (int)(share < 4 ? 4 : (share + 3) / 4 * 4);        // 4 wavefronts a workgroup
  U.at = (int64_t)blockIdx.x * U.share;
  U.end = U.at + U.share < all ? U.at + U.share : all;
  if (U.at >= U.end) return false;
  int64_t before = upto - total;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (U.at >= before && U.at < before + work[k]) {
      found[0] = X[k].b;
      found[1] = X[k].s0;
      found[2] = X[k].rows;
      found[3] = X[k].pos0;
      found[4] = X[k].lim;
      found[5] = first[k];
      found[6] = tiles[k];
      from = U.at - before;
    }
    before += work[k];
  }
  __syncthreads();
  T.b = uniform(found[0]);
  T.s0 = uniform(found[1]);
  T.rows = uniform(found[2]);
  T.pos0 = uniform(found[3]);
  T.lim = uniform(found[4]);
  U.first = uniform(found[5]);
  U.tiles = uniform(found[6]);
  const int64_t t = uniform64(from);
  const int row_tile = (int)(t / (U.tiles + KV_TURN));
  T.r0 = row_tile * R;
  U.into = (int)(t - (int64_t)row_tile * (U.tiles + KV_TURN));
  return true;
}

// On to the next row tile.
__device__ __forceinline__ void kv_deal_next(const AttnArgs& A, int R, RowTile& T, Deal& U) {
  U.into = 0;
  T.r0 += R;
  if (T.r0 < T.rows) return;
  T.r0 = 0;
  for (int b = T.b + 1; b <= A.S.batch; b += 64) {             // the next sequence that has tokens
    const int e = b + (threadIdx.x & 63);
    const uint64_t some = __ballot(e <= A.S.batch && kv_start(A.S, e + 1) > kv_start(A.S, e));
    if (some) {
      kv_sequence(A, b + __builtin_ctzll(some), T, U.first, U.tiles);
      return;
    }
  }
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

// A value that every lane wants and that no kernel of the launch writes, through the scalar cache.
__device__ __forceinline__ float scalar_load(const float* p) {
  return *(const __attribute__((address_space(4))) float*)uniform_ptr(p);
}

// Over the lanes l, l ^ 32.
__device__ __forceinline__ float max_halves(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
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
// size fit in fp16 then.  With fp16's smallest step 2^-24 a bf16 value keeps all its bits down to 2^-30 of
// the row's largest (an fp16 one to 2^-27); smaller ones lose some, and what is below 2^-38 of it is zero.
// load_q issues the loads, make_q returns the factor of the row's sums, score scale and power of two; NaN for a
// row that is not finite.
template <int D>
__device__ __forceinline__ void load_q(const AttnArgs& A, int token, int hq, int g, bool real, u32x4 (*w)[2]) {
  const uint16_t* p = A.q + (int64_t)token * A.q_st + (int64_t)hq * A.q_sh + 16 * g;
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      w[j][e] = u32x4{0, 0, 0, 0};
      if (!real) continue;
      const uint16_t* x = p + 64 * j + 8 * e;
      if (A.q_vec) {
        w[j][e] = *reinterpret_cast<const u32x4*>(x);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[j][e][k] = (uint32_t)x[2 * k] | (uint32_t)x[2 * k + 1] << 16;
      }
    }
}

// PARTS 16-byte pieces of a row as halves; the row's other pieces are in the lanes lane ^ FROM, lane ^ 2 FROM .. .
template <typename IO, int PARTS, int FROM>
__device__ __forceinline__ float scale_q(const AttnArgs& A, const u32x4* w, f16x8* q) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < PARTS; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, mag(IO::get((uint16_t)(w[j][k / 2] >> (16 * (k & 1))))));
#pragma unroll
  for (int o = FROM; o < 64; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  const bool finite = top < 0x7f800000u;
  const int ex = top == 0 || !finite ? 0 : 14 - __builtin_amdgcn_frexp_expf(__uint_as_float(top));
#pragma unroll
  for (int j = 0; j < PARTS; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) q[j][k] = (f16)ldexpf(IO::get((uint16_t)(w[j][k / 2] >> (16 * (k & 1)))), ex);
  return finite ? ldexpf(A.scale, -ex) : NAN;
}

template <typename IO, int D>
__device__ __forceinline__ float make_q(const AttnArgs& A, const u32x4 (*w)[2], f16x8 (*q)[2]) {
  return scale_q<IO, D / 32, 16>(A, &w[0][0], &q[0][0]);
}

// The same for 32 rows a product: lane half hh holds values 16 c + 8 hh + 0..7 as q[c].
template <typename IO, int D>
__device__ __forceinline__ float many_q(const AttnArgs& A, int token, int hq, int hh, bool real, f16x8* q) {
  const uint16_t* p = A.q + (int64_t)token * A.q_st + (int64_t)hq * A.q_sh + 8 * hh;
  u32x4 w[D / 16];
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    w[c] = u32x4{0, 0, 0, 0};
    if (!real) continue;
    if (A.q_vec) {
      w[c] = *reinterpret_cast<const u32x4*>(p + 16 * c);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[c][k] = (uint32_t)p[16 * c + 2 * k] | (uint32_t)p[16 * c + 2 * k + 1] << 16;
    }
  }
  return scale_q<IO, D / 16, 32>(A, w, q);
}

// (m, l, v) takes the part (mp, lp, w), both sums of 2^(s - their reference).
template <int W>
__device__ __forceinline__ void join_part(float& m, float& l, float* v, float mp, float lp, const float* w) {
  const float mn = fmaxf(m, mp);
  const float f = mp == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mp - mn);      // 1: nothing seen, 0 * 1
  const float keep = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
  m = mn;
  l = l * keep + lp * f;
#pragma unroll
  for (int k = 0; k < W; ++k) v[k] = v[k] * keep + w[k] * f;
}

// 1 / l, and 0 for a row that saw nothing; a NaN stays.
__device__ __forceinline__ float kv_inverse(float l) { return l == 0.f ? 0.f : 1.0f / l; }
__device__ __forceinline__ float kv_lse(float ref, float l) {
  return l == 0.f ? -INFINITY : (ref + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

template <typename IO>
__device__ __forceinline__ void store4(uint16_t* p, f32x4 v) {
  u32x2 w;
  w[0] = (uint32_t)IO::put(v[0]) | (uint32_t)IO::put(v[1]) << 16;
  w[1] = (uint32_t)IO::put(v[2]) | (uint32_t)IO::put(v[3]) << 16;
  *reinterpret_cast<u32x2*>(p) = w;
}

struct AttnPlan {
  int64_t rows;       // rows of a row tile: 16, 32 (few rows a sequence and head), 128 or 256 (many)
  int64_t shares, grid, bytes, counts;
};

// Prompts (kv_attn_many.hip).
int kv_attn_many(const AttnArgs& A, const AttnPlan& P, int D, int codes, int dtype, hipStream_t st);

}  // namespace pp
