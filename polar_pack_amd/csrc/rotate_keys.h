// Keys turned on their way into a cache, and the queries' rows beside them (kv_rotate.hip, kv_cache4.hip).
//
// A workgroup that writes a piece of a page computes the sines and cosines of its tokens once, into LDS, and then
// takes its heads one after another: they cost about as much as the values of one head.  Workgroups behind those turn
// the rows of queries, so that a step's rotation and append are one launch.
#pragma once

#include "kv_append.h"
#include "rotary.h"

namespace pp {

constexpr int64_t ROT_TABLE_MAX = 65536;       // bytes of LDS; a larger table is not made: each value its own

// [token lo ..][frequency]; null: no table
template <typename T>
__device__ __forceinline__ void rot_table(const Rot& R, const Piece& P, Trig<T>* tab) {
  const int n = (P.hi - P.lo) * R.half;
  for (int e = threadIdx.x; e < n; e += blockDim.x) {
    const int t = e / R.half, f = e - t * R.half;
    tab[e] = rot_trig<T>(R, f, R.pos ? rot_position(R, f, P.row0 + P.lo + t) : P.pos0 + P.lo + t);
  }
}

// The turned values of thread (tg, dg): tokens 4 tg + i, d 8 dg + j; the other half of a pair is read beside them.
template <typename IO, typename T, int D>
__device__ __forceinline__ void load_turned(const Rot& R, const Piece& P, const uint16_t* src, int64_t st, int vec, bool mine,
                                            const Trig<T>* tab, T (*out)[8]) {
  const int tg = threadIdx.x / (D / 8), dg = threadIdx.x % (D / 8), h8 = R.half / 8;
  const bool turned = dg < 2 * h8, low = dg < h8;
  const int other = R.neighbours || !turned ? dg : low ? dg + h8 : dg - h8;
  const int f0 = R.neighbours ? 4 * dg : low ? 8 * dg : 8 * (dg - h8);
  const T sign = low ? (T)-1 : (T)1;
  u32x4 x[4], y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * tg + i;
    x[i] = y[i] = u32x4{0, 0, 0, 0};
    if (!mine || t < P.lo || t >= P.hi) continue;
    const uint16_t* row = src + (P.row0 + t) * st;
    x[i] = load8(row + 8 * dg, vec);
    y[i] = load8(row + 8 * other, vec);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * tg + i;
#pragma unroll
    for (int j = 0; j < 8; ++j) out[i][j] = (T)half_of<IO>(x[i], j);
    if (!turned || !mine || t < P.lo || t >= P.hi) continue;
    auto trig = [&](int f) {
      if (tab) return tab[(t - P.lo) * R.half + f];
      return rot_trig<T>(R, f, R.pos ? rot_position(R, f, P.row0 + t) : P.pos0 + t);
    };
    if (R.neighbours) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const Trig<T> w = trig(f0 + j / 2);
        const T a = out[i][j], b = out[i][j + 1];
        out[i][j] = a * w.c - b * w.s;
        out[i][j + 1] = b * w.c + a * w.s;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const Trig<T> w = trig(f0 + j);
        out[i][j] = out[i][j] * w.c + sign * (T)half_of<IO>(y[i], j) * w.s;
      }
    }
  }
}

// Block qb of those that turn the queries' rows; every wavefront of the workgroup calls it.
template <typename IO>
__device__ __forceinline__ void rotate_queries(const KvSeqs& S, const Rot& R, const RotRows& Q, int qb) {
  const int units = rot_units(R.half, Q.D), rows = blockDim.x / units, tiles = (Q.tokens + rows - 1) / rows;
  const int group = qb / tiles, first = (qb - group * tiles) * rows;
  const int y = threadIdx.x / units, token = first + y;
  const bool real = y < rows && token < Q.tokens;
  int64_t own = 0;
  bool none = false;
  if (R.pos == nullptr) {
    int b = token;
    if (S.cu != nullptr) {
      int lo = kv_find(S, first, 1, 0, 0);
      int span = kv_find(S, min(first + rows, Q.tokens) - 1, 1, 0, 0) - lo + 1;     // the answer is in [lo, lo + span)
      while (span > 1) {
        const int half = span / 2;
        const bool up = kv_start(S, lo + half) <= token;
        lo = up ? lo + half : lo;
        span = up ? span - half : half;
      }
      b = lo;
    }
    none = b >= S.batch;
    if (real && !none) own = (int64_t)S.lengths[b] - kv_start(S, b + 1) + token;
  }
  if (real) rotate_unit<IO>(R, Q, token, threadIdx.x - y * units, group, own, none);
}
inline int64_t query_blocks(const Rot& R, const RotRows& Q, unsigned threads) {
  if (Q.x == nullptr || Q.tokens == 0) return 0;
  const int rows = (int)threads / rot_units(R.half, Q.D);
  return (int64_t)((Q.tokens + rows - 1) / rows) * ((Q.heads + Q.per - 1) / Q.per);
}

// Heads a workgroup takes: more of them share the sines and cosines, as long as there are four workgroups a CU.
inline int heads_per(int64_t units, int heads) {
  const int64_t per = units * heads / (4 * (int64_t)device_cu_count());
  return per < 1 ? 1 : per < heads ? (int)per : heads;
}

}  // namespace pp
