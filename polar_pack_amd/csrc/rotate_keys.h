// Keys turned on their way into a cache, and the queries' rows beside them (kv_rotate.hip, kv_cache4.hip).
//
// A workgroup that writes a piece of a page computes the sines and cosines of its tokens once, into LDS, for several
// heads side by side: they cost more than the values of one head, and heads one after another cost their latencies (16
// ragged prompts, 8 heads of 128 in 4 bits: 45 us, against 18 for an append of keys as they are).  Workgroups behind
// those turn the rows of queries, so that a step's rotation and append are one launch.
#pragma once

#include "kv_append.h"
#include "rotary.h"

namespace pp {

// [token lo ..][frequency], the frequencies 0, 8, 16 .. first, then 1, 9, .. : what the lanes of a row read at once lies side
// by side, and rows begin in other banks.
__host__ __device__ inline int rot_stride(const Rot& R) { return R.half + 2; }
__device__ __forceinline__ int rot_place(const Rot& R, int f) { return (f & 7) * (R.half >> 3) + (f >> 3); }

template <typename T>
__device__ __forceinline__ void rot_table(const Rot& R, const Piece& P, Trig<T>* tab) {
  const int n = (P.hi - P.lo) * R.half;
  for (int e = threadIdx.x; e < n; e += blockDim.x) {
    const int t = e / R.half, f = e - t * R.half;
    tab[t * rot_stride(R) + rot_place(R, f)] =
        rot_trig<T>(R, f, R.pos ? rot_position(R, f, P.row0 + P.lo + t) : P.pos0 + P.lo + t);
  }
}

// The turned values of thread (tg, dg), d 8 dg + j of tokens 4 tg + i, as use(i, values) for one token after another (so
// that those of one at a time are in registers); the other half of a pair is read beside them.  Tokens that are not of
// the piece give zeros.
template <typename IO, typename T, int D, typename F>
__device__ __forceinline__ void load_turned(const Rot& R, const Piece& P, const uint16_t* src, int64_t st, int vec, int tid, bool mine,
                                            const Trig<T>* tab, F use) {
  const int tg = tid / (D / 8), dg = tid % (D / 8), h8 = R.half / 8;
  const bool turned = dg < 2 * h8, low = dg < h8;
  const int other = R.neighbours || !turned ? dg : low ? dg + h8 : dg - h8;
  const int f0 = R.neighbours ? 4 * dg : low ? 8 * dg : 8 * (dg - h8);
  u32x4 x[4], y[4];
  load_rows(P, src, st, vec, tg, 8 * dg, x);
  load_rows(P, src, st, vec, tg, 8 * other, y);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * tg + i;
#pragma unroll
    for (int k = 0; k < 4; ++k) asm volatile("" : "+v"(x[i][k]), "+v"(y[i][k]));      // not converted before its turn
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (T)half_of<IO>(x[i], j);
    const bool in = mine && t >= P.lo && t < P.hi;
    if (turned && in) {
      const Trig<T>* const row = tab + (t - P.lo) * rot_stride(R);
      auto trig = [&](int f) { return row[rot_place(R, f)]; };
      if (R.neighbours) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const Trig<T> w = trig(f0 + j / 2);
          const T a = v[j], b = v[j + 1];
          v[j] = a * w.c - b * w.s;
          v[j + 1] = b * w.c + a * w.s;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const Trig<T> w = trig(f0 + j);
          const T b = (T)half_of<IO>(y[i], j) * w.s;
          v[j] = v[j] * w.c + (low ? -b : b);
        }
      }
    }
    if (!in) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0;
    }
    use(i, v);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Block qb of those that turn the queries' rows; every wavefront of the workgroup calls it.
template <typename IO, int AHEAD>
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
  if (real) rotate_unit<IO, AHEAD>(R, Q, token, threadIdx.x - y * units, group, own, none);
}
inline int64_t query_blocks(const Rot& R, const RotRows& Q, unsigned threads) {
  if (Q.x == nullptr || Q.tokens == 0) return 0;
  const int rows = (int)threads / rot_units(R.half, Q.D);
  return (int64_t)((Q.tokens + rows - 1) / rows) * ((Q.heads + Q.per - 1) / Q.per);
}

// Workgroups that append, bound by instructions, and those that turn queries, bound by memory, alternate over the grid in
// the proportion of their numbers: block b is the index-th of either.
struct Roles {
  uint64_t step;          // append units a block, times 2^32, rounded up
  __device__ __forceinline__ bool appends(unsigned b, unsigned& index) const {
    const uint64_t at = b * step;
    const unsigned before = (unsigned)(at >> 32);
    const bool yes = (unsigned)((at + step) >> 32) != before;
    index = yes ? before : b - before;
    return yes;
  }
};
inline Roles roles(int64_t units, int64_t blocks) { return Roles{(((uint64_t)units << 32) + blocks - 1) / blocks}; }

// Heads a workgroup of `threads` a head takes side by side; a single token has few sines to share.
inline int heads_beside(const KvSeqs& S, unsigned threads, int heads) {
  const int n = S.cu ? (int)(512 / threads) : 1;
  return n < 1 ? 1 : n < heads ? n : heads;
}

}  // namespace pp
