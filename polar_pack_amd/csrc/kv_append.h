// Appending to a cache: the call's work items, and how a page of 8-bit codes is written.
#pragma once

#include "kv_common.h"

namespace pp {

// One workgroup takes the new tokens of one page and head, of the keys or of the values
// (kv_unit): nobody else touches that page's scale or codes.
// A page's tokens are split over the threads in units of 4 tokens x 8 values, one unit a thread
// (block * D / 32 threads), so the values are read once and stay in registers between the
// maximum and the rounding, and a unit of V is 8 words of 4 neighbouring tokens.  16 ragged prompts, 8
// heads of 128 in e4m3 (58 MB read, 29 written): 23 us, 3.9 TB/s with the vector units 66 % busy, and 26 when every byte was moved by a
// shift and a mask; one token of four sequences 7.4 us, the latency of lengths, pages, values and old scale one after another.
struct AppendArgs {
  KvCache C;
  KvSeqs S;
  const uint16_t* x[2];
  int64_t st[2], sh[2];
  int vec;
};

// Work item `at`: the call's tokens of one sequence that share a page.  A sequence's n tokens touch at
// most n / block + 2 of the position ranges [i * block, (i + 1) * block); i may be negative (a length
// below n) or past the table, and then, as where the table names no page, `page` is -1.  Tokens past
// the last sequence make items of their own, also without a page.
struct Piece {
  int64_t row0;       // the token at place t is row row0 + t of the call's tokens
  int64_t pos0;       // and has position pos0 + t
  int lo, hi, page;   // places lo..hi-1, from place `from` of the page on
  int from;
};

// Where a page holds more than one piece (4 bits), pieces are of 2^shift tokens.
__device__ __forceinline__ bool kv_piece(const KvCache& C, const KvSeqs& S, int at, int shift, Piece& P) {
  int b = at, slot = 0;
  if (S.cu != nullptr) {
    b = kv_find(S, at, 1, shift, 2);
    slot = at - kv_begin(S, b, 1, shift, 2);
  }
  const int s0 = kv_start(S, b), n = kv_start(S, b + 1) - s0;
  if (n <= 0) return false;
  const bool real = b < S.batch;
  const int64_t len = real ? S.lengths[b] : n, first = len - n;
  const int64_t piece = (first >> shift) + slot, p0 = piece << shift, blk = p0 >> C.shift;
  const int64_t lo = first > p0 ? first : p0, hi = len < p0 + (1 << shift) ? len : p0 + (1 << shift);
  if (lo >= hi) return false;
  P.row0 = s0 + p0 - first;
  P.pos0 = p0;
  P.from = (int)(p0 - (blk << C.shift));
  P.lo = (int)(lo - p0);
  P.hi = (int)(hi - p0);
  P.page = real && blk >= 0 && blk < S.width ? S.table[(int64_t)b * S.ld + blk] : -1;
  if (P.page >= C.pages) P.page = -1;
  return true;
}

// Workgroup -> work item, keys or values, head, the head first: neighbouring workgroups read
// neighbouring pieces of the tokens' rows (16 ragged prompts, append and read: 55.1 -> 54.2 us).
struct Unit {
  int item, isv, head;
};
__device__ __forceinline__ Unit kv_unit(const KvCache& C) {
  const uint32_t n = 2 * (uint32_t)C.heads, item = blockIdx.x / n, r = blockIdx.x - item * n;
  const bool isv = r >= (uint32_t)C.heads;
  return Unit{(int)item, isv, (int)(isv ? r - C.heads : r)};
}

// Codes and scale of one page, head and side (8 bits): thread (tg, dg) holds the values of tokens 4 tg .. 4 tg + 3 and
// d 8 dg .. 8 dg + 7, value(i, j).  `top`: the thread's largest magnitude, of which bits(top) are the word as
// a float; any order-keeping words do for the maximum.  red is 16 words of LDS, tile D * (block / 4 + 1) for V.  The page is
// that of threads tid = 0 .. nthr - 1, whole wavefronts, of a workgroup whose other threads make the same call for other
// heads; not `active`: for none.
template <int CODES, int D, typename B, typename V>
__device__ __forceinline__ void append_page(const KvCache& C, const Piece& P, int head, int isv, uint32_t top, B bits_of,
                                            uint32_t* red, uint32_t* tile, int tid, int nthr, bool active, V value) {
  using Q = KvCodes<CODES>;
  const int held = P.lo, end = P.hi;                   // new tokens held..end-1 of the page
  const int tg = tid / (D / 8), dg = tid % (D / 8);
  const bool mine = active && tid < (C.block / 4) * (D / 8);
  top = wave_umax(top);
  if ((tid & 63) == 0) red[tid >> 6] = top;
  const int64_t ph = (int64_t)P.page * C.heads + head;
  float* scale_at = (isv ? C.vs : C.ks) + ph;
  const float was = held && active ? *scale_at : 0.f;
  __syncthreads();
  for (int w = 0; w < (nthr + 63) / 64; ++w) top = max(top, red[w]);
  top = bits_of(top);
  // unsigned order: scales are not negative, and a NaN stays
  const uint32_t need = mag(__uint_as_float(top) / Q::kMax);
  const uint32_t bits = max(need, max(mag(was), mag(KV_SCALE_MIN)));
  const float now = __uint_as_float(bits);
  const bool finite = bits < 0x7f800000u;
  const bool grown = held && mag(was) < bits;
  const float ratio = finite ? was / now : 0.f;
  // qmax / max|x| is rounded once, 1 / scale of a rounded scale twice: half as many codes on the wrong
  // side of a tie
  const float inv = !finite ? 0.f : need == bits ? Q::kMax / __uint_as_float(top) : 1.0f / now;
  if (tid == 0 && active) *scale_at = now;

  uint32_t w8[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      w8[i][j] = finite ? Q::pack(value(i, 4 * j) * inv, value(i, 4 * j + 1) * inv, value(i, 4 * j + 2) * inv,
                                  value(i, 4 * j + 3) * inv)
                        : 0u;
  auto rescale = [&](uint32_t w) {
    float f[4];
    Q::unpack(w, f);
    return finite ? Q::pack(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio) : 0u;
  };
  const int64_t base = ph * (C.block * D);
  if (!isv) {
    uint8_t* k = C.k + base;
    if (mine) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 4 * tg + i;
        if (t >= held && t < end) *reinterpret_cast<u32x2*>(k + t * D + 8 * dg) = u32x2{w8[i][0], w8[i][1]};
      }
    }
    if (grown && active)
      for (int w = tid; w < held * (D / 4); w += nthr) {
        uint32_t* p = reinterpret_cast<uint32_t*>(k) + w;
        *p = rescale(*p);
      }
    return;
  }
  // V: four tokens of a value make a word; words that hold older or later tokens are merged.
  const int ld = C.block / 4 + 1;
  if (mine) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t c[4] = {w8[0][j], w8[1][j], w8[2][j], w8[3][j]};
      swap_bytes(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) tile[(8 * dg + 4 * j + i) * ld + tg] = c[i];
    }
  }
  __syncthreads();
  if (!active) return;
  uint32_t* v = reinterpret_cast<uint32_t*>(C.v + base);
  const int wl = C.shift - 2, words = D << wl;
  if (held == 0 && end == C.block) {                   // all new: whole 16-byte pieces
    const int ql = wl - 2;
    for (int w = tid; w < D << ql; w += nthr) {
      const uint32_t* t = tile + (w >> ql) * ld + 4 * (w & ((1 << ql) - 1));
      reinterpret_cast<u32x4*>(v)[w] = u32x4{t[0], t[1], t[2], t[3]};
    }
    return;
  }
  for (int w = tid; w < words; w += nthr) {
    const int d = w >> wl, g = w & ((1 << wl) - 1), t0 = 4 * g;
    if (t0 >= end || (t0 + 4 <= held && !grown)) continue;
    uint32_t out = tile[d * ld + g];
    if (t0 < held || t0 + 4 > end) {
      const uint32_t old = v[w], kept = grown ? rescale(old) : old;
      uint32_t r = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t from = t0 + i < held ? kept : t0 + i < end ? out : old;
        r |= from & (255u << (8 * i));
      }
      out = r;
    }
    v[w] = out;
  }
}

// Values `at` .. at + 7 of the rows of a piece's tokens 4 tg .. 4 tg + 3; where one is not of the piece, of its nearest row.
// No branch lies between the loads, which would make the compiler wait for each.
__device__ __forceinline__ void load_rows(const Piece& P, const uint16_t* src, int64_t st, int vec, int tg, int at, u32x4* x) {
  const uint16_t* row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) row[i] = src + (P.row0 + min(max(4 * tg + i, P.lo), P.hi - 1)) * st + at;
  if (vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = load8(row[i], true);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = load8(row[i], false);
  }
}

// The 16-bit values of a piece that thread (tg, dg) holds, zeros where there are none, and the largest word of
// magnitudes: those of 16-bit values are ordered like their words, NaN last.
template <int D>
__device__ __forceinline__ uint32_t load_unit(const Piece& P, const uint16_t* src, int64_t st, int vec, int tid, bool mine,
                                              u32x4* x) {
  const int tg = tid / (D / 8), dg = tid % (D / 8);
  u16x2 big = {0, 0};
  load_rows(P, src, st, vec, tg, 8 * dg, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = mine && 4 * tg + i >= P.lo && 4 * tg + i < P.hi;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[i][j] = in ? x[i][j] : 0u;
      big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, x[i][j] & 0x7fff7fffu));
    }
  }
  return max((uint32_t)big[0], (uint32_t)big[1]);
}

template <typename IO>
__device__ __forceinline__ float half_of(const u32x4& w, int j) {
  return IO::get((uint16_t)(w[j / 2] >> (16 * (j & 1))));
}

// An append of 16-bit values as they are (kv_cache.hip) or turned (kv_rotate.hip).
inline unsigned unit_threads(int block, int D) { return (unsigned)((block * D / 32 + 63) / 64 * 64); }
inline unsigned tile_bytes(int block, int D) { return (unsigned)(D * (block / 4 + 1) * 4); }
inline int64_t kv_pieces(const KvSeqs& S, int shift) {
  return S.cu ? (S.tokens >> shift) + 2 * (int64_t)S.batch + 2 : S.batch;
}

template <typename F>
int by_width(int D, F&& f) {
  switch (D) {
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
    case 192: return f(std::integral_constant<int, 192>());
    default: return f(std::integral_constant<int, 256>());
  }
}

// The values' part of an append's arguments, checked.
int append_check(const char* name, const pp_kv_cache* cache, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                 int64_t v_st, int64_t v_sh, int dtype, int64_t tokens, const int32_t* table, int64_t table_ld,
                 int64_t table_width, const int32_t* lengths, const int32_t* cu, int64_t batch, AppendArgs* A);

}  // namespace pp
