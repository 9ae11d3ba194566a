// Rotary positions: pair f of a row is turned by the angle position * frequency(f).
//
// A frequency is kept as the 64-bit fraction of a turn that one step of position is, so that position * frequency mod 2^64
// is the angle of that fraction, exact for every 64-bit position (a float32 product would be off by 2^-24 * position radians), and
// takes no table of positions: nothing has to arrive from memory but the position and a few frequencies.  What the fraction was
// rounded by, up to 2^-65 of a turn, the position multiplies: 2e-13 radians at 10^6, 5e-8 at 2^38, most of a radian at 2^62.  The
// sine and cosine of the rest below an eighth of a turn are their power series.
//
// In float32 (rows, and keys on their way into 8 bits) a sine or cosine is within 9.8e-8, 2.0e-8 in the mean square, where one
// rounding of the exact value leaves 3.0e-8 and 1.5e-8: the angle is 32 bits of a turn as a float, and the last two
// steps round.  Rows of 16 bits are rounded by up to 2^-11 afterwards; an 8-bit code differs from that of the exact key only
// where the key is within 2^-22 of its pair's magnitude of a tie.  Keys on their way into 4 bits take the series in 64 bits.
#pragma once

#include "kv_common.h"

namespace pp {

struct Rot {
  const uint64_t* turns;     // [half]
  const uint8_t* axes;       // [half], or null: one axis
  const void* pos;           // [axis][token], or null: each token's own place in its sequence
  int64_t pos_ld;
  int n_axes;
  int half;                  // frequencies; values 0 .. 2 half - 1 are turned
  int neighbours;            // pair f is values 2f, 2f + 1; otherwise f, f + half
  int wide;                  // positions are int64, otherwise int32
  float scaling;
};

template <typename T>
struct Trig {
  T c, s;
};

// cos and sin of the fraction t / 2^64 of a turn.
__device__ __forceinline__ void turn_trig(uint64_t t, Trig<double>& o) {
  const uint32_t k = (uint32_t)((t + (1ull << 61)) >> 62);            // the nearest quarter
  const double x = (double)(int64_t)(t - ((uint64_t)k << 62)) * 3.4061215800865545e-19;   // 2 pi / 2^64
  const double z = x * x;
  // terms to x^15 and x^16: what is left out is below 2^-53 at pi / 4 (x^17 / 17! 2^-54, x^18 / 18! 2^-59), and with the
  // roundings both are within 1.9e-16 (to x^14 the cosine was 1.1e-15 off, and a 4-bit code beside a border the wrong one)
  double s = -7.647163731819816e-13;
  s = fma(s, z, 1.6059043836821613e-10);
  s = fma(s, z, -2.505210838544172e-08);
  s = fma(s, z, 2.7557319223985893e-06);
  s = fma(s, z, -1.9841269841269841e-04);
  s = fma(s, z, 8.3333333333333332e-03);
  s = fma(s, z, -1.6666666666666666e-01);
  s = fma(s * z, x, x);
  double c = 4.779477332387385e-14;
  c = fma(c, z, -1.1470745597729725e-11);
  c = fma(c, z, 2.08767569878681e-09);
  c = fma(c, z, -2.7557319223985888e-07);
  c = fma(c, z, 2.4801587301587302e-05);
  c = fma(c, z, -1.3888888888888889e-03);
  c = fma(c, z, 4.1666666666666664e-02);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.0);
  const double a = k & 1 ? s : c, b = k & 1 ? c : s;
  o.c = (k + 1) & 2 ? -a : a;
  o.s = k & 2 ? -b : b;
}
__device__ __forceinline__ void turn_trig(uint64_t t, Trig<float>& o) {
  const uint32_t h = (uint32_t)(t >> 32);                              // 2^-32 of a turn: 1.5e-9
  const uint32_t k = (h + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(h - (k << 30)) * 1.4629180792671596e-09f;              // 2 pi / 2^32
  const float z = x * x;
  float s = 2.7557319e-06f;                                            // terms to x^9 and x^10: below 2^-27
  s = fmaf(s, z, -1.9841270e-04f);
  s = fmaf(s, z, 8.3333333e-03f);
  s = fmaf(s, z, -1.6666667e-01f);
  s = fmaf(s * z, x, x);
  float c = -2.7557319e-07f;
  c = fmaf(c, z, 2.4801587e-05f);
  c = fmaf(c, z, -1.3888889e-03f);
  c = fmaf(c, z, 4.1666667e-02f);
  c = fmaf(c, z, -0.5f);
  c = fmaf(c, z, 1.0f);
  const float a = k & 1 ? s : c, b = k & 1 ? c : s;
  o.c = (k + 1) & 2 ? -a : a;
  o.s = k & 2 ? -b : b;
}

// A token's position on an axis, below n_axes.
__device__ __forceinline__ int64_t rot_load(const Rot& R, int axis, int64_t token) {
  const int64_t at = axis * R.pos_ld + token;
  return R.wide ? reinterpret_cast<const int64_t*>(R.pos)[at] : reinterpret_cast<const int32_t*>(R.pos)[at];
}
__device__ __forceinline__ int64_t rot_position(const Rot& R, int f, int64_t token) {
  return rot_load(R, R.axes ? min((int)R.axes[f], R.n_axes - 1) : 0, token);
}

template <typename T>
__device__ __forceinline__ Trig<T> rot_trig(const Rot& R, int f, int64_t position) {
  Trig<T> o;
  turn_trig((uint64_t)position * R.turns[f], o);
  o.c *= (T)R.scaling;
  o.s *= (T)R.scaling;
  return o;
}

// 8 consecutive values as they lie in memory; `vec`: at a 16-byte boundary.
template <typename IO>
struct Row8 {
  u32x4 w[sizeof(typename IO::raw) / 2];
  __device__ __forceinline__ void load(const typename IO::raw* p, bool vec) {
    if constexpr (sizeof(typename IO::raw) == 4) {
      if (vec) {
        w[0] = reinterpret_cast<const u32x4*>(p)[0];
        w[1] = reinterpret_cast<const u32x4*>(p)[1];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i / 4][i % 4] = __float_as_uint(p[i]);
      }
    } else {
      w[0] = load8(p, vec);
    }
  }
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(typename IO::raw) == 4) x[i] = __uint_as_float(w[i / 4][i % 4]);
      else x[i] = IO::get((uint16_t)(w[0][i / 2] >> (16 * (i & 1))));
    }
  }
};
template <typename IO>
__device__ __forceinline__ void store_row(typename IO::raw* p, bool vec, const float* x) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = IO::put(x[i]);
    return;
  }
  if constexpr (sizeof(typename IO::raw) == 4) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    *reinterpret_cast<u32x4*>(p) = u32x4{IO::put2(x[0], x[1]), IO::put2(x[2], x[3]), IO::put2(x[4], x[5]),
                                         IO::put2(x[6], x[7])};
  }
}

// Rows (token, head) of D values; a thread takes 8 pairs of a token, or 16 values that are not turned, of
// some of its heads: unit u of rot_units.  Their sines and cosines stay in registers over the heads.
struct RotRows {
  const void* x;
  void* out;
  int64_t x_st, x_sh, o_st, o_sh;
  int tokens, heads, D, per;     // `per` heads a thread
  int vec;
};
__host__ __device__ inline int rot_units(int half, int D) { return half / 8 + (D - 2 * half + 15) / 16; }

// `none`: a token of no sequence, whose row is zero.  AHEAD heads are read before the first of them is written: rows may
// be turned where they lie, so that no load may pass a store before it.  2 beside an append in 4 bits, whose 108
// registers leave room for few wavefronts (16 ragged prompts 100.5 -> 98.3 us; 3 98.2); 1 beside one in 8 bits, of 78
// (4 prompts 26.5 us, with 2 27.3), and where rows are all there is (16,200 tokens 26.8 us, with 2 27.2).
template <typename IO, int AHEAD>
__device__ __forceinline__ void rotate_unit(const Rot& R, const RotRows& A, int token, int u, int group, int64_t own,
                                            bool none) {
  typedef typename IO::raw raw;
  const int h0 = group * A.per, h1 = min(A.heads, h0 + A.per);
  const raw* x = reinterpret_cast<const raw*>(A.x) + token * A.x_st + h0 * A.x_sh;
  raw* o = reinterpret_cast<raw*>(A.out) + token * A.o_st + h0 * A.o_sh;
  const int units = R.half / 8;
  int at0, at1;                   // the unit's two pieces of 8 values
  Trig<float> w[8];
  if (u < units && R.pos && R.axes) {
    // Up to four axes: the token's positions first, all at once, then a choice for each frequency.
    at0 = R.neighbours ? 16 * u : 8 * u;
    at1 = R.neighbours ? at0 + 8 : at0 + R.half;
    int64_t p[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) p[a] = rot_load(R, min(a, R.n_axes - 1), token);
    uint8_t axis[8];
    __builtin_memcpy(axis, R.axes + 8 * u, 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int a = axis[i];
      int64_t at = a == 0 ? p[0] : a == 1 ? p[1] : a == 2 ? p[2] : p[3];
      if (R.n_axes > 4) at = rot_load(R, min(a, R.n_axes - 1), token);
      w[i] = rot_trig<float>(R, 8 * u + i, at);
    }
  } else if (u < units) {
    if (R.pos) own = rot_load(R, 0, token);
    at0 = R.neighbours ? 16 * u : 8 * u;
    at1 = R.neighbours ? at0 + 8 : at0 + R.half;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = rot_trig<float>(R, 8 * u + i, own);
  } else {
    at0 = 2 * R.half + 16 * (u - units);
    at1 = at0 + 8 < A.D ? at0 + 8 : at0;
  }
  const bool turned = u < units, pairs = R.neighbours;
#pragma unroll 2
  for (int h = h0; h < h1; h += AHEAD, x += AHEAD * A.x_sh, o += AHEAD * A.o_sh) {
    Row8<IO> wa[AHEAD], wb[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const raw* const from = x + min(k, h1 - 1 - h) * A.x_sh;
      wa[k].load(from + at0, A.vec);
      wb[k].load(from + at1, A.vec);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      float a[8], b[8];
      wa[k].get(a);
      wb[k].get(b);
      if (turned) {
        if (pairs) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = a[2 * i], q = a[2 * i + 1], r = b[2 * i], t = b[2 * i + 1];
            a[2 * i] = p * w[i].c - q * w[i].s;
            a[2 * i + 1] = q * w[i].c + p * w[i].s;
            b[2 * i] = r * w[4 + i].c - t * w[4 + i].s;
            b[2 * i + 1] = t * w[4 + i].c + r * w[4 + i].s;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p = a[i], q = b[i];
            a[i] = p * w[i].c - q * w[i].s;
            b[i] = q * w[i].c + p * w[i].s;
          }
        }
      }
      if (none) {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
      }
      if (h + k < h1) {
        store_row<IO>(o + k * A.o_sh + at0, A.vec, a);
        store_row<IO>(o + k * A.o_sh + at1, A.vec, b);
      }
    }
  }
}

// Host side.
// Threads that share a unit's heads: as many as make `threads` a CU, since a thread's sines and cosines cost as much as
// two or three heads.  512 where rows are all there is (16,200 tokens of 18 heads of 128: 26.7 us, with 1024 27.5); 1024
// beside an append (16 ragged prompts of 32 query heads 99.9 us, with 512 104.9, with 4096 102.7; 4 prompts of 16 27.1,
// 26.9, 35.3).
inline int64_t rot_groups(int64_t units, int64_t heads, int threads) {
  const int64_t want = ((int64_t)device_cu_count() * threads + units - 1) / units;
  return want < 1 ? 1 : want < heads ? want : heads;
}
int rot_check(const pp_rotary* r, const void* positions, int64_t pos_ld, int pos_type, int64_t tokens, int64_t head_dim,
              bool needed, Rot* out);

}  // namespace pp
