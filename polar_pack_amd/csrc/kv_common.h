// The key/value cache in 8 or 4 bits: its layout, the sequences of a call and the codes.
//
// A cache is `pages` pages of `block` tokens (16, 32, 64 or 128) for `heads` heads of D values:
//   K codes [page][head][token][D], V codes [page][head][D][token], one byte a value, and one
//   float32 scale for each page and head of either; a value is code * scale.
// V is kept transposed because a matrix-core operand of the product with the weights wants
// consecutive tokens of one d in a lane: here those are 16 consecutive bytes, and no kernel
// transposes V through LDS.
//
// In 4 bits (PP_KV_E2M1) a byte holds two codes, of neighbouring d (K) or tokens (V), and every 32 values d of a
// token and head have a scale of their own, a power of two as an e5m2 byte: K [page][head][token][D / 32],
// V [page][head][D / 32][token].  Powers of two make the codes exact functions of the values, whatever the order of
// operations, let the conversion to halves take K's scale along, and leave code * scale exact in fp16; as the upper
// byte of an fp16 number a V scale becomes a factor by one permute.  A token's codes depend on no other token, so an
// append never rounds again what is there.
#pragma once

#include "pp_common.h"

namespace pp {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float KV_SCALE_MIN = 5.421010862427522e-20f;   // 2^-64

struct KvCache {
  uint8_t* k;
  uint8_t* v;
  float* ks;        // in 4 bits bytes: scales_k, scales_v
  float* vs;
  int64_t pages;
  int heads, block, shift;   // block == 1 << shift
};
__device__ __forceinline__ uint8_t* scales_k(const KvCache& C) { return reinterpret_cast<uint8_t*>(C.ks); }
__device__ __forceinline__ uint8_t* scales_v(const KvCache& C) { return reinterpret_cast<uint8_t*>(C.vs); }

// The sequences of a call: token t of sequence b lies in page table[b*ld + t / block].  The call's
// tokens cu[b] .. cu[b+1]-1 are the last of sequence b's lengths[b] tokens; without cu every
// sequence has one.  Everything read from the device is held to its range before it is used as an
// index: cu to [0, tokens], pages to [0, pages), positions to [0, width * block).
struct KvSeqs {
  const int32_t* table;
  int64_t ld;
  const int32_t* lengths;
  const int32_t* cu;
  int width, batch, tokens;
};

// First token of sequence b, b in [0, batch + 1]: sequence `batch` is what lies past cu[batch].
__device__ __forceinline__ int kv_start(const KvSeqs& S, int b) {
  if (b <= 0) return 0;
  if (b > S.batch) return S.tokens;
  if (S.cu == nullptr) return b < S.tokens ? b : S.tokens;
  const int c = S.cu[b];
  return c < 0 ? 0 : c > S.tokens ? S.tokens : c;
}

// The sequence whose work items hold item `at`, where sequence b's begin at
// (start(b) * mul >> shift) + slack * b: the last b in [0, batch] that begins at or before `at`.
// A wavefront looks at 64 sequences a step.  Every wavefront of the workgroup calls it.
__device__ __forceinline__ int kv_begin(const KvSeqs& S, int b, int mul, int shift, int slack) {
  return (int)((int64_t)kv_start(S, b) * mul >> shift) + slack * b;
}

__device__ __forceinline__ int kv_find(const KvSeqs& S, int at, int mul, int shift, int slack) {
  const int lane = threadIdx.x & 63;
  int lo = 0, span = S.batch + 1;            // the answer is in [lo, lo + span)
  while (span > 1) {
    const int step = (span + 63) / 64;
    const int b = lo + lane * step;
    const bool ok = b < lo + span && kv_begin(S, b, mul, shift, slack) <= at;
    const uint64_t mask = __ballot(ok || lane == 0);
    const int last = 63 - __builtin_clzll(mask);
    const int end = lo + span;
    lo = lo + last * step;
    span = end - lo < step ? end - lo : step;
  }
  return uniform(lo);
}

// NaN-keeping maximum of magnitudes: as unsigned words the order is that of the values, NaN last.
__device__ __forceinline__ uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t w = __shfl_xor(v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}

template <int CODES>
struct KvCodes;

template <>
struct KvCodes<PP_KV_INT8> {
  static constexpr float kMax = 127.f;
  // Beside 1.5 * 2^23 a float has no bits below 1: the sum is rounded, ties to even, and its last byte is the
  // code.  Numbers only.
  static __device__ __forceinline__ uint32_t code(float x) {
    return __float_as_uint(__builtin_amdgcn_fmed3f(x, -127.f, 127.f) + 12582912.f);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {
    return __builtin_amdgcn_perm(code(b), code(a), 0x0c0c0400u) | __builtin_amdgcn_perm(code(d), code(c), 0x04000c0cu);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  }
  // Four codes as fp16, exactly: byte ^ 0x80 under the exponent byte of 1024 is 1024 + 128 + code.
  static __device__ __forceinline__ void halves(uint32_t w, f16x2& lo, f16x2& hi) {
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 off = {(f16)1152.f, (f16)1152.f};
    lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
    hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
  }
};

template <>
struct KvCodes<PP_KV_E4M3> {
  static constexpr float kMax = 448.f;
  static __device__ __forceinline__ float hold(float x) { return __builtin_amdgcn_fmed3f(x, -448.f, 448.f); }
  static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(hold(a), hold(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hold(c), hold(d), w, true);
  }
  static __device__ __forceinline__ void halves(uint32_t w, f16x2& lo, f16x2& hi) {
    lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float* x) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = lo[0]; x[1] = lo[1]; x[2] = hi[0]; x[3] = hi[1];
  }
};

// Scales of 4-bit codes: the exponent of the smallest power of two from 2^-14 to 2^13 that is a seventh of the
// magnitude `bits` or more, its float and its byte.
__device__ __forceinline__ int scale4(uint32_t bits) {
  const int e = (int)((bits + 0x1fffffu) >> 23) - 129;      // past 1.75 * 2^k: one more
  return min(max(e, -14), 13);
}
__device__ __forceinline__ float scale4_value(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ uint32_t scale4_byte(int e) { return (uint32_t)(e + 15) << 2; }
constexpr uint32_t SCALE4_NAN = 0x7f;

// 16-bit values in memory as float and back.
struct IoF16 {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(uint16_t u) { return (float)__builtin_bit_cast(f16, u); }
  static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (f16)x); }
  static __device__ __forceinline__ uint32_t put2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
  }
};
struct IoBf16 {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
  static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
  static __device__ __forceinline__ uint32_t put2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
  }
};
struct IoF32 {
  typedef float raw;
  static __device__ __forceinline__ float get(float u) { return u; }
  static __device__ __forceinline__ float put(float x) { return x; }
};

// 8 consecutive 16-bit values; `vec`: at a 16-byte boundary.
__device__ __forceinline__ u32x4 load8(const uint16_t* p, bool vec) {
  if (vec) return *reinterpret_cast<const u32x4*>(p);
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
  return w;
}

// Byte i of word j becomes byte j of word i.
__device__ __forceinline__ void swap_bytes(uint32_t* w) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Host side: the checks every entry point makes of a cache and its sequences.
int kv_check_cache(const pp_kv_cache* c, KvCache* out);
int kv_check_seqs(const KvCache& c, const int32_t* table, int64_t ld, int64_t width, const int32_t* lengths, const int32_t* cu,
                  int64_t batch, int64_t tokens, KvSeqs* out);

}  // namespace pp
