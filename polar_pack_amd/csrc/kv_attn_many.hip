// Attention of many rows a sequence and head (prompts, pieces of prompts) to the 8-bit cache.
//
// A workgroup of 4 or 8 wavefronts takes 32 rows a wavefront of one sequence and key/value head and
// walks the keys in tiles of 64.  The codes of a tile become fp16 once, on their way
// into LDS, for all wavefronts; both products run on v_mfma_f32_32x32x16_f16.
//
// S^T = K Q^T leaves a lane 16 scores of one row (column lane % 32) for each 32 keys.  Which key is
// which row of the product is free: row m takes the key whose bits 2 and 3 are those of m swapped, so
// that the 8 scores of a lane that make one operand of O^T = V^T P^T belong to 8 consecutive keys,
// 16 c + 8 (lane / 32) + 0..7, and V's operand is one 16-byte read of a row of the transposed V.
// LDS rows are swizzled in 16-byte chunks so that 16 lanes of a read touch every bank once.
#include "kv_attn.h"

namespace pp {

constexpr float KV_NONE = -1e30f, KV_NEAR = 12.f, KV_FAR = 15.9f;

// 16-byte chunk c of row r: rows of a multiple of 256 bytes by r % 16, of an odd multiple of 128 by r / 2 % 8.
template <int BYTES>
__device__ __forceinline__ int swizzled(int r, int c) {
  return BYTES % 256 == 0 ? r * BYTES + 16 * (c ^ (r & 15)) : r * BYTES + 16 * (c ^ ((r >> 1) & 7));
}

template <int CODES, typename IO, int D, int WAVES, int NP>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void kv_attn_many_kernel(const AttnArgs A) {
  constexpr int KS = D / 16, DT = D / 32, R = 32 * WAVES, THREADS = 64 * WAVES;
  constexpr int CH = 4 * D < THREADS ? 1 : 4 * D / THREADS;            // chunks of 16 codes of K and of V a thread stages
  constexpr int KB = 64 * D * 2;                                       // bytes of a tile of K or V
  __shared__ __align__(16) uint8_t lds[2][2 * KB];
  const KvCache& C = A.C;
  const KvSeqs& S = A.S;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), m32 = lane & 31, hh = lane >> 5;
  const int h = blockIdx.y, shift = C.shift, bs = C.block;
  RowTile T;
  Deal U;
  ManyPart* const desc = A.desc ? A.desc + (int64_t)h * A.shares + blockIdx.x : nullptr;
  if (A.shares) {
    if (tid == 0) desc->runs = 0;
    if (!kv_deal<THREADS>(A, R, T, U)) return;
  } else {
    // the last row tiles first: they see the most keys
    if (!kv_row_tile(A, gridDim.x - 1 - blockIdx.x, R, T)) return;
    U = Deal{0, 1, 1, T.lo >> 6, 1, 0};
  }
  for (;; kv_deal_next(A, R, T, U)) {
  int a = T.lo >> 6, z = T.hi > T.lo ? (T.hi + 63) >> 6 : a, run = 0, runs = 1, owner = 0;
  if (A.shares) {
    const int64_t begin = U.at - U.into + KV_TURN;             // of its tiles that hold keys
    const int left = U.tiles + KV_TURN - U.into;
    const int take = U.end - U.at < left ? (int)(U.end - U.at) : left;
    const int t0 = max(U.into - KV_TURN, 0), t1 = U.into + take - KV_TURN;
    U.at += take;
    if (t1 <= 0) return;                                       // the share ends before them
    owner = (int)(begin / U.share);
    runs = (int)((begin + U.tiles - 1) / U.share) - owner + 1;
    run = blockIdx.x - owner;
    kv_tile_range(A, R, T);
    a = max(U.first + t0, T.lo >> 6);
    z = min(U.first + t1, T.hi > T.lo ? (T.hi + 63) >> 6 : 0);
    z = max(a, z);
  } else {
    U.at = U.end;
  }

  // this lane's row: column m32 of the wavefront's row tile
  f16x8 q[KS];
  int lo, hi;
  const int rr = 32 * wave + m32, row = T.r0 + rr;
  const bool real = row < T.rows;
  const int token = real ? row / A.group : 0, gq = real ? row - token * A.group : 0;
  kv_visible(A, T, token, real, lo, hi);
  const float rf = many_q<IO, D>(A, T.s0 + token, h * A.group + gq, hh, real, q);
  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int k = 0; k < 16; ++k) o[d][k] = 0.f;
  // Weights are e^(s - ref) vs: ref is 2^12 below the largest exponent seen when it was set, and is
  // set anew only where a weight would pass 2^KV_FAR, so that most tiles need no maximum over a row's lanes.
  float ref = KV_NONE, l = 0.f;

  // Staging: thread t holds, of each THREADS chunks of 16 codes of a tile, K chunk t (key t / (D / 16)) and V
  // chunk t (value t / 4, keys 16 (t % 4) ..).  Lane e of a wavefront holds table entry ids0 + e.
  const int32_t* table = S.table + (int64_t)T.b * S.ld;
  int ids = -1, ids0 = INT32_MIN / 2;
  u32x4 kw[CH], vw[CH];
  float ks_n[NP], vs_n[NP];
  int ok_n = 0;
  auto load = [&](int tile) {
    const int e0 = (tile * 64) >> shift;
    if (e0 < ids0 || e0 + NP > ids0 + 64) {
      ids0 = e0;
      ids = (int64_t)e0 + lane < S.width ? table[e0 + lane] : -1;
      ids = ids < C.pages ? ids : -1;
    }
    int page[NP];
    ok_n = 0;
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      page[e] = lane_read(ids, e0 - ids0 + e);
      ok_n |= (page[e] >= 0 ? (1 << (4 / NP)) - 1 : 0) << (4 / NP * e);
      page[e] = page[e] < 0 ? 0 : page[e];
      const int64_t ph = (int64_t)page[e] * C.heads + h;
      ks_n[e] = C.ks[ph];
      vs_n[e] = C.vs[ph];
    }
    auto pick = [&](int group) {
      int p = page[0];
#pragma unroll
      for (int e = 1; e < NP; ++e) p = group * NP / 4 == e ? page[e] : p;
      return ((int64_t)p * C.heads + h) * (bs * D);
    };
    if (4 * D < THREADS && tid >= 4 * D) return;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = tid + THREADS * c, key = at / KS, part = at % KS;
      kw[c] = *reinterpret_cast<const u32x4*>(C.k + pick(key >> 4) + ((tile * 64 + key) & (bs - 1)) * D + 16 * part);
      const int d = at >> 2, group = at & 3;
      vw[c] = *reinterpret_cast<const u32x4*>(C.v + pick(group) + d * bs + ((tile * 64 + 16 * group) & (bs - 1)));
    }
  };
  auto store = [&](int tile, int buf) {
    if (4 * D < THREADS && tid >= 4 * D) return;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = tid + THREADS * c, key = at / KS, part = at % KS, d = at >> 2, group = at & 3;
      f16x8 x, y;
      to_halves<CODES>(kw[c], x, y);
      *reinterpret_cast<f16x8*>(&lds[buf][swizzled<2 * D>(key, 2 * part)]) = x;
      *reinterpret_cast<f16x8*>(&lds[buf][swizzled<2 * D>(key, 2 * part + 1)]) = y;
      if (CODES == PP_KV_E4M3) {                 // codes past the length may be NaN
        const int seen = ok_n >> group & 1 ? T.lim - tile * 64 - 16 * group : 0;
        if (seen < 16) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int left = seen - 4 * w;
            vw[c][w] &= left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
          }
        }
      }
      to_halves<CODES>(vw[c], x, y);
      *reinterpret_cast<f16x8*>(&lds[buf][KB + swizzled<128>(d, 2 * group)]) = x;
      *reinterpret_cast<f16x8*>(&lds[buf][KB + swizzled<128>(d, 2 * group + 1)]) = y;
    }
  };

  const int mk = (m32 & 0x13) | (m32 & 4) << 1 | (m32 & 8) >> 1;       // key of row m32: bits 2 and 3 swapped
  if (a < z) {
    load(a);
    store(a, 0);
  }
  __syncthreads();
  for (int tile = a; tile < z; ++tile) {
    const int buf = (tile - a) & 1, okv = ok_n;
    float ks[NP], vs[NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) { ks[e] = ks_n[e]; vs[e] = vs_n[e]; }
    load(min(tile + 1, z - 1));
    const int t0 = tile * 64;
    if (__any((t0 < hi) & (t0 + 64 > lo))) {
      const uint8_t* const kb = lds[buf];
      const uint8_t* const vb = lds[buf] + KB;
      f32x16 s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f16x8 ka[KS];
#pragma unroll
        for (int c = 0; c < KS; ++c) ka[c] = *reinterpret_cast<const f16x8*>(kb + swizzled<2 * D>(32 * t + mk, 2 * c + hh));
#pragma unroll
        for (int k = 0; k < 16; ++k) s[t][k] = 0.f;
#pragma unroll
        for (int c = 0; c < KS; ++c) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[c], q[c], s[t], 0, 0, 0);
      }
      float lv[NP], iv[NP], kq[NP];
      bool vbad = false;
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        const bool bad = mag(vs[e]) >= 0x7f800000u;
        vbad |= bad;
        const float vq = bad ? 1.f : fmaxf(vs[e], KV_SCALE_MIN);
        lv[e] = __builtin_amdgcn_logf(vq);
        iv[e] = __builtin_amdgcn_rcpf(vq);
        kq[e] = ks[e] * rf;
      }
      const bool edge = __any((okv != 15) | (t0 < lo) | (t0 + 64 > hi));
      float e[4][8], top = -INFINITY;
      auto exponents = [&](float from) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int k = 0; k < 8; ++k) e[g][k] = s[g / 2][8 * (g & 1) + k] * kq[g * NP / 4] + (lv[g * NP / 4] - from);
        if (edge) {
          const int k0 = lo - t0 - 8 * hh, k1 = hi - t0 - 8 * hh;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int a0 = okv >> g & 1 ? k0 : 64;
#pragma unroll
            for (int k = 0; k < 8; ++k) e[g][k] = ((16 * g + k >= a0) & (16 * g + k < k1)) ? e[g][k] : -INFINITY;
          }
        }
        top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int k = 0; k < 8; ++k) top = fmaxf(top, e[g][k]);
      };
      exponents(ref);
      if (__any(top > KV_FAR)) {
        exponents(0.f);
        top = max_halves(top);
        const float next = fmaxf(ref, top - KV_NEAR);
        const float f = __builtin_amdgcn_exp2f(ref - next);
        ref = next;
        l *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
        exponents(ref);
      }
      f16x8 p[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          const f32x2 w = {__builtin_amdgcn_exp2f(e[g][k]), __builtin_amdgcn_exp2f(e[g][k + 1])};
          sum += w[0];
          sum += w[1];
          const f16x2 w16 = __builtin_convertvector(w, f16x2);
          p[g][k] = w16[0];
          p[g][k + 1] = w16[1];
        }
        l += sum * iv[g * NP / 4];
      }
      if (vbad) {                                              // the same in every lane
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int key = t0 + 16 * g + 8 * hh + k;
            const bool see = (okv >> g & 1) & (key >= lo) & (key < hi) & (mag(vs[g * NP / 4]) >= 0x7f800000u);
            p[g][k] = see ? (f16)NAN : p[g][k];
          }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f16x8 va[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) va[d] = *reinterpret_cast<const f16x8*>(vb + swizzled<128>(32 * d + m32, 2 * g + hh));
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[d], p[g], o[d], 0, 0, 0);
      }
    }
    store(tile + 1, buf ^ 1);
    __syncthreads();
  }

  // a lane holds values 32 d + 8 k + 4 hh + 0..3 of its row
  l = sum_halves(l);
  if (real) {
    if (runs == 1) {
      const int64_t at = (int64_t)(T.s0 + token) * A.q_heads + h * A.group + gq;
      const float inv = kv_inverse(l);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          store4<IO>(A.out + at * D + 32 * d + 8 * k + 4 * hh,
                     f32x4{o[d][4 * k] * inv, o[d][4 * k + 1] * inv, o[d][4 * k + 2] * inv, o[d][4 * k + 3] * inv});
      if (A.lse && hh == 0) A.lse[at] = kv_lse(ref + KV_P_LOG2, l);
    } else {
      // workgroup owner + i has part i; the owner's is its second
      float* part = A.parts + (((int64_t)h * A.shares + blockIdx.x) * 2 + (run == 0)) * R * (D + 4) + (int64_t)rr * (D + 4);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<f32x4*>(part + 32 * d + 8 * k + 4 * hh) =
              f32x4{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]};
      if (hh == 0) {
        part[D] = ref + KV_P_LOG2;
        part[D + 1] = l;
      }
    }
  }
  if (runs > 1 && run == 0 && tid == 0) *desc = ManyPart{runs, T.s0, T.r0, min(R, T.rows - T.r0)};
  if (U.at >= U.end) return;
  }
}

// The parts of shared row tiles: workgroup (owner, 16 of its row tile's rows, head), 16 threads a row.
template <typename IO, int D>
__global__ __launch_bounds__(256) void kv_attn_many_join_kernel(const AttnArgs A, int R) {
  constexpr int W = D / 16;
  const int pieces = R / 16, owner = blockIdx.x / pieces, h = blockIdx.y;
  const ManyPart P = A.desc[(int64_t)h * A.shares + owner];
  const int rr = blockIdx.x % pieces * 16 + (threadIdx.x >> 4), d0 = (threadIdx.x & 15) * W;
  if (P.runs < 2 || rr >= P.rows) return;
  const float* part = A.parts + ((int64_t)h * A.shares + owner) * (2 * R) * (D + 4) + (int64_t)rr * (D + 4);
  float m = -INFINITY, l = 0.f, v[W];
#pragma unroll
  for (int k = 0; k < W; ++k) v[k] = 0.f;
#pragma unroll 4
  for (int i = 0; i < P.runs; ++i) {
    const float* e = part + (int64_t)(i == 0 ? 1 : 2 * i) * R * (D + 4);
    f32x4 w[W / 4];
#pragma unroll
    for (int k = 0; k < W / 4; ++k) w[k] = *reinterpret_cast<const f32x4*>(e + d0 + 4 * k);
    join_part<W>(m, l, v, e[D], e[D + 1], reinterpret_cast<const float*>(w));
  }
  const int r = P.r0 + rr, i = r / A.group;
  const int64_t at = (int64_t)(P.s0 + i) * A.q_heads + h * A.group + (r - i * A.group);
  const float inv = kv_inverse(l);
#pragma unroll
  for (int k = 0; k < W; k += 4)
    store4<IO>(A.out + at * D + d0 + k, f32x4{v[k] * inv, v[k + 1] * inv, v[k + 2] * inv, v[k + 3] * inv});
  if (A.lse && d0 == 0) A.lse[at] = kv_lse(m, l);
}

template <int CODES, typename IO, int D>
static int many_launch(const AttnArgs& A, const AttnPlan& P, hipStream_t st) {
  const dim3 grid((unsigned)P.grid, (unsigned)A.C.heads);
  auto pick = [&](auto waves) {
    constexpr int WAVES = decltype(waves)::value;
    auto kern = A.C.block >= 64 ? kv_attn_many_kernel<CODES, IO, D, WAVES, 1>
                : A.C.block == 32 ? kv_attn_many_kernel<CODES, IO, D, WAVES, 2> : kv_attn_many_kernel<CODES, IO, D, WAVES, 4>;
    hipLaunchKernelGGL(kern, grid, dim3(64 * WAVES), 0, st, A);
  };
  if constexpr (D <= 128) {
    if (P.rows == 256) pick(std::integral_constant<int, 8>());
    else pick(std::integral_constant<int, 4>());
  } else {
    pick(std::integral_constant<int, 4>());
  }
  PP_LAUNCH_CHECK();
  if (P.shares) {
    hipLaunchKernelGGL((kv_attn_many_join_kernel<IO, D>), dim3((unsigned)(P.shares * (P.rows / 16)), (unsigned)A.C.heads),
                       dim3(256), 0, st, A, (int)P.rows);
    PP_LAUNCH_CHECK();
  }
  return PP_OK;
}

template <int CODES, typename IO>
static int many_width(const AttnArgs& A, const AttnPlan& P, int D, hipStream_t st) {
  switch (D) {
    case 64: return many_launch<CODES, IO, 64>(A, P, st);
    case 128: return many_launch<CODES, IO, 128>(A, P, st);
    case 192: return many_launch<CODES, IO, 192>(A, P, st);
    default: return many_launch<CODES, IO, 256>(A, P, st);
  }
}

int kv_attn_many(const AttnArgs& A, const AttnPlan& P, int D, int codes, int dtype, hipStream_t st) {
  if (codes == PP_KV_INT8)
    return dtype == PP_F16 ? many_width<PP_KV_INT8, IoF16>(A, P, D, st) : many_width<PP_KV_INT8, IoBf16>(A, P, D, st);
  return dtype == PP_F16 ? many_width<PP_KV_E4M3, IoF16>(A, P, D, st) : many_width<PP_KV_E4M3, IoBf16>(A, P, D, st);
}

}  // namespace pp
