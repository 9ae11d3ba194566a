// Attention of many rows a sequence and head (prompts, pieces of prompts) to the 8-bit cache.
//
// A workgroup of 4 wavefronts takes 128 NQ rows of one sequence and key/value head, a wavefront 32 NQ
// of them, and walks the keys in tiles of 64.  The codes of a tile become fp16 once, on their way
// into LDS, for all four wavefronts; both products run on v_mfma_f32_32x32x16_f16.
//
// S^T = K Q^T leaves a lane 16 scores of one row (column lane % 32) for each 32 keys.  Which key is
// which row of the product is free: row m takes the key whose bits 2 and 3 are those of m swapped, so
// that the 8 scores of a lane that make one operand of O^T = V^T P^T belong to 8 consecutive keys,
// 16 c + 8 (lane / 32) + 0..7, and V's operand is one 16-byte read of a row of the transposed V.
// LDS rows are swizzled in 16-byte chunks so that 16 lanes of a read touch every bank once.
#include "kv_attn.h"

namespace pp {

// 16-byte chunk c of row r: rows of a multiple of 256 bytes by r % 16, of an odd multiple of 128 by r / 2 % 8.
template <int BYTES>
__device__ __forceinline__ int swizzled(int r, int c) {
  return BYTES % 256 == 0 ? r * BYTES + 16 * (c ^ (r & 15)) : r * BYTES + 16 * (c ^ ((r >> 1) & 7));
}

template <int CODES, typename IO, int D, int NQ, int NP>
__global__ __launch_bounds__(256, 1) void kv_attn_many_kernel(const AttnArgs A) {
  constexpr int KS = D / 16, DT = D / 32, R = 128 * NQ, CH = D / 64;   // chunks of 16 codes a thread stages
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
    if (!kv_deal(A, R, T, U)) return;
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

  // this lane's rows: column m32 of the wavefront's NQ row tiles
  f16x8 q[NQ][KS];
  float rf[NQ];
  int lo[NQ], hi[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = T.r0 + 32 * (NQ * wave + n) + m32;
    const bool real = r < T.rows;
    const int i = real ? r / A.group : 0, gq = real ? r - i * A.group : 0;
    kv_visible(A, T, i, real, lo[n], hi[n]);
    rf[n] = many_q<IO, D>(A, T.s0 + i, h * A.group + gq, hh, real, q[n]);
  }
  f32x16 o[NQ][DT];
  float mx[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    mx[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int k = 0; k < 16; ++k) o[n][d][k] = 0.f;
  }

  // Staging: thread t holds, of each 256 chunks of 16 codes of a tile, K chunk t (key t / (D / 16)) and V
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
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = tid + 256 * c, key = at / KS, part = at % KS;
      kw[c] = *reinterpret_cast<const u32x4*>(C.k + pick(key >> 4) + ((tile * 64 + key) & (bs - 1)) * D + 16 * part);
      const int d = at >> 2, group = at & 3;
      vw[c] = *reinterpret_cast<const u32x4*>(C.v + pick(group) + d * bs + ((tile * 64 + 16 * group) & (bs - 1)));
    }
  };
  auto store = [&](int tile, int buf) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = tid + 256 * c, key = at / KS, part = at % KS, d = at >> 2, group = at & 3;
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
    bool any = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) any |= (t0 < hi[n]) & (t0 + 64 > lo[n]);
    if (__any(any)) {
      f32x16 s[NQ][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int k = 0; k < 16; ++k) s[n][t][k] = 0.f;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          const f16x8 ka = *reinterpret_cast<const f16x8*>(&lds[buf][swizzled<2 * D>(32 * t + mk, 2 * c + hh)]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, q[n][c], s[n][t], 0, 0, 0);
        }
      }
      float lv[4], iv[4], kq[4];
      bool vbad = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = vs[e * NP / 4];
        const bool bad = mag(v) >= 0x7f800000u;
        vbad |= bad;
        const float vq = bad ? 1.f : fmaxf(v, KV_SCALE_MIN);
        lv[e] = __builtin_amdgcn_logf(vq);
        iv[e] = 1.0f / vq;
        kq[e] = ks[e * NP / 4];
      }
      f16x8 p[NQ][4];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float e[2][16], top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int k = 0; k < 16; ++k) e[t][k] = s[n][t][k] * (kq[2 * t + k / 8] * rf[n]) + lv[2 * t + k / 8];
        if (__any((okv != 15) | (t0 < lo[n]) | (t0 + 64 > hi[n]))) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int key = t0 + 32 * t + 16 * (k / 8) + 8 * hh + k % 8;
              const bool see = (okv >> (2 * t + k / 8) & 1) & (key >= lo[n]) & (key < hi[n]);
              e[t][k] = see ? e[t][k] : -INFINITY;
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int k = 0; k < 16; ++k) top = fmaxf(top, e[t][k]);
        top = max_halves(top);
        if (__any(top > mx[n])) {
          const float mn = fmaxf(mx[n], top);
          const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx[n] - mn);
          mx[n] = mn;
          l[n] *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[n][d] *= f;
        }
        const float ref = (mx[n] == -INFINITY ? 0.f : mx[n]) - KV_P_LOG2;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float w = __builtin_amdgcn_exp2f(e[g / 2][8 * (g & 1) + k] - ref);
            sum += w;
            p[n][g][k] = (f16)w;
          }
          l[n] += sum * iv[g];
        }
        if (__any(vbad)) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int key = t0 + 16 * g + 8 * hh + k;
              const bool see = (okv >> g & 1) & (key >= lo[n]) & (key < hi[n]) & (mag(vs[g * NP / 4]) >= 0x7f800000u);
              p[n][g][k] = see ? (f16)NAN : p[n][g][k];
            }
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const f16x8 va = *reinterpret_cast<const f16x8*>(&lds[buf][KB + swizzled<128>(32 * d + m32, 2 * g + hh)]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) o[n][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, p[n][g], o[n][d], 0, 0, 0);
        }
    }
    store(tile + 1, buf ^ 1);
    __syncthreads();
  }

  // a lane holds values 32 d + 8 k + 4 hh + 0..3 of its rows
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] = sum_halves(l[n]);
    const int rr = 32 * (NQ * wave + n) + m32, r = T.r0 + rr;
    if (r >= T.rows) continue;
    if (runs == 1) {
      const int i = r / A.group;
      const int64_t at = (int64_t)(T.s0 + i) * A.q_heads + h * A.group + (r - i * A.group);
      const float inv = kv_inverse(l[n]);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          store4<IO>(A.out + at * D + 32 * d + 8 * k + 4 * hh,
                     f32x4{o[n][d][4 * k] * inv, o[n][d][4 * k + 1] * inv, o[n][d][4 * k + 2] * inv, o[n][d][4 * k + 3] * inv});
      if (A.lse && hh == 0) A.lse[at] = kv_lse(mx[n], l[n]);
    } else {
      // workgroup owner + i has part i; the owner's is its second
      float* part = A.parts + (((int64_t)h * A.shares + blockIdx.x) * 2 + (run == 0)) * R * (D + 4) + (int64_t)rr * (D + 4);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<f32x4*>(part + 32 * d + 8 * k + 4 * hh) =
              f32x4{o[n][d][4 * k], o[n][d][4 * k + 1], o[n][d][4 * k + 2], o[n][d][4 * k + 3]};
      if (hh == 0) {
        part[D] = mx[n];
        part[D + 1] = l[n];
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
  auto pick = [&](auto nq) {
    constexpr int NQ = decltype(nq)::value;
    auto kern = A.C.block >= 64 ? kv_attn_many_kernel<CODES, IO, D, NQ, 1>
                : A.C.block == 32 ? kv_attn_many_kernel<CODES, IO, D, NQ, 2> : kv_attn_many_kernel<CODES, IO, D, NQ, 4>;
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, A);
  };
  if constexpr (D <= 128) {
    if (P.rows == 256) pick(std::integral_constant<int, 2>());
    else pick(std::integral_constant<int, 1>());
  } else {
    pick(std::integral_constant<int, 1>());
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
