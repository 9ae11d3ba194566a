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
//
// What bounds it: LDS and the vector unit as much as the matrix cores.  A tile of 64 keys and 256
// rows is 1024 cycles of products a wavefront, two a SIMD; its operands are 34 KB a wavefront, 2200 LDS cycles a
// CU with the staging; its weights are 32 exponentials a lane at a quarter of the rate, with the rest 1200-1500
// cycles.  Counted in the kernel: weights and staging ~1700 cycles, products ~1900, against 5600 a tile before
// the two halves of the wavefronts ran a barrier apart.  Four prompts of 2048 tokens, 16 query and 2 key
// heads of 128: 102 us, 0.67 PFLOP/s of 1.35 that the library's fp16 product reaches; 509 tokens behind
// 32,192: 166 us, 0.82.  Measured on the way (prompts / piece): wavefronts of 64 rows, one a SIMD 395 / 442 us (registers spilled),
// 8 of 32 rows 142 / 182, a barrier apart 144 / 167, heavy row tiles first and priority 103 / 164.
// 192 and 256 values a head: sums and queries of 32 rows take 144 and 192 registers, so 4 wavefronts, one a SIMD,
// whose products wait for their weights; at 256 28 bytes a lane spill.  The same prompts with 12 query and 4 key heads of 192
// 175 us, 0.44 PFLOP/s (a piece 272, 0.56), with 16 and 1 of 256 278, 0.50 (424, 0.64).
#include "kv_attn.h"

namespace pp {

// A barrier that nothing is scheduled across.
__device__ __forceinline__ void phase() {
  __builtin_amdgcn_sched_barrier(0);
  __syncthreads();
  __builtin_amdgcn_sched_barrier(0);
}

template <int I>
using Int = std::integral_constant<int, I>;

typedef const __attribute__((address_space(1))) u32x4* GlobalCodes;    // not a flat address, whose loads wait for LDS

constexpr float KV_NONE = -3.40282347e38f, KV_NEAR = 12.f, KV_FAR = 65000.f;   // no reference yet: no score is less

template <int CODES, typename IO, int D, int WAVES, int NP>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void kv_attn_many_kernel(const AttnArgs A) {
  constexpr int KS = D / 16, DT = D / 32, R = 32 * WAVES, THREADS = 64 * WAVES;
  constexpr int CH = 4 * D < THREADS ? 1 : 4 * D / THREADS;            // chunks of 16 codes of K and of V a thread stages
  constexpr bool PING = WAVES == 8;
  // Rows in LDS are 16 bytes longer than their halves, so that 16 rows' chunks of a column lie in all the banks
  // and every chunk of an operand is one address and a constant.
  constexpr int KR = 2 * D + 16, VR = 2 * 64 + 16, KB = 64 * KR, VB = D * VR, RING = PING ? 3 : 2;
  __shared__ __align__(16) uint8_t lds[RING * (KB + VB)];
  const KvCache& C = A.C;
  const KvSeqs& S = A.S;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), m32 = lane & 31, hh = lane >> 5;
  const int h = A.shares ? blockIdx.y : blockIdx.x % C.heads, shift = C.shift, bs = C.block;
  RowTile T;
  Deal U;
  ManyPart* const desc = A.desc ? A.desc + (int64_t)h * A.shares + blockIdx.x : nullptr;
  if (A.shares) {
    if (tid == 0) desc->runs = 0;
    if (!kv_deal<THREADS>(A, R, T, U)) return;
  } else {
    if (!kv_row_tile_from_last(A, blockIdx.x / C.heads, R, T)) return;
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
  // The same in every lane, and said so: what is asked of them becomes a branch then, and no lanes are switched off.
  // Where they were, hipcc 7.2 saved registers at the join before it switched the lanes on again, and loaded back
  // garbage (192 and 256 values a head in pages of 32, writes through such addresses; tests/test_device_code.py).
  a = uniform(a);
  z = uniform(z);
  T.lim = uniform(T.lim);

  // this lane's row: column m32 of the wavefront's row tile
  f16x8 q[KS];
  int lo, hi;
  const int rr = 32 * wave + m32, row = T.r0 + rr;
  const bool real = row < T.rows;
  const int token = real ? row / A.group : 0, gq = real ? row - token * A.group : 0;
  kv_visible(A, T, token, real, lo, hi);
  const float rf = many_q<IO, D>(A, T.s0 + token, h * A.group + gq, hh, real, q);
  if (!real) hi = T.lim;                                     // a row that is not there needs no mask
  const int all_lo = wave_max(lo), all_hi = wave_min(hi);    // keys that all the wavefront's rows see
  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int k = 0; k < 16; ++k) o[d][k] = 0.f;
  // Weights are e^(s - ref) vs: ref was the largest exponent less 12 when it was set, and is set anew
  // only where the weights of 8 keys pass what fp16 holds, so that most tiles need no maximum.
  float ref = KV_NONE, l = 0.f;

  // Staging: thread t holds, of each THREADS chunks of 16 codes of a tile, K chunk t (key t / (D / 16)) and V
  // chunk t (value t / 4, keys 16 (t % 4) ..).  Lane e of a wavefront holds table entry ids0 + e.
  const int32_t* table = S.table + (int64_t)T.b * S.ld;
  int ids = -1, ids0 = INT32_MIN / 2;
  struct Pages {
    int p[NP];
  };
  auto pages = [&](int tile) {                               // of the tile, or of the last one
    const int e0 = (min(tile, z - 1) * 64) >> shift;
    if (e0 < ids0 || e0 + NP > ids0 + 64) {
      ids0 = e0;
      ids = (int64_t)e0 + lane < S.width ? table[e0 + lane] : -1;
      ids = ids < C.pages ? ids : -1;
    }
    Pages P;
#pragma unroll
    for (int e = 0; e < NP; ++e) P.p[e] = lane_read(ids, e0 - ids0 + e);
    return P;
  };
  // A page's codes of this head: its first tile's address the same in every lane where a tile lies in
  // one page, so that a load is that and the thread's own offset.
  auto codes = [&](const uint8_t* all, const Pages& P, int group, int in_page) {
    int p = P.p[0];
#pragma unroll
    for (int e = 1; e < NP; ++e) p = group * NP / 4 == e ? P.p[e] : p;
    const uint8_t* at = all + ((int64_t)(p < 0 ? 0 : p) * C.heads + h) * (bs * D) + in_page;
    return NP == 1 ? uniform_ptr(at) : at;
  };
  u32x4 kw[CH], vw[CH];
  const bool stages = 4 * D >= THREADS || tid < 4 * D;
  auto load_k = [&](const Pages& P, int tile) {
    if (!stages) return;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = tid + THREADS * c, key = at / KS, part = at % KS;
      const uint32_t mine = (key & (NP == 1 ? 63 : bs - 1)) * D + 16 * part;
      kw[c] = *(GlobalCodes)(codes(C.k, P, key >> 4, NP == 1 ? ((tile * 64) & (bs - 1)) * D : 0) + mine);
    }
  };
  auto load_v = [&](const Pages& P, int tile) {
    if (!stages) return;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = tid + THREADS * c, d = at >> 2, group = at & 3;
      const uint32_t mine = d * bs + ((16 * group) & (NP == 1 ? 63 : bs - 1));
      vw[c] = *(GlobalCodes)(codes(C.v, P, group, NP == 1 ? (tile * 64) & (bs - 1) : 0) + mine);
    }
  };
  auto store_k = [&](int at_ring) {
    if (!stages) return;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = tid + THREADS * c, key = at / KS, part = at % KS;
      f16x8 x, y;
      to_halves<CODES>(kw[c], x, y);
      uint8_t* const k = lds + at_ring * KB + key * KR + 32 * part;
      *reinterpret_cast<f16x8*>(k) = x;
      *reinterpret_cast<f16x8*>(k + 16) = y;
    }
  };
  // Codes of e4m3 past the length, or of no page, may be NaN: zeros instead.
  auto clear_v = [&](const Pages& P, int tile) {
    if (CODES != PP_KV_E4M3) return;
    bool all = (tile + 1) * 64 <= T.lim;
#pragma unroll
    for (int e = 0; e < NP; ++e) all &= P.p[e] >= 0;
    if (all) return;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int group = (tid + THREADS * c) & 3;
      int p = P.p[0];
#pragma unroll
      for (int e = 1; e < NP; ++e) p = group * NP / 4 == e ? P.p[e] : p;
      const int seen = p >= 0 ? T.lim - tile * 64 - 16 * group : 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int left = seen - 4 * w;
        vw[c][w] &= left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
      }
    }
  };
  auto store_v = [&](int at_ring) {
    if (!stages) return;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = tid + THREADS * c, d = at >> 2, group = at & 3;
      f16x8 x, y;
      to_halves<CODES>(vw[c], x, y);
      uint8_t* const v = lds + RING * KB + at_ring * VB + d * VR + 32 * group;
      *reinterpret_cast<f16x8*>(v) = x;
      *reinterpret_cast<f16x8*>(v + 16) = y;
    }
  };
  struct Scales {
    float k[NP], v[NP];
    int ok;
  };
  auto scales = [&](const Pages& P) {
    Scales X;
    X.ok = 0;
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      const int64_t ph = (int64_t)(P.p[e] < 0 ? 0 : P.p[e]) * C.heads + h;
      X.k[e] = scalar_load(C.ks + ph);
      X.v[e] = scalar_load(C.vs + ph);
      X.ok |= (P.p[e] >= 0 ? (1 << (4 / NP)) - 1 : 0) << (4 / NP * e);
    }
    return X;
  };

  const int mk = (m32 & 0x13) | (m32 & 4) << 1 | (m32 & 8) >> 1;       // key of row m32: bits 2 and 3 swapped
  const uint8_t* const kl = lds + mk * KR + 16 * hh;
  const uint8_t* const vl = lds + RING * KB + m32 * VR + 16 * hh;
  f32x16 s[2];
  f16x8 p[4];

  // One step of a wavefront: the weights of tile i, a barrier, the products (the weighted values of
  // tile i and the scores of tile i + 1) and beside them the staging of later tiles, a barrier.  With 8 wavefronts
  // the second four, which share the SIMDs with the first, run one barrier behind, so that one
  // wavefront of a SIMD has the matrix cores, and the priority, while the other has the vector unit.  Operands are read
  // from LDS a group of products ahead, and no further: all at once they would not leave
  // registers for the sums.
  f16x8 va[2][DT], ka[2][4];
  auto read_v = [&](auto buf, const uint8_t* v, int g) {
#pragma unroll
    for (int d = 0; d < DT; ++d) va[decltype(buf)::value][d] = *reinterpret_cast<const f16x8*>(v + 32 * d * VR + 32 * g);
  };
  auto read_k = [&](auto buf, const uint8_t* k, int c) {      // chunks c and c + 1
#pragma unroll
    for (int e = 0; e < 4; ++e)
      ka[decltype(buf)::value][e] = *reinterpret_cast<const f16x8*>(k + 32 * (e & 1) * KR + 32 * (c + (e >> 1)));
  };
  auto score = [&](auto buf, int c) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s[e & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[decltype(buf)::value][e], q[c + (e >> 1)],
                                                        c + (e >> 1) == 0 ? f32x16{} : s[e & 1], 0, 0, 0);
  };
  auto scores = [&](const uint8_t* k) {                       // the first group is read
#pragma unroll
    for (int c = 0; c < KS; c += 4) {
      read_k(Int<1>(), k, c + 2);
      score(Int<0>(), c);
      __builtin_amdgcn_sched_barrier(0);
      if (c + 4 < KS) read_k(Int<0>(), k, c + 4);
      score(Int<1>(), c + 2);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto value = [&](auto buf, int g) {
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[decltype(buf)::value][d], p[g], o[d], 0, 0, 0);
  };
  // What a tile's scales make of its scores and sums, with the reference as it is.
  float lv[NP], iv[NP], kq[NP], from = 0.f;
  bool vbad = false;
  auto weigh = [&](const Scales& X) {
    from = ref == KV_NONE ? 0.f : ref;
    vbad = false;
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      const bool bad = mag(X.v[e]) >= 0x7f800000u;
      vbad |= bad;
      const float vq = bad ? 1.f : fmaxf(X.v[e], KV_SCALE_MIN);
      lv[e] = __builtin_amdgcn_logf(vq) - from;
      iv[e] = __builtin_amdgcn_rcpf(vq);
      kq[e] = X.k[e] * rf;
    }
  };
  if (a < z) {
    Pages p1 = pages(a), p2 = pages(a + 1), p3;
    load_k(p1, a);
    load_v(p1, a);
    Scales sc = scales(p1);
    store_k(0);
    clear_v(p1, a);
    store_v(0);
    load_k(p2, min(a + 1, z - 1));
    store_k(1);
    p3 = pages(a + 2);
    load_k(p3, min(a + 2, z - 1));
    load_v(p2, min(a + 1, z - 1));
    __syncthreads();
    read_k(Int<0>(), kl, 0);
    scores(kl);
    weigh(sc);
    // The rings: beside the weights of tile i, V of tile i + 1 and K of tile i + 2 are written over what the products of
    // an earlier step read last, with a barrier between them.  K of the first tile is read just above instead, and
    // with two slots the first tile's weights already write over it: so a barrier here.  With three slots the
    // second tile's do; there the barrier is the one by which the second four run behind.
    if (!PING || wave >= WAVES / 2) phase();
    int r0 = 0;                                               // ring of V of tile i, and of K
    for (int i = a; i < z; ++i) {
      const int t0 = i * 64, r1 = r0 + 1 == RING ? 0 : r0 + 1, r2 = r1 + 1 == RING ? 0 : r1 + 1;
      float sum[4];
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          s[g / 2][8 * (g & 1) + k] = s[g / 2][8 * (g & 1) + k] * kq[g * NP / 4] + lv[g * NP / 4];
      const int k0 = lo - t0 - 8 * hh, k1 = hi - t0 - 8 * hh;   // the row's keys, 16 g + k of them this lane's
      if ((sc.ok != 15) | (t0 < all_lo) | (t0 + 64 > all_hi)) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int a0 = sc.ok >> g & 1 ? k0 : 64;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int at = 8 * (g & 1) + k;
            s[g / 2][at] = ((16 * g + k >= a0) & (16 * g + k < k1)) ? s[g / 2][at] : -INFINITY;
          }
        }
      }
      auto weights = [&]() {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          sum[g] = 0.f;
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            const int at = 8 * (g & 1) + k;
            const f32x2 w = {__builtin_amdgcn_exp2f(s[g / 2][at]), __builtin_amdgcn_exp2f(s[g / 2][at + 1])};
            sum[g] += w[0];
            sum[g] += w[1];
            const f16x2 w16 = __builtin_convertvector(w, f16x2);
            p[g][k] = w16[0];
            p[g][k + 1] = w16[1];
          }
        }
      };
      weights();
      const float most = fmaxf(fmaxf(sum[0], sum[1]), fmaxf(sum[2], sum[3]));
      if (__any((ref == KV_NONE) | (most > KV_FAR))) {       // for the rows that need it: no row sways another
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fmaxf(s[0][e], s[1][e]));
        top = max_halves(top);
        const bool need = (ref == KV_NONE) | (max_halves(most) > KV_FAR);
        const float next = need ? fmaxf(ref, top + from - KV_NEAR) : ref;
        const float f = __builtin_amdgcn_exp2f(ref - next);
        // Past 2^24 the reference is rounded so far that the largest exponent can be 16 and more, whose weight fp16
        // does not hold: it is 0 there.
        const float to = (need && top + (from - next) > 15.f) ? -top : from - next;
        l *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[0][e] += to;
          s[1][e] += to;
        }
        ref = next;
        weights();
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) l += sum[g] * iv[g * NP / 4];
      if (vbad) {                                            // the same in every lane
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const bool see = (sc.ok >> g & 1) & (16 * g + k >= k0) & (16 * g + k < k1) &
                             (mag(sc.v[g * NP / 4]) >= 0x7f800000u);
            p[g][k] = see ? (f16)NAN : p[g][k];
          }
      }
      const Pages p4 = pages(i + 3);
      clear_v(p2, i + 1);
      store_v(r1);
      store_k(r2);
      phase();
      __builtin_amdgcn_s_setprio(1);
      const uint8_t* const v = vl + r0 * VB;
      read_v(Int<0>(), v, 0);
      read_v(Int<1>(), v, 1);
      value(Int<0>(), 0);
      __builtin_amdgcn_sched_barrier(0);
      read_v(Int<0>(), v, 2);
      value(Int<1>(), 1);
      __builtin_amdgcn_sched_barrier(0);
      read_v(Int<1>(), v, 3);
      value(Int<0>(), 2);
      load_v(p3, min(i + 2, z - 1));
      __builtin_amdgcn_sched_barrier(0);
      read_k(Int<0>(), kl + r1 * KB, 0);
      value(Int<1>(), 3);
      load_k(p4, min(i + 3, z - 1));
      sc = scales(p2);
      __builtin_amdgcn_sched_barrier(0);
      scores(kl + r1 * KB);
      weigh(sc);
      p2 = p3;
      p3 = p4;
      __builtin_amdgcn_s_setprio(0);
      phase();
      r0 = r1;
    }
    if (PING && wave < WAVES / 2) phase();
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
      if (A.lse && hh == 0) A.lse[at] = kv_lse(ref, l);
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
        part[D] = ref;
        part[D + 1] = l;
      }
    }
  }
  if (runs > 1 && run == 0 && tid == 0) *desc = ManyPart{runs, T.s0, T.r0, min(R, T.rows - T.r0)};
  if (U.at >= U.end) return;
  __syncthreads();                       // the rings are read
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
  const dim3 grid((unsigned)(P.shares ? P.grid : P.grid * A.C.heads), P.shares ? (unsigned)A.C.heads : 1u);
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
