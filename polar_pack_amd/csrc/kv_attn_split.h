// Attention of a call's tokens to the cache, few rows a sequence and head.
//
// Row (token, query head) with position p = lengths[b] - n_b + i sees the keys j of
// (p - window, p] (causal) or of [0, length):
//   s_j = scale * ks * sum_d q_d kcode_jd,   o_d = sum_j e^(s_j - m) vs vcode_jd / sum_j e^(s_j - m).
#pragma once

#include "kv_attn.h"

namespace pp {

// Few rows a sequence and head (single tokens, drafts).  A workgroup takes 16 * RT rows of one
// sequence and key/value head and a run of 64-token tiles, dealt to its 4 wavefronts in turn.  Where a row
// tile has several runs, each leaves its sums in the workspace and counts itself done; the one that
// counts last reads them all in their order, writes the rows and sets the count back to zero.
//
// The codes go from memory to the matrix cores without LDS: S^T = K Q^T takes rows of K as they lie
// (16 bytes a lane), O^T = V^T P^T rows of the transposed V.  Which token is which row of a product is
// free, so S^T's rows are numbered such that the 16 scores a lane holds of a tile, tokens
// 16 g + 0..15 of lane group g = lane / 16, are the ones whose V codes its 16-byte load brings:
// row m of product t is token 16 (m / 4) + 4 t + m % 4, and P needs no exchange between lanes.
// Scales stay out of the codes: ks multiplies a lane's scores, log2 vs is added to the exponent,
// so that weights e^(s - m) vs are at most 2^14 in fp16 whatever the scales, and the sum of
// e^(s - m) takes them times 1 / vs.
//
// What bounds it: the codes' way from memory.  A copy that only loads takes as long as the kernel
// (attend_batch 131.7 against 134.9 us when that was measured).  Four sequences of 100-131 k tokens,
// 248 MB: 52 us, of which the loads stream for 36 (6.9 TB/s, what any kernel reads here), 5 until
// the first codes arrive (lengths, pages, codes: three round trips), 3 for a share's sums to be in memory and
// 5-7 for the join.  64 sequences of 77-8190 tokens, 559 MB: 100 us (5.6 TB/s): a workgroup's 2 shares
// of row tiles each fill the loads' pipeline anew.  Equal shares against one workgroup a row
// tile 100 / 124 us; one workgroup a CU with two tiles on their way against two with one 112 / 118
// (and 65 / 69 at the long sequences, whose join reads half as many parts); a turn counted as 16 tiles
// against 4 66.4 -> 63.2.  With 64 values a head a workgroup's registers leave room for a second on the CU, and
// a tile is half the bytes on its way: 24 sequences of 5 drafted tokens in a window of 2000, 34.5 -> 30.7 us with
// two.  64 sequences of 77-8190 with 4 key heads of 192: 80 us (5.2 TB/s); of 256 105 (5.3), where 48-76 bytes a lane
// spill in tiles of 16 rows and 152-200 in tiles of 32.  V with the streaming cache policy, since a load takes whole lines of it; not K,
// whose lines two loads share.
//
// In 4 bits (PP_KV_E2M1) the codes become halves on their way into the products, K's with their scale, V's times theirs (all
// exact), and no scale is left for scores or weights.  One tile on its way and two workgroups a CU: converting takes as long
// as the loads, and a SIMD issues an instruction of one wavefront every 8 clocks, of two every 4 to 5.  64 sequences of
// 77-8190 tokens and 8 key heads (297 MB) 64 us, 4.6 TB/s, with one workgroup of two tiles a CU 73; loads alone take
// 62.  4 sequences of 200-262 k and 2 (263 MB) 57 us: there two workgroups a CU would leave twice the parts to join (61).
// Wider heads, in turn with 8 bits, us: 64 of 77-8190 with 4 key heads of 192 60 / 88 (3.8 TB/s), of 256 72 / 117 (4.3); 4 of 100-131 k
// with 2 of 192 50 / 76, of 256 59 / 100 (4.3).  In tiles of 32 rows the registers are full: 24 sequences of 500-8000 and 5 drafted
// tokens with 8 key heads of 128 54 / 61, 4 of 192 49 / 52, 4 of 256 84 / 76, where 208-212 bytes a lane spill; elsewhere nothing does.
// The scaled products that take 4-bit codes as they are were no way: against queries split over three e4m3 terms they are off
// by 2^-15 of the sum of magnitudes, where float32 sums are by 2^-24.
template <int CODES, typename IO, int D, int RT, int NP>
__global__ __launch_bounds__(256, D == 64 || (CODES == PP_KV_E2M1 && D * RT == 128) ? 2 : 1) void kv_attn_split_kernel(const AttnArgs A) {
  constexpr bool FOUR = CODES == PP_KV_E2M1;
  constexpr int DT = D / 16, R = 16 * RT, BUF = !FOUR && D * RT <= 256 ? 2 : 1;
  constexpr int EL = FOUR && D % 128 == 0 ? 32 : 16, J = D / (4 * EL), PIECES = EL / 8;   // codes a load of K, loads a row
  typedef std::conditional_t<FOUR && EL == 16, u32x2, u32x4> KWords;
  typedef std::conditional_t<FOUR, u32x2, u32x4> VWords;
  const KvCache& C = A.C;
  const KvSeqs& S = A.S;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), m16 = lane & 15, g = lane >> 4;
  const int h = blockIdx.y;
  RowTile T;
  Deal U;
  if (A.shares) {
    if (!kv_deal<256>(A, R, T, U)) return;
  } else {
    if (!kv_row_tile(A, blockIdx.x, R, T)) return;
    U = Deal{0, 1, 1, T.lo >> 6, 1, 0};
  }
  const int shift = C.shift, bs = C.block;
  for (;; kv_deal_next(A, R, T, U)) {
  int a = T.lo >> 6, z = T.hi > T.lo ? (T.hi + 63) >> 6 : 0, run = 0, runs = 1, owner = 0;
  if (A.shares) {
    const int64_t begin = U.at - U.into + KV_TURN;             // of its tiles that hold keys
    const int left = U.tiles + KV_TURN - U.into;
    const int take = U.end - U.at < left ? (int)(U.end - U.at) : left;
    const int t0 = max(U.into - KV_TURN, 0), t1 = U.into + take - KV_TURN;
    U.at += take;
    if (t1 <= 0) return;                                       // the share ends before them
    owner = (int)quotient(begin, U.share);
    runs = (int)quotient(begin + U.tiles - 1, U.share) - owner + 1;
    run = blockIdx.x - owner;
    kv_tile_range(A, R, T);
    a = max(U.first + t0, T.lo >> 6);
    z = min(U.first + t1, T.hi > T.lo ? (T.hi + 63) >> 6 : 0);
  } else {
    U.at = U.end;
  }

  f32x4 o[RT][DT];
  float mx[RT], l[RT];
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    mx[x] = -INFINITY;
    l[x] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[x][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Tiles of this wavefront: a + wave, a + wave + 4, ...; lane e holds the table's entry e % NP of
  // tile e / NP of the next 64 / NP tiles.
  const int32_t* table = S.table + (int64_t)T.b * S.ld;
  int ids = 0;
  const int km = NP == 1 ? 0 : (16 * (m16 >> 2)) >> shift, vm = NP == 1 ? 0 : (16 * g) >> shift;   // page of the tile
  auto page_of = [&](int step, int which) {
    int p = lane_read(ids, (step % (64 / NP)) * NP);
#pragma unroll
    for (int e = 1; e < NP; ++e) {
      const int pe = lane_read(ids, (step % (64 / NP)) * NP + e);
      p = which == e ? pe : p;
    }
    return p;
  };
  // BUF tiles are on their way while one is worked on, each in registers of its own.  The loads of a
  // tile past the last are made all the same, every lane's from the cache's first bytes: a branch
  // around them would make the compiler wait for all loads at its end.
  KWords kc[BUF][4][J];
  VWords vc[BUF][DT];
  float ks[BUF], vs[BUF];
  // 4 bits: the scales.  Every lane loads one word, not the bytes and words that it wants: with 32 codes a load of K those of a
  // token's groups, which then change places with the lanes of the same row; of V those of four tokens and a group, which the
  // lane's 16 neighbours then read from it.  6 loads a tile less (64 sequences of 77-8190 tokens 75.2 -> 73.2 us).
  constexpr int KL = EL == 32 ? J : 4 * J, VL = (D / 32 * 4 + 15) / 16;
  uint32_t k4[BUF][KL], v4[BUF][VL];
  int ok[BUF];
  int64_t vat[BUF];
  auto load_k = [&](auto buf, int tile, int step) {
    constexpr int I = decltype(buf)::value;
    const bool there = tile < z;
    if (there && step % (64 / NP) == 0) {
      const int64_t at = (((int64_t)tile + 4 * (lane / NP)) * 64 >> shift) + lane % NP;
      ids = at < S.width ? table[at] : -1;
      ids = ids < C.pages ? ids : -1;
    }
    const int pk = page_of(step, km), pv = page_of(step, vm);
    const int64_t hk = (int64_t)((there & (pk >= 0)) ? pk : 0) * C.heads + (there ? h : 0);
    const int tok = (tile * 64 + 16 * (m16 >> 2)) & (bs - 1);
    if constexpr (FOUR) {
      const int64_t ph = (int64_t)((there & (pv >= 0)) ? pv : 0) * C.heads + (there ? h : 0);
      ok[I] = pv >= 0;
      const int64_t row = hk * bs + (there ? tok + (m16 & 3) : 0);
      const uint8_t* at = C.k + row * (D / 2) + EL / 2 * g;
      const uint8_t* sat = scales_k(C) + row * (D / 32) + (EL == 32 ? 4 * g * (D / 32) : EL * g / 32);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < J; ++j) {
          kc[I][t][j] = *reinterpret_cast<const KWords*>(at + 4 * t * (D / 2) + 2 * EL * j);
          if constexpr (EL == 16) k4[I][4 * j + t] = sat[4 * t * (D / 32) + EL / 8 * j];
        }
      if constexpr (EL == 32) {
#pragma unroll
        for (int j = 0; j < J; ++j) k4[I][j] = *reinterpret_cast<const uint32_t*>(sat + 4 * j);      // of token t = g
      }
      vat[I] = ph * (bs * D) + (there ? (tile * 64 + 16 * g) & (bs - 1) : 0);      // as codes of a byte
      return;
    }
    const uint8_t* at = C.k + hk * (bs * D) + (there ? (tok + (m16 & 3)) * D + 16 * g : 0);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < J; ++j) kc[I][t][j] = *reinterpret_cast<const KWords*>(at + 4 * t * D + 64 * j);
    ok[I] = pv >= 0;
    const int64_t ph = (int64_t)((there & (pv >= 0)) ? pv : 0) * C.heads + (there ? h : 0);
    ks[I] = C.ks[ph];
    vs[I] = C.vs[ph];
    vat[I] = ph * (bs * D) + (there ? ((tile * 64 + 16 * g) & (bs - 1)) + m16 * bs : 0);
  };
  auto load_v = [&](auto buf) {
    constexpr int I = decltype(buf)::value;
    if constexpr (FOUR) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
        vc[I][d] = __builtin_nontemporal_load(reinterpret_cast<const VWords*>(C.v + (vat[I] >> 1) + (16 * d + m16) * (bs / 2)));
      const int64_t page = vat[I] & ~(int64_t)(bs - 1);        // page and head * bs * D
      const uint8_t* at = scales_v(C) + (page >> 5) + (vat[I] - page);
#pragma unroll
      for (int i = 0; i < VL; ++i)
        v4[I][i] = *reinterpret_cast<const uint32_t*>(at + min(4 * i + (m16 >> 2), D / 32 - 1) * bs + 4 * (m16 & 3));
      return;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
      vc[I][d] = __builtin_nontemporal_load(reinterpret_cast<const VWords*>(C.v + vat[I] + d * 16 * bs));
  };

  // This lane's rows: column m16 of row tile x.
  int tile = a + wave, step = 0;
  u32x4 qw[RT][D / 32];
  int lo[RT], hi[RT];
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int r = T.r0 + 16 * x + m16;
    const bool real = r < T.rows;
    const int i = real ? r / A.group : 0, gq = real ? r - i * A.group : 0;
    kv_visible(A, T, i, real, lo[x], hi[x]);
    load_q<D, EL>(A, T.s0 + i, h * A.group + gq, g, real, qw[x]);
  }
  load_k(Int<0>(), tile, 0);
  load_v(Int<0>());
  if constexpr (BUF == 2) {
    load_k(Int<BUF - 1>(), tile + 4, 1);
    load_v(Int<BUF - 1>());
  }
  f16x8 q[RT][D / 32];
  float rf[RT];
#pragma unroll
  for (int x = 0; x < RT; ++x) rf[x] = make_q<IO, D>(A, qw[x], q[x]);

  auto work = [&](auto buf) {
    constexpr int I = decltype(buf)::value;
    f32x4 s[RT][4];
    if constexpr (FOUR && EL == 32) {
#pragma unroll
      for (int j = 0; j < J; ++j) k4[I][j] = turn_bytes(k4[I][j], g);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int x = 0; x < RT; ++x) s[x][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if constexpr (FOUR) {
          const float ks4 = EL == 16 ? __builtin_amdgcn_cvt_f32_bf8(k4[I][EL == 16 ? 4 * j + t : 0], 0) : bf8_byte(k4[I][j], t);
#pragma unroll
          for (int w = 0; w < PIECES; ++w) {
            const f16x8 ka = halves4(kc[I][t][j][w], ks4);
#pragma unroll
            for (int x = 0; x < RT; ++x)
              s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q[x][PIECES * j + w], s[x][t], 0, 0, 0);
          }
        } else {
          f16x8 ka, kb;
          to_halves<CODES>(kc[I][t][j], ka, kb);
#pragma unroll
          for (int x = 0; x < RT; ++x) {
            s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q[x][2 * j], s[x][t], 0, 0, 0);
            s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, q[x][2 * j + 1], s[x][t], 0, 0, 0);
          }
        }
      }
    }
    const bool okv = ok[I];
    // scores to weights
    bool vbad = false;
    float lv = 0.f, iv = 1.f, kscale = 1.f;                      // 4 bits: scales are in the operands
    if constexpr (!FOUR) {
      vbad = mag(vs[I]) >= 0x7f800000u;                          // the values are NaN, the sum of weights is not
      const float vq = vbad ? 1.f : fmaxf(vs[I], KV_SCALE_MIN);
      lv = __builtin_amdgcn_logf(vq), iv = 1.0f / vq, kscale = ks[I];
    }
    load_k(buf, tile + 4 * BUF, step + BUF);
    const int t0 = tile * 64 + 16 * g;
    f16x8 p[RT][2];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      const float c = kscale * rf[x];
      const bool edge = __any(!okv | (t0 < lo[x]) | (t0 + 16 > hi[x]));
      float e[16], top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) e[4 * t + r] = FOUR ? s[x][t][r] * c : s[x][t][r] * c + lv;
      if (edge) {
        const int from = okv ? lo[x] - t0 : 16, to = hi[x] - t0;
#pragma unroll
        for (int k = 0; k < 16; ++k) e[k] = ((k >= from) & (k < to)) ? e[k] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) top = fmaxf(top, e[k]);
      top = max_groups(top);
      const float next = kv_ref(top);
      if (__any(next > mx[x])) {
        const float mn = fmaxf(mx[x], next);
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx[x] - mn);
        mx[x] = mn;
        l[x] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[x][d] *= f;
      }
      const float ref = mx[x] == -INFINITY ? 0.f : mx[x];
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        e[k] = __builtin_amdgcn_exp2f(e[k] - ref);
        sum += e[k];
        p[x][k / 8][k % 8] = (f16)e[k];
      }
      l[x] += sum * iv;
      if (!FOUR && __any(vbad)) {
        const int from = (okv & vbad) ? lo[x] - t0 : 16, to = hi[x] - t0;
#pragma unroll
        for (int k = 0; k < 16; ++k) p[x][k / 8][k % 8] = ((k >= from) & (k < to)) ? (f16)NAN : p[x][k / 8][k % 8];
      }
    }
    if (CODES != PP_KV_INT8) {                   // past the length codes may be NaN, and scales of 4 bits
      const int seen = okv ? T.lim - t0 : 0;
      if (__any(seen < 16)) {
        if constexpr (FOUR) {
          const uint32_t keep = keep_bytes(seen - 4 * (m16 & 3));
#pragma unroll
          for (int i = 0; i < VL; ++i) v4[I][i] &= keep;
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t keep = keep_bytes(seen - 4 * w);
#pragma unroll
            for (int d = 0; d < DT; ++d) vc[I][d][w] &= keep;
          }
        }
      }
    }
    if constexpr (FOUR) {
      f16x8 sa, sb;                              // of the tokens' scales
      each<DT>([&](auto dt) {
        constexpr int d = decltype(dt)::value;
        if constexpr (d % 2 == 0) {
          constexpr int at = 2 * d % 16;
          const uint32_t w = v4[I][d / 8];
          sa = scales4(row_bcast<at>(w), row_bcast<at + 1>(w));
          sb = scales4(row_bcast<at + 2>(w), row_bcast<at + 3>(w));
        }
        const f16x8 va = halves4(vc[I][d][0], 1.f) * sa, vb = halves4(vc[I][d][1], 1.f) * sb;
#pragma unroll
        for (int x = 0; x < RT; ++x) {
          o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[x][0], o[x][d], 0, 0, 0);
          o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb, p[x][1], o[x][d], 0, 0, 0);
        }
      });
    } else {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        f16x8 va, vb;
        to_halves<CODES>(vc[I][d], va, vb);
#pragma unroll
        for (int x = 0; x < RT; ++x) {
          o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[x][0], o[x][d], 0, 0, 0);
          o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb, p[x][1], o[x][d], 0, 0, 0);
        }
      }
    }
    load_v(buf);
    tile += 4;
    ++step;
  };
  while (tile < z) {
    work(Int<0>());
    if constexpr (BUF == 2) {
      if (tile >= z) break;
      work(Int<BUF - 1>());
    }
  }

  // The 4 wavefronts' sums meet in LDS; a thread then holds D / 16 neighbouring values of a row (of
  // RT rows), of the run or, where the tile has several and this one is the last to end, of all.
  constexpr int W = D / 16;
  __shared__ float so[4][R][D + 4];
  __shared__ float sm[4][R], sl[4][R];
  __shared__ uint32_t done;
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int r = 16 * x + m16;
    l[x] = sum_groups(l[x]);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&so[wave][r][16 * d + 4 * g]) = o[x][d];
    if (g == 0) { sm[wave][r] = mx[x]; sl[wave][r] = l[x]; }
  }
  __syncthreads();
  float v[RT][W], m[RT], sum[RT];
  const int d0 = (threadIdx.x & 15) * W;
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int r = 16 * x + (threadIdx.x >> 4);
    m[x] = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
    sum[x] = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) v[x][k] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = sm[w][r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sm[w][r] - m[x]);   // 0 * 1: nothing seen
      sum[x] += sl[w][r] * f;
#pragma unroll
      for (int k = 0; k < W; ++k) v[x][k] += so[w][r][d0 + k] * f;
    }
  }
  bool last = true;
  if (runs > 1) {
    // A run's sums go to memory past the caches that other XCDs do not see (agent-scope stores) and
    // are waited for before the tile's count goes up; the last run reads them all, in order, so that
    // the result does not depend on which one is last.
    // workgroup owner + i has part i; the owner's is its second
    float* const part = A.parts + ((int64_t)h * A.shares + owner) * (2 * R) * (D + 4);
    auto place = [&](int i) { return part + (int64_t)(i == 0 ? 1 : 2 * i) * R * (D + 4); };
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      const int r = 16 * x + (threadIdx.x >> 4);
      if (T.r0 + r >= T.rows) continue;
      float* p = place(run) + r * (D + 4);
#pragma unroll
      for (int k = 0; k < W; ++k) __hip_atomic_store(p + d0 + k, v[x][k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (d0 == 0) {
        __hip_atomic_store(p + D, m[x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(p + D + 1, sum[x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint32_t* const count = A.counts + (int64_t)h * A.shares + owner;
    if (threadIdx.x == 0) done = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    last = done == (uint32_t)(runs - 1);
    if (last) {
    if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    // 16 threads a row and share of the runs: with few rows in the tile several shares a row
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      const int left = T.rows - T.r0 - 16 * x;
      const int bits = left >= 9 ? 4 : left >= 5 ? 3 : left >= 3 ? 2 : left == 2 ? 1 : 0;
      const int team = threadIdx.x >> 4, row = team & ((1 << bits) - 1), shares = 16 >> bits;
      m[x] = -INFINITY;
      sum[x] = 0.f;
#pragma unroll
      for (int k = 0; k < W; ++k) v[x][k] = 0.f;
      if (row < left) {
        constexpr int AHEAD = W <= 8 ? 8 : 4;
        for (int i0 = team >> bits; i0 < runs; i0 += AHEAD * shares) {
          f32x4 w[AHEAD][W / 4];
          f32x2 ml[AHEAD];
#pragma unroll
          for (int u = 0; u < AHEAD; ++u) {
            const int i = min(i0 + u * shares, runs - 1);
            const float* e = place(i) + (16 * x + row) * (D + 4);
            ml[u] = *reinterpret_cast<const f32x2*>(e + D);
#pragma unroll
            for (int k = 0; k < W / 4; ++k) w[u][k] = *reinterpret_cast<const f32x4*>(e + d0 + 4 * k);
          }
#pragma unroll
          for (int u = 0; u < AHEAD; ++u)
            if (i0 + u * shares < runs)
              join_part<W>(m[x], sum[x], v[x], ml[u][0], ml[u][1], reinterpret_cast<const float*>(&w[u][0]));
        }
      }
      __syncthreads();
      float* mine = &so[0][team][0];
#pragma unroll
      for (int k = 0; k < W; ++k) mine[d0 + k] = v[x][k];
      if (d0 == 0) { sm[0][team] = m[x]; sl[0][team] = sum[x]; }
      __syncthreads();
      for (int t = 1; t < shares; ++t) {
        const int other = (row | t << bits) & 15;
        if (team < 1 << bits) join_part<W>(m[x], sum[x], v[x], sm[0][other], sl[0][other], &so[0][other][d0]);
      }
    }
    }
  }
  if (last) {
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int r = T.r0 + 16 * x + (threadIdx.x >> 4);
    if (r >= T.rows) continue;
    const int i = r / A.group;
    const int64_t at = (int64_t)(T.s0 + i) * A.q_heads + h * A.group + (r - i * A.group);
    const float inv = kv_inverse(sum[x]);
#pragma unroll
    for (int k = 0; k < W; k += 4)
      store4<IO>(A.out + at * D + d0 + k, f32x4{v[x][k] * inv, v[x][k + 1] * inv, v[x][k + 2] * inv, v[x][k + 3] * inv});
    if (A.lse && d0 == 0) A.lse[at] = kv_lse(m[x], sum[x]);
  }
  }
  if (U.at >= U.end) return;
  __syncthreads();                       // the sums in LDS are read
  }
}

template <int CODES, typename IO, int D>
int attn_launch(const AttnArgs& A, const AttnPlan& P, hipStream_t st) {
  const dim3 grid((unsigned)P.grid, (unsigned)A.C.heads);
  auto pick = [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    auto kern = A.C.block >= 64 ? kv_attn_split_kernel<CODES, IO, D, RT, 1>
                : A.C.block == 32 ? kv_attn_split_kernel<CODES, IO, D, RT, 2> : kv_attn_split_kernel<CODES, IO, D, RT, 4>;
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, A);
  };
  if (P.rows == 16) pick(std::integral_constant<int, 1>());
  else pick(std::integral_constant<int, 2>());
  PP_LAUNCH_CHECK();
  return PP_OK;
}

template <int CODES, typename IO>
int attn_width(const AttnArgs& A, const AttnPlan& P, int D, hipStream_t st) {
  switch (D) {
    case 64: return attn_launch<CODES, IO, 64>(A, P, st);
    case 128: return attn_launch<CODES, IO, 128>(A, P, st);
    case 192: return attn_launch<CODES, IO, 192>(A, P, st);
    default: return attn_launch<CODES, IO, 256>(A, P, st);
  }
}

}  // namespace pp
