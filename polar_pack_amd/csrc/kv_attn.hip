// Attention of a call's tokens to the 8-bit cache.
//
// Row (token, query head) with position p = lengths[b] - n_b + i sees the keys j of
// (p - window, p] (causal) or of [0, length):
//   s_j = scale * ks * sum_d q_d kcode_jd,   o_d = sum_j e^(s_j - m) vs vcode_jd / sum_j e^(s_j - m).
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
template <int I>
using Int = std::integral_constant<int, I>;

template <int CODES, typename IO, int D, int RT, int NP>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void kv_attn_split_kernel(const AttnArgs A) {
  constexpr int J = D / 64, DT = D / 16, R = 16 * RT, BUF = D * RT <= 256 ? 2 : 1;
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
    owner = (int)(begin / U.share);
    runs = (int)((begin + U.tiles - 1) / U.share) - owner + 1;
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
  u32x4 kc[BUF][4][J], vc[BUF][DT];
  float ks[BUF], vs[BUF];
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
    const uint8_t* at = C.k + hk * (bs * D) + (there ? (tok + (m16 & 3)) * D + 16 * g : 0);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < J; ++j) kc[I][t][j] = *reinterpret_cast<const u32x4*>(at + 4 * t * D + 64 * j);
    ok[I] = pv >= 0;
    const int64_t ph = (int64_t)((there & (pv >= 0)) ? pv : 0) * C.heads + (there ? h : 0);
    ks[I] = C.ks[ph];
    vs[I] = C.vs[ph];
    vat[I] = ph * (bs * D) + (there ? ((tile * 64 + 16 * g) & (bs - 1)) + m16 * bs : 0);
  };
  auto load_v = [&](auto buf) {
    constexpr int I = decltype(buf)::value;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      vc[I][d] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(C.v + vat[I] + d * 16 * bs));
  };

  // This lane's rows: column m16 of row tile x.
  int tile = a + wave, step = 0;
  u32x4 qw[RT][J][2];
  int lo[RT], hi[RT];
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int r = T.r0 + 16 * x + m16;
    const bool real = r < T.rows;
    const int i = real ? r / A.group : 0, gq = real ? r - i * A.group : 0;
    kv_visible(A, T, i, real, lo[x], hi[x]);
    load_q<D>(A, T.s0 + i, h * A.group + gq, g, real, qw[x]);
  }
  load_k(Int<0>(), tile, 0);
  load_v(Int<0>());
  if constexpr (BUF == 2) {
    load_k(Int<BUF - 1>(), tile + 4, 1);
    load_v(Int<BUF - 1>());
  }
  f16x8 q[RT][J][2];
  float rf[RT];
#pragma unroll
  for (int x = 0; x < RT; ++x) rf[x] = make_q<IO, D>(A, qw[x], q[x]);

  auto work = [&](auto buf) {
    constexpr int I = decltype(buf)::value;
    f32x4 s[RT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int x = 0; x < RT; ++x) s[x][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        f16x8 ka, kb;
        to_halves<CODES>(kc[I][t][j], ka, kb);
#pragma unroll
        for (int x = 0; x < RT; ++x) {
          s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q[x][j][0], s[x][t], 0, 0, 0);
          s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, q[x][j][1], s[x][t], 0, 0, 0);
        }
      }
    }
    const bool okv = ok[I];
    // scores to weights
    const bool vbad = mag(vs[I]) >= 0x7f800000u;                 // the values are NaN, the sum of weights is not
    const float vq = vbad ? 1.f : fmaxf(vs[I], KV_SCALE_MIN);
    const float lv = __builtin_amdgcn_logf(vq), iv = 1.0f / vq, kscale = ks[I];
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
        for (int r = 0; r < 4; ++r) e[4 * t + r] = s[x][t][r] * c + lv;
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
      if (__any(vbad)) {
        const int from = (okv & vbad) ? lo[x] - t0 : 16, to = hi[x] - t0;
#pragma unroll
        for (int k = 0; k < 16; ++k) p[x][k / 8][k % 8] = ((k >= from) & (k < to)) ? (f16)NAN : p[x][k / 8][k % 8];
      }
    }
    if (CODES == PP_KV_E4M3) {                   // codes past the length may be NaN
      const int seen = okv ? T.lim - t0 : 0;
      if (__any(seen < 16)) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int left = seen - 4 * w;
          const uint32_t keep = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
#pragma unroll
          for (int d = 0; d < DT; ++d) vc[I][d][w] &= keep;
        }
      }
    }
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

// The row tile by the mean rows of a sequence and head (tokens x query heads a key head), in us on both sides,
// sequences of int8 codes of 16 query and 2 key heads of 128 unless said:
// * 16 or 32 rows at 24: 4 sequences of 4000 tokens 17.6 / 24.4, 64 of 8000 90 / 65.  From 17 rows on 32, which a
//   large batch reads its codes once for.
// * 32 rows or the many-row kernel's 128: at 48 rows 4 of 40,000 50 / 67, 64 of 2000 31 / 65, 200 of 1000 76 / 87; at
//   64, 4 of 4000 26.6 / 26.6, 64 of 8000 107 / 158 (8 query and key heads, e4m3, 64 of up to 500: 55 / 50); at 128,
//   75 / 72, 57 / 70 and 183 / 167.  To 64 rows 32.  At 256 values a head the two are even sooner: at 48, 4 of 4000 45 / 37,
//   64 of 2000 58 / 101, 24 of 4000 74 / 75; to 32 rows there.
// * 128 rows or 256, which 8 wavefronts share, at 128: 72 / 70, 167 / 152 (64 values a head, 8 key heads: 24 of 4000
//   100 / 105, 64 of 8000 469 / 409); 256 from 129 on, and never for more than 128 values, whose sums fill the registers.
// A batch of prompts and single tokens takes what its mean asks for: a prompt of 2000 and 60 single tokens of
// 1000-8000 125 (152 in tiles of 32), of 500 105 (57 in tiles of 32).
//
// Shares for a workgroup a CU, two of few rows with 64 values a head (kv_attn_split_kernel): one / two at 16 rows, 24
// sequences in a window of 2000 26 / 23, 64 of up to 8190 63 / 56, 4 of 40,000 36 / 37; at 32 rows 32 / 29, 83 / 68,
// 50 / 48; alike with e4m3 and pages of 16.  None for batches that one workgroup cannot count, and none for
// prompts of two row tiles a CU and more.  Cut / whole, 4 prompts: 256 row tiles 53 / 50, 384 117 / 68, 512 144 / 99,
// 1024 503 / 333; behind 4000 tokens each 128 115 / 144, 256 193 / 172, 320 246 / 288, 384 301 / 308, 448 363 / 328.
// What lies behind a prompt only the device knows; whole tiles never lose from 448 on.
static AttnPlan attn_plan(int64_t heads, int64_t D, int64_t block, int64_t width, int64_t batch, int64_t tokens,
                          int64_t q_heads) {
  const int64_t group = q_heads / heads, rows = (tokens * group + batch - 1) / batch, cus = device_cu_count();
  AttnPlan P;
  P.rows = rows <= 16 ? 16 : rows <= (D <= 192 ? 64 : 32) ? 32 : rows <= 128 || D > 128 ? 128 : 256;
  const int64_t row_tiles = tokens * group / P.rows + batch + 1;
  P.shares = ((P.rows <= 32 && D == 64 ? 2 : 1) * cus + heads - 1) / heads;
  const int64_t most = row_tiles * ((width * block + 255) / 256 + 1);       // of 4 tiles each
  if (P.shares > most) P.shares = most;
  if (batch > KV_DEAL_BATCH || (P.rows > 32 && tokens * q_heads / P.rows >= 2 * cus)) P.shares = 0;
  P.grid = P.shares ? P.shares : row_tiles;
  P.bytes = heads * P.shares * (2 * P.rows * (D + 4) * 4 + (int64_t)sizeof(ManyPart));
  P.counts = P.rows <= 32 ? heads * P.shares * 4 : 0;
  return P;
}

template <int CODES, typename IO, int D>
static int attn_launch(const AttnArgs& A, const AttnPlan& P, hipStream_t st) {
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
static int attn_width(const AttnArgs& A, const AttnPlan& P, int D, hipStream_t st) {
  switch (D) {
    case 64: return attn_launch<CODES, IO, 64>(A, P, st);
    case 128: return attn_launch<CODES, IO, 128>(A, P, st);
    case 192: return attn_launch<CODES, IO, 192>(A, P, st);
    default: return attn_launch<CODES, IO, 256>(A, P, st);
  }
}

}  // namespace pp

using namespace pp;

static bool attn_sizes(int64_t heads, int64_t D, int64_t block, int64_t width, int64_t batch, int64_t tokens,
                       int64_t q_heads, AttnPlan* P) {
  if (heads <= 0 || D <= 0 || block <= 0 || width <= 0 || batch <= 0 || tokens <= 0 || q_heads < heads) return false;
  *P = attn_plan(heads, D, block, width, batch, tokens, q_heads);
  return true;
}

extern "C" int64_t pp_kv_attention_workspace_size(int64_t heads, int64_t head_dim, int64_t block, int64_t table_width,
                                                  int64_t batch, int64_t tokens, int64_t q_heads) {
  AttnPlan P;
  return attn_sizes(heads, head_dim, block, table_width, batch, tokens, q_heads, &P) ? P.bytes : 0;
}

extern "C" int64_t pp_kv_attention_counts_size(int64_t heads, int64_t head_dim, int64_t block, int64_t table_width,
                                               int64_t batch, int64_t tokens, int64_t q_heads) {
  AttnPlan P;
  return attn_sizes(heads, head_dim, block, table_width, batch, tokens, q_heads, &P) ? P.counts : 0;
}

extern "C" int pp_kv_attention(const pp_kv_cache* cache, const void* q, int64_t q_st, int64_t q_sh, int64_t q_heads,
                               int dtype, int64_t tokens, const int32_t* table, int64_t table_ld, int64_t table_width,
                               const int32_t* lengths, const int32_t* cu, int64_t batch, int causal, int64_t window,
                               float scale, void* out, float* lse, void* workspace, int64_t workspace_size,
                               void* counts, int64_t counts_size, void* stream) {
  AttnArgs A;
  int rc = kv_check_cache(cache, &A.C);
  if (rc) return rc;
  rc = kv_check_seqs(A.C, table, table_ld, table_width, lengths, cu, batch, tokens, &A.S);
  if (rc) return rc;
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16, "pp_kv_attention: dtype %d is not PP_F16 or PP_BF16", dtype);
  PP_REQUIRE(q_heads > 0 && q_heads % A.C.heads == 0 && q_heads <= 65535,
             "pp_kv_attention: %lld query heads over %d heads", (long long)q_heads, A.C.heads);
  PP_REQUIRE(tokens * q_heads <= INT32_MAX, "pp_kv_attention: too many rows");
  PP_REQUIRE(window >= 0 && (causal || window == 0), "pp_kv_attention: a window needs causal attention");
  if (tokens == 0) return PP_OK;
  PP_REQUIRE(q && out, "pp_kv_attention: null queries or output");
  PP_REQUIRE(aligned(q, 2) && aligned(out, 16), "pp_kv_attention: queries or output are not aligned");
  const AttnPlan P = attn_plan(A.C.heads, cache->head_dim, A.C.block, table_width, batch, tokens, q_heads);
  PP_REQUIRE(P.bytes == 0 || (workspace && workspace_size >= P.bytes && aligned(workspace, 16)),
             "pp_kv_attention: workspace of %lld bytes at a 16-byte boundary needed", (long long)P.bytes);
  PP_REQUIRE(P.counts == 0 || (counts && counts_size >= P.counts && aligned(counts, 4)),
             "pp_kv_attention: %lld bytes of counts, zero, needed", (long long)P.counts);
  A.q = (const uint16_t*)q;
  A.q_st = q_st; A.q_sh = q_sh;
  A.q_vec = aligned(q, 16) && q_st % 8 == 0 && q_sh % 8 == 0;
  A.out = (uint16_t*)out;
  A.lse = lse;
  A.parts = (float*)workspace;
  A.q_heads = (int)q_heads;
  A.group = (int)q_heads / A.C.heads;
  A.window = (int)(window < INT32_MAX ? window : 0);
  A.causal = causal;
  A.shares = (int)P.shares;
  A.desc = P.shares ? (ManyPart*)(A.parts + A.C.heads * P.shares * 2 * P.rows * (cache->head_dim + 4)) : nullptr;
  A.counts = (uint32_t*)counts;
  PP_REQUIRE(P.grid <= INT32_MAX, "pp_kv_attention: too many rows");
  A.scale = scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
  const int D = cache->head_dim;
  if (P.rows > 32) return kv_attn_many(A, P, D, cache->codes, dtype, st);
  if (cache->codes == PP_KV_INT8)
    return dtype == PP_F16 ? attn_width<PP_KV_INT8, IoF16>(A, P, D, st) : attn_width<PP_KV_INT8, IoBf16>(A, P, D, st);
  return dtype == PP_F16 ? attn_width<PP_KV_E4M3, IoF16>(A, P, D, st) : attn_width<PP_KV_E4M3, IoBf16>(A, P, D, st);
}
