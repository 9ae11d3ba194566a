// Writing keys and values into the 8-bit cache, and reading them back.
#include "kv_common.h"

namespace pp {

int kv_check_cache(const pp_kv_cache* c, KvCache* out) {
  PP_REQUIRE(c != nullptr, "kv cache: null");
  PP_REQUIRE(c->k && c->v && c->k_scale && c->v_scale, "kv cache: null codes or scales");
  PP_REQUIRE(c->pages > 0 && c->pages <= INT32_MAX, "kv cache: pages %lld", (long long)c->pages);
  PP_REQUIRE(c->heads > 0 && c->heads <= 65535, "kv cache: heads %d not in 1..65535", c->heads);
  PP_REQUIRE(c->block == 16 || c->block == 32 || c->block == 64 || c->block == 128,
             "kv cache: block %d is not 16, 32, 64 or 128", c->block);
  PP_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 192 || c->head_dim == 256,
             "kv cache: head_dim %d is not 64, 128, 192 or 256", c->head_dim);
  PP_REQUIRE(c->codes == PP_KV_INT8 || c->codes == PP_KV_E4M3, "kv cache: codes %d", c->codes);
  PP_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16), "kv cache: codes are not 16-byte aligned");
  *out = KvCache{(uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale, c->pages, c->heads, c->block,
                 c->block == 16 ? 4 : c->block == 32 ? 5 : c->block == 64 ? 6 : 7};
  return PP_OK;
}

int kv_check_seqs(const KvCache& c, const int32_t* table, int64_t ld, int64_t width, const int32_t* lengths, const int32_t* cu,
                  int64_t batch, int64_t tokens, KvSeqs* out) {
  PP_REQUIRE(table && lengths, "kv: null block table or lengths");
  PP_REQUIRE(batch > 0 && batch <= (1 << 24), "kv: batch %lld not in 1..2^24", (long long)batch);
  PP_REQUIRE(tokens >= 0 && tokens <= (1 << 28), "kv: tokens %lld not in 0..2^28", (long long)tokens);
  PP_REQUIRE(width > 0 && width <= (1 << 30) >> c.shift, "kv: a block table of %lld pages holds no or over 2^30 tokens",
             (long long)width);
  PP_REQUIRE(ld >= width || batch == 1, "kv: block table rows of %lld overlap (stride %lld)", (long long)width,
             (long long)ld);
  PP_REQUIRE(cu != nullptr || tokens == batch, "kv: %lld tokens of %lld sequences need cu", (long long)tokens,
             (long long)batch);
  *out = KvSeqs{table, ld, lengths, cu, (int)width, (int)batch, (int)tokens};
  return PP_OK;
}

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
  int64_t row0;       // the token at place t of the page is row row0 + t of the call's tokens
  int lo, hi, page;   // places lo..hi-1 of the page
};

__device__ __forceinline__ bool kv_piece(const KvCache& C, const KvSeqs& S, int at, Piece& P) {
  int b = at, slot = 0;
  if (S.cu != nullptr) {
    b = kv_find(S, at, 1, C.shift, 2);
    slot = at - kv_begin(S, b, 1, C.shift, 2);
  }
  const int s0 = kv_start(S, b), n = kv_start(S, b + 1) - s0;
  if (n <= 0) return false;
  const bool real = b < S.batch;
  const int64_t len = real ? S.lengths[b] : n, first = len - n;
  const int64_t blk = (first >> C.shift) + slot, p0 = blk << C.shift;
  const int64_t lo = first > p0 ? first : p0, hi = len < p0 + C.block ? len : p0 + C.block;
  if (lo >= hi) return false;
  P.row0 = s0 + p0 - first;
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

template <int CODES, typename IO, int D>
__global__ __launch_bounds__(1024) void kv_append_kernel(const AppendArgs A) {
  using Q = KvCodes<CODES>;
  const KvCache& C = A.C;
  Piece P;
  const Unit N = kv_unit(C);
  if (!kv_piece(C, A.S, N.item, P) || P.page < 0) return;
  const int head = N.head, isv = N.isv;
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int held = P.lo, end = P.hi;                   // new tokens held..end-1 of the page
  __shared__ uint32_t red[16];
  extern __shared__ uint32_t tile[];                   // V codes: [D][block / 4 + 1] words

  const int tg = tid / (D / 8), dg = tid % (D / 8);    // tokens 4*tg.., values 8*dg..
  const bool mine = tid < (C.block / 4) * (D / 8);
  // Magnitudes of 16-bit values are ordered like their words, NaN last, so the maximum is taken of those.
  u32x4 x[4];
  u16x2 big = {0, 0};
  const uint16_t* src = A.x[isv] + (int64_t)head * A.sh[isv];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * tg + i;
    x[i] = u32x4{0, 0, 0, 0};
    if (mine && t >= held && t < end) x[i] = load8(src + (P.row0 + t) * A.st[isv] + 8 * dg, A.vec);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, x[i][j] & 0x7fff7fffu));
  uint32_t top = wave_umax(max((uint32_t)big[0], (uint32_t)big[1]));
  if ((tid & 63) == 0) red[tid >> 6] = top;
  const int64_t ph = (int64_t)P.page * C.heads + head;
  float* scale_at = (isv ? C.vs : C.ks) + ph;
  const float was = held ? *scale_at : 0.f;
  __syncthreads();
  for (int w = 0; w < (nthr + 63) / 64; ++w) top = max(top, red[w]);
  top = mag(IO::get((uint16_t)top));
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
  if (tid == 0) *scale_at = now;

  uint32_t w8[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t u = x[i][2 * j], v = x[i][2 * j + 1];
      w8[i][j] = finite ? Q::pack(IO::get((uint16_t)u) * inv, IO::get((uint16_t)(u >> 16)) * inv,
                                  IO::get((uint16_t)v) * inv, IO::get((uint16_t)(v >> 16)) * inv)
                        : 0u;
    }
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
    if (grown)
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

// Reading back: the same units, each output row written once; tokens that lie on no page, or past
// the last sequence, read zero.
struct ReadArgs {
  KvCache C;
  KvSeqs S;
  void* out[2];
};

template <int CODES, typename IO, int D>
__global__ __launch_bounds__(1024) void kv_read_kernel(const ReadArgs A) {
  using Q = KvCodes<CODES>;
  const KvCache& C = A.C;
  Piece P;
  const Unit N = kv_unit(C);
  if (!kv_piece(C, A.S, N.item, P)) return;
  const int head = N.head, isv = N.isv;
  const int tid = threadIdx.x, nthr = blockDim.x;
  extern __shared__ uint32_t tile[];
  const bool none = P.page < 0;                        // read page 0, write zeros
  const int64_t ph = (int64_t)(none ? 0 : P.page) * C.heads + head, base = ph * (C.block * D);
  const float scale = none ? 0.f : (isv ? C.vs : C.ks)[ph];
  const int tg = tid / (D / 8), dg = tid % (D / 8);
  const bool mine = tid < (C.block / 4) * (D / 8);
  uint32_t w8[4][2];
  if (isv) {
    const u32x4* v = reinterpret_cast<const u32x4*>(C.v + base);
    const int ql = C.shift - 4, ld = C.block / 4 + 1;
    for (int w = tid; w < D << ql; w += nthr) {
      const u32x4 c = v[w];
      uint32_t* t = tile + (w >> ql) * ld + 4 * (w & ((1 << ql) - 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = c[i];
    }
    __syncthreads();
    if (!mine) return;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = tile[(8 * dg + 4 * j + i) * ld + tg];
      swap_bytes(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) w8[i][j] = c[i];
    }
  } else {
    if (!mine) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(C.k + base + (4 * tg + i) * D + 8 * dg);
      w8[i][0] = w[0];
      w8[i][1] = w[1];
    }
  }
  typedef typename IO::raw raw;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * tg + i;
    if (t < P.lo || t >= P.hi) continue;
    raw* o = reinterpret_cast<raw*>(A.out[isv]) + ((P.row0 + t) * C.heads + head) * D + 8 * dg;
    float x[8];
    Q::unpack(none ? 0u : w8[i][0], x);
    Q::unpack(none ? 0u : w8[i][1], x + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= scale;
    if constexpr (sizeof(raw) == 4) {
      reinterpret_cast<f32x4*>(o)[0] = f32x4{x[0], x[1], x[2], x[3]};
      reinterpret_cast<f32x4*>(o)[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
      *reinterpret_cast<u32x4*>(o) = u32x4{IO::put2(x[0], x[1]), IO::put2(x[2], x[3]), IO::put2(x[4], x[5]),
                                           IO::put2(x[6], x[7])};
    }
  }
}

template <typename F>
static int by_width(int D, F&& f) {
  switch (D) {
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
    case 192: return f(std::integral_constant<int, 192>());
    default: return f(std::integral_constant<int, 256>());
  }
}

static unsigned unit_threads(int block, int D) { return (unsigned)((block * D / 32 + 63) / 64 * 64); }
static unsigned tile_bytes(int block, int D) { return (unsigned)(D * (block / 4 + 1) * 4); }
static int64_t pieces(const KvCache& C, const KvSeqs& S) {
  return S.cu ? S.tokens / C.block + 2 * (int64_t)S.batch + 2 : S.batch;
}

}  // namespace pp

using namespace pp;

extern "C" int pp_kv_append(const pp_kv_cache* cache, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                            int64_t v_st, int64_t v_sh, int dtype, int64_t tokens, const int32_t* table,
                            int64_t table_ld, int64_t table_width, const int32_t* lengths, const int32_t* cu,
                            int64_t batch, void* stream) {
  AppendArgs A;
  int rc = kv_check_cache(cache, &A.C);
  if (rc) return rc;
  rc = kv_check_seqs(A.C, table, table_ld, table_width, lengths, cu, batch, tokens, &A.S);
  if (rc) return rc;
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16, "pp_kv_append: dtype %d is not PP_F16 or PP_BF16", dtype);
  if (tokens == 0) return PP_OK;
  PP_REQUIRE(k && v, "pp_kv_append: null keys or values");
  PP_REQUIRE(aligned(k, 2) && aligned(v, 2), "pp_kv_append: keys or values are not 2-byte aligned");
  A.x[0] = (const uint16_t*)k;
  A.x[1] = (const uint16_t*)v;
  A.st[0] = k_st; A.st[1] = v_st;
  A.sh[0] = k_sh; A.sh[1] = v_sh;
  A.vec = aligned(k, 16) && aligned(v, 16) && k_st % 8 == 0 && k_sh % 8 == 0 && v_st % 8 == 0 && v_sh % 8 == 0;
  const int64_t items = pieces(A.C, A.S);
  const dim3 wg(unit_threads(A.C.block, cache->head_dim));
  PP_REQUIRE(items * 2 * A.C.heads <= UINT32_MAX / wg.x, "pp_kv_append: too many tokens and sequences");
  const dim3 grid((unsigned)(items * 2 * A.C.heads));
  const unsigned lds = tile_bytes(A.C.block, cache->head_dim);
  return by_width(cache->head_dim, [&](auto d) -> int {
    constexpr int D = decltype(d)::value;
    const bool i8 = cache->codes == PP_KV_INT8, h = dtype == PP_F16;
    auto kern = i8 ? (h ? kv_append_kernel<PP_KV_INT8, IoF16, D> : kv_append_kernel<PP_KV_INT8, IoBf16, D>)
                   : (h ? kv_append_kernel<PP_KV_E4M3, IoF16, D> : kv_append_kernel<PP_KV_E4M3, IoBf16, D>);
    hipLaunchKernelGGL(kern, grid, wg, lds, (hipStream_t)stream, A);
    PP_LAUNCH_CHECK();
    return PP_OK;
  });
}

extern "C" int pp_kv_read(const pp_kv_cache* cache, const int32_t* table, int64_t table_ld, int64_t table_width,
                          const int32_t* lengths, const int32_t* cu, int64_t batch, int64_t tokens, int dtype,
                          void* k_out, void* v_out, void* stream) {
  ReadArgs A;
  int rc = kv_check_cache(cache, &A.C);
  if (rc) return rc;
  rc = kv_check_seqs(A.C, table, table_ld, table_width, lengths, cu, batch, tokens, &A.S);
  if (rc) return rc;
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16 || dtype == PP_F32, "pp_kv_read: dtype %d", dtype);
  if (tokens == 0) return PP_OK;
  PP_REQUIRE(k_out && v_out, "pp_kv_read: null outputs");
  PP_REQUIRE(aligned(k_out, 16) && aligned(v_out, 16), "pp_kv_read: outputs are not 16-byte aligned");
  A.out[0] = k_out;
  A.out[1] = v_out;
  const int64_t items = pieces(A.C, A.S);
  const dim3 wg(unit_threads(A.C.block, cache->head_dim));
  PP_REQUIRE(items * 2 * A.C.heads <= UINT32_MAX / wg.x, "pp_kv_read: too many tokens and sequences");
  const dim3 grid((unsigned)(items * 2 * A.C.heads));
  const unsigned lds = tile_bytes(A.C.block, cache->head_dim);
  return by_width(cache->head_dim, [&](auto d) -> int {
    constexpr int D = decltype(d)::value;
    const bool i8 = cache->codes == PP_KV_INT8;
    auto kern = dtype == PP_F16    ? (i8 ? kv_read_kernel<PP_KV_INT8, IoF16, D> : kv_read_kernel<PP_KV_E4M3, IoF16, D>)
                : dtype == PP_BF16 ? (i8 ? kv_read_kernel<PP_KV_INT8, IoBf16, D> : kv_read_kernel<PP_KV_E4M3, IoBf16, D>)
                                   : (i8 ? kv_read_kernel<PP_KV_INT8, IoF32, D> : kv_read_kernel<PP_KV_E4M3, IoF32, D>);
    hipLaunchKernelGGL(kern, grid, wg, lds, (hipStream_t)stream, A);
    PP_LAUNCH_CHECK();
    return PP_OK;
  });
}
