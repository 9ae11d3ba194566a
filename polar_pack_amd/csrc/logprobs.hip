// Log probabilities of given tokens, entropy and the most likely alternatives of rows of logits.
//
//   lse = m + log s,  s = sum e^(x - m),  t = sum (x - m) e^(x - m),  m = max x,
//   logprob = x[token] - lse,  entropy = lse - sum p x = log s - t / s,
//   alternatives: the k largest x, equal ones by the lower index, with x - lse.
//
// One pass over the logits: a workgroup reads a part of a row in steps of 16 logits a thread and
// keeps (m, s, t) per thread.  The alternatives ride along: every logit is a 64-bit key (its order
// in the high word, ~index in the low one, so no two are equal and a larger key is a better one),
// and keys at or above a threshold that at least k keys reach go to a list in LDS, from which they
// are picked whenever it has grown.  Few rows are split into parts, joined by a second launch.
//
// What bounds it: without alternatives the reading (2047 rows of 151,936 in float32, 1.24 GB: 219 us, 5.7
// TB/s); with alternatives instructions and latency (250 rows in bf16 with 20 alternatives, 76 MB: 47 us; 22
// instructions a logit, the vector units 56 % busy, two barriers a step).  A first floor from the threads'
// largest logits and tests as floats before keys are made took it from 56 to 47; 4 workgroups a CU
// instead of 2 cost 69 (each part picks its own list), 1 a CU 62.
#include "kv_common.h"

namespace pp {

constexpr int LP_THREADS = 256;
constexpr int LP_PER = 16;                        // logits a thread and step
constexpr int LP_STEP = LP_THREADS * LP_PER;
constexpr int LP_TIDY = 128;                      // a longer list is picked after the step
constexpr int LP_LIST = LP_STEP + LP_TIDY;
constexpr int LP_TOP_MAX = 64;

struct LpArgs {
  const void* x;
  int64_t x_st;
  const int64_t* tokens;
  int64_t t_st;
  float* logprob;
  float* entropy;
  int64_t* ids;
  float* top_lp;
  float* stats;          // [row][part][4]: m, s, t
  uint64_t* keys;        // [row][part][k]
  int rows, V, per_row, k, parts, part;   // `part` logits a part, a multiple of LP_STEP
};

__device__ __forceinline__ uint64_t lp_key(float x, int index) {
  const uint32_t u = __float_as_uint(x + 0.f);    // -0 counts as 0
  const uint32_t o = x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return ((uint64_t)o << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

struct LpStat {
  float m, s, t;
};
__device__ __forceinline__ float lp_ref(float m) { return m == -INFINITY ? 0.f : m; }
// A difference to the maximum, held where e^d is 0 all the same: d * e^d and d * s stay numbers.
__device__ __forceinline__ float lp_far(float d) { return fmaxf(d, -1e30f); }
__device__ __forceinline__ LpStat lp_join(const LpStat& a, const LpStat& b) {
  const float m = fmaxf(a.m, b.m), r = lp_ref(m);
  const float da = lp_far(a.m - r), db = lp_far(b.m - r);
  const float ea = __expf(da), eb = __expf(db);
  return LpStat{m, a.s * ea + b.s * eb, ea * (a.t + da * a.s) + eb * (b.t + db * b.s)};
}

struct LpShared {
  uint64_t list[LP_LIST];
  uint64_t group[64];
  uint64_t best[LP_TOP_MAX];
  int count;
  uint64_t floor;
};

struct LpNone {};
template <bool TOP>
struct LpLds { typedef LpShared type; };
template <>
struct LpLds<false> { typedef LpNone type; };
__device__ __forceinline__ const uint64_t* lp_best(const LpShared& L) { return L.best; }
__device__ __forceinline__ const uint64_t* lp_best(const LpNone&) { return nullptr; }

// Raises the floor to the k-th largest of 64 groups' largest keys (thread t's in group t % 64): k keys at
// least reach it.
__device__ __forceinline__ void lp_floor(LpShared& L, uint64_t top, int k) {
  const int tid = threadIdx.x;
  if (tid < 64) L.group[tid] = 0;
  __syncthreads();
  atomicMax((unsigned long long*)&L.group[tid & 63], (unsigned long long)top);
  __syncthreads();
  if (tid < 64) {
    const uint64_t g = L.group[tid];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < 64; ++i) rank += L.group[i] > g || (L.group[i] == g && i < tid);
    if (rank == k - 1 && g > L.floor) L.floor = g;
  }
  __syncthreads();
}

// Keys of `list` below a floor that k of them reach leave it.
__device__ __forceinline__ void lp_tidy(LpShared& L, int k) {
  const int tid = threadIdx.x;
  const int n = L.count;
  uint64_t mine[(LP_LIST + LP_THREADS - 1) / LP_THREADS];
  uint64_t top = 0;
#pragma unroll
  for (int i = 0; i < (LP_LIST + LP_THREADS - 1) / LP_THREADS; ++i) {
    const int at = tid + i * LP_THREADS;
    mine[i] = at < n ? L.list[at] : 0;
    top = mine[i] > top ? mine[i] : top;
  }
  __syncthreads();
  if (tid == 0) L.count = 0;
  lp_floor(L, top, k);
  const uint64_t fl = L.floor;
#pragma unroll
  for (int i = 0; i < (LP_LIST + LP_THREADS - 1) / LP_THREADS; ++i)
    if (mine[i] != 0 && mine[i] >= fl) L.list[atomicAdd(&L.count, 1)] = mine[i];
  __syncthreads();
}

// The k best keys of the list in order, in L.best; the list may be longer than LP_TIDY.
__device__ __forceinline__ void lp_pick(LpShared& L, int k) {
  const int n0 = L.count;
  __syncthreads();
  if (n0 > LP_TIDY) lp_tidy(L, k);
  const int n = L.count;
  for (int at = threadIdx.x; at < n; at += LP_THREADS) {
    const uint64_t key = L.list[at];
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += L.list[i] > key;
    if (rank < k) L.best[rank] = key;
  }
  __syncthreads();
}

// A list longer than LP_TIDY to at most that: where bounds do not do it, to its k best.
__device__ __forceinline__ void lp_shorten(LpShared& L, int k) {
  lp_tidy(L, k);
  const int n = L.count;
  __syncthreads();
  if (n <= LP_TIDY) return;
  lp_pick(L, k);
  if (threadIdx.x < k) L.list[threadIdx.x] = L.best[threadIdx.x];
  if (threadIdx.x == 0) {
    L.count = k;
    L.floor = L.best[k - 1];
  }
  __syncthreads();
}

__device__ __forceinline__ LpStat lp_block_join(LpStat v, float* sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    v = lp_join(v, LpStat{__shfl_xor(v.m, o, 64), __shfl_xor(v.s, o, 64), __shfl_xor(v.t, o, 64)});
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) { sh[3 * w] = v.m; sh[3 * w + 1] = v.s; sh[3 * w + 2] = v.t; }
  __syncthreads();
  v = LpStat{sh[0], sh[1], sh[2]};
  for (int i = 1; i < LP_THREADS / 64; ++i) v = lp_join(v, LpStat{sh[3 * i], sh[3 * i + 1], sh[3 * i + 2]});
  return v;
}

template <typename IO>
__device__ __forceinline__ float lp_at(const LpArgs& A, int row, int64_t i) {
  return IO::get(reinterpret_cast<const typename IO::raw*>(A.x)[(int64_t)row * A.x_st + i]);
}

// What a row's joined statistics and best keys give.
template <typename IO>
__device__ __forceinline__ void lp_write(const LpArgs& A, int row, const LpStat& v, const uint64_t* best) {
  const float logs = logf(v.s), lse = v.m + logs;
  if (threadIdx.x == 0) A.entropy[row] = logs - v.t / v.s;
  for (int j = threadIdx.x; j < A.per_row; j += LP_THREADS) {
    const int64_t t = A.tokens[(int64_t)row * A.t_st + j];
    A.logprob[(int64_t)row * A.per_row + j] = t >= 0 && t < A.V ? lp_at<IO>(A, row, t) - lse : NAN;
  }
  for (int j = threadIdx.x; j < A.k; j += LP_THREADS) {
    A.ids[(int64_t)row * A.k + j] = (int64_t)(uint32_t)~(uint32_t)best[j];
    A.top_lp[(int64_t)row * A.k + j] = lp_value(best[j]) - lse;
  }
}

template <typename IO, bool TOP>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(const LpArgs A) {
  typedef typename IO::raw raw;
  constexpr int VE = 16 / sizeof(raw);             // logits a load
  __shared__ float sh[3 * LP_THREADS / 64];
  __shared__ typename LpLds<TOP>::type L;
  const int row = blockIdx.x / A.parts, part = blockIdx.x % A.parts, tid = threadIdx.x;
  const raw* x = reinterpret_cast<const raw*>(A.x) + (int64_t)row * A.x_st;
  // loads at 16-byte boundaries: logit i lies in load (i + skew) / VE
  const int skew = (int)((reinterpret_cast<uintptr_t>(x) % 16) / sizeof(raw));
  const int lo = part * A.part, hi = min(A.V + skew, lo + A.part);
  LpStat v{-INFINITY, 0.f, 0.f};
  if constexpr (TOP) {
    if (tid == 0) { L.count = 0; L.floor = 0; }
    __syncthreads();
  }
  // The logits of the next two steps are on their way while a step's are worked on.
  constexpr int LOADS = LP_PER / VE;
  auto fetch = [&](u32x4* w, int c) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int at = c + (u * LP_THREADS + tid) * VE - skew;   // first logit of the load
      if (at >= 0 && at + VE <= A.V && c < hi) {
        w[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x + at));
      } else {
        raw e[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) e[i] = c < hi && at + i >= 0 && at + i < A.V ? x[at + i] : IO::put(-INFINITY);
        __builtin_memcpy(&w[u], e, 16);
      }
    }
  };
  auto step = [&](const u32x4* w, int c) {
    float f[LP_PER];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      raw e[VE];
      __builtin_memcpy(e, &w[u], 16);
#pragma unroll
      for (int i = 0; i < VE; ++i) f[u * VE + i] = IO::get(e[i]);
    }
    float top = f[0];
#pragma unroll
    for (int i = 1; i < LP_PER; ++i) top = fmaxf(top, f[i]);
    if (top > v.m) {
      if (v.m != -INFINITY) {
        const float d = lp_far(v.m - top), e = __expf(d);
        v.t = e * (v.t + d * v.s);
        v.s *= e;
      }
      v.m = top;
    }
    const float r = lp_ref(v.m);
#pragma unroll
    for (int i = 0; i < LP_PER; ++i) {
      const float d = f[i] - r, e = __expf(d);
      v.s += e;
      v.t += lp_far(d) * e;
    }
    if constexpr (TOP) {
      auto each = [&](auto f2) {
#pragma unroll
        for (int u = 0; u < LP_PER / VE; ++u)
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const int at = c + (u * LP_THREADS + tid) * VE - skew + i;
            f2(f[u * VE + i], at);
          }
      };
      if (c == lo) {                                 // a first floor, so that the list starts short
        uint64_t best = 0;
        each([&](float x, int at) {
          const uint64_t key = at >= 0 && at < A.V ? lp_key(x, at) : 0;
          best = key > best ? key : best;
        });
        lp_floor(L, best, A.k);
      }
      const uint64_t fl = L.floor;
      // few threads hold a candidate: a logit not below the floor's, or a NaN, which the sums show
      const float least = lp_value(fl);              // a NaN while there is no floor: nothing is below it
      if (!(top < least) || v.s != v.s)
        each([&](float x, int at) {
          if (x < least || at < 0 || at >= A.V) return;
          const uint64_t key = lp_key(x, at);
          if (key >= fl) L.list[atomicAdd(&L.count, 1)] = key;
        });
      __syncthreads();
      const int n = L.count;
      __syncthreads();                               // all have read the count before the next step adds to it
      if (n > LP_TIDY) lp_shorten(L, A.k);
    }
  };
  u32x4 w0[LOADS], w1[LOADS];
  fetch(w0, lo);
  fetch(w1, lo + LP_STEP);
  for (int c = lo; c < hi; c += 2 * LP_STEP) {
    step(w0, c);
    fetch(w0, c + 2 * LP_STEP);
    if (c + LP_STEP >= hi) break;
    step(w1, c + LP_STEP);
    fetch(w1, c + 3 * LP_STEP);
  }
  v = lp_block_join(v, sh);
  if constexpr (TOP) {
    for (int j = tid; j < A.k; j += LP_THREADS) L.best[j] = 0;
    __syncthreads();
    lp_pick(L, A.k);
  }
  if (A.parts == 1) {
    lp_write<IO>(A, row, v, lp_best(L));
    return;
  }
  const int64_t at = (int64_t)row * A.parts + part;
  if (tid == 0) {
    A.stats[4 * at] = v.m; A.stats[4 * at + 1] = v.s; A.stats[4 * at + 2] = v.t;
  }
  if constexpr (TOP)
    for (int j = tid; j < A.k; j += LP_THREADS) A.keys[at * A.k + j] = L.best[j];
}

template <typename IO, bool TOP>
__global__ __launch_bounds__(LP_THREADS) void logprobs_join_kernel(const LpArgs A) {
  __shared__ float sh[3 * LP_THREADS / 64];
  __shared__ typename LpLds<TOP>::type L;
  const int row = blockIdx.x, tid = threadIdx.x;
  LpStat v{-INFINITY, 0.f, 0.f};
  for (int p = tid; p < A.parts; p += LP_THREADS) {
    const float* s = A.stats + 4 * ((int64_t)row * A.parts + p);
    v = lp_join(v, LpStat{s[0], s[1], s[2]});
  }
  v = lp_block_join(v, sh);
  if constexpr (TOP) {
    if (tid == 0) { L.count = 0; L.floor = 0; }
    __syncthreads();
    const uint64_t* keys = A.keys + (int64_t)row * A.parts * A.k;
    for (int j = tid; j < A.parts * A.k; j += LP_THREADS)
      if (keys[j] != 0) L.list[atomicAdd(&L.count, 1)] = keys[j];
    __syncthreads();
    lp_pick(L, A.k);
  }
  lp_write<IO>(A, row, v, lp_best(L));
}

// Parts a row: one from 2 workgroups a CU on; otherwise as many as that takes, of whole steps, and
// no more candidates than the join's list holds.
static void lp_plan(int64_t rows, int64_t V, int64_t k, int64_t* parts, int64_t* part) {
  const int64_t steps = (V + 16 + LP_STEP - 1) / LP_STEP;      // 16: the row's skew
  int64_t p = (2 * device_cu_count() + rows - 1) / rows;
  if (k > 0 && p > LP_LIST / k) p = LP_LIST / k;
  if (p > steps) p = steps;
  if (p < 1) p = 1;
  const int64_t per = (steps + p - 1) / p;
  *part = per * LP_STEP;
  *parts = (steps + per - 1) / per;
}

template <bool TOP>
static int lp_launch(const LpArgs& A, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)A.rows * A.parts));
  auto kern = dtype == PP_F16 ? logprobs_kernel<IoF16, TOP>
              : dtype == PP_BF16 ? logprobs_kernel<IoBf16, TOP> : logprobs_kernel<IoF32, TOP>;
  hipLaunchKernelGGL(kern, grid, dim3(LP_THREADS), 0, st, A);
  PP_LAUNCH_CHECK();
  if (A.parts == 1) return PP_OK;
  auto join = dtype == PP_F16 ? logprobs_join_kernel<IoF16, TOP>
              : dtype == PP_BF16 ? logprobs_join_kernel<IoBf16, TOP> : logprobs_join_kernel<IoF32, TOP>;
  hipLaunchKernelGGL(join, dim3((unsigned)A.rows), dim3(LP_THREADS), 0, st, A);
  PP_LAUNCH_CHECK();
  return PP_OK;
}

}  // namespace pp

using namespace pp;

extern "C" int64_t pp_logprobs_workspace_size(int64_t rows, int64_t V, int64_t top) {
  if (rows <= 0 || V <= 0 || top < 0) return 0;
  int64_t parts, part;
  lp_plan(rows, V, top, &parts, &part);
  return parts == 1 ? 0 : rows * parts * (16 + 8 * top);
}

extern "C" int pp_logprobs(const void* logits, int64_t l_st, int dtype, int64_t rows, int64_t V,
                           const int64_t* tokens, int64_t t_st, int64_t per_row, int64_t top, float* logprob,
                           float* entropy, int64_t* top_ids, float* top_logprobs, void* workspace,
                           int64_t workspace_size, void* stream) {
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16 || dtype == PP_F32, "pp_logprobs: dtype %d", dtype);
  PP_REQUIRE(rows >= 0 && rows <= (1 << 24), "pp_logprobs: rows %lld not in 0..2^24", (long long)rows);
  PP_REQUIRE(V > 0 && V <= (1 << 30), "pp_logprobs: %lld logits a row", (long long)V);
  PP_REQUIRE(top >= 0 && top <= LP_TOP_MAX && top <= V, "pp_logprobs: top %lld not in 0..min(%d, logits)",
             (long long)top, LP_TOP_MAX);
  PP_REQUIRE(per_row >= 0 && per_row <= INT32_MAX, "pp_logprobs: %lld tokens a row", (long long)per_row);
  if (rows == 0) return PP_OK;
  PP_REQUIRE(logits && entropy, "pp_logprobs: null logits or entropy");
  PP_REQUIRE(aligned(logits, dtype == PP_F32 ? 4 : 2), "pp_logprobs: logits are not aligned to their type");
  PP_REQUIRE(per_row == 0 || (tokens && logprob), "pp_logprobs: null tokens or logprob");
  PP_REQUIRE(top == 0 || (top_ids && top_logprobs), "pp_logprobs: null alternatives");
  LpArgs A;
  int64_t parts, part;
  lp_plan(rows, V, top, &parts, &part);
  PP_REQUIRE(rows * parts <= INT32_MAX, "pp_logprobs: too many rows");
  const int64_t need = parts == 1 ? 0 : rows * parts * (16 + 8 * top);
  PP_REQUIRE(need == 0 || (workspace && workspace_size >= need && aligned(workspace, 16)),
             "pp_logprobs: workspace of %lld bytes at a 16-byte boundary needed", (long long)need);
  A.x = logits; A.x_st = l_st;
  A.tokens = tokens; A.t_st = t_st;
  A.logprob = logprob; A.entropy = entropy; A.ids = top_ids; A.top_lp = top_logprobs;
  A.stats = (float*)workspace;
  A.keys = (uint64_t*)((char*)workspace + rows * parts * 16);
  A.rows = (int)rows; A.V = (int)V; A.per_row = (int)per_row; A.k = (int)top;
  A.parts = (int)parts; A.part = (int)part;
  return top ? lp_launch<true>(A, dtype, (hipStream_t)stream) : lp_launch<false>(A, dtype, (hipStream_t)stream);
}
