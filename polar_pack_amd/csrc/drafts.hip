// Drafted tokens against the target's probabilities.
//
// Sequence b drafted c tokens d_i from distributions q_i; p_0 .. p_c are the target's.  With given numbers u:
//   accepted = the first i with not (u_i q_i(d_i) < p_i(d_i)), or c,
//   the token after them is drawn with u_n from r = max(p_i - q_i, 0) (refused at i) or r = p_c: the first t whose
//   sum r_0 + .. + r_t passes u_n times the sum of all.
// Tokens are whole numbers, so the sums are held in 64 bits: in 32 a vocabulary's sum is off by more than the
// smallest probabilities, and neighbouring tokens would change places.
//
// Only the row that is drawn from is read, cut into parts over workgroups.  Each finds the row by itself (two round
// trips: tokens, then their probabilities), sums its part, and counts itself done; the one that counts last finds the
// part in which the sum passes, reads that again and finds the token.  One launch, and the order of the sums is
// fixed by the parts.
#include "kv_common.h"

namespace pp {

constexpr int DR_THREADS = 256;
constexpr int DR_PER = 16;                          // entries a thread and step
constexpr int DR_STEP = DR_THREADS * DR_PER;

struct DraftArgs {
  const void* p;
  const void* q;          // null: the drafts were certain
  const int64_t* tokens;
  const float* u;
  const int32_t* counts;  // null: n of every sequence
  int64_t* out;
  int64_t* accepted;
  double* sums;           // [sequence][part]: of r
  uint32_t* done;         // [sequence]: parts that are done; 0 before and after
  int64_t p_sb, p_sr, q_sb, q_sr, t_sb, u_sb;
  int batch, n, V, parts, part;       // `part` entries a part, a multiple of DR_STEP
};

// What counts as a probability: a positive number, otherwise 0.
__device__ __forceinline__ float dr_clean(float x) { return x > 0.f && x < INFINITY ? x : 0.f; }

template <typename IO>
struct DraftRow {
  const typename IO::raw* p;
  const typename IO::raw* q;    // null: nothing to take off but `without`
  int without;                  // an entry that counts 0, or -1
};

// Entries c + (l * DR_THREADS + tid) * VE + 0 .. VE - 1 of a row for l = 0 .. DR_PER / VE - 1.
template <typename IO>
__device__ __forceinline__ void dr_load(const typename IO::raw* x, int c, int V, float* f) {
  typedef typename IO::raw raw;
  constexpr int VE = 16 / sizeof(raw);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0;
#pragma unroll
  for (int l = 0; l < DR_PER / VE; ++l) {
    const int at = c + (l * DR_THREADS + (int)threadIdx.x) * VE;
    if (vec && at + VE <= V) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(x + at);
      raw e[VE];
      __builtin_memcpy(e, &w, 16);
#pragma unroll
      for (int i = 0; i < VE; ++i) f[l * VE + i] = dr_clean(IO::get(e[i]));
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) f[l * VE + i] = at + i < V ? dr_clean(IO::get(x[at + i])) : 0.f;
    }
  }
}

// r of these entries; `all`: of p alone.
template <typename IO>
__device__ __forceinline__ void dr_rest(const DraftRow<IO>& R, int c, int V, bool all, double* r) {
  constexpr int VE = 16 / sizeof(typename IO::raw);
  float f[DR_PER], g[DR_PER];
  dr_load<IO>(R.p, c, V, f);
  if (R.q && !all) {
    dr_load<IO>(R.q, c, V, g);
#pragma unroll
    for (int i = 0; i < DR_PER; ++i) r[i] = fmax((double)f[i] - (double)g[i], 0.0);
  } else {
#pragma unroll
    for (int i = 0; i < DR_PER; ++i) {
      const int at = c + (i / VE * DR_THREADS + (int)threadIdx.x) * VE + i % VE;
      r[i] = at == R.without && !all ? 0.0 : (double)f[i];
    }
  }
}

__device__ __forceinline__ double dr_shfl_up(double v, int o) { return __shfl_up(v, o, 64); }
__device__ __forceinline__ double dr_scan(double v) {           // inclusive, over the wavefront
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double w = dr_shfl_up(v, o);
    v += (int)(threadIdx.x & 63) >= o ? w : 0.0;
  }
  return v;
}
__device__ __forceinline__ double dr_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <typename IO>
__global__ __launch_bounds__(DR_THREADS) void verify_drafts_kernel(const DraftArgs A) {
  typedef typename IO::raw raw;
  constexpr int VE = 16 / sizeof(raw), LOADS = DR_PER / VE;
  __shared__ double waves[DR_THREADS / 64], totals[LOADS][DR_THREADS / 64];
  __shared__ uint32_t last;
  __shared__ int found;
  const int b = blockIdx.x / A.parts, part = blockIdx.x - b * A.parts;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const raw* const p = reinterpret_cast<const raw*>(A.p) + b * A.p_sb;
  const raw* const q = A.q ? reinterpret_cast<const raw*>(A.q) + b * A.q_sb : nullptr;
  const int64_t* const tokens = A.tokens + b * A.t_sb;
  const float* const u = A.u + b * A.u_sb;

  // every wavefront looks at 64 drafts a round
  const int count = A.counts ? min(max(A.counts[b], 0), A.n) : A.n;
  int accepted = count;
  for (int i0 = 0; i0 < A.n; i0 += 64) {
    const int i = i0 + lane;
    bool bad = i >= count;
    if (i < A.n) {
      const int64_t t = tokens[i];
      const bool in = t >= 0 && t < A.V;
      const float pd = in ? dr_clean(IO::get(p[i * A.p_sr + t])) : 0.f;
      const float qd = !q ? 1.f : in ? dr_clean(IO::get(q[i * A.q_sr + t])) : 0.f;
      bad |= !((double)u[i] * (double)qd < (double)pd);
    }
    const uint64_t mask = __ballot(bad);
    if (mask) {
      accepted = min(count, i0 + __builtin_ctzll(mask));
      break;
    }
  }
  const bool refused = accepted < count;
  DraftRow<IO> R;
  R.p = p + accepted * A.p_sr;
  R.q = refused && q ? q + accepted * A.q_sr : nullptr;
  R.without = -1;
  if (refused && !q) {
    const int64_t t = tokens[accepted];
    R.without = t >= 0 && t < A.V ? (int)t : -1;
  }

  // over the workgroup, the same in every thread
  auto block_sum = [&](double v) {
    v = dr_sum(v);
    if (lane == 0) waves[wave] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < DR_THREADS / 64; ++w) v += waves[w];
    __syncthreads();
    return v;
  };
  auto range_sum = [&](int lo, int hi, bool all) {
    double v = 0.0;
    for (int c = lo; c < hi; c += DR_STEP) {
      double r[DR_PER];
      dr_rest<IO>(R, c, A.V, all, r);
#pragma unroll
      for (int i = 0; i < DR_PER; ++i) v += r[i];
    }
    return block_sum(v);
  };
  const double mine = range_sum(part * A.part, min(A.V, (part + 1) * A.part), false);
  double* const sums = A.sums + (int64_t)b * A.parts;
  if (tid == 0) {
    __hip_atomic_store(sums + part, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = __hip_atomic_fetch_add(A.done + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(A.parts - 1);
  }
  __syncthreads();
  if (!last) return;
  if (tid == 0) __hip_atomic_store(A.done + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");

  // the part: every wavefront looks for itself, 64 parts a round
  auto part_sum = [&](int i) {
    return i < A.parts ? __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
  };
  double total = 0.0;
  for (int i = 0; i < A.parts; i += 64) total += __shfl(dr_scan(part_sum(i + lane)), 63, 64);
  const double drawn = fmax((double)u[A.n], 0.0);
  int lo = 0, hi = 0;                                          // where the entry is
  double before = 0.0;
  const bool all = !(total > 0.0);
  if (all) {
    // Nothing is left (p below q at every entry but for rounding): p's own row, which this workgroup reads alone.
    total = range_sum(0, A.V, true);
    hi = total > 0.0 ? A.V : 0;
  } else {
    int at = -1;
    bool passed = false;
    for (int i = 0; i < A.parts; i += 64) {
      const double v = part_sum(i + lane), upto = before + dr_scan(v);
      const uint64_t pass = __ballot(upto > drawn * total && v > 0.0), some = __ballot(v > 0.0);
      if (pass) {
        const int k = __builtin_ctzll(pass);
        at = i + k;
        before = __shfl(upto - v, k, 64);
        passed = true;
        break;
      }
      if (some) at = i + 63 - __builtin_clzll(some);           // u so near 1 that no sum passes: the last one
      before = __shfl(upto, 63, 64);
    }
    if (!passed) before = -INFINITY;                           // nor does one of its entries
    lo = at * A.part;
    hi = min(A.V, lo + A.part);
  }
  const double target = drawn * total;
  if (tid == 0) found = -1;
  __syncthreads();
  if (hi > lo) {
    int best = -1;                                             // the last entry that is not 0
    for (int c = lo; c < hi; c += DR_STEP) {
      double r[DR_PER], s[LOADS], upto[LOADS];
      dr_rest<IO>(R, c, A.V, all, r);
#pragma unroll
      for (int l = 0; l < LOADS; ++l) {
        s[l] = 0.0;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          s[l] += r[l * VE + e];
          if (r[l * VE + e] > 0.0) best = c + (l * DR_THREADS + tid) * VE + e;
        }
        upto[l] = dr_scan(s[l]);
        if (lane == 63) totals[l][wave] = upto[l];
      }
      __syncthreads();
      double run = before;
      int hit = -1;
#pragma unroll
      for (int l = 0; l < LOADS; ++l)
        for (int w = 0; w < DR_THREADS / 64; ++w) {
          const double v = totals[l][w];
          if (hit < 0 && w == wave) {
            const uint64_t pass = __ballot(run + upto[l] > target && s[l] > 0.0);
            if (pass) {
              const int k = __builtin_ctzll(pass);
              if (lane == k) {
                double t = run + (upto[l] - s[l]);
                int index = -1;
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                  const bool take = r[l * VE + e] > 0.0 && (index < 0 || t <= target);
                  if (take) index = c + (l * DR_THREADS + tid) * VE + e;
                  t += r[l * VE + e];
                }
                hit = index;
              }
              hit = __shfl(hit, k, 64);
            }
          }
          run += v;
        }
      // the first wavefront's hit, in the order of the entries
      if (hit >= 0 && lane == 0) atomicMin(reinterpret_cast<unsigned int*>(&found), (unsigned)hit);
      __syncthreads();
      if (found >= 0) break;
      before = run;
    }
    if (found < 0) {                                           // uniform: read after a barrier
      __syncthreads();
      if (best >= 0) atomicMax(&found, best);
      __syncthreads();
    }
  }
  const int pick = found;
  for (int i = tid; i <= A.n; i += DR_THREADS)
    A.out[(int64_t)b * (A.n + 1) + i] = i < accepted ? tokens[i] : i == accepted ? pick : -1;
  if (tid == 0) A.accepted[b] = accepted;
}

// Parts of a row: as many as give 6 workgroups a CU, of whole steps.
static void dr_plan(int64_t batch, int64_t V, int64_t* parts, int64_t* part) {
  const int64_t steps = (V + DR_STEP - 1) / DR_STEP;
  int64_t n = (6 * (int64_t)device_cu_count() + batch - 1) / batch;
  if (n > steps) n = steps;
  const int64_t per = (steps + n - 1) / n;
  *part = per * DR_STEP;
  *parts = (steps + per - 1) / per;
}

}  // namespace pp

using namespace pp;

extern "C" int64_t pp_verify_drafts_workspace_size(int64_t batch, int64_t V) {
  if (batch <= 0 || V <= 0) return 0;
  int64_t parts, part;
  dr_plan(batch, V, &parts, &part);
  return batch * parts * 8;
}

extern "C" int pp_verify_drafts(const void* target, int64_t p_sb, int64_t p_sr, const void* draft, int64_t q_sb,
                                int64_t q_sr, int dtype, int64_t batch, int64_t n, int64_t V, const int64_t* tokens,
                                int64_t t_sb, const float* uniforms, int64_t u_sb, const int32_t* counts, int64_t* out,
                                int64_t* accepted, void* workspace, int64_t workspace_size, void* done, int64_t done_size,
                                void* stream) {
  PP_REQUIRE(dtype == PP_F16 || dtype == PP_BF16 || dtype == PP_F32, "pp_verify_drafts: dtype %d", dtype);
  PP_REQUIRE(batch >= 0 && batch <= (1 << 24), "pp_verify_drafts: batch %lld not in 0..2^24", (long long)batch);
  PP_REQUIRE(n >= 0 && n <= (1 << 16), "pp_verify_drafts: %lld drafts a sequence not in 0..2^16", (long long)n);
  PP_REQUIRE(V > 0 && V <= (1 << 30), "pp_verify_drafts: %lld probabilities a row", (long long)V);
  if (batch == 0) return PP_OK;
  PP_REQUIRE(target && uniforms && out && accepted && (tokens || n == 0), "pp_verify_drafts: null operands");
  const int es = dtype == PP_F32 ? 4 : 2;
  PP_REQUIRE(aligned(target, es) && aligned(draft, es), "pp_verify_drafts: probabilities are not aligned to their type");
  int64_t parts, part;
  dr_plan(batch, V, &parts, &part);
  PP_REQUIRE(batch * parts <= INT32_MAX, "pp_verify_drafts: too many sequences");
  PP_REQUIRE(workspace && workspace_size >= batch * parts * 8 && aligned(workspace, 8),
             "pp_verify_drafts: workspace of %lld bytes at an 8-byte boundary needed", (long long)(batch * parts * 8));
  PP_REQUIRE(done && done_size >= 4 * batch && aligned(done, 4), "pp_verify_drafts: %lld bytes of counts, zero, needed",
             (long long)(4 * batch));
  const DraftArgs A{target, n ? draft : nullptr, tokens, uniforms, counts, out, accepted, (double*)workspace, (uint32_t*)done,
                    p_sb, p_sr, q_sb, q_sr, t_sb, u_sb, (int)batch, (int)n, (int)V, (int)parts, (int)part};
  auto kern = dtype == PP_F16 ? verify_drafts_kernel<IoF16>
              : dtype == PP_BF16 ? verify_drafts_kernel<IoBf16> : verify_drafts_kernel<IoF32>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(batch * parts)), dim3(DR_THREADS), 0, (hipStream_t)stream, A);
  PP_LAUNCH_CHECK();
  return PP_OK;
}
