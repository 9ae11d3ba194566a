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
// trips: tokens, then their probabilities), leaves the sum of every 1024 entries in the workspace, and counts itself
// done; of the one that counts last a wavefront finds the 1024 in which the sum passes, reads those again and finds
// the token.  One launch, and the order of the sums is fixed.
//
// What bounds it: the reading, where there are many sequences: 128 of 5 drafts over 151,936 float32 probabilities (150 MB
// where every sequence refuses one) 29 us, of which finding the row is 3 and the last 1024 entries 4; 8 workgroups a CU
// against 6 29.1 / 29.4, 12 31.9, 20 44.  4 sequences 9.6 us, the chain of six round trips.  Rows that do not begin at a 16-byte
// boundary, most of an odd vocabulary's, are read an entry a load: 128 sequences of 5 random drafts over 151,935 56 us in float32 and 49 in
// bf16, where 151,936 take 34 and 25; without a draft's probabilities 31 and 31, 26 and 21.
#include "kv_common.h"

namespace pp {

constexpr int DR_THREADS = 256;
constexpr int DR_PER = 16;                          // entries a lane and chunk
constexpr int DR_CHUNK = 64 * DR_PER;
constexpr int DR_STEP = DR_THREADS * DR_PER;        // a chunk for each wavefront

struct DraftArgs {
  const void* p;
  const void* q;          // null: the drafts were certain
  const int64_t* tokens;
  const float* u;
  const int32_t* counts;  // null: n of every sequence
  int64_t* out;
  int64_t* accepted;
  double* sums;           // [sequence][chunk]: of r
  uint32_t* done;         // [sequence]: parts that are done; 0 before and after
  int64_t p_sb, p_sr, q_sb, q_sr, t_sb, u_sb;
  int batch, n, V, parts, part;       // `part` entries a part, a multiple of DR_STEP
  int chunks;
};

// What counts as a probability: NaN and what is below 0 as 0, infinity as the largest float.
__device__ __forceinline__ float dr_clean(float x) { return __builtin_amdgcn_fmed3f(x, 0.f, 3.40282347e38f); }

// A lane's entries of the chunk at c: c + (64 l + lane) * VE + 0 .. VE - 1 for l = 0 .. LOADS - 1, as they lie in
// memory, zeros past V.
template <typename IO>
struct DraftWords {
  static constexpr int VE = 16 / sizeof(typename IO::raw), LOADS = DR_PER / VE;
  u32x4 w[LOADS];
  __device__ __forceinline__ void load(const typename IO::raw* x, int c, int V) {
    const int lane = threadIdx.x & 63;
    if (reinterpret_cast<uintptr_t>(x) % 16 == 0 && c + DR_CHUNK <= V) {     // the same in every lane
#pragma unroll
      for (int l = 0; l < LOADS; ++l) w[l] = *reinterpret_cast<const u32x4*>(x + c + (64 * l + lane) * VE);
      return;
    }
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const int at = c + (64 * l + lane) * VE;
      typename IO::raw e[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) e[i] = at + i < V ? x[at + i] : (typename IO::raw)0;
      __builtin_memcpy(&w[l], e, 16);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    typename IO::raw e[VE];
    __builtin_memcpy(e, &w[i / VE], 16);
    return dr_clean(IO::get(e[i % VE]));
  }
};

// The row that is drawn from: p less q, or p but for one entry.
template <typename IO>
struct DraftRow {
  const typename IO::raw* p;
  const typename IO::raw* q;    // null: nothing to take off but `without`
  int without;                  // an entry that counts 0, or -1
  struct Step {
    DraftWords<IO> p, q;
  };
  __device__ __forceinline__ void load(Step& S, int c, int V) const {
    S.p.load(p, c, V);
    if (q) S.q.load(q, c, V);
  }
  __device__ __forceinline__ void rest(const Step& S, int c, double* r) const {
    constexpr int VE = DraftWords<IO>::VE;
    if (q) {
#pragma unroll
      for (int i = 0; i < DR_PER; ++i) {
        const float x = S.q.get(i);
        r[i] = (double)fmaxf(S.p.get(i), x) - (double)x;
      }
    } else {
#pragma unroll
      for (int i = 0; i < DR_PER; ++i)
        r[i] = c + (64 * (i / VE) + (int)(threadIdx.x & 63)) * VE + i % VE == without ? 0.0 : (double)S.p.get(i);
    }
  }
};

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
  __shared__ uint32_t last;
  const int b = blockIdx.x / A.parts, part = blockIdx.x - b * A.parts;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const raw* const p = reinterpret_cast<const raw*>(A.p) + b * A.p_sb;
  const raw* const q = A.q ? reinterpret_cast<const raw*>(A.q) + b * A.q_sb : nullptr;
  const int64_t* const tokens = A.tokens + b * A.t_sb;
  const float* const u = A.u + b * A.u_sb;

  // every wavefront looks at 64 drafts a round
  const int count = A.counts ? min(max(A.counts[b], 0), A.n) : A.n;
  int accepted = count;
  for (int i0 = 0; i0 < count; i0 += 64) {
    const int i = i0 + lane;
    bool bad = false;
    if (i < count) {
      const int64_t t = tokens[i];
      const bool in = t >= 0 && t < A.V;
      const float pd = in ? dr_clean(IO::get(p[i * A.p_sr + t])) : 0.f;
      const float qd = !q ? 1.f : in ? dr_clean(IO::get(q[i * A.q_sr + t])) : 0.f;
      bad = !((double)u[i] * (double)qd < (double)pd);
    }
    const uint64_t mask = __ballot(bad);
    if (mask) {
      accepted = i0 + __builtin_ctzll(mask);
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

  // The wavefront's chunks lo, lo + by .. of W; the entries of one are on their way while those of the one before are
  // added.
  auto sum_chunks = [&](const DraftRow<IO>& W, int lo, int hi, int by, auto done) {
    typename DraftRow<IO>::Step now, next;
    W.load(now, lo, A.V);
    for (int c = lo; c < hi; c += by) {
      if (c + by < hi) W.load(next, c + by, A.V);
      double r[DR_PER], v = 0.0;
      W.rest(now, c, r);
#pragma unroll
      for (int i = 0; i < DR_PER; ++i) v += r[i];
      done(c, dr_sum(v));
      now = next;
    }
  };
  double* const sums = A.sums + (int64_t)b * A.chunks;
  auto put = [&](int c, double v) {
    if (lane == 0) __hip_atomic_store(sums + c / DR_CHUNK, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  const int begin = part * A.part + wave * DR_CHUNK, end = min(A.V, (part + 1) * A.part);
  if (begin < end) sum_chunks(R, begin, end, DR_STEP, put);
  // Sums go to memory past the caches that other XCDs do not see, are waited for before the count goes up, and are
  // read past them too: nothing else that another workgroup wrote is read, so no cache is emptied (which costs
  // 10 us where 128 sequences end while others still read: 46 -> 36).
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) last = __hip_atomic_fetch_add(A.done + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(A.parts - 1);
  __syncthreads();
  if (!last || wave != 0) return;
  if (lane == 0) __hip_atomic_store(A.done + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  auto chunk_sum = [&](int i) {
    return i < A.chunks ? __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
  };
  auto total_of = [&]() {
    double v = 0.0;
    for (int i = 0; i < A.chunks; i += 64) v += __shfl(dr_scan(chunk_sum(i + lane)), 63, 64);
    return v;
  };
  const double drawn = fmax((double)u[A.n], 0.0);
  double total = total_of();
  if (!(total > 0.0)) {
    // Nothing is left (p below q at every entry but for rounding): p's own row, which this wavefront sums alone.
    R.q = nullptr;
    R.without = -1;
    sum_chunks(R, 0, A.V, DR_CHUNK, put);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    total = total_of();
  }
  const double target = drawn * total;
  int pick = -1, at = -1;
  double before = 0.0;
  bool passed = false;
  for (int i = 0; i < A.chunks && !passed; i += 64) {
    const double v = chunk_sum(i + lane), upto = before + dr_scan(v);
    const uint64_t pass = __ballot(upto > target && v > 0.0), some = __ballot(v > 0.0);
    passed = pass != 0;
    if (passed) {
      at = i + __builtin_ctzll(pass);
      before = __shfl(upto - v, at - i, 64);
    } else {
      if (some) at = i + 63 - __builtin_clzll(some);           // u so near 1 that no sum passes: the last one
      before = __shfl(upto, 63, 64);
    }
  }
  if (at >= 0) {
    const int c = at * DR_CHUNK;
    double r[DR_PER], run = passed ? before : -INFINITY;       // where no sum passes, none of its entries does
    typename DraftRow<IO>::Step S;
    R.load(S, c, A.V);
    R.rest(S, c, r);
    int best = -1;                                             // the last entry that is not 0
    bool found = false;
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      double s = 0.0;
#pragma unroll
      for (int e = 0; e < VE; ++e) s += r[l * VE + e];
      const double upto = dr_scan(s);
      const uint64_t pass = __ballot(run + upto > target && s > 0.0);
      int index = -1;                                          // the lane's entry that passes, or its last
      double t = run + (upto - s);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        if (r[l * VE + e] > 0.0 && (index < 0 || !pass || t <= target)) index = c + (64 * l + lane) * VE + e;
        t += r[l * VE + e];
      }
      if (!found && pass) {
        found = true;
        pick = __shfl(index, __builtin_ctzll(pass), 64);
      }
      best = max(best, index);
      run += __shfl(upto, 63, 64);
    }
    if (!found) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) best = max(best, __shfl_xor(best, o, 64));
      pick = best;
    }
  }
  for (int i = lane; i <= A.n; i += 64)
    A.out[(int64_t)b * (A.n + 1) + i] = i < accepted ? tokens[i] : i == accepted ? pick : -1;
  if (lane == 0) A.accepted[b] = accepted;
}

// Parts of a row: as many as give 8 workgroups a CU, of whole steps.
static void dr_plan(int64_t batch, int64_t V, int64_t* parts, int64_t* part) {
  const int64_t steps = (V + DR_STEP - 1) / DR_STEP;
  int64_t n = (8 * (int64_t)device_cu_count() + batch - 1) / batch;
  if (n > steps) n = steps;
  const int64_t per = (steps + n - 1) / n;
  *part = per * DR_STEP;
  *parts = (steps + per - 1) / per;
}

static int64_t dr_chunks(int64_t V) { return (V + DR_CHUNK - 1) / DR_CHUNK; }

}  // namespace pp

using namespace pp;

extern "C" int64_t pp_verify_drafts_workspace_size(int64_t batch, int64_t V) {
  if (batch <= 0 || V <= 0) return 0;
  return batch * dr_chunks(V) * 8;
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
  const int64_t need = batch * dr_chunks(V) * 8;
  PP_REQUIRE(workspace && workspace_size >= need && aligned(workspace, 8),
             "pp_verify_drafts: workspace of %lld bytes at an 8-byte boundary needed", (long long)need);
  PP_REQUIRE(done && done_size >= 4 * batch && aligned(done, 4), "pp_verify_drafts: %lld bytes of counts, zero, needed",
             (long long)(4 * batch));
  const DraftArgs A{target, n ? draft : nullptr, tokens, uniforms, counts, out, accepted, (double*)workspace, (uint32_t*)done,
                    p_sb, p_sr, q_sb, q_sr, t_sb, u_sb, (int)batch, (int)n, (int)V, (int)parts, (int)part,
                    (int)dr_chunks(V)};
  auto kern = dtype == PP_F16 ? verify_drafts_kernel<IoF16>
              : dtype == PP_BF16 ? verify_drafts_kernel<IoBf16> : verify_drafts_kernel<IoF32>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(batch * parts)), dim3(DR_THREADS), 0, (hipStream_t)stream, A);
  PP_LAUNCH_CHECK();
  return PP_OK;
}
