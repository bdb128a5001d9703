// Token scores from a row of logits: the log probability of a given token, the
// entropy of the row's distribution and its likeliest tokens, in one pass.
//
// With z = x / T, m = max z and d = z - m:
//   S = sum e^d,  U = sum e^d d
//   log p(token) = d(token) - log S,   entropy = log S - U / S
// and the alternatives are the top_k largest logits, ties to the lowest index.
// S and U are kept online (a running maximum; both are rescaled when it moves)
// in fp32, exponents in units of log2.
#include <cfloat>
#include <cstdint>

#include "common.cuh"
#include "kvcache.cuh"

namespace wx {

constexpr int kScoreThreads = 256, kScoreWarps = kScoreThreads / 32;
constexpr int kScoreMaxCtas = 8;    // CTAs (one cluster) on a row
constexpr int kScoreMaxTop = 32;    // one lane each
constexpr int kScoreVecs = 2;       // 16-byte vectors of a thread's step
constexpr int kScoreStages = 4;     // steps in flight

struct ScoreArgs {
  const void* logits;
  int64_t ld;
  const int64_t* tokens;
  float *logprob, *entropy, *top_logprob;
  int32_t* top_index;
  int64_t vocab;
  int top_k;
  float inv_t;
};

// max and the three-input max that hand NaN on
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Order of logits as unsigned integers: NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.0f);   // -0 + 0 = +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
  if (k == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// (value, lowest index first) as one number; 0 is below every entry
__device__ __forceinline__ uint64_t entry(float x, uint32_t index) {
  return ((uint64_t)order_key(x) << 32) | ~index;
}

// The running sums of one thread or of a part of a row.
struct Sums {
  float m, s, u;   // reference logit, sum 2^d, sum 2^d d (d = (logit - m) c, log2 units)
};

// x with the reference m in place of its own, m at least x.m; c = log2(e) / T
__device__ __forceinline__ Sums refer(Sums x, float m, float c) {
  // a part without weight (nothing in it, or all -inf) keeps none
  if (x.s == 0.0f) return {m, 0.0f, 0.0f};
  const float d = (x.m - m) * c, f = fast_exp2(d);
  // s d f -> 0 as f -> 0: what is too small to count adds nothing
  return {m, x.s * f, f == 0.0f ? 0.0f : (x.u + x.s * d) * f};
}
// The lanes' parts joined, a fixed tree: every lane gets the whole.
__device__ __forceinline__ float warp_max(float m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
__device__ __forceinline__ Sums join_lanes(Sums x, float c) {
  x = refer(x, warp_max(x.m), c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    x.s += __shfl_xor_sync(0xffffffffu, x.s, o);
    x.u += __shfl_xor_sync(0xffffffffu, x.u, o);
  }
  return x;
}

template <typename T>
struct Lanes;
template <>
struct Lanes<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& w, float (&v)[4]) {
    v[0] = __uint_as_float(w.x);
    v[1] = __uint_as_float(w.y);
    v[2] = __uint_as_float(w.z);
    v[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <>
struct Lanes<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& w, float (&v)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __uint_as_float(a[i] << 16);
      v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ float one(const uint16_t* p) {
    return __uint_as_float((uint32_t)*p << 16);
  }
};

__device__ __forceinline__ uint32_t cluster_peer(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float peer_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t peer_u64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void score_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}

constexpr int kCandidates = 768;

// A CTA's candidates for the alternatives, in no order, and the best of them.
struct Candidates {
  uint64_t list[kCandidates];
  uint64_t best[kScoreMaxTop];
  uint64_t part[kScoreWarps];
  uint32_t sorted[kScoreWarps][32];   // each warp's largest logits, descending
  uint32_t reach;                     // the top_k-th largest of them: top_k reach it
  int n, n_in_step, n_owners;
  // threads whose largest logit reaches it: with the one step that has it (step <<
  // 8), or, where another step's do too, for all their steps
  uint32_t in_step[kScoreThreads];
  uint8_t owners[kScoreThreads];
};

// Sets c.reach from each thread's largest logit (its order_key; 0: it has none), and
// the lists of threads that reach it: `step` has the largest, `other` is the largest
// of the other steps. Called by every thread, after a barrier; ends with one.
__device__ __forceinline__ void find_reach(Candidates& c, uint32_t key, int step, float other,
                                           int top_k) {
  const int lane = lane_id(), w = warp_id();
  int r = 0;
#pragma unroll
  for (int j = 0; j < 32; j++) {
    const uint32_t y = __shfl_sync(0xffffffffu, key, j);
    r += y > key || (y == key && j < lane);
  }
  c.sorted[w][r] = key;
  __syncthreads();
  // the CTA's top_k-th is among its warps' first top_k
  if (threadIdx.x < kScoreWarps * top_k) {
    const uint32_t mine = c.sorted[threadIdx.x / top_k][threadIdx.x % top_k];
    int above = 0;   // largest logits above this one, by a search in each warp's
#pragma unroll
    for (int u = 0; u < kScoreWarps; u++) {
      int at = 0;
#pragma unroll
      for (int step = 16; step > 0; step >>= 1)
        if (c.sorted[u][at + step - 1] > mine) at += step;
      above += at + (c.sorted[u][at] > mine ? 1 : 0);
    }
    if (above < top_k) atomicMin(&c.reach, mine);
  }
  __syncthreads();
  if (key && key >= c.reach) {
    if (order_key(other) >= c.reach)
      c.owners[atomicAdd(&c.n_owners, 1)] = (uint8_t)threadIdx.x;
    else
      c.in_step[atomicAdd(&c.n_in_step, 1)] = ((uint32_t)step << 8) | threadIdx.x;
  }
  __syncthreads();
}
static_assert(kScoreThreads <= 256, "a thread's number is kept in a byte");

// The first top_k of c.list's n <= kCandidates entries (distinct but for 0) to c.best,
// 0 past their number: an entry's place is the number of entries above it. Called by
// every thread, after a barrier; ends with one.
__device__ __forceinline__ void rank_candidates(Candidates& c, int n, int top_k) {
  if (threadIdx.x < kScoreMaxTop) c.best[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kScoreThreads) {
    const uint64_t e = c.list[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; j++) r += c.list[j] > e;
    if (e && r < top_k) c.best[r] = e;
  }
  __syncthreads();
}

// A CTA's vectors of a row: thread t's are i(it, j) + 32 j for each step it.
template <typename T>
struct Slice {
  const uint4* vec;
  int lead, v0, v1, n_steps;
  static constexpr int kStep = kScoreThreads * kScoreVecs;
  static __device__ __forceinline__ int at(int step, int j, int t) {
    return step * kStep + (t >> 5) * 32 * kScoreVecs + j * 32 + (t & 31);
  }
};

// The largest entry up to `bar`, itself included, among thread t's vectors, found by
// t's whole warp (each lane gets it). NaN at token 0 is the largest number there is.
template <typename T>
__device__ __forceinline__ uint64_t best_up_to(const Slice<T>& s, int t, uint64_t bar) {
  constexpr int N = Lanes<T>::N;
  uint64_t mx = 0;
  for (int i = lane_id(); i < s.n_steps * kScoreVecs; i += 32) {
    const int k = s.v0 + Slice<T>::at(i / kScoreVecs, i % kScoreVecs, t);
    if (k >= s.v1) continue;
    float v[N];
    Lanes<T>::unpack(s.vec[k], v);
#pragma unroll
    for (int e = 0; e < N; e++) {
      const uint64_t y = entry(v[e], (uint32_t)(s.lead + k * N + e));
      if (y <= bar && y > mx) mx = y;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t y = __shfl_xor_sync(0xffffffffu, mx, o);
    mx = y > mx ? y : mx;
  }
  return mx;
}

// c.best by taking the largest entry top_k times, for rows where too many logits
// reach the threshold (most tokens masked, long runs of equal logits): `edge` is
// an entry of the thread's own besides its vectors, or 0.
template <typename T>
__device__ __noinline__ void take_best(const Slice<T>& s, Candidates& c, int top_k,
                                       uint64_t edge) {
  const int lane = lane_id(), w = warp_id();
  uint64_t mine = 0;   // the thread's largest vector entry not yet taken
  for (int l = 0; l < 32; l++) {
    const uint64_t y = best_up_to(s, w * 32 + l, ~0ull);
    if (l == lane) mine = y;
  }
  for (int r = 0; r < top_k; r++) {
    const uint64_t own = edge > mine ? edge : mine;
    uint64_t mx = own;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t y = __shfl_xor_sync(0xffffffffu, mx, o);
      mx = y > mx ? y : mx;
    }
    if (lane == 0) c.part[w] = mx;
    __syncthreads();
    uint64_t all = 0;
    for (int u = 0; u < kScoreWarps; u++) all = c.part[u] > all ? c.part[u] : all;
    if (threadIdx.x == 0) c.best[r] = all;
    __syncthreads();
    if (all && mx == all) {   // this warp's: the lane that holds it looks for its next
      const uint32_t who = __ballot_sync(0xffffffffu, own == all && edge != all);
      if (edge == all) edge = 0;
      if (who) {
        const int l = __ffs(who) - 1;
        const uint64_t y = best_up_to(s, w * 32 + l, all - 1);
        if (l == lane) mine = y;
      }
    }
  }
  __syncthreads();
}

// Row blockIdx.y by a cluster of gridDim.x CTAs, each a contiguous part of it.
//
// A thread takes kScoreVecs 16-byte vectors a step, copied kScoreStages - 1 steps
// ahead into shared memory; the warp shares the reference of its sums. For the
// alternatives the pass keeps each thread's largest logit, its step, and the largest
// of the other steps. The top_k-th of the threads' largest is a logit that top_k reach,
// so the alternatives are among the logits of the few threads whose largest reaches
// it: that step, or all of theirs where another reaches it too, is gone over again
// (from shared memory or L2), and the logits that reach it are listed and put in order
// by counting ranks. The parts are joined in shared memory, then over the cluster's.
//
// Measured (B200): 2048 rows of 100003 bf16 logits (410 MB) 70 us without and 80 us
// with 5 alternatives (5.8 and 5.1 TB/s), bound by the issue of some seven
// instructions a logit, one of them the exponential; 1024 such rows of fp32 67 us
// without, 78 with 20 (6.1 and 5.3 TB/s), near the memory's bandwidth. 5 rows of 50001
// fp32 with 10 alternatives 7.5 us (4.4 without), bound by the latency of the steps
// after the pass. Sorted lists that every warp kept through the pass took 115 us where
// this takes 80: a newcomer cost a warp some 300 cycles. CTAs that stay for several
// rows and read ahead took 95 against 88 (3.5 rows a CTA leave a round half empty).
template <typename T, bool TOP>
__global__ void __launch_bounds__(kScoreThreads, 4) token_score_kernel(const ScoreArgs a) {
  constexpr int N = Lanes<T>::N;
  __shared__ Sums sums[kScoreWarps];
  __shared__ Sums cta_sums;
  __shared__ uint4 ring[kScoreStages][kScoreVecs][kScoreThreads];
  __shared__ Candidates cand;
  const int lane = lane_id(), w = warp_id();
  const int rank = blockIdx.x, n_ctas = gridDim.x;
  const int64_t row = blockIdx.y;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const float c = 1.4426950408889634f * a.inv_t;
  pdl_wait();

  // the elements before the first and past the last whole vector are left for the
  // end
  Slice<T> s;
  s.lead = (int)min(a.vocab, (int64_t)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
  const int n_vec = (int)((a.vocab - s.lead) / N);
  s.vec = reinterpret_cast<const uint4*>(x + s.lead);
  s.v0 = (int)((int64_t)n_vec * rank / n_ctas);
  s.v1 = (int)((int64_t)n_vec * (rank + 1) / n_ctas);
  s.n_steps = (s.v1 - s.v0 + Slice<T>::kStep - 1) / Slice<T>::kStep;
  // each thread copies its vectors ahead into slots that only it reads
  auto fetch = [&](int it) {
#pragma unroll
    for (int j = 0; j < kScoreVecs; j++) {
      const int i = s.v0 + Slice<T>::at(it, j, threadIdx.x);
      if (i < s.v1)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         smem_u32(&ring[it % kScoreStages][j][threadIdx.x])),
                     "l"(s.vec + i)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int it = 0; it < kScoreStages - 1; it++) fetch(it);
  if (TOP && threadIdx.x == 0) {
    cand.reach = 0xFFFFFFFFu;
    cand.n = cand.n_in_step = cand.n_owners = 0;
  }

  float m = -INFINITY;
  float2 s2 = {0.0f, 0.0f}, u2 = {0.0f, 0.0f};
  // the thread's largest logit, its step, and the largest of its other steps
  float largest = -INFINITY, other = -INFINITY;
  int largest_step = 0;
  // the reference moves to the warp's maximum where a logit passes it by more than
  // 2^8 in weight: once or twice a row, since the warp's lanes share it
  const float slack = 8.0f / c;
  auto raise = [&](float vm) {
    if (!__any_sync(0xffffffffu, !(vm <= m + slack))) return;
    const float to = max_nan(m, warp_max(vm));
    const Sums x = refer({m, s2.x, u2.x}, to, c), y = refer({m, s2.y, u2.y}, to, c);
    s2 = {x.s, y.s};
    u2 = {x.u, y.u};
    m = to;
  };

#pragma unroll 1
  for (int it = 0; it < s.n_steps; it++) {
    fetch(it + kScoreStages - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kScoreStages - 1) : "memory");
    float v[kScoreVecs][N];
#pragma unroll
    for (int j = 0; j < kScoreVecs; j++)
      Lanes<T>::unpack(ring[it % kScoreStages][j][threadIdx.x], v[j]);
    if (it + 1 == s.n_steps) {
#pragma unroll
      for (int j = 0; j < kScoreVecs; j++)
        if (s.v0 + Slice<T>::at(it, j, threadIdx.x) >= s.v1) {
#pragma unroll
          for (int e = 0; e < N; e++) v[j][e] = -INFINITY;
        }
    }
    float vm = v[0][0];
#pragma unroll
    for (int j = 0; j < kScoreVecs; j++)
#pragma unroll
      for (int e = 0; e < N; e += 2) vm = max_nan(vm, v[j][e], v[j][e + 1]);
    if (TOP) {
      const bool up = vm > largest;   // NaN: among the others, and so gone over
      other = max_nan(other, up ? largest : vm);
      largest_step = up ? it : largest_step;
      largest = up ? vm : largest;
    }
    raise(vm);
    const float ref = m == -INFINITY ? 0.0f : m;
    const float2 neg = {-ref, -ref}, c2 = {c, c};
#pragma unroll
    for (int j = 0; j < kScoreVecs; j++)
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        float2 d = __fmul2_rn(__fadd2_rn(make_float2(v[j][e], v[j][e + 1]), neg), c2);
        // the bound keeps d finite where its power is 0 (a masked logit)
        d.x = max_nan(d.x, -1e4f);
        d.y = max_nan(d.y, -1e4f);
        const float2 p = {fast_exp2(d.x), fast_exp2(d.y)};
        s2 = __fadd2_rn(s2, p);
        u2 = __ffma2_rn(p, d, u2);
      }
  }
  pdl_launch_dependents();
  // the row's edges
  uint64_t edge = 0;
  if (rank == 0 && w == 0) {
    const int tail = s.lead + n_vec * N + lane - 16;
    const bool is = lane < 16 ? lane < s.lead : tail < a.vocab;
    const int at = lane < 16 ? lane : tail;
    const float y = is ? Lanes<T>::one(x + at) : -INFINITY;
    raise(y);
    const float d = max_nan((y - (m == -INFINITY ? 0.0f : m)) * c, -1e4f), p = fast_exp2(d);
    s2.x += p;
    u2.x = fmaf(p, d, u2.x);
    if (is) edge = entry(y, (uint32_t)at);
  }

  // the warp's, the CTA's, the row's
  Sums acc = join_lanes({m, s2.x + s2.y, u2.x + u2.y}, c);
  if (lane == 0) sums[w] = acc;
  __syncthreads();   // reach, n and n_owners are set too
  if (w == 0) {
    acc = join_lanes(lane < kScoreWarps ? sums[lane] : Sums{-INFINITY, 0.0f, 0.0f}, c);
    if (lane == 0) cta_sums = acc;
  }
  if (TOP) {
    const bool has = s.v0 + Slice<T>::at(0, 0, threadIdx.x) < s.v1;
    find_reach(cand, has ? order_key(max_nan(largest, other)) : 0, largest_step, other, a.top_k);
    const uint32_t reach = cand.reach;
    auto list = [&](uint64_t e) {
      const int at = atomicAdd(&cand.n, 1);
      if (at < kCandidates) cand.list[at] = e;
    };
    if (edge && (uint32_t)(edge >> 32) >= reach) list(edge);
    // vector j of thread t's step it; what is left in the ring is there
    const bool in_ring = s.n_steps <= kScoreStages;
    auto go_over = [&](int it, int j, int t) {
      const int k = s.v0 + Slice<T>::at(it, j, t);
      if (k >= s.v1) return;
      float v[N];
      Lanes<T>::unpack(in_ring ? ring[it][j][t] : s.vec[k], v);
      float vm = v[0];
#pragma unroll
      for (int e = 0; e < N; e += 2) vm = max_nan(vm, v[e], v[e + 1]);
      if (order_key(vm) < reach) return;
#pragma unroll
      for (int e = 0; e < N; e++) {
        const uint32_t y = order_key(v[e]);
        if (y >= reach) list(((uint64_t)y << 32) | ~(uint32_t)(s.lead + k * N + e));
      }
    };
    // dealt out over the CTA: the threads' one step, and all steps of the few others
    const int n_one = cand.n_in_step * kScoreVecs, per = s.n_steps * kScoreVecs;
    const int n_all = n_one + cand.n_owners * per;
#pragma unroll 1
    for (int i = threadIdx.x; i < n_all; i += kScoreThreads) {
      const int u = i < n_one ? 0 : (i - n_one) / per, f = i < n_one ? i : i - n_one - u * per;
      const uint32_t o = i < n_one ? cand.in_step[i / kScoreVecs]
                                   : (uint32_t)(f / kScoreVecs) << 8 | cand.owners[u];
      go_over((int)(o >> 8), f % kScoreVecs, (int)(o & 255));
    }
    __syncthreads();
    if (cand.n <= kCandidates)
      rank_candidates(cand, cand.n, a.top_k);
    else
      take_best(s, cand, a.top_k, edge);
  }
  if (n_ctas > 1) {
    score_cluster_sync();
    if (rank == 0) {
      if (w == 0) {
        const uint32_t p = cluster_peer(&cta_sums, lane < n_ctas ? lane : 0);
        acc = {peer_f32(p), peer_f32(p + 4), peer_f32(p + 8)};
        acc = join_lanes(lane < n_ctas ? acc : Sums{-INFINITY, 0.0f, 0.0f}, c);
      }
      // CTA u's list by warp u
      if (TOP && w < n_ctas && lane < a.top_k)
        cand.list[w * a.top_k + lane] = peer_u64(cluster_peer(cand.best + lane, w));
    }
    // a CTA's shared memory outlives its readers, whose values are in use by now:
    // nothing is handed over
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;"
                 ::: "memory");
    if (rank != 0) return;
    if (TOP) rank_candidates(cand, n_ctas * a.top_k, a.top_k);
  }
  if (rank != 0 || w != 0) return;

  const bool empty = acc.m == -INFINITY;   // every token is masked
  const float log_s = logf(acc.s);
  auto logprob = [&](float v) { return empty ? -INFINITY : (v - acc.m) * a.inv_t - log_s; };
  if (lane == 0) {
    if (a.logprob) {
      const int64_t t = a.tokens[row];
      a.logprob[row] = t < 0 ? 0.0f : t >= a.vocab ? -INFINITY : logprob(Lanes<T>::one(x + t));
    }
    if (a.entropy)
      a.entropy[row] = empty ? 0.0f : log_s - 0.6931471805599453f * (acc.u / acc.s);
  }
  if (TOP && lane < a.top_k) {
    const uint64_t e = cand.best[lane];
    a.top_logprob[row * a.top_k + lane] = logprob(order_value((uint32_t)(e >> 32)));
    a.top_index[row * a.top_k + lane] = (int32_t)~(uint32_t)e;
  }
}
static_assert(kScoreMaxCtas <= kScoreWarps, "a CTA's list for each warp of the first");
static_assert(kScoreMaxCtas * kScoreMaxTop <= kCandidates, "");

template <typename T, bool TOP>
static cudaError_t launch_score(const ScoreArgs& a, int ctas, int64_t rows, cudaStream_t st) {
  return launch_after(token_score_kernel<T, TOP>, dim3((unsigned)ctas, (unsigned)rows),
                      kScoreThreads, 0, ctas, st, a);
}

}  // namespace wx

extern "C" int wx_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab,
                                 int64_t ld, const int64_t* tokens, int64_t top_k,
                                 float temperature, float* logprob, float* entropy,
                                 float* top_logprob, int32_t* top_index, void* stream) {
  using namespace wx;
  if (dtype != WX_DTYPE_BF16 && dtype != WX_DTYPE_F32)
    return fail(WX_ERR_INVALID, "token_logprobs: bad dtype %d", dtype);
  if (rows < 0 || vocab < 1 || vocab > 0x7fffffff || (rows > 1 && ld < vocab))
    return fail(WX_ERR_INVALID, "token_logprobs: bad shape %lld x %lld, row stride %lld",
                (long long)rows, (long long)vocab, (long long)ld);
  if (top_k < 0 || top_k > kScoreMaxTop || top_k > vocab)
    return fail(WX_ERR_INVALID, "token_logprobs: top_k %lld not in [0, min(%d, vocabulary)]",
                (long long)top_k, kScoreMaxTop);
  // the kernel's factor, log2(e) / temperature, has to be finite too
  if (!(temperature > 0.0f) || !(1.4426950408889634f * (1.0f / temperature) <= FLT_MAX) ||
      !(temperature <= FLT_MAX))
    return fail(WX_ERR_INVALID, "token_logprobs: temperature must be positive and finite");
  if (rows == 0) return WX_OK;
  const int es = dtype == WX_DTYPE_BF16 ? 2 : 4;
  if (!logits || ((uintptr_t)logits % es))
    return fail(WX_ERR_INVALID, "token_logprobs: logits NULL or not aligned to their type");
  if (logprob && !tokens)
    return fail(WX_ERR_INVALID, "token_logprobs: log probabilities asked for without tokens");
  if (top_k && (!top_logprob || !top_index))
    return fail(WX_ERR_INVALID, "token_logprobs: top_k without its outputs");
  ScoreArgs a = {logits, ld,    tokens,     logprob, entropy, top_logprob, top_index,
                 vocab,  (int)top_k, 1.0f / temperature};
  // rows alone fill the GPU from two CTAs an SM on; below that a row is split (320 rows
  // of 50001 logits: 17 us whole, 21 in two parts, whose ends cost as much as they save)
  int ctas = 1;
  while (ctas < kScoreMaxCtas && rows * ctas < 2 * sm_count() &&
         vocab * es / (2 * ctas) >= kScoreThreads * 16)
    ctas *= 2;
  cudaStream_t st = as_stream(stream);
  constexpr int64_t kMaxGridY = 65535;
  for (int64_t r = 0; r < rows; r += kMaxGridY) {
    const int64_t n = rows - r < kMaxGridY ? rows - r : kMaxGridY;
    cudaError_t e;
    if (es == 2)
      e = top_k ? launch_score<uint16_t, true>(a, ctas, n, st)
                : launch_score<uint16_t, false>(a, ctas, n, st);
    else
      e = top_k ? launch_score<float, true>(a, ctas, n, st)
                : launch_score<float, false>(a, ctas, n, st);
    WX_CUDA_TRY(e);
    a.logits = static_cast<const char*>(a.logits) + n * ld * es;
    if (a.tokens) a.tokens += n;
    if (a.logprob) a.logprob += n;
    if (a.entropy) a.entropy += n;
    if (a.top_logprob) a.top_logprob += n * top_k;
    if (a.top_index) a.top_index += n * top_k;
  }
  return check_launch("token_logprobs");
}
