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

namespace wx {

constexpr int kScoreThreads = 256, kScoreWarps = kScoreThreads / 32;
constexpr int kScoreMaxCtas = 8;    // CTAs (one cluster) on a row
constexpr int kScoreMaxTop = 32;    // one lane each
constexpr int kScoreVecs = 2;       // 16-byte vectors of a thread's step
constexpr int kScoreStages = 5;     // steps in flight

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
  float m, s, u;   // maximum logit, sum 2^d, sum 2^d d (d in log2 units)
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

// The warp's best entries, one a lane, best first; the first top_k count.
struct TopList {
  uint64_t mine = 0;   // this lane's entry
  uint64_t last = 0;   // entry top_k - 1: what a newcomer has to beat

  // each lane's x, sorted: the list's first contents
  __device__ __forceinline__ void start(uint64_t x, int top_k) {
    const int lane = lane_id();
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
      for (int j = k >> 1; j > 0; j >>= 1) {
        const uint64_t y = __shfl_xor_sync(0xffffffffu, x, j);
        const bool keep_max = ((lane & k) == 0) == ((lane & j) == 0);
        x = keep_max == (x > y) ? x : y;
      }
    mine = x;
    last = __shfl_sync(0xffffffffu, mine, top_k - 1);
  }
  // x (the same in all lanes) takes its place
  __device__ __forceinline__ void insert(uint64_t x, int top_k) {
    const int lane = lane_id();
    const uint64_t up = __shfl_up_sync(0xffffffffu, mine, 1);
    const int at = __popc(__ballot_sync(0xffffffffu, mine > x));
    if (lane == at) mine = x;
    if (lane > at) mine = up;
    last = __shfl_sync(0xffffffffu, mine, top_k - 1);
  }
  // each lane's x where it beats the list
  __device__ __forceinline__ void offer(uint64_t x, int top_k) {
    uint32_t who = __ballot_sync(0xffffffffu, x > last);
    while (who) {
      const int from = __ffs(who) - 1;
      insert(__shfl_sync(0xffffffffu, x, from), top_k);
      who &= who - 1;
      who &= __ballot_sync(0xffffffffu, x > last);
    }
  }
};

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

// The first top_k of n entries (n <= kScoreThreads, distinct but for 0) in order:
// every thread counts the entries above its own. Called by the whole CTA.
__device__ __forceinline__ void rank_entries(const uint64_t* from, int n, int top_k,
                                             uint64_t* to) {
  const int t = threadIdx.x;
  if (t < n) {
    const uint64_t x = from[t];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < n; i++) rank += from[i] > x;
    if (x && rank < top_k) to[rank] = x;
  }
}

// Row blockIdx.y by a cluster of gridDim.x CTAs, each a contiguous part of it.
//
// A thread takes kScoreVecs 16-byte vectors a step, copied kScoreStages - 1 steps
// ahead into shared memory, and rescales its sums when its
// own maximum moves. A warp's list starts as its lanes' first maxima, sorted. From
// then on a vector is looked into only if its largest logit passes the list's last
// one and is not below `bound`, the CTA's top_k-th logit so far, which the lists
// are joined for after steps 1, 4, 16 and so on: about top_k logits of a row pass
// each time the logits seen have grown fourfold. The parts are joined in shared
// memory, then over the cluster's, the lists by counting ranks.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kScoreThreads) token_score_kernel(const ScoreArgs a) {
  constexpr int N = Lanes<T>::N;
  __shared__ Sums sums[kScoreWarps];
  __shared__ Sums cta_sums;
  __shared__ uint64_t lists[kScoreThreads];   // of kScoreWarps warps or kScoreMaxCtas CTAs
  __shared__ uint64_t cta_list[kScoreMaxTop], best[kScoreMaxTop];
  __shared__ uint4 ring[kScoreStages][kScoreVecs][kScoreThreads];
  static_assert(kScoreMaxCtas * kScoreMaxTop <= kScoreThreads && kScoreMaxCtas <= 32, "");
  const int lane = lane_id(), w = warp_id();
  const int rank = blockIdx.x, n_ctas = gridDim.x;
  const int64_t row = blockIdx.y;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const float c = 1.4426950408889634f * a.inv_t;
  if (TOP) {
    if (threadIdx.x < kScoreMaxTop) cta_list[threadIdx.x] = best[threadIdx.x] = 0;
    __syncthreads();
  }

  float m = -INFINITY;
  float2 s2 = {0.0f, 0.0f}, u2 = {0.0f, 0.0f};
  // the warp's maximum becomes that of vm where it is larger: seldom after a few
  // steps, since the warp's lanes share it
  auto raise = [&](float vm) {
    if (!__any_sync(0xffffffffu, !(vm <= m))) return;
    const float to = max_nan(m, warp_max(vm));
    const Sums x = refer({m, s2.x, u2.x}, to, c), y = refer({m, s2.y, u2.y}, to, c);
    s2 = {x.s, y.s};
    u2 = {x.u, y.u};
    m = to;
  };
  TopList top;
  // a logit is looked at unless it is <= pass: the list's last one, since later
  // steps have higher indices and an equal logit comes after, or just below the
  // CTA's top_k-th so far, since against other warps it may come before
  float pass = -INFINITY;
  uint32_t floor = 0;        // order_key of the CTA's top_k-th logit so far
  auto set_pass = [&](bool equals) {
    const uint32_t own = (uint32_t)(top.last >> 32);
    uint32_t k = max(own - (equals && own ? 1 : 0), floor ? floor - 1 : 0);
    if (k == 0x7FFFFFFFu) k--;   // -0, which compares equal to the 0 above it
    pass = k ? order_value(k) : __uint_as_float(0x7FC00000u);   // NaN: everything passes
  };

  // the elements before the first and past the last whole vector: `edges`, at the
  // end, by the first CTA's first warp
  const int lead = (int)min(a.vocab, (int64_t)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
  const int n_vec = (int)((a.vocab - lead) / N);
  const uint4* xv = reinterpret_cast<const uint4*>(x + lead);
  const int v0 = (int)((int64_t)n_vec * rank / n_ctas);
  const int v1 = (int)((int64_t)n_vec * (rank + 1) / n_ctas);
  constexpr int kStep = kScoreThreads * kScoreVecs;
  const int n_steps = (v1 - v0 + kStep - 1) / kStep;
  // each thread copies its vectors ahead into slots that only it reads
  auto fetch = [&](int it) {
    const int i = v0 + it * kStep + w * 32 * kScoreVecs + lane;
#pragma unroll
    for (int j = 0; j < kScoreVecs; j++)
      if (i + j * 32 < v1)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         smem_u32(&ring[it % kScoreStages][j][threadIdx.x])),
                     "l"(xv + i + j * 32)
                     : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int it = 0; it < kScoreStages - 1; it++) fetch(it);
  int refresh = 1;
  for (int it = 0; it < n_steps; it++) {
    // a warp's vectors of a step lie side by side, so its indices only grow
    const int i = v0 + it * kStep + w * 32 * kScoreVecs + lane;
    fetch(it + kScoreStages - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kScoreStages - 1) : "memory");
    float v[kScoreVecs][N], vmax[kScoreVecs];
#pragma unroll
    for (int j = 0; j < kScoreVecs; j++)
      Lanes<T>::unpack(ring[it % kScoreStages][j][threadIdx.x], v[j]);
    if (it + 1 == n_steps) {
#pragma unroll
      for (int j = 0; j < kScoreVecs; j++)
        if (i + j * 32 >= v1) {
#pragma unroll
          for (int e = 0; e < N; e++) v[j][e] = -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < kScoreVecs; j++) {
      vmax[j] = max_nan(v[j][0], v[j][1]);
#pragma unroll
      for (int e = 2; e < N; e += 2) vmax[j] = max_nan(vmax[j], v[j][e], v[j][e + 1]);
    }
    float vm = vmax[0];
#pragma unroll
    for (int j = 1; j < kScoreVecs; j++) vm = max_nan(vm, vmax[j]);
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
    if (!TOP) continue;

    const uint32_t at0 = (uint32_t)lead + (uint32_t)i * N;   // vector j: + 32 N j
    uint32_t own = 0xFFFFFFFFu;   // the lane's entry of the list's start
    if (it == 0) {
      bool got = false;
#pragma unroll
      for (int j = 0; j < kScoreVecs; j++)
#pragma unroll
        for (int e = 0; e < N; e++)
          if (!got && (v[j][e] == vm || v[j][e] != v[j][e])) {
            got = true;
            own = at0 + 32 * N * j + e;
          }
      top.start(i < v1 ? entry(vm, own) : 0, a.top_k);
    }
    if (it == 0) set_pass(true);
    if (__any_sync(0xffffffffu, !(vm <= pass))) {
#pragma unroll
      for (int j = 0; j < kScoreVecs; j++) {
        if (!__any_sync(0xffffffffu, !(vmax[j] <= pass))) continue;
        const bool valid = i + j * 32 < v1;
#pragma unroll
        for (int e = 0; e < N; e++) {
          const uint32_t at = at0 + 32 * N * j + e;
          const bool in = valid && at != own && !(v[j][e] <= pass);
          if (__any_sync(0xffffffffu, in)) {
            top.offer(in ? entry(v[j][e], at) : 0, a.top_k);
            set_pass(it == 0);
          }
        }
      }
    }
    if (it == 0) set_pass(false);
    if (it + 1 == refresh && it + 1 < n_steps) {
      refresh *= 4;
      if (lane < a.top_k) lists[w * a.top_k + lane] = top.mine;
      __syncthreads();
      rank_entries(lists, kScoreWarps * a.top_k, a.top_k, best);
      __syncthreads();
      floor = (uint32_t)(best[a.top_k - 1] >> 32);
      set_pass(false);
    }
  }
  if (rank == 0 && w == 0) {
    const int tail = lead + n_vec * N + lane - 16;
    const bool is = lane < 16 ? lane < lead : tail < a.vocab;
    const int at = lane < 16 ? lane : tail;
    const float y = is ? Lanes<T>::one(x + at) : -INFINITY;
    raise(y);
    const float d = max_nan((y - (m == -INFINITY ? 0.0f : m)) * c, -1e4f), p = fast_exp2(d);
    s2.x += p;
    u2.x = fmaf(p, d, u2.x);
    if (TOP) top.offer(is ? entry(y, (uint32_t)at) : 0, a.top_k);
  }

  // the warp's, the CTA's, the row's
  Sums acc = join_lanes({m, s2.x + s2.y, u2.x + u2.y}, c);
  if (lane == 0) sums[w] = acc;
  if (TOP && lane < a.top_k) lists[w * a.top_k + lane] = top.mine;
  __syncthreads();
  if (w == 0) {
    acc = join_lanes(lane < kScoreWarps ? sums[lane] : Sums{-INFINITY, 0.0f, 0.0f}, c);
    if (lane == 0) cta_sums = acc;
  }
  if (TOP) rank_entries(lists, kScoreWarps * a.top_k, a.top_k, n_ctas > 1 ? cta_list : best);
  if (n_ctas > 1) {
    score_cluster_sync();
    if (rank == 0) {
      if (w == 0) {
        const uint32_t p = cluster_peer(&cta_sums, lane < n_ctas ? lane : 0);
        acc = {peer_f32(p), peer_f32(p + 4), peer_f32(p + 8)};
        acc = join_lanes(lane < n_ctas ? acc : Sums{-INFINITY, 0.0f, 0.0f}, c);
      }
      if (TOP) {
        if (threadIdx.x < n_ctas * a.top_k) {
          const int r = threadIdx.x / a.top_k;
          lists[threadIdx.x] =
              peer_u64(cluster_peer(cta_list + (threadIdx.x - r * a.top_k), r));
        }
        __syncthreads();
        rank_entries(lists, n_ctas * a.top_k, a.top_k, best);
      }
    }
    score_cluster_sync();   // a CTA's shared memory outlives its readers
  } else if (TOP) {
    __syncthreads();
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
    const uint64_t e = best[lane];
    a.top_logprob[row * a.top_k + lane] = logprob(order_value((uint32_t)(e >> 32)));
    a.top_index[row * a.top_k + lane] = (int32_t)~(uint32_t)e;
  }
}

template <typename T, bool TOP>
static cudaError_t launch_score(const ScoreArgs& a, int ctas, int64_t rows, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, (unsigned)rows);
  cfg.blockDim = dim3(kScoreThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, token_score_kernel<T, TOP>, a);
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
  if (!(temperature > 0.0f) || !(1.0f / temperature <= FLT_MAX) || !(temperature <= FLT_MAX))
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
  // rows alone fill the GPU from two CTAs an SM on; below that a row is split
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
