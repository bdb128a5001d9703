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
constexpr int kScoreVecs = 4;       // 16-byte loads in flight a thread

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
__device__ __forceinline__ uint64_t entry(float x, int64_t index) {
  return ((uint64_t)order_key(x) << 32) | (uint32_t)~(uint32_t)index;
}

// The running sums of one thread or of a part of a row.
struct Sums {
  float m, s, u;   // maximum logit, sum 2^d, sum 2^d d (d in log2 units)
};

// a joined with b; c = log2(e) / T
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
  // a part without weight (nothing in it, or all -inf) leaves the other as it is
  if (b.s == 0.0f) return {max_nan(a.m, b.m), a.s, a.u};
  if (a.s == 0.0f) return {max_nan(a.m, b.m), b.s, b.u};
  const float m = max_nan(a.m, b.m);
  const float da = (a.m - m) * c, db = (b.m - m) * c;
  const float fa = exp2f(da), fb = exp2f(db);
  // f d -> 0 as f -> 0: a part too small to count adds nothing
  const float ua = fa == 0.0f ? 0.0f : (a.u + a.s * da) * fa;
  const float ub = fb == 0.0f ? 0.0f : (b.u + b.s * db) * fb;
  return {m, a.s * fa + b.s * fb, ua + ub};
}

// The warp's best top_k entries, one a lane, best first.
struct TopList {
  uint64_t mine = 0;   // this lane's entry
  uint64_t last = 0;   // entry top_k - 1: what a newcomer has to beat

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

// best top_k of n sorted lists of top_k entries each (n <= 32), list l read by
// lane l through at(i): every round the best head leaves its list
template <typename At>
__device__ __forceinline__ uint64_t merge_lists(int n, int top_k, At at) {
  const int lane = lane_id();
  int i = 0;
  uint64_t head = lane < n ? at(0) : 0, mine = 0;
  for (int r = 0; r < top_k; r++) {
    uint64_t best = head;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t x = __shfl_xor_sync(0xffffffffu, best, o);
      best = x > best ? x : best;
    }
    if (lane == r) mine = best;
    if (head == best && best != 0) {   // entries are distinct: one lane's head
      i++;
      head = i < top_k ? at(i) : 0;
    }
  }
  return mine;
}

// Row blockIdx.y by a cluster of gridDim.x CTAs, each a contiguous part of it.
// A thread takes kScoreVecs 16-byte vectors a step, rescales its sums when its
// own maximum moves, and the warp looks for newcomers to its list of top_k only
// when some lane holds a logit that is not below the list's last. The parts are
// joined in shared memory, then over the cluster's: always in the same order.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kScoreThreads) token_score_kernel(const ScoreArgs a) {
  constexpr int N = Lanes<T>::N;
  __shared__ Sums sums[kScoreWarps];
  __shared__ Sums cta_sums;
  __shared__ uint64_t lists[kScoreWarps][kScoreMaxTop];
  __shared__ uint64_t cta_list[kScoreMaxTop];
  const int lane = lane_id(), w = warp_id();
  const int rank = blockIdx.x, n_ctas = gridDim.x;
  const int64_t row = blockIdx.y;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const float c = 1.4426950408889634f * a.inv_t;

  Sums acc = {-INFINITY, 0.0f, 0.0f};
  TopList top;
  float seen = -INFINITY;   // the list's last logit

  // one step: `count` valid logits of v in this lane, index of the first
  auto step = [&](auto& v, auto index_of, auto valid) {
    constexpr int K = sizeof(v) / sizeof(float);
    float vm = -INFINITY;
#pragma unroll
    for (int i = 0; i < K; i++) vm = max_nan(vm, v[i]);
    if (!(vm <= acc.m)) {
      const Sums fresh = {vm, 0.0f, 0.0f};
      const float d = (acc.m - vm) * c, f = acc.s == 0.0f ? 0.0f : exp2f(d);
      acc.u = f == 0.0f ? 0.0f : (acc.u + acc.s * d) * f;
      acc.s *= f;
      acc.m = fresh.m;
    }
    const float m = acc.m == -INFINITY ? 0.0f : acc.m;
#pragma unroll
    for (int i = 0; i < K; i++) {
      // the bound keeps d finite where e is 0 (a masked logit)
      const float d = max_nan((v[i] - m) * c, -1e4f);
      const float e = fast_exp2(d);
      acc.s += e;
      acc.u = fmaf(e, d, acc.u);
    }
    if (TOP && __any_sync(0xffffffffu, !(vm < seen))) {
#pragma unroll
      for (int i = 0; i < K; i++) top.offer(valid(i) ? entry(v[i], index_of(i)) : 0, a.top_k);
      seen = top.last ? order_value((uint32_t)(top.last >> 32)) : -INFINITY;
    }
  };

  // head and tail: the elements before the first and past the last whole vector
  const int64_t lead = min(a.vocab, (int64_t)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int64_t n_vec = (a.vocab - lead) / N;
  if (rank == 0 && w == 0) {
    float v[1] = {lane < lead ? Lanes<T>::one(x + lane) : -INFINITY};
    step(v, [&](int) { return (int64_t)lane; }, [&](int) { return lane < lead; });
  }
  const uint4* xv = reinterpret_cast<const uint4*>(x + lead);
  const int64_t v0 = n_vec * rank / n_ctas, v1 = n_vec * (rank + 1) / n_ctas;
  // a warp's vectors of a step lie side by side, so its indices only grow
  for (int64_t i = v0 + w * 32 * kScoreVecs; i < v1; i += kScoreThreads * kScoreVecs) {
    float v[kScoreVecs * N];
#pragma unroll
    for (int j = 0; j < kScoreVecs; j++) {
      const int64_t k = i + j * 32 + lane;
      float p[N];
      if (k < v1) {
        Lanes<T>::unpack(__ldg(xv + k), p);
      } else {
#pragma unroll
        for (int e = 0; e < N; e++) p[e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < N; e++) v[j * N + e] = p[e];
    }
    step(
        v,
        [&](int e) { return lead + (i + (e / N) * 32 + lane) * N + e % N; },
        [&](int e) { return i + (e / N) * 32 + lane < v1; });
  }
  if (rank == n_ctas - 1 && w == kScoreWarps - 1) {
    const int64_t k = lead + n_vec * N + lane;
    float v[1] = {k < a.vocab ? Lanes<T>::one(x + k) : -INFINITY};
    step(v, [&](int) { return k; }, [&](int) { return k < a.vocab; });
  }

  // the warp's, the CTA's, the row's
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums b = {__shfl_xor_sync(0xffffffffu, acc.m, o), __shfl_xor_sync(0xffffffffu, acc.s, o),
              __shfl_xor_sync(0xffffffffu, acc.u, o)};
    acc = join(acc, b, c);
  }
  if (lane == 0) sums[w] = acc;
  if (TOP) lists[w][lane] = top.mine;
  __syncthreads();
  if (w == 0) {
    for (int i = 1; i < kScoreWarps; i++) acc = join(acc, sums[i], c);
    if (lane == 0) cta_sums = acc;
    if (TOP)
      cta_list[lane] = merge_lists(kScoreWarps, a.top_k, [&](int i) { return lists[lane][i]; });
  }
  if (n_ctas > 1) {
    score_cluster_sync();
    if (rank == 0 && w == 0) {
      for (int r = 1; r < n_ctas; r++) {
        const uint32_t p = cluster_peer(&cta_sums, r);
        acc = join(acc, Sums{peer_f32(p), peer_f32(p + 4), peer_f32(p + 8)}, c);
      }
      if (TOP) {
        const uint32_t p = cluster_peer(cta_list, lane < n_ctas ? lane : 0);
        top.mine = merge_lists(n_ctas, a.top_k, [&](int i) { return peer_u64(p + 8 * i); });
      }
    }
    score_cluster_sync();   // a CTA's shared memory outlives its readers
  } else if (TOP && w == 0) {
    top.mine = cta_list[lane];
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
    a.top_logprob[row * a.top_k + lane] = logprob(order_value((uint32_t)(top.mine >> 32)));
    a.top_index[row * a.top_k + lane] = (int32_t)~(uint32_t)top.mine;
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
