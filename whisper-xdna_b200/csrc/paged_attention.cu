// Attention of one new token a sequence over a paged key-value cache.
//
// For sequence i, key-value head h and each of the head's `group` query rows
//   s_j = scale q . k_j   for start_i <= j < len_i
//   lse = log sum_j e^(s_j),   o = sum_j e^(s_j - lse) v_j
// in one pass over the cache with a running maximum and sum in fp32 (exponents
// in units of log2). A row without keys gives o = 0 and lse = -inf. The cache's
// length is split over CTAs where sequences and heads alone do not fill the
// GPU; the parts' (maximum, sum, o) are then joined, always in the same order.
#include <cstdint>

#include "common.cuh"
#include "kvcache.cuh"

namespace wx {

static __device__ int g_attend_err;

int paged_attention_take_error(int* flags, bool clear) {
  int v = 0;
  WX_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_attend_err, sizeof(int)));
  *flags |= v;
  const int zero = 0;
  if (v && clear) WX_CUDA_TRY(cudaMemcpyToSymbol(g_attend_err, &zero, sizeof(int)));
  return WX_OK;
}

struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;             // (sequences, heads, group) or NULL
  float* part_o;          // (rows, splits, head_dim): parts, where splits > 1
  float2* part_ml;        // (rows, splits): maximum (log2 units) and sum
  const int32_t *table, *lens, *starts;
  int64_t q_seq, q_head, q_group, o_seq, o_head, o_group;   // elements
  int64_t page_stride, tok_stride, head_stride, ld_table;
  int64_t n_pages;
  int n_heads, group, page_size, max_len, splits, chunk;
  float scale_log2;       // scale * log2(e)
};

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int N = 4;   // elements in 16 bytes
  static __device__ __forceinline__ void unpack(const uint4& w, float (&v)[4]) {
    v[0] = __uint_as_float(w.x);
    v[1] = __uint_as_float(w.y);
    v[2] = __uint_as_float(w.z);
    v[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float x) { *p = x; }
};
template <>
struct Elem<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& w, float (&v)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __uint_as_float(a[i] << 16);
      v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ float load(const uint16_t* p) {
    return __uint_as_float((uint32_t)*p << 16);
  }
  static __device__ __forceinline__ void store(uint16_t* p, float x) {
    *p = (uint16_t)bf16_bits<RND_RNE>(x);
  }
};

// The keys that sequence `seq` attends to, as far as the table reaches.
__device__ __forceinline__ void key_range(const PagedArgs& a, int seq, int* first, int* end) {
  int n = a.lens[seq];
  if (n > a.max_len) {
    atomicOr(&g_attend_err, WX_DEVERR_PAGE);
    n = a.max_len;
  }
  *end = max(n, 0);
  *first = a.starts ? max(a.starts[seq], 0) : 0;
}

constexpr int kPagedThreads = 128;
constexpr int kPagedWarps = kPagedThreads / 32;

// GT query rows of one (sequence, head) against the keys of one split, products
// on the FMA pipe. Each group of `lanes` lanes holds a key row (16 bytes a
// lane); the groups of the CTA take tokens in turn, keep sums of their own and
// are joined at the end.
template <typename T, int HD, int GT>
__global__ void __launch_bounds__(kPagedThreads) paged_attention_fma_kernel(const PagedArgs a) {
  constexpr int N = Elem<T>::N, kLanes = HD / N;     // lanes on a row
  constexpr int kRows = 32 / kLanes;                 // rows a warp reads at once
  constexpr int kStreams = kPagedWarps * kRows;      // token streams of the CTA
  constexpr int U = 4;                               // tokens of a stream in flight
  static_assert(kLanes <= 32 && 32 % kLanes == 0, "");
  __shared__ float sh_o[kStreams][GT][HD];
  __shared__ float sh_m[kStreams][GT], sh_l[kStreams][GT];

  const int tiles = (a.group + GT - 1) / GT;
  const int split = blockIdx.x / tiles, tile = blockIdx.x - split * tiles;
  const int head = blockIdx.y, seq = blockIdx.z;
  const int g0 = tile * GT, g_n = min(GT, a.group - g0);
  int first, end;
  key_range(a, seq, &first, &end);
  const int c0 = max(first, split * a.chunk), c1 = min(end, (split + 1) * a.chunk);
  if (c0 >= c1 && a.splits > 1) return;   // the join skips it too

  const int lane = lane_id(), sub = lane % kLanes;
  const int stream = warp_id() * kRows + lane / kLanes;
  const T* q = static_cast<const T*>(a.q) + seq * a.q_seq + head * a.q_head;
  const T* kp = static_cast<const T*>(a.k) + head * a.head_stride + sub * N;
  const T* vp = static_cast<const T*>(a.v) + head * a.head_stride + sub * N;
  const int32_t* row = a.table + seq * a.ld_table;

  float qr[GT][N], o[GT][N], m[GT], l[GT];
#pragma unroll
  for (int g = 0; g < GT; g++) {
    m[g] = -INFINITY;
    l[g] = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e++) {
      o[g][e] = 0.0f;
      qr[g][e] = g < g_n ? Elem<T>::load(q + (g0 + g) * a.q_group + sub * N + e) * a.scale_log2
                         : 0.0f;
    }
  }
  for (int t0 = c0 + stream; t0 - stream < c1; t0 += kStreams * U) {
    uint4 kw[U], vw[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int t = t0 + u * kStreams;
      ok[u] = t < c1;
      kw[u] = vw[u] = make_uint4(0, 0, 0, 0);
      if (ok[u]) {
        const int slot = t / a.page_size;
        const int page = row[slot];
        if (page < 0 || page >= a.n_pages) {
          atomicOr(&g_attend_err, WX_DEVERR_PAGE);
          ok[u] = false;
        } else {
          const int64_t at = page * a.page_stride + (t - slot * a.page_size) * a.tok_stride;
          kw[u] = *reinterpret_cast<const uint4*>(kp + at);
          vw[u] = *reinterpret_cast<const uint4*>(vp + at);
        }
      }
    }
    float s[U][GT];
#pragma unroll
    for (int u = 0; u < U; u++) {
      float kf[N];
      Elem<T>::unpack(kw[u], kf);
#pragma unroll
      for (int g = 0; g < GT; g++) {
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++) x = fmaf(qr[g][e], kf[e], x);
#pragma unroll
        for (int w = kLanes / 2; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
        s[u][g] = ok[u] ? x : -INFINITY;
      }
    }
#pragma unroll
    for (int g = 0; g < GT; g++) {
      float mx = m[g];
#pragma unroll
      for (int u = 0; u < U; u++) mx = fmaxf(mx, s[u][g]);
      const float mu = mx == -INFINITY ? 0.0f : mx;
      const float f = fast_exp2(m[g] - mu);
      m[g] = mx;
      l[g] *= f;
#pragma unroll
      for (int e = 0; e < N; e++) o[g][e] *= f;
#pragma unroll
      for (int u = 0; u < U; u++) {
        s[u][g] = fast_exp2(s[u][g] - mu);
        l[g] += s[u][g];
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      float vf[N];
      Elem<T>::unpack(vw[u], vf);
#pragma unroll
      for (int g = 0; g < GT; g++)
#pragma unroll
        for (int e = 0; e < N; e++) o[g][e] = fmaf(s[u][g], vf[e], o[g][e]);
    }
  }
#pragma unroll
  for (int g = 0; g < GT; g++) {
#pragma unroll
    for (int e = 0; e < N; e++) sh_o[stream][g][sub * N + e] = o[g][e];
    if (sub == 0) {
      sh_m[stream][g] = m[g];
      sh_l[stream][g] = l[g];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < g_n * HD; i += kPagedThreads) {
    const int g = i / HD, d = i - g * HD;
    float mx = -INFINITY;
    for (int w = 0; w < kStreams; w++) mx = fmaxf(mx, sh_m[w][g]);
    const float mu = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f, x = 0.0f;
    for (int w = 0; w < kStreams; w++) {
      const float f = fast_exp2(sh_m[w][g] - mu);
      sum = fmaf(sh_l[w][g], f, sum);
      x = fmaf(sh_o[w][g][d], f, x);
    }
    const int64_t r = ((int64_t)seq * a.n_heads + head) * a.group + g0 + g;
    if (a.splits > 1) {
      a.part_o[(r * a.splits + split) * HD + d] = x;
      if (d == 0) a.part_ml[r * a.splits + split] = make_float2(mx, sum);
    } else {
      T* out = static_cast<T*>(a.out) + seq * a.o_seq + head * a.o_head + (g0 + g) * a.o_group;
      Elem<T>::store(out + d, sum == 0.0f ? 0.0f : x / sum);
      if (d == 0 && a.lse)
        a.lse[r] = sum == 0.0f ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
    }
  }
}

// One warp a query row: the parts of the splits that held keys, joined in order.
template <typename T, int HD>
__global__ void __launch_bounds__(kPagedThreads) paged_attention_join_kernel(const PagedArgs a,
                                                                             int64_t rows) {
  pdl_wait();
  const int64_t r = (int64_t)blockIdx.x * kPagedWarps + warp_id();
  if (r >= rows) return;
  constexpr int N = HD / 32;
  const int lane = lane_id();
  const int g = (int)(r % a.group);
  const int64_t sh = r / a.group;
  const int head = (int)(sh % a.n_heads), seq = (int)(sh / a.n_heads);
  int first, end;
  key_range(a, seq, &first, &end);
  const int s0 = first / a.chunk, s1 = first < end ? (end + a.chunk - 1) / a.chunk : s0;
  float mx = -INFINITY;
  for (int s = s0; s < s1; s++) mx = fmaxf(mx, a.part_ml[r * a.splits + s].x);
  const float mu = mx == -INFINITY ? 0.0f : mx;
  float sum = 0.0f, x[N] = {};
  for (int s = s0; s < s1; s++) {
    const float2 ml = a.part_ml[r * a.splits + s];
    const float f = fast_exp2(ml.x - mu);
    sum = fmaf(ml.y, f, sum);
    const float* p = a.part_o + (r * a.splits + s) * HD;
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = fmaf(p[e * 32 + lane], f, x[e]);
  }
  T* out = static_cast<T*>(a.out) + seq * a.o_seq + head * a.o_head + g * a.o_group;
#pragma unroll
  for (int e = 0; e < N; e++)
    Elem<T>::store(out + e * 32 + lane, sum == 0.0f ? 0.0f : x[e] / sum);
  if (lane == 0 && a.lse)
    a.lse[r] = sum == 0.0f ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
}

// How a call's work is cut: query rows a CTA takes, splits of the cache's length
// and the tokens of one.
struct PagedCut {
  int tile, splits, chunk;
};

static PagedCut paged_cut(int64_t n_seqs, int64_t n_heads, int64_t group, int64_t max_len) {
  PagedCut c;
  c.tile = 1;
  while (c.tile < 8 && c.tile < group) c.tile *= 2;
  const int64_t items = n_seqs * n_heads * ((group + c.tile - 1) / c.tile);
  const int64_t want = 4 * 148;      // CTAs
  int64_t chunk = max_len * items / want;
  chunk = chunk < 128 ? 128 : chunk > 1024 ? 1024 : chunk;
  chunk = (chunk + 63) / 64 * 64;
  c.chunk = (int)chunk;
  c.splits = (int)((max_len + chunk - 1) / chunk);
  if (c.splits < 1) c.splits = 1;
  return c;
}

static int64_t paged_space(int64_t rows, const PagedCut& c, int64_t head_dim) {
  return c.splits > 1 ? rows * c.splits * (head_dim * 4 + 8) : 0;
}

template <typename T, int HD>
static cudaError_t run_paged(const PagedArgs& a, const PagedCut& c, int64_t n_seqs,
                             cudaStream_t st) {
  const int tiles = (a.group + c.tile - 1) / c.tile;
  const dim3 grid((unsigned)(c.splits * tiles), (unsigned)a.n_heads, (unsigned)n_seqs);
  cudaError_t e;
  switch (c.tile) {
    case 1:
      e = launch_k(paged_attention_fma_kernel<T, HD, 1>, grid, dim3(kPagedThreads), 0, st, a);
      break;
    case 2:
      e = launch_k(paged_attention_fma_kernel<T, HD, 2>, grid, dim3(kPagedThreads), 0, st, a);
      break;
    case 4:
      e = launch_k(paged_attention_fma_kernel<T, HD, 4>, grid, dim3(kPagedThreads), 0, st, a);
      break;
    default:
      e = launch_k(paged_attention_fma_kernel<T, HD, 8>, grid, dim3(kPagedThreads), 0, st, a);
  }
  if (e != cudaSuccess || c.splits == 1) return e;
  const int64_t rows = n_seqs * a.n_heads * a.group;
  PdlScope pdl(true);
  return launch_k(paged_attention_join_kernel<T, HD>,
                  dim3((unsigned)((rows + kPagedWarps - 1) / kPagedWarps)), dim3(kPagedThreads),
                  0, st, a, rows);
}

static int check_cut(const char* what, int64_t n_seqs, int64_t n_heads, int64_t group,
                     int64_t head_dim, int64_t max_len) {
  if (n_seqs < 0 || n_seqs > 65535 || n_heads < 1 || n_heads > 65535 || group < 1 ||
      group > 65535 || max_len < 0 || max_len > (1 << 30))
    return fail(WX_ERR_INVALID,
                "%s: bad shape: %lld sequences, %lld heads, group %lld, max_len %lld", what,
                (long long)n_seqs, (long long)n_heads, (long long)group, (long long)max_len);
  if (head_dim != 64 && head_dim != 128)
    return fail(WX_ERR_UNSUPPORTED, "%s: head dim %lld (64 and 128 are supported)", what,
                (long long)head_dim);
  return WX_OK;
}

}  // namespace wx

extern "C" {

int64_t wx_paged_attention_workspace(int64_t n_seqs, int64_t n_heads, int64_t group,
                                     int64_t head_dim, int64_t max_len) {
  using namespace wx;
  const int s = check_cut("paged_attention_workspace", n_seqs, n_heads, group, head_dim, max_len);
  if (s != WX_OK) return s;
  return paged_space(n_seqs * n_heads * group, paged_cut(n_seqs, n_heads, group, max_len),
                     head_dim);
}

int wx_paged_attention(const void* q, int64_t q_seq_stride, int64_t q_head_stride,
                       int64_t q_group_stride, const void* k_cache, const void* v_cache,
                       int64_t page_stride, int64_t tok_stride, int64_t head_stride,
                       const int32_t* table, int64_t ld_table, const int32_t* lens,
                       const int32_t* starts, void* out, int64_t o_seq_stride,
                       int64_t o_head_stride, int64_t o_group_stride, float* lse, int64_t n_seqs,
                       int64_t n_heads, int64_t group, int64_t head_dim, int64_t n_pages,
                       int64_t page_size, int64_t max_len, float scale, int dtype,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace wx;
  WX_TRY(check_cut("paged_attention", n_seqs, n_heads, group, head_dim, max_len));
  WX_TRY(check_pool("paged_attention", k_cache, v_cache, page_stride, tok_stride, head_stride,
                    n_heads, head_dim, n_pages, page_size, dtype));
  if (n_seqs == 0) return WX_OK;
  if (!q || !out || !lens || !table || ld_table < 1)
    return fail(WX_ERR_INVALID, "paged_attention: NULL argument or empty page table");
  if (ld_table * page_size < max_len)
    return fail(WX_ERR_INVALID, "paged_attention: max_len %lld is past the table's %lld pages",
                (long long)max_len, (long long)ld_table);
  const int es = dtype == WX_DTYPE_BF16 ? 2 : 4;
  if (((uintptr_t)q | (uintptr_t)out) % es)
    return fail(WX_ERR_INVALID, "paged_attention: q or out not aligned to its type");
  const PagedCut c = paged_cut(n_seqs, n_heads, group, max_len);
  const int64_t rows = n_seqs * n_heads * group, want = paged_space(rows, c, head_dim);
  if (want && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < want))
    return fail(WX_ERR_INVALID,
                "paged_attention: workspace of %lld bytes (16-byte aligned) needed, got %lld",
                (long long)want, (long long)workspace_bytes);
  PagedArgs a = {};
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.out = out;
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * c.splits * head_dim);
  a.table = table;
  a.lens = lens;
  a.starts = starts;
  a.q_seq = q_seq_stride;
  a.q_head = q_head_stride;
  a.q_group = q_group_stride;
  a.o_seq = o_seq_stride;
  a.o_head = o_head_stride;
  a.o_group = o_group_stride;
  a.page_stride = page_stride;
  a.tok_stride = tok_stride;
  a.head_stride = head_stride;
  a.ld_table = ld_table;
  a.n_pages = n_pages;
  a.n_heads = (int)n_heads;
  a.group = (int)group;
  a.page_size = (int)page_size;
  a.max_len = (int)max_len;
  a.splits = c.splits;
  a.chunk = c.chunk;
  a.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = as_stream(stream);
  if (dtype == WX_DTYPE_BF16)
    WX_CUDA_TRY((head_dim == 64 ? run_paged<uint16_t, 64> : run_paged<uint16_t, 128>)(a, c,
                                                                                      n_seqs, st));
  else
    WX_CUDA_TRY((head_dim == 64 ? run_paged<float, 64> : run_paged<float, 128>)(a, c, n_seqs, st));
  return check_launch("paged_attention");
}

}  // extern "C"
