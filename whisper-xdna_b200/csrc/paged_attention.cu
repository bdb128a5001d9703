// Attention of one new token a sequence over a paged key-value cache.
//
// For sequence i, key-value head h and each of the head's `group` query rows
//   s_j = scale q . k_j   for start_i <= j < len_i
//   lse = log sum_j e^(s_j),   o = sum_j e^(s_j - lse) v_j
// in one pass over the cache with a running maximum and sum in fp32 (exponents
// in units of log2). A row without keys gives o = 0 and lse = -inf. The cache's
// length is split over CTAs where sequences and heads alone do not fill the
// GPU; the parts' (maximum, sum, o) are then joined, always in the same order.
#include <atomic>
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
  uint32_t div_mul, div_shift;   // t / page_size = (umulhi(t, mul) + t) >> shift
  float scale_log2;       // scale * log2(e)
};

__device__ __forceinline__ int page_slot(const PagedArgs& a, int t) {
  return (int)((__umulhi((uint32_t)t, a.div_mul) + (uint32_t)t) >> a.div_shift);
}

__device__ __forceinline__ void store_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_out(uint16_t* p, float x) {
  *p = (uint16_t)bf16_bits<RND_RNE>(x);
}

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

// GT query rows of one (sequence, head) against the keys of one split, fp32:
// products on the FMA pipe, which keeps all of their bits. Each group of `lanes` lanes holds a key row (16 bytes a
// lane); the groups of the CTA take tokens in turn, keep sums of their own and
// are joined at the end.
template <int HD, int GT>
__global__ void __launch_bounds__(kPagedThreads) paged_attention_fma_kernel(const PagedArgs a) {
  constexpr int N = 4, kLanes = HD / N;     // lanes on a row
  constexpr int kRows = 32 / kLanes;                 // rows a warp reads at once
  constexpr int kStreams = kPagedWarps * kRows;      // token streams of the CTA
  constexpr int U = 4;                               // tokens of a stream in flight
  static_assert(kLanes <= 32 && 32 % kLanes == 0, "");
  __shared__ float sh_o[kStreams][GT][HD];
  __shared__ float sh_m[kStreams][GT], sh_l[kStreams][GT];
  pdl_launch_dependents();   // the join waits for this kernel's end

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
  const float* q = static_cast<const float*>(a.q) + seq * a.q_seq + head * a.q_head;
  const float* kp = static_cast<const float*>(a.k) + head * a.head_stride + sub * N;
  const float* vp = static_cast<const float*>(a.v) + head * a.head_stride + sub * N;
  const int32_t* row = a.table + seq * a.ld_table;

  float qr[GT][N], o[GT][N], m[GT], l[GT];
#pragma unroll
  for (int g = 0; g < GT; g++) {
    m[g] = -INFINITY;
    l[g] = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e++) {
      o[g][e] = 0.0f;
      qr[g][e] = g < g_n ? q[(g0 + g) * a.q_group + sub * N + e] * a.scale_log2 : 0.0f;
    }
  }
  for (int t0 = c0 + stream; t0 - stream < c1; t0 += kStreams * U) {
    float4 kw[U], vw[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int t = t0 + u * kStreams;
      ok[u] = t < c1;
      kw[u] = vw[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (ok[u]) {
        const int slot = page_slot(a, t);
        const int page = row[slot];
        if (page < 0 || page >= a.n_pages) {
          atomicOr(&g_attend_err, WX_DEVERR_PAGE);
          ok[u] = false;
        } else {
          const int64_t at = page * a.page_stride + (t - slot * a.page_size) * a.tok_stride;
          kw[u] = *reinterpret_cast<const float4*>(kp + at);
          vw[u] = *reinterpret_cast<const float4*>(vp + at);
        }
      }
    }
    float s[U][GT];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const float kf[N] = {kw[u].x, kw[u].y, kw[u].z, kw[u].w};
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
      const float vf[N] = {vw[u].x, vw[u].y, vw[u].z, vw[u].w};
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
      float* out = static_cast<float*>(a.out) + seq * a.o_seq + head * a.o_head + (g0 + g) * a.o_group;
      out[d] = sum == 0.0f ? 0.0f : x / sum;
      if (d == 0 && a.lse)
        a.lse[r] = sum == 0.0f ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
    }
  }
}

// ---------------------------------------------------------------- tensor cores

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  // src_size 0 reads nothing and writes zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(ok ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// d += a (16 x 16, row) * b (16 x 8, col), bf16 in, fp32 out
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit values, one row in each four lanes, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

constexpr int kTok = 16;   // keys of one tile

template <int HD>
struct MmaCfg {
  static constexpr int kStages = HD == 64 ? 4 : 3;
  static constexpr int kTileBytes = kTok * HD * 2;               // K or V of one tile
  static constexpr int kWarpBytes = kStages * 2 * kTileBytes;
  static constexpr int kSmem = kPagedWarps * kWarpBytes;
};

// Up to 8 NT query rows of one (sequence, head) against the keys of one split, bf16.
//
// The keys stand where a matrix product has its rows: S^T = K Q^T is 16 keys x 8
// query rows a product and O^T = V^T P^T is 16 dimensions x 8 query rows, so one
// query row costs what eight do and the softmax needs no shared memory: P^T is
// S^T's accumulator, transposed 8 x 8 at a time in registers. Each warp takes
// tiles of 16 keys in turn through a ring of its own, filled by asynchronous
// 16-byte copies (any page size, layout and start: each row has an address of its
// own, rows out of range are zeros), and keeps sums of its own: no barrier until
// the four warps' parts are joined at the end. The rows' reference maximum moves
// only when a score passes it by more than 2^8, so weights stay below 2^8 and
// the rescaling is rare.
template <int HD, int NT>
__global__ void __launch_bounds__(kPagedThreads) paged_attention_mma_kernel(const PagedArgs a) {
  using Cfg = MmaCfg<HD>;
  constexpr int kRows = 8 * NT, kSteps = HD / 16, kCpr = HD / 8;   // 16-byte chunks of a row
  constexpr int kLoads = kTok * kCpr / 32;                         // a lane, K or V
  extern __shared__ __align__(128) char smem[];
  __shared__ float sh_m[kPagedWarps][kRows], sh_l[kPagedWarps][kRows];
  pdl_launch_dependents();   // the join waits for this kernel's end

  const int tiles = (a.group + kRows - 1) / kRows;
  const int split = blockIdx.x / tiles, g0 = (blockIdx.x - split * tiles) * kRows;
  const int g_n = min(kRows, a.group - g0);
  const int head = blockIdx.y, seq = blockIdx.z;
  int first, end;
  key_range(a, seq, &first, &end);
  const int c0 = max(first, split * a.chunk), c1 = min(end, (split + 1) * a.chunk);
  if (c0 >= c1 && a.splits > 1) return;   // the join skips it too

  const int lane = lane_id(), w = warp_id();
  const uint16_t* kp = static_cast<const uint16_t*>(a.k) + head * a.head_stride;
  const uint16_t* vp = static_cast<const uint16_t*>(a.v) + head * a.head_stride;
  const int32_t* row = a.table + seq * a.ld_table;
  const uint32_t ring = smem_u32(smem) + w * Cfg::kWarpBytes;

  // the warp's tiles: kTok keys from base + 4 kTok i on
  const int base = c0 / kTok * kTok + w * kTok;
  const int n_mine = base < c1 ? (c1 - base + kPagedWarps * kTok - 1) / (kPagedWarps * kTok) : 0;

  // where key (tile i, lane % 16) is, -1: nowhere
  auto locate = [&](int i) -> int64_t {
    const int t = base + i * kPagedWarps * kTok + (lane & 15);
    if (t < c0 || t >= c1) return -1;
    const int slot = page_slot(a, t);
    const int page = __ldg(row + slot);
    if (page < 0 || page >= a.n_pages) {
      atomicOr(&g_attend_err, WX_DEVERR_PAGE);
      return -1;
    }
    return page * a.page_stride + (t - slot * a.page_size) * a.tok_stride;
  };
  // copies tile i (its keys at `where`) into its slot of the ring; returns which
  // keys have none
  auto fetch = [&](int i, int64_t where) {
    const uint32_t slot = ring + (i % Cfg::kStages) * 2 * Cfg::kTileBytes;
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      const int r = j * (32 / kCpr) + lane / kCpr, c = lane % kCpr;
      const int64_t at = __shfl_sync(0xffffffffu, where, r);
      const uint32_t dst = slot + r * HD * 2 + ((c ^ (r & 7)) << 4);
      const int64_t from = at < 0 ? 0 : at + c * 8;
      cp_async16(dst, kp + from, at >= 0);
      cp_async16(dst + Cfg::kTileBytes, vp + from, at >= 0);
    }
  };

  int64_t next = n_mine > 0 ? locate(0) : -1;
  uint32_t live[Cfg::kStages];   // bit r: key r of the tile in this slot is one
#pragma unroll
  for (int i = 0; i < Cfg::kStages - 1; i++) {
    live[i] = __ballot_sync(0xffffffffu, next >= 0);
    if (i < n_mine) fetch(i, next);
    cp_async_commit();
    next = i + 1 < n_mine ? locate(i + 1) : -1;
  }

  // Q^T in fragments: row n = lane / 4, dimensions 2 (lane % 4) + {0, 1, 8, 9}
  uint32_t qf[NT][kSteps][2];
  {
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + seq * a.q_seq + head * a.q_head;
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int g = n * 8 + lane / 4;
      const uint16_t* p = q + (g0 + g) * a.q_group + (lane & 3) * 2;
#pragma unroll
      for (int k = 0; k < kSteps; k++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          qf[n][k][h] = g < g_n ? (uint32_t)p[k * 16 + h * 8] |
                                      ((uint32_t)p[k * 16 + h * 8 + 1] << 16)
                                : 0;
    }
  }

  float o[NT][kSteps][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; n++) {
#pragma unroll
    for (int k = 0; k < kSteps; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[n][k][e] = 0.0f;
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.0f;
  }
  const int lr = lane & 7, l8 = lane >> 3;

#pragma unroll 1
  for (int i = 0; i < n_mine; i++) {
    {
      const int f = i + Cfg::kStages - 1;
      __syncwarp();   // every lane has read the slot that is filled now
      const uint32_t bits = __ballot_sync(0xffffffffu, next >= 0);
      if (f < n_mine) fetch(f, next);
      cp_async_commit();
      next = f + 1 < n_mine ? locate(f + 1) : -1;
      live[Cfg::kStages - 1] = bits;
    }
    cp_async_wait<Cfg::kStages - 1>();
    __syncwarp();
    const uint32_t kt = ring + (i % Cfg::kStages) * 2 * Cfg::kTileBytes;
    const uint32_t vt = kt + Cfg::kTileBytes;

    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
    for (int k = 0; k < kSteps; k++) {
      uint32_t kf[4];
      const int r = (l8 & 1) * 8 + lr, c = k * 2 + (l8 >> 1);
      ldmatrix4(kf, kt + r * HD * 2 + ((c ^ lr) << 4));
#pragma unroll
      for (int n = 0; n < NT; n++) mma_bf16(s[n], kf, qf[n][k][0], qf[n][k][1]);
    }
    // keys lane / 4 and lane / 4 + 8, query rows 2 (lane % 4) + {0, 1}
    const bool in0 = live[0] >> (lane >> 2) & 1, in1 = live[0] >> ((lane >> 2) + 8) & 1;
    uint32_t pf[NT][2], pl[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; e++)
        x[e] = (e < 2 ? in0 : in1) ? s[n][e] * a.scale_log2 : -INFINITY;
      const float m0 = fmaxf(x[0], x[2]), m1 = fmaxf(x[1], x[3]);
      if (__any_sync(0xffffffffu, m0 > m[n][0] + 8.0f || m1 > m[n][1] + 8.0f)) {
        float y[2] = {m0, m1};
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1)
            y[h] = fmaxf(y[h], __shfl_xor_sync(0xffffffffu, y[h], d));
          y[h] = fmaxf(y[h], m[n][h]);
          const float f = m[n][h] == -INFINITY ? 0.0f : fast_exp2(m[n][h] - y[h]);
          m[n][h] = y[h];
          l[n][h] *= f;
#pragma unroll
          for (int k = 0; k < kSteps; k++) {
            o[n][k][h] *= f;
            o[n][k][2 + h] *= f;
          }
        }
      }
      // a row that has met no score above -inf yet: its reference is 0
      const float r0 = m[n][0] == -INFINITY ? 0.0f : m[n][0];
      const float r1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];
      x[0] = fast_exp2(x[0] - r0);
      x[1] = fast_exp2(x[1] - r1);
      x[2] = fast_exp2(x[2] - r0);
      x[3] = fast_exp2(x[3] - r1);
      l[n][0] += x[0] + x[2];
      l[n][1] += x[1] + x[3];
      // the weights in two bf16 parts, the upper half of their bits and the rest
      // (15 bits or more in all): the product with V then loses nothing that the
      // result's type could hold. The rest of a weight above 0 is kept above 0, so
      // that an infinite v gives an infinity and not 0 * inf.
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; e++)
        y[e] = fmaxf(x[e] - __uint_as_float(__float_as_uint(x[e]) & 0xFFFF0000u),
                     x[e] * 0x1p-30f);
      pf[n][0] = transpose8(pack_bf16x2<RND_TRUNC>(x[0], x[1]));
      pf[n][1] = transpose8(pack_bf16x2<RND_TRUNC>(x[2], x[3]));
      pl[n][0] = transpose8(pack_bf16x2_rne(y[0], y[1]));
      pl[n][1] = transpose8(pack_bf16x2_rne(y[2], y[3]));
    }
#pragma unroll
    for (int k = 0; k < kSteps; k++) {
      uint32_t vf[4];
      const int r = (l8 >> 1) * 8 + lr, c = k * 2 + (l8 & 1);
      ldmatrix4_trans(vf, vt + r * HD * 2 + ((c ^ lr) << 4));
#pragma unroll
      for (int n = 0; n < NT; n++) {
        mma_bf16(o[n][k], vf, pf[n][0], pf[n][1]);
        mma_bf16(o[n][k], vf, pl[n][0], pl[n][1]);
      }
    }
#pragma unroll
    for (int j = 0; j + 1 < Cfg::kStages; j++) live[j] = live[j + 1];
  }
  cp_async_wait<0>();
  __syncthreads();   // the rings become the warps' parts of o

  float* part = reinterpret_cast<float*>(smem);   // [warp][row][HD]
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float sum = l[n][h];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const int g = n * 8 + (lane & 3) * 2 + h;
      if (lane < 4) {
        sh_m[w][g] = m[n][h];
        sh_l[w][g] = sum;
      }
      float* p = part + (w * kRows + g) * HD + (lane >> 2);
#pragma unroll
      for (int k = 0; k < kSteps; k++) {
        p[k * 16] = o[n][k][h];
        p[k * 16 + 8] = o[n][k][2 + h];
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < g_n * HD; i += kPagedThreads) {
    const int g = i / HD, d = i - g * HD;
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kPagedWarps; u++) mx = fmaxf(mx, sh_m[u][g]);
    const float mu = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f, x = 0.0f;
#pragma unroll
    for (int u = 0; u < kPagedWarps; u++) {
      const float f = fast_exp2(sh_m[u][g] - mu);
      sum = fmaf(sh_l[u][g], f, sum);
      x = fmaf(part[(u * kRows + g) * HD + d], f, x);
    }
    const int64_t r = ((int64_t)seq * a.n_heads + head) * a.group + g0 + g;
    if (a.splits > 1) {
      a.part_o[(r * a.splits + split) * HD + d] = x;
      if (d == 0) a.part_ml[r * a.splits + split] = make_float2(mx, sum);
    } else {
      uint16_t* out = static_cast<uint16_t*>(a.out) + seq * a.o_seq + head * a.o_head +
                      (g0 + g) * a.o_group;
      out[d] = (uint16_t)bf16_bits<RND_RNE>(sum == 0.0f ? 0.0f : x / sum);
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
    store_out(out + e * 32 + lane, sum == 0.0f ? 0.0f : x[e] / sum);
  if (lane == 0 && a.lse)
    a.lse[r] = sum == 0.0f ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
}

// How a call's work is cut: query rows a CTA takes, splits of the cache's length
// and the tokens of one.
struct PagedCut {
  int tile, splits, chunk;
};

static PagedCut paged_cut(int64_t n_seqs, int64_t n_heads, int64_t group, int64_t max_len,
                          int dtype) {
  PagedCut c;
  if (dtype == WX_DTYPE_BF16) {
    c.tile = group <= 8 ? 8 : 16;
  } else {
    c.tile = 1;
    while (c.tile < 8 && c.tile < group) c.tile *= 2;
  }
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

template <int HD, int NT>
static cudaError_t run_mma(const PagedArgs& a, dim3 grid, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};   // bit: a device whose limit has been raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(done.load(std::memory_order_acquire) >> dev & 1)) {
    e = cudaFuncSetAttribute(paged_attention_mma_kernel<HD, NT>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, MmaCfg<HD>::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  }
  return launch_k(paged_attention_mma_kernel<HD, NT>, grid, dim3(kPagedThreads),
                  MmaCfg<HD>::kSmem, st, a);
}

template <int HD>
static cudaError_t run_fma(const PagedArgs& a, int tile, dim3 grid, cudaStream_t st) {
  const dim3 block(kPagedThreads);
  switch (tile) {
    case 1: return launch_k(paged_attention_fma_kernel<HD, 1>, grid, block, 0, st, a);
    case 2: return launch_k(paged_attention_fma_kernel<HD, 2>, grid, block, 0, st, a);
    case 4: return launch_k(paged_attention_fma_kernel<HD, 4>, grid, block, 0, st, a);
    default: return launch_k(paged_attention_fma_kernel<HD, 8>, grid, block, 0, st, a);
  }
}

template <typename T, int HD>
static cudaError_t run_paged(const PagedArgs& a, const PagedCut& c, int64_t n_seqs,
                             cudaStream_t st) {
  const int tiles = (a.group + c.tile - 1) / c.tile;
  const dim3 grid((unsigned)(c.splits * tiles), (unsigned)a.n_heads, (unsigned)n_seqs);
  cudaError_t e;
  if constexpr (sizeof(T) == 2)
    e = c.tile == 8 ? run_mma<HD, 1>(a, grid, st) : run_mma<HD, 2>(a, grid, st);
  else
    e = run_fma<HD>(a, c.tile, grid, st);
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
                                     int64_t head_dim, int64_t max_len, int dtype) {
  using namespace wx;
  const int s = check_cut("paged_attention_workspace", n_seqs, n_heads, group, head_dim, max_len);
  if (s != WX_OK) return s;
  return paged_space(n_seqs * n_heads * group, paged_cut(n_seqs, n_heads, group, max_len, dtype),
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
  const PagedCut c = paged_cut(n_seqs, n_heads, group, max_len, dtype);
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
  // Granlund and Montgomery's division by an invariant, for t < 2^31
  a.div_shift = 0;
  while ((1ll << a.div_shift) < page_size) a.div_shift++;
  a.div_mul = (uint32_t)((((1ull << a.div_shift) - page_size) << 32) / page_size + 1);
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
