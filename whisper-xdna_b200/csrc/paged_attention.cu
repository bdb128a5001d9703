// Attention of one new token a sequence over a paged key-value cache.
//
// For sequence i, key-value head h and each of the head's `group` query rows
//   s_j = scale q . k_j   for start_i <= j < len_i
//   lse = log sum_j e^(s_j),   o = sum_j e^(s_j - lse) v_j
// in one pass over the cache with a running maximum and sum in fp32 (exponents
// in units of log2). A row without keys gives o = 0 and lse = -inf. The cache's
// length is split over CTAs where sequences and heads alone do not fill the
// GPU; the parts' (maximum, sum, o) are then joined, always in the same order.
#include <algorithm>
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
  float* part_o;          // (rows, splits, head_dim): parts, where chunk > 0
  float2* part_ml;        // (rows, splits): maximum (log2 units) and sum
  const int32_t *table, *lens, *starts;
  int64_t q_seq, q_head, q_group, o_seq, o_head, o_group;   // elements
  int64_t page_stride, tok_stride, head_stride, ld_table;
  int64_t n_pages;
  int n_seqs, n_heads, group, page_size, max_len, tiles;   // tiles: of a group's rows
  // how the cache's length is split: chunk > 0: in chunks of that many keys or more
  // (pick_chunk), `splits` at most, their parts joined by another kernel; else in
  // `splits` even parts of each sequence's keys, by the CTAs of a cluster
  int splits, chunk;
  int slots;              // CTAs that are resident at once
  int* picked;            // the chunk, for the joining kernel
  Div by_page;            // page_size
  float scale_log2;       // scale * log2(e)
};

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

// The page of a key, read a turn before its place is worked out: the load is not
// waited for in between.
struct PagedKey {
  int t, page;   // the key, -1: none
};
__device__ __forceinline__ PagedKey read_page(const PagedArgs& a, const int32_t* row, int t,
                                              bool is) {
  PagedKey k = {is ? t : -1, 0};
  if (is) k.page = row[a.by_page(t)];
  return k;
}
// Where it is, in elements from the head's first; -1: nowhere.
__device__ __forceinline__ int64_t place_key(const PagedArgs& a, const PagedKey& k) {
  if (k.t < 0) return -1;
  if (k.page < 0 || k.page >= a.n_pages) {
    atomicOr(&g_attend_err, WX_DEVERR_PAGE);
    return -1;
  }
  return k.page * a.page_stride + (k.t - a.by_page(k.t) * a.page_size) * a.tok_stride;
}

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

constexpr int kMaxChunk = 1024;

// The keys of a chunk: as many as make the calls' keys one wave of CTAs, within
// [a.chunk, kMaxChunk]. The host sees only a bound of the lengths, often the table's
// whole width: cut by that, 44 K keys of a 65 K window kept 342 CTAs on 444 places.
// Every thread of a CTA calls it.
__device__ __forceinline__ int pick_chunk(const PagedArgs& a) {
  __shared__ int64_t sh_keys[kPagedWarps];
  if (a.chunk >= kMaxChunk) return a.chunk;
  int64_t keys = 0;
  if ((int)threadIdx.x < a.n_seqs) {
    const int end = min(a.lens[threadIdx.x], a.max_len);
    keys = max(end - (a.starts ? max(a.starts[threadIdx.x], 0) : 0), 0);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) keys += __shfl_xor_sync(0xffffffffu, keys, d);
  if (lane_id() == 0) sh_keys[warp_id()] = keys;
  __syncthreads();
  keys = 0;
#pragma unroll
  for (int u = 0; u < kPagedWarps; u++) keys += sh_keys[u];
  const int64_t want = keys * a.n_heads * a.tiles / a.slots;
  return (int)min(max(want + 15, (int64_t)a.chunk), (int64_t)kMaxChunk) / 16 * 16;
}

// What a CTA (WPI = 4: its four warps share an item) or a warp (WPI = 1: each has an
// item of its own) works on: query rows [g0, g0 + g_n) of a (sequence, head), keys
// [c0, c1).
struct PagedItem {
  int seq, head, split, g0, g_n, c0, c1;
  bool any;   // false: there is no such item
};

template <int WPI, int ROWS, int TOK>
__device__ __forceinline__ PagedItem paged_item(const PagedArgs& a) {
  PagedItem t;
  int tile;
  if constexpr (WPI == 1) {
    const uint32_t i = blockIdx.x * kPagedWarps + warp_id();   // at most 2^31 + 3
    const uint32_t row = i / (uint32_t)a.tiles;
    tile = (int)(i - row * a.tiles);
    t.seq = (int)(row / (uint32_t)a.n_heads);
    t.head = (int)(row - (uint32_t)t.seq * a.n_heads);
    t.split = 0;
    t.any = t.seq < a.n_seqs;
    if (!t.any) return t;
  } else {
    tile = blockIdx.x / a.splits;
    t.split = blockIdx.x - tile * a.splits;
    t.head = blockIdx.y;
    t.seq = blockIdx.z;
    t.any = true;
  }
  t.g0 = tile * ROWS;
  t.g_n = min(ROWS, a.group - t.g0);
  int first, end;
  key_range(a, t.seq, &first, &end);
  if (WPI > 1 && a.chunk > 0) {
    t.c0 = t.c1 = 0;
    if ((int64_t)t.split * a.chunk >= end) {   // empty whatever the chunk
      t.any = t.split == 0 && t.seq == 0 && t.head == 0;
      if (!t.any) return t;
    }
    const int chunk = pick_chunk(a);
    if (t.seq == 0 && t.head == 0 && blockIdx.x == 0 && threadIdx.x == 0) *a.picked = chunk;
    t.c0 = max(first, t.split * chunk);
    t.c1 = min(end, (t.split + 1) * chunk);
  } else {
    const int from = first / TOK * TOK;
    const int n = max(end - from, 0);
    const int per = ((n + TOK - 1) / TOK + a.splits - 1) / a.splits * TOK;
    t.c0 = max(first, from + t.split * per);
    t.c1 = min(end, from + (t.split + 1) * per);
  }
  return t;
}

template <int WPI>
__device__ __forceinline__ void item_sync() {
  if constexpr (WPI == 1)
    __syncwarp();
  else
    __syncthreads();
}

__device__ __forceinline__ float peer_f32(const float* p, int rank) {
  uint32_t r;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
  return v;
}

__device__ __forceinline__ float4 peer_f32x4(const float4* p, int rank) {
  uint32_t r;
  float4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(r)
               : "memory");
  return v;
}

__device__ __forceinline__ float add_scaled(float o, float x, float f) { return fmaf(x, f, o); }
__device__ __forceinline__ float4 add_scaled(float4 o, float4 x, float f) {
  return make_float4(fmaf(x.x, f, o.x), fmaf(x.y, f, o.y), fmaf(x.z, f, o.z), fmaf(x.w, f, o.w));
}

// Parts of one query row's elements joined: (maximum, sum, o) of `n` parts.
template <typename V>
struct Joined {
  float m, l;
  V o;
  template <typename M, typename L, typename O>
  __device__ __forceinline__ Joined(int n, M ms, L ls, O os) : m(-INFINITY), l(0.0f), o{} {
#pragma unroll
    for (int u = 0; u < n; u++) m = fmaxf(m, ms(u));
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int u = 0; u < n; u++) {
      const float f = fast_exp2(ms(u) - ref);
      l = fmaf(ls(u), f, l);
      o = add_scaled(o, os(u), f);
    }
  }
};

// four elements of a row, in one store where their place allows it
__device__ __forceinline__ void store_out4(float* p, float4 x) {
  if (((uintptr_t)p & 15) == 0) {
    *reinterpret_cast<float4*>(p) = x;
  } else {
    p[0] = x.x;
    p[1] = x.y;
    p[2] = x.z;
    p[3] = x.w;
  }
}
__device__ __forceinline__ void store_out4(uint16_t* p, float4 x) {
  const uint32_t lo = pack_bf16x2_rne(x.x, x.y), hi = pack_bf16x2_rne(x.z, x.w);
  if (((uintptr_t)p & 7) == 0) {
    *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
  } else {
    p[0] = (uint16_t)lo;
    p[1] = (uint16_t)(lo >> 16);
    p[2] = (uint16_t)hi;
    p[3] = (uint16_t)(hi >> 16);
  }
}

// The item's warps' parts in shared memory, o as (warp, row, HD), joined and written:
// as the result, as a part for the joining kernel, or over the cluster's CTAs. `mine`
// (ROWS * (HD + 2) floats) is the CTA's own part in a cluster. A thread takes four
// elements of a row at a time: one by one, 40 items of 16 keys of 128 with 13 rows each
// took 6.6 us.
template <typename T, int HD, int ROWS, int WPI>
__device__ __forceinline__ void finish_item(const PagedArgs& a, const PagedItem& t,
                                            const float* part, const float (*sh_m)[ROWS],
                                            const float (*sh_l)[ROWS], float* mine) {
  constexpr int kQuads = HD / 4;
  const int tid = threadIdx.x % (32 * WPI);
  const int64_t row0 = ((int64_t)t.seq * a.n_heads + t.head) * a.group + t.g0;
  T* out = static_cast<T*>(a.out) + t.seq * a.o_seq + t.head * a.o_head + t.g0 * a.o_group;
  auto write = [&](int g, int d, const Joined<float4>& j) {
    const float f = 1.0f / j.l;
    float4 x = make_float4(j.o.x * f, j.o.y * f, j.o.z * f, j.o.w * f);
    if (j.l == 0.0f) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    store_out4(out + g * a.o_group + 4 * d, x);
    if (d == 0 && a.lse)
      a.lse[row0 + g] = j.l == 0.0f ? -INFINITY : (j.m + log2f(j.l)) * 0.6931471805599453f;
  };
  const float4* part4 = reinterpret_cast<const float4*>(part);
  float4* mine4 = reinterpret_cast<float4*>(mine);
  for (int i = tid; i < t.g_n * kQuads; i += 32 * WPI) {
    const int g = i / kQuads, d = i - g * kQuads;
    const Joined<float4> j(
        WPI, [&](int u) { return sh_m[u][g]; }, [&](int u) { return sh_l[u][g]; },
        [&](int u) { return part4[(u * ROWS + g) * kQuads + d]; });
    if (a.chunk > 0) {
      const int64_t at = (row0 + g) * a.splits + t.split;
      reinterpret_cast<float4*>(a.part_o)[at * kQuads + d] = j.o;
      if (d == 0) a.part_ml[at] = make_float2(j.m, j.l);
    } else if (WPI > 1 && a.splits > 1) {
      mine4[g * kQuads + d] = j.o;
      if (d == 0) {
        mine[ROWS * HD + g] = j.m;
        mine[ROWS * (HD + 1) + g] = j.l;
      }
    } else {
      write(g, d, j);
    }
  }
  if (WPI > 1 && a.chunk == 0 && a.splits > 1) {
    asm volatile(
        "barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
            : "memory");
    // each CTA writes its share of the rows
    for (int i = t.split * kPagedThreads + tid; i < t.g_n * kQuads;
         i += a.splits * kPagedThreads) {
      const int g = i / kQuads, d = i - g * kQuads;
      write(g, d,
            Joined<float4>(
                a.splits, [&](int u) { return peer_f32(mine + ROWS * HD + g, u); },
                [&](int u) { return peer_f32(mine + ROWS * (HD + 1) + g, u); },
                [&](int u) { return peer_f32x4(mine4 + g * kQuads + d, u); }));
    }
    // a CTA's shared memory outlives its readers, whose values are in use by now:
    // nothing is handed over
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::
                     : "memory");
  }
}

// ---------------------------------------------------------------- fp32

// Values x[0 .. NV) summed over groups of L lanes, NV <= L: lane i of a group gets
// the sum of x[i / (L / NV)]. Each round halves the values that a lane keeps and
// hands its partner the rest, so NV sums cost NV - 1 shuffles and log2(L / NV) more.
template <int L, int NV>
__device__ __forceinline__ float sum_lanes(float (&x)[NV]) {
  const int lane = lane_id();
#pragma unroll
  for (int n = NV, d = L / 2; n > 1; n >>= 1, d >>= 1) {
    const bool up = lane & d;
#pragma unroll
    for (int i = 0; i < n / 2; i++) {
      const float keep = up ? x[n / 2 + i] : x[i], give = up ? x[i] : x[n / 2 + i];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
    }
  }
#pragma unroll
  for (int d = L / NV / 2; d > 0; d >>= 1) x[0] += __shfl_xor_sync(0xffffffffu, x[0], d);
  return x[0];
}

template <int HD>
struct FmaCfg {
  static constexpr int kTok = 4;                           // keys of one tile
  static constexpr int kStages = HD == 64 ? 4 : 2;
  static constexpr int kTileBytes = kTok * HD * 4;         // K or V of one tile
  static constexpr int kWarpBytes = kStages * 2 * kTileBytes;
  static constexpr int kSmem = kPagedWarps * kWarpBytes;
};

// GT query rows of one (sequence, head) against the keys of one split, fp32:
// products on the FMA pipe, which keeps all of their bits. Each warp takes tiles of
// four keys through a ring of its own, as the bf16 kernel does. A group of HD / 4
// lanes holds a key row, 16 bytes a lane: HD = 64 makes two groups, which take two
// keys of a tile each. A tile's scores are summed over the lanes so that each lane
// ends with one (key, query row) and takes one exponential; the weights come back
// to all lanes through shared memory.
//
// Measured (B200): 64 items of 4096 keys of 128, 2 and 4 rows each, 44 and 46 us (6.1 and
// 5.9 TB/s), 8 rows 59: bound by the issue of some 17 instructions a key and row. From 3
// rows on the tensor cores take over (keys of 64, 4 rows: 320 items of 1500 keys 46 us here
// and 48 there, 64 of 4096 29.9 and 28.4, 44 of up to 2180 13.8 and 11.4; with 2 rows 42.8
// and 47.7, 26.1 and 27.9, 12.9 and 11.3), but short items of 3 or 4 rows stay (1280 of up
// to 256 keys of 128 23.9 and 28.8, of up to 64 11.8 and 17.6), and short ones that are
// many, up to 8 rows at a time (see PagedCut).
template <int HD, int GT, int WPI>
__global__ void __launch_bounds__(kPagedThreads, 4) paged_attention_fma_kernel(const PagedArgs a) {
  using Cfg = FmaCfg<HD>;
  constexpr int kLanes = HD / 4, kGroups = 32 / kLanes;
  constexpr int kKeys = Cfg::kTok / kGroups;         // of a group
  constexpr int NV = kKeys * GT, kDup = kLanes / NV; // lanes with the same score
  static_assert(NV <= kLanes, "");
  extern __shared__ __align__(128) char smem[];
  __shared__ float sh_m[kPagedWarps][GT], sh_l[kPagedWarps][GT];
  __shared__ __align__(16) float sh_p[kPagedWarps][Cfg::kTok * GT];
  pdl_wait();

  const PagedItem it = paged_item<WPI, GT, Cfg::kTok>(a);
  // nothing to do; in a cluster the others still wait for this CTA
  if (!it.any || (it.c0 >= it.c1 && a.chunk > 0)) return;
  const int seq = it.seq, head = it.head, g0 = it.g0, g_n = it.g_n, c0 = it.c0, c1 = it.c1;

  const int lane = lane_id(), w = warp_id(), sub = lane % kLanes, grp = lane / kLanes;
  const float* kp = static_cast<const float*>(a.k) + head * a.head_stride;
  const float* vp = static_cast<const float*>(a.v) + head * a.head_stride;
  const int32_t* row = a.table + seq * a.ld_table;
  char* ring = smem + w * Cfg::kWarpBytes;
  const uint32_t ring_at = smem_u32(ring);

  constexpr int kTurn = WPI * Cfg::kTok;   // keys of one turn of the item's warps
  const int base = c0 + w % WPI * Cfg::kTok;
  const int n_mine = base < c1 ? (c1 - base + kTurn - 1) / kTurn : 0;
  // key (tile i, lane % kTok)
  auto locate = [&](int i) {
    const int t = base + i * kTurn + lane % Cfg::kTok;
    return read_page(a, row, t, i < n_mine && t < c1);
  };
  auto fetch = [&](int i, int64_t where) {
    const uint32_t slot = ring_at + (i % Cfg::kStages) * 2 * Cfg::kTileBytes;
#pragma unroll
    for (int j = 0; j < kKeys; j++) {
      const int r = j * kGroups + grp;
      const int64_t at = __shfl_sync(0xffffffffu, where, r);
      const uint32_t dst = slot + r * HD * 4 + sub * 16;
      const int64_t from = at < 0 ? 0 : at + sub * 4;
      cp_async16(dst, kp + from, at >= 0);
      cp_async16(dst + Cfg::kTileBytes, vp + from, at >= 0);
    }
  };
  PagedKey next = locate(0);
  uint32_t live[Cfg::kStages];   // bit r: key r of the tile in this slot is one
#pragma unroll
  for (int i = 0; i < Cfg::kStages - 1; i++) {
    const int64_t where = place_key(a, next);
    next = locate(i + 1);
    live[i] = __ballot_sync(0xffffffffu, where >= 0);
    if (i < n_mine) fetch(i, where);
    cp_async_commit();
  }

  // query rows in pairs, so that one packed FMA serves two of them (GT = 1: one row
  // and a zero one)
  constexpr int GP = (GT + 1) / 2;
  const float* q = static_cast<const float*>(a.q) + seq * a.q_seq + head * a.q_head;
  float2 qr[GP][4], o[GP][4];
#pragma unroll
  for (int g = 0; g < GP; g++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      o[g][e] = make_float2(0.0f, 0.0f);
      const float* p = q + (g0 + 2 * g) * a.q_group + sub * 4 + e;
      qr[g][e].x = 2 * g < g_n ? p[0] * a.scale_log2 : 0.0f;
      qr[g][e].y = 2 * g + 1 < g_n ? p[a.q_group] * a.scale_log2 : 0.0f;
    }
  // this lane's score: key my_r of the tile (r counts as the ring's rows), row my_g
  const int my = sub / kDup, my_g = my % GT, my_r = my / GT * kGroups + grp;
  float m = -INFINITY, l = 0.0f;   // of row my_g: the warp's reference, this lane's sum

#pragma unroll 1
  for (int i = 0; i < n_mine; i++) {
    {
      const int f = i + Cfg::kStages - 1;
      const int64_t where = place_key(a, next);
      next = locate(f + 1);
      live[Cfg::kStages - 1] = __ballot_sync(0xffffffffu, where >= 0);
      __syncwarp();   // every lane has read the slot that is filled now
      if (f < n_mine) fetch(f, where);
      cp_async_commit();
    }
    cp_async_wait<Cfg::kStages - 1>();
    __syncwarp();
    const float4* kt = reinterpret_cast<const float4*>(
        ring + (i % Cfg::kStages) * 2 * Cfg::kTileBytes);
    const float4* vt = kt + Cfg::kTileBytes / 16;

    float s[NV];
#pragma unroll
    for (int u = 0; u < kKeys; u++) {
      const float4 k = kt[(u * kGroups + grp) * kLanes + sub];
      const float kd[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int g = 0; g < GP; g++) {
        float2 x = __fmul2_rn(qr[g][0], make_float2(kd[0], kd[0]));
#pragma unroll
        for (int e = 1; e < 4; e++) x = __ffma2_rn(qr[g][e], make_float2(kd[e], kd[e]), x);
        s[u * GT + 2 * g] = x.x;
        if (GT > 1) s[u * GT + (2 * g + 1) % GT] = x.y;
      }
    }
    float x = sum_lanes<kLanes, NV>(s);
    if (!(live[0] >> my_r & 1)) x = -INFINITY;
    if (__any_sync(0xffffffffu, x > m + 8.0f)) {
      // a new reference: the row's largest score so far, over keys and groups
      float y = x;
#pragma unroll
      for (int d = kLanes / 2; d >= GT * kDup; d >>= 1)
        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
      if (kGroups == 2) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
      y = fmaxf(y, m);
      const float f = m == -INFINITY ? 0.0f : fast_exp2(m - y);
      m = y;
      l *= f;
#pragma unroll
      for (int g = 0; g < GP; g++) {
        const float2 fg = {__shfl_sync(0xffffffffu, f, 2 * g * kDup),
                           __shfl_sync(0xffffffffu, f, (2 * g + 1) % GT * kDup)};
#pragma unroll
        for (int e = 0; e < 4; e++) o[g][e] = __fmul2_rn(o[g][e], fg);
      }
    }
    x = fast_exp2(x - (m == -INFINITY ? 0.0f : m));
    l += x;
    if (kDup == 1 || sub % kDup == 0) sh_p[w][my_r * GT + my_g] = x;
    __syncwarp();
#pragma unroll
    for (int u = 0; u < kKeys; u++) {
      const int r = u * kGroups + grp;
      const float4 v = vt[r * kLanes + sub];
      const float vd[4] = {v.x, v.y, v.z, v.w};
      float2 p[GP];
      if constexpr (GT >= 4) {
#pragma unroll
        for (int g = 0; g < GP; g += 2) {
          const float4 x = *reinterpret_cast<const float4*>(&sh_p[w][r * GT + 2 * g]);
          p[g] = make_float2(x.x, x.y);
          p[g + 1] = make_float2(x.z, x.w);
        }
      } else {
        p[0] = make_float2(sh_p[w][r * GT], GT > 1 ? sh_p[w][r * GT + GT - 1] : 0.0f);
      }
#pragma unroll
      for (int g = 0; g < GP; g++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          o[g][e] = __ffma2_rn(p[g], make_float2(vd[e], vd[e]), o[g][e]);
    }
#pragma unroll
    for (int j = 0; j + 1 < Cfg::kStages; j++) live[j] = live[j + 1];
  }
  // the row's sum over its keys' lanes and the groups
#pragma unroll
  for (int d = kLanes / 2; d >= GT * kDup; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  if (kGroups == 2) {
    l += __shfl_xor_sync(0xffffffffu, l, 16);
#pragma unroll
    for (int g = 0; g < GP; g++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        o[g][e].x += __shfl_xor_sync(0xffffffffu, o[g][e].x, 16);
        o[g][e].y += __shfl_xor_sync(0xffffffffu, o[g][e].y, 16);
      }
  }
  cp_async_wait<0>();
  pdl_launch_dependents();
  item_sync<WPI>();   // the item's rings become its warps' parts of o

  float* part = reinterpret_cast<float*>(smem + (WPI == 1 ? w * Cfg::kWarpBytes : 0));
  float* my_part = part + w % WPI * GT * HD;
  if (lane < kLanes) {
#pragma unroll
    for (int g = 0; g < GP; g++) {
      *reinterpret_cast<float4*>(my_part + 2 * g * HD + sub * 4) =
          make_float4(o[g][0].x, o[g][1].x, o[g][2].x, o[g][3].x);
      if (GT > 1)
        *reinterpret_cast<float4*>(my_part + (2 * g + 1) * HD + sub * 4) =
            make_float4(o[g][0].y, o[g][1].y, o[g][2].y, o[g][3].y);
    }
    if (my_r == 0 && sub % kDup == 0) {
      sh_m[w][my_g] = m;
      sh_l[w][my_g] = l;
    }
  }
  item_sync<WPI>();
  const int w0 = WPI == 1 ? w : 0;
  finish_item<float, HD, GT, WPI>(a, it, part, sh_m + w0, sh_l + w0, part + WPI * GT * HD);
}

// ---------------------------------------------------------------- tensor cores

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
  static constexpr int kStages = 2;
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
// the rescaling is rare. A decode step has 1 to 16 query rows a head: 128-row
// accumulators in tensor memory would stand nearly empty, and mma.sync is far from its
// limit here.
//
// Bound by the memory: measured (B200), 16 clips' 1500 frames of 20 heads of 64, five
// beams each (123 MB) 24.6 us, 5.0 TB/s; 64 clips 88 us, 5.6 TB/s; 64 sequences of 1 to
// 16384 tokens, 8 heads of 128 with 4 query rows (504 MB) 89 us, 5.7 TB/s; 5 beams'
// first tokens 2.9 us, a launch. Products on the FMA pipe took 110 and 200 us for the
// first and third; four-stage rings, with fewer CTAs on an SM, 34 and 99.
template <int HD, int NT, int WPI>
__global__ void __launch_bounds__(kPagedThreads) paged_attention_mma_kernel(const PagedArgs a) {
  using Cfg = MmaCfg<HD>;
  constexpr int kRows = 8 * NT, kSteps = HD / 16, kCpr = HD / 8;   // 16-byte chunks of a row
  constexpr int kLoads = kTok * kCpr / 32;                         // a lane, K or V
  extern __shared__ __align__(128) char smem[];
  __shared__ float sh_m[kPagedWarps][kRows], sh_l[kPagedWarps][kRows];
  pdl_wait();

  const PagedItem it = paged_item<WPI, kRows, kTok>(a);
  // nothing to do; in a cluster the others still wait for this CTA
  if (!it.any || (it.c0 >= it.c1 && a.chunk > 0)) return;
  const int seq = it.seq, head = it.head, g0 = it.g0, g_n = it.g_n, c0 = it.c0, c1 = it.c1;

  const int lane = lane_id(), w = warp_id();
  const uint16_t* kp = static_cast<const uint16_t*>(a.k) + head * a.head_stride;
  const uint16_t* vp = static_cast<const uint16_t*>(a.v) + head * a.head_stride;
  const int32_t* row = a.table + seq * a.ld_table;
  const uint32_t ring = smem_u32(smem) + w * Cfg::kWarpBytes;

  // the warp's tiles: kTok keys from base + kTurn i on
  constexpr int kTurn = WPI * kTok;
  const int base = c0 / kTok * kTok + w % WPI * kTok;
  const int n_mine = base < c1 ? (c1 - base + kTurn - 1) / kTurn : 0;

  // key (tile i, lane % 16)
  auto locate = [&](int i) {
    const int t = base + i * kTurn + (lane & 15);
    return read_page(a, row, t, i < n_mine && t >= c0 && t < c1);
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

  PagedKey next = locate(0);
  uint32_t live[Cfg::kStages];   // bit r: key r of the tile in this slot is one
#pragma unroll
  for (int i = 0; i < Cfg::kStages - 1; i++) {
    const int64_t where = place_key(a, next);
    next = locate(i + 1);
    live[i] = __ballot_sync(0xffffffffu, where >= 0);
    if (i < n_mine) fetch(i, where);
    cp_async_commit();
  }

  // Q^T in fragments: row n = lane / 4, dimensions 2 (lane % 4) + {0, 1, 8, 9}
  uint32_t qf[NT][kSteps][2];
  {
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + seq * a.q_seq + head * a.q_head;
    auto load = [&](auto pair) {
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const int g = n * 8 + lane / 4;
        const uint16_t* p = q + (g0 + g) * a.q_group + (lane & 3) * 2;
#pragma unroll
        for (int k = 0; k < kSteps; k++)
#pragma unroll
          for (int h = 0; h < 2; h++) qf[n][k][h] = g < g_n ? pair(p + k * 16 + h * 8) : 0;
      }
    };
    if ((((uintptr_t)q | (uint64_t)(a.q_group * 2)) & 3) == 0)
      load([](const uint16_t* p) { return *reinterpret_cast<const uint32_t*>(p); });
    else
      load([](const uint16_t* p) { return (uint32_t)p[0] | ((uint32_t)p[1] << 16); });
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
      const int64_t where = place_key(a, next);
      next = locate(f + 1);
      live[Cfg::kStages - 1] = __ballot_sync(0xffffffffu, where >= 0);
      __syncwarp();   // every lane has read the slot that is filled now
      if (f < n_mine) fetch(f, where);
      cp_async_commit();
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
  pdl_launch_dependents();
  item_sync<WPI>();   // the item's rings become its warps' parts of o

  float* part = reinterpret_cast<float*>(smem + (WPI == 1 ? w * Cfg::kWarpBytes : 0));
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
      float* p = part + (w % WPI * kRows + g) * HD + (lane >> 2);
#pragma unroll
      for (int k = 0; k < kSteps; k++) {
        p[k * 16] = o[n][k][h];
        p[k * 16 + 8] = o[n][k][2 + h];
      }
    }
  item_sync<WPI>();
  const int w0 = WPI == 1 ? w : 0;
  finish_item<uint16_t, HD, kRows, WPI>(a, it, part, sh_m + w0, sh_l + w0,
                                        part + WPI * kRows * HD);
}

// ---------------------------------------------------------------- fp32 on tensor cores

// d += a (16 x 8, row) * b (8 x 8, col), tf32 in (fp32 whose lowest 13 bits are 0),
// fp32 out
__device__ __forceinline__ void mma_tf32(float (&d)[4], const float (&a)[4], float b0, float b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
        "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// x in two parts of 11 bits, the first rounded (to infinity at the very top, which the
// kernel meets as it does infinities), the second cut: within 2^-22 of x together. NaN
// stays NaN in the second.
__device__ __forceinline__ float tf32_hi(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xFFFFE000u);
}
__device__ __forceinline__ float tf32_lo(float x, float hi) {
  return __uint_as_float(__float_as_uint(x - hi) & 0xFFFFE000u);
}
__device__ __forceinline__ void split_tf32(const float (&x)[4], float (&hi)[4], float (&lo)[4]) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    hi[e] = tf32_hi(x[e]);
    lo[e] = tf32_lo(x[e], hi[e]);
  }
}

// outside [2^-102, 2^64], 0 aside; by exponents, since compares of floats with their
// branches were 2 us of a call with 16 rows
__device__ __forceinline__ bool far_from_one(float x) {
  const uint32_t b = __float_as_uint(x) << 1;
  return (b != 0) & (b - (25u << 24) > (166u << 24));
}

template <int HD, int HALVES>
struct Tf32Cfg {
  static constexpr int kTileBytes = kTok * HD * 4;           // K or V of one tile
  static constexpr int kWarpBytes = HALVES * kTileBytes;     // a ring of K and V tiles
  static constexpr int kQueryBytes = HD / 8 * 32 * 16;   // 8 rows in two parts or 16 whole
  static constexpr int kSmem = kPagedWarps * kWarpBytes + kQueryBytes;
};

// Up to 8 NT query rows of one (sequence, head) against the keys of one split, fp32: the
// products of the bf16 kernel (S^T = K Q^T, O^T = V^T P^T) on tf32 operands. Each number
// is in two parts and three of the four products of parts are taken, the fourth being
// below 2^-22 of a product: 2^-20 in all, a few roundings of fp32. A part below 2^-126
// counts as 0: an error of 2^-126 |v| in a weight's share of o and of 2^-126 p in a value's,
// and in the scores none that shows, since a query with numbers so small or so large that
// it could (see `whole`) gets its scores as sums of whole products. A key of 128 costs
// some 90 instructions for up to 8 rows, mostly the splitting, where the FMA kernel takes
// 17 a row.
//
// A warp's ring holds K and V tiles in turn: three of them, so that K of the next tile is
// under way while this tile's V waits, or two, which for keys of 128 leaves room for a
// third CTA on an SM. Which dimension stands in which column of a product is
// free as long as both operands agree (and for V, which row), so every operand is read
// four dimensions at a time: K's columns t and t + 4 of two steps are dimensions
// 4 t .. 4 t + 3 of 16, V's rows g and g + 8 of two tiles are 4 g .. 4 g + 3 of 32.
//
// Measured (B200), the FMA kernel (8 rows at a time) in brackets: 320 items of 1500 keys
// of 64, 5 rows each, 47 us (81); 64 items of 4096 keys, 8 rows: of 64 29 (40), of 128 47
// (59), 16 rows: 38 (70) and 60 (108). Few warps carry it, twelve on an SM: bound by
// latency, of the copies and of the chain from a tile's scores to its weights (5.2 TB/s
// for 5 rows of 64; for 8 of 128 with eight warps, issue 37 % and tensor cores 23 % of
// their cycles). Four CTAs on an SM in place of three for keys of 64, with 128 registers:
// 58.7 us where three took 53.6. First parts cut in place of rounded: twice the error, and
// no faster. Two tiles in place of three for keys of 128 and 5 rows: 320 items of 1500 keys
// 81 us and 115 (444 places for CTAs, not 296), 44 items of up to 2180 16.4 and 22.5, but
// 25.9 and 24.9 for 87 K keys in chunks, where the places are filled either way.
template <int HD, int NT, int HALVES>
__global__ void __launch_bounds__(kPagedThreads, HD == 64 || (NT == 1 && HALVES == 2) ? 3 : 2)
    paged_attention_tf32_kernel(const PagedArgs a) {
  using Cfg = Tf32Cfg<HD, HALVES>;
  constexpr int kRows = 8 * NT, kSteps = HD / 8, kBlocks = HD / 32, kCpr = HD / 4;
  constexpr int kLoads = kTok * kCpr / 32;   // a lane, K or V
  constexpr int kLd = NT == 1 ? 8 : 24;      // of a key's weights: no bank is met twice
  extern __shared__ __align__(128) char smem[];
  __shared__ float sh_m[kPagedWarps][kRows], sh_l[kPagedWarps][kRows];
  __shared__ __align__(16) float sh_p[kPagedWarps][kTok][kLd];
  pdl_wait();

  const PagedItem it = paged_item<4, kRows, kTok>(a);
  // nothing to do; in a cluster the others still wait for this CTA
  if (!it.any || (it.c0 >= it.c1 && a.chunk > 0)) return;
  const int seq = it.seq, head = it.head, g0 = it.g0, g_n = it.g_n, c0 = it.c0, c1 = it.c1;

  const int lane = lane_id(), w = warp_id(), g = lane >> 2, t = lane & 3;
  const float* kp = static_cast<const float*>(a.k) + head * a.head_stride;
  const float* vp = static_cast<const float*>(a.v) + head * a.head_stride;
  const float* q = static_cast<const float*>(a.q) + seq * a.q_seq + head * a.q_head;
  const int32_t* row = a.table + seq * a.ld_table;
  char* ring = smem + w * Cfg::kWarpBytes;
  const uint32_t ring_at = smem_u32(ring);
  char* sh_q = smem + kPagedWarps * Cfg::kWarpBytes;

  constexpr int kTurn = kPagedWarps * kTok;
  const int base = c0 / kTok * kTok + w * kTok;
  const int n_mine = base < c1 ? (c1 - base + kTurn - 1) / kTurn : 0;
  auto locate = [&](int i) {
    const int key = base + i * kTurn + (lane & 15);
    return read_page(a, row, key, i < n_mine && key >= c0 && key < c1);
  };
  // half h: K (even) or V (odd) of tile h / 2, whose keys are at `where`. Chunks of 16
  // bytes are exchanged within a row so that a warp's reads meet no bank twice: K's
  // eight lanes read two rows, V's four. A tile with all its keys needs no tests (16
  // clips' frames 53.7 -> 48.3 us)
  auto fetch = [&](int h, int64_t where) {
    const uint32_t slot = ring_at + h % HALVES * Cfg::kTileBytes;
    const float* from = (h & 1 ? vp : kp) + lane % kCpr * 4;
    auto rows = [&](auto copy) {
#pragma unroll
      for (int j = 0; j < kLoads; j++) {
        const int r = j * (32 / kCpr) + lane / kCpr;
        const int64_t at = __shfl_sync(0xffffffffu, where, r);
        const int mix = h & 1 ? (r & 3) << 1 : (r & 1) << 2;
        copy(slot + r * HD * 4 + ((lane % kCpr ^ mix) << 4), at);
      }
    };
    if (__all_sync(0xffffffffu, where >= 0))
      rows([&](uint32_t to, int64_t at) { cp_async16(to, from + at, true); });
    else
      rows([&](uint32_t to, int64_t at) { cp_async16(to, from + (at < 0 ? 0 : at), at >= 0); });
  };
  PagedKey next = locate(0);
  int64_t where = place_key(a, next);   // of the tile fetched last
  next = locate(1);
  uint32_t live = __ballot_sync(0xffffffffu, where >= 0), live_next = 0;
  if (n_mine > 0) fetch(0, where);
  cp_async_commit();
  if (HALVES == 3) {
    if (n_mine > 0) fetch(1, where);
    cp_async_commit();
  }

  // Q^T's fragments in the order of the steps: in two parts for one tile of rows, and
  // whole for two, which leaves room for two CTAs on an SM
  auto query = [&](int r, int d) {
    return r < g_n ? q[(g0 + r) * a.q_group + d] * a.scale_log2 : 0.0f;
  };
  bool extreme = false;
  constexpr int kFrags = kSteps * 32 / kPagedThreads;   // a thread's
  float2 qf[kFrags][NT];
#pragma unroll
  for (int j = 0; j < kFrags; j++) {
    const int i = threadIdx.x + j * kPagedThreads;
    const int d = (i >> 6) * 16 + (i & 3) * 4 + (i >> 5 & 1) * 2, r = i >> 2 & 7;
#pragma unroll
    for (int z = 0; z < NT; z++) qf[j][z] = make_float2(query(r + 8 * z, d), query(r + 8 * z, d + 1));
  }
#pragma unroll
  for (int j = 0; j < kFrags; j++) {
    const float x = qf[j][0].x, y = qf[j][0].y, hx = tf32_hi(x), hy = tf32_hi(y);
#pragma unroll
    for (int z = 0; z < NT; z++) extreme |= far_from_one(qf[j][z].x) | far_from_one(qf[j][z].y);
    reinterpret_cast<float4*>(sh_q)[threadIdx.x + j * kPagedThreads] =
        NT == 1 ? make_float4(hx, hy, tf32_lo(x, hx), tf32_lo(y, hy))
                : make_float4(x, y, qf[j][NT - 1].x, qf[j][NT - 1].y);
  }
  // what parts below 2^-126 cost a score: of k, hd 2^-126 |q| at most; of q, 2^-126 / |q|
  // of the product. Neither shows while q is within these bounds.
  const bool whole = __syncthreads_or(extreme);

  // o[z][b][i][e]: dimensions 32 b + 4 g + 2 i (e < 2) and the next, rows 8 z + 2 t + e % 2
  float o[NT][kBlocks][2][4] = {}, m[NT][2], l[NT][2] = {};
#pragma unroll
  for (int z = 0; z < NT; z++) m[z][0] = m[z][1] = -INFINITY;

#pragma unroll 1
  for (int i = 0; i < n_mine; i++) {
    __syncwarp();   // every lane has read the slot that is filled now
    if (HALVES == 2) fetch(2 * i + 1, where);
    where = place_key(a, next);
    next = locate(i + 2);
    live_next = __ballot_sync(0xffffffffu, where >= 0);
    if (HALVES == 3 && i + 1 < n_mine) fetch(2 * i + 2, where);
    cp_async_commit();
    cp_async_wait<HALVES - 1>();
    __syncwarp();
    const float4* kt =
        reinterpret_cast<const float4*>(ring + 2 * i % HALVES * Cfg::kTileBytes);
    // six chains of products for a tile of rows: one would wait for each step's result
    float s[NT][2][3][4] = {};
#pragma unroll
    for (int j = 0; j < kSteps / 2; j++) {
      const int c = (4 * j + t) ^ ((g & 1) << 2);
      const float4 x = kt[g * kCpr + c], y = kt[(g + 8) * kCpr + c];
      const float k[2][4] = {{x.x, y.x, x.y, y.y}, {x.z, y.z, x.w, y.w}};
#pragma unroll
      for (int u = 0; u < 2; u++) {
        float hi[4], lo[4];
        split_tf32(k[u], hi, lo);
        const float4 b = reinterpret_cast<const float4*>(sh_q)[(2 * j + u) * 32 + lane];
        const float q_all[4] = {b.x, b.y, b.z, b.w};
        float q_hi[4], q_lo[4];
        if constexpr (NT > 1) split_tf32(q_all, q_hi, q_lo);
#pragma unroll
        for (int z = 0; z < NT; z++) {
          const float h0 = NT > 1 ? q_hi[2 * z] : b.x, h1 = NT > 1 ? q_hi[2 * z + 1] : b.y;
          const float l0 = NT > 1 ? q_lo[2 * z] : b.z, l1 = NT > 1 ? q_lo[2 * z + 1] : b.w;
          mma_tf32(s[z][u][0], hi, h0, h1);
          mma_tf32(s[z][u][1], hi, l0, l1);
          mma_tf32(s[z][u][2], lo, h0, h1);
        }
      }
    }
    // keys g and g + 8, query rows 8 z + 2 t + {0, 1}
    const bool in0 = live >> g & 1, in1 = live >> (g + 8) & 1;
    float x[NT][4];
    bool odd = whole;
#pragma unroll
    for (int z = 0; z < NT; z++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        x[z][e] = (s[z][0][0][e] + s[z][1][0][e]) +
                  ((s[z][0][1][e] + s[z][1][1][e]) + (s[z][0][2][e] + s[z][1][2][e]));
        odd |= x[z][e] != x[z][e];
      }
    if (__any_sync(0xffffffffu, odd)) {
      // an infinite number has no parts: the scores as sums of whole products
#pragma unroll
      for (int e = 0; e < 4 * NT; e++) {
        const int r = g + (e >> 1 & 1) * 8;
        float y = 0.0f;
        for (int d = 0; d < HD; d++) {
          const float kd = reinterpret_cast<const float*>(
              kt)[r * HD + (((d >> 2) ^ ((r & 1) << 2)) << 2) + (d & 3)];
          y = fmaf(query((e >> 2) * 8 + 2 * t + (e & 1), d), kd, y);
        }
        x[e >> 2][e & 3] = y;
      }
    }
    float most[NT][2];
    bool more = false;
#pragma unroll
    for (int z = 0; z < NT; z++) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (!(e < 2 ? in0 : in1)) x[z][e] = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        most[z][h] = fmaxf(x[z][h], x[z][2 + h]);
        more |= most[z][h] > m[z][h] + 8.0f;
      }
    }
    if (__any_sync(0xffffffffu, more)) {
#pragma unroll
      for (int z = 0; z < NT; z++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float y = most[z][h];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
          y = fmaxf(y, m[z][h]);
          const float f = m[z][h] == -INFINITY ? 0.0f : fast_exp2(m[z][h] - y);
          m[z][h] = y;
          l[z][h] *= f;
#pragma unroll
          for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[z][b][e >> 1][(e & 1) * 2 + h] *= f;
        }
    }
#pragma unroll
    for (int z = 0; z < NT; z++) {
      // a row that has met no score above -inf yet: its reference is 0
      const float r0 = m[z][0] == -INFINITY ? 0.0f : m[z][0];
      const float r1 = m[z][1] == -INFINITY ? 0.0f : m[z][1];
#pragma unroll
      for (int e = 0; e < 4; e++) x[z][e] = fast_exp2(x[z][e] - (e & 1 ? r1 : r0));
      l[z][0] += x[z][0] + x[z][2];
      l[z][1] += x[z][1] + x[z][3];
      // from accumulators to operands: keys t and t + 4 of either eight, row g
      *reinterpret_cast<float2*>(&sh_p[w][g][8 * z + 2 * t]) = make_float2(x[z][0], x[z][1]);
      *reinterpret_cast<float2*>(&sh_p[w][g + 8][8 * z + 2 * t]) = make_float2(x[z][2], x[z][3]);
    }
    __syncwarp();   // also: every lane has read K's slot
    if (i + 1 < n_mine) fetch(2 * i + HALVES, where);
    cp_async_commit();
    float p_hi[NT][4], p_lo[NT][4];
#pragma unroll
    for (int z = 0; z < NT; z++) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; e++) p[e] = sh_p[w][t + 4 * e][8 * z + g];
      split_tf32(p, p_hi[z], p_lo[z]);
    }
    cp_async_wait<HALVES - 1>();
    __syncwarp();
    const float4* vt =
        reinterpret_cast<const float4*>(ring + (2 * i + 1) % HALVES * Cfg::kTileBytes);
    // a tile's products are summed by themselves, then added in fp32; two blocks of
    // dimensions share a vote on what has no parts
#pragma unroll
    for (int b0 = 0; b0 < kBlocks; b0 += 2) {
      float d[NT][2][2][4] = {};
#pragma unroll
      for (int b = 0; b < 2; b++) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int c = (8 * (b0 + b) + g) ^ (t << 1);
          const float4 v0 = vt[(8 * u + t) * kCpr + c], v1 = vt[(8 * u + t + 4) * kCpr + c];
          const float v[2][4] = {{v0.x, v0.y, v1.x, v1.y}, {v0.z, v0.w, v1.z, v1.w}};
#pragma unroll
          for (int n = 0; n < 2; n++) {
            float hi[4], lo[4];
            split_tf32(v[n], hi, lo);
#pragma unroll
            for (int z = 0; z < NT; z++) {
              mma_tf32(d[z][b][n], lo, p_hi[z][2 * u], p_hi[z][2 * u + 1]);
              mma_tf32(d[z][b][n], hi, p_lo[z][2 * u], p_lo[z][2 * u + 1]);
              mma_tf32(d[z][b][n], hi, p_hi[z][2 * u], p_hi[z][2 * u + 1]);
            }
          }
        }
      }
      odd = false;
#pragma unroll
      for (int e = 0; e < 16 * NT; e++) {
        const float y = d[e >> 4][e >> 3 & 1][e >> 2 & 1][e & 3];
        odd |= y != y;
      }
      if (__any_sync(0xffffffffu, odd)) {
        // as above
#pragma unroll
        for (int e = 0; e < 16 * NT; e++) {
          const int b = e >> 3 & 1, n = e >> 2 & 1;
          const int dim = 32 * (b0 + b) + 4 * g + 2 * n + (e >> 1 & 1);
          float y = 0.0f;
          for (int r = 0; r < kTok; r++) {
            const float vd = reinterpret_cast<const float*>(
                vt)[r * HD + (((dim >> 2) ^ ((r & 3) << 1)) << 2) + (dim & 3)];
            y = fmaf(sh_p[w][r][8 * (e >> 4) + 2 * t + (e & 1)], vd, y);
          }
          d[e >> 4][b][n][e & 3] = y;
        }
      }
#pragma unroll
      for (int e = 0; e < 16 * NT; e++)
        o[e >> 4][b0 + (e >> 3 & 1)][e >> 2 & 1][e & 3] +=
            d[e >> 4][e >> 3 & 1][e >> 2 & 1][e & 3];
    }
    live = live_next;
  }
  cp_async_wait<0>();
  pdl_launch_dependents();
  __syncthreads();   // the rings become the warps' parts of o

  float* part = reinterpret_cast<float*>(smem);   // [warp][row][HD]
#pragma unroll
  for (int z = 0; z < NT; z++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float sum = l[z][h];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const int r = 8 * z + 2 * t + h;
      if (lane < 4) {
        sh_m[w][r] = m[z][h];
        sh_l[w][r] = sum;
      }
#pragma unroll
      for (int b = 0; b < kBlocks; b++)
#pragma unroll
        for (int n = 0; n < 2; n++)
          *reinterpret_cast<float2*>(part + (w * kRows + r) * HD + 32 * b + 4 * g + 2 * n) =
              make_float2(o[z][b][n][h], o[z][b][n][2 + h]);
    }
  __syncthreads();
  finish_item<float, HD, kRows, 4>(a, it, part, sh_m, sh_l, part + kPagedWarps * kRows * HD);
}

// A query row's parts joined by W warps, which take the splits that held keys in turn
// and are joined in order: one where rows are many (four rows a CTA), 32 where they are
// few and their splits many. Measured (B200) with 273 parts for each of 16 rows, the
// whole call: W = 32 29 us, 8 33, 1 87.
template <typename T, int HD, int W>
__global__ void __launch_bounds__(W == 1 ? kPagedThreads : 32 * W)
    paged_attention_join_kernel(const PagedArgs a, int64_t rows) {
  pdl_begin();
  constexpr int N = HD / 32;
  __shared__ float sh_m[W], sh_l[W], sh_o[W][W == 1 ? 1 : HD];
  const int lane = lane_id(), w = W == 1 ? 0 : warp_id();
  // at most 2^31 - 1 rows
  const uint32_t row = W == 1 ? blockIdx.x * kPagedWarps + warp_id() : blockIdx.x;
  if (row >= rows) return;
  const uint32_t item = row / (uint32_t)a.group, seq = item / (uint32_t)a.n_heads;
  const int g = (int)(row - item * a.group), head = (int)(item - seq * a.n_heads);
  const int64_t r = row;
  int first, end;
  key_range(a, seq, &first, &end);
  const int chunk = a.chunk >= kMaxChunk ? a.chunk : *a.picked;
  // this warp's splits: s0 + W i for i < n
  const int s0 = first / chunk + w, s1 = first < end ? (end + chunk - 1) / chunk : 0;
  const int n = s0 < s1 ? (s1 - s0 + W - 1) / W : 0;
  const float2* ml = a.part_ml + r * a.splits + s0;
  const float* p = a.part_o + (r * a.splits + s0) * HD + lane * N;
  auto read = [&](int i) { return i < n ? ml[W * i] : make_float2(-INFINITY, 0.0f); };
  float2 my = read(lane);   // lane i - i0 holds part i
  float mx = my.x;
  for (int i = 32 + lane; i < n; i += 32) mx = fmaxf(mx, read(i).x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  const float ref = mx == -INFINITY ? 0.0f : mx;
  float sum = 0.0f, x[N] = {};
  for (int i0 = 0; i0 < n; i0 += 32) {
    if (i0 > 0) my = read(i0 + lane);
    const float f = fast_exp2(my.x - ref);
    sum = fmaf(my.y, f, sum);
    const int m = min(32, n - i0);
    constexpr int kAhead = 8;   // parts in flight
    for (int i = 0; i < m; i += kAhead) {
      float y[kAhead][N];
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        if (i + j >= m) continue;
        const float* from = p + (int64_t)(W * (i0 + i + j)) * HD;
        if constexpr (N == 4)
          *reinterpret_cast<float4*>(y[j]) = *reinterpret_cast<const float4*>(from);
        else
          *reinterpret_cast<float2*>(y[j]) = *reinterpret_cast<const float2*>(from);
      }
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        if (i + j >= m) continue;
        const float fi = __shfl_sync(0xffffffffu, f, i + j);
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = fmaf(y[j][e], fi, x[e]);
      }
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  T* out = static_cast<T*>(a.out) + seq * a.o_seq + head * a.o_head + g * a.o_group;
  auto lse = [](float m, float l) {
    return l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  };
  if constexpr (W == 1) {
#pragma unroll
    for (int e = 0; e < N; e++) store_out(out + lane * N + e, sum == 0.0f ? 0.0f : x[e] / sum);
    if (lane == 0 && a.lse) a.lse[r] = lse(mx, sum);
  } else {
#pragma unroll
    for (int e = 0; e < N; e++) sh_o[w][lane * N + e] = x[e];
    if (lane == 0) {
      sh_m[w] = mx;
      sh_l[w] = sum;
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d < HD) {
      const Joined<float> j(
          W, [&](int u) { return sh_m[u]; }, [&](int u) { return sh_l[u]; },
          [&](int u) { return sh_o[u][d]; });
      store_out(out + d, j.l == 0.0f ? 0.0f : j.o / j.l);
      if (d == 0 && a.lse) a.lse[r] = lse(j.m, j.l);
    }
  }
}

constexpr int64_t kJoinRows = 8 * 148;   // rows from which on a warp each will do

// How a call's work is cut: query rows of a tile, warps on an item (1 or 4), and for
// long caches chunks of keys that a second kernel joins. In between, a launch splits
// an item over a cluster where that keeps every CTA in the first wave (launch_paged).
//
// Measured (B200), a warp and a CTA for each item of up to 16, 64, 128, 256 keys of 64,
// us: in bf16 with 5 rows, 640 items 4.1 and 4.7, 5.8 and 4.7, 8.4 and 5.6, 12.5 and 6.8;
// 2000 items 5.7 and 9.5, 7.4 and 10.3, 10.0 and 11.3, 15.8 and 13.8; 8000 items 13 and 31,
// 18 and 35, 23 and 39, 32 and 44 (6400 of up to 448 keys: 124 and 116). In fp32 with one
// row, 2000 items 5.0 and 8.1, 11.6 and 10.6, 20 and 14, 37 and 20; 8000 items 12 and 26,
// 24 and 35, 36 and 42, 59 and 54; with 8 rows 26 and 65, 41 and 72, 59 and 80, 94 and 93.
// Tiles of 16 rows against two of 8, 64 items of 4096 keys, 16 rows each: 31.7 and 36.2.
// 320 items of 1500 keys, a cluster of 1, 2, 4, 8 for each: 27.3, 25.8, 31.0, 38.4 us
// (two waves from 4 on; 3 CTAs, which divide no GPC: 33.0; all a us less since queries are
// read in pairs); 20 such items 20.3, 13.3, 8.7, 7.3. 64 sequences to 16384 keys, chunks of at most 512, 1024, 2048: 98, 91, 95;
// their 2048 rows joined by a warp and by 32 warps each, the whole call: 89 and 127.
struct PagedCut {
  int tile, warps, splits, chunk;
};
// An item of short sequences gets a warp where items are many: its time grows with the
// keys, a CTA's with the waves.
constexpr int64_t kShortKeys = 256, kShortItems = 300, kShortBf16 = 10, kShortFp32 = 30;
constexpr int64_t kClusterKeys = 4096;
constexpr int64_t kEarlyKeys = 65536;
constexpr int64_t kMinChunk = 128, kChunkCtas = 32 * 148;
constexpr int64_t kMostParts = 32768;   // bounds the workspace of many long sequences

static PagedCut paged_cut(int64_t n_seqs, int64_t n_heads, int64_t group, int64_t max_len,
                          int dtype) {
  PagedCut c = {};
  if (dtype == WX_DTYPE_BF16) {
    c.tile = group <= 8 ? 8 : 16;
  } else {
    c.tile = group <= 2 ? (int)group
             : group <= 4 && max_len <= kShortKeys ? 4
             : group <= 8 ? 8 : 16;
  }
  c.splits = 1;
  c.warps = 4;
  const int64_t pairs = n_seqs * n_heads, items = pairs * ((group + c.tile - 1) / c.tile);
  const bool fp32 = dtype == WX_DTYPE_F32;
  // a warp's tile in fp32, where it works on the FMA pipe
  const int narrow = !fp32 || c.tile <= 4 ? c.tile : 8;
  const int64_t short_items = pairs * ((group + narrow - 1) / narrow);
  if (max_len <= (fp32 ? kShortKeys / 2 : kShortKeys) &&
      short_items >= kShortItems + max_len * (fp32 ? kShortFp32 : kShortBf16)) {
    c.warps = 1;
    c.tile = narrow;
  } else if (max_len > kClusterKeys) {
    int64_t chunk = max_len * items / kChunkCtas;
    chunk = chunk < kMinChunk ? kMinChunk : chunk > kMaxChunk ? kMaxChunk : chunk;
    if (n_seqs > kPagedThreads) chunk = kMaxChunk;   // pick_chunk leaves it at that
    chunk = std::min(std::max(chunk, max_len * items / kMostParts), max_len);
    chunk = (chunk + 15) / 16 * 16;
    c.chunk = (int)chunk;
    c.splits = (int)((max_len + chunk - 1) / chunk);
  }
  return c;
}

static int64_t paged_space(int64_t rows, const PagedCut& c, int64_t head_dim) {
  return c.chunk > 0 ? 16 + rows * c.splits * (head_dim * 4 + 8) : 0;
}

// What a kernel needs to know of a device before its first launch there: its dynamic
// shared memory's limit is raised, and the CTAs that are resident at once counted.
static cudaError_t prepare_paged(std::atomic<int> (&resident)[64], const void* kernel, int smem,
                                 int* ctas) {
  int dev = 0, n = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64) n = resident[dev].load(std::memory_order_acquire);
  if (n == 0) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kPagedThreads, smem);
    if (e != cudaSuccess) return e;
    n = (n < 1 ? 1 : n) * sm_count();
    if (dev < 64) resident[dev].store(n, std::memory_order_release);
  }
  *ctas = n;
  return cudaSuccess;
}

template <void (*kernel)(const PagedArgs)>
static cudaError_t launch_paged(PagedArgs a, const PagedCut& c, int smem, cudaStream_t st) {
  static std::atomic<int> resident[64] = {};
  int ctas = 0;
  cudaError_t e = prepare_paged(resident, reinterpret_cast<const void*>(kernel), smem, &ctas);
  if (e != cudaSuccess) return e;
  a.slots = ctas;
  const int64_t n_items = (int64_t)a.n_seqs * a.n_heads * a.tiles;
  if (c.chunk == 0 && c.warps > 1)
    while (a.splits < 8 && n_items * a.splits * 2 <= ctas && a.max_len >= 128 * a.splits)
      a.splits *= 2;
  dim3 grid((unsigned)(a.splits * a.tiles), (unsigned)a.n_heads, (unsigned)a.n_seqs);
  if (c.warps == 1) grid = dim3((unsigned)((n_items + kPagedWarps - 1) / kPagedWarps));
  // Placed while the kernel before it ends, a wave of CTAs lands on the SMs that are free
  // first, unevenly: 33.5 us became 36.8 (64 items of 4096 keys). A call of a few us
  // gains half of what a launch costs. Early and not, bf16, heads of 64, us: 100 items of
  // a table of 448 keys (45 K) 5.5 and 6.0, one clip's frames (30 K) 6.0 and 6.4; 320 of
  // 224 (72 K) 7.3 and 7.0, of 448 (143 K) 11.2 and 10.7, of 1500 (481 K) 24.5 and 24.0.
  // Calls of several waves would gain that half again, which this rule leaves: 6400 items
  // of 224 (1.4 M) 59.3 and 60.0.
  const bool early = n_items * a.max_len <= kEarlyKeys;
  return launch(early, kernel, grid, kPagedThreads, smem, c.chunk == 0 ? a.splits : 1, st, a);
}

template <int HD>
static cudaError_t run_mma(const PagedArgs& a, const PagedCut& c, cudaStream_t st) {
  constexpr int smem = MmaCfg<HD>::kSmem;
  if (c.warps == 1)
    return c.tile == 8 ? launch_paged<paged_attention_mma_kernel<HD, 1, 1>>(a, c, smem, st)
                       : launch_paged<paged_attention_mma_kernel<HD, 2, 1>>(a, c, smem, st);
  return c.tile == 8 ? launch_paged<paged_attention_mma_kernel<HD, 1, 4>>(a, c, smem, st)
                     : launch_paged<paged_attention_mma_kernel<HD, 2, 4>>(a, c, smem, st);
}

template <int HD>
static cudaError_t run_fp32(const PagedArgs& a, const PagedCut& c, cudaStream_t st) {
  constexpr int smem = FmaCfg<HD>::kSmem, ring = HD == 128 ? 2 : 3;
  constexpr int smem3 = Tf32Cfg<HD, 3>::kSmem, smem_r = Tf32Cfg<HD, ring>::kSmem;
  if (c.warps == 1) {
    switch (c.tile) {
      case 1: return launch_paged<paged_attention_fma_kernel<HD, 1, 1>>(a, c, smem, st);
      case 2: return launch_paged<paged_attention_fma_kernel<HD, 2, 1>>(a, c, smem, st);
      case 4: return launch_paged<paged_attention_fma_kernel<HD, 4, 1>>(a, c, smem, st);
      default: return launch_paged<paged_attention_fma_kernel<HD, 8, 1>>(a, c, smem, st);
    }
  }
  switch (c.tile) {
    case 1: return launch_paged<paged_attention_fma_kernel<HD, 1, 4>>(a, c, smem, st);
    case 2: return launch_paged<paged_attention_fma_kernel<HD, 2, 4>>(a, c, smem, st);
    case 4: return launch_paged<paged_attention_fma_kernel<HD, 4, 4>>(a, c, smem, st);
    case 8:
      return c.chunk > 0
                 ? launch_paged<paged_attention_tf32_kernel<HD, 1, 3>>(a, c, smem3, st)
                 : launch_paged<paged_attention_tf32_kernel<HD, 1, ring>>(a, c, smem_r, st);
    default: return launch_paged<paged_attention_tf32_kernel<HD, 2, ring>>(a, c, smem_r, st);
  }
}

template <typename T, int HD>
static cudaError_t run_paged(const PagedArgs& a, const PagedCut& c, cudaStream_t st) {
  cudaError_t e;
  if constexpr (sizeof(T) == 2)
    e = run_mma<HD>(a, c, st);
  else
    e = run_fp32<HD>(a, c, st);
  if (e != cudaSuccess || c.chunk == 0) return e;
  const int64_t rows = (int64_t)a.n_seqs * a.n_heads * a.group;
  if (rows >= kJoinRows)
    return launch_after(paged_attention_join_kernel<T, HD, 1>,
                        dim3((unsigned)((rows + kPagedWarps - 1) / kPagedWarps)), kPagedThreads, 0,
                        1, st, a, rows);
  return launch_after(paged_attention_join_kernel<T, HD, 32>, dim3((unsigned)rows), 32 * 32, 0, 1,
                      st, a, rows);
}

static int check_cut(const char* what, int64_t n_seqs, int64_t n_heads, int64_t group,
                     int64_t head_dim, int64_t max_len) {
  if (n_seqs < 0 || n_seqs > 65535 || n_heads < 1 || n_heads > 65535 || group < 1 ||
      group > 65535 || n_seqs * n_heads * group > 0x7fffffff || max_len < 0 ||
      max_len > (1 << 29))
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
  return paged_space(n_seqs * n_heads * group,
                     paged_cut(n_seqs, n_heads, group, max_len, dtype), head_dim);
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
                    n_heads, head_dim, n_pages, page_size, dtype, false));
  if (n_seqs == 0) return WX_OK;
  if (!q || !out || !lens || !table || ld_table < 1)
    return fail(WX_ERR_INVALID, "paged_attention: NULL argument or empty page table");
  if (ld_table * page_size < max_len)
    return fail(WX_ERR_INVALID, "paged_attention: max_len %lld is past the table's %lld pages",
                (long long)max_len, (long long)ld_table);
  const int es = dtype == WX_DTYPE_BF16 ? 2 : 4;
  if (((uintptr_t)q | (uintptr_t)out) % es)
    return fail(WX_ERR_INVALID, "paged_attention: q or out not aligned to its type");
  if (rows_overlap(n_seqs, o_seq_stride, head_dim) ||
      rows_overlap(n_heads, o_head_stride, head_dim) ||
      rows_overlap(group, o_group_stride, head_dim))
    return fail(WX_ERR_INVALID, "paged_attention: out's rows share memory (strides %lld, %lld, %lld)",
                (long long)o_seq_stride, (long long)o_head_stride, (long long)o_group_stride);
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
  a.picked = static_cast<int*>(workspace);
  a.part_o = static_cast<float*>(workspace) + 4;
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
  a.n_seqs = (int)n_seqs;
  a.tiles = (int)((group + c.tile - 1) / c.tile);
  a.splits = c.splits;
  a.chunk = c.chunk;
  a.by_page = Div((uint32_t)page_size);
  a.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = as_stream(stream);
  if (dtype == WX_DTYPE_BF16)
    WX_CUDA_TRY((head_dim == 64 ? run_paged<uint16_t, 64> : run_paged<uint16_t, 128>)(a, c, st));
  else
    WX_CUDA_TRY((head_dim == 64 ? run_paged<float, 64> : run_paged<float, 128>)(a, c, st));
  return check_launch("paged_attention");
}

}  // extern "C"
