// The paged key-value cache of a text decoder on the encoder's features:
// writing tokens into it (append), continuing, ending and growing sequences
// with copy on write (fork), and moving its pages together (compact). No call
// waits for the host: the page plan is made on the device, and the copy kernel
// that follows reads it there.
//
// A cache is two pools (K and V) of n_pages pages of page_size tokens for each
// layer; a row of the page table names a sequence's pages in order, -1 past the
// last. refs[p] counts the table entries that name page p; 0 is free.
#include <cstdint>

#include "common.cuh"
#include "kvcache.cuh"

namespace wx {

// WX_DEVERR_PAGE, kept apart from the library's error word: the bounded waits
// of the other kernels give up when they see that word set.
static __device__ int g_kv_err;

int kv_take_error(int* flags, bool clear) {
  int v = 0;
  WX_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_kv_err, sizeof(int)));
  *flags |= v;
  const int zero = 0;
  if (v && clear) WX_CUDA_TRY(cudaMemcpyToSymbol(g_kv_err, &zero, sizeof(int)));
  return WX_OK;
}

__device__ __forceinline__ void kv_error() { atomicOr(&g_kv_err, WX_DEVERR_PAGE); }

// ---------------------------------------------------------------- append

struct AppendArgs {
  const char* src[2];       // K, V rows
  char* dst[2];             // pools
  int64_t s_seq, s_tok, s_head;                 // source strides, bytes
  int64_t page_stride, tok_stride, head_stride;  // pool strides, bytes
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lens;
  const int32_t* counts;
  int n_tokens, n_heads, row_units;   // units of sizeof(U) bytes in one head's row
  int page_size, width;
  int64_t n_pages;
};

// One thread moves units of sizeof(U) bytes: (token, head, unit) of sequence
// blockIdx.y, K or V by blockIdx.z. Consecutive threads take consecutive units
// of a row, so both sides are full lines. Bound by latency for one token (a
// launch), by the memory's bandwidth for a prompt's or a clip's worth.
template <typename U>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendArgs a) {
  const int seq = blockIdx.y;
  const int len = a.lens[seq];
  int count = a.counts ? a.counts[seq] : a.n_tokens;
  count = min(max(count, 0), a.n_tokens);
  const uint32_t per_token = (uint32_t)a.n_heads * a.row_units;
  const uint32_t total = (uint32_t)count * per_token;
  const char* src = a.src[blockIdx.z] + seq * a.s_seq;
  char* dst = a.dst[blockIdx.z];
  const int32_t* row = a.table + seq * a.ld_table;
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += gridDim.x * blockDim.x) {
    const int t = (int)(i / per_token);
    const int r = (int)(i - (uint32_t)t * per_token);
    const int h = r / a.row_units, u = r - h * a.row_units;
    const int pos = len - count + t;
    const int slot = pos / a.page_size;
    const int page = pos >= 0 && slot < a.width ? row[slot] : -1;
    if (page < 0 || page >= a.n_pages) {
      kv_error();
      continue;
    }
    const int in_page = pos - slot * a.page_size;
    const U x = *reinterpret_cast<const U*>(src + t * a.s_tok + h * a.s_head +
                                            u * (int64_t)sizeof(U));
    *reinterpret_cast<U*>(dst + page * a.page_stride + in_page * a.tok_stride +
                          h * a.head_stride + u * (int64_t)sizeof(U)) = x;
  }
}

// ---------------------------------------------------------------- page plans

// The planning kernels run as one cluster of kPlanCtas CTAs: their phases are
// parted by the cluster's hardware barrier, so a plan is one launch.
constexpr int kPlanCtas = 8;
constexpr int kPlanThreads = 1024;

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}

// Inclusive scan over the CTA's kPlanThreads values; *total gets their sum.
// Every thread calls it; `part` is 32 words of shared memory.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* part, int64_t* total) {
  const int lane = lane_id(), w = warp_id();
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();   // the previous call's readers are done with part
  if (lane == 31) part[w] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int i = 0; i < kPlanThreads / 32; i++) {
    const int64_t p = part[i];
    if (i < w) before += p;
    all += p;
  }
  *total = all;
  return v + before;
}

// One page copy: the first n_tok tokens of page src, every layer and head.
struct PageCopy {
  int32_t src, dst, n_tok, pad;
};

// The workspace of a plan.
struct PlanSpace {
  PageCopy* copies;     // max(n_seqs, n_pages)
  int32_t* list;        // n_pages: free pages or holes, ascending
  int32_t* remap;       // n_pages: where compaction moves a page
  int64_t* scan;        // n_seqs: pages and copies asked for before this sequence
  int32_t* need;        // n_seqs: pages asked for, bit 30: one of them is a copy
  int32_t* seg;         // 3 * kPlanCtas counts
  int32_t* n_copies;
};

static int64_t align16(int64_t n) { return (n + 15) & ~(int64_t)15; }

static int64_t plan_space(PlanSpace* p, void* base, int64_t n_seqs, int64_t n_pages) {
  char* b = static_cast<char*>(base);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* q = b + at;
    at += align16(bytes);
    return q;
  };
  PlanSpace s;
  s.n_copies = reinterpret_cast<int32_t*>(take(4));
  s.seg = reinterpret_cast<int32_t*>(take(4 * 3 * kPlanCtas));
  s.copies = reinterpret_cast<PageCopy*>(
      take((int64_t)sizeof(PageCopy) * (n_seqs > n_pages ? n_seqs : n_pages)));
  s.list = reinterpret_cast<int32_t*>(take(4 * n_pages));
  s.remap = reinterpret_cast<int32_t*>(take(4 * n_pages));
  s.scan = reinterpret_cast<int64_t*>(take(8 * n_seqs));
  s.need = reinterpret_cast<int32_t*>(take(4 * n_seqs));
  if (p) *p = s;
  return at;
}

struct ForkArgs {
  const int32_t *table, *lens, *refs, *parents, *grow;
  int32_t *table_out, *lens_out, *refs_out, *grown, *status;
  PlanSpace ws;
  int n_seqs, width, page_size, n_pages;
};

constexpr int kNeedsCopy = 1 << 30;

// Sequence i goes on as parents[i] did, with room for grow[i] more tokens:
//   1 the lengths, and the reference counts as they were
//   2 the rows of the page table; references given back and taken (integer
//     atomics: the counts do not depend on their order)
//   3 what each sequence asks for: pages for its new tokens, and one more where
//     its last page is partly filled and another sequence refers to it too. Of
//     the sequences that share such a page the longest (the first among equals)
//     keeps it: what it writes lies past the others' lengths. The rest copy it.
//     A page stands at the same place in the rows of all sequences that share
//     it, so the sharers are found by comparing one column.
//   4 the free pages in ascending order, and the running sum of the requests
//   5 the k-th page asked for is the k-th free page; sequences past the pool's
//     end are not grown
// Integer work of a few bytes a page, bound by the latency of its phases.
__global__ void __launch_bounds__(kPlanThreads, 1) kv_fork_kernel(const ForkArgs a) {
  __shared__ int64_t part[32];
  pdl_launch_dependents();
  const int cta = blockIdx.x;
  const int tid = cta * kPlanThreads + threadIdx.x;
  constexpr int kAll = kPlanCtas * kPlanThreads;
  const int lane = lane_id(), gw = tid >> 5;
  constexpr int kWarps = kAll / 32;
  const int ps = a.page_size;
  const int64_t capacity = (int64_t)a.width * ps;

  // 1
  for (int p = tid; p < a.n_pages; p += kAll) a.refs_out[p] = a.refs[p];
  for (int i = tid; i < a.n_seqs; i += kAll) {
    const int par = a.parents ? a.parents[i] : i;
    int now = 0;
    if (par >= 0 && par < a.n_seqs) {
      now = a.lens[par];
      if (now < 0 || now > capacity) {
        kv_error();
        now = now < 0 ? 0 : (int)capacity;
      }
    } else if (par >= a.n_seqs) {
      kv_error();
    }
    a.lens_out[i] = now;
  }
  if (tid == 0) *a.ws.n_copies = 0;
  cluster_sync();

  // 2
  for (int i = gw; i < a.n_seqs; i += kWarps) {
    const int par = a.parents ? a.parents[i] : i;
    const int held = (__ldcg(a.lens_out + i) + ps - 1) / ps;
    const int32_t* from = a.table + (int64_t)(par >= 0 && par < a.n_seqs ? par : i) * a.width;
    const int32_t* old = a.table + (int64_t)i * a.width;
    int32_t* to = a.table_out + (int64_t)i * a.width;
    for (int c = lane; c < a.width; c += 32) {
      const int was = old[c];
      int is = c < held ? from[c] : -1;
      if (is >= a.n_pages || (is < 0 && c < held)) {
        kv_error();
        is = -1;
      }
      to[c] = is;
      if (was != is) {
        if (was >= 0 && was < a.n_pages) atomicSub(a.refs_out + was, 1);
        if (is >= 0) atomicAdd(a.refs_out + is, 1);
      }
    }
  }
  cluster_sync();

  // 3
  for (int i = gw; i < a.n_seqs; i += kWarps) {
    const int now = __ldcg(a.lens_out + i);
    const int grow = a.grow ? max(a.grow[i], 0) : 0;
    const bool wants = grow > 0 && (int64_t)now + grow <= capacity;
    int need = 0;
    if (wants) {
      const int col = now / ps;
      need = (int)(((int64_t)now + grow + ps - 1) / ps) - (now + ps - 1) / ps;
      if (now % ps) {
        const int page = __ldcg(a.table_out + (int64_t)i * a.width + col);
        const int refs = page >= 0 ? __ldcg(a.refs_out + page) : 0;
        if (refs > 1) {
          int mates = 0;
          bool better = false;
          for (int j = lane; j < a.n_seqs; j += 32) {
            const int nj = __ldcg(a.lens_out + j);
            if (nj > col * ps && __ldcg(a.table_out + (int64_t)j * a.width + col) == page) {
              mates++;
              better |= nj > now || (nj == now && j < i);
            }
          }
          mates = __reduce_add_sync(0xffffffffu, mates);
          better = __any_sync(0xffffffffu, better);
          if (better || mates != refs) need = (need + 1) | kNeedsCopy;
        }
      }
    }
    if (lane == 0) a.ws.need[i] = need;
  }
  const int seg = (a.n_pages + kPlanCtas - 1) / kPlanCtas;
  const int p0 = min(a.n_pages, cta * seg), p1 = min(a.n_pages, p0 + seg);
  int64_t total;
  {
    int n = 0;
    for (int p = p0 + threadIdx.x; p < p1; p += kPlanThreads) n += __ldcg(a.refs_out + p) == 0;
    block_scan(n, part, &total);
    if (threadIdx.x == 0) a.ws.seg[cta] = (int)total;
  }
  cluster_sync();

  // 4
  int n_free = 0, base = 0;
  for (int c = 0; c < kPlanCtas; c++) {
    const int n = __ldcg(a.ws.seg + c);
    if (c < cta) base += n;
    n_free += n;
  }
  for (int p = p0; p < p1; p += kPlanThreads) {
    const int q = p + threadIdx.x;
    const int f = q < p1 && __ldcg(a.refs_out + q) == 0;
    const int64_t upto = block_scan(f, part, &total);
    if (f) a.ws.list[base + upto - 1] = q;
    base += (int)total;
  }
  if (cta == 0) {
    int64_t run = 0;   // pages asked for, and the copies among them in the low half
    for (int i = 0; i < a.n_seqs; i += kPlanThreads) {
      const int q = i + threadIdx.x;
      const int need = q < a.n_seqs ? __ldcg(a.ws.need + q) : 0;
      const int64_t v = ((int64_t)(need & ~kNeedsCopy) << 32) | (need & kNeedsCopy ? 1 : 0);
      const int64_t upto = block_scan(v, part, &total);
      if (q < a.n_seqs) a.ws.scan[q] = run + upto - v;
      run += total;
    }
    if (threadIdx.x == 0) {
      const int64_t asked = run >> 32;
      a.status[1] = (int)(asked > n_free ? asked - n_free : 0);
      a.status[0] = n_free;   // less what phase 5 takes
    }
  }
  cluster_sync();

  // 5
  for (int i = gw; i < a.n_seqs; i += kWarps) {
    const int now = __ldcg(a.lens_out + i);
    const int grow = a.grow ? max(a.grow[i], 0) : 0;
    const bool wants = grow > 0 && (int64_t)now + grow <= capacity;
    const int asked = __ldcg(a.ws.need + i);
    const int need = asked & ~kNeedsCopy;
    const int64_t scan = __ldcg(a.ws.scan + i);
    const int64_t before = scan >> 32;
    const bool granted = wants && (need == 0 || before + need <= n_free);
    __syncwarp();
    if (lane == 0) {
      a.lens_out[i] = granted ? now + grow : now;
      if (a.grown) a.grown[i] = granted ? grow : 0;
      if (granted && need) atomicSub(a.status, need);
    }
    if (!granted || need == 0) continue;
    int32_t* row = a.table_out + (int64_t)i * a.width;
    int64_t next = before;
    if (asked & kNeedsCopy) {
      const int col = now / ps;
      if (lane == 0) {
        const int src = __ldcg(row + col), dst = __ldcg(a.ws.list + next);
        atomicSub(a.refs_out + src, 1);
        a.refs_out[dst] = 1;
        row[col] = dst;
        a.ws.copies[(int32_t)scan] = {src, dst, now % ps, 0};
        atomicAdd(a.ws.n_copies, 1);
      }
      next++;
    }
    const int fresh = need - (asked & kNeedsCopy ? 1 : 0);
    const int held = (now + ps - 1) / ps;
    for (int c = lane; c < fresh; c += 32) {
      const int page = __ldcg(a.ws.list + next + c);
      row[held + c] = page;
      a.refs_out[page] = 1;
    }
  }
}

struct CompactArgs {
  const int32_t *table, *refs;
  int32_t *table_out, *refs_out, *status;
  PlanSpace ws;
  int64_t n_entries;
  int page_size, n_pages;
};

// The used pages past the first n_used go to the free ones among them, both in
// ascending order: the fewest moves that leave the pool dense.
__global__ void __launch_bounds__(kPlanThreads, 1) kv_compact_kernel(const CompactArgs a) {
  __shared__ int64_t part[32];
  pdl_launch_dependents();
  const int cta = blockIdx.x;
  const int64_t tid = cta * kPlanThreads + threadIdx.x;
  constexpr int kAll = kPlanCtas * kPlanThreads;
  const int seg = (a.n_pages + kPlanCtas - 1) / kPlanCtas;
  const int p0 = min(a.n_pages, cta * seg), p1 = min(a.n_pages, p0 + seg);
  int64_t total;

  // used pages of each CTA's part
  int n = 0;
  for (int p = p0 + threadIdx.x; p < p1; p += kPlanThreads) n += a.refs[p] > 0;
  block_scan(n, part, &total);
  if (threadIdx.x == 0) a.ws.seg[cta] = (int)total;
  cluster_sync();
  int n_used = 0;
  for (int c = 0; c < kPlanCtas; c++) n_used += __ldcg(a.ws.seg + c);

  // holes below n_used, movers from it on: a count of either in a page's part
  n = 0;
  for (int p = p0 + threadIdx.x; p < p1; p += kPlanThreads)
    n += (a.refs[p] > 0) == (p >= n_used);
  // a part that holds n_used has both kinds: count the holes apart
  int holes = 0;
  for (int p = p0 + threadIdx.x; p < min(p1, n_used); p += kPlanThreads) holes += a.refs[p] <= 0;
  block_scan(((int64_t)holes << 32) | (uint32_t)(n - holes), part, &total);
  if (threadIdx.x == 0) {
    a.ws.seg[kPlanCtas + cta] = (int)(total >> 32);
    a.ws.seg[2 * kPlanCtas + cta] = (int)(total & 0xffffffff);
  }
  cluster_sync();
  int hole_at = 0, mover_at = 0, n_movers = 0;
  for (int c = 0; c < kPlanCtas; c++) {
    const int h = __ldcg(a.ws.seg + kPlanCtas + c), m = __ldcg(a.ws.seg + 2 * kPlanCtas + c);
    if (c < cta) {
      hole_at += h;
      mover_at += m;
    }
    n_movers += m;
  }
  for (int p = p0; p < p1; p += kPlanThreads) {
    const int q = p + threadIdx.x;
    const int r = q < p1 ? a.refs[q] : 0;
    const bool hole = q < p1 && q < n_used && r <= 0;
    const bool mover = q < p1 && q >= n_used && r > 0;
    const int64_t upto = block_scan(((int64_t)hole << 32) | (uint32_t)mover, part, &total);
    if (hole) a.ws.list[hole_at + (int)(upto >> 32) - 1] = q;
    if (mover) a.ws.copies[mover_at + (int)(upto & 0xffffffff) - 1].src = q;
    if (q < p1) a.refs_out[q] = q < n_used ? max(r, 0) : 0;
    hole_at += (int)(total >> 32);
    mover_at += (int)(total & 0xffffffff);
  }
  if (tid == 0) {
    a.status[0] = n_used;
    a.status[1] = n_movers;
    *a.ws.n_copies = n_movers;
  }
  cluster_sync();
  for (int64_t m = tid; m < n_movers; m += kAll) {
    const int src = __ldcg(&a.ws.copies[m].src), dst = __ldcg(a.ws.list + m);
    a.ws.copies[m] = {src, dst, a.page_size, 0};
    a.ws.remap[src] = dst;
    a.refs_out[dst] = a.refs[src];
  }
  cluster_sync();
  for (int64_t i = tid; i < a.n_entries; i += kAll) {
    int page = a.table[i];
    if (page >= a.n_pages) {
      kv_error();
      page = -1;
    } else if (page >= n_used) {
      // a page that the table names and the counts call free has no place to go
      if (a.refs[page] > 0) {
        page = __ldcg(a.ws.remap + page);
      } else {
        kv_error();
        page = -1;
      }
    }
    a.table_out[i] = page;
  }
}

// ---------------------------------------------------------------- page copies

struct CopyArgs {
  char *k, *v;
  const PageCopy* copies;
  const int32_t* n_copies;
  int64_t layer_stride, page_stride, tok_stride, head_stride;   // bytes
  int n_layers, n_heads, row_chunks;   // 16-byte chunks of one head's row
  bool head_major;                     // a page is stored head by head
};

constexpr int kCopyThreads = 256, kCopyUnroll = 4;

// One CTA a (copy, layer, K or V) at a time: the tokens of a page, 16 bytes a
// thread, kCopyUnroll loads in flight before their stores. Source and target
// pages are never the same page, nor is a target another copy's source: plans
// copy pages in use to free ones. Bound by the memory's bandwidth, read + write.
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(const CopyArgs a) {
  pdl_wait();   // the plan
  const int64_t units = (int64_t)*a.n_copies * a.n_layers * 2;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int which = (int)(u & 1);
    const int64_t v = u >> 1;
    const int layer = (int)(v % a.n_layers);
    const PageCopy c = a.copies[v / a.n_layers];
    char* pool = (which ? a.v : a.k) + layer * a.layer_stride;
    const char* src = pool + c.src * a.page_stride;
    char* dst = pool + c.dst * a.page_stride;
    const int n = c.n_tok * a.n_heads * a.row_chunks;
    for (int i0 = 0; i0 < n; i0 += kCopyThreads * kCopyUnroll) {
      uint4 x[kCopyUnroll];
      int64_t at[kCopyUnroll];
#pragma unroll
      for (int j = 0; j < kCopyUnroll; j++) {
        const int i = i0 + j * kCopyThreads + threadIdx.x;
        const int r = i / a.row_chunks, k = i - r * a.row_chunks;
        const int inner = a.head_major ? c.n_tok : a.n_heads;
        const int hi = r / inner, lo = r - hi * inner;
        const int t = a.head_major ? lo : hi, h = a.head_major ? hi : lo;
        at[j] = t * a.tok_stride + h * a.head_stride + k * 16;
        if (i < n) x[j] = *reinterpret_cast<const uint4*>(src + at[j]);
      }
#pragma unroll
      for (int j = 0; j < kCopyUnroll; j++)
        if (i0 + j * kCopyThreads + (int)threadIdx.x < n)
          *reinterpret_cast<uint4*>(dst + at[j]) = x[j];
    }
  }
}

// ---------------------------------------------------------------- host

int check_pool(const char* what, const void* k, const void* v, int64_t page_stride,
               int64_t tok_stride, int64_t head_stride, int64_t n_heads, int64_t head_dim,
               int64_t n_pages, int64_t page_size, int dtype) {
  if (dtype != WX_DTYPE_BF16 && dtype != WX_DTYPE_F32)
    return fail(WX_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (n_heads < 1 || n_heads > 65535 || head_dim < 1 || n_pages < 1 || page_size < 1 ||
      n_pages > 0x7fffffff || page_size > 65536)
    return fail(WX_ERR_INVALID,
                "%s: bad cache: %lld pages of %lld tokens, %lld heads of %lld", what,
                (long long)n_pages, (long long)page_size, (long long)n_heads,
                (long long)head_dim);
  const int64_t es = dtype == WX_DTYPE_BF16 ? 2 : 4;
  if (head_dim * es % 16 || page_stride * es % 16 || tok_stride * es % 16 ||
      head_stride * es % 16 || ((uintptr_t)k & 15) || ((uintptr_t)v & 15))
    return fail(WX_ERR_INVALID,
                "%s: the cache's rows must be 16-byte aligned (head_dim %lld, strides %lld, "
                "%lld, %lld)",
                what, (long long)head_dim, (long long)page_stride, (long long)tok_stride,
                (long long)head_stride);
  if (page_stride < 0 || tok_stride < 0 || head_stride < 0)
    return fail(WX_ERR_INVALID, "%s: negative stride", what);
  if (!k || !v) return fail(WX_ERR_INVALID, "%s: NULL cache", what);
  return WX_OK;
}

template <typename Args>
static cudaError_t launch_cluster(void (*kernel)(Args), const Args& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kPlanCtas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kPlanCtas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

struct Pool {
  void *k, *v;
  int64_t n_layers, layer_stride, page_stride, tok_stride, head_stride, n_heads, head_dim;
  int dtype;
};

// The copies of a plan of at most max_copies, as a programmatic dependent of the
// planning kernel: its CTAs are in place when the plan is done.
static int launch_copies(const char* what, const Pool& p, const PlanSpace& ws,
                         int64_t max_copies, cudaStream_t st) {
  const int64_t es = p.dtype == WX_DTYPE_BF16 ? 2 : 4;
  CopyArgs a = {};
  a.k = static_cast<char*>(p.k);
  a.v = static_cast<char*>(p.v);
  a.copies = ws.copies;
  a.n_copies = ws.n_copies;
  a.layer_stride = p.layer_stride * es;
  a.page_stride = p.page_stride * es;
  a.tok_stride = p.tok_stride * es;
  a.head_stride = p.head_stride * es;
  a.n_layers = (int)p.n_layers;
  a.n_heads = (int)p.n_heads;
  a.row_chunks = (int)(p.head_dim * es / 16);
  a.head_major = p.tok_stride < p.head_stride;
  const int64_t units = max_copies * p.n_layers * 2, most = (int64_t)sm_count() * 8;
  PdlScope pdl(true);
  WX_CUDA_TRY(launch_k(kv_copy_kernel, dim3((unsigned)(units < most ? units : most)),
                       dim3(kCopyThreads), 0, st, a));
  return check_launch(what);
}

static int check_plan(const char* what, int64_t n_layers, int64_t layer_stride, int64_t es,
                      int64_t n_seqs, int64_t width, const void* ws, int64_t ws_bytes,
                      int64_t n_pages) {
  if (n_layers < 1 || n_layers > 65536 || layer_stride < 0 || layer_stride * es % 16)
    return fail(WX_ERR_INVALID, "%s: bad layers: %lld, stride %lld", what, (long long)n_layers,
                (long long)layer_stride);
  if (n_seqs < 1 || n_seqs > (1 << 20) || width < 1 || width > 0x7fffffff)
    return fail(WX_ERR_INVALID, "%s: bad page table: %lld x %lld", what, (long long)n_seqs,
                (long long)width);
  const int64_t want = plan_space(nullptr, nullptr, n_seqs, n_pages);
  if (!ws || ((uintptr_t)ws & 15) || ws_bytes < want)
    return fail(WX_ERR_INVALID, "%s: workspace of %lld bytes (16-byte aligned) needed, got %lld",
                what, (long long)want, (long long)ws_bytes);
  return WX_OK;
}

}  // namespace wx

extern "C" {

int wx_kv_append(const void* k, const void* v, int64_t src_seq_stride, int64_t src_tok_stride,
                 int64_t src_head_stride, void* k_cache, void* v_cache, int64_t page_stride,
                 int64_t tok_stride, int64_t head_stride, const int32_t* table, int64_t ld_table,
                 const int32_t* lens, const int32_t* counts, int64_t n_seqs, int64_t n_tokens,
                 int64_t n_heads, int64_t head_dim, int64_t n_pages, int64_t page_size,
                 int dtype, void* stream) {
  using namespace wx;
  WX_TRY(check_pool("kv_append", k_cache, v_cache, page_stride, tok_stride, head_stride, n_heads,
                    head_dim, n_pages, page_size, dtype));
  if (n_seqs < 0 || n_seqs > 65535 || n_tokens < 0 || n_tokens > 0x7fffffff)
    return fail(WX_ERR_INVALID, "kv_append: bad shape: %lld sequences, %lld tokens",
                (long long)n_seqs, (long long)n_tokens);
  if (head_dim > 65536 || n_tokens * n_heads * head_dim > 0x7fffffff)
    return fail(WX_ERR_INVALID, "kv_append: %lld tokens of %lld heads of %lld: over 2^31 - 1",
                (long long)n_tokens, (long long)n_heads, (long long)head_dim);
  if (n_seqs == 0 || n_tokens == 0) return WX_OK;
  if (!k || !v || !table || !lens || ld_table < 1)
    return fail(WX_ERR_INVALID, "kv_append: NULL argument or empty page table");
  const int64_t es = dtype == WX_DTYPE_BF16 ? 2 : 4;
  AppendArgs a = {};
  a.src[0] = static_cast<const char*>(k);
  a.src[1] = static_cast<const char*>(v);
  a.dst[0] = static_cast<char*>(k_cache);
  a.dst[1] = static_cast<char*>(v_cache);
  a.s_seq = src_seq_stride * es;
  a.s_tok = src_tok_stride * es;
  a.s_head = src_head_stride * es;
  a.page_stride = page_stride * es;
  a.tok_stride = tok_stride * es;
  a.head_stride = head_stride * es;
  a.table = table;
  a.ld_table = ld_table;
  a.lens = lens;
  a.counts = counts;
  a.n_tokens = (int)n_tokens;
  a.n_heads = (int)n_heads;
  a.page_size = (int)page_size;
  a.width = (int)(ld_table < 0x7fffffff ? ld_table : 0x7fffffff);
  a.n_pages = n_pages;
  // 16 bytes a thread where the source rows allow it, else one element
  const bool vec = !((a.s_seq | a.s_tok | a.s_head | (int64_t)(uintptr_t)k |
                      (int64_t)(uintptr_t)v) & 15);
  const int64_t unit = vec ? 16 : es;
  a.row_units = (int)(head_dim * es / unit);
  const int64_t units = n_tokens * n_heads * a.row_units;
  const int64_t blocks = (units + 255) / 256;
  const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536), (unsigned)n_seqs, 2);
  cudaStream_t st = as_stream(stream);
  if (vec)
    WX_CUDA_TRY(launch_k(kv_append_kernel<uint4>, grid, dim3(256), 0, st, a));
  else if (es == 2)
    WX_CUDA_TRY(launch_k(kv_append_kernel<uint16_t>, grid, dim3(256), 0, st, a));
  else
    WX_CUDA_TRY(launch_k(kv_append_kernel<uint32_t>, grid, dim3(256), 0, st, a));
  return check_launch("kv_append");
}

int64_t wx_kv_workspace(int64_t n_seqs, int64_t n_pages) {
  if (n_seqs < 0 || n_pages < 0) return 0;
  return wx::plan_space(nullptr, nullptr, n_seqs, n_pages);
}

int wx_kv_fork(void* k_cache, void* v_cache, int64_t n_layers, int64_t layer_stride,
               int64_t page_stride, int64_t tok_stride, int64_t head_stride, int64_t n_heads,
               int64_t head_dim, int64_t n_pages, int64_t page_size, int dtype,
               const int32_t* table, const int32_t* lens, const int32_t* refs,
               const int32_t* parents, const int32_t* grow, int64_t n_seqs, int64_t width,
               int32_t* table_out, int32_t* lens_out, int32_t* refs_out, int32_t* grown_out,
               int32_t* status_out, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace wx;
  WX_TRY(check_pool("kv_fork", k_cache, v_cache, page_stride, tok_stride, head_stride, n_heads,
                    head_dim, n_pages, page_size, dtype));
  WX_TRY(check_plan("kv_fork", n_layers, layer_stride, dtype == WX_DTYPE_BF16 ? 2 : 4, n_seqs,
                    width, workspace, workspace_bytes, n_pages));
  if (!table || !lens || !refs || !table_out || !lens_out || !refs_out || !status_out)
    return fail(WX_ERR_INVALID, "kv_fork: NULL argument");
  if (table == table_out || lens == lens_out || refs == refs_out)
    return fail(WX_ERR_INVALID, "kv_fork: the new page table cannot be written over the old one");
  if (n_heads * head_dim * page_size > 0x7fffffff || width * page_size > 0x7fffffff)
    return fail(WX_ERR_INVALID, "kv_fork: a page or a sequence of over 2^31 - 1 elements or tokens");
  ForkArgs a = {};
  a.table = table;
  a.lens = lens;
  a.refs = refs;
  a.parents = parents;
  a.grow = grow;
  a.table_out = table_out;
  a.lens_out = lens_out;
  a.refs_out = refs_out;
  a.grown = grown_out;
  a.status = status_out;
  plan_space(&a.ws, workspace, n_seqs, n_pages);
  a.n_seqs = (int)n_seqs;
  a.width = (int)width;
  a.page_size = (int)page_size;
  a.n_pages = (int)n_pages;
  cudaStream_t st = as_stream(stream);
  WX_CUDA_TRY(launch_cluster(kv_fork_kernel, a, st));
  WX_TRY(check_launch("kv_fork"));
  if (!grow) return WX_OK;   // nothing is written, so nothing is copied
  const Pool p = {k_cache, v_cache, n_layers, layer_stride, page_stride, tok_stride,
                  head_stride, n_heads, head_dim, dtype};
  return launch_copies("kv_fork copies", p, a.ws, n_seqs, st);
}

int wx_kv_compact(void* k_cache, void* v_cache, int64_t n_layers, int64_t layer_stride,
                  int64_t page_stride, int64_t tok_stride, int64_t head_stride, int64_t n_heads,
                  int64_t head_dim, int64_t n_pages, int64_t page_size, int dtype,
                  const int32_t* table, const int32_t* refs, int64_t n_seqs, int64_t width,
                  int32_t* table_out, int32_t* refs_out, int32_t* status_out, void* workspace,
                  int64_t workspace_bytes, void* stream) {
  using namespace wx;
  WX_TRY(check_pool("kv_compact", k_cache, v_cache, page_stride, tok_stride, head_stride, n_heads,
                    head_dim, n_pages, page_size, dtype));
  WX_TRY(check_plan("kv_compact", n_layers, layer_stride, dtype == WX_DTYPE_BF16 ? 2 : 4, n_seqs,
                    width, workspace, workspace_bytes, n_pages));
  if (!table || !refs || !table_out || !refs_out || !status_out)
    return fail(WX_ERR_INVALID, "kv_compact: NULL argument");
  if (refs == refs_out)
    return fail(WX_ERR_INVALID, "kv_compact: the new counts cannot be written over the old ones");
  if (n_heads * head_dim * page_size > 0x7fffffff)
    return fail(WX_ERR_INVALID, "kv_compact: a page of over 2^31 - 1 elements");
  CompactArgs a = {};
  a.table = table;
  a.refs = refs;
  a.table_out = table_out;
  a.refs_out = refs_out;
  a.status = status_out;
  plan_space(&a.ws, workspace, n_seqs, n_pages);
  a.n_entries = n_seqs * width;
  a.page_size = (int)page_size;
  a.n_pages = (int)n_pages;
  cudaStream_t st = as_stream(stream);
  WX_CUDA_TRY(launch_cluster(kv_compact_kernel, a, st));
  WX_TRY(check_launch("kv_compact"));
  const Pool p = {k_cache, v_cache, n_layers, layer_stride, page_stride, tok_stride,
                  head_stride, n_heads, head_dim, dtype};
  return launch_copies("kv_compact copies", p, a.ws, n_pages / 2 + 1, st);
}

}  // extern "C"
