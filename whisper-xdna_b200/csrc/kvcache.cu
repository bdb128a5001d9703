// The paged key-value cache of a text decoder on the encoder's features:
// writing tokens into it (append), continuing, ending and growing sequences
// with copy on write (fork), and moving its pages together (compact). No call
// waits for the host: the page plan is made on the device, and the copy kernel
// that follows reads it there.
//
// A cache is two pools (K and V) of n_pages pages of page_size tokens for each
// layer; a row of the page table names a sequence's pages in order, -1 past the
// last. refs[p] counts the table entries that name page p; 0 is free.
#include <algorithm>
#include <atomic>
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
  Div by_token, by_row, by_page;      // units of a token, units of a row, page_size
  int width;
  int64_t n_pages;
};

constexpr int kAppendUnroll = 4;

// A thread moves units of sizeof(U) bytes, kAppendUnroll of them in flight: (token,
// head, unit) of sequence blockIdx.y, K or V by blockIdx.z. Consecutive threads take
// consecutive units of a row, so both sides are full lines. Measured (B200): 64 clips
// of 1500 frames, 20 heads of 64 in bf16 (983 MB read and written) 146 us, 6.7 TB/s,
// the memory's bandwidth; one unit in flight a thread and hardware divisions 198 us.
// One token of 320 sequences 2.0 us, a launch.
template <typename U>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendArgs a) {
  pdl_begin();
  const int seq = blockIdx.y;
  // a count past the rows given still says where row 0 goes; none is below 0
  const int asked = a.counts ? a.counts[seq] : a.n_tokens;
  const int count = min(max(asked, 0), a.n_tokens);
  // row 0's position; cut off where all positions are below 0 anyhow
  const int first = (int)max((int64_t)a.lens[seq] - asked, (int64_t)INT32_MIN);
  const uint32_t per_token = (uint32_t)a.n_heads * a.row_units;
  const uint32_t total = (uint32_t)count * per_token;
  const char* src = a.src[blockIdx.z] + seq * a.s_seq;
  char* dst = a.dst[blockIdx.z];
  const int32_t* row = a.table + seq * a.ld_table;
  for (uint32_t i0 = blockIdx.x * blockDim.x * kAppendUnroll + threadIdx.x; i0 < total;
       i0 += gridDim.x * blockDim.x * kAppendUnroll) {
    U x[kAppendUnroll];
    int64_t to[kAppendUnroll];
#pragma unroll
    for (int j = 0; j < kAppendUnroll; j++) {
      const uint32_t i = i0 + j * blockDim.x;
      to[j] = -1;
      if (i >= total) continue;
      const int t = a.by_token((int)i), r = (int)(i - (uint32_t)t * per_token);
      const int h = a.by_row(r), u = r - h * a.row_units;
      x[j] = *reinterpret_cast<const U*>(src + t * a.s_tok + h * a.s_head +
                                         u * (int64_t)sizeof(U));
      const int pos = first + t;
      const int slot = a.by_page(max(pos, 0));
      const int page = pos >= 0 && slot < a.width ? row[slot] : -1;
      if (page < 0 || page >= a.n_pages)
        kv_error();
      else
        to[j] = page * a.page_stride + (pos - slot * (int)a.by_page.d) * a.tok_stride +
                h * a.head_stride + u * (int64_t)sizeof(U);
    }
#pragma unroll
    for (int j = 0; j < kAppendUnroll; j++)
      if (to[j] >= 0) *reinterpret_cast<U*>(dst + to[j]) = x[j];
  }
  if (asked != count && (threadIdx.x | blockIdx.x | blockIdx.z) == 0) kv_error();
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
// Every thread calls it; `part` is 33 words of shared memory.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* part, int64_t* total) {
  const int lane = lane_id(), w = warp_id();
  auto warp_scan = [&](int64_t x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += u;
    }
    return x;
  };
  v = warp_scan(v);
  __syncthreads();   // the previous call's readers are done with part
  if (lane == 31) part[w + 1] = v;
  __syncthreads();
  if (w == 0) {
    const int64_t x = warp_scan(part[lane + 1]);
    part[lane + 1] = x;
    if (lane == 0) part[0] = 0;
  }
  __syncthreads();
  *total = part[32];
  return v + part[w];
}
static_assert(kPlanThreads == 1024, "block_scan: a warp scans the warps' sums");

// The one-CTA plans' scans: two 32-bit values side by side, exclusive, in place; their
// sums in a0 and b0. `part` is 66 words.
__device__ __forceinline__ void block_scan2(uint32_t& a, uint32_t& b, uint32_t* part, uint32_t* a0,
                                            uint32_t* b0) {
  const int lane = lane_id(), w = warp_id();
  const uint32_t a_in = a, b_in = b;
  auto warp_scan = [&](uint32_t& x, uint32_t& y) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += u;
        y += v;
      }
    }
  };
  warp_scan(a, b);
  if (lane == 31) {
    part[w + 1] = a;
    part[33 + w + 1] = b;
  }
  __syncthreads();
  if (w == 0) {
    uint32_t x = part[lane + 1], y = part[33 + lane + 1];
    warp_scan(x, y);
    part[lane + 1] = x;
    part[33 + lane + 1] = y;
    if (lane == 0) part[0] = part[33] = 0;
  }
  __syncthreads();
  *a0 = part[32];
  *b0 = part[33 + 32];
  a += part[w] - a_in;
  b += part[33 + w] - b_in;
}
// The sum of every thread's value; `part` is 32 words, not in use before.
__device__ __forceinline__ uint32_t block_sum(uint32_t v, uint32_t* part) {
  v = __reduce_add_sync(0xffffffffu, v);
  if (lane_id() == 0) part[warp_id()] = v;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, part[lane_id()]);
}

// One page copy: the first n_tok tokens of page src, every layer and head.
struct PageCopy {
  int32_t src, dst, n_tok, pad;
};

// The workspace of a plan.
struct PlanSpace {
  PageCopy* copies;     // max(n_seqs, n_pages)
  int32_t* list;        // n_pages: free pages or holes, ascending
  int32_t* remap;       // n_pages: where a page is after a compaction, -1: nobody's
  unsigned long long* keeper;   // n_pages: the longest sharer of a page to be written
  int32_t* sharers;     // n_pages: how many share it, 0 before
  int32_t* column;      // n_pages: its column + 1, 0: not to be written
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
  s.keeper = reinterpret_cast<unsigned long long*>(take(8 * n_pages));
  s.sharers = reinterpret_cast<int32_t*>(take(4 * n_pages));
  s.column = reinterpret_cast<int32_t*>(take(4 * n_pages));
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
  Div by_page, by_width;   // page_size, width
};

constexpr int kNeedsCopy = 1 << 30;

// The steps of a fork for one sequence or table entry, shared by its two forms.

// sequence i's parent, -1: none
__device__ __forceinline__ int fork_parent(const ForkArgs& a, int i) {
  const int par = a.parents ? a.parents[i] : i;
  if (par >= a.n_seqs) {
    kv_error();
    return -1;
  }
  return par < 0 ? -1 : par;
}
// the length it goes on from
__device__ __forceinline__ int fork_length(const ForkArgs& a, int par) {
  const int n = par < 0 ? 0 : a.lens[par];
  const int64_t most = (int64_t)a.width * a.page_size;
  if (n < 0 || n > most) {
    kv_error();
    return n < 0 ? 0 : (int)most;
  }
  return n;
}
// a row's entry in column c, `from` standing in the parent's row
__device__ __forceinline__ int fork_entry(const ForkArgs& a, int from, int c, int now) {
  if (c * a.page_size >= now) return -1;
  if (from < 0 || from >= a.n_pages) {
    kv_error();
    return -1;
  }
  return from;
}
__device__ __forceinline__ void fork_refs(const ForkArgs& a, int32_t* refs, int was, int is) {
  if (was == is) return;
  if (was >= 0 && was < a.n_pages) atomicSub(refs + was, 1);
  if (is >= 0) atomicAdd(refs + is, 1);
}
// the tokens that a sequence of `now` is to grow by, as far as its row has room for g
__device__ __forceinline__ int fork_grow(const ForkArgs& a, int g, int now) {
  return g > 0 && (int64_t)now + g <= (int64_t)a.width * a.page_size ? g : 0;
}
__device__ __forceinline__ unsigned long long keeper_rank(int now, int i) {
  return ((unsigned long long)(uint32_t)now << 32) | (uint32_t)~i;
}

// Sequence i goes on as parents[i] did, with room for grow[i] more tokens:
//   1 the lengths, and the reference counts as they were
//   2 the rows of the page table; references given back and taken (integer
//     atomics: the counts do not depend on their order)
//   3 the partly filled last pages that are to be written and are shared
//   4 their sharers: the longest (the first among equals) keeps the page, since
//     what it writes lies past the others' lengths. A page stands at the same place
//     in the rows of all sequences that share it.
//   5 what each sequence asks for: pages for its new tokens, and one more where it
//     has to copy a shared page
//   6 the free pages in ascending order, and the running sum of the requests
//   7 the k-th page asked for is the k-th free page; sequences past the pool's
//     end are not grown
// Integer work of a few bytes a page, bound by the latency of its phases. This form
// keeps its arrays in global memory, parted by a cluster's barrier: for tables that
// do not fit one CTA's shared memory. Measured (B200): 58 K table entries 31 us.
__global__ void __launch_bounds__(kPlanThreads, 1) kv_fork_kernel(const ForkArgs a) {
  __shared__ int64_t part[33];
  pdl_begin();
  const int cta = blockIdx.x;
  const int tid = cta * kPlanThreads + threadIdx.x;
  constexpr int kAll = kPlanCtas * kPlanThreads;
  const int lane = lane_id(), gw = tid >> 5;
  constexpr int kWarps = kAll / 32;
  const int ps = a.page_size;

  // 1
  for (int p = tid; p < a.n_pages; p += kAll) {
    a.refs_out[p] = a.refs[p];
    a.ws.keeper[p] = 0;
    a.ws.sharers[p] = a.ws.column[p] = 0;
  }
  for (int i = tid; i < a.n_seqs; i += kAll) a.lens_out[i] = fork_length(a, fork_parent(a, i));
  if (tid == 0) *a.ws.n_copies = 0;
  cluster_sync();

  // 2
  for (int i = gw; i < a.n_seqs; i += kWarps) {
    const int par = a.parents ? a.parents[i] : i, now = __ldcg(a.lens_out + i);
    const int32_t* from = a.table + (int64_t)(par >= 0 && par < a.n_seqs ? par : i) * a.width;
    const int32_t* old = a.table + (int64_t)i * a.width;
    int32_t* to = a.table_out + (int64_t)i * a.width;
    for (int c = lane; c < a.width; c += 32) {
      const int is = fork_entry(a, from[c], c, now);
      to[c] = is;
      fork_refs(a, a.refs_out, old[c], is);
    }
  }
  cluster_sync();

  // 3
  for (int i = tid; i < a.n_seqs; i += kAll) {
    const int now = __ldcg(a.lens_out + i);
    const int col = a.by_page(now);
    if (now == col * ps || !fork_grow(a, a.grow ? a.grow[i] : 0, now)) continue;
    const int page = __ldcg(a.table_out + (int64_t)i * a.width + col);
    if (page >= 0 && __ldcg(a.refs_out + page) > 1) atomicMax(a.ws.column + page, col + 1);
  }
  cluster_sync();

  // 4
  for (int i = gw; i < a.n_seqs; i += kWarps) {
    const int now = __ldcg(a.lens_out + i);
    for (int c = lane; c * ps < now; c += 32) {
      const int page = __ldcg(a.table_out + (int64_t)i * a.width + c);
      if (page < 0 || __ldcg(a.ws.column + page) != c + 1) continue;
      atomicMax(a.ws.keeper + page, keeper_rank(now, i));
      atomicAdd(a.ws.sharers + page, 1);
    }
  }
  cluster_sync();

  // 5
  for (int i = tid; i < a.n_seqs; i += kAll) {
    const int now = __ldcg(a.lens_out + i), grow = fork_grow(a, a.grow ? a.grow[i] : 0, now);
    int need = 0;
    if (grow) {
      const int col = a.by_page(now);
      need = a.by_page(now + grow - 1) - a.by_page(now + ps - 1) + 1;
      const int page = now != col * ps ? __ldcg(a.table_out + (int64_t)i * a.width + col) : -1;
      const int refs = page >= 0 ? __ldcg(a.refs_out + page) : 0;
      if (refs > 1 && (__ldcg(a.ws.keeper + page) != keeper_rank(now, i) ||
                       __ldcg(a.ws.sharers + page) != refs ||
                       __ldcg(a.ws.column + page) != col + 1))
        need = (need + 1) | kNeedsCopy;
    }
    a.ws.need[i] = need;
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

  // 6
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
      a.status[0] = n_free;   // less what phase 7 takes
    }
  }
  cluster_sync();

  // 7
  for (int i = gw; i < a.n_seqs; i += kWarps) {
    const int now = __ldcg(a.lens_out + i), grow = fork_grow(a, a.grow ? a.grow[i] : 0, now);
    const int asked = __ldcg(a.ws.need + i), need = asked & ~kNeedsCopy;
    const int64_t scan = __ldcg(a.ws.scan + i), before = scan >> 32;
    const bool granted = grow && (need == 0 || before + need <= n_free);
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
      const int col = a.by_page(now);
      if (lane == 0) {
        const int src = __ldcg(row + col), dst = __ldcg(a.ws.list + next);
        atomicSub(a.refs_out + src, 1);
        a.refs_out[dst] = 1;
        row[col] = dst;
        a.ws.copies[(int32_t)scan] = {src, dst, now - col * ps, 0};
        atomicAdd(a.ws.n_copies, 1);
      }
      next++;
    }
    const int fresh = need - (asked & kNeedsCopy ? 1 : 0);
    const int held = a.by_page(now + ps - 1);
    for (int c = lane; c < fresh; c += 32) {
      const int page = __ldcg(a.ws.list + next + c);
      row[held + c] = page;
      a.refs_out[page] = 1;
    }
  }
}

// Words of shared memory that the one-CTA form of a fork takes.
__host__ __device__ constexpr int64_t fork_words(int64_t n_seqs, int64_t width, int64_t n_pages) {
  return 2 * n_seqs * width + 6 * n_pages + 5 * n_seqs + 2;
}

// The same plan by one CTA, its arrays in shared memory: a phase costs a barrier and
// not a trip through L2. Bound by one SM's instruction issue as the table grows.
// Measured (B200), with the copies' launch, here against the cluster's form: 5 beams
// 6.7 and 16 us, 320 beams (4800 entries, 77 MB copied) 25 and 35, 256 sequences of
// 57 pages (14.6 K entries) 16.6 and 18.4: kCtaEntries is about where they meet.
__global__ void __launch_bounds__(kPlanThreads, 1) kv_fork_cta_kernel(const ForkArgs a) {
  extern __shared__ __align__(16) int32_t words[];
  __shared__ uint32_t part[66];
  __shared__ int n_copies, taken;
  pdl_begin();
  const int tid = threadIdx.x;
  const int n_entries = a.n_seqs * a.width, ps = a.page_size;
  unsigned long long* keeper = reinterpret_cast<unsigned long long*>(words);   // n_pages
  int32_t* refs = words + 2 * a.n_pages;
  int32_t *sharers = refs + a.n_pages, *column = sharers + a.n_pages, *list = column + a.n_pages;
  int32_t *is = list + a.n_pages, *was = is + n_entries;      // rows after and before
  int32_t *len = was + n_entries, *need = len + a.n_seqs;
  int32_t *pages_before = need + a.n_seqs, *copies_before = pages_before + a.n_seqs;
  int32_t* grow_by = copies_before + a.n_seqs;

  // 1: counts, lengths and parents' rows as they stand. The loads that do not hang on
  // one another go first, so that two trips to memory are waited for and not six.
  constexpr int kAhead = 4;
  int par0 = tid, grow0 = 0, refs0 = 0, from[kAhead], now[kAhead], then[kAhead];
  if (tid < a.n_seqs) {
    if (a.parents) par0 = a.parents[tid];
    if (a.grow) grow0 = a.grow[tid];
  }
  if (tid < a.n_pages) refs0 = a.refs[tid];
  auto parent_of = [&](int e) {
    return e < n_entries && a.parents ? a.parents[a.by_width(e)] : a.by_width(e);
  };
#pragma unroll
  for (int j = 0; j < kAhead; j++) from[j] = parent_of(tid + j * kPlanThreads);
  for (int e0 = tid; e0 < n_entries; e0 += kPlanThreads * kAhead) {
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int e = e0 + j * kPlanThreads, i = a.by_width(e);
      if (e >= n_entries) continue;
      now[j] = a.table[from[j] < 0 || from[j] >= a.n_seqs ? e : e + (from[j] - i) * a.width];
      then[j] = a.table[e];
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++) from[j] = parent_of(e0 + (j + kAhead) * kPlanThreads);
    if (e0 == tid && tid < a.n_seqs) {
      if (par0 >= a.n_seqs) kv_error();
      len[tid] = fork_length(a, par0 >= a.n_seqs || par0 < 0 ? -1 : par0);
      grow_by[tid] = grow0;
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int e = e0 + j * kPlanThreads;
      if (e >= n_entries) continue;
      is[e] = now[j];
      was[e] = then[j];
    }
  }
  for (int i = tid + kPlanThreads; i < a.n_seqs; i += kPlanThreads) {
    len[i] = fork_length(a, fork_parent(a, i));
    grow_by[i] = a.grow ? a.grow[i] : 0;
  }
  for (int p = tid; p < a.n_pages; p += kPlanThreads) {
    refs[p] = p == tid ? refs0 : a.refs[p];
    keeper[p] = 0;
    sharers[p] = column[p] = 0;
  }
  if (tid == 0) n_copies = taken = 0;
  __syncthreads();

  // 2
#pragma unroll 4
  for (int e = tid; e < n_entries; e += kPlanThreads) {
    const int i = a.by_width(e), page = fork_entry(a, is[e], e - i * a.width, len[i]);
    is[e] = page;
    fork_refs(a, refs, was[e], page);
  }
  __syncthreads();

  // 3
  for (int i = tid; i < a.n_seqs; i += kPlanThreads) {
    const int now = len[i], col = a.by_page(now);
    if (now == col * ps || !fork_grow(a, grow_by[i], now)) continue;
    const int page = is[i * a.width + col];
    if (page >= 0 && refs[page] > 1) atomicMax(column + page, col + 1);
  }
  __syncthreads();

  // 4
#pragma unroll 4
  for (int e = tid; e < n_entries; e += kPlanThreads) {
    const int page = is[e];
    if (page < 0 || column[page] == 0) continue;
    const int i = a.by_width(e);
    if (column[page] != e - i * a.width + 1) continue;
    atomicMax(keeper + page, keeper_rank(len[i], i));
    atomicAdd(sharers + page, 1);
  }
  __syncthreads();

  // 5 and 6: each thread a run of sequences and of pages
  const int per = (a.n_seqs + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(a.n_seqs, tid * per), i1 = min(a.n_seqs, i0 + per);
  // pages asked for, and the copies among them in the low 15 bits: with at most 2^14
  // entries neither passes its field
  uint32_t asked = 0;
  for (int i = i0; i < i1; i++) {
    const int now = len[i], grow = fork_grow(a, grow_by[i], now);
    int n = 0;
    if (grow) {
      const int col = a.by_page(now);
      n = a.by_page(now + grow - 1) - a.by_page(now + ps - 1) + 1;
      const int page = now != col * ps ? is[i * a.width + col] : -1;
      if (page >= 0 && refs[page] > 1 &&
          (keeper[page] != keeper_rank(now, i) || sharers[page] != refs[page] ||
           column[page] != col + 1))
        n = (n + 1) | kNeedsCopy;
    }
    need[i] = n;
    asked += ((uint32_t)(n & ~kNeedsCopy) << 15) | (n & kNeedsCopy ? 1 : 0);
  }
  const int per_p = (a.n_pages + kPlanThreads - 1) / kPlanThreads;
  const int p0 = min(a.n_pages, tid * per_p), p1 = min(a.n_pages, p0 + per_p);
  uint32_t free = 0, total, n_free;
  for (int p = p0; p < p1; p++) free += refs[p] == 0;
  block_scan2(asked, free, part, &total, &n_free);
  for (int i = i0; i < i1; i++) {
    pages_before[i] = (int)(asked >> 15);
    copies_before[i] = (int)(asked & 0x7fff);
    asked += ((uint32_t)(need[i] & ~kNeedsCopy) << 15) | (need[i] & kNeedsCopy ? 1 : 0);
  }
  for (int p = p0; p < p1; p++)
    if (refs[p] == 0) list[free++] = p;
  __syncthreads();

  // 7
  for (int i = tid; i < a.n_seqs; i += kPlanThreads) {
    const int now = len[i], grow = fork_grow(a, grow_by[i], now);
    const int n = need[i] & ~kNeedsCopy, copy = need[i] & kNeedsCopy ? 1 : 0;
    const int before = pages_before[i];
    const bool granted = grow && (n == 0 || before + n <= (int)n_free);
    a.lens_out[i] = granted ? now + grow : now;
    if (a.grown) a.grown[i] = granted ? grow : 0;
    if (!granted || n == 0) continue;
    atomicAdd(&taken, n);
    int32_t* row = is + i * a.width;
    if (copy) {
      const int col = a.by_page(now), src = row[col], dst = list[before];
      atomicSub(refs + src, 1);
      refs[dst] = 1;
      row[col] = dst;
      a.ws.copies[copies_before[i]] = {src, dst, now - col * ps, 0};
      atomicAdd(&n_copies, 1);
    }
    const int held = a.by_page(now + ps - 1);
    for (int c = 0; c < n - copy; c++) {
      const int page = list[before + copy + c];
      row[held + c] = page;
      refs[page] = 1;
    }
  }
  __syncthreads();
  for (int e = tid; e < n_entries; e += kPlanThreads) a.table_out[e] = is[e];
  for (int p = tid; p < a.n_pages; p += kPlanThreads) a.refs_out[p] = refs[p];
  if (tid == 0) {
    const int pages = (int)(total >> 15);
    *a.ws.n_copies = n_copies;
    a.status[0] = (int)n_free - taken;
    a.status[1] = max(pages - (int)n_free, 0);
  }
}

struct CompactArgs {
  const int32_t *table, *refs;
  int32_t *table_out, *refs_out, *status;
  PlanSpace ws;
  int64_t n_entries;
  int page_size, n_pages;
};

// A table entry after a compaction. One that names no page, or a page that the counts
// call free, has no tokens: kept, it could name the page that another sequence's are
// moved to.
template <typename Load>
__device__ __forceinline__ int compact_entry(const CompactArgs& a, int page, Load remap) {
  if (page < 0) return page;
  const int to = page < a.n_pages ? remap(page) : -1;
  if (to < 0) kv_error();
  return to;
}

// The used pages past the first n_used go to the free ones among them, both in
// ascending order: the fewest moves that leave the pool dense. This form keeps its
// arrays in global memory, for pools that do not fit one CTA's shared memory.
__global__ void __launch_bounds__(kPlanThreads, 1) kv_compact_kernel(const CompactArgs a) {
  __shared__ int64_t part[33];
  pdl_begin();
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
    if (q < p1) {
      a.refs_out[q] = q < n_used ? max(r, 0) : 0;
      a.ws.remap[q] = r > 0 ? q : -1;   // a mover's is set below
    }
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
  for (int64_t i = tid; i < a.n_entries; i += kAll)
    a.table_out[i] =
        compact_entry(a, a.table[i], [&](int p) { return __ldcg(a.ws.remap + p); });
}

// Words of shared memory that the one-CTA form of a compaction takes.
__host__ __device__ constexpr int64_t compact_words(int64_t n_pages) { return 4 * n_pages; }

// The same by one CTA, its arrays in shared memory. Measured (B200): 96 pages, 11 of
// them moved, 4.9 us with the copies; in the cluster's form 13.1.
__global__ void __launch_bounds__(kPlanThreads, 1) kv_compact_cta_kernel(const CompactArgs a) {
  extern __shared__ __align__(16) int32_t words[];
  __shared__ uint32_t part[66], sums[32];
  pdl_begin();
  const int tid = threadIdx.x;
  int32_t *refs = words, *holes = refs + a.n_pages, *movers = holes + a.n_pages,
          *remap = movers + a.n_pages;
#pragma unroll 4
  for (int p = tid; p < a.n_pages; p += kPlanThreads) refs[p] = a.refs[p];
  __syncthreads();
  // each thread a run of pages
  const int per = (a.n_pages + kPlanThreads - 1) / kPlanThreads;
  const int p0 = min(a.n_pages, tid * per), p1 = min(a.n_pages, p0 + per);
  uint32_t n = 0;
  for (int p = p0; p < p1; p++) n += refs[p] > 0;
  const int n_used = (int)block_sum(n, sums);
  uint32_t hole = 0, mover = 0, n_holes, n_movers_u;
  for (int p = p0; p < p1; p++) {
    hole += p < n_used && refs[p] <= 0;
    mover += p >= n_used && refs[p] > 0;
  }
  block_scan2(hole, mover, part, &n_holes, &n_movers_u);
  const int n_movers = (int)n_movers_u;
  for (int p = p0; p < p1; p++) {
    remap[p] = refs[p] > 0 ? p : -1;   // a mover's is set below
    if (p < n_used && refs[p] <= 0) holes[hole++] = p;
    if (p >= n_used && refs[p] > 0) movers[mover++] = p;
  }
  __syncthreads();
  for (int m = tid; m < n_movers; m += kPlanThreads) {
    const int src = movers[m], dst = holes[m];
    a.ws.copies[m] = {src, dst, a.page_size, 0};
    remap[src] = dst;
    refs[dst] = refs[src];
  }
  if (tid == 0) {
    a.status[0] = n_used;
    a.status[1] = n_movers;
    *a.ws.n_copies = n_movers;
  }
  __syncthreads();
  for (int p = tid; p < a.n_pages; p += kPlanThreads)
    a.refs_out[p] = p < n_used ? max(refs[p], 0) : 0;
#pragma unroll 4
  for (int64_t i = tid; i < a.n_entries; i += kPlanThreads)
    a.table_out[i] = compact_entry(a, a.table[i], [&](int p) { return remap[p]; });
}

// ---------------------------------------------------------------- page copies

struct CopyArgs {
  char *k, *v;
  const PageCopy* copies;
  const int32_t* n_copies;
  int64_t layer_stride, page_stride, tok_stride, head_stride;   // bytes
  int n_layers, n_heads, row_chunks;   // 16-byte chunks of one head's row
  int n_parts;                         // parts of kCopyPart chunks in a whole page
  Div by_row, by_head, by_part;        // row_chunks, n_heads, n_parts
  int run;                             // a page's first `run` tokens are one run of memory,
                                       // or any number of tokens if it is 1
  bool head_major;                     // a page is stored head by head
};

constexpr int kCopyThreads = 256, kCopyUnroll = 8;
constexpr int kCopyResident = 4;   // CTAs on an SM (registers)

constexpr int kCopyPart = kCopyThreads * kCopyUnroll;   // 16-byte chunks

// One CTA a part of a copy at a time, K or V of layer blockIdx.y / 2: 32 KiB of the
// page's tokens, 16 bytes a thread, kCopyUnroll loads in flight before their stores.
// Source and target pages are never the same page, nor is a target another copy's
// source: plans copy pages in use to free ones. Bound by the memory's bandwidth, read
// + write. Measured (B200): 734 MB (700 pages of 64 KB in 4 layers) 134 us with the
// plan, 5.5 TB/s; 16 KiB parts and 4 loads in flight 132, but 30 against 27 us
// for a fork of 320 beams (77 MB).
__global__ void __launch_bounds__(kCopyThreads, kCopyResident) kv_copy_kernel(const CopyArgs a) {
  pdl_begin();   // waits for the plan
  const int which = blockIdx.y & 1, layer = blockIdx.y >> 1;
  const int units = *a.n_copies * a.n_parts;   // at most the pool's pages * n_parts
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int item = a.by_part(u);
    const PageCopy c = a.copies[item];
    const int n = c.n_tok * a.n_heads * a.row_chunks;
    const int i0 = (u - item * a.n_parts) * kCopyPart + threadIdx.x;
    char* pool = (which ? a.v : a.k) + layer * a.layer_stride;
    const char* src = pool + c.src * a.page_stride;
    char* dst = pool + c.dst * a.page_stride;
    const bool run = a.run == 1 || a.run == c.n_tok;
    uint4 x[kCopyUnroll];
    int64_t at[kCopyUnroll];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; j++) {
      const int i = i0 + j * kCopyThreads;
      at[j] = (int64_t)i * 16;
      if (!run) {
        const int r = a.by_row(i), k = i - r * a.row_chunks;
        const int hi = a.head_major ? r / c.n_tok : a.by_head(r);
        const int lo = r - hi * (a.head_major ? c.n_tok : a.n_heads);
        const int t = a.head_major ? lo : hi, h = a.head_major ? hi : lo;
        at[j] = t * a.tok_stride + h * a.head_stride + k * 16;
      }
      if (i < n) x[j] = *reinterpret_cast<const uint4*>(src + at[j]);
    }
#pragma unroll
    for (int j = 0; j < kCopyUnroll; j++)
      if (i0 + j * kCopyThreads < n) *reinterpret_cast<uint4*>(dst + at[j]) = x[j];
  }
}

// ---------------------------------------------------------------- host

int check_pool(const char* what, const void* k, const void* v, int64_t page_stride,
               int64_t tok_stride, int64_t head_stride, int64_t n_heads, int64_t head_dim,
               int64_t n_pages, int64_t page_size, int dtype, bool written) {
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
  if (written && (rows_overlap(n_pages, page_stride, head_dim) ||
                  rows_overlap(page_size, tok_stride, head_dim) ||
                  rows_overlap(n_heads, head_stride, head_dim)))
    return fail(WX_ERR_INVALID,
                "%s: the cache is written, but its rows share memory (strides %lld, %lld, %lld)",
                what, (long long)page_stride, (long long)tok_stride, (long long)head_stride);
  if (!k || !v) return fail(WX_ERR_INVALID, "%s: NULL cache", what);
  return WX_OK;
}

// The one-CTA forms' bound: what one CTA reads before a cluster of eight overtakes it,
// within its shared memory.
constexpr int64_t kCtaEntries = 16384;
constexpr int64_t kCtaWords = 220 * 1024 / 4;
static_assert(kCtaEntries <= 1 << 14, "a fork's running sums: 17 and 15 bits");

template <typename Args>
static cudaError_t launch_cta(void (*kernel)(Args), std::atomic<uint64_t>& done, const Args& a,
                              int64_t words, cudaStream_t st) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(done.load(std::memory_order_acquire) >> dev & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)(kCtaWords * 4));
    if (e != cudaSuccess) return e;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  }
  return launch_after(kernel, dim3(1), kPlanThreads, (int)words * 4, 1, st, a);
}

struct Pool {
  void *k, *v;
  int64_t n_layers, layer_stride, page_stride, tok_stride, head_stride, n_heads, head_dim,
      page_size;
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
  a.by_row = Div((uint32_t)a.row_chunks);
  a.by_head = Div((uint32_t)a.n_heads);
  a.head_major = p.tok_stride < p.head_stride;
  a.run = 0;
  if (p.head_stride == p.head_dim && p.tok_stride == p.n_heads * p.head_dim)
    a.run = 1;
  else if (p.tok_stride == p.head_dim && p.head_stride == p.page_size * p.head_dim)
    a.run = (int)p.page_size;
  const int64_t chunks = p.page_size * p.n_heads * a.row_chunks;
  a.n_parts = (int)((chunks + kCopyPart - 1) / kCopyPart);
  a.by_part = Div((uint32_t)a.n_parts);
  const int64_t units = max_copies * a.n_parts, y = 2 * p.n_layers;
  const int64_t most = std::max<int64_t>(1, (int64_t)sm_count() * kCopyResident / y);
  WX_CUDA_TRY(launch_after(kv_copy_kernel, dim3((unsigned)std::min(units, most), (unsigned)y),
                           kCopyThreads, 0, 1, st, a));
  return check_launch(what);
}

static int check_plan(const char* what, int64_t n_layers, int64_t layer_stride,
                      int64_t head_dim, int64_t es, int64_t n_seqs, int64_t width,
                      const void* ws, int64_t ws_bytes, int64_t n_pages) {
  if (n_layers < 1 || n_layers > 32767 || layer_stride < 0 || layer_stride * es % 16 ||
      rows_overlap(n_layers, layer_stride, head_dim))
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
                    head_dim, n_pages, page_size, dtype, true));
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
  a.by_page = Div((uint32_t)page_size);
  a.width = (int)(ld_table < 0x7fffffff ? ld_table : 0x7fffffff);
  a.n_pages = n_pages;
  // 16 bytes a thread where the source rows allow it, else one element
  const bool vec = !((a.s_seq | a.s_tok | a.s_head | (int64_t)(uintptr_t)k |
                      (int64_t)(uintptr_t)v) & 15);
  const int64_t unit = vec ? 16 : es;
  a.row_units = (int)(head_dim * es / unit);
  a.by_row = Div((uint32_t)a.row_units);
  a.by_token = Div((uint32_t)(a.row_units * a.n_heads));
  const int64_t units = n_tokens * n_heads * a.row_units;
  const int64_t blocks = (units + 256 * kAppendUnroll - 1) / (256 * kAppendUnroll);
  const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536), (unsigned)n_seqs, 2);
  cudaStream_t st = as_stream(stream);
  if (vec)
    WX_CUDA_TRY(launch_after(kv_append_kernel<uint4>, grid, 256, 0, 1, st, a));
  else if (es == 2)
    WX_CUDA_TRY(launch_after(kv_append_kernel<uint16_t>, grid, 256, 0, 1, st, a));
  else
    WX_CUDA_TRY(launch_after(kv_append_kernel<uint32_t>, grid, 256, 0, 1, st, a));
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
                    head_dim, n_pages, page_size, dtype, true));
  WX_TRY(check_plan("kv_fork", n_layers, layer_stride, head_dim, dtype == WX_DTYPE_BF16 ? 2 : 4,
                    n_seqs, width, workspace, workspace_bytes, n_pages));
  if (!table || !lens || !refs || !table_out || !lens_out || !refs_out || !status_out)
    return fail(WX_ERR_INVALID, "kv_fork: NULL argument");
  if (table == table_out || lens == lens_out || refs == refs_out)
    return fail(WX_ERR_INVALID, "kv_fork: the new page table cannot be written over the old one");
  if (n_heads * head_dim * page_size > 0x7fffffff || width * page_size > (1 << 30))
    return fail(WX_ERR_INVALID, "kv_fork: a page of over 2^31 - 1 elements or a row of over 2^30 tokens");
  // the running sum of pages asked for is in 32 bits, a row's width and a copy each at most
  if (n_seqs * width > (1 << 30))
    return fail(WX_ERR_INVALID, "kv_fork: a page table of over 2^30 entries: %lld x %lld",
                (long long)n_seqs, (long long)width);
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
  a.by_page = Div((uint32_t)page_size);
  a.by_width = Div((uint32_t)width);
  cudaStream_t st = as_stream(stream);
  const int64_t words = fork_words(n_seqs, width, n_pages);
  static std::atomic<uint64_t> ready{0};
  if (n_seqs * width <= kCtaEntries && words <= kCtaWords)
    WX_CUDA_TRY(launch_cta(kv_fork_cta_kernel, ready, a, words, st));
  else
    WX_CUDA_TRY(launch_after(kv_fork_kernel, dim3(kPlanCtas), kPlanThreads, 0, kPlanCtas, st, a));
  WX_TRY(check_launch("kv_fork"));
  if (!grow) return WX_OK;   // nothing is written, so nothing is copied
  const Pool p = {k_cache, v_cache, n_layers, layer_stride, page_stride, tok_stride,
                  head_stride, n_heads, head_dim, page_size, dtype};
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
                    head_dim, n_pages, page_size, dtype, true));
  WX_TRY(check_plan("kv_compact", n_layers, layer_stride, head_dim,
                    dtype == WX_DTYPE_BF16 ? 2 : 4, n_seqs, width, workspace, workspace_bytes,
                    n_pages));
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
  const int64_t words = compact_words(n_pages);
  static std::atomic<uint64_t> ready{0};
  if (a.n_entries <= kCtaEntries && words <= kCtaWords)
    WX_CUDA_TRY(launch_cta(kv_compact_cta_kernel, ready, a, words, st));
  else
    WX_CUDA_TRY(
        launch_after(kv_compact_kernel, dim3(kPlanCtas), kPlanThreads, 0, kPlanCtas, st, a));
  WX_TRY(check_launch("kv_compact"));
  const Pool p = {k_cache, v_cache, n_layers, layer_stride, page_stride, tok_stride,
                  head_stride, n_heads, head_dim, page_size, dtype};
  return launch_copies("kv_compact copies", p, a.ws, n_pages / 2 + 1, st);
}

}  // extern "C"
