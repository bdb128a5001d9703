// Shared by the operators on the paged key-value cache.
#pragma once
#include "common.cuh"
#include "wxb200_internal.h"

namespace wx {

// Division of n < 2^31 by an invariant d (Granlund and Montgomery, "Division by
// invariant integers using multiplication", 1994): a multiply, an add and a shift
// where the hardware's division takes some twenty instructions.
struct Div {
  uint32_t d, mul, shift;
  Div() = default;
  explicit Div(uint32_t by) : d(by), shift(0) {
    while ((1ull << shift) < by) shift++;
    mul = (uint32_t)((((1ull << shift) - by) << 32) / by + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int operator()(int n) const {
    return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift);
  }
#endif
};

// The decoder's kernels are launched one after another, each of a few microseconds, so
// each is a programmatic dependent of the kernel before it on the stream: it may take
// its place while that one ends. pdl_begin() comes before a kernel's first access to
// memory: it returns when all that was on the stream before is complete and visible,
// and then lets the next kernel be placed. Every thread calls it, so that a kernel that
// is complete stands for all before it. (The long kernels call pdl_wait() there, and
// pdl_launch_dependents() when their loops are done.) Nothing that another kernel may
// write is read by a read-only load: that would promise that it stays as it is from this
// kernel's start on, when the kernel before it may still be writing.
#ifdef __CUDACC__
__device__ __forceinline__ void pdl_begin() {
  pdl_wait();
  pdl_launch_dependents();
}
#endif

// Launches a kernel so, or (early false) once the stream's last kernel has ended, in
// clusters of `cluster` CTAs along x.
template <typename... KArgs, typename... Args>
inline cudaError_t launch(bool early, void (*kernel)(KArgs...), dim3 grid, int threads, int smem,
                          int cluster, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (early) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    n++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = (unsigned)n;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}
template <typename... KArgs, typename... Args>
inline cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, int threads, int smem,
                                int cluster, cudaStream_t st, Args&&... args) {
  return launch(true, kernel, grid, threads, smem, cluster, st, std::forward<Args>(args)...);
}

// Whether rows of head_dim elements, `stride` apart, lie over one another.
inline bool rows_overlap(int64_t n, int64_t stride, int64_t head_dim) {
  return n > 1 && stride < head_dim && stride > -head_dim;
}

// Checks a pool's types, sizes, strides (elements) and alignment; `written`: and that no
// two of its rows share memory, which a pool that is only read may do.
int check_pool(const char* what, const void* k, const void* v, int64_t page_stride,
               int64_t tok_stride, int64_t head_stride, int64_t n_heads, int64_t head_dim,
               int64_t n_pages, int64_t page_size, int dtype, bool written);

// WX_DEVERR_PAGE as recorded by the cache's kernels on the current device: OR it
// into *flags, and clear it when asked.
int kv_take_error(int* flags, bool clear);
int paged_attention_take_error(int* flags, bool clear);

}  // namespace wx
