// Shared by the operators on the paged key-value cache.
#pragma once
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

// Checks a pool's types, sizes, strides (elements) and alignment.
int check_pool(const char* what, const void* k, const void* v, int64_t page_stride,
               int64_t tok_stride, int64_t head_stride, int64_t n_heads, int64_t head_dim,
               int64_t n_pages, int64_t page_size, int dtype);

// WX_DEVERR_PAGE as recorded by the cache's kernels on the current device: OR it
// into *flags, and clear it when asked.
int kv_take_error(int* flags, bool clear);
int paged_attention_take_error(int* flags, bool clear);

}  // namespace wx
