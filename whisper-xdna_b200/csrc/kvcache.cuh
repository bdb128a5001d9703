// Shared by the operators on the paged key-value cache.
#pragma once
#include "wxb200_internal.h"

namespace wx {

// Checks a pool's types, sizes, strides (elements) and alignment.
int check_pool(const char* what, const void* k, const void* v, int64_t page_stride,
               int64_t tok_stride, int64_t head_stride, int64_t n_heads, int64_t head_dim,
               int64_t n_pages, int64_t page_size, int dtype);

// WX_DEVERR_PAGE as recorded by the cache's kernels on the current device: OR it
// into *flags, and clear it when asked.
int kv_take_error(int* flags, bool clear);
int paged_attention_take_error(int* flags, bool clear);

}  // namespace wx
