// What the kernels of the paged 8-bit KV cache share: limits, argument checks, dispatch.
#pragma once
#include <type_traits>

#include "common.hpp"

namespace sfl {

// Of a page's scale 2^e: pages of zeros have it, and values below 2^-110 no codes of their
// own. Codes under it are normal numbers of bf16.
constexpr int kLeastExponent = -100;

// A barrier after which every thread of the workgroup sees what the others stored: their
// stores have arrived.
__device__ __forceinline__ void settle() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

inline int log2_of(int x) {
  int n = 0;
  while ((1 << n) < x) ++n;
  return n;
}

inline int check_paged(const char* what, int batch, int places, int pages, int page_size) {
  if (batch <= 0 || places <= 0 || pages <= 0) return set_error(SFL_ERR_INVALID, "%s: batch, places and pages must be positive", what);
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: unsupported page size %d", what, page_size);
  if (long(places) * page_size > SFL_CACHE_MAX_SLOTS)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: at most %d slots", what, SFL_CACHE_MAX_SLOTS);
  if (pages > SFL_PAGE_MAX_PAGES) return set_error(SFL_ERR_UNSUPPORTED, "%s: at most %d pages", what, SFL_PAGE_MAX_PAGES);
  return SFL_OK;
}

inline int check_head_dim(const char* what, int head_dim) {
  if (head_dim != 16 && head_dim != 32 && head_dim != 64 && head_dim != 128)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: unsupported head dim %d", what, head_dim);
  return SFL_OK;
}

template <typename T, typename F>
int paged_dims(int dim, F&& f) {
  switch (dim) {
    case 16: return f(T{}, std::integral_constant<int, 16>{});
    case 32: return f(T{}, std::integral_constant<int, 32>{});
    case 64: return f(T{}, std::integral_constant<int, 64>{});
    default: return f(T{}, std::integral_constant<int, 128>{});
  }
}
template <typename F>
int paged_types(int dtype, int dim, F&& f) {
  switch (dtype) {
    case SFL_DTYPE_F32: return paged_dims<float>(dim, f);
    case SFL_DTYPE_BF16: return paged_dims<bf16_t>(dim, f);
    default: return paged_dims<f16_t>(dim, f);
  }
}

}  // namespace sfl
