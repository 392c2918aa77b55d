// Paged K/V cache: how the device code of pages.hip and page_attention.hip addresses it, and the
// host's checks of a qe_pages (include/qe.h).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/qe.h"

namespace qe {

constexpr uint32_t kPageDim = 128;  // head_dim
constexpr uint32_t kPageRun = 16;   // positions transposed together in a V page

// A checked qe_pages in the widths the kernels use. Everything that the plan (table, lens, starts)
// says is device data and is bounds-checked where it is used.
struct PagePlan {
  const int32_t *table, *lens, *starts;
  uint32_t n_seqs, n_pages, n_kv, page_shift, table_stride;
};
struct PageStore {
  uint8_t *k, *v, *k_exp, *v_exp;
};

// Checks a qe_pages and splits it; QE_OK or the status after set_error.
int check_pages(const qe_pages* p, PagePlan* plan, PageStore* store);

#ifdef __HIPCC__
// Positions the table has entries for.
__device__ __forceinline__ int64_t capacity_of(const PagePlan& p) { return int64_t(p.table_stride) << p.page_shift; }

// Page of position pos of sequence s, or -1 where there is none (0 <= pos < capacity).
__device__ __forceinline__ int32_t page_of(const PagePlan& p, uint32_t s, int64_t pos) {
  const int32_t page = p.table[size_t(s) * p.table_stride + size_t(pos >> p.page_shift)];
  return uint32_t(page) < p.n_pages ? page : -1;
}

// Row index (page, KV head, offset) of a position, counted in rows of 128 elements; also the index
// of its exponent byte.
__device__ __forceinline__ size_t page_row(const PagePlan& p, int32_t page, uint32_t head, uint32_t off) {
  return ((size_t(page) * p.n_kv + head) << p.page_shift) + off;
}
// Element index in a V page of that row's dim 0; dim d is 16 d further.
__device__ __forceinline__ size_t v_element(const PagePlan& p, int32_t page, uint32_t head, uint32_t off) {
  return page_row(p, page, head, off & ~(kPageRun - 1)) * kPageDim + (off & (kPageRun - 1));
}

// 2^(e - 127) for an exponent byte e (0 would be 2^-127: taken as 0, which no append writes).
__device__ __forceinline__ float exp_scale(uint32_t e) { return __uint_as_float(e << 23); }
#endif

}  // namespace qe
