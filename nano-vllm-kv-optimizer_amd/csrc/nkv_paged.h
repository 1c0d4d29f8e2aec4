// The paged cache of the dense path, as its kernels see it: keys and values
// [pages][Hkv][page][D] (any strides but the innermost), bf16, or int8 codes
// with an fp32 scale a row [pages][Hkv][page].
#pragma once

#include "nkv_common.h"

namespace nkv {

struct PagedCache {
  char* k;
  char* v;
  float* ks;       // nullptr: bf16
  float* vs;
  int64_t sp, sh, st;   // elements from page to page, head to head, token to token
  int pages, hkv, page, shift;   // page = 1 << shift tokens
};

// Checks the cache arguments that every paged entry point takes and fills c.
int fill_paged(const char* who, void* k, void* v, float* k_scale, float* v_scale, int64_t page_stride,
               int64_t head_stride, int64_t token_stride, int pages, int num_kv_heads, int page_size, int head_dim,
               PagedCache* c);

// Rows whose largest magnitude is below are zero in 8 bits (127 / a stays finite).
constexpr float kTinyRow = 0x1p-119f;

// Element offset of a slot's row of head h (slot in [0, pages * page)).
__device__ __forceinline__ int64_t paged_row(const PagedCache& c, int slot, int h) {
  return c.sp * (slot >> c.shift) + c.sh * h + c.st * (slot & (c.page - 1));
}
// The row's place in the scales.
__device__ __forceinline__ int64_t paged_scale(const PagedCache& c, int slot, int h) {
  return ((static_cast<int64_t>(slot >> c.shift) * c.hkv + h) << c.shift) + (slot & (c.page - 1));
}
__device__ __forceinline__ bool paged_slot_ok(const PagedCache& c, int slot) {
  return slot >= 0 && (slot >> c.shift) < c.pages;
}

}  // namespace nkv
