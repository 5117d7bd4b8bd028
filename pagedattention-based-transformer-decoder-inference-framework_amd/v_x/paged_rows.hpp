// A batch of rows of tokens in a caller's pages (kv_quant.hip, pa_tree.hip): what is checked
// on the host, and where a token lies.
#pragma once

#include <string>

#include "common.hpp"
#include "pa_decode.hpp"

namespace llm {

// Bytes per element of the pools that a batch of rows may lie in (0: others).
inline int paged_elem_size(int kvt) {
  return kvt == LLM_I8 || kvt == LLM_E4M3 ? 1 : kvt == LLM_F16 || kvt == LLM_BF16 ? 2 : 0;
}
inline int value_size(int dtype) {
  return dtype == LLM_F32 ? 4 : dtype == LLM_F16 || dtype == LLM_BF16 ? 2 : 0;
}
inline size_t paged_stride(const pa_kv_view& v) {
  return v.page_stride > 0 ? (size_t)v.page_stride
                           : (size_t)v.page_size * v.head_dim * paged_elem_size(v.kv_dtype);
}
inline bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// The view's own sizes, the same for every call on it.
inline int check_paged_view(const char* name, const pa_kv_view* kv, const pa_kv_scales* scales) {
  const std::string who = std::string(name) + ": ";
  LLM_REQUIRE(kv, who + "kv view is NULL");
  LLM_REQUIRE(kv->k_pool && kv->v_pool && kv->page_table, who + "kv pointers NULL");
  LLM_REQUIRE(paged_elem_size(kv->kv_dtype) > 0,
              who + "kv_dtype must be LLM_F16, LLM_BF16, LLM_I8 or LLM_E4M3");
  LLM_REQUIRE(kv->num_pages > 0 && kv->num_beams > 0 && kv->num_heads > 0 && kv->max_tiles > 0 &&
                  kv->page_size > 0 && kv->head_dim > 0,
              who + "empty kv view");
  LLM_REQUIRE((long long)kv->max_tiles * kv->page_size <= 1 << 30,
              who + "max_tiles * page_size above 2^30 tokens");
  const size_t stride = paged_stride(*kv);
  LLM_REQUIRE(kv->page_stride >= 0 && stride % 16 == 0 &&
                  stride >= (size_t)kv->page_size * kv->head_dim * paged_elem_size(kv->kv_dtype),
              who + "page_stride must be 0 or >= one page, and pages multiples of 16 bytes");
  LLM_REQUIRE((long long)kv->num_pages <= (1LL << 47) / (long long)stride, who + "pool too large");
  LLM_REQUIRE(aligned16(kv->k_pool) && aligned16(kv->v_pool), who + "pools must be 16-byte aligned");
  if (!scales) return LLM_OK;
  LLM_REQUIRE(scales->k_scale && scales->v_scale, who + "scale pointers NULL");
  LLM_REQUIRE(scales->page_stride == 0 || scales->page_stride >= kv->page_size,
              who + "the scales' page_stride must be 0 or >= page_size");
  return LLM_OK;
}

__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return min(max(x, lo), hi); }

}  // namespace llm
