// Host-side checks shared by the paged-cache entries (cache_rows.cu, cache_attention.cu,
// verify_drafts.cu): the cache's form, and layouts of activations beside it.
#pragma once

#include "plan_common.h"

namespace t4a {
namespace cache {

constexpr int kMaxDim = 256;
constexpr int kRowAlign = 16;  // bytes: a row's start, so that 16-byte copies serve every row

inline int element_size(int dtype) {
  switch (dtype) {
    case T4A_CUDA_F32: return 4;
    case T4A_F16:
    case T4A_BF16: return 2;
    case T4A_I8:
    case T4A_E4M3: return 1;
    default: return 0;
  }
}

inline bool is_cache_kind(int kind) { return kind == T4A_F16 || kind == T4A_BF16 || kind == T4A_I8 || kind == T4A_E4M3; }
inline bool is_quantised(int kind) { return kind == T4A_I8 || kind == T4A_E4M3; }
inline bool is_row_dtype(int dtype) { return dtype == T4A_CUDA_F32 || dtype == T4A_F16 || dtype == T4A_BF16; }

inline bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// A layout of `rank` axes within its buffer.
inline int check_tensor(const t4a_cuda_layout* l, int rank, long long len, int element_bytes) {
  T4A_TRY(plan::check_layout(l));
  if (l->rank != rank) return T4A_ERR_RANK_LENGTH;
  return plan::check_span(*l, len, element_bytes);
}

// Rows along axis 0: unit stride there.
inline int check_rows(const t4a_cuda_layout* l, int rank, long long len, int element_bytes) {
  T4A_TRY(check_tensor(l, rank, len, element_bytes));
  if (l->extents[0] > 1 && l->strides[0] != 1) return T4A_ERR_INVALID_STRIDE;
  return T4A_OK;
}

// A destination's elements are apart; one without elements is.
inline int check_destination(const t4a_cuda_layout& l) {
  for (int d = 0; d < l.rank; ++d)
    if (l.extents[d] == 0) return T4A_OK;
  return plan::require_destination(l);
}

// Whether the rows of `l` start on multiples of `bytes`.
inline bool rows_aligned(const void* base, const t4a_cuda_layout& l, int element_bytes, unsigned bytes) {
  if (!aligned(static_cast<const char*>(base) + l.offset * element_bytes, bytes)) return false;
  for (int d = 1; d < l.rank; ++d)
    if (l.extents[d] > 1 && (l.strides[d] * element_bytes) % static_cast<long long>(bytes) != 0) return false;
  return true;
}

// What the kernels take of one of the cache's tensors: a base and strides in elements.
struct Pages {
  unsigned char* base;
  float* scale;
  long long head, place, page;                    // strides of the rows, in bytes
  long long scale_head, scale_place, scale_page;  // strides of the scales, in elements
};

struct View {
  Pages k, v;
  long long pages;
  int page_size, heads, dim;
};

inline int check_side(int kind, void* base, float* scale, const t4a_cuda_layout& l, long long len,
                      const t4a_cuda_layout& sl, long long scale_len, bool written, bool pointers, Pages* out) {
  const int esize = element_size(kind);
  T4A_TRY(check_rows(&l, 4, len, esize));
  if (l.extents[0] <= 0 || l.extents[0] % 16 != 0 || l.extents[0] > kMaxDim) return T4A_ERR_SHAPE_MISMATCH;
  if (written) T4A_TRY(check_destination(l));
  long long count;
  T4A_TRY(plan::element_count(l, &count));
  if (pointers && count != 0 && base == nullptr) return T4A_ERR_NULL_ARGUMENT;
  if (count != 0 && !rows_aligned(base, l, esize, kRowAlign)) return T4A_ERR_INVALID_STRIDE;
  out->base = static_cast<unsigned char*>(base) + l.offset * esize;
  out->head = l.strides[1] * esize;
  out->place = l.strides[2] * esize;
  out->page = l.strides[3] * esize;
  out->scale = nullptr;
  out->scale_head = out->scale_place = out->scale_page = 0;
  if (is_quantised(kind)) {
    T4A_TRY(check_tensor(&sl, 3, scale_len, 4));
    if (written) T4A_TRY(check_destination(sl));
    for (int d = 0; d < 3; ++d)
      if (sl.extents[d] != l.extents[d + 1]) return T4A_ERR_SHAPE_MISMATCH;
    if (pointers && count != 0 && scale == nullptr) return T4A_ERR_NULL_ARGUMENT;
    if (!aligned(scale, 4)) return T4A_ERR_INVALID_STRIDE;
    out->scale = scale + sl.offset;
    out->scale_head = sl.strides[0];
    out->scale_place = sl.strides[1];
    out->scale_page = sl.strides[2];
  }
  return T4A_OK;
}

// The cache as the kernels take it; `written`: its rows are destinations; `pointers`: its buffers
// are given, not the layouts alone.
inline int check_cache(const t4a_kv_cache* c, bool written, bool pointers, View* out) {
  if (c == nullptr) return T4A_ERR_NULL_ARGUMENT;
  if (!is_cache_kind(c->kind)) return T4A_ERR_UNSUPPORTED_DTYPE;
  T4A_TRY(check_side(c->kind, c->k, c->k_scale, c->k_layout, c->k_len, c->k_scale_layout, c->k_scale_len, written,
                     pointers, &out->k));
  T4A_TRY(check_side(c->kind, c->v, c->v_scale, c->v_layout, c->v_len, c->v_scale_layout, c->v_scale_len, written,
                     pointers, &out->v));
  for (int d = 0; d < 4; ++d)
    if (c->k_layout.extents[d] != c->v_layout.extents[d]) return T4A_ERR_SHAPE_MISMATCH;
  const long long* e = c->k_layout.extents;
  if (e[1] > INT_MAX || e[2] > INT_MAX || e[3] > INT_MAX) return T4A_ERR_DOMAIN_TOO_LARGE;
  long long places;
  if (plan::mul_overflows(e[2], e[3], &places)) return T4A_ERR_OVERFLOW;
  out->pages = e[3];
  out->page_size = static_cast<int>(e[2]);
  out->heads = static_cast<int>(e[1]);
  out->dim = static_cast<int>(e[0]);
  return T4A_OK;
}

}  // namespace cache
}  // namespace t4a
