// Internals shared by the paged-cache kernels (paged_norm.cu, paged_attention.cu,
// paged_attention_tc.cu): the batch as the kernels see it and its checks.
#pragma once
#include <climits>
#include "ie_common.cuh"

namespace ie {

// The sequences of a call (device arrays). Every index derived from them is
// checked against these extents before it addresses memory, so a bad table
// or length gives a status word, never a stray access.
struct PagedBatch {
  const int* q_start;     // [B + 1]
  const int* kv_len;      // [B]
  const int* page_table;  // [B][max_pages], row stride ld_table
  int64_t ld_table;
  int B, T, max_pages;
};

struct PagedLayout {
  int num_pages, page_size, page_log2, n_kv_heads;
  int64_t page_stride, head_stride, row_stride;  // elements
};

// Checks of the arguments every paged entry point shares.
inline int check_paged(const ie_paged_cache* c, int B, int T, const int* page_table, int64_t ld_table, int max_pages,
                       const int* q_start, const int* kv_len) {
  if (!c || B < 0 || T < 0) return IE_ERR_INVALID_ARG;
  if (!c->k || !c->v || c->num_pages <= 0 || c->n_kv_heads <= 0) return IE_ERR_INVALID_ARG;
  if (c->head_dim != 64 && c->head_dim != 128) return IE_ERR_UNSUPPORTED;
  const int ps = c->page_size;
  if (ps < 16 || ps > 256 || (ps & (ps - 1))) return IE_ERR_UNSUPPORTED;
  // a row, a head's rows and a page do not overlap their neighbours: either
  // [page][head][row] or [page][row][head] order, padded or not
  if (c->row_stride < c->head_dim || c->head_stride < c->head_dim || c->page_stride < c->head_dim)
    return IE_ERR_INVALID_ARG;
  const int64_t row_span = (int64_t)(ps - 1) * c->row_stride, head_span = (int64_t)(c->n_kv_heads - 1) * c->head_stride;
  if (c->row_stride > (INT64_C(1) << 40) || c->head_stride > (INT64_C(1) << 40) ||
      c->page_stride > (INT64_C(1) << 36))
    return IE_ERR_INVALID_ARG;
  const bool head_major = c->n_kv_heads == 1 || c->head_stride >= row_span + c->head_dim;
  const bool row_major = c->row_stride >= head_span + c->head_dim;
  if (!head_major && !row_major) return IE_ERR_INVALID_ARG;
  if (c->num_pages > 1 && c->page_stride < row_span + head_span + c->head_dim) return IE_ERR_INVALID_ARG;
  if (!aligned16(c->k) || !aligned16(c->v) || c->row_stride % 8 || c->head_stride % 8 || c->page_stride % 8)
    return IE_ERR_ALIGNMENT;
  if (B == 0 || T == 0) return IE_OK;
  if (!page_table || !q_start || !kv_len || max_pages <= 0 || ld_table < max_pages) return IE_ERR_INVALID_ARG;
  for (const void* p : {(const void*)page_table, (const void*)q_start, (const void*)kv_len})
    if (reinterpret_cast<uintptr_t>(p) & 3u) return IE_ERR_ALIGNMENT;
  // positions are 32-bit, rounded up to whole blocks of keys and tiles of tokens included
  if ((int64_t)max_pages * ps > INT_MAX - 1023) return IE_ERR_INVALID_ARG;
  return IE_OK;
}

inline PagedLayout paged_layout(const ie_paged_cache* c) {
  PagedLayout l;
  l.num_pages = c->num_pages;
  l.page_size = c->page_size;
  l.page_log2 = 31 - __builtin_clz((unsigned)c->page_size);
  l.n_kv_heads = c->n_kv_heads;
  l.page_stride = c->page_stride;
  l.head_stride = c->head_stride;
  l.row_stride = c->row_stride;
  return l;
}

// Sequence that owns row `token`: the last b with q_start[b] <= token, -1
// before the first and B behind the last. Called by a whole warp; each round
// narrows the range 32-fold with one load per lane.
__device__ __forceinline__ int paged_owner(const int* __restrict__ q_start, int B, int token) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = B + 1;  // the answer + 1 = number of entries <= token; entries below lo are
  while (n > 0) {
    const int step = (n + 31) >> 5;
    const int i = lo + (lane + 1) * step - 1;  // last entry of this lane's part
    const bool le = i < lo + n && q_start[i] <= token;
    const int full = __popc(__ballot_sync(0xffffffffu, le));
    const int end = lo + n;
    lo += full * step;
    n = min(step - 1, end - lo);  // the part after the full ones, without its last entry when that one was tested
    if (full == 32) break;
  }
  return lo - 1;
}

}  // namespace ie
