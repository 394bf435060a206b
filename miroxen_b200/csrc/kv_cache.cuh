// What the kernels that fill and read the paged key/value cache share (include/mxk.h: MxkKvCache).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace mxk {

// The code the kernels leave in the device error word when an index read on the device is out of range.
constexpr int kErrBadIndex = MXK_DEVICE_ERR_BAD_INDEX;

template <bool E4M3> struct KvElem { using type = uint16_t; };
template <> struct KvElem<true> { using type = uint8_t; };

// Host-side checks of a cache descriptor that need no GPU.
inline int check_cache(const char* name, const MxkKvCache* c) {
  if (!c) return fail(MXK_ERR_INVALID_ARG, "%s: null cache", name);
  if (c->type != MXK_KV_BF16 && c->type != MXK_KV_E4M3) return fail(MXK_ERR_INVALID_ARG, "%s: unknown cache type %d", name, c->type);
  const int vec = c->type == MXK_KV_BF16 ? 8 : 16;  // elements in 16 bytes
  if (c->D < vec || c->D > MXK_ATTN_MAX_HEAD_DIM || c->D % vec != 0)
    return fail(MXK_ERR_INVALID_ARG, "%s: head dimension %d must be a multiple of %d and at most %d", name, c->D, vec, MXK_ATTN_MAX_HEAD_DIM);
  if (c->Hkv <= 0 || c->page_size <= 0 || c->n_seqs < 0 || c->max_pages < 0 || c->num_pages < 0)
    return fail(MXK_ERR_INVALID_ARG, "%s: Hkv=%d page_size=%d n_seqs=%d max_pages=%d num_pages=%lld", name, c->Hkv, c->page_size, c->n_seqs,
                c->max_pages, (long long)c->num_pages);
  if (int64_t(c->max_pages) * c->page_size >= (int64_t(1) << 31))
    return fail(MXK_ERR_TOO_LARGE, "%s: max_pages * page_size = %lld tokens per sequence", name, (long long)c->max_pages * c->page_size);
  if (c->num_pages >= (int64_t(1) << 31)) return fail(MXK_ERR_TOO_LARGE, "%s: num_pages=%lld", name, (long long)c->num_pages);
  if (c->page_stride % vec != 0 || c->token_stride % vec != 0 || c->head_stride % vec != 0 || c->page_stride < 0 || c->token_stride < 0 ||
      c->head_stride < 0 || c->table_stride < 0)
    return fail(MXK_ERR_INVALID_ARG, "%s: cache strides must be multiples of 16 bytes", name);
  if ((c->Hkv > 1 && c->head_stride < c->D) || (c->page_size > 1 && c->token_stride < c->D) || (c->num_pages > 1 && c->page_stride < c->D))
    return fail(MXK_ERR_INVALID_ARG, "%s: cache strides smaller than a head's D=%d channels", name, c->D);
  if (!aligned(static_cast<const char*>(c->k), 16) || !aligned(static_cast<const char*>(c->v), 16))
    return fail(MXK_ERR_INVALID_ARG, "%s: cache pointers must be 16-byte aligned", name);
  if (c->type == MXK_KV_BF16 && (c->k_scale || c->v_scale)) return fail(MXK_ERR_INVALID_ARG, "%s: scales belong to an e4m3 cache", name);
  return MXK_OK;
}

// Pointers a call that has work to do needs.
inline int check_cache_pointers(const char* name, const MxkKvCache* c) {
  if (!c->k || !c->v || !c->page_table) return fail(MXK_ERR_INVALID_ARG, "%s: null cache pages or page table", name);
  return MXK_OK;
}

// Element offset of token `pos` of sequence `seq` (head 0), or -1 when the token or its page is out of range.
__device__ __forceinline__ int64_t kv_token_offset(const MxkKvCache& c, int seq, int pos) {
  if (seq < 0 || seq >= c.n_seqs || pos < 0) return -1;
  const int page_i = pos / c.page_size;
  if (page_i >= c.max_pages) return -1;
  const int page = c.page_table[int64_t(seq) * c.table_stride + page_i];
  if (page < 0 || page >= c.num_pages) return -1;
  return int64_t(page) * c.page_stride + int64_t(pos - page_i * c.page_size) * c.token_stride;
}

}  // namespace mxk
