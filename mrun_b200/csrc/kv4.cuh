// The 4-bit paged K/V pool: uint8 [pages, kv_heads, page_size / 16, block_bytes].
//
// A block holds 16 consecutive tokens of one KV head, contiguous so that one bulk copy moves
// it: K codes [16][D / 2], V codes [16][D / 2] (two dimensions a byte, the even one in the low
// nibble), then [16][D / G] pairs (scale, minimum) of bf16 for K and the same for V. A group of
// G dimensions x is held as m = bf16(min x), s = bf16((max x - m) / 15) and codes
// c = round_half_even((x - m) / s) clipped to 0..15, and stands for m + s * c.
#pragma once

#include "common.cuh"

#include <math.h>

namespace mrb {

constexpr int KV4_TILE = 16;

__host__ __device__ constexpr int kv4_codes_bytes(int d) { return KV4_TILE * d / 2; }
__host__ __device__ constexpr int kv4_params_bytes(int d, int g) { return KV4_TILE * (d / g) * 4; }
__host__ __device__ constexpr int kv4_block_bytes(int d, int g) {
  return 2 * (kv4_codes_bytes(d) + kv4_params_bytes(d, g));
}

inline bool kv4_shape_ok(int64_t d, int64_t g) {
  return (d == 64 || d == 128) && (g == 32 || g == 64 || g == 128) && g <= d;
}

// The pool as every kernel gets it.
struct Kv4Pool {
  unsigned char* base;
  int64_t stride_page, stride_head;  // bytes
  int page_size, num_pages;
  int hkv;
  // block of `tok` (a position inside its page) for a page and KV head: 64-bit, a pool may
  // pass 4 GiB
  __device__ __forceinline__ unsigned char* block(int64_t page, int head, int tok, int block_bytes) const {
    return base + page * stride_page + head * stride_head + (int64_t)(tok / KV4_TILE) * block_bytes;
  }
};

// The checks that every entry point with a pool shares (host).
inline int kv4_check_pool(const char* what, const void* pool, int64_t num_pages, int64_t hkv, int64_t page_size,
                          int64_t stride_page, int64_t stride_head, int64_t d, int64_t g, Kv4Pool* out) {
  if (!kv4_shape_ok(d, g))
    return fail(MRB_ERR_UNSUPPORTED, "%s: head_dim 64 or 128 with groups of 32, 64 or 128 dimensions", what);
  if (hkv < 1 || num_pages < 1 || page_size < 1) return fail(MRB_ERR_ARG, "%s: bad pool sizes", what);
  if (page_size % KV4_TILE) return fail(MRB_ERR_UNSUPPORTED, "%s: page_size must be a multiple of 16", what);
  if (num_pages * page_size > INT32_MAX)
    return fail(MRB_ERR_UNSUPPORTED, "%s: the pool's slots must be numbered in 32 bits", what);
  if (!pool) return fail(MRB_ERR_ARG, "%s: null pool", what);
  const int64_t head_bytes = page_size / KV4_TILE * kv4_block_bytes((int)d, (int)g);
  if (!aligned(pool, 16) || stride_page % 128 || stride_head % 128)
    return fail(MRB_ERR_ARG, "%s: the pool must be 16-byte aligned and its strides multiples of 128 bytes", what);
  if (stride_head < head_bytes || stride_page < head_bytes)
    return fail(MRB_ERR_ARG, "%s: the pool's strides are smaller than its blocks", what);
  out->base = (unsigned char*)pool;
  out->stride_page = stride_page;
  out->stride_head = stride_head;
  out->page_size = (int)page_size;
  out->num_pages = (int)num_pages;
  out->hkv = (int)hkv;
  return MRB_OK;
}

constexpr int KV4_MAX_GROUP = 16;  // query heads a KV head

// The checks that the two attention entry points share (host).
inline int kv4_check_attention(const char* what, const void* q, int64_t tokens, int64_t rows, int64_t hq, int64_t hkv,
                               int64_t head_dim, int64_t group, const void* pool, int64_t num_pages, int64_t page_size,
                               int64_t stride_page, int64_t stride_head, const int32_t* block_table,
                               int64_t num_seqs, int64_t block_table_stride, int64_t max_pages_per_seq, const int32_t* row_len,
                               float scale, const void* out, Kv4Pool* p) {
  const int rc = kv4_check_pool(what, pool, num_pages, hkv, page_size, stride_page, stride_head, head_dim, group, p);
  if (rc != MRB_OK) return rc;
  if (tokens < 0 || rows < 0 || hq < 1 || hq % hkv || num_seqs < 1 || max_pages_per_seq < 1 ||
      block_table_stride < max_pages_per_seq)
    return fail(MRB_ERR_ARG, "%s: bad sizes", what);
  if (hq / hkv > KV4_MAX_GROUP) return fail(MRB_ERR_UNSUPPORTED, "%s: at most 16 query heads a KV head", what);
  // (the kernels round positions up to their steps of 128 tokens)
  if (max_pages_per_seq > (INT32_MAX - 128) / page_size || hkv > 65535 || tokens > INT32_MAX || rows > INT32_MAX)
    return fail(MRB_ERR_UNSUPPORTED, "%s: positions and rows must be numbered in 32 bits", what);
  if (!isfinite(scale)) return fail(MRB_ERR_ARG, "%s: scale must be finite", what);
  if (tokens == 0 || rows == 0) return MRB_OK;
  if (!q || !out || !block_table || !row_len) return fail(MRB_ERR_ARG, "%s: null pointer", what);
  if (!aligned(q, 16) || !aligned(out, 16)) return fail(MRB_ERR_ARG, "%s: q and out must be 16-byte aligned", what);
  return MRB_OK;
}

}  // namespace mrb
