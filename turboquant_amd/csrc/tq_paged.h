// tq_paged.h -- what the entries over a paged cache share: the checks of their
// arguments, and the store of large outputs.
#pragma once

#include "tq_common.h"

#include <initializer_list>

namespace tqh {

// log2(page_size), or -1 for a size that pages do not have.  Sixteen tokens
// at least, so that a 16-token tile never crosses pages.
inline int page_shift(int page_size) {
  for (int s = 4; s <= 10; s++)
    if (page_size == 1 << s) return s;
  return -1;
}

// Checks a paged cache's shape; fills shift and the codec of its records.
inline int check_pages(long long num_pages, int num_kv_heads, int page_size, int head_dim, int bits,
                       size_t outlier_blocks, int norm_mode, int &shift, PolarCodec &codec) {
  shift = page_shift(page_size);
  if (shift < 0) return fail(TQ_ERR_INVALID_ARGUMENT, "page_size %d is no power of two from 16 to 1024", page_size);
  if (head_dim <= 0 || head_dim % 32 != 0)
    return fail(TQ_ERR_INVALID_ARGUMENT, "head_dim (%d) must be divisible by QUANT_BLOCK_SIZE (32)", head_dim);
  if (num_kv_heads <= 0 || num_kv_heads > 65535)
    return fail(TQ_ERR_INVALID_ARGUMENT, "num_kv_heads %d outside 1 to 65,535", num_kv_heads);
  if (num_pages < 0 || num_pages >= 1ll << 31)
    return fail(TQ_ERR_INVALID_ARGUMENT, "num_pages %lld outside 0 to 2^31 - 1", num_pages);
  const int rc = polar_codec(bits, norm_mode, outlier_blocks, head_dim / 32, codec);
  if (rc) return rc;
  if (codec.mixed)
    return fail(TQ_ERR_INVALID_ARGUMENT, "paged records take outlier_blocks 0 or all");
  return TQ_OK;
}

// Refuses a pool that does not start on a 16-byte boundary (null: there is none).
inline int check_pools(std::initializer_list<const void *> pools) {
  for (const void *p : pools)
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0)
      return fail(TQ_ERR_INVALID_ARGUMENT, "code, scale and sign pools start on 16-byte boundaries");
  return TQ_OK;
}

// Whether rows of `stride` elements of `size` bytes from p start on 16-byte boundaries.
inline bool rows_aligned(const void *p, long long stride, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}

// A 16-byte store; `through`: with no wish to find it in a cache again.  Output
// of more than kThroughBytes, the size of the dies' L2s, is not there when it is
// read, and its lines push out what the kernel still reads (8,192 tokens' heads
// normed and rotated in 38.6 us, through 36.4; 64,000 tokens' records loaded in
// 74, through 53).
constexpr long long kThroughBytes = 32ll << 20;
typedef uint32_t words4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void store16(void *p, words4 v, int through) {
  if (through) {
    asm volatile("");  // one on each side keeps the two stores apart: merged, they are the plain one
    __builtin_nontemporal_store(v, static_cast<words4 *>(p));
    asm volatile("");
  } else {
    *static_cast<words4 *>(p) = v;
  }
}

inline int dtype_size(int dt) { return dt == TQ_DTYPE_F32 ? 4 : 2; }

}  // namespace tqh
