// kv4.cuh — addresses inside the paged 4-bit K/V cache (layout in include/moestream_cuda.h).
#pragma once
#include <stdint.h>

#include "../../include/moestream_cuda.h"

namespace ms {

// byte offsets in a block of 16 tokens of one head: K codes (8 hd), K scales (2 hd), V codes (8 hd), V scales (2 hd)
__host__ __device__ constexpr int kv4_block_bytes(int hd) { return 20 * hd; }
__host__ __device__ constexpr int kv4_k_scales(int hd) { return 8 * hd; }
__host__ __device__ constexpr int kv4_v_codes(int hd) { return 10 * hd; }
__host__ __device__ constexpr int kv4_v_scales(int hd) { return 18 * hd; }

// where chunk C (16 dims) of token pair p stands: the permutation puts the 16-byte units that the 8 lanes of
// one shared-memory phase read (2 chunks x 4 pairs) into different banks
template <int HD>
__device__ __forceinline__ int kv4_v_chunk(int C, int pair) {
  return HD == 64 ? C ^ (pair & 2) : C ^ ((pair & 3) << 1);
}

// the block of token pos of a sequence, counted in blocks from the start of the pages, or -1 where position or page
// number are outside their tables
__device__ __forceinline__ int64_t kv4_block(const ms_kv4_cache& c, int seq, int pos, int head) {
  if (pos < 0) return -1;
  const int j = pos / c.page_tokens;
  if (j >= c.max_pages) return -1;
  const int page = c.block_table[(int64_t)seq * c.max_pages + j];
  if (page < 0 || page >= c.n_pages) return -1;
  return ((int64_t)page * c.kv_heads + head) * (c.page_tokens / 16) + (pos % c.page_tokens) / 16;
}

}  // namespace ms
