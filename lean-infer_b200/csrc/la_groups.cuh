// Groups of consecutive batch rows that share the pages of a prefix, as every
// kernel of la_paged_decode_shared_prefix reads them from device memory.
#pragma once
#include <cstdint>

#include "la_internal.h"

namespace la {

struct PrefixGroups {
  const int* cu;    // [n + 1] first row of each group, or null: no groups
  const int* lens;  // [n] keys of each group's prefix
  int n;
  int batch;
  int block_size;
  int bs_shift;   // log2(block_size) when it is a power of two, else -1
  long long cap;  // keys that a block table has room for
};

// Group g: its first row, its rows, and the keys taken as shared, whole pages
// of them. A group of one row shares nothing (the row-by-row pass reads its
// keys just as well), and one that is no run of the batch's rows is empty.
struct PrefixGroup {
  int first, rows, keys;
};

__device__ __forceinline__ PrefixGroup prefix_group(const PrefixGroups& G, int g) {
  PrefixGroup r;
  r.first = G.cu[g];
  const int last = G.cu[g + 1];
  const long long n = min(static_cast<long long>(max(G.lens[g], 0)), G.cap);
  const bool sound = r.first >= 0 && r.first <= last && last <= G.batch;
  r.rows = sound ? last - r.first : 0;
  const int blocks = G.bs_shift >= 0 ? static_cast<int>(n) >> G.bs_shift : static_cast<int>(n) / G.block_size;
  r.keys = r.rows >= 2 ? blocks * G.block_size : 0;
  return r;
}

// The last group that begins at or before row b, or -1.
__device__ __forceinline__ int prefix_group_of(const PrefixGroups& G, int b) {
  int lo = -1, hi = G.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (G.cu[mid] <= b)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Keys of row b that its group's pass covers; the row reads those behind them
// by itself. None where the row ends before they do: every row of a group
// that takes part sees all the shared keys, so no key is masked for one row
// and seen by another (a masked NaN would reach the first through 0 * NaN).
__device__ __forceinline__ int prefix_keys(const PrefixGroups& G, int b, int ctx) {
  const int g = prefix_group_of(G, b);
  if (g < 0) return 0;
  const PrefixGroup r = prefix_group(G, g);
  return b < r.first + r.rows && ctx >= r.keys ? r.keys : 0;
}

// The pass over the keys that each row reads by itself (la_decode.cu): the
// arguments of la_paged_decode, checked the same way, and where its partials
// go: slot (row + CTA) of part_o [batch + #SMs][Hq][D] and part_lse
// [batch + #SMs][Hq] (base-2 logarithm), fp32, O normalised. Row b's parts
// are those of CTAs cf..cl, from its units of `16 * 8 / Hkv` keys and the even
// split of all rows' units. Rows without a prefix that lie within one CTA are
// written to out and softmax_lse.
struct OwnKeysPass {
  PrefixGroups groups;
  float* part_o;
  float* part_lse;
};

int decode_own_keys(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache,
                    const void* v_cache, int64_t kv_block_stride, int64_t kv_token_stride, int64_t kv_head_stride,
                    int64_t num_blocks, int block_size, const int32_t* block_table, int64_t bt_seq_stride,
                    int max_blocks_per_seq, const int32_t* cache_seqlens, int batch, int num_q_heads,
                    int num_kv_heads, int head_dim, float softmax_scale, void* out, int64_t out_batch_stride,
                    int64_t out_head_stride, float* softmax_lse, int* dev_error, cudaStream_t stream,
                    const OwnKeysPass& own);

}  // namespace la
