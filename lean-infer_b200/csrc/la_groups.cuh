// Groups of consecutive batch rows that share the pages of a prefix, as
// la_paged_decode_shared_prefix reads them from device memory.
#pragma once
#include <cstdint>

#include "la_internal.h"

namespace la {

struct PrefixGroups {
  const int* cu;    // [n + 1] first row of each group
  const int* lens;  // [n] keys of each group's prefix
  int n;
  int batch;
  int block_size;
  int bs_shift;   // log2(block_size) when it is a power of two, else -1
  long long cap;  // keys that a block table has room for
};

// Group g: its first row, its rows, and the keys taken as shared, whole pages
// of them. A group of one row shares nothing (the row reads its keys by itself
// just as well), and one that is no run of the batch's rows is empty.
struct PrefixGroup {
  int first, rows, keys;
};

// Bounds that run backwards can make groups overlap that are runs of rows each
// for itself, and no two warps need agree on whose a row is then. So where one
// group is no run of the batch's rows, all are empty, and every row reads its
// keys by itself.
__device__ __forceinline__ bool run_of_rows(const PrefixGroups& G, int first, int last) {
  return first >= 0 && first <= last && last <= G.batch;
}

__device__ __forceinline__ PrefixGroup group_from(const PrefixGroups& G, int first, int last, int len) {
  PrefixGroup r;
  r.first = first;
  const long long n = min(static_cast<long long>(max(len, 0)), G.cap);
  r.rows = run_of_rows(G, first, last) ? last - r.first : 0;
  const int blocks = G.bs_shift >= 0 ? static_cast<int>(n) >> G.bs_shift : static_cast<int>(n) / G.block_size;
  r.keys = r.rows >= 2 ? blocks * G.block_size : 0;
  return r;
}
// Through L2 only: it may be read before the kernel in front is done, and no
// stale line may stay in L1.
__device__ __forceinline__ PrefixGroup load_group(const PrefixGroups& G, int g) {
  return group_from(G, __ldcg(G.cu + g), __ldcg(G.cu + g + 1), __ldcg(G.lens + g));
}

// The CTA's table: up to kMaxGroups groups. Of more, which are read where they
// are needed, its first entry says whether all are runs of rows (rows: 1 or 0).
constexpr int kMaxGroups = 512;
__device__ __forceinline__ PrefixGroup prefix_group(const PrefixGroups& G, const PrefixGroup* tab, int g) {
  if (G.n <= kMaxGroups) return tab[g];
  PrefixGroup r = load_group(G, g);
  if (tab->rows == 0) r.rows = r.keys = 0;
  return r;
}

// Keys of row b that its group's pass covers; the row reads those behind them
// by itself. None where the row ends before they do: every row of a group
// that takes part sees all the shared keys, so no key is masked for one row
// and seen by another (a masked NaN would reach the first through 0 * NaN).
__device__ __forceinline__ int prefix_keys(const PrefixGroups& G, const PrefixGroup* tab, int b, int ctx) {
  int lo = -1, hi = G.n;  // the last group that begins at or before row b
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((G.n <= kMaxGroups ? tab[mid].first : G.cu[mid]) <= b)
      lo = mid;
    else
      hi = mid;
  }
  if (lo < 0) return 0;
  const PrefixGroup r = prefix_group(G, tab, lo);
  return b < r.first + r.rows && ctx >= r.keys ? r.keys : 0;
}

}  // namespace la
