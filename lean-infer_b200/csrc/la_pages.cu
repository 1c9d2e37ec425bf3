// Pages of the paged K/V cache copied and moved inside the pools of all layers.
//
//   la_copy_blocks:  pool[l, dst[i], :n_i] = pool[l, src[i], :n_i] for every layer l, in K and in V
//   la_move_blocks:  the same for whole pages, and every block-table entry src[i] becomes dst[i]
//
// Both run over data that stays in place (a fork's copy-on-write, a
// compaction), so they do no arithmetic and are bound by HBM: every byte is
// read once and written once.
//
// One launch: the first CTAs rewrite the table, the others copy.
//
// A pair may be copied in any order relative to the others, so a pair whose
// destination is another pair's source, or the destination of a pair before
// it, is skipped and reported (LA_DEVERR_BLOCK_PAIR): what the others do does
// not depend on timing.
#include <cuda_runtime.h>

#include <cstdint>

#include "la_internal.h"
#include "la_ptx.cuh"

namespace la {
namespace pages {

constexpr int kThreads = 256;
constexpr int kPer = 4;                       // 16-byte units of a chunk per thread, all in flight at once
constexpr int kChunk = kPer * kThreads;       // units that a CTA copies: 16 KB
constexpr int kTablePairs = 2048;             // pairs that a table CTA keeps in shared memory

struct Params {
  uint8_t* pool[2];
  long long layer_bytes, block_bytes, token_bytes, head_bytes;  // strides
  int layers, heads;
  int block_size;
  int row_units;    // 16-byte units of one token of one head
  int token_units;  // of one token
  int flat;         // a page is one run of bytes (kFlat)
  int chunks;       // of a whole page
  int parts;        // chunks of a pair in all tensors of all layers
  int per;          // of them, those that one CTA copies
  long long num_blocks;
  const int* src;
  const int* dst;
  const int* tokens;  // or null: whole pages
  int n;
  int* table;  // or null
  long long table_stride;
  int table_rows, table_cols;
  int table_ctas;  // the first ones of the grid
  int* err;
};

__device__ __forceinline__ void report(const Params& p, int code) {
  if (p.err) atomicCAS(p.err, 0, code);
}

__device__ __forceinline__ bool in_pool(const Params& p, int s, int d) {
  return s >= 0 && s < p.num_blocks && d >= 0 && d < p.num_blocks;
}

// One chunk of one pair in one tensor of one layer per CTA, the pairs in turn,
// so that what runs at a time is spread over all their pages; CTAs behind a
// partly filled page's tokens leave at once. The loads are issued before it is
// known whether the pair meets another, the stores wait for that. To see it the
// CTA reads all pairs, which is little beside its chunk up to some 1000 of them
// (8 KB); behind that it copies more chunks of its pair (per_cta). Measured
// (times of a copy at the rate of a plain tensor copy in brackets): 96 pages of
// 28 layers 832 us (873), 64 partly filled ones 304 us (309), 3 pages 28.8 us
// (27.3), one partly filled 9.5 us (8.2). 32 KB per CTA took up to 3 % longer,
// 8 KB up to 18 %, the pages one after another 4 % longer, without the streaming
// hints 9 % longer for the one page and 1.5 % less for the 64; a persistent
// grid with equal ranges 25 % longer.
template <bool kFlat>
__device__ __forceinline__ void copy_part(const Params& p, long long x) {
  const int i = static_cast<int>(x % p.n);
  const int part0 = static_cast<int>(x / p.n) * p.per;
  const int tid = threadIdx.x;
  const int s = p.src[i], d = p.dst[i], n = p.tokens ? p.tokens[i] : p.block_size;
  const bool first = part0 == 0 && tid == 0;
  if (s < 0 || s >= p.num_blocks || d < 0 || d >= p.num_blocks) {
    if (first) report(p, LA_DEVERR_BLOCK_ID);
    return;
  }
  if (n < 0 || n > p.block_size) {
    if (first) report(p, LA_DEVERR_SEQLEN);
    return;
  }
  const int units = n * p.token_units;
  if (s == d) return;
  bool judged = false;
  for (int part = part0; part < min(part0 + p.per, p.parts); ++part) {
    const int piece = part / p.chunks, chunk = part - piece * p.chunks;
    if (chunk * kChunk >= units) continue;
    uint8_t* base = p.pool[piece & 1] + (piece >> 1) * p.layer_bytes;
    const uint8_t* from = base + s * p.block_bytes;
    uint8_t* to = base + d * p.block_bytes;
    // byte offset in the page of this thread's e-th unit
    const int x0 = chunk * kChunk + tid;
    auto at_unit = [&](int e) -> long long {
      const int u = x0 + e * kThreads;
      if (kFlat) return static_cast<long long>(u) * 16;
      const int tok = u / p.token_units, r = u - tok * p.token_units;
      const int h = r / p.row_units;
      return tok * p.token_bytes + h * p.head_bytes + (r - h * p.row_units) * 16;
    };
    uint4 v[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (x0 + e * kThreads < units) v[e] = __ldcs(reinterpret_cast<const uint4*>(from + at_unit(e)));
    if (!judged) {
      bool meets = false;
      for (int j = tid; j < p.n; j += kThreads) meets |= j != i && (p.src[j] == d || (j < i && p.dst[j] == d));
      if (__syncthreads_or(meets)) {
        if (first) report(p, LA_DEVERR_BLOCK_PAIR);
        return;
      }
      judged = true;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (x0 + e * kThreads < units) __stcs(reinterpret_cast<uint4*>(to + at_unit(e)), v[e]);
  }
}

// Entries of the table, one per thread: the first sound pair that moves the
// page it names. The pairs are held in shared memory as far as they fit. A warp
// compares its entries with kLook pairs after another; a pair that some entry
// names is judged by all its lanes together. (Each lane by itself, one after
// another, 1201 pairs under 131 x 77 entries took 1.8 ms. One pair at a time, a
// table that names none of them took longer than the copies beside it, 187 us,
// since the copies' loads are in front of each look.)
constexpr int kLook = 8;
__device__ void table_part(const Params& p) {
  __shared__ int2 s_pair[kTablePairs];
  const int held = min(p.n, kTablePairs);
  for (int i = threadIdx.x; i < held; i += kThreads) s_pair[i] = make_int2(p.src[i], p.dst[i]);
  __syncthreads();
  const auto pair = [&](int i) { return i < held ? s_pair[i] : make_int2(p.src[i], p.dst[i]); };
  const int lane = threadIdx.x & 31;
  const long long x = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  const bool in = x < static_cast<long long>(p.table_rows) * p.table_cols;
  int* e = in ? p.table + (x / p.table_cols) * p.table_stride + x % p.table_cols : nullptr;
  int id = in ? *e : -1;  // below 0: no entry, one that names no page, or one that has been replaced
  for (int i0 = 0; i0 < p.n; i0 += kLook) {
    bool here = false;
    if (i0 + kLook <= held) {
#pragma unroll
      for (int u = 0; u < kLook; ++u) here |= s_pair[i0 + u].x == id;
    } else {
#pragma unroll
      for (int u = 0; u < kLook; ++u) here |= i0 + u < p.n && p.src[i0 + u] == id;
    }
    if (!__any_sync(0xffffffffu, here && id >= 0)) continue;
    for (int i = i0; i < min(i0 + kLook, p.n); ++i) {
      const int2 m = pair(i);
      const bool named = m.x == id && m.y != id && in_pool(p, m.x, m.y);
      if (!__any_sync(0xffffffffu, named)) continue;
      bool meets = false;
#pragma unroll 4
      for (int j = lane; j < p.n; j += 32) {
        const int2 o = pair(j);
        meets |= j != i && (o.x == m.y || (j < i && o.y == m.y));
      }
      if (__any_sync(0xffffffffu, meets) || !named) continue;
      *e = m.y;
      id = -1;
    }
    if (__all_sync(0xffffffffu, id < 0)) return;
  }
}

template <bool kFlat>
__global__ void __launch_bounds__(kThreads) pages_kernel(const Params p) {
  grid_dependency_wait();
  if (static_cast<int>(blockIdx.x) < p.table_ctas)
    table_part(p);
  else
    copy_part<kFlat>(p, static_cast<long long>(blockIdx.x) - p.table_ctas);
}

static int setup(Params* p, void* k_pool, void* v_pool, int64_t layer_stride, int64_t block_stride,
                 int64_t token_stride, int64_t head_stride, int num_layers, int64_t num_blocks, int block_size,
                 int num_kv_heads, int head_dim, int element_size, const int32_t* src, const int32_t* dst,
                 int num_pairs, int* dev_error) {
  if (num_pairs < 0 || num_layers < 0 || num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || head_dim <= 0)
    return LA_ERR_INVALID_ARGUMENT;
  if (element_size != 1 && element_size != 2 && element_size != 4) return LA_ERR_UNSUPPORTED;
  if (num_pairs > 0 && num_layers > 0 && (!k_pool || !v_pool || !src || !dst)) return LA_ERR_INVALID_ARGUMENT;
  if (layer_stride < 0 || block_stride <= 0 || token_stride <= 0 || head_stride <= 0) return LA_ERR_INVALID_ARGUMENT;
  const int64_t strides[] = {layer_stride, block_stride, token_stride, head_stride, head_dim};
  for (int64_t s : strides)
    if (s * element_size % 16) return LA_ERR_ALIGNMENT;
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(src, 4) || !aligned(dst, 4)) return LA_ERR_ALIGNMENT;
  if (num_blocks > 0x7fffffffLL || num_layers > 0x3fff) return LA_ERR_UNSUPPORTED;
  p->pool[0] = static_cast<uint8_t*>(k_pool);
  p->pool[1] = static_cast<uint8_t*>(v_pool);
  p->layer_bytes = layer_stride * element_size;
  p->block_bytes = block_stride * element_size;
  p->token_bytes = token_stride * element_size;
  p->head_bytes = head_stride * element_size;
  p->layers = num_layers;
  p->heads = num_kv_heads;
  p->block_size = block_size;
  p->row_units = head_dim * element_size / 16;
  p->token_units = num_kv_heads * p->row_units;
  if (static_cast<int64_t>(block_size) * num_kv_heads * p->row_units > 0x7fff0000LL) return LA_ERR_UNSUPPORTED;
  const int64_t row = static_cast<int64_t>(head_dim) * element_size;
  p->flat = (num_kv_heads == 1 || p->head_bytes == row) && (block_size == 1 || p->token_bytes == num_kv_heads * row);
  p->num_blocks = num_blocks;
  p->src = src;
  p->dst = dst;
  p->n = num_pairs;
  p->err = dev_error;
  return LA_OK;
}

// Chunks of a pair that a CTA copies: for each 16 KB that it copies it reads at
// most 16 KB of pairs, as long as the pair has chunks enough. (With one chunk
// each, 16000 pages of 16 tokens in 7 layers took 9970 us, 2508 so; their bytes
// take 2274 at the rate of a plain tensor copy.)
static int per_cta(int pairs, int parts) { return pairs < 2048 ? 1 : pairs / 1024 < parts ? pairs / 1024 : parts; }

static int launch(Params& p, cudaStream_t stream) {
  if (p.n == 0) return LA_OK;
  const int64_t entries = static_cast<int64_t>(p.table_rows) * p.table_cols;
  const int64_t table = (entries + kThreads - 1) / kThreads;
  p.chunks = (p.block_size * p.token_units + kChunk - 1) / kChunk;
  const int64_t parts = 2 * static_cast<int64_t>(p.layers) * p.chunks;
  if (parts > 0x7fffffffLL) return LA_ERR_UNSUPPORTED;
  p.parts = static_cast<int>(parts);
  p.per = per_cta(p.n, p.parts);
  const int64_t ctas = table + (parts > 0 ? p.n * ((parts + p.per - 1) / p.per) : 0);
  if (ctas == 0) return LA_OK;
  if (ctas > 0x7fffffffLL) return LA_ERR_UNSUPPORTED;
  p.table_ctas = static_cast<int>(table);
  return cuda_status(launch_pdl(p.flat ? pages_kernel<true> : pages_kernel<false>, dim3(static_cast<unsigned>(ctas)),
                                dim3(kThreads), 0, stream, p));
}

}  // namespace pages
}  // namespace la

extern "C" int la_copy_blocks(void* k_pool, void* v_pool, int64_t layer_stride, int64_t block_stride,
                              int64_t token_stride, int64_t head_stride, int num_layers, int64_t num_blocks,
                              int block_size, int num_kv_heads, int head_dim, int element_size,
                              const int32_t* src_blocks, const int32_t* dst_blocks, const int32_t* num_tokens,
                              int num_pairs, int* dev_error, cudaStream_t stream) {
  la::pages::Params p = {};
  const int st = la::pages::setup(&p, k_pool, v_pool, layer_stride, block_stride, token_stride, head_stride,
                                  num_layers, num_blocks, block_size, num_kv_heads, head_dim, element_size,
                                  src_blocks, dst_blocks, num_pairs, dev_error);
  if (st != LA_OK) return st;
  if (!la::aligned(num_tokens, 4)) return LA_ERR_ALIGNMENT;
  p.tokens = num_tokens;
  return la::pages::launch(p, stream);
}

extern "C" int la_move_blocks(void* k_pool, void* v_pool, int64_t layer_stride, int64_t block_stride,
                              int64_t token_stride, int64_t head_stride, int num_layers, int64_t num_blocks,
                              int block_size, int num_kv_heads, int head_dim, int element_size,
                              const int32_t* src_blocks, const int32_t* dst_blocks, int num_pairs,
                              int32_t* block_table, int64_t bt_seq_stride, int batch, int max_blocks_per_seq,
                              int* dev_error, cudaStream_t stream) {
  la::pages::Params p = {};
  const int st = la::pages::setup(&p, k_pool, v_pool, layer_stride, block_stride, token_stride, head_stride,
                                  num_layers, num_blocks, block_size, num_kv_heads, head_dim, element_size,
                                  src_blocks, dst_blocks, num_pairs, dev_error);
  if (st != LA_OK) return st;
  if (batch < 0 || max_blocks_per_seq < 0 || bt_seq_stride < max_blocks_per_seq) return LA_ERR_INVALID_ARGUMENT;
  const int64_t entries = static_cast<int64_t>(batch) * max_blocks_per_seq;
  if (entries > 0 && !block_table) return LA_ERR_INVALID_ARGUMENT;
  if (!la::aligned(block_table, 4)) return LA_ERR_ALIGNMENT;
  p.table = block_table;
  p.table_stride = bt_seq_stride;
  p.table_rows = batch;
  p.table_cols = max_blocks_per_seq;
  return la::pages::launch(p, stream);
}
