// Pages of the paged K/V cache copied and moved inside the pools of all layers.
//
//   la_copy_blocks:  pool[l, dst[i], :n_i] = pool[l, src[i], :n_i] for every layer l, in K and in V
//   la_move_blocks:  the same for whole pages, and every block-table entry src[i] becomes dst[i]
//
// Both run over data that stays in place (a fork's copy-on-write, a
// compaction), so they do no arithmetic and are bound by HBM: every byte is
// read once and written once.
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

struct Params {
  uint8_t* pool[2];
  long long layer_bytes, block_bytes, token_bytes, head_bytes;  // strides
  int layers, heads;
  int block_size;
  int row_units;  // 16-byte units of one token of one head
  long long num_blocks;
  const int* src;
  const int* dst;
  const int* tokens;  // or null: whole pages
  int n;
  int* table;  // or null
  long long table_stride;
  int table_rows, table_cols;
  int* err;
};

__device__ __forceinline__ void report(const Params& p, int code) {
  if (p.err) atomicCAS(p.err, 0, code);
}

// Whether pair i names pages of the pool and meets no other pair (block-collective).
__device__ bool pair_ok(const Params& p, int i) {
  const int s = p.src[i], d = p.dst[i];
  if (s < 0 || s >= p.num_blocks || d < 0 || d >= p.num_blocks) {
    if (threadIdx.x == 0) report(p, LA_DEVERR_BLOCK_ID);
    return false;
  }
  if (s == d) return false;  // already there
  bool meets = false;
  for (int j = threadIdx.x; j < p.n; j += blockDim.x) meets |= j != i && (p.src[j] == d || (j < i && p.dst[j] == d));
  if (__syncthreads_or(meets)) {
    if (threadIdx.x == 0) report(p, LA_DEVERR_BLOCK_PAIR);
    return false;
  }
  return true;
}

// One pair, tensor and layer per CTA.
__global__ void __launch_bounds__(kThreads) copy_kernel(const Params p) {
  grid_dependency_wait();
  const int i = blockIdx.x, t = blockIdx.y & 1, l = blockIdx.y >> 1;
  if (!pair_ok(p, i)) return;
  int n = p.tokens ? p.tokens[i] : p.block_size;
  if (n < 0 || n > p.block_size) {
    if (threadIdx.x == 0) report(p, LA_DEVERR_SEQLEN);
    return;
  }
  const uint8_t* s = p.pool[t] + l * p.layer_bytes + p.src[i] * p.block_bytes;
  uint8_t* d = p.pool[t] + l * p.layer_bytes + p.dst[i] * p.block_bytes;
  const int per_token = p.heads * p.row_units;
  for (int x = threadIdx.x; x < n * per_token; x += kThreads) {
    const int tok = x / per_token, r = x - tok * per_token;
    const int h = r / p.row_units, u = r - h * p.row_units;
    const long long at = tok * p.token_bytes + h * p.head_bytes + u * 16;
    *reinterpret_cast<uint4*>(d + at) = *reinterpret_cast<const uint4*>(s + at);
  }
}

// One table entry per thread: the first sound pair that moves its page.
__global__ void __launch_bounds__(kThreads) table_kernel(const Params p) {
  grid_dependency_wait();
  const long long x = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  if (x >= static_cast<long long>(p.table_rows) * p.table_cols) return;
  int* e = p.table + (x / p.table_cols) * p.table_stride + x % p.table_cols;
  const int id = *e;
  for (int i = 0; i < p.n; ++i) {
    const int d = p.dst[i];
    if (p.src[i] != id || d == id || d < 0 || d >= p.num_blocks) continue;
    bool meets = false;
    for (int j = 0; j < p.n; ++j) meets |= j != i && (p.src[j] == d || (j < i && p.dst[j] == d));
    if (meets) continue;
    *e = d;
    return;
  }
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
  if (static_cast<int64_t>(block_size) * num_kv_heads * p->row_units > 0x7fffffffLL) return LA_ERR_UNSUPPORTED;
  p->num_blocks = num_blocks;
  p->src = src;
  p->dst = dst;
  p->n = num_pairs;
  p->err = dev_error;
  return LA_OK;
}

static int launch_copy(const Params& p, cudaStream_t stream) {
  if (p.n == 0 || p.layers == 0) return LA_OK;
  return cuda_status(launch_pdl(copy_kernel, dim3(p.n, 2 * p.layers), dim3(kThreads), 0, stream, p));
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
  return la::pages::launch_copy(p, stream);
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
  const int c = la::pages::launch_copy(p, stream);
  if (c != LA_OK || entries == 0 || num_pairs == 0) return c;
  const int64_t ctas = (entries + la::pages::kThreads - 1) / la::pages::kThreads;
  if (ctas > 0x7fffffffLL) return LA_ERR_UNSUPPORTED;
  return la::cuda_status(la::launch_pdl(la::pages::table_kernel, dim3(static_cast<unsigned>(ctas)),
                                        dim3(la::pages::kThreads), 0, stream, p));
}
