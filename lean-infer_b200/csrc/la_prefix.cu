// Paged GQA decode attention for a batch whose rows share long prefixes.
//
// out[b, h] = softmax(scale * q[b, h] . K_b^T) V_b over keys 0..cache_seqlens[b]-1
// of row b, read through block_table[b]: what la_paged_decode computes. Rows
// cu_prefix_rows[g] .. cu_prefix_rows[g+1]-1 hold the same pages for their
// first prefix_lens[b] keys.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "la_internal.h"
#include "la_ptx.cuh"

namespace la {
namespace prefix {

constexpr int kD = 128;

struct Params {
  const __nv_bfloat16* q;
  long long q_bs, q_hs;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  long long kv_block, kv_token, kv_head;
  long long num_blocks;
  int block_size;
  const int* table;
  long long table_stride;
  int max_blocks;
  const int* lens;
  const int* cu;
  int groups, batch;
  int hq, group;
  float scale_log2;
  __nv_bfloat16* out;
  long long out_bs, out_hs;
  float* lse;
  int* err;
};

// One warp per (row, query head), four dims per lane, keys one after another.
__global__ void __launch_bounds__(32) row_kernel(const Params p) {
  grid_dependency_wait();
  const int b = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const float ninf = -__int_as_float(0x7f800000);
  if (b == 0 && h == 0)
    for (int g = lane; p.groups > 0 && g <= p.groups; g += 32)
      if ((p.cu[g] < (g ? p.cu[g - 1] : 0) || p.cu[g] > p.batch) && p.err) atomicCAS(p.err, 0, LA_DEVERR_PREFIX);
  int ctx = p.lens[b];
  if (ctx > static_cast<long long>(p.max_blocks) * p.block_size) {
    if (p.err) atomicCAS(p.err, 0, LA_DEVERR_SEQLEN);
    ctx = p.max_blocks * p.block_size;
  }
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = ninf, l = 0.f;
  for (int e = 0; e < 4; ++e) q[e] = __bfloat162float(p.q[b * p.q_bs + h * p.q_hs + lane * 4 + e]) * p.scale_log2;
  for (int t = 0; t < ctx; ++t) {
    const int id = p.table[b * p.table_stride + t / p.block_size];
    float kx[4] = {0.f, 0.f, 0.f, 0.f}, vx[4] = {0.f, 0.f, 0.f, 0.f};
    if (id >= 0 && id < p.num_blocks) {
      const long long at = id * p.kv_block + (t % p.block_size) * p.kv_token + (h / p.group) * p.kv_head + lane * 4;
      for (int e = 0; e < 4; ++e) {
        kx[e] = __bfloat162float(p.k[at + e]);
        vx[e] = __bfloat162float(p.v[at + e]);
      }
    } else if (p.err) {
      atomicCAS(p.err, 0, LA_DEVERR_BLOCK_ID);
    }
    float s = q[0] * kx[0] + q[1] * kx[1] + q[2] * kx[2] + q[3] * kx[3];
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s), a = ex2(m - mn), w = ex2(s - mn);
    for (int e = 0; e < 4; ++e) o[e] = o[e] * a + w * vx[e];
    l = l * a + w;
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int e = 0; e < 4; ++e)
    p.out[b * p.out_bs + h * p.out_hs + lane * 4 + e] = __float2bfloat16_rn(o[e] * inv);
  if (p.lse && lane == 0)
    p.lse[static_cast<long long>(b) * p.hq + h] = l == 0.f ? ninf : (m + __log2f(l)) * 0.6931471805599453f;
}

}  // namespace prefix
}  // namespace la

extern "C" int la_paged_decode_shared_prefix_workspace_size(int device, int batch, int num_groups, int num_q_heads,
                                                            int num_kv_heads, int head_dim, size_t* bytes) {
  if (!bytes || batch < 0 || num_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim != 128 ||
      num_kv_heads > 8 || 8 % num_kv_heads != 0 || num_q_heads % num_kv_heads != 0)
    return head_dim != 128 ? LA_ERR_UNSUPPORTED : LA_ERR_INVALID_ARGUMENT;
  if (la::num_sms(device) <= 0) return LA_ERR_CUDA;
  *bytes = 256;
  return LA_OK;
}

extern "C" int la_paged_decode_shared_prefix(
    const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache, const void* v_cache,
    int64_t kv_block_stride, int64_t kv_token_stride, int64_t kv_head_stride, int64_t num_blocks, int block_size,
    const int32_t* block_table, int64_t bt_seq_stride, int max_blocks_per_seq, const int32_t* cache_seqlens,
    const int32_t* prefix_lens, const int32_t* cu_prefix_rows, int num_groups, int batch, int num_q_heads,
    int num_kv_heads, int head_dim, float softmax_scale, void* out, int64_t out_batch_stride, int64_t out_head_stride,
    float* softmax_lse, void* workspace, size_t workspace_bytes, int* dev_error, cudaStream_t stream) {
  using namespace la;
  if (!q || !k_cache || !v_cache || !block_table || !cache_seqlens || !out ||
      (num_groups > 0 && (!prefix_lens || !cu_prefix_rows)))
    return LA_ERR_INVALID_ARGUMENT;
  if (batch < 0 || num_groups < 0 || num_blocks <= 0 || block_size <= 0 || max_blocks_per_seq <= 0)
    return LA_ERR_INVALID_ARGUMENT;
  if (batch == 0) return LA_OK;
  if (head_dim != prefix::kD) return LA_ERR_UNSUPPORTED;
  if (num_kv_heads <= 0 || num_kv_heads > 8 || 8 % num_kv_heads != 0) return LA_ERR_UNSUPPORTED;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads != 0) return LA_ERR_INVALID_ARGUMENT;
  if (num_q_heads / num_kv_heads > 8) return LA_ERR_UNSUPPORTED;
  if (block_size % 16 != 0) return LA_ERR_UNSUPPORTED;
  if (!(softmax_scale > 0.f)) return LA_ERR_INVALID_ARGUMENT;
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16)) return LA_ERR_ALIGNMENT;
  if (q_batch_stride % 8 || q_head_stride % 8 || kv_block_stride % 8 || kv_token_stride % 8 || kv_head_stride % 8)
    return LA_ERR_ALIGNMENT;
  if (q_batch_stride <= 0 || q_head_stride <= 0 || kv_block_stride <= 0 || kv_token_stride <= 0 ||
      kv_head_stride <= 0 || out_batch_stride <= 0 || out_head_stride <= 0)
    return LA_ERR_INVALID_ARGUMENT;
  if (!aligned(out, 8) || out_batch_stride % 4 || out_head_stride % 4) return LA_ERR_ALIGNMENT;
  const int device = current_device();
  if (device < 0) return LA_ERR_CUDA;
  size_t need = 0;
  const int st = la_paged_decode_shared_prefix_workspace_size(device, batch, num_groups, num_q_heads, num_kv_heads,
                                                              head_dim, &need);
  if (st != LA_OK) return st;
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256)) return LA_ERR_WORKSPACE;
  prefix::Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_bs = q_batch_stride;
  p.q_hs = q_head_stride;
  p.k = static_cast<const __nv_bfloat16*>(k_cache);
  p.v = static_cast<const __nv_bfloat16*>(v_cache);
  p.kv_block = kv_block_stride;
  p.kv_token = kv_token_stride;
  p.kv_head = kv_head_stride;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.table = block_table;
  p.table_stride = bt_seq_stride;
  p.max_blocks = max_blocks_per_seq;
  p.lens = cache_seqlens;
  p.cu = cu_prefix_rows;
  p.groups = num_groups;
  p.batch = batch;
  p.hq = num_q_heads;
  p.group = num_q_heads / num_kv_heads;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_bs = out_batch_stride;
  p.out_hs = out_head_stride;
  p.lse = softmax_lse;
  p.err = dev_error;
  return cuda_status(launch_pdl(prefix::row_kernel, dim3(batch, num_q_heads), dim3(32), 0, stream, p));
}
