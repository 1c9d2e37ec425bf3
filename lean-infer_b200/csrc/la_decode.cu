// (b) Paged GQA decode attention for sm_100a: a persistent, warp-specialised
// split-KV kernel plus a combine kernel.
//
// Semantics (leaninfer/qwen3/model.py:60-67 -> flash_attn_with_kvcache with a
// block table, one query token, causal bottom-right alignment, which at
// q_len = 1 means "all keys 0..cache_seqlens[b]-1"):
//   out[b, h] = softmax(scale * q[b, h] . K[b, :, h / G]^T) . V[b, :, h / G]
// where K[b, t] = k_cache[block_table[b, t / BS], t % BS].
//
// Work decomposition. The key range of every sequence is cut into units of
// TC = 16 * (8 / Hkv) tokens; a unit is one pipeline stage: 128 (token, kv
// head) rows of K and of V, 32 KB each. The units of all sequences, laid end
// to end, are split into gridDim.x equal contiguous ranges, one per CTA
// (grid = #SMs, one CTA per SM), so every SM streams the same number of bytes
// whatever the length mix. The partition is recomputed on the device from
// cache_seqlens, so the launch shape never depends on device data and the
// call can be captured in a CUDA graph. A CTA range covers whole sequences
// (written straight to `out`) and at most two partial sequences at its ends
// (written as fp32 (O, lse) partials to the workspace and merged by the
// combine kernel).
//
// CTA: warps 8 and 9 are the producers (partition walk, block-table lookups,
// TMA issue), taking even and odd units in turn; warps 0-7 consume. Consumer warp w handles kv head w % Hkv and the
// 16-token sub-chunk w / Hkv of each stage: S^T = K Q^T and O^T += V^T P^T on
// mma.m16n8k16 (bf16 in, fp32 accumulate) with K/V fragments read by ldmatrix
// from 128-byte-swizzled TMA tiles, online softmax in fp32 with warp-shuffle
// max reductions, P transposed into the B operand with movmatrix.
#include <utility>

#include "la_decode_body.cuh"

namespace la {
namespace decode {

// Total units over all sequences, computed by one warp.
__device__ long long total_units(const Params& p, int lane) {
  long long tot = 0;
  for (int base = 0; base < p.batch; base += 32) {
    const int b = base + lane;
    int n = (b < p.batch) ? units_of(seq_ctx(p, b), p.tc) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    tot += n;
  }
  return tot;
}

// The split for up to 32 x kChunks sequences from their lengths held in
// registers, lane l holding the kChunks consecutive sequences l * kChunks + i:
// total units T, this CTA's range [u0, u1), the sequence b0 it starts in and
// that sequence's first unit pb0. Each lane sums its own sequences, one warp
// scan orders the lanes, and the lane whose sequences hold unit u0 walks its
// registers (a scan per 32 sequences, one after another, took 18k clocks at
// 1024 sequences before the first copy could be issued).
template <int kChunks>
__device__ __forceinline__ void split_from_regs(const Params& p, int lane, const int (&un)[kChunks], long long& T,
                                                long long& u0, long long& u1, int& b0, long long& pb0) {
  long long own = 0;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) own += un[i];
  long long incl = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  const long long excl = incl - own;
  T = __shfl_sync(0xffffffffu, incl, 31);
  const long long G = gridDim.x;
  u0 = cta_start(blockIdx.x, T, G);
  u1 = cta_start(blockIdx.x + 1, T, G);
  b0 = p.batch;
  pb0 = T;
  if (u1 <= u0) return;
  const unsigned hit = __ballot_sync(0xffffffffu, excl <= u0 && u0 < incl);
  const int src = __ffs(hit) - 1;  // u0 < T, so exactly one lane holds it
  int bl = 0;
  long long pbl = 0;
  if (lane == src) {
    long long acc = excl;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      if (!found && u0 < acc + un[i]) {
        found = true;
        bl = lane * kChunks + i;
        pbl = acc;
      }
      acc += un[i];
    }
  }
  b0 = __shfl_sync(0xffffffffu, bl, src);
  pb0 = __shfl_sync(0xffffffffu, pbl, src);
}

// The lengths of sequences lane * kChunks + i (0 past the batch), read
// through L2 only; 16-byte loads where the run is aligned and inside the
// batch.
template <int kChunks>
__device__ __forceinline__ void load_lens(const Params& p, int lane, int (&raw)[kChunks]) {
  static_assert(kChunks % 4 == 0, "lengths are loaded four at a time");
  const int b0 = lane * kChunks;
  const bool vec = (reinterpret_cast<uintptr_t>(p.seqlens) & 15) == 0;
#pragma unroll
  for (int v = 0; v < kChunks / 4; ++v) {
    const int b = b0 + 4 * v;
    if (vec && b + 3 < p.batch) {
      const int4 x = __ldcg(reinterpret_cast<const int4*>(p.seqlens + b));
      raw[4 * v] = x.x;
      raw[4 * v + 1] = x.y;
      raw[4 * v + 2] = x.z;
      raw[4 * v + 3] = x.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[4 * v + e] = (b + e < p.batch) ? __ldcg(p.seqlens + b + e) : 0;
    }
  }
}

// kChunks: the split is held in registers for up to 32 x kChunks sequences
// (8 for the engine's batches, 32 for the many short rows of the KV-head-
// sharded partition).
template <int kStages, int kChunks>
__global__ void __launch_bounds__(kThreads, 1)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_k1,
                        const __grid_constant__ CUtensorMap tm_v1, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ctrl = smem + kStages * p.stage_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(ctrl);
  uint64_t* empty = full + kMaxStages;
  StageDesc* descs = reinterpret_cast<StageDesc*>(ctrl + 128);
  uint8_t* zero_row = ctrl + 256;
  long long* sched = reinterpret_cast<long long*>(ctrl + 384);
  uint64_t* mg_full = reinterpret_cast<uint64_t*>(ctrl + 448);   // all consumer warps wrote their state
  uint64_t* mg_empty = reinterpret_cast<uint64_t*>(ctrl + 456);  // the j = 0 warps read it
  float* merge = reinterpret_cast<float*>(ctrl + 1024);          // [8 warps][TQ][8][36] fp32 (nsub > 1)

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kCWarps);
    }
    mbar_init(mg_full, kCWarps);
    mbar_init(mg_empty, p.hkv);
    fence_barrier_init();
  }
  if (threadIdx.x < 32) reinterpret_cast<uint32_t*>(zero_row)[threadIdx.x] = 0u;
  if (warp == kCWarps && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // The split is computed speculatively before the dependency wait from the
  // lengths as they are now (read through L2 only, so no stale line stays in
  // L1), then the lengths are read again after the wait: if any changed (the
  // previous kernel wrote them) the split is recomputed from the final ones.
  const bool spec = p.batch <= 32 * kChunks;
  int raw[kChunks];
  long long sT = 0, su0 = 0, su1 = 0, spb0 = 0;
  int sb0 = 0;
  if (warp >= kCWarps && spec) {
    int un[kChunks];
    const long long cap = static_cast<long long>(p.max_blocks) * p.block_size;
    load_lens(p, lane, raw);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const long long c = raw[i] < 0 ? 0 : (raw[i] > cap ? cap : raw[i]);
      un[i] = units_of(static_cast<int>(c), p.tc);
    }
    split_from_regs(p, lane, un, sT, su0, su1, sb0, spb0);
  }
  // Everything below may read data written by the previous kernel in the stream.
  grid_dependency_wait();

  // The windows of the first sequence are loaded with the speculative split,
  // together with the re-read that checks it.
  Windows<false> w;
  if (warp >= kCWarps) {
    if (spec && su1 > su0) {
      w.load_swin(p, lane, sb0);
      w.load_bwin(p, lane, sb0, static_cast<int>((su0 - spb0) * p.tc / p.block_size));
    }
    bool same = spec;
    if (spec) {
      int now[kChunks];
      load_lens(p, lane, now);
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
        if (now[i] != raw[i]) same = false;
      same = __all_sync(0xffffffffu, same);
    }
    // Partition: this CTA's unit range and the sequence it starts in.
    const long long T = same ? sT : total_units(p, lane);
    const long long G = gridDim.x;
    const long long u0 = same ? su0 : cta_start(blockIdx.x, T, G);
    const long long u1 = same ? su1 : cta_start(blockIdx.x + 1, T, G);
    long long acc = 0;
    int b0 = same ? sb0 : p.batch;
    long long pb0 = same ? spb0 : T;
    if (!same && u1 > u0) {
      for (int base = 0; base < p.batch; base += 32) {
        const int b = base + lane;
        const int n = (b < p.batch) ? units_of(seq_ctx(p, b), p.tc) : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int t = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += t;
        }
        const long long end = acc + incl;  // cumulative end of sequence b
        const unsigned hit = __ballot_sync(0xffffffffu, b < p.batch && end > u0);
        if (hit) {
          const int src = __ffs(hit) - 1;
          const int incl_src = __shfl_sync(0xffffffffu, incl, src);
          const int n_src = __shfl_sync(0xffffffffu, n, src);
          b0 = base + src;
          pb0 = acc + incl_src - n_src;
          break;
        }
        acc += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (u1 > u0 && b0 < p.batch) {
        w.load_swin(p, lane, b0);
        w.load_bwin(p, lane, b0, static_cast<int>((u0 - pb0) * p.tc / p.block_size));
      }
    }
    if (warp == kCWarps && lane == 0) {
      sched[0] = u0;
      sched[1] = (u1 > u0) ? u1 : u0;
      sched[2] = b0;
      sched[3] = pb0;
    }
  }
  __syncthreads();
  // The next kernel (the combine pass) may start its launch now; it waits for
  // this grid's completion before reading the partials.
  grid_launch_dependents();

  const long long u0 = sched[0];
  const long long n_units = sched[1] - sched[0];
  if (warp >= kCWarps)
    produce<kStages, false>(tm_q, tm_k, tm_v, tm_k1, tm_v1, p, smem, full, empty, descs, w, u0, n_units,
                            static_cast<int>(sched[2]), sched[3], static_cast<int>(blockIdx.x), warp - kCWarps,
                            static_cast<int>(blockDim.x >> 5) - kCWarps, lane);
  else
    consume<kStages, false>(p, smem, full, empty, descs, zero_row, mg_full, mg_empty, merge, n_units, warp, lane);
}

// ------------------------------------------------------------------ combine
// Grid (batch, Hq / warps per CTA), one warp per (sequence, query head) (a
// CTA is one warp, or up to kCombinePeerWarps with peer stores); lane l owns
// dims 4l..4l+3. Sequences whose key range lies inside one CTA's range were
// written directly by the decode kernel and are skipped. Rows over a few
// CTAs (at most kCombineFew) merge their slots one after another. The others
// merge their partials: up to 32 slots per round, one per lane (each lane finds
// its CTA's slot with its own two divisions and loads that slot's lse, so a
// round costs one division latency whatever the slot count); the round's
// max and weight sum are warp reductions, then the O rows are read 8 at a
// time with independent loads.
constexpr int kCombineBatch = 8;
constexpr int kCombineFew = 4;  // rows over at most this many CTAs take the sequential merge

__device__ __forceinline__ float warp_max_all(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum_all(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// With peer stores (the KV-head-sharded all-gather) a CTA holds kCombinePeerWarps
// warps, one query head each, so that it ends with one system-scope fence for
// all of them: one fence per one-warp CTA, 2048 of them at 256 rows x 8 heads,
// cost 6.4 us per layer on one GPU. Otherwise a CTA is one warp.
constexpr int kCombinePeerWarps = 4;

// kMany: the instance for small batches, whose rows are split over many
// CTAs (one round of up to 32 slots): the round's first kManyBatch O rows
// are loaded together with its lse values, so a row over up to 16 CTAs is
// merged after one load round trip (the general path loads the lse, then the
// O rows of the slots that hold keys 8 at a time: four dependent round trips
// for a row over 18 CTAs). Slots are read whether or not they hold keys;
// those without are skipped by a warp-uniform test, never weighted by zero,
// so whatever they hold does not reach the sum.
constexpr int kManyBatch = 16;

template <bool kMany>
__global__ void __launch_bounds__(32 * kCombinePeerWarps, 1) paged_decode_combine_kernel(const Params p, int grid) {
  const int b = blockIdx.x;
  const int hh = blockIdx.y * static_cast<int>(blockDim.x >> 5) + static_cast<int>(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const float NEG_INF = -__int_as_float(0x7f800000);

  // T (all units) and P_b (units before sequence b). They depend only on
  // cache_seqlens, which were final before the decode grid started (it does
  // not write them), so they are computed while that grid still runs; every
  // CTA waits for it before touching outputs or partials. Each lane sums its
  // own sequences (lane + 32 i, coalesced, 16 independent loads at a time)
  // and two warp sums finish: a round trip per 512 sequences. (A warp sum
  // after every 32 sequences, one round trip each, took ~15 us at 1024
  // sequences, and the combine CTAs that launch only as decode CTAs leave
  // run it after the decode grid.)
  long long T = 0, Pb = 0;
  {
    constexpr int kLoads = 16;
    int own = 0, before = 0;
    for (int base = 0; base < p.batch; base += 32 * kLoads) {
      int n[kLoads];
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const int bb = base + 32 * k + lane;
        n[k] = (bb < p.batch) ? units_of(seq_ctx(p, bb), p.tc) : 0;
      }
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        own += n[k];
        if (base + 32 * k + lane < b) before += n[k];
      }
    }
    long long o = own, bf = before;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
      o += __shfl_xor_sync(0xffffffffu, o, x);
      bf += __shfl_xor_sync(0xffffffffu, bf, x);
    }
    T = o;
    Pb = bf;
  }
  const int nb = units_of(seq_ctx(p, b), p.tc);
  const long long Gl = grid;
  const long long oofs = static_cast<long long>(b) * p.out_b_stride + static_cast<long long>(hh) * p.out_h_stride +
                         lane * 4;
  float* lse = p.lse_out ? p.lse_out + static_cast<long long>(b) * p.hq + hh : nullptr;
  // The row's CTAs cf..cl and the partial slots they wrote, also from the
  // lengths alone (64-bit divisions), so after the wait only the loads and
  // the merge remain: for rows over a few CTAs every slot, for the others
  // this lane's slot of the first round of 32 (-1: no slot, or an empty
  // range, T < G, that wrote nothing).
  const long long cf = nb > 0 ? cta_of(Pb, T, Gl) : 0;
  const long long cl = nb > 0 ? cta_of(Pb + nb - 1, T, Gl) : -1;
  auto slot_of = [&](long long c) -> int {
    const long long s0 = cta_start(c, T, Gl);
    return s0 != cta_start(c + 1, T, Gl) ? 2 * static_cast<int>(c) + (s0 >= Pb ? 0 : 1) : -1;
  };
  int few[kCombineFew];
#pragma unroll
  for (int u = 0; u < kCombineFew; ++u)
    few[u] = (cf < cl && cl - cf < kCombineFew && cf + u <= cl) ? slot_of(cf + u) : -1;
  const int first_round = (cl - cf >= kCombineFew && cf + lane <= cl) ? slot_of(cf + lane) : -1;
  grid_dependency_wait();

  if (nb == 0) {
    for (int r = 0; r < p.nouts; ++r) *reinterpret_cast<uint2*>(p.outs[r] + oofs) = make_uint2(0u, 0u);
    if (lse && lane == 0) *lse = NEG_INF;
  } else {
    if (cf == cl) {  // written by the decode pass; forward it to the peers
      if (p.peer_stores) {
        const uint2 v = *reinterpret_cast<const uint2*>(p.out + oofs);
        for (int r = 0; r < p.nouts; ++r)
          if (p.outs[r] != p.out) *reinterpret_cast<uint2*>(p.outs[r] + oofs) = v;
      }
    } else if (cl - cf < kCombineFew) {
      // A few slots (rows split across two to four CTAs, the usual case at
      // large batches): merge them one after another, all loads issued first.
      float m = NEG_INF, l = 0.f;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      float ls[kCombineFew];
      float4 ov[kCombineFew];
#pragma unroll
      for (int u = 0; u < kCombineFew; ++u) {
        ls[u] = NEG_INF;
        if (few[u] >= 0) {
          const long long slot = few[u];
          ls[u] = p.part_lse[slot * p.hq + hh];
          ov[u] = *reinterpret_cast<const float4*>(p.part_o + (slot * p.hq + hh) * kD + lane * 4);
        }
      }
#pragma unroll
      for (int u = 0; u < kCombineFew; ++u) {
        if (ls[u] != NEG_INF) {
          const float mn = fmaxf(m, ls[u]);
          const float a = ex2(m - mn), w = ex2(ls[u] - mn);
          acc[0] = acc[0] * a + w * ov[u].x;
          acc[1] = acc[1] * a + w * ov[u].y;
          acc[2] = acc[2] * a + w * ov[u].z;
          acc[3] = acc[3] * a + w * ov[u].w;
          l = l * a + w;
          m = mn;
        }
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      uint2 v;
      v.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
      v.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
      for (int r = 0; r < p.nouts; ++r) *reinterpret_cast<uint2*>(p.outs[r] + oofs) = v;
      if (lse && lane == 0) *lse = l > 0.f ? (m + __log2f(l)) * 0.6931471805599453f : NEG_INF;
    } else if constexpr (kMany) {
      float m = NEG_INF, l = 0.f;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (long long c0 = cf; c0 <= cl; c0 += 32) {
        const long long c = c0 + lane;
        const int slot = c0 == cf ? first_round : (c <= cl ? slot_of(c) : -1);
        const int nr = static_cast<int>(cl - c0 + 1 < 32 ? cl - c0 + 1 : 32);  // lanes of this round
        const float ls = slot >= 0 ? p.part_lse[static_cast<long long>(slot) * p.hq + hh] : NEG_INF;
        int su[kManyBatch];
        float4 ov[kManyBatch];
#pragma unroll
        for (int k = 0; k < kManyBatch; ++k) su[k] = __shfl_sync(0xffffffffu, slot, k);
#pragma unroll
        for (int k = 0; k < kManyBatch; ++k)
          ov[k] = (k < nr && su[k] >= 0) ? *reinterpret_cast<const float4*>(
                                               p.part_o + (static_cast<long long>(su[k]) * p.hq + hh) * kD + lane * 4)
                                         : make_float4(0.f, 0.f, 0.f, 0.f);
        const float mr = warp_max_all(ls);
        if (mr == NEG_INF) continue;  // warp-uniform: no keys in this round
        const float mn = fmaxf(m, mr);
        const float a = ex2(m - mn);  // 0 while m is -inf
        const bool use = slot >= 0 && ls != NEG_INF;
        const float wl = use ? ex2(ls - mn) : 0.f;
        l = l * a + warp_sum_all(wl);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] *= a;
        m = mn;
        const unsigned usem = __ballot_sync(0xffffffffu, use);
#pragma unroll
        for (int k = 0; k < kManyBatch; ++k) {
          const float w = __shfl_sync(0xffffffffu, wl, k);
          if ((usem >> k) & 1u) {
            acc[0] += w * ov[k].x;
            acc[1] += w * ov[k].y;
            acc[2] += w * ov[k].z;
            acc[3] += w * ov[k].w;
          }
        }
        for (int j0 = kManyBatch; j0 < nr; j0 += kManyBatch) {
#pragma unroll
          for (int k = 0; k < kManyBatch; ++k) su[k] = __shfl_sync(0xffffffffu, slot, (j0 + k) & 31);
#pragma unroll
          for (int k = 0; k < kManyBatch; ++k)
            ov[k] = (j0 + k < nr && ((usem >> ((j0 + k) & 31)) & 1u))
                        ? *reinterpret_cast<const float4*>(p.part_o + (static_cast<long long>(su[k]) * p.hq + hh) * kD +
                                                           lane * 4)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < kManyBatch; ++k) {
            const float w = __shfl_sync(0xffffffffu, wl, (j0 + k) & 31);
            if (j0 + k < nr && ((usem >> ((j0 + k) & 31)) & 1u)) {
              acc[0] += w * ov[k].x;
              acc[1] += w * ov[k].y;
              acc[2] += w * ov[k].z;
              acc[3] += w * ov[k].w;
            }
          }
        }
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      uint2 v;
      v.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
      v.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
      for (int r = 0; r < p.nouts; ++r) *reinterpret_cast<uint2*>(p.outs[r] + oofs) = v;
      if (lse && lane == 0) *lse = l > 0.f ? (m + __log2f(l)) * 0.6931471805599453f : NEG_INF;
    } else {
      float m = NEG_INF, l = 0.f;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (long long c0 = cf; c0 <= cl; c0 += 32) {
        const long long c = c0 + lane;
        const int slot = c0 == cf ? first_round : (c <= cl ? slot_of(c) : -1);
        const float ls = slot >= 0 ? p.part_lse[static_cast<long long>(slot) * p.hq + hh] : NEG_INF;
        const float mr = warp_max_all(ls);
        if (mr == NEG_INF) continue;  // warp-uniform: no keys in this round
        const float mn = fmaxf(m, mr);
        const float a = ex2(m - mn);  // 0 while m is -inf
        const bool use = slot >= 0 && ls != NEG_INF;
        const float wl = use ? ex2(ls - mn) : 0.f;
        l = l * a + warp_sum_all(wl);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] *= a;
        m = mn;
        unsigned todo = __ballot_sync(0xffffffffu, use);
        while (todo) {
          int su[kCombineBatch];
          float wu[kCombineBatch];
#pragma unroll
          for (int k = 0; k < kCombineBatch; ++k) {
            const int u = todo ? __ffs(todo) - 1 : 0;
            const bool have = todo != 0;
            todo &= todo - 1u;
            const int sv = __shfl_sync(0xffffffffu, slot, u);
            const float wv = __shfl_sync(0xffffffffu, wl, u);
            su[k] = have ? sv : -1;
            wu[k] = have ? wv : 0.f;
          }
          float4 ov[kCombineBatch];
#pragma unroll
          for (int k = 0; k < kCombineBatch; ++k)
            ov[k] = su[k] >= 0 ? *reinterpret_cast<const float4*>(
                                     p.part_o + (static_cast<long long>(su[k]) * p.hq + hh) * kD + lane * 4)
                               : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < kCombineBatch; ++k) {
            if (su[k] >= 0) {
              acc[0] += wu[k] * ov[k].x;
              acc[1] += wu[k] * ov[k].y;
              acc[2] += wu[k] * ov[k].z;
              acc[3] += wu[k] * ov[k].w;
            }
          }
        }
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      uint2 v;
      v.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
      v.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
      for (int r = 0; r < p.nouts; ++r) *reinterpret_cast<uint2*>(p.outs[r] + oofs) = v;
      if (lse && lane == 0) *lse = l > 0.f ? (m + __log2f(l)) * 0.6931471805599453f : NEG_INF;
    }
  }
  if (p.peer_stores) {
    // One system-scope fence per CTA: __syncthreads orders every thread's
    // peer stores before thread 0's fence, which is cumulative over them, so
    // the epoch the barrier kernel publishes next on this stream (a release
    // at system scope, after this grid completes) orders after all of them.
    __syncthreads();
    if (threadIdx.x == 0) __threadfence_system();
  }
}

// ------------------------------------------------------------------ host
static int stages_for(int stage_bytes, size_t ctrl_bytes, size_t* smem) {
  const size_t limit = 227 * 1024;
  for (int st = 3; st >= 2; --st) {
    const size_t need = 1024 /*align slack*/ + static_cast<size_t>(st) * stage_bytes + ctrl_bytes;
    if (need <= limit) {
      *smem = need;
      return st;
    }
  }
  return 0;
}

static int grid_for(int device) { return num_sms(device); }

}  // namespace decode

int decode_init(int device) {
  (void)device;
  const int lim = 227 * 1024;
  cudaError_t e = cudaFuncSetAttribute(decode::paged_decode_kernel<3, 8>, cudaFuncAttributeMaxDynamicSharedMemorySize, lim);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(decode::paged_decode_kernel<2, 8>, cudaFuncAttributeMaxDynamicSharedMemorySize, lim);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(decode::paged_decode_kernel<3, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, lim);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(decode::paged_decode_kernel<2, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, lim);
  if (e == cudaSuccess) {
    cudaFuncAttributes a;
    e = cudaFuncGetAttributes(&a, decode::paged_decode_combine_kernel<false>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, decode::paged_decode_combine_kernel<true>);
  }
  return cuda_status(e);
}

}  // namespace la

extern "C" int la_paged_decode_workspace_size(int device, int num_q_heads, int num_kv_heads, int head_dim,
                                              size_t* bytes) {
  if (!bytes || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim != 128 || num_kv_heads > 8 ||
      8 % num_kv_heads != 0)
    return LA_ERR_INVALID_ARGUMENT;
  const int grid = la::decode::grid_for(device);
  if (grid <= 0) return LA_ERR_CUDA;
  const size_t slots = static_cast<size_t>(2) * grid;
  const size_t o_bytes = slots * num_q_heads * head_dim * sizeof(float);
  const size_t l_bytes = slots * num_q_heads * sizeof(float);
  *bytes = ((o_bytes + 255) & ~size_t(255)) + ((l_bytes + 255) & ~size_t(255));
  return LA_OK;
}

namespace la {
namespace decode {

// Peer outputs of the KV-head-sharded all-gather (nullptr: local output only).
struct PeerOut {
  void* const* outs;  // [npeers] gather buffers, rank order (own included)
  int npeers;
};

int prepare_call(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache,
                 const void* v_cache, int64_t kv_block_stride, int64_t kv_token_stride, int64_t kv_head_stride,
                 int64_t num_blocks, int block_size, const int32_t* block_table, int64_t bt_seq_stride,
                 int max_blocks_per_seq, const int32_t* cache_seqlens, int batch, int num_q_heads, int num_kv_heads,
                 int head_dim, float softmax_scale, void* out, int64_t out_batch_stride, int64_t out_head_stride,
                 float* softmax_lse, int* dev_error, Call* call) {
  if (!q || !k_cache || !v_cache || !block_table || !cache_seqlens || !out) return LA_ERR_INVALID_ARGUMENT;
  if (batch < 0 || num_blocks <= 0 || block_size <= 0 || max_blocks_per_seq <= 0) return LA_ERR_INVALID_ARGUMENT;
  if (batch == 0) return LA_OK;
  if (head_dim != kD) return LA_ERR_UNSUPPORTED;
  if (num_kv_heads <= 0 || num_kv_heads > 8 || 8 % num_kv_heads != 0) return LA_ERR_UNSUPPORTED;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads != 0) return LA_ERR_INVALID_ARGUMENT;
  const int group = num_q_heads / num_kv_heads;
  if (group > 8 || num_q_heads > 256) return LA_ERR_UNSUPPORTED;
  if (block_size % kSub != 0) return LA_ERR_UNSUPPORTED;
  if (!(softmax_scale > 0.f)) return LA_ERR_INVALID_ARGUMENT;
  // TMA: 16-byte aligned bases and byte strides.
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16)) return LA_ERR_ALIGNMENT;
  if ((q_batch_stride * 2) % 16 || (q_head_stride * 2) % 16 || (kv_block_stride * 2) % 16 ||
      (kv_token_stride * 2) % 16 || (kv_head_stride * 2) % 16)
    return LA_ERR_ALIGNMENT;
  if (q_batch_stride <= 0 || q_head_stride <= 0 || kv_block_stride <= 0 || kv_token_stride <= 0 ||
      kv_head_stride <= 0 || out_batch_stride <= 0 || out_head_stride <= 0)
    return LA_ERR_INVALID_ARGUMENT;
  // the combine pass stores 4 bf16 per lane
  if (!aligned(out, 8) || out_batch_stride % 4 || out_head_stride % 4) return LA_ERR_ALIGNMENT;

  int st = LA_OK;
  CUtensorMap& tq = call->q;
  CUtensorMap& tk = call->k;
  CUtensorMap& tv = call->v;
  CUtensorMap& tk1 = call->k1;
  CUtensorMap& tv1 = call->v1;
  {
    const uint64_t dims[3] = {128, static_cast<uint64_t>(num_q_heads), static_cast<uint64_t>(batch)};
    const uint64_t strides[2] = {static_cast<uint64_t>(q_head_stride) * 2, static_cast<uint64_t>(q_batch_stride) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(num_q_heads), 1};
    if ((st = encode_tensor_map_bf16(&tq, q, 3, dims, strides, box, true)) != LA_OK) return st;
  }
  int big_box = 0;
  const int nsub = 8 / num_kv_heads;
  if (nsub >= 4 && block_size % (kSub * nsub) == 0) {
    // A whole unit (tc = 16 * nsub tokens of every kv head) per box: the
    // 16-token groups of a block as their own axis, after the heads, so the
    // box's rows come in the stage's order [group][head][token]. With one
    // kv head this replaces 32 boxes of 2 KB per stage by 4 of 16 KB (the
    // 8-GPU KV-head-sharded rank: 109 -> 89 us per layer at B = 1024), with
    // two 16 boxes of 4 KB (even); with four it measured slower than a box
    // per sub-chunk.
    const uint64_t dims[5] = {128, static_cast<uint64_t>(kSub), static_cast<uint64_t>(num_kv_heads),
                              static_cast<uint64_t>(block_size / kSub), static_cast<uint64_t>(num_blocks)};
    const uint64_t strides[4] = {static_cast<uint64_t>(kv_token_stride) * 2, static_cast<uint64_t>(kv_head_stride) * 2,
                                 static_cast<uint64_t>(kv_token_stride) * 2 * kSub,
                                 static_cast<uint64_t>(kv_block_stride) * 2};
    const uint32_t box[5] = {64, static_cast<uint32_t>(kSub), static_cast<uint32_t>(num_kv_heads),
                             static_cast<uint32_t>(nsub), 1};
    // The same layout with one 16-token group per box, for a sequence's
    // last unit when it is not full.
    const uint32_t box1[5] = {64, static_cast<uint32_t>(kSub), static_cast<uint32_t>(num_kv_heads), 1, 1};
    if (encode_tensor_map_bf16(&tk, k_cache, 5, dims, strides, box, true) == LA_OK &&
        encode_tensor_map_bf16(&tv, v_cache, 5, dims, strides, box, true) == LA_OK &&
        encode_tensor_map_bf16(&tk1, k_cache, 5, dims, strides, box1, true) == LA_OK &&
        encode_tensor_map_bf16(&tv1, v_cache, 5, dims, strides, box1, true) == LA_OK)
      big_box = 2;
  }
  if (!big_box) {
    // Token axis before the head axis, so one box covers all kv heads of 16
    // tokens (strides need not grow with the dimension index).
    const uint64_t dims[4] = {128, static_cast<uint64_t>(block_size), static_cast<uint64_t>(num_kv_heads),
                              static_cast<uint64_t>(num_blocks)};
    const uint64_t strides[3] = {static_cast<uint64_t>(kv_token_stride) * 2, static_cast<uint64_t>(kv_head_stride) * 2,
                                 static_cast<uint64_t>(kv_block_stride) * 2};
    const uint32_t box[4] = {64, static_cast<uint32_t>(kSub), static_cast<uint32_t>(num_kv_heads), 1};
    if (encode_tensor_map_bf16(&tk, k_cache, 4, dims, strides, box, true) == LA_OK &&
        encode_tensor_map_bf16(&tv, v_cache, 4, dims, strides, box, true) == LA_OK)
      big_box = 1;
  }
  if (!big_box) {
    const uint64_t dims[4] = {128, static_cast<uint64_t>(num_kv_heads), static_cast<uint64_t>(block_size),
                              static_cast<uint64_t>(num_blocks)};
    const uint64_t strides[3] = {static_cast<uint64_t>(kv_head_stride) * 2, static_cast<uint64_t>(kv_token_stride) * 2,
                                 static_cast<uint64_t>(kv_block_stride) * 2};
    const uint32_t box[4] = {64, 1, static_cast<uint32_t>(kSub), 1};
    if ((st = encode_tensor_map_bf16(&tk, k_cache, 4, dims, strides, box, true)) != LA_OK) return st;
    if ((st = encode_tensor_map_bf16(&tv, v_cache, 4, dims, strides, box, true)) != LA_OK) return st;
  }
  if (big_box != 2) {  // the one-group maps are read only with whole-unit boxes
    tk1 = tk;
    tv1 = tv;
  }

  Params& p = call->p;
  p = Params{};
  p.seqlens = cache_seqlens;
  p.block_table = block_table;
  p.bt_stride = bt_seq_stride;
  p.max_blocks = max_blocks_per_seq;
  p.batch = batch;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.group = group;
  p.nsub = 8 / num_kv_heads;
  p.block_size = block_size;
  p.bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(block_size)) : -1;
  p.num_blocks = num_blocks;
  p.tc = kSub * p.nsub;
  p.tc_shift = __builtin_ctz(static_cast<unsigned>(p.tc));
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_b_stride = out_batch_stride;
  p.out_h_stride = out_head_stride;
  p.nouts = 1;
  p.outs[0] = p.out;
  p.peer_stores = 0;
  p.lse_out = softmax_lse;
  p.err = dev_error;
  // Each Q half tile starts on a 1024-byte boundary (the 128-byte swizzle atom).
  p.big_box = big_box == 1;
  p.unit_box = big_box == 2;
  p.q_half_bytes = (num_q_heads * 128 + 1023) & ~1023;
  p.q_bytes = 2 * num_q_heads * 128;
  p.stage_bytes = 2 * kKVBytes + 2 * p.q_half_bytes;
  call->merge_bytes = (p.nsub > 1) ? kCWarps * ((group + 1) / 2) * 8 * 36 * 4 : 0;
  return LA_OK;
}

static int paged_decode_impl(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache,
                             const void* v_cache, int64_t kv_block_stride, int64_t kv_token_stride,
                             int64_t kv_head_stride, int64_t num_blocks, int block_size,
                             const int32_t* block_table, int64_t bt_seq_stride, int max_blocks_per_seq,
                             const int32_t* cache_seqlens, int batch, int num_q_heads, int num_kv_heads,
                             int head_dim, float softmax_scale, void* out, int64_t out_batch_stride,
                             int64_t out_head_stride, float* softmax_lse, void* workspace, size_t workspace_bytes,
                             int* dev_error, cudaStream_t stream, const PeerOut* peers) {
  Call call;
  int st = prepare_call(q, q_batch_stride, q_head_stride, k_cache, v_cache, kv_block_stride, kv_token_stride,
                        kv_head_stride, num_blocks, block_size, block_table, bt_seq_stride, max_blocks_per_seq,
                        cache_seqlens, batch, num_q_heads, num_kv_heads, head_dim, softmax_scale, out,
                        out_batch_stride, out_head_stride, softmax_lse, dev_error, &call);
  if (st != LA_OK || batch == 0) return st;
  Params& p = call.p;
  const CUtensorMap &tq = call.q, &tk = call.k, &tv = call.v, &tk1 = call.k1, &tv1 = call.v1;
  const int device = current_device();
  if (device < 0) return LA_ERR_CUDA;
  const int grid = grid_for(device);
  if (grid <= 0) return LA_ERR_CUDA;
  size_t need = 0;
  st = la_paged_decode_workspace_size(device, num_q_heads, num_kv_heads, head_dim, &need);
  if (st != LA_OK) return st;
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256)) return LA_ERR_WORKSPACE;
  if (peers) {
    if (peers->npeers < 1 || peers->npeers > kMaxPeers || !peers->outs) return LA_ERR_INVALID_ARGUMENT;
    p.nouts = peers->npeers;
    for (int r = 0; r < peers->npeers; ++r) {
      if (!peers->outs[r] || !aligned(peers->outs[r], 8)) return LA_ERR_INVALID_ARGUMENT;
      p.outs[r] = static_cast<__nv_bfloat16*>(peers->outs[r]);
    }
    p.peer_stores = 1;
  }
  const size_t slots = static_cast<size_t>(2) * grid;
  const size_t o_bytes = (slots * num_q_heads * kD * sizeof(float) + 255) & ~size_t(255);
  p.part_o = static_cast<float*>(workspace);
  p.part_lse = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + o_bytes);
  size_t smem = 0;
  const int stages = stages_for(p.stage_bytes, 1024 + call.merge_bytes, &smem);
  if (stages == 0) return LA_ERR_UNSUPPORTED;

  // A second producer warp pays off once units are many per CTA (at 1024
  // one-kv-head rows it took the pipeline off the producer's path); with a
  // few short sequences (B = 8) the extra warp measured slower.
  const int threads = (kCWarps + (batch >= 16 ? 2 : 1)) * 32;
  cudaError_t e;
  if (stages == 3)
    e = batch <= 256 ? launch_pdl(paged_decode_kernel<3, 8>, dim3(grid), dim3(threads), smem, stream, tq, tk, tv, tk1, tv1, p)
                     : launch_pdl(paged_decode_kernel<3, 32>, dim3(grid), dim3(threads), smem, stream, tq, tk, tv, tk1, tv1, p);
  else
    e = batch <= 256 ? launch_pdl(paged_decode_kernel<2, 8>, dim3(grid), dim3(threads), smem, stream, tq, tk, tv, tk1, tv1, p)
                     : launch_pdl(paged_decode_kernel<2, 32>, dim3(grid), dim3(threads), smem, stream, tq, tk, tv, tk1, tv1, p);
  if (e != cudaSuccess) return cuda_status(e);
  // peer stores: kCombinePeerWarps heads per CTA (fewer when they do not divide the heads)
  int wpc = 1;
  if (peers)
    for (int c = kCombinePeerWarps; c > 1; c >>= 1)
      if (num_q_heads % c == 0) {
        wpc = c;
        break;
      }
  // Rows over more than kCombineFew CTAs on average (batch * kCombineFew <
  // grid) take the many-slot instance.
  const dim3 cgrid(batch, num_q_heads / wpc), cblock(32 * wpc);
  e = static_cast<long long>(batch) * kCombineFew < grid
          ? launch_pdl(paged_decode_combine_kernel<true>, cgrid, cblock, 0, stream, p, grid)
          : launch_pdl(paged_decode_combine_kernel<false>, cgrid, cblock, 0, stream, p, grid);
  return cuda_status(e);
}

}  // namespace decode
}  // namespace la

extern "C" int la_paged_decode(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache,
                               const void* v_cache, int64_t kv_block_stride, int64_t kv_token_stride,
                               int64_t kv_head_stride, int64_t num_blocks, int block_size,
                               const int32_t* block_table, int64_t bt_seq_stride, int max_blocks_per_seq,
                               const int32_t* cache_seqlens, int batch, int num_q_heads, int num_kv_heads,
                               int head_dim, float softmax_scale, void* out, int64_t out_batch_stride,
                               int64_t out_head_stride, float* softmax_lse, void* workspace,
                               size_t workspace_bytes, int* dev_error, cudaStream_t stream) {
  return la::decode::paged_decode_impl(q, q_batch_stride, q_head_stride, k_cache, v_cache, kv_block_stride,
                                       kv_token_stride, kv_head_stride, num_blocks, block_size, block_table,
                                       bt_seq_stride, max_blocks_per_seq, cache_seqlens, batch, num_q_heads,
                                       num_kv_heads, head_dim, softmax_scale, out, out_batch_stride, out_head_stride,
                                       softmax_lse, workspace, workspace_bytes, dev_error, stream, nullptr);
}

extern "C" int la_paged_decode_allgather(
    const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache, const void* v_cache,
    int64_t kv_block_stride, int64_t kv_token_stride, int64_t kv_head_stride, int64_t num_blocks, int block_size,
    const int32_t* block_table, int64_t bt_seq_stride, int max_blocks_per_seq, const int32_t* cache_seqlens,
    int batch, int num_q_heads, int num_kv_heads, int head_dim, float softmax_scale, void* const* gather_bufs,
    int64_t out_batch_stride, int64_t out_head_stride, int rank, int world, void* workspace,
    size_t workspace_bytes, int* dev_error, cudaStream_t stream) {
  if (!gather_bufs || world < 1 || world > la::decode::kMaxPeers || rank < 0 || rank >= world)
    return LA_ERR_INVALID_ARGUMENT;
  // This rank's query heads sit at [rank * Hq_local, (rank + 1) * Hq_local) of
  // every gather buffer.
  void* outs[la::decode::kMaxPeers];
  const int64_t head0 = static_cast<int64_t>(rank) * num_q_heads * out_head_stride;
  for (int r = 0; r < world; ++r) {
    if (!gather_bufs[r]) return LA_ERR_INVALID_ARGUMENT;
    outs[r] = static_cast<__nv_bfloat16*>(gather_bufs[r]) + head0;
  }
  la::decode::PeerOut peers{outs, world};
  return la::decode::paged_decode_impl(q, q_batch_stride, q_head_stride, k_cache, v_cache, kv_block_stride,
                                       kv_token_stride, kv_head_stride, num_blocks, block_size, block_table,
                                       bt_seq_stride, max_blocks_per_seq, cache_seqlens, batch, num_q_heads,
                                       num_kv_heads, head_dim, softmax_scale, outs[rank], out_batch_stride,
                                       out_head_stride, nullptr, workspace, workspace_bytes, dev_error, stream,
                                       &peers);
}
