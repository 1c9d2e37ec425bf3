// The streaming part of paged GQA decode: producer and consumer warps over a
// CTA's range of units, shared by the decode kernel (la_decode.cu, which
// describes it) and by the pass over the rows' own keys beside shared
// prefixes (la_prefix.cu, kPrefix).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "la_groups.cuh"
#include "la_internal.h"
#include "la_ptx.cuh"

namespace la {
namespace decode {

constexpr int kD = 128;
constexpr int kSub = 16;                 // tokens per consumer warp per stage (MMA M)
constexpr int kCWarps = 8;               // consumer warps
constexpr int kMaxProducers = 2;  // producer warps (units alternate between them); the launch picks 1 or 2
constexpr int kThreads = (kCWarps + kMaxProducers) * 32;
constexpr int kTileBytes = kSub * 128;   // 16 rows x 64 dims bf16 (one swizzle-128B tile)
constexpr int kWarpBytes = 2 * kTileBytes;
constexpr int kKVHalf = kCWarps * kTileBytes;   // one 64-dim half of all warps' tiles: 16 KB
constexpr int kKVBytes = 2 * kKVHalf;           // 32 KB per tensor per stage
// Stage layout per tensor: [half][warp w][16 rows][128 B]; warp w = j*Hkv + h
// holds kv head h of sub-chunk j, so the Hkv heads of a sub-chunk are one
// contiguous run that a single TMA box [64 dims, 16 tokens, Hkv heads] fills.
constexpr int kMaxStages = 4;

constexpr int kMaxPeers = 8;  // ranks of a KV-head-sharded group
constexpr int kFlagFirst = 1;  // first stage of this CTA's segment of the sequence
constexpr int kFlagLast = 2;   // last stage of the segment
constexpr int kFlagWhole = 4;  // the segment is the whole sequence

struct StageDesc {
  int b;
  int tok0;
  int ctx;
  int flags;
  int slot;  // partial slot base (2*cta + 0/1) for segments that are not whole
  int pad[3];
};

struct Params {
  const int* seqlens;
  const int* block_table;
  long long bt_stride;
  int max_blocks;
  int batch;
  int hq, hkv, group, nsub;  // nsub = 8 / hkv consumer warps per kv head
  int block_size;
  int bs_shift;              // log2(block_size) when it is a power of two, else -1
  int tc_shift;              // log2(tc)
  long long num_blocks;
  int tc;                    // tokens per stage
  float scale_log2;
  __nv_bfloat16* out;
  long long out_b_stride, out_h_stride;
  // The decode pass writes `out` only. The combine pass stores every output
  // row to outs[0..nouts): `out` alone, or, for the KV-head-sharded
  // all-gather, every rank's gather buffer (peer pointers over NVLink; rows
  // the decode pass finished are forwarded from `out` with coalesced 8-byte
  // stores). With peer_stores set, each combine CTA then fences once at
  // system scope, so the epoch a later barrier publishes orders after its
  // stores.
  __nv_bfloat16* outs[kMaxPeers];
  int nouts;
  int peer_stores;
  float* lse_out;
  float* part_o;    // [slots][hq][D]
  float* part_lse;  // [slots][hq] (log2 domain, scaled)
  int* err;
  int q_bytes;      // Q bytes landed per stage (both halves)
  int q_half_bytes; // stride between the two Q halves (1024-byte aligned)
  int stage_bytes;
  int big_box;      // 1: K/V maps are [D, BS, Hkv, NB] with box (64, 16, Hkv, 1)
  // 1: one or two kv heads over blocks of a multiple of tc tokens: the K/V
  // maps are 5-D [D, 16 tokens, Hkv, BS / 16, NB] with box
  // (64, 16, Hkv, nsub, 1), whose rows land in the stage's order [sub-chunk
  // j][kv head][16 tokens]: a whole unit per half per tensor in one box.
  int unit_box;
  // kPrefix: another pass covers the keys that row b shares with its group,
  // and row b reads the ones behind them: its key positions and block-table
  // columns are counted from there on (what is shared ends with a page).
  // Rows that share keys, and rows split across CTAs, leave fp32 partials in
  // slot (row + CTA), distinct for every part: from one part to the next
  // along the line of units the row, the CTA or both go up by one. The first
  // and last CTA of a row's parts go to row_parts[2 b] and [2 b + 1].
  PrefixGroups groups;
  int* row_parts;
};

// Number of stage units of a sequence, with the same clamping everywhere.
__device__ __forceinline__ int seq_ctx(const Params& p, int b) {
  int c = p.seqlens[b];
  if (c < 0) c = 0;
  const long long cap = static_cast<long long>(p.max_blocks) * p.block_size;
  if (c > cap) {
    if (p.err) atomicCAS(p.err, 0, LA_DEVERR_SEQLEN);
    c = static_cast<int>(cap);
  }
  return c;
}
// Keys that row b reads by itself, and (kPrefix) the blocks before them.
template <bool kPrefix>
__device__ __forceinline__ int own_keys(const Params& p, const PrefixGroup* tab, int b, int* block0) {
  const int ctx = seq_ctx(p, b);
  if constexpr (!kPrefix) return ctx;
  const int n = prefix_keys(p.groups, tab, b, ctx);
  *block0 = p.bs_shift >= 0 ? (n >> p.bs_shift) : (n / p.block_size);
  return ctx - n;
}
__device__ __forceinline__ int units_of(int ctx, int tc) { return (ctx + tc - 1) / tc; }
// Division by the block size and the unit size on the producer's per-unit
// path: shifts (a division by a run-time value is a dependent chain of about
// twenty instructions, and the producer paced the pipeline at one kv head).
__device__ __forceinline__ int div_bs(const Params& p, int x) {
  return p.bs_shift >= 0 ? (x >> p.bs_shift) : (x / p.block_size);
}
__device__ __forceinline__ int units_p(const Params& p, int ctx) { return (ctx + p.tc - 1) >> p.tc_shift; }

__device__ __forceinline__ float warp_max_g(float v) {
  // max over the 8 lanes that share lane % 4
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
  return v;
}
__device__ __forceinline__ float warp_sum_g(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  v += __shfl_xor_sync(0xffffffffu, v, 16);
  return v;
}

// First unit of CTA c: floor(c * T / G).
__device__ __forceinline__ long long cta_start(long long c, long long T, long long G) { return c * T / G; }
// CTA whose range contains unit x: floor(((x + 1) * G - 1) / T).
__device__ __forceinline__ long long cta_of(long long x, long long T, long long G) { return ((x + 1) * G - 1) / T; }

// Producer lookups go through two windows held across its 32 lanes, so
// that a unit's copies wait on no global load in the common case: lane i
// holds the (clamped) length of sequence sb + i, and the raw block id of
// block wl + i of sequence bb. Entering a sequence also loads the first 32
// block ids of the next one, which are read at the next sequence change
// (with one kv head a sequence is ~6 units, and two dependent global round
// trips per unit made the producer the slowest part of the pipeline).
template <bool kPrefix>
struct Windows {
  const PrefixGroup* tab = nullptr;
  int sb = 0, swin = 0, bb = -1, wl = 0, bwin = -1;
  int owin = 0;  // kPrefix: the blocks before the sequence's own keys, beside swin
  __device__ __forceinline__ void load_swin(const Params& p, int lane, int base) {
    sb = base;
    swin = (sb + lane < p.batch) ? own_keys<kPrefix>(p, tab, sb + lane, &owin) : 0;
  }
  // The first block of sequence `seq` that it reads by itself (warp-uniform).
  __device__ __forceinline__ int block0(const Params& p, int seq) const {
    if constexpr (!kPrefix) return 0;
    if (seq >= sb && seq < sb + 32) return __shfl_sync(0xffffffffu, owin, seq - sb);
    int o = 0;
    if (seq < p.batch) own_keys<kPrefix>(p, tab, seq, &o);
    return o;
  }
  __device__ __forceinline__ int ids(const Params& p, int lane, int seq, int first) const {
    const int o = block0(p, seq);
    return (seq < p.batch && o + first + lane < p.max_blocks)
               ? p.block_table[static_cast<long long>(seq) * p.bt_stride + o + first + lane]
               : -1;
  }
  __device__ __forceinline__ void load_bwin(const Params& p, int lane, int seq, int first) {
    bb = seq;
    wl = first;
    bwin = ids(p, lane, seq, first);
  }
};

// Stage of unit k, and the parity of its phase. kStages 0: two or three, as
// `stages` says.
template <int kStages>
__device__ __forceinline__ int stage_of(int k, int stages, uint32_t& ph) {
  const int n = kStages > 0 ? k / kStages : stages == 2 ? k / 2 : k / 3;
  ph = static_cast<uint32_t>(n & 1);
  return k - n * (kStages > 0 ? kStages : stages);
}

// A producer warp: units u0 .. u0 + n_units - 1 of the line, from sequence b0
// (whose first unit is pb0) on, pid-th of nprod producers.
template <int kStages, bool kPrefix>
__device__ __forceinline__ void produce(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                        const CUtensorMap& tm_k1, const CUtensorMap& tm_v1, const Params& p,
                                        uint8_t* smem, uint64_t* full, uint64_t* empty, StageDesc* descs,
                                        Windows<kPrefix>& w, long long u0, long long n_units, int b0, long long pb0,
                                        int cta, int pid, int nprod, int lane, int stages = kStages) {
  const int hkv = p.hkv;
  // kPrefix: a row's own keys are read once, and beside them run CTAs that
  // read the shared ones, and code, from L2.
  [[maybe_unused]] const uint64_t once = kPrefix ? l2_evict_first() : 0;
  auto load4 = [&](void* dst, const CUtensorMap* tm, uint64_t* bar, int c0, int c1, int c2, int c3) {
    if constexpr (kPrefix)
      tma_load_4d(dst, tm, bar, c0, c1, c2, c3, once);
    else
      tma_load_4d(dst, tm, bar, c0, c1, c2, c3);
  };
  auto load5 = [&](void* dst, const CUtensorMap* tm, uint64_t* bar, int c0, int c1, int c2, int c3, int c4) {
    if constexpr (kPrefix)
      tma_load_5d(dst, tm, bar, c0, c1, c2, c3, c4, once);
    else
      tma_load_5d(dst, tm, bar, c0, c1, c2, c3, c4);
  };
  // Producer pid issues units k = pid, pid + nprod, ...; every producer
  // walks every unit to follow the sequences. One warp's per-unit path
  // (stage wait, descriptor, four TMA boxes whose issue alone takes ~650
  // clocks) paced the pipeline when sequences are short; two alternate.
  const int nu = static_cast<int>(n_units);
  int b = b0;
  int uis = static_cast<int>(u0 - pb0);  // unit of the current sequence at k
  int seq_k0 = -uis;                          // k of the current sequence's unit 0
  int ctx = (nu > 0) ? __shfl_sync(0xffffffffu, w.swin, 0) : 0;
  int nb = units_p(p, ctx);
  int nbb = -1, nbwin = -1;  // the next sequence's first block ids
  // This lane's warp slot (lanes 0..7): sub-chunk jl, kv head hl.
  const int jl = (lane < kCWarps) ? lane / hkv : 0;
  const int hl = (lane < kCWarps) ? lane - jl * hkv : 0;
  int k = 0;
  for (; k < nu; ++k, ++uis) {
    while (uis >= nb && b + 1 < p.batch) {
      ++b;
      uis = 0;
      seq_k0 = k;
      if (b - w.sb >= 32) w.load_swin(p, lane, b);
      ctx = __shfl_sync(0xffffffffu, w.swin, b - w.sb);
      nb = units_p(p, ctx);
    }
    if (uis >= nb) break;  // seqlens changed under the kernel: stop issuing
    if (k % nprod != pid) continue;
    const int tok0 = uis * p.tc;
    {
      // Blocks of this unit's sub-chunks that hold keys: [lbf, lbl].
      const int lbf = div_bs(p, tok0);
      const int lbl = div_bs(p, min(tok0 + p.tc, ctx) - 1);
      if (w.bb != b || lbf < w.wl || lbl >= w.wl + 32) {
        if (b == nbb && lbf == 0 && lbl < 32) {
          w.bb = b;
          w.wl = 0;
          w.bwin = nbwin;
        } else {
          w.load_bwin(p, lane, b, lbf);
        }
      }
      if (nbb <= b) {  // read at the next sequence change, not before
        nbb = b + 1;
        nbwin = w.ids(p, lane, nbb, 0);
      }
    }
    uint32_t ph;
    const int s = stage_of<kStages>(k, stages, ph);
    if (!mbar_wait(&empty[s], ph ^ 1u, p.err, LA_DEVERR_WAIT_TIMEOUT)) break;
    uint8_t* st = smem + s * p.stage_bytes;

    // Sub-chunk of warp-slot `lane` (lanes 0..7).
    bool active = false;
    int phys = -1, off = 0, head = 0, lb = 0;
    if (lane < kCWarps) {
      head = hl;
      const int t = tok0 + kSub * jl;
      if (t < ctx) {
        active = true;
        lb = div_bs(p, t);
        off = t - lb * p.block_size;
      }
    }
    // every lane takes part in the shuffle; inactive ones read lane 0
    const int id = __shfl_sync(0xffffffffu, w.bwin, active ? lb - w.wl : 0);
    if (active) {
      if (lb < p.max_blocks) {
        phys = id;
        // Out-of-pool ids are reported; TMA zero-fills the box for them.
        if ((phys < 0 || phys >= p.num_blocks) && p.err) atomicCAS(p.err, 0, LA_DEVERR_BLOCK_ID);
      } else if (p.err) {
        atomicCAS(p.err, 0, LA_DEVERR_SEQLEN);
      }
    }
    const unsigned act = __ballot_sync(0xffffffffu, active);
    const int shared = w.block0(p, b);
    if (lane == 0) {
      StageDesc d;
      d.b = b;
      d.tok0 = tok0;
      d.ctx = ctx;
      int flags = 0;
      if (k == 0 || uis == 0) flags |= kFlagFirst;
      if (k == nu - 1 || uis == nb - 1) flags |= kFlagLast;
      if (seq_k0 >= 0 && seq_k0 + nb <= nu && shared == 0) flags |= kFlagWhole;
      d.flags = flags;
      d.slot = kPrefix ? b + cta : 2 * cta + (seq_k0 <= 0 ? 0 : 1);
      if (kPrefix && uis == 0) p.row_parts[2 * b] = cta;
      if (kPrefix && uis == nb - 1) p.row_parts[2 * b + 1] = cta;
      descs[s] = d;
      // Q is read only on a sequence's first unit (kFlagFirst): load it there.
      const bool first = (flags & kFlagFirst) != 0;
      const bool whole_unit = tok0 + p.tc <= ctx;
      const uint32_t boxes =
          (p.unit_box && whole_unit) ? static_cast<uint32_t>(kCWarps) : static_cast<uint32_t>(__popc(act));
      const uint32_t bytes = boxes * (2 * kWarpBytes) + (first ? p.q_bytes : 0u);
      mbar_arrive_expect_tx(&full[s], bytes);
      if (first) {
        uint8_t* qs = st + 2 * kKVBytes;
        tma_load_3d(qs, &tm_q, &full[s], 0, 0, b);
        tma_load_3d(qs + p.q_half_bytes, &tm_q, &full[s], 64, 0, b);
      }
    }
    __syncwarp();
    if (phys < 0) phys = -1;  // outside the pool: TMA fills zeros
    // The four boxes of a sub-chunk (K and V, two 64-dim halves each) are
    // issued by four lanes in one instruction rather than one lane in four.
    const int piece = lane & 3;
    const int tens = piece >> 1, half = piece & 1;
    if (p.unit_box && tok0 + p.tc <= ctx) {
      // Lane 0's sub-chunk 0 starts the unit, inside one block.
      const int ph0 = __shfl_sync(0xffffffffu, phys, 0);
      const int grp = __shfl_sync(0xffffffffu, off, 0) / kSub;
      if (lane < 4)
        load5(st + tens * kKVBytes + half * kKVHalf, tens ? &tm_v : &tm_k, &full[s], half * 64, 0, 0, grp,
                    ph0);
    } else if (p.unit_box) {
      // A sequence's last unit, not full: only the sub-chunks that hold
      // keys, one box [64 dims, 16 tokens, Hkv heads] per half per tensor
      // each (the whole-unit box would read up to 7/8 of a unit of rows
      // past ctx: 8.5 % more bytes at one kv head over U[512, 1024]).
      // Rows past ctx inside the last active sub-chunk are loaded and
      // masked by its consumers; sub-chunks past ctx are neither loaded
      // nor read.
      if (active && head == 0) {
        const int grp = off / kSub;
        uint8_t* kd = st + lane * kTileBytes;
        uint8_t* vd = st + kKVBytes + lane * kTileBytes;
        load5(kd, &tm_k1, &full[s], 0, 0, 0, grp, phys);
        load5(kd + kKVHalf, &tm_k1, &full[s], 64, 0, 0, grp, phys);
        load5(vd, &tm_v1, &full[s], 0, 0, 0, grp, phys);
        load5(vd + kKVHalf, &tm_v1, &full[s], 64, 0, 0, grp, phys);
      }
    } else if (p.big_box) {
      // Sub-chunk j (all kv heads in one box per half, the lane of its head
      // 0 holding id and offset) is issued by lanes 4j .. 4j + 3.
      const int jj = lane >> 2;
      const int src = (jj < p.nsub ? jj : 0) * hkv;
      const int sph = __shfl_sync(0xffffffffu, phys, src);
      const int sof = __shfl_sync(0xffffffffu, off, src);
      const bool sact = __shfl_sync(0xffffffffu, active ? 1 : 0, src) != 0;
      if (jj < p.nsub && sact)
        load4(st + tens * kKVBytes + half * kKVHalf + src * kTileBytes, tens ? &tm_v : &tm_k, &full[s],
                    half * 64, sof, 0, sph);
    } else if (active) {
      uint8_t* kd = st + lane * kTileBytes;
      uint8_t* vd = st + kKVBytes + lane * kTileBytes;
      load4(kd, &tm_k, &full[s], 0, head, off, phys);
      load4(kd + kKVHalf, &tm_k, &full[s], 64, head, off, phys);
      load4(vd, &tm_v, &full[s], 0, head, off, phys);
      load4(vd + kKVHalf, &tm_v, &full[s], 64, head, off, phys);
    }
  }
  // On an early exit, let the copies this warp issued land before the CTA
  // releases its shared memory (bounded).
  if (k < nu) {
    for (int kk = (k > stages ? k - stages : 0); kk < k; ++kk) {
      uint32_t ph;
      const int s = stage_of<kStages>(kk, stages, ph);
      if (kk % nprod == pid) mbar_wait(&full[s], ph, nullptr, 0);
    }
  }
}

// A consumer warp (0..7).
template <int kStages, bool kPrefix>
__device__ __forceinline__ void consume(const Params& p, uint8_t* smem, uint64_t* full, uint64_t* empty,
                                        const StageDesc* descs, const uint8_t* zero_row, uint64_t* mg_full,
                                        uint64_t* mg_empty, float* merge, long long n_units, int warp, int lane,
                                        int stages = kStages) {
  const int hkv = p.hkv;
  const int w = warp;
  const int j = w / hkv;
  const int h = w - j * hkv;
  const int G = p.group;
  const int g = lane >> 2;
  const int tq = lane & 3;
  const float sl2 = p.scale_log2;
  const float NEG_INF = -__int_as_float(0x7f800000);

  float o[8][4];
  float m0 = NEG_INF, m1 = NEG_INF, l0 = 0.f, l1 = 0.f;
  uint32_t qf[8][2];
  int seg_ends = 0;  // segment ends seen (phase of the merge barriers)

  const int nu = static_cast<int>(n_units);
  for (int k = 0; k < nu; ++k) {
    uint32_t ph;
    const int s = stage_of<kStages>(k, stages, ph);
    if (!mbar_wait(&full[s], ph, p.err, LA_DEVERR_WAIT_TIMEOUT)) return;
    const StageDesc d = descs[s];
    uint8_t* st = smem + s * p.stage_bytes;

    if (d.flags & kFlagFirst) {
      m0 = m1 = NEG_INF;
      l0 = l1 = 0.f;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
      // Q^T B-fragments for the 8 k-steps (128 dims); rows n >= G read zeros.
      const uint8_t* qs = st + 2 * kKVBytes;
      const int n = lane & 7;
      const int mq = lane >> 3;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int chunk_all = 4 * kk + mq;  // 16-byte chunk index over 128 dims
        const int half = chunk_all >> 3;
        const int chunk = chunk_all & 7;
        uint32_t addr;
        if (n < G) {
          const int row = h * G + n;
          addr = smem_u32(qs + half * p.q_half_bytes) + swz128(row, chunk);
        } else {
          addr = smem_u32(zero_row);
        }
        uint32_t r[4];
        ldmatrix_x4(r, addr);
        qf[2 * kk][0] = r[0];
        qf[2 * kk][1] = r[1];
        qf[2 * kk + 1][0] = r[2];
        qf[2 * kk + 1][1] = r[3];
      }
    }

    const int t0 = d.tok0 + kSub * j;
    int valid = d.ctx - t0;
    valid = valid < 0 ? 0 : (valid > kSub ? kSub : valid);
    if (valid > 0) {
      const uint8_t* ks = st + w * kTileBytes;  // + half * kKVHalf
      uint8_t* vs = st + kKVBytes + w * kTileBytes;
      // S^T = K Q^T (16 tokens x 8 query columns)
      float sacc[4] = {0.f, 0.f, 0.f, 0.f};
      {
        const int mq = lane >> 3;
        const int r = (lane & 7) + ((mq & 1) << 3);
        const uint32_t kbase = smem_u32(ks);
#pragma unroll
        for (int kstep = 0; kstep < 8; ++kstep) {
          const int half = kstep >> 2;
          const int chunk = ((kstep & 3) << 1) + (mq >> 1);
          uint32_t a[4];
          ldmatrix_x4(a, kbase + half * kKVHalf + swz128(r, chunk));
          mma_bf16_16816(sacc, a, qf[kstep][0], qf[kstep][1]);
        }
      }
      // Mask, online softmax (columns 2tq, 2tq+1; tokens g, g+8).
      const bool v0 = g < valid, v1 = (g + 8) < valid;
      const float x0 = v0 ? sacc[0] * sl2 : NEG_INF;
      const float x1 = v0 ? sacc[1] * sl2 : NEG_INF;
      const float x2 = v1 ? sacc[2] * sl2 : NEG_INF;
      const float x3 = v1 ? sacc[3] * sl2 : NEG_INF;
      const float mn0 = fmaxf(m0, warp_max_g(fmaxf(x0, x2)));
      const float mn1 = fmaxf(m1, warp_max_g(fmaxf(x1, x3)));
      const float a0 = ex2(m0 - mn0), a1 = ex2(m1 - mn1);
      m0 = mn0;
      m1 = mn1;
      const float p0 = ex2(x0 - mn0), p1 = ex2(x1 - mn1), p2 = ex2(x2 - mn0), p3 = ex2(x3 - mn1);
      l0 = l0 * a0 + (p0 + p2);
      l1 = l1 * a1 + (p1 + p3);
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        o[mt][0] *= a0;
        o[mt][1] *= a1;
        o[mt][2] *= a0;
        o[mt][3] *= a1;
      }
      const uint32_t pb0 = movmatrix_trans(pack_bf16x2(p0, p1));
      const uint32_t pb1 = movmatrix_trans(pack_bf16x2(p2, p3));
      if (valid < kSub) {
        // Rows past the sequence end may hold anything (even NaN): zero them so
        // that P = 0 cannot meet a non-finite V in the MMA.
        for (int i = lane; i < (kSub - valid) * 16; i += 32) {
          const int row = valid + (i >> 4);
          const int half = (i >> 3) & 1;
          const int chunk = i & 7;
          *reinterpret_cast<uint4*>(vs + half * kKVHalf + row * 128 + chunk * 16) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      // O^T += V^T P^T
      {
        const int mq = lane >> 3;
        const int r = (lane & 7) + ((mq >> 1) << 3);  // token row
        const uint32_t vbase = smem_u32(vs);
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          const int dd = mt * 16 + ((mq & 1) << 3);
          const int half = dd >> 6;
          const int chunk = (dd & 63) >> 3;
          uint32_t a[4];
          ldmatrix_x4_trans(a, vbase + half * kKVHalf + swz128(r, chunk));
          mma_bf16_16816(o[mt], a, pb0, pb1);
        }
      }
      if (valid < kSub) fence_proxy_async_smem();  // generic writes before the next TMA into this stage
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);

    if (d.flags & kFlagLast) {
      float L0 = warp_sum_g(l0), L1 = warp_sum_g(l1);
      // kPrefix: a sum that is NaN counts, so that it reaches the result
      auto some = [](float l) { return kPrefix ? l != 0.f : l > 0.f; };
      const int c0 = 2 * tq, c1 = 2 * tq + 1;
      bool writer = true;
      if (p.nsub > 1) {
        // Several warps hold partial states of the same kv head (one per
        // sub-chunk j). They park them in shared memory and one of them
        // merges them, so every segment leaves one state per head, as with
        // nsub == 1. The merging warp rotates with the segment end (j =
        // seg_ends % nsub), so the merges of a CTA's many short sequences
        // (the KV-head-sharded rank crosses ~7 per CTA) are shared by the
        // warps instead of all landing on j = 0, whose lag held back every
        // stage's release. The merger folds the states in sub-chunk order
        // 0, 1, ..., nsub-1 whoever it is, so the result does not depend on
        // which warp merges.
        const int TQ = (G + 1) >> 1;  // lanes (per g) that hold real columns
        const uint32_t par = static_cast<uint32_t>(seg_ends & 1);
        const int jm = seg_ends & (p.nsub - 1);  // nsub is a power of two
        if (!mbar_wait(mg_empty, par ^ 1u, p.err, LA_DEVERR_WAIT_TIMEOUT)) return;
        if (tq < TQ) {
          float* slot = merge + ((w * TQ + tq) * 8 + g) * 36;
          slot[0] = m0;
          slot[1] = m1;
          slot[2] = L0;
          slot[3] = L1;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) slot[4 + mt * 4 + r] = o[mt][r];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(mg_full);
        writer = (j == jm);
        if (writer) {
          if (!mbar_wait(mg_full, par, p.err, LA_DEVERR_WAIT_TIMEOUT)) return;
          if (tq < TQ) {
            if (jm != 0) {  // start from sub-chunk 0's state (this warp's own is in its slot)
              const float* sl = merge + ((h * TQ + tq) * 8 + g) * 36;
              m0 = sl[0];
              m1 = sl[1];
              L0 = sl[2];
              L1 = sl[3];
#pragma unroll
              for (int mt = 0; mt < 8; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[mt][r] = sl[4 + mt * 4 + r];
            }
            for (int jj = 1; jj < p.nsub; ++jj) {
              const float* sl = merge + (((jj * hkv + h) * TQ + tq) * 8 + g) * 36;
              const float om0 = sl[0], om1 = sl[1], oL0 = sl[2], oL1 = sl[3];
              const float n0 = fmaxf(m0, om0), n1 = fmaxf(m1, om1);
              // a side with no keys (m = -inf) contributes nothing
              const float a0 = (m0 == NEG_INF) ? 0.f : ex2(m0 - n0), b0 = (om0 == NEG_INF) ? 0.f : ex2(om0 - n0);
              const float a1 = (m1 == NEG_INF) ? 0.f : ex2(m1 - n1), b1 = (om1 == NEG_INF) ? 0.f : ex2(om1 - n1);
#pragma unroll
              for (int mt = 0; mt < 8; ++mt) {
                o[mt][0] = o[mt][0] * a0 + sl[4 + mt * 4 + 0] * b0;
                o[mt][1] = o[mt][1] * a1 + sl[4 + mt * 4 + 1] * b1;
                o[mt][2] = o[mt][2] * a0 + sl[4 + mt * 4 + 2] * b0;
                o[mt][3] = o[mt][3] * a1 + sl[4 + mt * 4 + 3] * b1;
              }
              L0 = L0 * a0 + oL0 * b0;
              L1 = L1 * a1 + oL1 * b1;
              m0 = n0;
              m1 = n1;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(mg_empty);
        }
        ++seg_ends;
      }
      if (writer && (d.flags & kFlagWhole)) {
        const float i0 = L0 > 0.f ? 1.f / L0 : 0.f;
        const float i1 = L1 > 0.f ? 1.f / L1 : 0.f;
        {
          __nv_bfloat16* ob = p.out + static_cast<long long>(d.b) * p.out_b_stride;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            const int d0 = mt * 16 + g;
            if (c0 < G) {
              __nv_bfloat16* oh = ob + static_cast<long long>(h * G + c0) * p.out_h_stride;
              oh[d0] = __float2bfloat16_rn(o[mt][0] * i0);
              oh[d0 + 8] = __float2bfloat16_rn(o[mt][2] * i0);
            }
            if (c1 < G) {
              __nv_bfloat16* oh = ob + static_cast<long long>(h * G + c1) * p.out_h_stride;
              oh[d0] = __float2bfloat16_rn(o[mt][1] * i1);
              oh[d0 + 8] = __float2bfloat16_rn(o[mt][3] * i1);
            }
          }
        }
        if (p.lse_out && g == 0) {
          const float ln2 = 0.6931471805599453f;
          if (c0 < G) p.lse_out[static_cast<long long>(d.b) * p.hq + h * G + c0] = some(L0) ? (m0 + __log2f(L0)) * ln2 : NEG_INF;
          if (c1 < G) p.lse_out[static_cast<long long>(d.b) * p.hq + h * G + c1] = some(L1) ? (m1 + __log2f(L1)) * ln2 : NEG_INF;
        }
      } else if (writer) {
        float* po = p.part_o + static_cast<long long>(d.slot) * p.hq * kD;
        const float i0 = L0 > 0.f ? 1.f / L0 : 0.f;
        const float i1 = L1 > 0.f ? 1.f / L1 : 0.f;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          const int d0 = mt * 16 + g;
          if (c0 < G) {
            float* oh = po + (h * G + c0) * kD;
            oh[d0] = o[mt][0] * i0;
            oh[d0 + 8] = o[mt][2] * i0;
          }
          if (c1 < G) {
            float* oh = po + (h * G + c1) * kD;
            oh[d0] = o[mt][1] * i1;
            oh[d0 + 8] = o[mt][3] * i1;
          }
        }
        if (g == 0) {
          float* pl = p.part_lse + static_cast<long long>(d.slot) * p.hq;
          if (c0 < G) pl[h * G + c0] = some(L0) ? m0 + __log2f(L0) : NEG_INF;
          if (c1 < G) pl[h * G + c1] = some(L1) ? m1 + __log2f(L1) : NEG_INF;
        }
      }
    }
  }
}

// ------------------------------------------------------------------ host
// A checked call: tensor maps and the kernel's parameters but for where
// partials go, and the shared memory that merging sub-chunks takes.
struct Call {
  CUtensorMap q, k, v, k1, v1;
  Params p;
  int merge_bytes;
};

// The arguments of la_paged_decode, checked before anything else. LA_OK with
// a batch of 0 leaves the call empty.
int prepare_call(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache,
                 const void* v_cache, int64_t kv_block_stride, int64_t kv_token_stride, int64_t kv_head_stride,
                 int64_t num_blocks, int block_size, const int32_t* block_table, int64_t bt_seq_stride,
                 int max_blocks_per_seq, const int32_t* cache_seqlens, int batch, int num_q_heads, int num_kv_heads,
                 int head_dim, float softmax_scale, void* out, int64_t out_batch_stride, int64_t out_head_stride,
                 float* softmax_lse, int* dev_error, Call* call);

}  // namespace decode
}  // namespace la
