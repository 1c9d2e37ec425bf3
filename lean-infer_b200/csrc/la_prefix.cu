// Paged GQA decode attention for a batch whose rows share long prefixes, sm_100a.
//
// out[b, h] = softmax(scale * q[b, h] . K_b^T) V_b over keys 0..cache_seqlens[b]-1
// of row b, read through block_table[b]: what la_paged_decode computes. Rows
// cu_prefix_rows[g] .. cu_prefix_rows[g+1]-1 hold the same pages for their
// first keys, so the softmax is taken in two parts, joined by their maxima and
// sums: over the shared keys for all rows of a group at once, as matrix
// products (prefix_kernel), and over each row's own keys (the decode kernel of
// la_decode.cu). combine_kernel joins the parts of every row.
//
// prefix_kernel. For one kv head the group's rows x query heads of the kv head
// are the rows of Q; with 128-key tiles of K and V,
//   S = Q K^T,  P = exp2(S * scale * log2 e - m),  O += P V,  l += sum P
// run on tcgen05 with fp32 accumulators in tensor memory, m the running row
// maximum. Bound by HBM (the prefix once) while a kv head has at most ~256
// query rows, by the tensor cores and the exponentials above that.
//
// Work. An item is (group, kv head, pair of 128-row tiles); both tiles use
// each K/V tile that is staged. Where only one tile is left over, its two
// accumulators take the even and the odd key tiles instead, so that one
// tile's products still run while the other's exponentials do. A step is two
// tile products either way: one key tile of a pair of row tiles, or two key
// tiles of a single one. The steps of all items, laid end to end, are cut into
// equal ranges, one per CTA (one CTA per SM), whatever the number of groups;
// an item's part in a range is a segment, which leaves normalised fp32 O rows
// and base-2 logarithms of its sums. Everything is found on the device, so the
// launch does not depend on the groups.
//
// CTA, 16 warps: 0-3 and 4-7 softmax of tile 0 and 1 (a thread per row, the S
// row in registers), 8-11 store the segments' O, 12 issues the products, 13
// the TMA loads. Tensor memory: S0 S1 O0 O1, 128 columns each; P over S.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "la_groups.cuh"
#include "la_internal.h"
#include "la_ptx.cuh"

namespace la {
namespace prefix {

constexpr int kD = 128;
constexpr int kRows = 128;             // query rows per tile
constexpr int kKeys = 128;             // keys per K/V tile
constexpr int kHalf = 128 * 128;       // 64 dims of 128 rows: 16 KB
constexpr int kTile = 2 * kHalf;
constexpr int kStages = 4;             // K/V tiles in flight
constexpr int kThreads = 512;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;        // O_t at kColO + 128 t; S_t at 128 t
constexpr uint32_t kIdescQK = idesc_bf16_f32(128, kKeys, false, false);
constexpr uint32_t kIdescPV = idesc_bf16_f32(128, 128, false, true);
constexpr int kRegSoftmax = 160, kRegStore = 88, kRegOther = 104;
static_assert(256 * kRegSoftmax + 128 * kRegStore + 128 * kRegOther <= kThreads * 128,
              "the register split must fit in the registers the CTA is launched with");
// Shared memory: Q0 Q1 | K/V ring | staging of O (4 KB per storing warp) |
// row sums and maxima | barriers and the CTA's range.
constexpr int kOffKV = 2 * kTile;
constexpr int kOffStage = kOffKV + kStages * kTile;
constexpr int kStageBytes = 32 * 128;
constexpr int kOffStats = kOffStage + 4 * kStageBytes;
constexpr int kOffBar = kOffStats + 2 * 2 * kRows * 4;
constexpr int kOffWalk = kOffBar + 256;  // of the softmax warps, kept out of their registers
constexpr int kWalkBytes = 112;
constexpr size_t kSmemBytes = kOffWalk + 8 * kWalkBytes + 1024;  // + alignment to 1024 bytes at run time
static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");

struct Params {
  PrefixGroups groups;
  const int* table;
  long long table_stride;
  int max_blocks;
  int num_blocks;
  int box_keys;  // keys per TMA box, a power of two that divides the block size
  int hkv, group;
  int per_tile;   // sequences per row tile: 128 / group
  float scale_log2;
  float* part_o;    // [rows][D]
  float* part_lse;  // [rows], base 2
  int* err;
};

// How the steps of a group lie: kv heads one after another, in each the pairs
// of row tiles, the single tile last.
struct Shape {
  int tiles;    // key tiles
  int pairs;    // of row tiles, the single one included
  int single;   // 1: the last has one tile
  int per_head; // steps of one kv head
};

__device__ __forceinline__ Shape shape_of(const PrefixGroup& g, int per_tile) {
  Shape s;
  const int row_tiles = (g.rows + per_tile - 1) / per_tile;
  s.tiles = (g.keys + kKeys - 1) / kKeys;
  s.pairs = (row_tiles + 1) >> 1;
  s.single = row_tiles & 1;
  s.per_head = (s.pairs - s.single) * s.tiles + (s.single ? (s.tiles + 1) >> 1 : 0);
  return s;
}

__device__ __forceinline__ int steps_of(const Params& p, int g) {
  const PrefixGroup r = prefix_group(p.groups, g);
  return r.keys > 0 ? p.hkv * shape_of(r, p.per_tile).per_head : 0;
}

// The even split of T steps or units over at most `grid` CTAs, each with some.
__device__ __forceinline__ long long parts_of(long long T, int grid) { return T < grid ? (T > 0 ? T : 1) : grid; }
__device__ __forceinline__ long long part_start(long long c, long long T, long long G) { return c * T / G; }
__device__ __forceinline__ int part_of(long long x, long long T, long long G) {
  return static_cast<int>(((x + 1) * G - 1) / T);
}

// First partial row of item (g, h, r) in CTA c. An item's segments take up to
// 256 rows, those of two accumulators; from one segment to the next along the
// line of steps the item, the CTA or both go up, the item by at least the rows
// that one segment of it takes.
__device__ __forceinline__ int part_row(const Params& p, const PrefixGroup& g, int h, int r, int c) {
  return 2 * p.group * (p.hkv * g.first + h * g.rows + r * 2 * p.per_tile) + 2 * kRows * c;
}

// The CTA's range of steps and where it begins.
struct Range {
  long long u0, u1;  // steps
  long long before;  // steps before group g0
  int g0;
};

// Segments of the CTA's range, one after another (the same in every thread).
struct Walk {
  int left;  // steps of the range not yet taken
  int g, h, r, s;
  PrefixGroup grp;
  Shape shp;
};

struct Segment {
  int first, rows;  // sequences of the item: first row of the batch, how many
  int h;
  int table_row;    // of the batch: the group's first
  int two;          // two row tiles
  int tile0, tiles; // key tiles
  int keys;         // of the group
  int row0;         // first partial row
};

__device__ __forceinline__ void walk_group(const Params& p, Walk& w, int g) {
  w.g = g;
  w.grp = prefix_group(p.groups, g);
  w.shp = shape_of(w.grp, p.per_tile);
}

__device__ __forceinline__ void walk_start(const Params& p, const Range& R, Walk& w) {
  w.left = static_cast<int>(R.u1 - R.u0);
  if (w.left <= 0) return;
  walk_group(p, w, R.g0);
  const int x = static_cast<int>(R.u0 - R.before);
  w.h = x / w.shp.per_head;
  const int y = x - w.h * w.shp.per_head;
  w.r = min(y / w.shp.tiles, w.shp.pairs - 1);
  w.s = y - w.r * w.shp.tiles;
}

__device__ __forceinline__ bool walk_next(const Params& p, Walk& w, Segment& e) {
  if (w.left <= 0) return false;
  const bool one = w.shp.single && w.r == w.shp.pairs - 1;
  const int steps = one ? (w.shp.tiles + 1) >> 1 : w.shp.tiles;
  const int n = min(steps - w.s, w.left);
  const int seq0 = w.r * 2 * p.per_tile;
  e.first = w.grp.first + seq0;
  e.rows = min(w.grp.rows - seq0, 2 * p.per_tile);
  e.h = w.h;
  e.table_row = w.grp.first;
  e.two = one ? 0 : 1;
  e.tile0 = one ? 2 * w.s : w.s;
  e.tiles = one ? min(2 * n, w.shp.tiles - e.tile0) : n;
  e.keys = w.grp.keys;
  e.row0 = part_row(p, w.grp, w.h, w.r, blockIdx.x);
  w.left -= n;
  w.s += n;
  if (w.s == steps && w.left > 0) {
    w.s = 0;
    if (++w.r == w.shp.pairs) {
      w.r = 0;
      if (++w.h == p.hkv) {
        w.h = 0;
        int g = w.g;
        do {
          if (++g >= p.groups.n) {  // groups changed under the kernel
            w.left = 0;
            return true;
          }
          walk_group(p, w, g);
        } while (w.grp.keys == 0);
      }
    }
  }
  return true;
}

static_assert(sizeof(Walk) <= 64 && sizeof(Segment) + 64 <= kWalkBytes, "a softmax warp's walk");

// Key tiles that tile t's accumulator takes, and the i-th of them.
__device__ __forceinline__ int tiles_of(const Segment& e, int t) { return e.two ? e.tiles : (e.tiles + 1 - t) >> 1; }
// Query rows of tile t, and its first partial row.
__device__ __forceinline__ int rows_of(const Params& p, const Segment& e, int t) {
  const int seqs = e.two && t ? e.rows - p.per_tile : min(e.rows, p.per_tile);
  return seqs * p.group;
}

__device__ __forceinline__ uint64_t desc_kmajor(const uint8_t* tile) {
  return smem_desc_sw128(smem_u32(tile), 16, 1024);
}
__device__ __forceinline__ uint64_t desc_v(const uint8_t* tile) { return smem_desc_sw128(smem_u32(tile), kHalf, 1024); }

template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__global__ void __launch_bounds__(kThreads, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + kOffKV;
  float* stats = reinterpret_cast<float*>(smem + kOffStats);  // [tile][l | m][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* q_full = bars + 0;     // a segment's Q landed
  uint64_t* q_empty = bars + 1;    // its last S done
  uint64_t* kv_full = bars + 2;    // [kStages]
  uint64_t* kv_empty = bars + 6;   // [kStages]
  uint64_t* s_full = bars + 10;    // [2] S_t written
  uint64_t* s_free = bars + 12;    // [2] P_t V done
  uint64_t* p_full = bars + 14;    // [2] P_t written (128 arrivals)
  uint64_t* o_empty = bars + 16;   // [2] O_t read by the storing warps (128)
  uint64_t* st_full = bars + 18;   // [2] row sums and maxima of tile t written (128)
  uint64_t* st_empty = bars + 20;  // [2] ... and read (128)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
  Range* range = reinterpret_cast<Range*>(bars + 24);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int wg = warp >> 2;
  const float NEG_INF = -__int_as_float(0x7f800000);

  // Barriers and tensor memory: nothing that a kernel before this one writes.
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_empty[i], 128);
      mbar_init(&st_full[i], 128);
      mbar_init(&st_empty[i], 128);
    }
    fence_barrier_init();
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  if (warp == 13 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  grid_dependency_wait();
  // What came before is done and visible, so the row-by-row pass behind this
  // grid may start wherever an SM is free: it reads nothing written here.
  grid_launch_dependents();
  if (warp == 14) {
    // all steps, then the group that holds the CTA's first one
    const int n = p.groups.n;
    long long T = 0;
    for (int b = 0; b < n; b += 32) {
      const int g = b + lane;
      if (blockIdx.x == 0 && g < n && p.err) {
        const int lo = p.groups.cu[g], hi = p.groups.cu[g + 1];
        if (lo < 0 || hi < lo || hi > p.groups.batch) atomicCAS(p.err, 0, LA_DEVERR_PREFIX);
      }
      long long s = g < n ? steps_of(p, g) : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      T += s;
    }
    const long long G = parts_of(T, gridDim.x);
    const long long u0 = blockIdx.x < G ? part_start(blockIdx.x, T, G) : T;
    const long long u1 = blockIdx.x < G ? part_start(blockIdx.x + 1, T, G) : T;
    long long acc = 0, before = 0;
    int g0 = 0;
    for (int b = 0; u0 < u1 && b < n; b += 32) {
      const int g = b + lane;
      const int s = g < n ? steps_of(p, g) : 0;
      long long incl = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, acc + incl > u0);
      if (hit) {
        const int src = __ffs(hit) - 1;
        g0 = b + src;
        before = acc + __shfl_sync(0xffffffffu, incl - s, src);
        break;
      }
      acc += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) *range = Range{u0, u1, before, g0};
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (range->u0 >= range->u1) {  // no work
    if (warp == 12) tmem_dealloc(tmem, kTmemCols);
    return;
  }

  auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.err, LA_DEVERR_WAIT_TIMEOUT));
  };
  if (wg < 2) {
    regs_inc<kRegSoftmax>();
    // ------------------------------------------------------------ softmax of tile t
    const int t = wg;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t colS = t * 128, colO = kColO + t * 128;
    const float sl2 = p.scale_log2;
    Walk& w = *reinterpret_cast<Walk*>(smem + kOffWalk + warp * kWalkBytes);
    Segment& e = *reinterpret_cast<Segment*>(smem + kOffWalk + warp * kWalkBytes + 64);
    {
      Walk x;
      walk_start(p, *range, x);
      if (lane == 0) w = x;
      __syncwarp();
    }
    auto next = [&]() -> bool {
      Walk x = w;
      Segment y{};
      const bool more = walk_next(p, x, y);
      __syncwarp();  // every lane has read the old state
      if (lane == 0) {
        w = x;
        e = y;
      }
      __syncwarp();
      return more;
    };
    uint32_t seen = 0, nst = 0;  // S tiles, segments with statistics
    bool ok = true;
    while (ok && next()) {
      const int n = tiles_of(e, t);
      if (n == 0) continue;
      const bool active = quarter * 32 < rows_of(p, e, t);  // rows of this warp
      float m = NEG_INF, l = 0.f;
      for (int j = 0; j < n; ++j, ++seen) {
        if (!(ok = wait_all(&s_full[t], seen & 1))) break;
        if (!active) {
          mbar_arrive(&p_full[t]);
          continue;
        }
        tc_fence_after();
        float sv[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(taddr + colS + c * 32, sv[c]);
        tc_wait_ld();
        // keys of this tile, 128 but for the prefix's last
        const int nvis = e.keys - (e.tile0 + (e.two ? j : 2 * j + t)) * kKeys;
        float mx[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) mx[a] = NEG_INF;
        if (nvis >= kKeys) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int x = 0; x < 32; x += 2) mx[(x >> 1) & 7] = fmax3(mx[(x >> 1) & 7], sv[c][x], sv[c][x + 1]);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const float x0 = (c * 32 + x < nvis) ? sv[c][x] : NEG_INF;
              const float x1 = (c * 32 + x + 1 < nvis) ? sv[c][x + 1] : NEG_INF;
              sv[c][x] = x0;
              sv[c][x + 1] = x1;
              mx[(x >> 1) & 7] = fmax3(mx[(x >> 1) & 7], x0, x1);
            }
        }
        const float mt = fmaxf(fmax3(mx[0], mx[1], mx[2]), fmax3(fmax3(mx[3], mx[4], mx[5]), mx[6], mx[7])) * sl2;
        // The reference rises only by more than 2^8 (P stays below that, l
        // far below overflow), so that O is seldom rescaled.
        const float m_new = (mt > m + 8.f) ? mt : m;
        const float m_ref = (m_new == NEG_INF) ? 0.f : m_new;
        const float alpha = ex2(m - m_ref);
        const uint64_t sl2x2 = f2_pack(sl2, sl2), negm2 = f2_pack(-m_ref, -m_ref);
        uint64_t acc2[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) acc2[a] = 0ull;
        // P rounded to bf16, the type of V, for the product; l sums it unrounded.
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          float pk[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            const uint64_t y2 =
                f2_fma(f2_pack(sv[2 * c2 + (x >> 4)][(x & 15) * 2], sv[2 * c2 + (x >> 4)][(x & 15) * 2 + 1]), sl2x2, negm2);
            float e0, e1;
            f2_unpack(y2, e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            acc2[x & 3] = f2_add(acc2[x & 3], f2_pack(e0, e1));
            pk[x] = __uint_as_float(pack_bf16x2(e0, e1));
          }
          tmem_st32(taddr + colS + c2 * 32, pk);
        }
        float ps[8];
#pragma unroll
        for (int a = 0; a < 4; ++a) f2_unpack(acc2[a], ps[2 * a], ps[2 * a + 1]);
        l = l * alpha + (((ps[0] + ps[1]) + (ps[2] + ps[3])) + ((ps[4] + ps[5]) + (ps[6] + ps[7])));
        // O_t holds the products of the tiles before: S_t(j) was issued behind
        // them, and the next waits for this P.
        if (j >= 1 && __any_sync(0xffffffffu, m_new != m)) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float o[32];
            tmem_ld32(taddr + colO + c * 32, o);
            tc_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] *= alpha;
            tmem_st32(taddr + colO + c * 32, o);
          }
        }
        m = m_new;
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      if (!(ok = wait_all(&st_empty[t], (nst & 1) ^ 1u))) break;
      stats[(t * 2 + 0) * kRows + row] = l;
      stats[(t * 2 + 1) * kRows + row] = m;
      mbar_arrive(&st_full[t]);
      ++nst;
    }
  } else if (wg == 2) {
    regs_dec<kRegStore>();
    // ------------------------------------------------------------ segments' results
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    uint8_t* stage = smem + kOffStage + quarter * kStageBytes;
    Walk w;
    Segment e{};
    walk_start(p, *range, w);
    uint32_t done[2] = {0, 0};  // products P_t V, this segment's included
    uint32_t segs[2] = {0, 0};
    bool ok = true;
    while (ok && walk_next(p, w, e)) {
      for (int t = 0; t < 2 && ok; ++t) {
        const int rows = rows_of(p, e, t);
        const int n = tiles_of(e, t);
        const int row0 = e.row0 + t * rows_of(p, e, 0);
        if (n == 0) {  // a single key tile: none for the second accumulator
          if (row < rows) p.part_lse[row0 + row] = NEG_INF;
          continue;
        }
        done[t] += n;
        if (!(ok = wait_all(&st_full[t], segs[t] & 1))) break;
        const float l = stats[(t * 2 + 0) * kRows + row];
        const float m = stats[(t * 2 + 1) * kRows + row];
        mbar_arrive(&st_empty[t]);
        if (!(ok = wait_all(&s_free[t], (done[t] - 1) & 1))) break;  // the last product
        tc_fence_after();
        ++segs[t];
        if (quarter * 32 >= rows) {
          mbar_arrive(&o_empty[t]);
          continue;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (row < rows) p.part_lse[row0 + row] = l == 0.f ? NEG_INF : m + __log2f(l);
        // 32 columns at a time through the staging buffer (16-byte chunks
        // XORed by row), so that a store instruction writes 4 rows of 128 bytes.
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float o[32];
          tmem_ld32(taddr + kColO + t * 128 + c * 32, o);
          tc_wait_ld();
          if (c == 3) {
            tc_fence_before();
            mbar_arrive(&o_empty[t]);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x)
            *reinterpret_cast<float4*>(stage + lane * 128 + ((x ^ (lane & 7)) << 4)) =
                make_float4(o[4 * x] * inv, o[4 * x + 1] * inv, o[4 * x + 2] * inv, o[4 * x + 3] * inv);
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int r = x * 4 + (lane >> 3), ch = lane & 7;
            const float4 u = *reinterpret_cast<const float4*>(stage + r * 128 + ((ch ^ (r & 7)) << 4));
            if (quarter * 32 + r < rows)
              *reinterpret_cast<float4*>(p.part_o + static_cast<long long>(row0 + quarter * 32 + r) * kD + c * 32 +
                                         ch * 4) = u;
          }
          __syncwarp();
        }
      }
    }
  } else {
    regs_dec<kRegOther>();
    Walk w;
    Segment e{};
    if (warp == 13) {
      // ---------------------------------------------------------- TMA producer
      // Per segment Q, then the tiles in the order the products use them:
      // `lead` K tiles, then V(i), K(i + lead) in turn; lead is 1 for two row
      // tiles, 2 for the two accumulators of one.
      walk_start(p, *range, w);
      int kq = 0;
      uint32_t pos = 0;  // tiles loaded
      bool ok = true;
      const int boxes = kKeys / p.box_keys;
      auto load = [&](const CUtensorMap* tm, int tile) -> bool {
        const int st = pos % kStages;
        if (!wait_all(&kv_empty[st], ((pos / kStages) & 1) ^ 1u)) return false;
        uint8_t* dst = sKV + st * kTile;
        if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], kTile);
        __syncwarp();
        if (lane < 2 * boxes) {  // a box per lane: 64 dims of box_keys keys of one page
          const int key = tile * kKeys + (lane >> 1) * p.box_keys;
          // keys behind the prefix, and pages outside the pool, come from
          // block num_blocks, outside the tensor map: zeros
          int blk = p.num_blocks, off = 0;
          if (key < e.keys) {
            const int lb = p.groups.bs_shift >= 0 ? key >> p.groups.bs_shift : key / p.groups.block_size;
            off = key - lb * p.groups.block_size;
            const int id = __ldg(p.table + static_cast<long long>(e.table_row) * p.table_stride + lb);
            if (id >= 0 && id < p.num_blocks)
              blk = id;
            else if (p.err)
              atomicCAS(p.err, 0, LA_DEVERR_BLOCK_ID);
          }
          tma_load_4d(dst + (lane & 1) * kHalf + (lane >> 1) * p.box_keys * 128, tm, &kv_full[st], (lane & 1) * 64, off,
                      e.h, blk);
        }
        __syncwarp();
        ++pos;
        return true;
      };
      while (ok && walk_next(p, w, e)) {
        if (!(ok = wait_all(q_empty, (kq & 1) ^ 1u))) break;
        if (lane == 0) {
          const uint32_t half = 128u * p.group * p.per_tile;
          mbar_arrive_expect_tx(q_full, (1 + e.two) * 2 * half);
          for (int t = 0; t < 1 + e.two; ++t)
            for (int x = 0; x < 2; ++x)
              tma_load_3d(sQ + t * kTile + x * kHalf, &tm_q, q_full, x * 64, e.h * p.group, e.first + t * p.per_tile);
        }
        __syncwarp();
        ++kq;
        const int lead = 2 - e.two;
        for (int i = 0; ok && i < min(lead, e.tiles); ++i) ok = load(&tm_k, e.tile0 + i);
        for (int i = 0; ok && i < e.tiles; ++i) {
          ok = load(&tm_v, e.tile0 + i);
          if (ok && i + lead < e.tiles) ok = load(&tm_k, e.tile0 + i + lead);
        }
      }
      if (!ok && lane == 0) {  // early exit: let the copies already issued land (bounded)
        for (uint32_t u = (pos > kStages ? pos - kStages : 0); u < pos; ++u)
          mbar_wait(&kv_full[u % kStages], (u / kStages) & 1, nullptr, 0);
        if (kq > 0) mbar_wait(q_full, (kq - 1) & 1, nullptr, 0);
      }
      __syncwarp();
    } else if (warp == 12) {
      // ---------------------------------------------------------- products (lane 0 issues)
      // S_t over P_t is issued right behind the product that reads P_t: the
      // tensor core executes one thread's products in order.
      walk_start(p, *range, w);
      int kq = 0;
      uint32_t pos = 0;
      uint32_t cp[2] = {0, 0}, segs[2] = {0, 0};
      bool ok = true;
      auto wait_full = [&](uint32_t x) -> bool { return wait_all(&kv_full[x % kStages], (x / kStages) & 1); };
      auto issue_s = [&](int t, int q, uint32_t x) {
        if (lane == 0) {
          const uint64_t ad = desc_kmajor(sQ + q * kTile), bd = desc_kmajor(sKV + (x % kStages) * kTile);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const int o = ((ks >> 2) * kHalf + (ks & 3) * 32) >> 4;
            umma_f16_ss(tmem + t * 128, ad + o, bd + o, kIdescQK, ks > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[t]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, bool first, uint32_t x) -> bool {
        if (!wait_all(&p_full[t], cp[t] & 1)) return false;
        if (first) {  // O_t is overwritten: the previous segment's must have been read
          if (segs[t] > 0 && !wait_all(&o_empty[t], (segs[t] - 1) & 1)) return false;
          ++segs[t];
        }
        tc_fence_after();
        if (lane == 0) {
          const uint64_t vd = desc_v(sKV + (x % kStages) * kTile);
#pragma unroll
          for (int ks = 0; ks < kKeys / 16; ++ks)
            umma_f16_ts(tmem + kColO + t * 128, tmem + t * 128 + ks * 8, vd + ks * 128, kIdescPV,
                        (!first || ks > 0) ? 1u : 0u);
          umma_commit(&s_free[t]);
        }
        __syncwarp();
        ++cp[t];
        return true;
      };
      auto release = [&](uint64_t* bar) {
        if (lane == 0) umma_commit(bar);
        __syncwarp();
      };
      while (ok && walk_next(p, w, e)) {
        if (!(ok = wait_all(q_full, kq & 1))) break;
        ++kq;
        const int n = e.tiles, lead = 2 - e.two;
        for (int i = 0; ok && i < min(lead, n); ++i, ++pos) {
          if (!(ok = wait_full(pos))) break;
          if (e.two) {
            issue_s(0, 0, pos);
            issue_s(1, 1, pos);
          } else {
            issue_s(i, 0, pos);
          }
          release(&kv_empty[pos % kStages]);
        }
        if (!ok) break;
        if (n <= lead) release(q_empty);
        for (int i = 0; ok && i < n; ++i) {
          const uint32_t vp = pos++;
          const bool more = i + lead < n;
          const uint32_t kp = pos;
          if (more) ++pos;
          if (!(ok = wait_full(vp))) break;
          if (more && !(ok = wait_full(kp))) break;
          if (e.two) {
            if (!(ok = issue_pv(0, i == 0, vp))) break;
            if (more) issue_s(0, 0, kp);
            if (!(ok = issue_pv(1, i == 0, vp))) break;
            release(&kv_empty[vp % kStages]);
            if (more) issue_s(1, 1, kp);
          } else {
            if (!(ok = issue_pv(i & 1, i < 2, vp))) break;
            release(&kv_empty[vp % kStages]);
            if (more) issue_s(i & 1, 0, kp);
          }
          if (more) release(&kv_empty[kp % kStages]);
          if (more && i + 1 + lead == n) release(q_empty);  // the segment's last S
        }
      }
      __syncwarp();
    }
    // warps 14, 15: no role
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ------------------------------------------------------------------ combine
// A CTA per row, a warp per query head (heads behind the 16th in turn), lane l
// owning dims 4l..4l+3. The row's parts are those of its group's item, one per
// CTA that had a segment of it (two where the accumulators took alternate key
// tiles), and those of its own keys. Up to 32 parts per round, one per lane:
// the weights come from a warp maximum, then the O rows are read 16 at a time.
// Where they lie follows from the lengths and groups, which are final long
// before the parts are, so it is worked out before the wait for them.
constexpr int kCombineBatch = 16;
constexpr int kCombineWarps = 16;

struct CombineParams {
  PrefixGroups groups;
  const int* seqlens;
  int hq, hkv, group, per_tile;
  int grid;   // CTAs of both passes
  int tc;     // keys per unit of the row-by-row pass
  int own0;   // its first partial row
  const float* part_o;
  const float* part_lse;
  __nv_bfloat16* out;
  long long out_bs, out_hs;
  float* lse;
};

__device__ __forceinline__ int clamp_ctx(const CombineParams& p, int b) {
  const long long c = max(p.seqlens[b], 0);
  return static_cast<int>(c > p.groups.cap ? p.groups.cap : c);
}

__global__ void __launch_bounds__(32 * kCombineWarps) combine_kernel(const CombineParams p) {
  __shared__ long long red[2][kCombineWarps];
  __shared__ long long steps[2];
  const int b = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const float NEG_INF = -__int_as_float(0x7f800000);

  // All units, and those before this row.
  long long T = 0, before = 0;
  for (int x = threadIdx.x; x < p.groups.batch; x += blockDim.x) {
    const int ctx = clamp_ctx(p, x);
    const int n = ctx > 0 ? (ctx - prefix_keys(p.groups, x, ctx) + p.tc - 1) / p.tc : 0;
    T += n;
    if (x < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    T += __shfl_xor_sync(0xffffffffu, T, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) {
    red[0][warp] = T;
    red[1][warp] = before;
  }
  // All steps, and those before this row's group.
  const int ctx = clamp_ctx(p, b);
  const int gi = prefix_group_of(p.groups, b);
  Params sp;  // what steps_of reads
  sp.groups = p.groups;
  sp.hkv = p.hkv;
  sp.group = p.group;
  sp.per_tile = p.per_tile;
  if (warp == 0) {
    long long s = 0, sb = 0;
    for (int g = lane; g < p.groups.n; g += 32) {
      const int n = steps_of(sp, g);
      s += n;
      if (g < gi) sb += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      sb += __shfl_xor_sync(0xffffffffu, sb, o);
    }
    if (lane == 0) {
      steps[0] = s;
      steps[1] = sb;
    }
  }
  __syncthreads();
  T = before = 0;
  for (int x = 0; x < warps; ++x) {
    T += red[0][x];
    before += red[1][x];
  }
  const int shared = prefix_keys(p.groups, b, ctx);
  const int nb = (ctx - shared + p.tc - 1) / p.tc;
  const long long G = parts_of(T, p.grid);
  const int cf = nb > 0 ? part_of(before, T, G) : 0;
  const int own = nb > 0 ? part_of(before + nb - 1, T, G) - cf + 1 : 0;

  for (int hh = warp; hh < p.hq; hh += warps) {
    // the group's parts: CTAs pf.., `per` each, whose first row is row0
    int pn = 0, row0 = 0, per = 1, stride = 0;
    if (shared > 0) {
      const PrefixGroup g = prefix_group(p.groups, gi);
      const Shape s = shape_of(g, p.per_tile);
      const int h = hh / p.group;
      const int seq = b - g.first, r = seq / (2 * p.per_tile), in = seq - r * 2 * p.per_tile;
      const bool one = s.single && r == s.pairs - 1;
      const long long u0 = steps[1] + static_cast<long long>(h) * s.per_head + r * s.tiles;
      const int n = one ? (s.tiles + 1) >> 1 : s.tiles;
      const long long PG = parts_of(steps[0], p.grid);
      const int pf = part_of(u0, steps[0], PG), pl = part_of(u0 + n - 1, steps[0], PG);
      per = one ? 2 : 1;
      pn = (pl - pf + 1) * per;
      // rows of a tile: (sequence, query head of the kv head); the second
      // tile's, or accumulator's, behind those of the first
      const int tile = one ? 0 : in / p.per_tile;
      stride = one ? (g.rows - r * 2 * p.per_tile) * p.group : 0;
      row0 = part_row(sp, g, h, r, pf) + tile * p.per_tile * p.group + (in - tile * p.per_tile) * p.group + hh % p.group;
    }
    if (hh == warp) grid_dependency_wait();
    const int n = pn + own;
    __nv_bfloat16* out = p.out + b * p.out_bs + hh * p.out_hs + lane * 4;
    float* lse = p.lse ? p.lse + static_cast<long long>(b) * p.hq + hh : nullptr;
    if (shared == 0 && own == 1) continue;  // written by the row-by-row pass
    float m = NEG_INF, l = 0.f;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int e0 = 0; e0 < n; e0 += 32) {
      const int x = e0 + lane;
      int row = -1;
      if (x < pn)
        row = per == 2 ? row0 + (x >> 1) * 2 * kRows + (x & 1) * stride : row0 + x * 2 * kRows;
      else if (x < n)
        row = p.own0 + (b + cf + x - pn) * p.hq + hh;
      const float ls = row >= 0 ? p.part_lse[row] : NEG_INF;
      const int nr = min(n - e0, 32);
      int su[kCombineBatch];
      float4 ov[kCombineBatch];
#pragma unroll
      for (int k = 0; k < kCombineBatch; ++k) su[k] = __shfl_sync(0xffffffffu, row, k);
#pragma unroll
      for (int k = 0; k < kCombineBatch; ++k)
        ov[k] = k < nr ? *reinterpret_cast<const float4*>(p.part_o + static_cast<long long>(su[k]) * kD + lane * 4)
                       : make_float4(0.f, 0.f, 0.f, 0.f);
      // A part without keys has -inf and is left out by a test, never by a
      // weight of 0, so whatever its row holds does not count; NaN counts.
      const bool use = row >= 0 && ls != NEG_INF;
      const unsigned usem = __ballot_sync(0xffffffffu, use);
      if (usem == 0) continue;
      float mr = use ? ls : NEG_INF;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mr = fmaxf(mr, __shfl_xor_sync(0xffffffffu, mr, o));
      const float mn = fmaxf(m, mr);
      const float a = ex2(m - mn);
      const float wl = use ? ex2(ls - mn) : 0.f;
      float ws = wl;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
      l = l * a + ws;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] *= a;
      m = mn;
      for (int j0 = 0; j0 < nr; j0 += kCombineBatch) {
        if (j0 > 0) {
#pragma unroll
          for (int k = 0; k < kCombineBatch; ++k) su[k] = __shfl_sync(0xffffffffu, row, (j0 + k) & 31);
#pragma unroll
          for (int k = 0; k < kCombineBatch; ++k)
            ov[k] = j0 + k < nr
                        ? *reinterpret_cast<const float4*>(p.part_o + static_cast<long long>(su[k]) * kD + lane * 4)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int k = 0; k < kCombineBatch; ++k) {
          const float wk = __shfl_sync(0xffffffffu, wl, (j0 + k) & 31);
          if (j0 + k < nr && ((usem >> ((j0 + k) & 31)) & 1u)) {
            acc[0] += wk * ov[k].x;
            acc[1] += wk * ov[k].y;
            acc[2] += wk * ov[k].z;
            acc[3] += wk * ov[k].w;
          }
        }
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint2 v;
    v.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    v.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<uint2*>(out) = v;
    if (lse && lane == 0) *lse = l == 0.f ? NEG_INF : (m + __log2f(l)) * 0.6931471805599453f;
  }
}

// ------------------------------------------------------------------ host
// Partial rows: of the prefix pass, then of the row-by-row pass.
static int64_t prefix_rows(int64_t batch, int hq, int grid) { return 2 * batch * hq + 2 * kRows * grid; }
static int64_t own_rows(int64_t batch, int hq, int grid) { return (batch + grid) * hq; }

}  // namespace prefix

int prefix_init(int device) {
  (void)device;
  cudaError_t e = cudaFuncSetAttribute(prefix::prefix_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(prefix::kSmemBytes));
  cudaFuncAttributes a;
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, prefix::combine_kernel);
  return cuda_status(e);
}

}  // namespace la

extern "C" int la_paged_decode_shared_prefix_workspace_size(int device, int batch, int num_groups, int num_q_heads,
                                                            int num_kv_heads, int head_dim, size_t* bytes) {
  using namespace la::prefix;
  if (!bytes || batch < 0 || num_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim != kD ||
      num_kv_heads > 8 || 8 % num_kv_heads != 0 || num_q_heads % num_kv_heads != 0)
    return head_dim != kD ? LA_ERR_UNSUPPORTED : LA_ERR_INVALID_ARGUMENT;
  const int grid = la::num_sms(device);
  if (grid <= 0) return LA_ERR_CUDA;
  const int64_t rows = prefix_rows(batch, num_q_heads, grid) + own_rows(batch, num_q_heads, grid);
  if (rows > 0x7fffffffLL) return LA_ERR_UNSUPPORTED;
  *bytes = static_cast<size_t>(rows) * (kD + 1) * sizeof(float) + 256;
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
  using namespace la::prefix;
  if (!q || !k_cache || !v_cache || !block_table || !cache_seqlens || !out ||
      (num_groups > 0 && (!prefix_lens || !cu_prefix_rows)))
    return LA_ERR_INVALID_ARGUMENT;
  if (batch < 0 || num_groups < 0 || num_blocks <= 0 || block_size <= 0 || max_blocks_per_seq <= 0)
    return LA_ERR_INVALID_ARGUMENT;
  if (batch == 0) return LA_OK;
  if (head_dim != kD) return LA_ERR_UNSUPPORTED;
  if (num_kv_heads <= 0 || num_kv_heads > 8 || 8 % num_kv_heads != 0) return LA_ERR_UNSUPPORTED;
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads != 0) return LA_ERR_INVALID_ARGUMENT;
  const int group = num_q_heads / num_kv_heads;
  if (group > 8) return LA_ERR_UNSUPPORTED;
  if (block_size % 16 != 0 || num_blocks > 0x7ffffffeLL) return LA_ERR_UNSUPPORTED;
  if (!(softmax_scale > 0.f)) return LA_ERR_INVALID_ARGUMENT;
  if (q_batch_stride <= 0 || q_head_stride <= 0 || kv_block_stride <= 0 || kv_token_stride <= 0 ||
      kv_head_stride <= 0 || out_batch_stride <= 0 || out_head_stride <= 0)
    return LA_ERR_INVALID_ARGUMENT;
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16)) return LA_ERR_ALIGNMENT;
  if (q_batch_stride % 8 || q_head_stride % 8 || kv_block_stride % 8 || kv_token_stride % 8 || kv_head_stride % 8)
    return LA_ERR_ALIGNMENT;
  if (!aligned(out, 8) || out_batch_stride % 4 || out_head_stride % 4) return LA_ERR_ALIGNMENT;

  const int device = current_device();
  const int grid = device >= 0 ? num_sms(device) : 0;
  if (grid <= 0) return LA_ERR_CUDA;
  size_t need = 0;
  int st = la_paged_decode_shared_prefix_workspace_size(device, batch, num_groups, num_q_heads, num_kv_heads, head_dim,
                                                        &need);
  if (st != LA_OK) return st;
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256)) return LA_ERR_WORKSPACE;

  if (num_groups == 0 || batch < 2)  // nothing to share; the workspace is larger than that call's
    return la_paged_decode(q, q_batch_stride, q_head_stride, k_cache, v_cache, kv_block_stride, kv_token_stride,
                           kv_head_stride, num_blocks, block_size, block_table, bt_seq_stride, max_blocks_per_seq,
                           cache_seqlens, batch, num_q_heads, num_kv_heads, head_dim, softmax_scale, out,
                           out_batch_stride, out_head_stride, softmax_lse, workspace, workspace_bytes, dev_error, stream);

  PrefixGroups groups;
  groups.cu = cu_prefix_rows;
  groups.lens = prefix_lens;
  groups.n = num_groups;
  groups.batch = batch;
  groups.block_size = block_size;
  groups.bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(block_size)) : -1;
  groups.cap = static_cast<int64_t>(max_blocks_per_seq) * block_size;
  if (groups.cap > 0x7fffff00LL) groups.cap = 0x7fffff00LL / block_size * block_size;  // lengths are int32
  const int per_tile = kRows / group;
  // the steps of one group, counted in 32 bits
  const int64_t key_tiles = (groups.cap + kKeys - 1) / kKeys;
  if (key_tiles * num_kv_heads * (batch / (2 * per_tile) + 1) > 0x7fffffffLL) return LA_ERR_UNSUPPORTED;

  const int64_t rows = prefix_rows(batch, num_q_heads, grid), all = rows + own_rows(batch, num_q_heads, grid);
  float* part_o = static_cast<float*>(workspace);
  float* part_lse = part_o + all * kD;

  {
    CUtensorMap tq, tk, tv;
    {
      const uint64_t dims[3] = {128, static_cast<uint64_t>(num_q_heads), static_cast<uint64_t>(batch)};
      const uint64_t strides[2] = {static_cast<uint64_t>(q_head_stride) * 2, static_cast<uint64_t>(q_batch_stride) * 2};
      const uint32_t box[3] = {64, static_cast<uint32_t>(group), static_cast<uint32_t>(per_tile)};
      if ((st = encode_tensor_map_bf16(&tq, q, 3, dims, strides, box, true)) != LA_OK) return st;
    }
    int box_keys = kKeys;
    while (block_size % box_keys) box_keys >>= 1;
    {
      const uint64_t dims[4] = {128, static_cast<uint64_t>(block_size), static_cast<uint64_t>(num_kv_heads),
                                static_cast<uint64_t>(num_blocks)};
      const uint64_t strides[3] = {static_cast<uint64_t>(kv_token_stride) * 2, static_cast<uint64_t>(kv_head_stride) * 2,
                                   static_cast<uint64_t>(kv_block_stride) * 2};
      const uint32_t box[4] = {64, static_cast<uint32_t>(box_keys), 1, 1};
      if ((st = encode_tensor_map_bf16(&tk, k_cache, 4, dims, strides, box, true)) != LA_OK) return st;
      if ((st = encode_tensor_map_bf16(&tv, v_cache, 4, dims, strides, box, true)) != LA_OK) return st;
    }
    Params p;
    p.groups = groups;
    p.table = block_table;
    p.table_stride = bt_seq_stride;
    p.max_blocks = max_blocks_per_seq;
    p.num_blocks = static_cast<int>(num_blocks);
    p.box_keys = box_keys;
    p.hkv = num_kv_heads;
    p.group = group;
    p.per_tile = per_tile;
    p.scale_log2 = softmax_scale * 1.4426950408889634f;
    p.part_o = part_o;
    p.part_lse = part_lse;
    p.err = dev_error;
    st = cuda_status(launch_pdl(prefix_kernel, dim3(grid), dim3(kThreads), kSmemBytes, stream, tq, tk, tv, p));
    if (st != LA_OK) return st;
  }

  st = decode_own_keys(q, q_batch_stride, q_head_stride, k_cache, v_cache, kv_block_stride, kv_token_stride,
                       kv_head_stride, num_blocks, block_size, block_table, bt_seq_stride, max_blocks_per_seq,
                       cache_seqlens, batch, num_q_heads, num_kv_heads, head_dim, softmax_scale, out, out_batch_stride,
                       out_head_stride, softmax_lse, dev_error, stream,
                       OwnKeysPass{groups, part_o + rows * kD, part_lse + rows});
  if (st != LA_OK) return st;

  CombineParams c;
  c.groups = groups;
  c.seqlens = cache_seqlens;
  c.hq = num_q_heads;
  c.hkv = num_kv_heads;
  c.group = group;
  c.per_tile = per_tile;
  c.grid = grid;
  c.tc = 16 * (8 / num_kv_heads);
  c.own0 = static_cast<int>(rows);
  c.part_o = part_o;
  c.part_lse = part_lse;
  c.out = static_cast<__nv_bfloat16*>(out);
  c.out_bs = out_batch_stride;
  c.out_hs = out_head_stride;
  c.lse = softmax_lse;
  const int warps = num_q_heads < kCombineWarps ? num_q_heads : kCombineWarps;
  return cuda_status(launch_pdl(combine_kernel, dim3(batch), dim3(32 * warps), 0, stream, c));
}
