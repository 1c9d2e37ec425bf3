// Paged GQA decode attention for a batch whose rows share long prefixes, sm_100a.
//
// out[b, h] = softmax(scale * q[b, h] . K_b^T) V_b over keys 0..cache_seqlens[b]-1
// of row b, read through block_table[b]: what la_paged_decode computes. Rows
// cu_prefix_rows[g] .. cu_prefix_rows[g+1]-1 hold the same pages for their
// first keys, so the softmax is taken in two parts, joined by their maxima and
// sums: over the shared keys for all rows of a group at once, as matrix
// products, and over each row's own keys behind them, streamed row by row
// (the warps of la_decode_body.cuh).
//
// shared_prefix_kernel does both at once, each on its own SMs. The shared part
// is bound by the tensor cores and the exponentials when many rows share a
// prefix: a step (see below) is 2048 cycles of products and as many of
// exponentials on an SM and takes ~2.2 us (128 rows with 32768 shared keys only:
// 51 us, 0.67 PFLOP/s of products). The rows' own keys are bound by HBM, which
// about 64 SMs of streaming CTAs already draw 4.75 of its ~6 TB/s from (96: 5.7).
// One after the other on all SMs, the two took their sum, and each its own start
// (128 rows behind 32768 keys: 103 us); side by side they take little more than
// the longer one (62 us, 72 once the power limit has lowered the clock). Every CTA
// counts the steps and units of both parts and takes the same decision: P CTAs
// for the prefixes, as many as finish with the rest by a model of both, the
// others for the rows. combine_kernel joins the parts of every row.
//
// 128 rows, 16 query and 8 kv heads, mostly their own keys behind 2048 shared
// ones: 50.3 us, 88 % of HBM's measured rate; 4 rows: 11 us, of which ~4 pass
// before the plan is there and checked and ~3 between the last CTA's end and the
// combined row (instructions that run once cost ~10 ns each, from a cold cache).
//
// Shared part. For one kv head the group's rows x query heads of the kv head
// are the rows of Q; with 128-key tiles of K and V,
//   S = Q K^T,  P = exp2(S * scale * log2 e - m),  O += P V,  l += sum P
// run on tcgen05 with fp32 accumulators in tensor memory, m the running row
// maximum. An item is (group, kv head, pair of 128-row tiles); both tiles use
// each K/V tile that is staged. Where only one tile is left over, its two
// accumulators take the even and the odd key tiles instead, so that one
// tile's products still run while the other's exponentials do. A step is two
// tile products either way: one key tile of a pair of row tiles, or two key
// tiles of a single one. S and P go in halves of 64 keys, so that a tile's
// softmax of one half runs while the products of the other do (whole tiles:
// 80.6 us instead of 72.5 for 128 rows behind 32768 keys, although a product of
// half the width takes three quarters of the time). The steps of all items, laid
// end to end, are cut into P equal ranges; an item's part in a range is a
// segment, which leaves normalised fp32 O rows and base-2 logarithms of its sums.
//
// CTA, 12 warps. Shared part: 0-3 and 4-7 softmax of tile 0 and 1 (a thread
// per row, half a tile's S row in registers), which store the segments' O as
// well, 8 and 11 issue the products of tile 0 and 1, 9 the TMA loads; tensor
// memory holds S0 S1 O0 O1, 128 columns each, P over S. Own keys: 0-7 consume,
// 10 and 11 load. 10 makes the plan.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "la_decode_body.cuh"
#include "la_groups.cuh"
#include "la_internal.h"
#include "la_ptx.cuh"

namespace la {
namespace prefix {

constexpr int kD = 128;
constexpr int kRows = 128;             // query rows per tile
constexpr int kKeys = 128;             // keys per K/V tile
constexpr int kParts = 2;              // S and P of a key tile
constexpr int kPart = kKeys / kParts;  // keys of each
constexpr int kHalf = 128 * 128;       // 64 dims of 128 rows: 16 KB
constexpr int kTile = 2 * kHalf;
constexpr int kStages = 4;             // K/V tiles in flight
constexpr int kThreads = 384;          // 12 warps: 168 registers for each thread
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;        // O_t at kColO + 128 t; S_t of a tile's first half at 128 t, of the second 64 behind
constexpr uint32_t kIdescQK = idesc_bf16_f32(128, kPart, false, false);
constexpr uint32_t kIdescPV = idesc_bf16_f32(128, 128, false, true);
// Shared memory. Control, both parts' barriers apart: they are initialised
// before the CTA knows which part it takes. Then the part's data: Q0 Q1 and the
// K/V ring; or the stages and the merge area of the decode warps.
constexpr int kOffTmem = 224;
constexpr int kOffOwnBar = 256;
constexpr int kOffPlan = 384;
constexpr int kOffStale = 448;
constexpr int kOffDesc = 512;
constexpr int kOffZero = 640;
constexpr int kOffWalk = 768;          // of the softmax warps, kept out of their registers
constexpr int kWalkBytes = 120;
constexpr int kOffTable = 2048;
constexpr int kCtrlBytes = 8192;
constexpr int kOffQ = kCtrlBytes;
constexpr int kOffKV = kOffQ + 2 * kTile;
constexpr size_t kSmemBytes = kOffKV + kStages * kTile + 1024;  // + alignment to 1024 bytes at run time
static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
static_assert(kOffWalk + 8 * kWalkBytes <= kOffTable && kOffTable + kMaxGroups * sizeof(PrefixGroup) <= kCtrlBytes,
              "control area");
// Warps behind the eight of softmax or consumers. Shared part: the products of
// tile 0 and (kWarpSecond) 1, and the loads between them. Own keys: the last two
// load. kWarpPlan makes the plan.
constexpr int kWarpProduct = 8, kWarpLoad = 9, kWarpPlan = 10, kWarpSecond = 11;

// The time model that divides the SMs (shared_ctas). Microseconds on a B200,
// fitted to the times of 15 calls with 2 to 146 CTAs for the shared part: all get
// the division that measured fastest or one within 4 %
// (with fractional steps per CTA, 9 %). A step with two row tiles (64 KB of K and V), with one (128 KB);
// a unit (64 KB) of a row's own keys, without and with sub-chunks to merge
// (nsub > 1); 64 KB at the rate of HBM; a second segment of a CTA.
constexpr float kPairUs = 1.16f, kSingleUs = 2.14f, kUnitUs = 0.964f, kUnitMergedUs = 1.236f, kHbmUs = 0.0094f,
                kSegmentUs = 4.5f;

struct Params {
  decode::Params own;  // the rows' own keys; groups, tables, counts and scale of both parts
  // Of 64 KB, of the decode warps: three, or two where three do not fit (128 rows
  // behind 2048 keys, mostly their own: 50.2 us with three, 53.2 with two).
  int stages;
  int box_keys;        // keys per TMA box, a power of two that divides the block size
  int per_tile;        // sequences per row tile: 128 / group
  uint32_t tile_magic; // ceil(2^32 / per_tile): x / per_tile is the high word of x * magic for x < 2^25
  float* part_o;       // [rows][D]
  float* part_lse;     // [rows], base 2
  int4* items;         // [batch][hkv]: first partial row of the row's first head, distance of the second
                       // accumulator's (0: none), first and last CTA of its item
  int* flags;          // [batch]: kShares, kOwn
};
constexpr int kShares = 1, kOwn = 2;

// How the steps of a group lie: kv heads one after another, in each the pairs
// of row tiles, the single tile last.
struct Shape {
  int tiles;    // key tiles
  int pairs;    // of row tiles, the single one included
  int single;   // 1: the last has one tile
  int half;     // steps of that one
  int per_head; // steps of one kv head
};

__device__ __forceinline__ Shape shape_of(const Params& p, const PrefixGroup& g) {
  Shape s;
  const int row_tiles = static_cast<int>(__umulhi(g.rows + p.per_tile - 1, p.tile_magic));
  s.tiles = (g.keys + kKeys - 1) / kKeys;
  s.pairs = (row_tiles + 1) >> 1;
  s.single = row_tiles & 1;
  s.half = s.single ? (s.tiles + 1) >> 1 : 0;
  s.per_head = (s.pairs - s.single) * s.tiles + s.half;
  return s;
}

__device__ __forceinline__ int steps_of(const Params& p, const PrefixGroup& g) {
  return g.keys > 0 ? p.own.hkv * shape_of(p, g).per_head : 0;
}

// First partial row of item (g, h, r) in CTA c. An item's segments take up to
// 256 rows, those of two accumulators; from one segment to the next along the
// line of steps the item, the CTA or both go up, the item by at least the rows
// that one segment of it takes.
__device__ __forceinline__ int part_row(const Params& p, const PrefixGroup& g, int h, int r, int c) {
  return 2 * p.own.group * (p.own.hkv * g.first + h * g.rows + r * 2 * p.per_tile) + 2 * kRows * c;
}

// What the CTA does: its range of steps or of units, and where that begins.
struct Plan {
  long long u0, u1;
  long long before;  // steps before group `at`, or units before row `at`
  int at;
  int shared;        // takes part in the shared part
  int c;             // its number in its part
};

__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }
__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

// Lengths of rows base + 8 lane + i (0 past the batch), 16 bytes at a time
// where they can be; through L2 only, since the kernel in front may still
// write them (no stale line stays in L1).
__device__ __forceinline__ void load_lens8(const Params& p, int lane, int base, int (&raw)[8]) {
  const int* s = p.own.seqlens;
  const int b0 = base + 8 * lane;
  const bool vec = (reinterpret_cast<uintptr_t>(s) & 15) == 0;
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const int b = b0 + 4 * v;
    if (vec && b + 3 < p.own.batch) {
      const int4 x = __ldcg(reinterpret_cast<const int4*>(s + b));
      raw[4 * v] = x.x;
      raw[4 * v + 1] = x.y;
      raw[4 * v + 2] = x.z;
      raw[4 * v + 3] = x.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[4 * v + e] = b + e < p.own.batch ? __ldcg(s + b + e) : 0;
    }
  }
}

// What a plan for up to 256 rows and 32 groups was made from, one warp.
struct Seen {
  int raw[8];
  int lo, hi, len;
};
__device__ __forceinline__ Seen read_inputs(const Params& p, int lane) {
  Seen r;
  load_lens8(p, lane, 0, r.raw);
  const bool in = lane < p.own.groups.n;
  r.lo = in ? __ldcg(p.own.groups.cu + lane) : 0;
  r.hi = in ? __ldcg(p.own.groups.cu + lane + 1) : 0;
  r.len = in ? __ldcg(p.own.groups.lens + lane) : 0;
  return r;
}

// Units of those rows (kept in raw), and their sum. The first block's look-up
// of groups runs over the registers of the lanes that hold them (grp: lane g's
// group, the first of at most 32), the others search the table.
__device__ __forceinline__ int units8(const Params& p, const PrefixGroup* tab, const PrefixGroup& grp, bool in_regs,
                                      int lane, int base, int (&raw)[8]) {
  const int cap = static_cast<int>(p.own.groups.cap);
#pragma unroll
  for (int i = 0; i < 8; ++i) raw[i] = min(max(raw[i], 0), cap);
  if (in_regs) {
    int own[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) own[i] = raw[i];
    for (int g = 0; g < p.own.groups.n; ++g) {
      const int d = base + 8 * lane - __shfl_sync(0xffffffffu, grp.first, g);
      const unsigned rows = __shfl_sync(0xffffffffu, grp.rows, g);
      const int keys = __shfl_sync(0xffffffffu, grp.keys, g);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (static_cast<unsigned>(d + i) < rows && raw[i] >= keys) own[i] = raw[i] - keys;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = own[i];
  } else {
    for (int i = 0; i < 8; ++i) {
      const int c = raw[0];
#pragma unroll
      for (int e = 0; e < 7; ++e) raw[e] = raw[e + 1];
      raw[7] = c > 0 ? c - prefix_keys(p.own.groups, tab, base + 8 * lane + i, c) : 0;
    }
  }
  int sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    raw[i] = decode::units_p(p.own, raw[i]);
    sum += raw[i];
  }
  return sum;
}

// x / d for x < 2^16 and d < 2^10, rounded down: the quotient of x + 1/2 is at
// least 1 / (2 d) away from a whole number, far more than its rounding.
__device__ __forceinline__ int small_div(int x, float inv_d) {
  return static_cast<int>((static_cast<float>(x) + 0.5f) * inv_d);
}

// First of T steps or units of CTA c of G: floor(c T / G).
__device__ __forceinline__ long long part_start(int c, long long T, int G) { return c * T / G; }
__device__ __forceinline__ int part_start(int c, int T, int G, float inv_G) {
  const int q = T / G;
  return c * q + small_div(c * (T - q * G), inv_G);
}

// CTAs of the shared part, an even number, from its steps, the rows' units and
// the items: the one of least time by a model, 64 numbers of CTAs tried at
// once, of several the one with most, whose busy CTAs are the closest (8 rows
// 12 us instead of 12.7). The shared part takes the time of a CTA's steps, the
// other that of its units over its CTAs; where all CTAs together would load more
// than HBM gives, by a factor f, the steps with two row tiles, whose loads are
// needed soonest, take f^3 as long, the others, whose loads are twice as many,
// f^0.5. A CTA whose range is not within one item has two segments to store.
// Where there is a CTA for every step and unit, the model has nothing to weigh.
__device__ __forceinline__ int shared_ctas(const Params& p, float pair_steps, float single_steps, float units,
                                           int items, int grid, int lane) {
  const float steps = pair_steps + single_steps, avg = __fdividef(1.f, steps);
  if (steps + units < static_cast<float>(grid)) return (grid - static_cast<int>(units)) & ~1;
  const float a = pair_steps * kPairUs, b = single_steps * kSingleUs;
  const float unit = p.own.nsub > 1 ? kUnitMergedUs : kUnitUs, own_work = units * unit;
  const float loads = __fdividef(pair_steps + 2.f * single_steps, a + b) * kHbmUs;  // of one CTA, of HBM's rate
  const float own_loads = __fdividef(kHbmUs, unit), per_item = __fdividef(1.f, static_cast<float>(items));
  float best = 3e38f;
  int at = 2;
#pragma unroll 1
  for (int P = 2 + 2 * lane; P <= grid; P += 64) {
    const float x = static_cast<float>(P), cs = fminf(x, steps), co = fminf(static_cast<float>(grid - P), units);
    const float f = fmaxf(1.f, cs * loads + co * own_loads);
    // whole items per CTA or CTAs per item: P * per_item is whole up to rounding
    const float y = x * per_item, odd = x < steps && fabsf(y - rintf(y)) > 1e-3f ? kSegmentUs : 0.f;
    const float t = fmaxf((a * f * f * f + b * sqrtf(f)) * avg * ceilf(__fdividef(steps, cs) - 1e-3f) + odd,
                          units > 0.f ? __fdividef(own_work, fmaxf(co, 1e-6f)) : 0.f);
    if (t <= best) {
      best = t;
      at = P;
    }
  }
  // positive floats compare as their bits do
  const unsigned least = __reduce_min_sync(0xffffffffu, __float_as_uint(best));
  return static_cast<int>(__reduce_max_sync(0xffffffffu, __float_as_uint(best) == least ? at : 0));
}

// The part that the CTA takes, and its number there. Neighbouring CTAs mostly
// land on the two SMs of a TPC, next pairs on the same GPC. A pair has the same
// part (two that stream load 114 GB/s together, one beside a tensor core CTA
// ~48 GB/s while that one takes 1.3 times as long), and the pairs that stream
// are spread evenly among the others. Q: CTAs that stream, an even number.
__device__ __forceinline__ void take_part(Plan& r, int Q, int grid, bool any_shared) {
  const int pairs = grid >> 1, pair = static_cast<int>(blockIdx.x >> 1), half = Q >> 1;
  const float inv = __fdividef(1.f, static_cast<float>(pairs));
  const int before = small_div(pair * half, inv);
  r.shared = any_shared && (pair >= pairs || small_div((pair + 1) * half, inv) == before);
  r.c = static_cast<int>(blockIdx.x);
  if (any_shared) r.c = r.shared ? r.c - 2 * min(before, half) : 2 * before + (r.c & 1);
  r.u0 = r.u1 = r.before = 0;
  r.at = 0;
}

// One warp's work, for up to 256 rows and 32 groups: `in`, all in registers.
__device__ __forceinline__ Plan make_plan(const Params& p, PrefixGroup* tab, const Seen& in, int lane) {
  const PrefixGroups& G = p.own.groups;
  PrefixGroup grp{0, 0, 0};
  Shape h{0, 0, 0, 0, 0};
  const bool sound = __all_sync(0xffffffffu, lane >= G.n || run_of_rows(G, in.lo, in.hi));
  if (lane < G.n) {
    if (sound) grp = group_from(G, in.lo, in.hi, in.len);
    tab[lane] = grp;
    if (grp.keys > 0) h = shape_of(p, grp);
  }
  const int mine = p.own.hkv * h.per_head;
  const int S = warp_sum(mine), single = warp_sum(p.own.hkv * h.half);
  const int items = warp_sum(h.tiles ? p.own.hkv * h.pairs : 0);
  int raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) raw[i] = in.raw[i];
  const int first = units8(p, tab, grp, true, lane, 0, raw);
  const int U = warp_sum(first);
  const int grid = static_cast<int>(gridDim.x);
  const int Q = S > 0 ? (grid - shared_ctas(p, static_cast<float>(S - single), static_cast<float>(single),
                                            static_cast<float>(U), items, grid, lane)) & ~1
                      : grid;
  Plan r;
  take_part(r, Q, grid, S > 0);
  // no more CTAs than units, so that a row's parts are those of consecutive ones
  const int T = r.shared ? S : U, n = min(T, r.shared ? grid - Q : Q);
  if (r.c >= n) return r;
  const float inv = __fdividef(1.f, static_cast<float>(n));
  const int u0 = part_start(r.c, T, n, inv);
  r.u0 = u0;
  r.u1 = part_start(r.c + 1, T, n, inv);
  // the lane that holds the first one: a group each, or eight rows
  const int incl = warp_scan(r.shared ? mine : first, lane);
  const int src = __ffs(__ballot_sync(0xffffffffu, incl > u0)) - 1;
  int at = 0, before = incl - (r.shared ? mine : first);
  if (!r.shared) {
    bool found = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      found |= u0 < before + raw[i];
      if (!found) {
        before += raw[i];
        at = i + 1;
      }
    }
  }
  r.at = __shfl_sync(0xffffffffu, r.shared ? lane : 8 * lane + at, src);
  r.before = __shfl_sync(0xffffffffu, before, src);
  return r;
}

// The same for any number of rows and groups.
__device__ __noinline__ Plan make_large_plan(const Params& p, PrefixGroup* tab, int lane) {
  const PrefixGroups& G = p.own.groups;
  int raw[8];
  long long S = 0, single = 0, U = 0;
  int items = 0;
  const PrefixGroup none{0, 0, 0};
  bool sound = true;
  for (int b = 0; b < G.n; b += 32) {
    const int g = b + lane;
    Shape h{0, 0, 0, 0, 0};
    if (g < G.n) {
      const int lo = __ldcg(G.cu + g), hi = __ldcg(G.cu + g + 1);
      const PrefixGroup r = group_from(G, lo, hi, __ldcg(G.lens + g));
      sound &= run_of_rows(G, lo, hi);
      if (G.n <= kMaxGroups) tab[g] = r;
      if (r.keys > 0) h = shape_of(p, r);
    }
    S += warp_sum(p.own.hkv * h.per_head);
    single += warp_sum(p.own.hkv * h.half);
    items += warp_sum(h.tiles ? p.own.hkv * h.pairs : 0);
  }
  sound = __all_sync(0xffffffffu, sound);
  if (!sound) {
    S = single = 0;
    items = 0;
    for (int g = lane; g < min(G.n, kMaxGroups); g += 32) tab[g] = none;
  }
  if (G.n > kMaxGroups && lane == 0) tab->rows = sound;
  __syncwarp();
  for (int base = 0; base < G.batch; base += 256) {
    load_lens8(p, lane, base, raw);
    U += warp_sum(units8(p, tab, none, false, lane, base, raw));
  }
  const int grid = static_cast<int>(gridDim.x);
  const int Q = S > 0 ? (grid - shared_ctas(p, static_cast<float>(S - single), static_cast<float>(single),
                                            static_cast<float>(U), items, grid, lane)) & ~1
                      : grid;
  Plan r;
  take_part(r, Q, grid, S > 0);
  const long long T = r.shared ? S : U;
  const int most = r.shared ? grid - Q : Q, n = static_cast<int>(T < most ? T : most);
  if (r.c >= n) return r;
  r.u0 = part_start(r.c, T, n);
  r.u1 = part_start(r.c + 1, T, n);
  long long acc = 0;
  const int count = r.shared ? G.n : G.batch, stride = r.shared ? 32 : 256;
  for (int base = 0; base < count; base += stride) {
    int sum = 0;
    if (r.shared) {
      if (base + lane < G.n) sum = steps_of(p, prefix_group(G, tab, base + lane));
    } else {
      load_lens8(p, lane, base, raw);
      sum = units8(p, tab, none, false, lane, base, raw);
    }
    const int incl = warp_scan(sum, lane);
    const unsigned hit = __ballot_sync(0xffffffffu, acc + incl > r.u0);
    if (hit) {
      const int src = __ffs(hit) - 1;
      int at = 0;
      long long before = acc + incl - sum;
      if (!r.shared) {
        bool found = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          found |= r.u0 < before + raw[i];
          if (!found) {
            before += raw[i];
            at = i + 1;
          }
        }
      }
      r.at = base + __shfl_sync(0xffffffffu, r.shared ? lane : 8 * lane + at, src);
      r.before = __shfl_sync(0xffffffffu, before, src);
      break;
    }
    acc += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}

// Segments of the CTA's range, one after another (the same in every thread).
struct Walk {
  int left;  // steps of the range not yet taken
  int c;     // the CTA's number in the shared part
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
  int begin, end;   // of the item
  int c;            // the CTA's number in the shared part
};

__device__ __forceinline__ void walk_group(const Params& p, const PrefixGroup* tab, Walk& w, int g) {
  w.g = g;
  w.grp = prefix_group(p.own.groups, tab, g);
  w.shp = shape_of(p, w.grp);
}

__device__ __forceinline__ void walk_start(const Params& p, const PrefixGroup* tab, const Plan& R, Walk& w) {
  w.left = static_cast<int>(R.u1 - R.u0);
  w.c = R.c;
  if (w.left <= 0) return;
  walk_group(p, tab, w, R.at);
  const int x = static_cast<int>(R.u0 - R.before);
  w.h = x / w.shp.per_head;
  const int y = x - w.h * w.shp.per_head;
  w.r = min(y / w.shp.tiles, w.shp.pairs - 1);
  w.s = y - w.r * w.shp.tiles;
}

__device__ __forceinline__ bool walk_next(const Params& p, const PrefixGroup* tab, Walk& w, Segment& e) {
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
  e.c = w.c;
  e.row0 = part_row(p, w.grp, w.h, w.r, w.c);
  e.begin = w.s == 0;
  e.end = w.s + n == steps;
  w.left -= n;
  w.s += n;
  if (w.s == steps && w.left > 0) {
    w.s = 0;
    if (++w.r == w.shp.pairs) {
      w.r = 0;
      if (++w.h == p.own.hkv) {
        w.h = 0;
        int g = w.g;
        do {
          if (++g >= p.own.groups.n) {  // groups changed under the kernel
            w.left = 0;
            return true;
          }
          walk_group(p, tab, w, g);
        } while (w.grp.keys == 0);
      }
    }
  }
  return true;
}

static_assert(kOffDesc + 3 * sizeof(decode::StageDesc) <= kOffZero, "a descriptor per stage");
static_assert(sizeof(Walk) <= 64 && sizeof(Segment) + 64 <= kWalkBytes, "a softmax warp's walk");

// Key tiles that tile t's accumulator takes, and the i-th of them.
__device__ __forceinline__ int tiles_of(const Segment& e, int t) { return e.two ? e.tiles : (e.tiles + 1 - t) >> 1; }
// Query rows of tile t, and its first partial row.
__device__ __forceinline__ int rows_of(const Params& p, const Segment& e, int t) {
  const int seqs = e.two && t ? e.rows - p.per_tile : min(e.rows, p.per_tile);
  return seqs * p.own.group;
}

// Lane 0's value, which the compiler knows to be the same in every lane.
template <typename T>
__device__ __forceinline__ T uniform(T x) {
  return __shfl_sync(0xffffffffu, x, 0);
}

__device__ __forceinline__ uint64_t desc_kmajor(const uint8_t* tile) {
  return smem_desc_sw128(smem_u32(tile), 16, 1024);
}
__device__ __forceinline__ uint64_t desc_v(const uint8_t* tile) { return smem_desc_sw128(smem_u32(tile), kHalf, 1024); }

// The barriers of the shared part.
struct Bars {
  uint64_t* b;
  __device__ __forceinline__ uint64_t* q_full() const { return b + 0; }    // a segment's Q landed
  __device__ __forceinline__ uint64_t* q_empty() const { return b + 1; }   // both product warps' last S done
  __device__ __forceinline__ uint64_t* kv_full() const { return b + 2; }   // [kStages]
  __device__ __forceinline__ uint64_t* kv_empty() const { return b + 6; }  // [kStages] both product warps are through
  __device__ __forceinline__ uint64_t* s_full() const { return b + 10; }   // [2][2] S_t of each half written
  __device__ __forceinline__ uint64_t* p_full() const { return b + 14; }   // [2][2] P_t of each half written (128 arrivals)
  __device__ __forceinline__ uint64_t* pv_done() const { return b + 18; }  // [2] P_t V done
  __device__ __forceinline__ uint64_t* o_full() const { return b + 20; }   // [2] a segment's last P_t V done
  __device__ __forceinline__ uint64_t* o_empty() const { return b + 22; }  // [2] O_t stored (128)
  __device__ __forceinline__ uint64_t* planned() const { return b + 24; }  // the plan is in shared memory
  __device__ __forceinline__ uint64_t* checked() const { return b + 25; }  // it was checked after the wait
  __device__ __forceinline__ uint64_t* done() const { return b + 26; }     // a softmax warp is through (8)
  __device__ __forceinline__ uint64_t* again() const { return b + 27; }    // a warp has left the stale plan (11)
};

__device__ __forceinline__ bool wait_warp(const Params& p, uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.own.err, LA_DEVERR_WAIT_TIMEOUT));
}

// Softmax of tile t and the segments' results, four warps, a thread per row.
__device__ __forceinline__ void softmax_warp(const Params& p, const PrefixGroup* tab, const Plan& plan, uint8_t* smem,
                                             Bars bars, uint32_t tmem, int t, int warp, int lane) {
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return wait_warp(p, bar, parity); };
  uint64_t* s_full = bars.s_full() + kParts * t;
  uint64_t* p_full = bars.p_full() + kParts * t;
  uint64_t* pv_done = bars.pv_done() + t;
  uint64_t* o_full = bars.o_full() + t;
  uint64_t* o_empty = bars.o_empty() + t;
  const float NEG_INF = -__int_as_float(0x7f800000);
  const int quarter = warp & 3;
  const int row = quarter * 32 + lane;
  const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const uint32_t colS = t * 128, colO = kColO + t * 128;
  const float sl2 = p.own.scale_log2;
  Walk& w = *reinterpret_cast<Walk*>(smem + kOffWalk + warp * kWalkBytes);
  Segment& e = *reinterpret_cast<Segment*>(smem + kOffWalk + warp * kWalkBytes + 64);
  auto next = [&]() -> bool {
    Walk x = w;
    Segment y{};
    const bool more = walk_next(p, tab, x, y);
    __syncwarp();  // every lane has read the old state
    if (lane == 0) {
      w = x;
      e = y;
    }
    __syncwarp();
    return more;
  };
  uint32_t seen = 0, segs = 0;  // halves of key tiles, segments
  bool ok = true;
  {
    Walk x;
    walk_start(p, tab, plan, x);
    if (lane == 0) w = x;
    __syncwarp();
  }
  while (ok && next()) {
    const int n = tiles_of(e, t);
    const int rows = rows_of(p, e, t);
    const int row0 = e.row0 + t * rows_of(p, e, 0);
    if (n == 0) {  // a single key tile: none for the second accumulator
      if (row < rows) p.part_lse[row0 + row] = NEG_INF;
      continue;
    }
    const bool active = quarter * 32 < rows;  // rows of this warp
    float m = NEG_INF, l = 0.f;
#pragma unroll 1
    for (int j = 0; j < kParts * n; ++j, ++seen) {
      const int half = j % kParts;
      if (!(ok = wait_all(&s_full[half], (seen / kParts) & 1))) break;
      if (!active) {
        mbar_arrive(&p_full[half]);
        continue;
      }
      tc_fence_after();
      const uint32_t col = colS + half * kPart;
      float sv[kPart / 32][32];
#pragma unroll
      for (int c = 0; c < kPart / 32; ++c) tmem_ld32(taddr + col + c * 32, sv[c]);
      tc_wait_ld();
      // keys of this half, 64 but for the prefix's last tile
      const int nvis = e.keys - (e.tile0 + (e.two ? j / kParts : 2 * (j / kParts) + t)) * kKeys - half * kPart;
      float mx[8];
#pragma unroll
      for (int a = 0; a < 8; ++a) mx[a] = NEG_INF;
      if (nvis >= kPart) {
#pragma unroll
        for (int c = 0; c < kPart / 32; ++c)
#pragma unroll
          for (int x = 0; x < 32; x += 2) mx[(x >> 1) & 7] = fmax3(mx[(x >> 1) & 7], sv[c][x], sv[c][x + 1]);
      } else {
#pragma unroll
        for (int c = 0; c < kPart / 32; ++c)
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
      // O_t is rescaled when it holds the products of the halves before; the
      // next waits for this P. (The one but last is done, since S was issued
      // behind it: the parity means the last.)
      if (j >= 1 && __any_sync(0xffffffffu, m_new != m)) {
        if (!(ok = wait_all(pv_done, (seen - 1) & 1))) break;
        tc_fence_after();
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
      // P rounded to bf16, the type of V, for the product; l sums it unrounded.
#pragma unroll
      for (int c = 0; c < kPart / 32; ++c) {
        float pk[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const uint64_t y2 = f2_fma(f2_pack(sv[c][2 * x], sv[c][2 * x + 1]), sl2x2, negm2);
          float e0, e1;
          f2_unpack(y2, e0, e1);
          e0 = ex2(e0);
          e1 = ex2(e1);
          acc2[x & 3] = f2_add(acc2[x & 3], f2_pack(e0, e1));
          pk[x] = __uint_as_float(pack_bf16x2(e0, e1));
        }
        tmem_st16(taddr + col + c * 16, pk);
      }
      float ps[8];
#pragma unroll
      for (int a = 0; a < 4; ++a) f2_unpack(acc2[a], ps[2 * a], ps[2 * a + 1]);
      l = l * alpha + (((ps[0] + ps[1]) + (ps[2] + ps[3])) + ((ps[4] + ps[5]) + (ps[6] + ps[7])));
      m = m_new;
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[half]);
    }
    if (!ok) break;
    if (!(ok = wait_all(o_full, segs++ & 1))) break;  // the last product
    tc_fence_after();
    // What the combine pass has to know of the item: where its parts are.
    if ((e.begin || e.end) && (e.two || t == 0) && row < rows && row % p.own.group == 0) {
      int4* it = p.items + static_cast<long long>(e.first + t * p.per_tile + row / p.own.group) * p.own.hkv + e.h;
      if (e.begin) {
        it->x = row0 + row;
        it->y = e.two ? 0 : rows;
        it->z = e.c;
      }
      if (e.end) it->w = e.c;
    }
    if (row < rows) p.part_lse[row0 + row] = l == 0.f ? NEG_INF : m + __log2f(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    // Each thread stores its row, 32 bytes (a sector) at a time.
    float* dst = p.part_o + static_cast<long long>(row0 + row) * kD;
    if (active) {
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        float o[32];
        tmem_ld32(taddr + colO + c * 32, o);
        tc_wait_ld();
#pragma unroll
        for (int x = 0; x < 32; ++x) o[x] *= inv;
        if (row < rows) {
#pragma unroll
          for (int x = 0; x < 4; ++x) store_f32x8(dst + c * 32 + x * 8, o + x * 8);
        }
      }
    }
    tc_fence_before();
    mbar_arrive(o_empty);
  }
}

// The page ids of a segment's boxes, one box (64 dims of box_keys keys of one
// page) per lane: read 32 boxes at a time, the next 32 in advance.
struct Pages {
  const int* ids_of_row;
  int boxes, per_page;  // boxes of a tile, of a page
  int win, ids, next;
  // Not by the read-only path: the kernel in front may write the table after this
  // one has started, and such a load need not stay behind the wait for it.
  __device__ __forceinline__ int read(const Params& p, const Segment& e, int w0, int lane) const {
    const int x = w0 * 32 + lane;
    return x * p.box_keys < e.keys ? __ldcg(ids_of_row + x / per_page) : -1;
  }
  __device__ __forceinline__ void start(const Params& p, const Segment& e, int lane) {
    boxes = kKeys / p.box_keys;
    per_page = p.own.block_size / p.box_keys;
    ids_of_row = p.own.block_table + static_cast<long long>(e.table_row) * p.own.bt_stride;
    win = e.tile0 * boxes >> 5;
    ids = read(p, e, win, lane);
    next = read(p, e, win + 1, lane);
  }
  // The page of this lane's box (lane / 2) of a tile; tiles in ascending order.
  __device__ __forceinline__ int of(const Params& p, const Segment& e, int tile, int lane) {
    const int x = tile * boxes;
    if (x >> 5 != win) {
      win = x >> 5;
      ids = next;
      next = read(p, e, win + 1, lane);
    }
    return __shfl_sync(0xffffffffu, ids, (x & 31) + min(lane >> 1, boxes - 1));
  }
};

// TMA loads of the shared part, one warp, from segment e on, its page ids in
// `pages`. Per segment Q, then the tiles in the order the products use them:
// `lead` K tiles, then V(i), K(i + lead) in turn; lead is 1 for two row tiles,
// 2 for the two accumulators of one.
__device__ __forceinline__ void load_warp(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                          const Params& p, const PrefixGroup* tab, uint8_t* smem, Bars bars, Walk& w,
                                          Segment& e, Pages& pages, int lane) {
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return wait_warp(p, bar, parity); };
  uint64_t* q_full = bars.q_full();
  uint64_t* q_empty = bars.q_empty();
  uint64_t* kv_full = bars.kv_full();
  uint64_t* kv_empty = bars.kv_empty();
  uint8_t* sQ = smem + kOffQ;
  uint8_t* sKV = smem + kOffKV;
  int kq = 0;
  uint32_t pos = 0;  // tiles loaded
  bool ok = true;
  const int half = lane & 1, box = lane >> 1;
  int k_id = 0, v_id = 0;  // pages of the last K tile, and of the one before
  auto load = [&](const CUtensorMap* tm, int tile, int id) -> bool {
    const int st = pos % kStages;
    if (!wait_all(&kv_empty[st], ((pos / kStages) & 1) ^ 1u)) return false;
    uint8_t* dst = sKV + st * kTile;
    if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], kTile);
    __syncwarp();
    if (box < pages.boxes) {
      // keys behind the prefix, and pages outside the pool, come from block
      // num_blocks, outside the tensor map: zeros
      const int x = tile * pages.boxes + box;
      const bool in = x * p.box_keys < e.keys;
      const bool sound = id >= 0 && id < p.own.num_blocks;
      if (in && !sound && p.own.err) atomicCAS(p.own.err, 0, LA_DEVERR_BLOCK_ID);
      const int blk = in && sound ? id : static_cast<int>(p.own.num_blocks);
      tma_load_4d(dst + half * kHalf + box * p.box_keys * 128, tm, &kv_full[st], half * 64,
                  x % pages.per_page * p.box_keys, e.h, blk);
    }
    __syncwarp();
    ++pos;
    return true;
  };
  while (true) {
    if (!(ok = wait_all(q_empty, (kq & 1) ^ 1u))) break;
    if (lane == 0) {
      const uint32_t bytes = 128u * p.own.group * p.per_tile;
      mbar_arrive_expect_tx(q_full, (1 + e.two) * 2 * bytes);
      for (int t = 0; t < 1 + e.two; ++t)
        for (int x = 0; x < 2; ++x)
          tma_load_3d(sQ + t * kTile + x * kHalf, &tm_q, q_full, x * 64, e.h * p.own.group, e.first + t * p.per_tile);
    }
    __syncwarp();
    ++kq;
    // K(i) and V(i - lead), K first
    const int lead = 2 - e.two;
    for (int i = 0; ok && i < e.tiles + lead; ++i) {
      const int id = v_id;
      v_id = k_id;
      if (i >= lead) ok = load(&tm_v, e.tile0 + i - lead, lead == 2 ? id : v_id);
      if (i < e.tiles) {
        k_id = pages.of(p, e, e.tile0 + i, lane);
        ok = ok && load(&tm_k, e.tile0 + i, k_id);
      }
    }
    if (!ok || !walk_next(p, tab, w, e)) break;
    pages.start(p, e, lane);
  }
  if (!ok && lane == 0) {  // early exit: let the copies already issued land (bounded)
    for (uint32_t u = (pos > kStages ? pos - kStages : 0); u < pos; ++u)
      mbar_wait(&kv_full[u % kStages], (u / kStages) & 1, nullptr, 0);
    if (kq > 0) mbar_wait(q_full, (kq - 1) & 1, nullptr, 0);
  }
  __syncwarp();
}

// 1: a pair of row tiles, 0: the two accumulators of one.
template <int kTwo>
struct Pair {
  static constexpr int value = kTwo;
};

// Products of the shared part, from segment e on: a warp for each of the two
// row tiles or accumulators, so that one warp's waits and arithmetic pass while
// the other's products run (one warp for both: 128 rows behind 32768 shared keys
// 52.5 us instead of 50). One thread issues. What the instructions take is the same
// in every lane and known to be so (from lane 0's registers), and the issuing
// thread is chosen by elect.sync (issued under `lane == 0`, from each lane's own
// registers, they took 7 % longer).
__device__ __forceinline__ void product_warp(const Params& p, const PrefixGroup* tab, uint8_t* smem, Bars bars,
                                             uint32_t tmem_base, int tile, Walk& w, Segment& e, int lane) {
  const int t = uniform(tile);
  const uint32_t tmem = uniform(tmem_base), colS = tmem + t * 128, colO = tmem + kColO + t * 128;
  const uint64_t q_desc = uniform(desc_kmajor(smem + kOffQ)), k_desc = uniform(desc_kmajor(smem + kOffKV)),
                 v_desc = uniform(desc_v(smem + kOffKV));
  uint64_t *s_full = bars.s_full() + kParts * t, *p_full = bars.p_full() + kParts * t;
  uint64_t *pv_done = bars.pv_done() + t, *o_full = bars.o_full() + t, *o_empty = bars.o_empty() + t;
  uint32_t segs = 0, pos = 0, p_par = 0, o_par = 1;  // parities of the next phase
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_warp(p, bar, parity); };
  // S over P is issued right behind the product that reads P: the tensor core
  // executes one thread's products in order. A step: the products of V tile i
  // and K tile i + lead; of a pair's tiles each warp takes all, of a single
  // tile's those of its accumulator.
  auto segment = [&](auto pair) -> bool {
    constexpr int kTwo = decltype(pair)::value, kLead = 2 - kTwo;
    const int n = uniform(e.tiles);
#pragma unroll 1
    for (int i = -kLead; i < n; ++i) {
      const bool pv = i >= 0, more = i + kLead < n;
      const uint32_t vs = pos % kStages, v_par = (pos / kStages) & 1;
      pos += pv;
      const uint32_t ks = pos % kStages, k_par = (pos / kStages) & 1;
      pos += more;
      uint64_t *v_full = bars.kv_full() + vs, *k_full = bars.kv_full() + ks;
      const bool here = (!pv || mbar_try_wait(v_full, v_par)) & (!more || mbar_try_wait(k_full, k_par));
      if (!__all_sync(0xffffffffu, here)) {
        if (pv && !wait(v_full, v_par)) return false;
        if (more && !wait(k_full, k_par)) return false;
      }
      // A parity tells one phase of a stage from the next, not from the one after:
      // the other warp's tiles are waited for as well, and released by both.
      if (!kTwo && (i & 1) != t) {
        if (lane == 0) {
          if (pv) mbar_arrive(bars.kv_empty() + vs);
          if (more) mbar_arrive(bars.kv_empty() + ks);
        }
        __syncwarp();
        continue;
      }
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        const bool first = i < kLead && part == 0, last = part == kParts - 1;
        const uint32_t col = colS + part * kPart;
        if (pv) {
          if (first) {  // O is overwritten: the previous segment's must have been read
            if (!wait(o_empty, o_par)) return false;
            o_par ^= 1;
          }
          if (!wait(p_full + part, p_par)) return false;
          tc_fence_after();
        }
        if (elect_one()) {
          if (pv) {
            const uint64_t vd = v_desc + vs * (kTile >> 4) + part * (kPart * 128 >> 4);
#pragma unroll
            for (int k = 0; k < kPart / 16; ++k)
              umma_f16_ts(colO, col + k * 8, vd + k * 128, kIdescPV, (!first || k > 0) ? 1u : 0u);
            umma_commit(pv_done);
            if (last) {
              if (!more) umma_commit(o_full);
              umma_commit(bars.kv_empty() + vs);
            }
          }
          if (more) {
            const uint64_t qd = q_desc + kTwo * t * (kTile >> 4);
            const uint64_t kd = k_desc + ks * (kTile >> 4) + part * (kPart * 128 >> 4);
#pragma unroll
            for (int k = 0; k < kD / 16; ++k) {
              const int o = ((k >> 2) * kHalf + (k & 3) * 32) >> 4;
              umma_f16_ss(col, qd + o, kd + o, kIdescQK, k > 0 ? 1u : 0u);
            }
            umma_commit(s_full + part);
            if (last) {
              umma_commit(bars.kv_empty() + ks);
              if (i + 2 * kLead >= n) umma_commit(bars.q_empty());  // this warp's last S of the segment
            }
          }
        }
        __syncwarp();
      }
      p_par ^= pv;
    }
    if (!kTwo && t >= n && lane == 0) mbar_arrive(bars.q_empty());  // it had none
    return true;
  };
  do {
    if (!wait(bars.q_full(), segs++ & 1)) break;
    if (!(uniform(e.two) ? segment(Pair<1>{}) : segment(Pair<0>{}))) break;
  } while (walk_next(p, tab, w, e));
  __syncwarp();
}

// What the combine pass has to read of each row, and whether the groups are
// sound; one warp of the grid.
__device__ __forceinline__ void write_flags(const Params& p, const PrefixGroup* tab, int lane) {
  for (int g = lane; g < p.own.groups.n; g += 32) {
    const int lo = p.own.groups.cu[g], hi = p.own.groups.cu[g + 1];
    if (p.own.err && (lo < 0 || hi < lo || hi > p.own.batch)) atomicCAS(p.own.err, 0, LA_DEVERR_PREFIX);
  }
  for (int b = lane; b < p.own.batch; b += 32) {
    int block0;
    const int own = decode::own_keys<true>(p.own, tab, b, &block0);
    p.flags[b] = (block0 > 0 ? kShares : 0) | (own > 0 ? kOwn : 0);
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    shared_prefix_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap own_q,
                         const __grid_constant__ CUtensorMap own_k, const __grid_constant__ CUtensorMap own_v,
                         const __grid_constant__ CUtensorMap own_k1, const __grid_constant__ CUtensorMap own_v1,
                         const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const Bars bars{reinterpret_cast<uint64_t*>(smem)};
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kOffTmem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kOffOwnBar);
  uint64_t* empty = full + decode::kMaxStages;
  uint64_t* mg_full = empty + decode::kMaxStages;  // all consumer warps wrote their state
  uint64_t* mg_empty = mg_full + 1;                // the merging warp read it
  PrefixGroup* tab = reinterpret_cast<PrefixGroup*>(smem + kOffTable);
  Plan& plan = *reinterpret_cast<Plan*>(smem + kOffPlan);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // Barriers and tensor memory: nothing that a kernel before this one writes.
  if (warp == kWarpSecond && lane == 0) {
    mbar_init(bars.q_full(), 1);
    mbar_init(bars.q_empty(), 2);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bars.kv_full() + i, 1);
      mbar_init(bars.kv_empty() + i, 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars.pv_done() + i, 1);
      mbar_init(bars.o_full() + i, 1);
      mbar_init(bars.o_empty() + i, 128);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bars.s_full() + i, 1);
      mbar_init(bars.p_full() + i, 128);
    }
    mbar_init(bars.planned(), 1);
    mbar_init(bars.checked(), 1);
    mbar_init(bars.done(), 8);
    mbar_init(bars.again(), kThreads / 32 - 1);
    for (int s = 0; s < 3; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], decode::kCWarps);
    }
    mbar_init(mg_full, decode::kCWarps);
    mbar_init(mg_empty, p.own.hkv);
    fence_barrier_init();
  }
  if (warp == kWarpSecond) reinterpret_cast<uint32_t*>(smem + kOffZero)[lane] = 0u;
  if (warp == kWarpProduct) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  if (warp == kWarpLoad && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&own_q);
    tma_prefetch_desc(&own_k);
    tma_prefetch_desc(&own_v);
  }
  // The plan is made before the wait for the kernel in front, from the lengths
  // and groups as they are, and checked after it; if they changed, it is made
  // again. Beyond 256 rows or 32 groups it is made after the wait (257 rows behind
  // 2048 keys take 65 us, 256 of them 53).
  const bool early = p.own.batch <= 256 && p.own.groups.n <= 32;
  volatile int* stale = reinterpret_cast<volatile int*>(smem + kOffStale);
  Seen in;
  if (warp == kWarpPlan && early) in = read_inputs(p, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (!early) grid_dependency_wait();

  // Round 0 with the plan; before anything is done by it, the check has to be
  // back. If the plan was stale, round 1 with the new one, which is made when
  // all warps have left the old one.
  // (A round through each warp's code before the plan was there, to fetch it
  // into the instruction caches, made every size 3 to 35 % slower.)
  auto leave_plan = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(bars.again());
  };
  if (warp < 8) {
    bool ok = false;
    for (uint32_t round = 0; round < 2; ++round) {
      if (!wait_warp(p, bars.planned(), round)) break;
      grid_dependency_wait();
      if (round == 0) {
        if (!wait_warp(p, bars.checked(), 0)) break;
        if (*stale) {
          leave_plan();
          continue;
        }
      }
      ok = true;
      break;
    }
    if (ok && plan.shared)
      softmax_warp(p, tab, plan, smem, bars, tmem, warp >> 2, warp, lane);
    else if (ok)
      decode::consume<0, true>(p.own, smem + kCtrlBytes, full, empty,
                                        reinterpret_cast<const decode::StageDesc*>(smem + kOffDesc), smem + kOffZero,
                                        mg_full, mg_empty,
                                        reinterpret_cast<float*>(smem + kCtrlBytes + p.stages * p.own.stage_bytes),
                                        plan.u1 - plan.u0, warp, lane, p.stages);
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bars.done());
  } else {
    const bool maker = warp == kWarpPlan;
    Walk w;
    Segment e{};
    Pages pages;
    decode::Windows<true> win;
    win.tab = tab;
    for (uint32_t round = 0; round < 2; ++round) {
      if (maker) {
        const Plan r = early ? make_plan(p, tab, in, lane) : make_large_plan(p, tab, lane);
        __syncwarp();  // the entries of `tab` are all lanes' stores, lane 0 arrives for them
        if (lane == 0) {
          plan = r;
          mbar_arrive(bars.planned());
        }
        __syncwarp();
      } else if (!wait_warp(p, bars.planned(), round)) {
        break;
      }
      bool work = plan.shared ? !maker : plan.u1 > plan.u0 && warp >= kWarpPlan;
      if (work && plan.shared) {
        walk_start(p, tab, plan, w);
        work = walk_next(p, tab, w, e);
      }
      grid_dependency_wait();
      if (warp >= kWarpPlan) grid_launch_dependents();  // the combine pass waits for this grid's end before it reads
      if (maker && round == 0) {
        bool same = true;
        if (early) {
          const Seen now = read_inputs(p, lane);
          same = now.lo == in.lo && now.hi == in.hi && now.len == in.len;
#pragma unroll
          for (int i = 0; i < 8; ++i) same &= now.raw[i] == in.raw[i];
          same = __all_sync(0xffffffffu, same);
          in = now;
        }
        if (lane == 0) {
          *stale = !same;
          mbar_arrive(bars.checked());
        }
        __syncwarp();
      }
      if (work && !plan.shared) {
        win.load_swin(p.own, lane, plan.at);
        win.load_bwin(p.own, lane, plan.at,
                      static_cast<int>((plan.u0 - plan.before) * p.own.tc / p.own.block_size));
      } else if (work && warp == kWarpLoad) {
        pages.start(p, e, lane);
      }
      if (round == 0) {
        if (!wait_warp(p, bars.checked(), 0)) break;
        if (*stale) {
          if (!maker)
            leave_plan();
          else if (!wait_warp(p, bars.again(), 0))
            break;
          continue;
        }
      }
      if (work) {
        if (!plan.shared)
          decode::produce<0, true>(own_q, own_k, own_v, own_k1, own_v1, p.own, smem + kCtrlBytes, full, empty,
                                            reinterpret_cast<decode::StageDesc*>(smem + kOffDesc), win, plan.u0,
                                            plan.u1 - plan.u0, plan.at, plan.before, plan.c, maker ? 1 : 0, 2, lane,
                                            p.stages);
        else if (warp == kWarpLoad)
          load_warp(tm_q, tm_k, tm_v, p, tab, smem, bars, w, e, pages, lane);
        else
          product_warp(p, tab, smem, bars, tmem, warp == kWarpSecond, w, e, lane);
      }
      break;
    }
    if (warp == kWarpProduct) {
      // tensor memory is read by the eight warps until they are through
      wait_warp(p, bars.done(), 0);
      tc_fence_after();
      tmem_dealloc(tmem, kTmemCols);
    } else if (blockIdx.x == 0 && warp == (plan.shared ? kWarpPlan : kWarpLoad)) {
      write_flags(p, tab, lane);
    }
  }
}

// ------------------------------------------------------------------ combine
// kSplit: a CTA per (row, query head), whose four warps take every fourth run
// of 16 of the row's parts, and the first joins the warps' results; where there
// are enough rows and heads to fill the SMs, a warp for each. Lane l owns dims
// 4l..4l+3. The row's parts are those of its group's item, one per CTA that
// had a segment of it (two where the accumulators took alternate key tiles),
// and those of its own keys. In a run the weights come from a maximum over
// the lanes that hold the logarithms, and the O rows are requested together
// with them. Bound by the latency of its three dependent reads (one row over
// 148 parts in one warp took 20 us).
constexpr int kRun = 16;
constexpr int kCombineWarps = 4;

struct CombineParams {
  const int* flags;
  const int2* row_parts;
  const int4* items;
  int hq, hkv, group;
  int grid;   // CTAs that parts come from, at most
  int own0;   // first partial row of the rows' own keys
  int rows;   // all partial rows
  const float* part_o;
  const float* part_lse;
  __nv_bfloat16* out;
  long long out_bs, out_hs;
  float* lse;
};

template <bool kSplit>
__global__ void __launch_bounds__(32 * kCombineWarps) combine_kernel(const CombineParams p) {
  __shared__ float4 s_acc[kCombineWarps - 1][32];
  __shared__ float2 s_ml[kCombineWarps - 1];
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.x, hh = kSplit ? blockIdx.y : blockIdx.y * kCombineWarps + (threadIdx.x >> 5);
  const int warp = kSplit ? threadIdx.x >> 5 : 0;
  constexpr int kWarps = kSplit ? kCombineWarps : 1;
  const int h = hh / p.group;
  const float NEG_INF = -__int_as_float(0x7f800000);
  grid_dependency_wait();
  grid_launch_dependents();
  if (hh >= p.hq) return;
  const int flags = p.flags[b];
  const int2 rp = p.row_parts[b];
  const int4 it = p.items[static_cast<long long>(b) * p.hkv + h];
  // Groups that are reported as unsound leave entries unwritten: whatever they
  // hold, the reads below stay inside the workspace.
  int pn = 0, own = 0;
  if (flags & kShares) pn = max(0, min(it.w - it.z + 1, p.grid)) * (it.y ? 2 : 1);
  if (flags & kOwn) own = max(0, min(rp.y - rp.x + 1, p.grid));
  if (!(flags & kShares) && own == 1) return;  // written by the CTA that read the row
  const int n = pn + own;
  float m = NEG_INF, l = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int e0 = warp * kRun; e0 < n; e0 += kWarps * kRun) {
    const int x = e0 + (lane & (kRun - 1));
    int row = 0;
    if (x < pn)
      row = it.x + hh - h * p.group + (it.y ? (x >> 1) * 2 * kRows + (x & 1) * it.y : x * 2 * kRows);
    else if (x < n)
      row = p.own0 + (b + rp.x + x - pn) * p.hq + hh;
    row = min(max(row, 0), p.rows - 1);
    const float ls = x < n ? p.part_lse[row] : NEG_INF;
    float4 ov[kRun];
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      const int r = __shfl_sync(0xffffffffu, row, k);
      ov[k] = e0 + k < n ? *reinterpret_cast<const float4*>(p.part_o + static_cast<long long>(r) * kD + lane * 4)
                         : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // A part without keys has -inf and is left out by a test, never by a
    // weight of 0, so whatever its row holds does not count; NaN counts.
    const bool use = x < n && ls != NEG_INF;
    const unsigned usem = __ballot_sync(0xffffffffu, use);
    if (usem == 0) continue;
    float mr = use ? ls : NEG_INF;
#pragma unroll
    for (int o = kRun / 2; o > 0; o >>= 1) mr = fmaxf(mr, __shfl_xor_sync(0xffffffffu, mr, o));
    const float mn = fmaxf(m, mr);
    const float a = ex2(m - mn);
    const float wl = use ? ex2(ls - mn) : 0.f;
    float ws = wl;
#pragma unroll
    for (int o = kRun / 2; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
    l = l * a + ws;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] *= a;
    m = mn;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      const float wk = __shfl_sync(0xffffffffu, wl, k);
      if ((usem >> k) & 1u) {
        acc[0] += wk * ov[k].x;
        acc[1] += wk * ov[k].y;
        acc[2] += wk * ov[k].z;
        acc[3] += wk * ov[k].w;
      }
    }
  }
  if (kSplit && n > kRun) {  // the other warps' results, in their order
    if (warp > 0) {
      s_acc[warp - 1][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (lane == 0) s_ml[warp - 1] = make_float2(m, l);
    }
    __syncthreads();
  }
  if (warp > 0) return;
  for (int w = 1; w * kRun < n && w < kWarps; ++w) {
    const float2 ml = s_ml[w - 1];
    const float4 o = s_acc[w - 1][lane];
    if (ml.y == 0.f) continue;
    const float mn = fmaxf(m, ml.x);
    const float a = l == 0.f ? 0.f : ex2(m - mn), c = ex2(ml.x - mn);
    acc[0] = acc[0] * a + o.x * c;
    acc[1] = acc[1] * a + o.y * c;
    acc[2] = acc[2] * a + o.z * c;
    acc[3] = acc[3] * a + o.w * c;
    l = l * a + ml.y * c;
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint2 v;
  v.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  v.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<uint2*>(p.out + b * p.out_bs + hh * p.out_hs + lane * 4) = v;
  if (p.lse && lane == 0)
    p.lse[static_cast<long long>(b) * p.hq + hh] = l == 0.f ? NEG_INF : (m + __log2f(l)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ host
// The workspace: partial rows of the shared part and of the rows' own keys
// (O, then logarithms), and what the combine pass reads of each row.
struct Workspace {
  int64_t own0, rows;              // partial rows
  size_t lse, items, parts, flags;  // byte offsets; part_o is at 0
  size_t bytes;
};

static Workspace workspace_of(int64_t batch, int hq, int hkv, int64_t grid) {
  Workspace w;
  w.own0 = 2 * batch * hq + 2 * kRows * grid;
  w.rows = w.own0 + (batch + grid) * hq;
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  w.lse = up(static_cast<size_t>(w.rows) * kD * sizeof(float));
  w.items = up(w.lse + static_cast<size_t>(w.rows) * sizeof(float));
  w.parts = up(w.items + static_cast<size_t>(batch) * hkv * sizeof(int4));
  w.flags = up(w.parts + static_cast<size_t>(batch) * sizeof(int2));
  w.bytes = up(w.flags + static_cast<size_t>(batch) * sizeof(int));
  return w;
}

}  // namespace prefix

int prefix_init(int device) {
  (void)device;
  cudaError_t e = cudaFuncSetAttribute(prefix::shared_prefix_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       227 * 1024);
  cudaFuncAttributes a;
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, prefix::combine_kernel<true>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, prefix::combine_kernel<false>);
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
  const Workspace w = workspace_of(batch, num_q_heads, num_kv_heads, grid);
  if (w.rows > 0x7fffffffLL) return LA_ERR_UNSUPPORTED;
  *bytes = w.bytes;
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
  if (num_groups < 0 || (num_groups > 0 && (!prefix_lens || !cu_prefix_rows))) return LA_ERR_INVALID_ARGUMENT;
  decode::Call call;
  int st = decode::prepare_call(q, q_batch_stride, q_head_stride, k_cache, v_cache, kv_block_stride, kv_token_stride,
                                kv_head_stride, num_blocks, block_size, block_table, bt_seq_stride, max_blocks_per_seq,
                                cache_seqlens, batch, num_q_heads, num_kv_heads, head_dim, softmax_scale, out,
                                out_batch_stride, out_head_stride, softmax_lse, dev_error, &call);
  if (st != LA_OK || batch == 0) return st;
  if (num_blocks > 0x7ffffffeLL) return LA_ERR_UNSUPPORTED;
  const int device = current_device();
  const int grid = device >= 0 ? num_sms(device) & ~1 : 0;  // take_part and shared_ctas deal in pairs
  if (grid <= 0) return LA_ERR_CUDA;
  if (grid < 4) return LA_ERR_UNSUPPORTED;  // a pair for each part
  const Workspace w = workspace_of(batch, num_q_heads, num_kv_heads, grid);
  if (w.rows > 0x7fffffffLL) return LA_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < w.bytes || !aligned(workspace, 256)) return LA_ERR_WORKSPACE;
  if (num_groups == 0 || batch < 2)  // nothing to share; the workspace is larger than that call's
    return la_paged_decode(q, q_batch_stride, q_head_stride, k_cache, v_cache, kv_block_stride, kv_token_stride,
                           kv_head_stride, num_blocks, block_size, block_table, bt_seq_stride, max_blocks_per_seq,
                           cache_seqlens, batch, num_q_heads, num_kv_heads, head_dim, softmax_scale, out,
                           out_batch_stride, out_head_stride, softmax_lse, workspace, workspace_bytes, dev_error, stream);

  const int group = num_q_heads / num_kv_heads, per_tile = kRows / group;
  PrefixGroups& groups = call.p.groups;
  groups.cu = cu_prefix_rows;
  groups.lens = prefix_lens;
  groups.n = num_groups;
  groups.batch = batch;
  groups.block_size = block_size;
  groups.bs_shift = call.p.bs_shift;
  groups.cap = static_cast<int64_t>(max_blocks_per_seq) * block_size;
  if (groups.cap > 0x7fff0000LL) groups.cap = 0x7fff0000LL / block_size * block_size;  // lengths are int32
  // steps of all groups and units of 256 rows are counted in 32 bits
  const int64_t key_tiles = (groups.cap + kKeys - 1) / kKeys, most_groups = num_groups < batch ? num_groups : batch;
  if (key_tiles * num_kv_heads * (batch / (2 * per_tile) + most_groups) > 0x7fffffffLL ||
      256 * (groups.cap / call.p.tc + 1) > 0x7fffffffLL || batch > (1 << 24))
    return LA_ERR_UNSUPPORTED;

  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Params p;
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_lse = reinterpret_cast<float*>(ws + w.lse);
  p.items = reinterpret_cast<int4*>(ws + w.items);
  p.flags = reinterpret_cast<int*>(ws + w.flags);
  call.p.part_o = p.part_o + w.own0 * kD;
  call.p.part_lse = p.part_lse + w.own0;
  call.p.row_parts = reinterpret_cast<int*>(ws + w.parts);
  p.own = call.p;
  p.per_tile = per_tile;
  p.tile_magic = static_cast<uint32_t>(((1ull << 32) + per_tile - 1) / per_tile);
  p.box_keys = kKeys;
  while (block_size % p.box_keys) p.box_keys >>= 1;

  CUtensorMap tq, tk, tv;
  {
    const uint64_t dims[3] = {128, static_cast<uint64_t>(num_q_heads), static_cast<uint64_t>(batch)};
    const uint64_t strides[2] = {static_cast<uint64_t>(q_head_stride) * 2, static_cast<uint64_t>(q_batch_stride) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(group), static_cast<uint32_t>(per_tile)};
    if ((st = encode_tensor_map_bf16(&tq, q, 3, dims, strides, box, true)) != LA_OK) return st;
  }
  {
    const uint64_t dims[4] = {128, static_cast<uint64_t>(block_size), static_cast<uint64_t>(num_kv_heads),
                              static_cast<uint64_t>(num_blocks)};
    const uint64_t strides[3] = {static_cast<uint64_t>(kv_token_stride) * 2, static_cast<uint64_t>(kv_head_stride) * 2,
                                 static_cast<uint64_t>(kv_block_stride) * 2};
    const uint32_t box[4] = {64, static_cast<uint32_t>(p.box_keys), 1, 1};
    if ((st = encode_tensor_map_bf16(&tk, k_cache, 4, dims, strides, box, true)) != LA_OK) return st;
    if ((st = encode_tensor_map_bf16(&tv, v_cache, 4, dims, strides, box, true)) != LA_OK) return st;
  }
  const size_t two = kCtrlBytes + 2 * static_cast<size_t>(call.p.stage_bytes) + call.merge_bytes + 1024;
  p.stages = two + call.p.stage_bytes <= 227 * 1024 ? 3 : 2;
  const size_t own = two + (p.stages - 2) * static_cast<size_t>(call.p.stage_bytes);
  const size_t smem = own > kSmemBytes ? own : kSmemBytes;
  if (smem > 227 * 1024) return LA_ERR_UNSUPPORTED;
  st = cuda_status(launch_pdl(shared_prefix_kernel, dim3(grid), dim3(kThreads), smem, stream, tq, tk, tv, call.q, call.k,
                              call.v, call.k1, call.v1, p));
  if (st != LA_OK) return st;

  CombineParams c;
  c.flags = p.flags;
  c.row_parts = reinterpret_cast<const int2*>(ws + w.parts);
  c.items = p.items;
  c.hq = num_q_heads;
  c.hkv = num_kv_heads;
  c.group = group;
  c.grid = grid;
  c.own0 = static_cast<int>(w.own0);
  c.rows = static_cast<int>(w.rows);
  c.part_o = p.part_o;
  c.part_lse = p.part_lse;
  c.out = static_cast<__nv_bfloat16*>(out);
  c.out_bs = out_batch_stride;
  c.out_hs = out_head_stride;
  c.lse = softmax_lse;
  // A row has about #SMs parts over the number of rows: one warp goes through
  // them as fast as four once the rows and heads are four per SM.
  const bool split = static_cast<int64_t>(batch) * num_q_heads < 4 * grid;
  return cuda_status(launch_pdl(split ? combine_kernel<true> : combine_kernel<false>,
                                dim3(batch, split ? num_q_heads : (num_q_heads + kCombineWarps - 1) / kCombineWarps),
                                dim3(32 * kCombineWarps), 0, stream, c));
}
