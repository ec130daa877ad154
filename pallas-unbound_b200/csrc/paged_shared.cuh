// paged_shared.cuh — attention of one new token a sequence over a paged cache
// whose sequences hold the same first pages: those are read once for all of
// them.
//
// No counterpart in the reference (each sequence's dense cache is read whole,
// src/pallas_flash/kernels/decoding.py:86-115).
//
// A group's sequences times the query heads of one K/V head are the rows of an
// attention over the shared tokens:
//   S [rows x tokens] = Q K^T,  O [rows x D] = exp(S - m) V,
// 4 rows P D flops on 4 P D bytes of 16-bit pages, so from about 250 rows on
// (the ridge) it is bound by the tensor core and the exponents instead of the
// pages.  Three launches: the prefix (this file), each sequence's own tokens
// (paged_tc.cuh, in fp32), and the join of both by their maxima and sums.
//
// The prefix.  An item is (group, K/V head, 256 rows); its tiles of 128 tokens
// and those of all items, each item's cost of starting before them, lie in one
// line that is cut into as many equal parts as there are CTAs (one an SM), so
// lengths that the host does not know load every SM alike.  A CTA's run of one
// item's tiles leaves a record (m, l, O in fp32) of its 256 rows.
//
//   warps 0-7    softmax, a warpgroup for each of two slots; thread r owns row r
//                (TMEM lane r).  More than 128 rows: slot t takes rows 128 t and
//                on, every tile is used by both.  Fewer: both slots take the same
//                rows and every other tile, and leave two records.  Either way
//                products alternate between the slots, so the tensor core has one
//                slot's work while the other is in its exponents.
//   warp 8       page table lookups and TMA loads
//   warp 9       tcgen05 issue: S of job k + 2 behind P V of job k
//   warps 12-15  e4m3 pools: tiles as stored are staged and turned into f16
//                operands (every e4m3 value is an f16 value), which costs less
//                than splitting 128 x 128 weights into e4m3 parts; q as f16,
//                scaled by a power of two for each row if it is bf16
// P goes back over S's columns of TMEM as the product's left operand, rounded
// once to the operands' type; sums and maxima are fp32.
#pragma once

#include <cfloat>

#include "paged_tc.cuh"

namespace pu {
namespace decode {
namespace shared {

constexpr int BT = 128;                  // tokens of a tile
constexpr int kRows = 256;               // rows of an item
constexpr int kMaxGroups = 64;
constexpr int kItemCost = 2;             // what starting and ending an item costs, in tiles
// Whether sharing pays.  A pass over shared tokens and its join cost 8 to 12 us before their first tile, and each
// tile of 128 rows as much as 2 tiles that a sequence reads by itself (64 KB of keys and values, spread over all CTAs, from
// L2 where they fit), or 4 of 32 KB (heads of 64, e4m3).  A group for which that is more than its sequences' own
// tiles shares nothing, nor does a call that saves fewer than kWorth tiles.  Measured, shared against not, tiles saved:
//   64 KB: 4 sequences behind 8192 tokens 36.3 us, 30.7 (1024), 24 behind 1024 33.2, 31.4 (1408), 32: 34.6, 35.2 (1920),
//     40: 36.4, 39.0 (2304), 64: 44.2, 53.2 (3840), 256 behind 128 72.5, 78.3 (1920), 2 behind 40960 65.6, 62.0 (0)
//   32 KB: e4m3, 16 behind 2048 34.3, 31.4 (1536), 20: 36.5, 34.4 (2048), 24: 37.0, 37.8 (2560), 4 behind 16384 48.5, 37.4 (0);
//     heads of 64, 80 behind 2048 33.0, 31.5 (1920), 96: 32.1, 34.3 (2304)
constexpr int kWorth = 2048;
constexpr int kBadRing = 8;

template <typename T, typename KVT, int D>
struct Cfg {
  static constexpr bool kF8 = sizeof(KVT) == 1;
  using Op = typename std::conditional<kF8, __half, T>::type;          // operands of the products
  static constexpr bool kBf16 = std::is_same<Op, __nv_bfloat16>::value;
  // P = 2^(s - m), m = the maximum - kShift, moved once a score passes the maximum by kRescale:
  // f16 weights then use the range of their type, bf16 has fp32's
  static constexpr float kRescale = 8.f, kShift = kBf16 ? 0.f : 7.f;
  static constexpr int kThreads = kF8 ? 512 : 384;
  static constexpr int kSoftmaxRegs = kF8 ? 192 : 208, kRoleRegs = kF8 ? 56 : 88, kConvertRegs = 72;
  static constexpr int kBlocks = D / 64;                               // 128-byte swizzle blocks of a 16-bit row
  static constexpr int kTile = BT * D * 2;
  static constexpr int kTile8 = BT * D;                                // a staged e4m3 tile
  static constexpr int NK = D == 64 ? 4 : 2, NV = kF8 ? 1 : NK;        // 16-bit tiles of K and V
  static constexpr int NS = kF8 ? 2 : 0;                               // staged pairs
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + 2 * kTile;
  static constexpr int kOffV = kOffK + NK * kTile;
  static constexpr int kOffStage = kOffV + NV * kTile;
  static constexpr int kOffBar = kOffStage + NS * 2 * kTile8;
  // Kf[NK] Ke[NK] Vf[NV] Ve[NV] K8f K8e V8f V8e [NS each] S[2] P[2] O[2] Of[2] Q Qe drain
  static constexpr int kBars = 2 * NK + 2 * NV + 4 * NS + 8 + 3;
  static constexpr int kOffMisc = kOffBar + kBars * 8;                 // tmem base, abort flag
  static constexpr int kOffBad = kOffMisc + 8;                         // [kBadRing] which 16 tokens of a tile were not loaded
  static constexpr int kOffScale = kOffBad + kBadRing * 4;             // [2 runs][kRows] exponent of what undoes a row's scale (e4m3)
  static constexpr int kOffGroups = (kOffScale + (kF8 ? 2 * kRows : 0) + 7) / 8 * 8;
  static constexpr int kSmem = kOffGroups + 16 * (kMaxGroups + 1);
  static_assert(kSmem <= 232448, "shared memory of one CTA");
};

// TMEM columns of slot t
__host__ __device__ constexpr uint32_t col_s(int t) { return 128u * t; }
__host__ __device__ constexpr uint32_t col_o(int t) { return 256u + 128u * t; }

// A group as every CTA works it out and the join reads it.
struct Group {
  int start;                   // first sequence
  int tokens;                  // shared tokens, whole pages; 0: nothing is shared
  int rep;                     // the sequence whose table row is read
  int unit;                    // first unit of the line
};
static_assert(sizeof(Group) == 16, "");

struct Params {
  const void* q;               // [B][H][D]
  const int32_t* table;        // [B][max_pages]
  const int32_t* lens;         // [B]
  const int32_t* shared_lens;  // [groups]
  const int32_t* starts;       // [groups + 1] or nullptr: one group of all
  int32_t* skip;               // [B] tokens of each sequence that the prefix pass takes
  int32_t* in_group;           // [B] and its group
  int32_t* own_lens;           // [B] and those that are left
  Group* desc;                 // [kMaxGroups + 1]
  float* slabs;                // records
  int B, H, H_kv, group, slices, groups;
  int max_pages, num_pages, page_shift, box;
  int pass_cost;               // a tile of 128 rows of the prefix pass, in tiles that a sequence reads by itself
  float scale_log2;
};

// A record: {m, l} of 256 rows, then O in columns of four: [D / 4][256][4], so that a warp of
// consecutive rows writes and reads whole lines.
template <int D>
constexpr size_t kSlab = (size_t)kRows * (D + 2);

// The line of units and its parts.
struct Line {
  int q, rem, ctas;
  __device__ __forceinline__ Line(int units, int grid) {
    ctas = min(units, grid);
    q = ctas > 0 ? units / ctas : 0;
    rem = units - q * ctas;
  }
  __device__ __forceinline__ int part(int c) const { return c * q + min(c, rem); }
  // the part that holds unit x
  __device__ __forceinline__ int holder(int x) const {
    const int big = rem * (q + 1);
    return x < big ? x / (q + 1) : rem + (x - big) / q;
  }
};

__device__ __forceinline__ int tiles_of(const Group& g) { return (g.tokens + BT - 1) / BT; }

// Items of the groups before g.
__device__ __forceinline__ int items_before(const Group* gs, int g) {
  int n = 0;
  for (int i = 0; i < g; ++i) {
    const int tiles = tiles_of(gs[i]);
    if (tiles > 0) n += (gs[i + 1].unit - gs[i].unit) / (tiles + kItemCost);
  }
  return n;
}

// A CTA's runs of tiles, one item after the other.
struct Walk {
  const Group* groups;
  int H_kv, group, unit, end;            // units of the part that are left
  int g, r, pairs, tiles, t0, n, item;   // this run: group, item of it, tiles [t0, t0 + n)
  int rows;                              // rows of the item, up to 256
  int seg;
  bool split;                            // both slots on the same rows
  __device__ __forceinline__ Walk(const Group* gs, int H_kv_, int group_, int u0, int u1)
      : groups(gs), H_kv(H_kv_), group(group_), unit(u0), end(u1), g(0), seg(-1) {}
  // to the next run with tiles; false when there is none
  __device__ __forceinline__ bool next() {
    while (unit < end) {
      while (groups[g + 1].unit <= unit) ++g;
      const Group& a = groups[g];
      tiles = tiles_of(a);
      const int all = (groups[g + 1].start - a.start) * group;
      pairs = (all + kRows - 1) / kRows;
      const int per = tiles + kItemCost, in = unit - a.unit;
      r = in / per;
      const int first = a.unit + r * per + kItemCost;      // unit of the item's first tile
      t0 = max(unit, first) - first;
      const int stop = min(end, first + tiles);
      n = stop - (first + t0);
      unit = stop;
      if (n <= 0) {
        unit = max(unit, min(end, first));
        continue;
      }
      rows = min(kRows, all - (r % pairs) * kRows);
      split = rows <= kRows / 2;
      ++seg;
      return true;
    }
    return false;
  }
  __device__ __forceinline__ int head() const { return r / pairs; }
  __device__ __forceinline__ int row0() const { return (r % pairs) * kRows; }
  __device__ __forceinline__ int jobs() const { return split ? n : 2 * n; }
};

// Which group holds sequence b (-1: none).
__device__ __forceinline__ int group_of(const Group* gs, int groups, int b) {
  int a = -1, z = groups;                // last g with start <= b
  while (z - a > 1) {
    const int m = (a + z) >> 1;
    if (gs[m].start <= b) a = m;
    else z = m;
  }
  return a >= 0 && b < gs[a + 1].start ? a : -1;
}

// Groups from the caller's arrays, checked so that nothing below can leave its bounds: starts in
// order and inside the batch, shared tokens in whole pages that a sequence of the group holds.
__device__ __forceinline__ void make_groups(const Params& p, Group* gs, int tid, int threads) {
  const int lane = tid & 31;
  if (tid < 32) {
    int top = 0;                         // largest start so far
    for (int base = 0; base <= p.groups; base += 32) {
      const int i = base + lane;
      int s = 0;
      if (i <= p.groups) s = p.starts != nullptr ? p.starts[i] : i == 0 ? 0 : p.B;
      s = max(0, min(s, p.B));
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, off);
        if (lane >= off) s = max(s, y);
      }
      s = max(s, top);
      top = __shfl_sync(0xffffffffu, s, 31);
      if (i <= p.groups) {
        gs[i].start = s;
        gs[i].rep = 0x7fffffff;
        gs[i].unit = 0;                  // for now: sequences that hold the shared tokens
        gs[i].tokens = i < p.groups ? max(0, min(p.shared_lens[i], p.max_pages << p.page_shift)) >> p.page_shift << p.page_shift : 0;
      }
    }
  }
  __syncthreads();
  for (int b = tid; b < p.B; b += threads) {
    const int g = group_of(gs, p.groups, b);
    if (g >= 0 && p.lens[b] >= gs[g].tokens) {
      atomicMin(&gs[g].rep, b);
      atomicAdd(&gs[g].unit, 1);
    }
  }
  __syncthreads();
  if (tid < 32) {
    // tiles that sharing saves; one sequence alone shares with nobody
    long long saved = 0;
    for (int i = lane; i < p.groups; i += 32) {
      const int rows = (gs[i + 1].start - gs[i].start) * p.group, holders = gs[i].unit;
      const long long less = (long long)holders * p.slices - (long long)((rows + kRows / 2 - 1) / (kRows / 2)) * p.pass_cost;
      if (holders < 2 || less <= 0) gs[i].tokens = 0;
      saved += less * tiles_of(gs[i]);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) saved += __shfl_xor_sync(0xffffffffu, saved, off);
    const bool worth = saved * p.H_kv >= kWorth;
    int before = 0;
    for (int base = 0; base <= p.groups; base += 32) {
      const int i = base + lane;
      int units = 0;
      if (i < p.groups) {
        if (!worth) gs[i].tokens = 0;
        const int all = (gs[i + 1].start - gs[i].start) * p.group;
        if (gs[i].tokens > 0) units = (all + kRows - 1) / kRows * p.H_kv * (tiles_of(gs[i]) + kItemCost);
      }
      int x = units;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
      }
      if (i <= p.groups) gs[i].unit = before + x - units;
      before += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, typename KVT, int D>
__global__ void __launch_bounds__(Cfg<T, KVT, D>::kThreads, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ Params p) {
  using C = Cfg<T, KVT, D>;
  using Op = typename C::Op;
  constexpr bool kF8 = C::kF8;
  constexpr int NK = C::NK, NV = C::NV, NS = C::NS, kTile = C::kTile;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(smem) & 1023u) {
    if (tid == 0) record_device_error(PU_ERR_UNSUPPORTED, kSiteDecodeTc);
    return;
  }
  uint8_t* sQ = smem + C::kOffQ;
  uint8_t* sK = smem + C::kOffK;
  uint8_t* sV = smem + C::kOffV;
  uint8_t* sStage = smem + C::kOffStage;
  uint64_t* bKf = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* bKe = bKf + NK;
  uint64_t* bVf = bKe + NK;
  uint64_t* bVe = bVf + NV;
  uint64_t* bK8f = bVe + NV;             // [NS] staged K landed
  uint64_t* bK8e = bK8f + NS;            // [NS] turned into an operand
  uint64_t* bV8f = bK8e + NS;
  uint64_t* bV8e = bV8f + NS;
  uint64_t* bS = bV8e + NS;              // [2] S of the slot's job
  uint64_t* bP = bS + 2;                 // [2] its P written (128 arrivals)
  uint64_t* bO = bP + 2;                 // [2] the slot's last P V of the run
  uint64_t* bOf = bO + 2;                // [2] its O read (128 arrivals)
  uint64_t* bQ = bOf + 2;                // queries of the run in shared memory (256 arrivals)
  uint64_t* bQe = bQ + 1;                // the run's last S done
  uint64_t* bDrain = bQe + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);
  volatile uint32_t* s_bad = reinterpret_cast<volatile uint32_t*>(smem + C::kOffBad);
  uint8_t* s_scale = smem + C::kOffScale;
  Group* s_groups = reinterpret_cast<Group*>(smem + C::kOffGroups);

  if (tid == 0) {
    for (int s = 0; s < NK; ++s) {
      mbar_init(bKf + s, kF8 ? 128 : 1);
      mbar_init(bKe + s, 1);
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(bVf + s, kF8 ? 128 : 1);
      mbar_init(bVe + s, 1);
    }
    for (int s = 0; s < NS; ++s) {
      mbar_init(bK8f + s, 1);
      mbar_init(bK8e + s, 128);
      mbar_init(bV8f + s, 1);
      mbar_init(bV8e + s, 128);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bS + t, 1);
      mbar_init(bP + t, 128);
      mbar_init(bO + t, 1);
      mbar_init(bOf + t, 128);
    }
    mbar_init(bQ, kRows);
    mbar_init(bQe, 1);
    mbar_init(bDrain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  grid_dep_wait();
  grid_dep_launch_dependents();
  make_groups(p, s_groups, tid, C::kThreads);
  const Line line(s_groups[p.groups].unit, (int)gridDim.x);
  if (blockIdx.x == 0) {
    // for the passes that follow
    for (int i = tid; i <= p.groups; i += C::kThreads) p.desc[i] = s_groups[i];
    for (int b = tid; b < p.B; b += C::kThreads) {
      const int g = group_of(s_groups, p.groups, b);
      // a sequence that holds fewer tokens than its group shares attends them by itself
      const int skip = g >= 0 && p.lens[b] >= s_groups[g].tokens ? s_groups[g].tokens : 0;
      p.skip[b] = skip;
      p.in_group[b] = g;
      p.own_lens[b] = max(0, min(p.lens[b], p.max_pages << p.page_shift) - skip);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int cta = (int)blockIdx.x;
  const bool work = cta < line.ctas;
  Walk w(s_groups, p.H_kv, p.group, work ? line.part(cta) : 0, work ? line.part(cta + 1) : 0);

  if (warp >= 8 && warp < 12) {
    reg_dealloc<C::kRoleRegs>();
    if (warp == 8) {
      // ---------------- pages -> shared memory ----------------
      // entries of 32 boxes at a time, the next 32 on their way
      const int box_shift = 31 - __clz(p.box), boxes = BT >> box_shift, batch = 32 / boxes;
      const int lane_tile = lane / boxes, lane_row = (lane & (boxes - 1)) << box_shift;
      int j = 0, begun[2] = {0, 0};      // tiles so far, K and V tiles whose copies were begun
      bool ok = true;
      while (ok && w.next()) {
        const Group& g = s_groups[w.g];
        const int32_t* table = p.table + (size_t)g.rep * p.max_pages;
        const int head = w.head(), t1 = w.t0 + w.n;
        auto look_up = [&](int t) -> int {
          const int tile = t + lane_tile, row = tile * BT + lane_row;
          return tile < t1 && row < g.tokens ? table[row >> p.page_shift] : -1;
        };
        int entries = look_up(w.t0), ahead = look_up(w.t0 + batch);
        for (int t = w.t0; ok && t < t1; ++t, ++j) {
          const int k = (t - w.t0) % batch;
          if (k == 0 && t > w.t0) {
            entries = ahead;
            ahead = look_up(t + batch);
          }
          const int pg = __shfl_sync(0xffffffffu, entries, (k * boxes + lane) & 31), row0 = t * BT;
          const bool mine = lane < boxes && row0 + lane_row < g.tokens, good = mine && (unsigned)pg < (unsigned)p.num_pages;
          if (mine && !good) record_device_error(PU_ERR_INVALID_ARGUMENT, kSiteDecodePage);
          const unsigned loaded = __ballot_sync(0xffffffffu, good);
          const unsigned bad = __ballot_sync(0xffffffffu, lane < BT / 16 && !((loaded >> ((lane * 16) >> box_shift)) & 1u));
          const int outer = pg * p.H_kv + head, in = p.box < BT ? 0 : row0 & ((1 << p.page_shift) - 1);
          const uint32_t bytes = (uint32_t)__popc(loaded) * p.box * D * (uint32_t)sizeof(KVT);
          int at[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) at[i] = __shfl_sync(0xffffffffu, outer, i);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            // 16-bit tiles go to their operand's place, e4m3 tiles are staged
            const int many = kF8 ? NS : kv == 0 ? NK : NV, s = j % many, turn = j / many;
            uint64_t* full = kF8 ? (kv == 0 ? bK8f : bV8f) + s : (kv == 0 ? bKf : bVf) + s;
            uint64_t* empty = kF8 ? (kv == 0 ? bK8e : bV8e) + s : (kv == 0 ? bKe : bVe) + s;
            uint8_t* dst = kF8 ? sStage + (2 * s + kv) * C::kTile8 : (kv == 0 ? sK : sV) + s * kTile;
            // one answer for the warp: a lane that gave up alone would leave the others at the next vote
            if (turn > 0) ok = __all_sync(0xffffffffu, mbar_wait(empty, (turn - 1) & 1, abort_flag, kSiteDecodeTc));
            if (!ok) break;
            begun[kv] = j + 1;
            if (elect_one_sync()) {
              if (kv == 0) s_bad[j % kBadRing] = bad;
              mbar_arrive_expect_tx(full, bytes);
              constexpr int cols = kF8 ? 128 : 64, blocks = kF8 ? 1 : C::kBlocks;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if ((loaded >> i) & 1u) {
#pragma unroll
                  for (int cb = 0; cb < blocks; ++cb)
                    tma_load_3d(dst + cb * BT * 128 + i * p.box * 128, kv == 0 ? &tmK : &tmV, full, cb * cols, in, at[i]);
                }
              }
            }
            __syncwarp();
          }
        }
      }
      // copies still in flight land before the CTA may exit
      volatile int no_abort = 0;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int many = kF8 ? NS : kv == 0 ? NK : NV;
        uint64_t* full = kF8 ? (kv == 0 ? bK8f : bV8f) : kv == 0 ? bKf : bVf;
        for (int i = max(0, begun[kv] - many); i < begun[kv]; ++i) mbar_wait(full + i % many, (i / many) & 1, &no_abort, kSiteDecodeTc);
      }
    } else if (warp == 9) {
      // ---------------- tcgen05 issue ----------------
      if (elect_one_sync()) {
        constexpr uint32_t idS = make_idesc_16(BT, BT, 0, 0, C::kBf16), idO = make_idesc_16(BT, D, 0, 1, C::kBf16);
        const uint64_t dQ0 = make_sdesc_sw128(smem_u32(sQ), 16, 1024);
        const uint64_t dK0 = make_sdesc_sw128(smem_u32(sK), 16, 1024);
        const uint64_t dV0 = make_sdesc_sw128(smem_u32(sV), BT * 128, 1024);
        int jk = 0, jv = 0;              // K and V tiles used so far
        int np[2] = {0, 0};              // P tiles of the slot used so far
        bool ok = true;
        while (ok && w.next()) {
          const int jobs = w.jobs(), step = w.split ? 0 : 1;       // job k: tile k >> step
          ok = mbar_wait(bQ, w.seg & 1, abort_flag, kSiteDecodeTc);
          auto issue_s = [&](int k) {
            const int t = k & 1, s = (jk + (k >> step)) % NK;
            if (w.split || t == 0) ok = ok && mbar_wait(bKf + s, ((jk + (k >> step)) / NK) & 1, abort_flag, kSiteDecodeTc);
            // the run's first product of a slot overwrites what the last run left there
            if (!ok) return;
            tc_fence_after();
            const uint64_t dq = sdesc_add(dQ0, w.split ? 0 : t * kTile), dk = sdesc_add(dK0, s * kTile);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = (kk >> 2) * (BT * 128) + (kk & 3) * 32;
              mma_ss(tmem + col_s(t), sdesc_add(dq, off), sdesc_add(dk, off), idS, kk > 0);
            }
            mma_commit(bS + t);
            if (w.split || t == 1) mma_commit(bKe + s);
            if (k + 1 == jobs) mma_commit(bQe);
          };
          issue_s(0);
          if (jobs > 1) issue_s(1);
          for (int k = 0; ok && k < jobs; ++k) {
            const int t = k & 1, j = jv + (k >> step), s = j % NV;
            if (w.split || t == 0) ok = ok && mbar_wait(bVf + s, (j / NV) & 1, abort_flag, kSiteDecodeTc);
            if (k < 2 && w.seg > 0) {
              // the slot's O of its last run has been read (a run of one job leaves slot 1 out: its threads arrive all the same)
              ok = ok && mbar_wait(bOf + t, (w.seg - 1) & 1, abort_flag, kSiteDecodeTc);
            }
            ok = ok && mbar_wait(bP + t, np[t] & 1, abort_flag, kSiteDecodeTc);
            if (!ok) break;
            ++np[t];
            tc_fence_after();
            const uint64_t dv = sdesc_add(dV0, s * kTile);
#pragma unroll
            for (int kk = 0; kk < BT / 16; ++kk)
              mma_ts(tmem + col_o(t), tmem + col_s(t) + kk * 8, sdesc_add(dv, kk * 16 * 128), idO, k > 1 || kk > 0);
            if (w.split || t == 1) mma_commit(bVe + s);
            if (k + 2 < jobs) issue_s(k + 2);
            else mma_commit(bO + t);
          }
          if (jobs == 1) mma_commit(bO + 1);
          jk += w.n;
          jv += w.n;
        }
        // every issued product completes before TMEM and shared memory go away
        mma_commit(bDrain);
        volatile int no_abort = 0;
        mbar_wait(bDrain, 0, &no_abort, kSiteDecodeTc);
      }
    }
  } else if (warp >= 12) {
    if constexpr (kF8) {
      reg_dealloc<C::kConvertRegs>();
      // ---------------- staged e4m3 tiles -> f16 operands ----------------
      const int row0 = (tid & 127) >> 3, c = tid & 7;          // 16 rows at a time, eight lanes a row
      int j = 0;
      bool ok = true;
      while (ok && w.next()) {
        for (int t = 0; ok && t < w.n; ++t, ++j) {
          const int s8 = j % NS;
          uint32_t bad = 0;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int many = kv == 0 ? NK : NV, s = j % many, turn = j / many;
            ok = mbar_wait((kv == 0 ? bK8f : bV8f) + s8, (j / NS) & 1, abort_flag, kSiteDecodeTc);
            if (ok && turn > 0) ok = mbar_wait((kv == 0 ? bKe : bVe) + s, (turn - 1) & 1, abort_flag, kSiteDecodeTc);
            if (!ok) break;
            if (kv == 0) bad = s_bad[j % kBadRing];
            const uint8_t* src = sStage + (2 * s8 + kv) * C::kTile8;
            uint8_t* dst = (kv == 0 ? sK : sV) + s * kTile;
#pragma unroll 2
            for (int r = row0; r < BT; r += 16) {
              uint4 x = *reinterpret_cast<const uint4*>(src + r * 128 + ((c ^ (r & 7)) << 4));
              if ((bad >> (r >> 4)) & 1u) x = make_uint4(0u, 0u, 0u, 0u);  // not loaded
              const uint32_t in[4] = {x.x, x.y, x.z, x.w};
              uint32_t out[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const __half2 h(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(in[i >> 1] >> (16 * (i & 1))), __NV_E4M3));
                out[i] = *reinterpret_cast<const uint32_t*>(&h);
              }
              // 32 bytes of f16: chunks 2 c and 2 c + 1, the upper half of the lanes the other way
              // round, or both halves' blocks would meet in the same banks
              const int flip = c >> 2;
              uint8_t* at = dst + (c >> 2) * (BT * 128) + r * 128;
              const uint4 a = make_uint4(out[0], out[1], out[2], out[3]), b = make_uint4(out[4], out[5], out[6], out[7]);
              const int ch = (2 * c) & 7;
              *reinterpret_cast<uint4*>(at + (((ch + flip) ^ (r & 7)) << 4)) = flip ? b : a;
              *reinterpret_cast<uint4*>(at + (((ch + 1 - flip) ^ (r & 7)) << 4)) = flip ? a : b;
            }
            fence_proxy_async_smem();
            mbar_arrive((kv == 0 ? bKf : bVf) + s);
            mbar_arrive((kv == 0 ? bK8e : bV8e) + s8);
          }
        }
      }
    }
  } else {
    reg_alloc<C::kSoftmaxRegs>();
    // ---------------- softmax ----------------
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_base + col_s(t), tO = tmem + lane_base + col_o(t);
    int js = 0;                          // jobs of this slot so far
    int j0 = 0;                          // tiles of the CTA so far
    while (w.next()) {
      const Group& g = s_groups[w.g];
      const int head = w.head(), row0 = w.row0();
      // ---- this slot's part of the queries ----
      if (w.seg > 0) mbar_wait(bQe, (w.seg - 1) & 1, abort_flag, kSiteDecodeTc);
      {
        constexpr int kVecs = D / 8, kStep = 128 / kVecs, kLoads = 128 / kStep;    // lanes of a row, rows at once
        const int c = row % kVecs, lo = (w.split ? t * 64 : t * 128) + row / kVecs;
        // sequence and query head of the first row; kStep rows on, without a division
        const int first = row0 + lo, dseq = kStep / p.group, dhead = kStep - dseq * p.group;
        int seq = first / p.group, at = first - seq * p.group;
        const T* q = static_cast<const T*>(p.q) + ((size_t)g.start * p.H + (size_t)head * p.group) * D + c * 8;
        uint4 v[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          v[u] = make_uint4(0u, 0u, 0u, 0u);
          if ((!w.split || u < kLoads / 2) && lo + u * kStep < w.rows) v[u] = *reinterpret_cast<const uint4*>(q + ((size_t)seq * p.H + at) * D);
          seq += dseq;
          at += dhead;
          if (at >= p.group) {
            at -= p.group;
            ++seq;
          }
        }
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          if (w.split && u >= kLoads / 2) break;
          const int r = lo + u * kStep;
          if constexpr (kF8) {
            float x[8];
            unpack8<T>(v[u], x);
            int down = 127;              // of 2^0
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
              // by a power of two that puts the row's largest |q| into [2^14, 2^15): bf16's 8 bits
              // are f16 values down to 2^-31 of it
              float mx = 0.f;
#pragma unroll
              for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fabsf(x[k]));
#pragma unroll
              for (int off = kVecs / 2; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
              const int e = (mx > 0.f && isfinite(mx)) ? ((__float_as_int(mx) >> 23) & 0xff) - 127 : 14;
              const int sh = min(126, 14 - e);
              const float up = __int_as_float((127 + sh) << 23);
              down = 127 - sh;
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] *= up;
            }
            // Two buffers: both slots' threads stage rows that both slots read, and where a run has two
            // jobs a slot can end it, and stage the next, before a warp of the other has read its scale.
            // The run after that has products only once every thread has staged its part of the next.
            if (c == 0) s_scale[(w.seg & 1) * kRows + r] = (uint8_t)down;
            v[u] = make_uint4(pack16<__half>(x[0], x[1]), pack16<__half>(x[2], x[3]), pack16<__half>(x[4], x[5]), pack16<__half>(x[6], x[7]));
          }
          *reinterpret_cast<uint4*>(sQ + (r >> 7) * kTile + (c >> 3) * (BT * 128) + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[u];
        }
        fence_proxy_async_smem();
        mbar_arrive(bQ);
      }
      const int item_row = w.split ? row : t * 128 + row;
      const bool active = (item_row & ~31) < w.rows;     // a warp without rows only takes part in the barriers
      float scale = p.scale_log2;
      if constexpr (kF8) {
        mbar_wait(bQ, w.seg & 1, abort_flag, kSiteDecodeTc);
        scale *= __uint_as_float((uint32_t)s_scale[(w.seg & 1) * kRows + item_row] << 23);
      }
      float m = -INFINITY, l = 0.f;
      const int jobs = w.jobs(), step = w.split ? 0 : 1;
      for (int k = t; k < jobs; k += 2, ++js) {
        const int j = j0 + (k >> step);
        mbar_wait(bS + t, js & 1, abort_flag, kSiteDecodeTc);
        __syncwarp();
        tc_fence_after();
        const uint32_t bad = s_bad[j % kBadRing];
        if (!kF8 && bad) {
          // rows of V that were not loaded count as zeros (a converted tile has them)
          const int sv = j % NV;
          mbar_wait(bVf + sv, (j / NV) & 1, abort_flag, kSiteDecodeTc);
          if ((bad >> (row >> 4)) & 1u) {
#pragma unroll
            for (int cb = 0; cb < C::kBlocks; ++cb)
#pragma unroll
              for (int c = 0; c < 8; ++c)
                reinterpret_cast<uint4*>(sV + sv * kTile + cb * BT * 128 + row * 128)[c] = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
        if (!active) {
          tc_fence_before();
          mbar_arrive(bP + t);
          continue;
        }
        uint32_t s[BT];
        tmem_ld32(tS, *reinterpret_cast<uint32_t(*)[32]>(s));
        tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
        tmem_ld32(tS + 64, *reinterpret_cast<uint32_t(*)[32]>(s + 64));
        tmem_ld32(tS + 96, *reinterpret_cast<uint32_t(*)[32]>(s + 96));
        tmem_wait_ld();
        reg_fence(s);
        if (bad) {                       // tokens that were not loaded have no scores
#pragma unroll
          for (int c = 0; c < BT; ++c)
            if ((bad >> (c >> 4)) & 1u) s[c] = __float_as_uint(-INFINITY);
        }
        float mx8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mx8[i] = __uint_as_float(s[i]);
#pragma unroll
        for (int c = 8; c < BT; ++c) mx8[c & 7] = fmaxf(mx8[c & 7], __uint_as_float(s[c]));
        const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])), fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
        const float top = mx * scale - C::kShift;
        float alpha = 1.f;
        if (top > m + C::kRescale || m == -INFINITY) {
          alpha = m == -INFINITY ? 0.f : ex2(m - top);
          m = top;
        }
        // O of the slot is quiescent: the commit behind this S covered the P V before it
        if (k >= 2 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t ov[32];
            tmem_ld32(tO + c * 32, ov);
            tmem_wait_ld();
            reg_fence(ov);
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
            tmem_st32(tO + c * 32, ov);
          }
        }
        // nothing seen so far: exp2(-inf - 0) = 0
        const float ref = m == -INFINITY ? 0.f : m;
        const uint64_t scale2 = f2_pack(scale, scale), negm2 = f2_pack(-ref, -ref);
        uint64_t rs2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int c = h * 64 + 2 * i;
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale2, negm2), x0, x1);
            const float p0 = ex2(x0), p1 = ex2(x1);
            rs2[i & 3] = f2_add(rs2[i & 3], f2_pack(p0, p1));
            pk[i] = pack16<Op>(p0, p1);
          }
          tmem_st32(tS + h * 32, pk);
        }
        float ra, rb, rc, rd;
        f2_unpack(f2_add(rs2[0], rs2[1]), ra, rb);
        f2_unpack(f2_add(rs2[2], rs2[3]), rc, rd);
        l = l * alpha + ((ra + rb) + (rc + rd));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bP + t);
      }
      j0 += w.n;
      // ---- the record ----
      mbar_wait(bO + t, w.seg & 1, abort_flag, kSiteDecodeTc);
      __syncwarp();
      tc_fence_after();
      const bool whole = w.n == w.tiles;
      float* slab = p.slabs + (size_t)(whole ? 2 * (int)gridDim.x + items_before(s_groups, w.g) + w.r : 2 * cta + (w.seg > 0)) * kSlab<D>;
      const int place = t * 128 + row;
      reinterpret_cast<float2*>(slab)[place] = make_float2(m, l);
      if (active) {
        float4* o = reinterpret_cast<float4*>(slab + 2 * kRows) + place;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t ov[32];
          tmem_ld32(tO + c * 32, ov);
          tmem_wait_ld();
          reg_fence(ov);
          if (t >= jobs) {               // no tile for this slot
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = 0u;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            o[(c * 8 + i) * kRows] = make_float4(__uint_as_float(ov[4 * i]), __uint_as_float(ov[4 * i + 1]), __uint_as_float(ov[4 * i + 2]),
                                                 __uint_as_float(ov[4 * i + 3]));
        }
      }
      tc_fence_before();
      mbar_arrive(bOf + t);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// the join: a thread a row and four columns, a warp 32 rows of one K/V head
// ---------------------------------------------------------------------------
struct JoinParams {
  const Group* desc;
  const int32_t* skip;         // [B]
  const int32_t* in_group;     // [B]
  const float* slabs;
  const float* own_o;          // [B * H][D] fp32, the own tokens' output
  const float* own_lse;        // [B * H]
  __nv_bfloat16* o;
  float* lse;                  // or nullptr
  int B, H, H_kv, group, groups, grid;     // grid: CTAs of the prefix pass
  float o_scale;
};

constexpr int kJoinWarps = 8;

// Many records are asked for at once, weights and columns together (first weights, then columns where they
// count, with four records at once and 16 columns a thread: 64 sequences, 19 records a row, 18 us).
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const JoinParams p) {
  grid_dep_wait();
  grid_dep_launch_dependents();
  constexpr int kParts = D / 4 / kJoinWarps;
  const int rows = p.B * p.group, x = (int)blockIdx.x * 32 + (int)(threadIdx.x & 31);       // row of the head, sequences first
  const int head = (int)(blockIdx.y / kParts), col = (int)(blockIdx.y % kParts) * kJoinWarps + (int)(threadIdx.x >> 5);
  if (x >= rows) return;
  const int b = x / p.group;
  const size_t out = (size_t)b * p.H + (size_t)head * p.group + (x - b * p.group);
  // the sequence's own tokens; an output of no weight is not there
  float M = p.own_lse[out] * kLog2e, L = 1.f;
  float4 acc = reinterpret_cast<const float4*>(p.own_o + out * D)[col];
  const int skip = p.skip[b], g = p.in_group[b], units = p.desc[p.groups].unit;
  if (M == -INFINITY) {
    L = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (skip > 0) {
    const Group a = p.desc[g];
    const Line line(units, p.grid);
    const int all = (p.desc[g + 1].start - a.start) * p.group, pairs = (all + kRows - 1) / kRows, tiles = tiles_of(a);
    const int at = x - a.start * p.group, pair = at / kRows;
    const int r = head * pairs + pair, item0 = a.unit + r * (tiles + kItemCost), first = item0 + kItemCost;
    const int c0 = line.holder(first), c1 = line.holder(first + tiles - 1);
    // both slots of a CTA leave a record where they shared the rows
    const int shift = min(kRows, all - pair * kRows) <= kRows / 2 ? 1 : 0, many = (c1 - c0 + 1) << shift;
    const bool second = line.part(c0) < item0;     // the item is not the first run of its first CTA
    const size_t only = c0 == c1 ? (size_t)(2 * p.grid + items_before(p.desc, g) + r) : 0;
    constexpr int kAhead = 16;
    for (int i0 = 0; i0 < many; i0 += kAhead) {
      float2 ml[kAhead];
      float4 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        ml[u] = make_float2(-INFINITY, 0.f);
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int i = i0 + u, c = c0 + (i >> shift), place = at % kRows + (shift ? (i & 1) * (kRows / 2) : 0);
        if (i < many) {
          const float* slab = p.slabs + (only ? only : (size_t)(2 * c + (c == c0 && second))) * kSlab<D>;
          ml[u] = __ldcg(reinterpret_cast<const float2*>(slab) + place);
          v[u] = __ldcg(reinterpret_cast<const float4*>(slab + 2 * kRows) + col * kRows + place);
        }
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) top = fmaxf(top, ml[u].x);
      const float keep = M == -INFINITY ? 0.f : ex2(M - top);
      L *= keep;
      acc.x *= keep;
      acc.y *= keep;
      acc.z *= keep;
      acc.w *= keep;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float wt = ml[u].x == -INFINITY ? 0.f : ex2(ml[u].x - top), wo = wt * p.o_scale;
        L = fmaf(wt, ml[u].y, L);
        acc.x = fmaf(wo, v[u].x, acc.x);
        acc.y = fmaf(wo, v[u].y, acc.y);
        acc.z = fmaf(wo, v[u].z, acc.z);
        acc.w = fmaf(wo, v[u].w, acc.w);
      }
      M = top;
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint2 y;
  y.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  y.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  reinterpret_cast<uint2*>(p.o + out * D)[col] = y;
  if (col == 0 && p.lse != nullptr) p.lse[out] = L == 0.f ? -INFINITY : (M + lg2(L)) * kLn2;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct Layout {
  size_t own, own_lse, skip, in_group, own_lens, desc, slabs, total;   // byte offsets behind the own tokens' decode
};

inline Layout layout(long long B, long long H, long long H_kv, long long D, long long groups) {
  Layout l{};
  const size_t rows = (size_t)B * H;
  l.own = round_up(ptc::workspace_bytes(D), 256);
  l.own_lse = l.own + round_up(rows * D * sizeof(float), 256);
  l.skip = l.own_lse + round_up(rows * sizeof(float), 256);
  l.in_group = l.skip + round_up((size_t)B * sizeof(int32_t), 256);
  l.own_lens = l.in_group + round_up((size_t)B * sizeof(int32_t), 256);
  l.desc = l.own_lens + round_up((size_t)B * sizeof(int32_t), 256);
  l.slabs = l.desc + round_up((kMaxGroups + 1) * sizeof(Group), 256);
  const size_t items = (size_t)H_kv * ((size_t)(B * (H / H_kv)) / kRows + (size_t)groups);
  l.total = l.slabs + (2 * (size_t)sm_count() + items) * kRows * (D + 2) * sizeof(float);
  return l;
}

inline bool eligible(long long D, int q_dtype, int kv_dtype) {
  if (q_dtype != PU_DTYPE_F16 && q_dtype != PU_DTYPE_BF16) return false;
  if (kv_dtype == PU_DTYPE_FP8_E4M3) return D == 128;
  return (D == 64 || D == 128) && q_dtype == kv_dtype;
}

template <typename T, typename KVT, int D>
int launch_as(const CUtensorMap& tk, const CUtensorMap& tv, const Params& prm, cudaStream_t st) {
  using C = Cfg<T, KVT, D>;
  const int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(prefix_kernel<T, KVT, D>), C::kSmem, "shared prefix shared memory");
  if (rc) return rc;
  return check_cuda(launch_pdl(prefix_kernel<T, KVT, D>, dim3((unsigned)sm_count()), dim3(C::kThreads), C::kSmem, st, tk, tv, prm),
                    "shared prefix launch");
}

}  // namespace shared
}  // namespace decode
}  // namespace pu

extern "C" {

size_t pu_decode_paged_shared_workspace_size(int64_t B, int64_t H, int64_t H_kv, int64_t groups, int64_t D) {
  if (B <= 0 || H <= 0 || H_kv <= 0 || H % H_kv || groups <= 0 || D <= 0) return 0;
  return pu::decode::shared::layout(B, H, H_kv, D, groups).total;
}

int pu_decode_paged_shared(const void* q, int q_dtype, const void* k_pool, const void* v_pool, int kv_dtype,
                           const int32_t* page_table, int64_t max_pages_per_seq, int64_t num_pages, int64_t page_size,
                           const int32_t* kv_lens, const int32_t* shared_lens, const int32_t* group_starts, int64_t groups,
                           void* o, float* lse, void* workspace, size_t workspace_bytes, int64_t B, int64_t H, int64_t H_kv,
                           int64_t D, float sm_scale, float k_scale, float v_scale, void* stream) {
  using namespace pu::decode;
  int shift = 0;
  int rc = pu::paged::check_pages(page_table, max_pages_per_seq, num_pages, page_size, &shift);
  if (rc) return rc;
  rc = check_args(q, q_dtype, k_pool, v_pool, kv_dtype, B, H, max_pages_per_seq * page_size, D, true, false);
  if (rc) return rc;
  if (!o || !kv_lens || !shared_lens) return pu::set_error(PU_ERR_INVALID_ARGUMENT, "null output or lengths");
  if (!pu::aligned16(o) || !pu::aligned16(workspace))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "the output and the workspace must be 16-byte aligned");
  if (H_kv <= 0 || H % H_kv != 0)
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "H = %lld is not a multiple of H_kv = %lld", (long long)H, (long long)H_kv);
  if (num_pages > 2147483647ll / H_kv) return pu::set_error(PU_ERR_UNSUPPORTED, "page pool too large");
  if (!(k_scale > 0.f) || !(v_scale > 0.f) || !isfinite(k_scale) || !isfinite(v_scale))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "k_scale and v_scale must be positive and finite");
  if (groups < 1 || groups > shared::kMaxGroups || (groups > 1 && !group_starts))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "%lld shared prefixes (1 to %d, with group_starts from 2 on)", (long long)groups, shared::kMaxGroups);
  if (!shared::eligible(D, q_dtype, kv_dtype))
    return pu::set_error(PU_ERR_UNSUPPORTED, "a shared prefix needs q and pools of one 16-bit type, or e4m3 pools with D = 128");
  // units of the line are 32-bit: items times (tiles + cost)
  const long long tiles = (max_pages_per_seq * page_size + shared::BT - 1) / shared::BT + shared::kItemCost;
  const long long items = H_kv * (B * (H / H_kv) / shared::kRows + groups);
  if (B > ptc::kMaxB || H > kMaxBH || H_kv * (D / 4 / shared::kJoinWarps) > 65535 || items > 2147483647ll / tiles)
    return pu::set_error(PU_ERR_UNSUPPORTED, "shared prefix of %lld sequences with %lld heads over %lld tokens", (long long)B, (long long)H,
                         (long long)(max_pages_per_seq * page_size));
  const shared::Layout l = shared::layout(B, H, H_kv, D, groups);
  if (!workspace || workspace_bytes < l.total)
    return pu::set_error(PU_ERR_WORKSPACE, "shared prefix workspace needs %zu bytes, got %zu", l.total, workspace_bytes);
  char* ws = static_cast<char*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f8 = kv_dtype == PU_DTYPE_FP8_E4M3, h = q_dtype == PU_DTYPE_F16;

  shared::Params prm{};
  prm.q = q;
  prm.table = page_table;
  prm.lens = kv_lens;
  prm.shared_lens = shared_lens;
  prm.starts = group_starts;
  prm.skip = reinterpret_cast<int32_t*>(ws + l.skip);
  prm.in_group = reinterpret_cast<int32_t*>(ws + l.in_group);
  prm.own_lens = reinterpret_cast<int32_t*>(ws + l.own_lens);
  prm.desc = reinterpret_cast<shared::Group*>(ws + l.desc);
  prm.slabs = reinterpret_cast<float*>(ws + l.slabs);
  prm.B = (int)B;
  prm.H = (int)H;
  prm.H_kv = (int)H_kv;
  prm.group = (int)(H / H_kv);
  prm.slices = (prm.group + ptc::NP - 1) / ptc::NP;
  prm.groups = (int)groups;
  prm.max_pages = (int)max_pages_per_seq;
  prm.num_pages = (int)num_pages;
  prm.page_shift = shift;
  prm.box = (int)std::min<long long>(page_size, shared::BT);
  prm.pass_cost = D == 128 && !f8 ? 2 : 4;
  prm.scale_log2 = sm_scale * k_scale * kLog2e;

  ptc::Params own{};
  own.q = q;
  own.table = page_table;
  own.lens = prm.own_lens;
  own.skip = prm.skip;
  own.o32 = reinterpret_cast<float*>(ws + l.own);
  own.lse = reinterpret_cast<float*>(ws + l.own_lse);
  own.count = static_cast<int*>(workspace);
  own.rec = reinterpret_cast<float*>(ws + kCountBytes);
  own.B = prm.B;
  own.H = prm.H;
  own.pool_heads = prm.H_kv;
  own.lists = 1;
  own.group = prm.group;
  own.slices = prm.slices;
  own.inner = prm.H_kv * own.slices;
  own.max_pages = prm.max_pages;
  own.num_pages = prm.num_pages;
  own.page_shift = shift;
  own.box = prm.box;
  own.scale_log2 = prm.scale_log2;
  own.o_scale = v_scale;

  CUtensorMap tk, tv;
  rc = ptc::make_maps(&tk, &tv, k_pool, v_pool, kv_dtype, num_pages, H_kv, shift, prm.box, (int)D);
  if (rc) return rc;
  // All tokens are each sequence's own where the call can save too little whatever its lengths (two launches less: four
  // sequences of 1224 tokens 14.6 us instead of 21.2), and where the scale is not a positive number: the prefix pass
  // masks scores and takes their maximum before it scales them, which saves a product a score and is the same only for
  // a positive factor (NaN is none).
  const long long most = (B * prm.slices - prm.pass_cost) * H_kv * (tiles - shared::kItemCost);
  if (B < 2 || most < shared::kWorth || !(prm.scale_log2 >= FLT_MIN && prm.scale_log2 <= FLT_MAX)) {
    own.lens = kv_lens;
    own.skip = nullptr;
    own.o32 = nullptr;
    own.o = static_cast<__nv_bfloat16*>(o);
    own.lse = lse;
    return ptc::launch_with(tk, tv, own, q_dtype, kv_dtype, (int)D, st);
  }
  if (f8)
    rc = h ? shared::launch_as<__half, __nv_fp8_e4m3, 128>(tk, tv, prm, st)
           : shared::launch_as<__nv_bfloat16, __nv_fp8_e4m3, 128>(tk, tv, prm, st);
  else if (D == 128)
    rc = h ? shared::launch_as<__half, __half, 128>(tk, tv, prm, st) : shared::launch_as<__nv_bfloat16, __nv_bfloat16, 128>(tk, tv, prm, st);
  else
    rc = h ? shared::launch_as<__half, __half, 64>(tk, tv, prm, st) : shared::launch_as<__nv_bfloat16, __nv_bfloat16, 64>(tk, tv, prm, st);
  if (rc) return rc;
  rc = ptc::launch_with(tk, tv, own, q_dtype, kv_dtype, (int)D, st);
  if (rc) return rc;

  shared::JoinParams jp{};
  jp.desc = prm.desc;
  jp.skip = prm.skip;
  jp.in_group = prm.in_group;
  jp.slabs = prm.slabs;
  jp.own_o = own.o32;
  jp.own_lse = own.lse;
  jp.o = static_cast<__nv_bfloat16*>(o);
  jp.lse = lse;
  jp.B = prm.B;
  jp.H = prm.H;
  jp.H_kv = prm.H_kv;
  jp.group = prm.group;
  jp.groups = prm.groups;
  jp.grid = pu::sm_count();
  jp.o_scale = v_scale;
  const dim3 grid((unsigned)((B * prm.group + 31) / 32), (unsigned)(H_kv * (D / 4 / shared::kJoinWarps))), block(shared::kJoinWarps * 32);
  return pu::check_cuda(D == 128 ? launch_pdl(shared::join_kernel<128>, grid, block, 0, st, jp)
                                 : launch_pdl(shared::join_kernel<64>, grid, block, 0, st, jp),
                        "shared prefix join launch");
}

}  // extern "C"
