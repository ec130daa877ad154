// paged_tc.cuh — attention of one new token over a paged cache with grouped
// heads, on the tensor core: 16-bit caches of q's type with G = H / H_kv >= 2
// (D = 64 or 128), e4m3 caches with any G (D = 128).
//
// No counterpart in the reference (dense caches, one K/V head per query head:
// src/pallas_flash/kernels/decoding.py:86-115).  The products are those of
// the dense grouped kernel, with the rows of a 128-token tile as the MMA's M
// and up to 16 query heads as its N:
//   S [128 rows x 16 heads] = K_tile Q^T,   O^T [D x 16 heads] += V_tile^T P^T
// about 64 D flops per row of 4 D bytes: far below the ridge, so the kernel
// is bound by reading the pages once.
//
// Work.  The tiles of all (sequence, K/V head, slice of 16 query heads) are
// numbered in one line, an item's cost of starting and ending before its
// tiles, and cut into as many equal parts as there are CTAs (one per SM), so a
// ragged batch keeps every SM equally busy whatever the lengths, which the host
// does not know; a grid cut by the table's capacity leaves most SMs idle when
// sequences are shorter than the table.  A part may begin and end inside a
// sequence: such an end is written as a record (m, l, o) and the last CTA of
// the sequence joins its records; a CTA has at most two of them, so the
// workspace is a few MB whatever the batch.  No CTA waits for another.
//
// Roles (512 threads, registers shared out with setmaxnreg):
//   warps 0-7   two softmax groups; group t & 1 takes tile t, each with its
//               own running maximum, sums and accumulator (row r of the tile
//               = TMEM lane r = thread r).  One group alone left the tensor
//               core and the loads waiting on e4m3 tiles, whose softmax takes
//               longer than their bytes.
//   warp 8      page table lookups and TMA loads
//   warp 9      tcgen05 issue of the S products; also owns the TMEM
//   warp 10     queries of the next segments into shared memory (e4m3: scaled
//               by a power of two and split into parts)
//   warp 11     tcgen05 issue of the P V products
//   warps 12-15 the end of each segment: both groups' accumulators and sums
//               into the output or a record, and the joins.  The accumulators
//               are double buffered over segments, so the softmax groups go on
//               with the next sequence at once (done by them, the end took
//               longer than two tiles: 2048 sequences of 128 tokens 107 us).
// One thread issues, elected with elect.sync inside a warp-uniform branch:
// that tells the compiler that a single thread runs there.  Behind
// `lane == 0` it wraps each tensor or TMA instruction in a loop over the active
// lanes, and a product of 40 clocks took 154 to issue.
// K/V tiles run through one ring across segments, so a new sequence's first
// pages are on their way while the previous one ends.
//
// e4m3: K and V tiles are operands as stored; q and P are split into e4m3
// parts stacked along N: q into two parts if bf16 (8 significant bits are
// two e4m3 parts exactly) and three if f16 (11 bits), P into three.  The parts of
// q share the scale of the head's largest element, so an element is off by at most
// 2^-17 of that one.  With 16-bit pages P is rounded once to their type (the fp32
// sums l are taken before): outputs differ from an fp32 P's inside bf16's last step.
//
// Pages.  Only pages that hold tokens of the sequence are read.  An entry
// outside the pool is not followed: it is reported (detail 302) and its
// tokens are left out.  Rows past the length and rows not loaded are masked,
// and their V rows are zeroed in shared memory, so stale values never count.
//
// Measured (calls back to back on pools that do not fit L2; the copy rate of
// this GPU is 6.4 TB/s): 8 sequences of 4096 to 131072 tokens, 32 heads over 8
// of 128, f16, 64-token pages: 2.51 GB in 357 us = 7.0 TB/s; 24 sequences of up
// to 32768 tokens, 64 heads over 8, e4m3, 32-token pages: 0.98 GB in 157 to 166 us =
// 5.9 to 6.3 TB/s (the splitting of P shares the issue slots with everything else); 256
// sequences of up to 2048 tokens, 16 heads over 2 of 64, 16-token pages: 135 MB
// in 39 us, of which 28 us are the loads alone, the rest the start, the last
// tile's chain and the joins; one sequence of 1000 tokens: 11 us.
#pragma once

#include "gqa_tc.cuh"

namespace pu {
namespace decode {
namespace ptc {

using tc::to16;

constexpr int BT = 128;                    // cache rows per tile (MMA M)
constexpr int NP = 16;                     // query heads per slice (MMA N per part)
constexpr int kGroups = 2;                 // softmax groups of 128 threads
constexpr int kSoftmax = kGroups * 128;
constexpr int kLoadWarp = 8, kScoreWarp = 9, kQueryWarp = 10, kValueWarp = 11;
constexpr int kEndWarps = 12;               // first of four
constexpr int kCtaThreads = 512;
// registers a thread: softmax 256 x 152, roles 128 x 80, ends 128 x 128 = the launch's 512 x 128 (with 160 / 72 / 120
// the e4m3 kernels spilled: 24 sequences up to 32768 tokens 172 us instead of 166)
constexpr int kSoftmaxRegs = 152, kRoleRegs = 80, kEndRegs = 128;
constexpr int kMaxB = 8192;                // sequences, as many as a page plan takes (each CTA reads all lengths)
constexpr int kHead = 4;                   // floats before o in a record: m, l, and two that keep o 16-byte aligned

template <typename T, typename KVT, int D>
struct Cfg {
  static constexpr bool kF8 = sizeof(KVT) == 1;
  static constexpr int kQParts = !kF8 ? 1 : std::is_same<T, __nv_bfloat16>::value ? 2 : 3;
  static constexpr int kPParts = kF8 ? 3 : 1;
  // P = 2^(s - m) with m = the running maximum - kShift; m moves (and the
  // accumulator is rescaled) once a score passes the maximum by kRescale, so
  // P <= 2^(kShift + kRescale), near the top of its type: a long tail of
  // small weights then stays above the type's smallest step (f16 2^-24, three
  // e4m3 parts 2^-19; bf16 has fp32's range and needs no shift).
  static constexpr float kRescale = kF8 ? 2.f : 8.f;
  static constexpr float kShift = kF8 ? 6.f : std::is_same<T, __nv_bfloat16>::value ? 0.f : 7.f;
  static constexpr int kRowBytes = D * (int)sizeof(KVT);
  static constexpr int kBlocks = kRowBytes / 128;          // 128-byte swizzle blocks of a tile
  static_assert(kRowBytes % 128 == 0, "rows are whole swizzle blocks");
  // What starting and ending a segment costs, in tiles: parts are cut by tiles
  // plus this for each item (200 e4m3 sequences of up to 4000 tokens, 4 K/V
  // heads: 115 us with 2, 121 with 1, 128 with 0; 64 KB tiles: 1 and 2 the same).
  static constexpr int kItemCost = BT * kRowBytes == 32768 ? 1 : 2;
  static constexpr int kTile = BT * kRowBytes;
  // ring stages: 192 KB in flight (16 x 16384 tokens of e4m3, 4 K/V heads: 55.5 us; with 5 stages 57.5)
  static constexpr int NS = kTile == 32768 ? 3 : 6;
  static constexpr int kQSlots = kF8 ? 3 : 4;              // segments whose queries are staged ahead
  static constexpr int kQBlock = NP * 128;                 // one swizzle block of one part of q or P
  static constexpr int kQBytes = (kF8 ? kQParts : kBlocks) * kQBlock;
  static constexpr int kPBytes = (kF8 ? kPParts : 2) * kQBlock;   // 16 heads x 128 rows
  static constexpr int kOffKV = 0;                         // stage: V, then K
  static constexpr int kOffQ = NS * 2 * kTile;
  static constexpr int kOffP = kOffQ + kQSlots * kQBytes;
  static constexpr int kOffBar = kOffP + kGroups * kPBytes;
  // full[NS], empty[NS], qfull[4], qfree[4], sfull[4], sfree[4], pfull[2], pvdone[2], sums[2], odone[2], ofree[2], drain[2]
  static constexpr int kBars = 2 * NS + 2 * kQSlots + 8 + 2 * kGroups + 8;
  static constexpr int kOffMisc = (kOffBar + kBars * 8 + 15) / 16 * 16;   // tmem base, abort flag, last-CTA flag
  static constexpr int kOffBad = kOffMisc + 16;            // [NS] boxes of the stage that were not loaded
  static constexpr int kOffMax = kOffBad + 32;             // [2 groups][2][4 warps][NP] tile maxima
  static constexpr int kOffM = kOffMax + kGroups * 2 * 4 * NP * 4;   // [2 parities][2 groups][NP]
  static constexpr int kOffL = kOffM + 2 * kGroups * NP * 4;     // [2 parities][2 groups][4 warps][NP]
  static constexpr int kOffFac = kOffL + 2 * kGroups * 4 * NP * 4;    // [4 warps][2 groups][NP]
  static constexpr int kOffQinv = kOffFac + 4 * 2 * NP * 4;           // [4 slots][NP]
  static constexpr int kOffStart = (kOffQinv + kQSlots * NP * 4 + 15) / 16 * 16;
  static constexpr int kSmem = kOffStart + 96;
  static constexpr int kSCols = kQParts * NP, kOCols = kPParts * NP;
  static constexpr int kColO = 4 * kSCols;                 // four S buffers, then two accumulators per group
  static constexpr int kCols = kColO + 2 * kGroups * kOCols;
  static constexpr uint32_t kTmemCols = kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kSmem <= 232448, "shared memory of one CTA");
  static_assert(kOffBar % 8 == 0 && kOffMax % 16 == 0, "barriers, and maxima that are read as float4");
};

struct Params {
  const void* q;               // [B, H, D]
  const int32_t* table;        // [B][max_pages]
  const int32_t* lens;         // [B]
  __nv_bfloat16* o;            // [B, H, D]
  float* lse;                  // [B, H] or nullptr
  int* count;                  // [CTAs] zero between calls
  float* rec;                  // [CTAs][2][NP][D + kHead]
  int B, H, H_kv, group, slices;
  int max_pages, num_pages, page_shift;
  int box;                     // rows of one TMA box: min(page size, 128)
  float scale_log2, o_scale;
};

// x as N e4m3 parts, x ~ sum_i part_i / kPartScale^i: each part is the e4m3
// rounding of what the ones before left, times kPartScale when `scaled` (a
// remainder of a value up to 256 is at most 8, so 32 keeps it below 256).
constexpr float kPartScale = 32.f;

template <bool scaled, int N>
__device__ __forceinline__ void split_e4m3(float a, float b, uint16_t (&part)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const __nv_fp8x2_storage_t h2 = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    part[i] = (uint16_t)h2;
    if (i + 1 < N) {
      const float2 hf = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(h2, __NV_E4M3)));
      a = (a - hf.x) * (scaled ? kPartScale : 1.f);
      b = (b - hf.y) * (scaled ? kPartScale : 1.f);
    }
  }
}

// The tiles of this CTA in order.  An item is (sequence b, inner index r =
// K/V head * slices + slice); a segment is the CTA's run of one item's tiles.
struct Walk {
  const Params* p;
  int b, r, t, tiles, len, inner, left, seg, loc, cost;   // left: the part's units from this tile on
  __device__ __forceinline__ int len_of(int i) const {
    const int n = p->lens[i], cap = p->max_pages << p->page_shift;
    return n < 0 ? 0 : n > cap ? cap : n;
  }
  __device__ __forceinline__ int tiles_of(int i) const { return (len_of(i) + BT - 1) / BT; }
  // is the current tile the last of its segment?
  __device__ __forceinline__ bool last() const { return left == 1 || t + 1 == tiles; }
  // to the next tile, or over all n tiles of the segment
  __device__ __forceinline__ void next(int n = 1) {
    left -= n;
    t += n;
    loc += n;
    if (left <= 0 || t < tiles) return;
    left -= cost;
    if (left <= 0) return;
    t = loc = 0;
    ++seg;
    if (++r < inner) return;
    r = 0;
    do len = len_of(++b);
    while (len == 0);
    tiles = (len + BT - 1) / BT;
  }
};

// A CTA's part of the line of units (an item's cost, then its tiles).
struct Start {
  long long ctas, q, rem, first, end;    // parts of q or (the first rem) q + 1 units; this one's
  long long item0;                       // first unit of sequence b
  int b, r, t, tiles, len, left, cost;   // the Walk's first tile
};

template <int kItemCost>
__device__ __forceinline__ void find_start(const Params& p, int lane, Start* out) {
  constexpr int kHold = 8;
  const int inner = p.H_kv * p.slices, cap = p.max_pages << p.page_shift;
  int len[kHold];
  // lengths of sequences base + 8 lane + k, in a lane's registers
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      const int i = base + lane * kHold + k;
      len[k] = i < p.B ? p.lens[i] : 0;
    }
#pragma unroll
    for (int k = 0; k < kHold; ++k) len[k] = max(0, min(len[k], cap));
  };
  long long tiles = 0;
  int items = 0;
  for (int base = 0; base < p.B; base += 32 * kHold) {
    load(base);
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      tiles += (len[k] + BT - 1) / BT;
      items += len[k] > 0;
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    tiles += __shfl_xor_sync(0xffffffffu, tiles, off);
    items += __shfl_xor_sync(0xffffffffu, items, off);
  }
  // with no more tiles than CTAs each has one of its own
  Start s;
  s.cost = tiles * inner <= (long long)gridDim.x ? 0 : kItemCost;
  const long long all = (tiles + (long long)items * s.cost) * inner;
  // no part is empty, so every CTA between an item's first and last has a record
  s.ctas = min((long long)gridDim.x, all);
  if (all <= 0xffffffffll) {             // 32-bit division where it does (the 64-bit one takes 1 us)
    s.q = s.ctas > 0 ? (unsigned)all / (unsigned)s.ctas : 0;
  } else {
    s.q = all / s.ctas;
  }
  s.rem = all - s.q * s.ctas;
  const long long c = blockIdx.x;
  s.first = c < s.ctas ? c * s.q + min(c, s.rem) : 0;
  s.end = c < s.ctas ? (c + 1) * s.q + min(c + 1, s.rem) : 0;
  s.left = (int)(s.end - s.first);
  s.item0 = 0;
  s.b = s.r = s.t = s.tiles = s.len = 0;
  if (s.left > 0) {
    long long before = 0;
    for (int base = 0;; base += 32 * kHold) {
      if (p.B > 32 * kHold) load(base);  // otherwise they are still there
      long long mine = 0;
#pragma unroll
      for (int k = 0; k < kHold; ++k) mine += len[k] > 0 ? (len[k] + BT - 1) / BT + s.cost : 0;
      long long x = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, (before + x) * inner > s.first);
      if (hit) {
        // the lane that holds the sequence finds it among its eight
        const int src = __ffs(hit) - 1;
        long long at = before + x - mine;
        bool found = false;
#pragma unroll
        for (int k = 0; k < kHold; ++k) {
          const int n = (len[k] + BT - 1) / BT, units = len[k] > 0 ? n + s.cost : 0;
          if (!found && (at + units) * inner > s.first) {
            found = true;
            s.b = base + lane * kHold + k;
            s.tiles = n;
            s.len = len[k];
            s.item0 = at * inner;
          }
          at += units;
        }
        if (lane == src) {
          const long long in = s.first - s.item0;
          const int per = s.tiles + s.cost;
          if (in <= 0xffffffffll) {
            s.r = (int)((unsigned)in / (unsigned)per);
          } else {
            s.r = (int)(in / per);
          }
          s.t = (int)(in - (long long)s.r * per) - s.cost;
          if (s.t < 0) {                 // the part begins inside an item's cost
            s.left += s.t;
            s.t = 0;
          }
          *out = s;
        }
        return;
      }
      before += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  if (lane == 0) *out = s;
}

// Sum or maximum of the warp's 16 values per lane over its 32 lanes: lanes 2 h
// and 2 h + 1 return head h's (each step halves the values a lane still holds).
template <bool kMax>
__device__ __forceinline__ float join(float a, float b) { return kMax ? fmaxf(a, b) : a + b; }

template <bool kMax>
__device__ __forceinline__ float reduce16(const float (&v)[NP], int lane) {
  float a[8], b[4], c[2], d;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float keep = lane & 16 ? v[i + 8] : v[i], give = lane & 16 ? v[i] : v[i + 8];
    a[i] = join<kMax>(keep, __shfl_xor_sync(0xffffffffu, give, 16));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float keep = lane & 8 ? a[i + 4] : a[i], give = lane & 8 ? a[i] : a[i + 4];
    b[i] = join<kMax>(keep, __shfl_xor_sync(0xffffffffu, give, 8));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float keep = lane & 4 ? b[i + 2] : b[i], give = lane & 4 ? b[i] : b[i + 2];
    c[i] = join<kMax>(keep, __shfl_xor_sync(0xffffffffu, give, 4));
  }
  d = join<kMax>(lane & 2 ? c[1] : c[0], __shfl_xor_sync(0xffffffffu, lane & 2 ? c[0] : c[1], 2));
  return join<kMax>(d, __shfl_xor_sync(0xffffffffu, d, 1));
}

template <typename T, typename KVT, int D>
__global__ void __launch_bounds__(kCtaThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ Params p) {
  using C = Cfg<T, KVT, D>;
  constexpr int NS = C::NS, kQSlots = C::kQSlots, kQParts = C::kQParts, kPParts = C::kPParts, kTile = C::kTile;
  constexpr bool kF8 = C::kF8;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(smem) & 1023u) {
    if (tid == 0) record_device_error(PU_ERR_UNSUPPORTED, kSiteDecodeTc);
    return;
  }
  uint8_t* sKV = smem + C::kOffKV;
  uint8_t* sQ = smem + C::kOffQ;
  uint8_t* sP = smem + C::kOffP;
  uint64_t* bFull = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* bEmpty = bFull + NS;
  uint64_t* bQfull = bEmpty + NS;        // [kQSlots] queries of segment s in slot s % kQSlots
  uint64_t* bQfree = bQfull + kQSlots;   // [kQSlots] its products (and scales, e4m3) have been read
  uint64_t* bSf = bQfree + kQSlots;      // [4] S of tile t in buffer t & 3
  uint64_t* bSfree = bSf + 4;            // [4] read into registers (an arrival per warp)
  uint64_t* bPf = bSfree + 4;            // [2] P of the group's tile written (128 arrivals)
  uint64_t* bPv = bPf + kGroups;         // [2] the group's P V product done
  uint64_t* bSums = bPv + kGroups;       // [2] maxima and sums of segment s in buffer s & 1 (an arrival per warp)
  uint64_t* bOdone = bSums + 2;          // [2] its products done
  uint64_t* bOfree = bOdone + 2;         // [2] its accumulators and sums read (128 arrivals)
  uint64_t* bDrain = bOfree + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);
  int* s_last = reinterpret_cast<int*>(smem + C::kOffMisc + 8);
  volatile uint32_t* s_bad = reinterpret_cast<volatile uint32_t*>(smem + C::kOffBad);
  float* s_max = reinterpret_cast<float*>(smem + C::kOffMax);
  float* s_m = reinterpret_cast<float*>(smem + C::kOffM);
  float* s_l = reinterpret_cast<float*>(smem + C::kOffL);
  Start* s_start = reinterpret_cast<Start*>(smem + C::kOffStart);
  static_assert(sizeof(Start) <= 96, "room for the start");
  float* s_fac = reinterpret_cast<float*>(smem + C::kOffFac);
  float* s_qinv = reinterpret_cast<float*>(smem + C::kOffQinv);

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(bFull + s, 1);
      mbar_init(bEmpty + s, 1);
    }
    for (int s = 0; s < kQSlots; ++s) {
      mbar_init(bQfull + s, 32);
      mbar_init(bQfree + s, kF8 ? 1 + kGroups : 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(bSf + s, 1);
      mbar_init(bSfree + s, 4);
    }
    for (int g = 0; g < kGroups; ++g) {
      mbar_init(bPf + g, 128);
      mbar_init(bPv + g, 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(bSums + g, kSoftmax / 32);
      mbar_init(bOdone + g, 1);
      mbar_init(bOfree + g, 128);
    }
    mbar_init(bDrain, 1);
    mbar_init(bDrain + 1, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kScoreWarp) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  if (warp == kLoadWarp && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  grid_dep_wait();
  grid_dep_launch_dependents();

  // Where this CTA's tiles begin.  One warp looks, 256 lengths at a time with
  // all of a lane's eight loads in flight (32 at a time in every warp took 2 to
  // 4 us for 256 sequences), and leaves it in shared memory.
  if (warp == kEndWarps) find_start<C::kItemCost>(p, lane, s_start);

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Start st = *s_start;
  // CTA c: units [c q + min(c, rem), ...), q or q + 1 of them
  const long long q = st.q, rem = st.rem, first = st.first, end = st.end;
  auto part = [&](long long c) { return c * q + min(c, rem); };
  long long item0 = st.item0;
  Walk w0;
  w0.p = &p;
  w0.inner = p.H_kv * p.slices;
  w0.b = st.b;
  w0.r = st.r;
  w0.t = st.t;
  w0.tiles = st.tiles;
  w0.len = st.len;
  w0.left = st.left;
  w0.cost = st.cost;
  w0.seg = w0.loc = 0;

  if (warp >= kSoftmax / 32 && warp < kEndWarps) {
    reg_dealloc<kRoleRegs>();
    if (warp == kLoadWarp) {
      // ---------------- pages -> ring ----------------
      // The table is read for up to 8 tiles of a segment at a time (lane j * boxes
      // + i: box i of the j-th), two such batches ahead, or each tile's loads
      // would wait for its entries first.
      const int box_shift = 31 - __clz(p.box), boxes = BT >> box_shift, batch = min(32 / boxes, 8);
      const int lane_tile = lane / boxes, lane_row = (lane & (boxes - 1)) << box_shift, per_page = 1 << p.page_shift;
      Walk wl = w0;                          // the first tile of the next batch
      auto look_up = [&]() -> int {
        const int cnt = min(min(wl.left, wl.tiles - wl.t), batch);
        const int row = (wl.t + lane_tile) * BT + lane_row;
        const int32_t* at = p.table + (size_t)wl.b * p.max_pages + (row >> p.page_shift);
        int pg = -1;
        asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n @q ld.global.b32 %0, [%1];\n}"
                     : "+r"(pg) : "l"(at), "r"((int)(lane_tile < cnt && row < wl.len)));
        if (cnt > 0) wl.next(cnt);
        return pg;
      };
      int entries = 0, next1 = look_up(), next2 = look_up();
      int n = 0, j = 0, cnt = 0, s = 0, turn = 0, seg = -1, head = 0;   // stage s for the turn-th time
      for (Walk w = w0; w.left > 0; w.next(), ++n, ++j) {
        if (j == cnt) {
          j = 0;
          cnt = min(min(w.left, w.tiles - w.t), batch);
          entries = next1;
          next1 = next2;
          next2 = look_up();
        }
        if (w.seg != seg) {
          seg = w.seg;
          head = w.r / p.slices;
        }
        const int pg = __shfl_sync(0xffffffffu, entries, (j * boxes + lane) & 31), row0 = w.t * BT;
        const bool mine = lane < boxes && row0 + lane_row < w.len;
        const bool good = mine && (unsigned)pg < (unsigned)p.num_pages;
        if (mine && !good) record_device_error(PU_ERR_INVALID_ARGUMENT, kSiteDecodePage);
        const unsigned loaded = __ballot_sync(0xffffffffu, good);
        const int outer = pg * p.H_kv + head, in = p.box < BT ? 0 : row0 & (per_page - 1);
        // one answer for the warp: a lane that gave up alone would leave the others at the next vote
        if (turn > 0 && !__all_sync(0xffffffffu, mbar_wait(bEmpty + s, (turn - 1) & 1, abort_flag, kSiteDecodeTc))) break;
        // box i's coordinates to the issuing thread (all of them ahead of it: a
        // shuffle and a branch for each box put the boxes one behind the other)
        int at[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) at[i] = __shfl_sync(0xffffffffu, outer, i);
        if (elect_one_sync()) {
          s_bad[s] = ~loaded;
          mbar_arrive_expect_tx(bFull + s, (uint32_t)__popc(loaded) * 2 * p.box * C::kRowBytes);
          uint8_t* dV = sKV + s * 2 * kTile;
          const int step = p.box * 128;
          constexpr int cols = kF8 ? 128 : 64;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if ((loaded >> i) & 1u) {
#pragma unroll
              for (int cb = 0; cb < C::kBlocks; ++cb)
                tma_load_3d(dV + kTile + cb * BT * 128 + i * step, &tmK, bFull + s, cb * cols, in, at[i]);
#pragma unroll
              for (int cb = 0; cb < C::kBlocks; ++cb)
                tma_load_3d(dV + cb * BT * 128 + i * step, &tmV, bFull + s, cb * cols, in, at[i]);
            }
          }
        }
        __syncwarp();
        if (++s == NS) {
          s = 0;
          ++turn;
        }
      }
      // copies still in flight land before the CTA may exit
      volatile int no_abort = 0;
      for (int i = max(0, n - NS); i < n; ++i) mbar_wait(bFull + i % NS, (i / NS) & 1, &no_abort, kSiteDecodeTc);
    } else if (warp == kQueryWarp) {
      // ---------------- queries -> shared memory ----------------
      int done = -1;                         // last segment staged
      for (Walk w = w0; w.left > 0; w.next()) {
        if (w.seg == done) continue;
        done = w.seg;
        const int slot = w.seg % kQSlots;
        if (w.seg >= kQSlots &&
            !__all_sync(0xffffffffu, mbar_wait(bQfree + slot, (w.seg / kQSlots - 1) & 1, abort_flag, kSiteDecodeTc)))
          break;
        const int slice = w.r % p.slices, heads = min(NP, p.group - slice * NP);
        const T* q = static_cast<const T*>(p.q) + ((size_t)w.b * p.H + (w.r / p.slices) * p.group + slice * NP) * D;
        uint8_t* dst = sQ + slot * C::kQBytes;
        constexpr int kVecs = D / 8;         // 16-byte vectors of a row
        constexpr int kHold = NP * kVecs / 64;   // vectors a lane holds, in two rounds
#pragma unroll
        for (int i0 = 0; i0 < 2 * kHold; i0 += kHold) {
          uint4 v[kHold];
#pragma unroll
          for (int i = 0; i < kHold; ++i) {
            const int h = ((i0 + i) * 32 + lane) / kVecs, c = ((i0 + i) * 32 + lane) % kVecs;
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (h < heads) v[i] = *reinterpret_cast<const uint4*>(q + (size_t)h * D + c * 8);
          }
#pragma unroll
          for (int i = 0; i < kHold; ++i) {
            const int h = ((i0 + i) * 32 + lane) / kVecs, c = ((i0 + i) * 32 + lane) % kVecs;
            if constexpr (!kF8) {
              *reinterpret_cast<uint4*>(dst + (c >> 3) * C::kQBlock + h * 128 + (((c & 7) ^ (h & 7)) << 4)) = v[i];
            } else {
              // scaled by a power of two so that the head's largest |q| lies in
              // [128, 256), then split; 16 lanes hold a head
              float x[8];
              unpack8<T>(v[i], x);
              float mx = 0.f;
#pragma unroll
              for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fabsf(x[k]));
#pragma unroll
              for (int off = 8; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
              const int e = (mx > 0.f && isfinite(mx)) ? ((__float_as_int(mx) >> 23) & 0xff) - 127 : 7;
              const int sh = min(126, 7 - e);      // -120 at least: 2^sh and 2^-sh are both normal numbers
              const float up = __int_as_float((127 + sh) << 23), down = __int_as_float((127 - sh) << 23);
              uint32_t wd[kQParts][2];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint16_t pr[kQParts];
                split_e4m3<false>(x[2 * k] * up, x[2 * k + 1] * up, pr);
#pragma unroll
                for (int j = 0; j < kQParts; ++j)
                  wd[j][k >> 1] = (k & 1) ? (wd[j][k >> 1] | ((uint32_t)pr[j] << 16)) : (uint32_t)pr[j];
              }
              const int at = h * 128 + (((c >> 1) ^ (h & 7)) << 4) + (c & 1) * 8;
#pragma unroll
              for (int j = 0; j < kQParts; ++j)
                *reinterpret_cast<uint2*>(dst + j * C::kQBlock + at) = make_uint2(wd[j][0], wd[j][1]);
              // a head that is not finite makes its scores NaN, as it would in 16 bits
              if (c == 0) s_qinv[slot * NP + h] = isfinite(mx) ? down : mx - mx;
            }
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(bQfull + slot);
      }
    } else if (warp == kScoreWarp) {
      // ---------------- tcgen05: S products ----------------
      if (elect_one_sync()) {
        constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
        constexpr uint32_t idS = kF8 ? make_idesc_e4m3(BT, C::kSCols, 0, 0) : make_idesc_16(BT, NP, 0, 0, kBf16);
        const uint64_t dQ0 = make_sdesc_sw128(smem_u32(sQ), 16, 1024);
        const uint64_t dK0 = make_sdesc_sw128(smem_u32(sKV + kTile), 16, 1024);
        int t = 0;
        for (Walk w = w0; w.left > 0; w.next(), ++t) {
          const int slot = w.seg % kQSlots, buf = t & 3;
          if (w.loc == 0 && !mbar_wait(bQfull + slot, (w.seg / kQSlots) & 1, abort_flag, kSiteDecodeTc)) break;
          if (t >= 4 && !mbar_wait(bSfree + buf, ((t >> 2) - 1) & 1, abort_flag, kSiteDecodeTc)) break;
          if (!mbar_wait(bFull + t % NS, (t / NS) & 1, abort_flag, kSiteDecodeTc)) break;
          tc_fence_after();
          const uint64_t dk = sdesc_add(dK0, (t % NS) * 2 * kTile), dq = sdesc_add(dQ0, slot * C::kQBytes);
          const uint32_t col = tmem + buf * C::kSCols;
          if constexpr (kF8) {
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) mma_ss_f8(col, sdesc_add(dk, kk * 32), sdesc_add(dq, kk * 32), idS, kk > 0);
          } else {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              mma_ss(col, sdesc_add(dk, (kk >> 2) * (BT * 128) + (kk & 3) * 32),
                     sdesc_add(dq, (kk >> 2) * C::kQBlock + (kk & 3) * 32), idS, kk > 0);
          }
          mma_commit(bSf + buf);
          if (w.last()) mma_commit(bQfree + slot);
        }
        // every issued product completes before TMEM and shared memory go away
        mma_commit(bDrain);
        volatile int no_abort = 0;
        mbar_wait(bDrain, 0, &no_abort, kSiteDecodeTc);
      }
    } else if (warp == kValueWarp) {
      // ---------------- tcgen05: P V products ----------------
      if (elect_one_sync()) {
        constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
        constexpr uint32_t idO = kF8 ? make_idesc_e4m3(128, C::kOCols, 1, 0) : make_idesc_16(128, NP, 1, 0, kBf16);
        const uint64_t dP0 = make_sdesc_sw128(smem_u32(sP), 16, 1024);
        // D = 64: M is still 128, with the K tile's 64 columns behind V's as
        // the other half; its rows of the accumulator are never read
        const uint64_t dV0 = make_sdesc_sw128(smem_u32(sKV), D == 64 ? kTile : BT * 128, 1024);
        int t = 0;
        for (Walk w = w0; w.left > 0; w.next(), ++t) {
          const int grp = t & 1;
          const int par = w.seg & 1;
          if (w.loc == 0 && w.seg > 1 && !mbar_wait(bOfree + par, ((w.seg >> 1) - 1) & 1, abort_flag, kSiteDecodeTc)) break;
          if (!mbar_wait(bPf + grp, (t >> 1) & 1, abort_flag, kSiteDecodeTc)) break;
          tc_fence_after();
          const uint64_t dv = sdesc_add(dV0, (t % NS) * 2 * kTile), dp = sdesc_add(dP0, grp * C::kPBytes);
          const uint32_t col = tmem + C::kColO + (par * kGroups + grp) * C::kOCols;
          const bool more = w.loc >= kGroups;    // the group's accumulator already holds tiles of this segment
          if constexpr (kF8) {
#pragma unroll
            for (int kk = 0; kk < BT / 32; ++kk)
              mma_ss_f8(col, sdesc_add(dv, kk * 32 * 128), sdesc_add(dp, kk * 32), idO, more || kk > 0);
          } else {
#pragma unroll
            for (int kk = 0; kk < BT / 16; ++kk)
              mma_ss(col, sdesc_add(dv, kk * 16 * 128), sdesc_add(dp, (kk >> 2) * C::kQBlock + (kk & 3) * 32), idO, more || kk > 0);
          }
          mma_commit(bPv + grp);
          mma_commit(bEmpty + t % NS);
          if (w.last()) mma_commit(bOdone + par);
        }
        mma_commit(bDrain + 1);
        volatile int no_abort = 0;
        mbar_wait(bDrain + 1, 0, &no_abort, kSiteDecodeTc);
      }
    }
  } else if (warp < kSoftmax / 32) {
    reg_alloc<kSoftmaxRegs>();
    // ---------------- softmax groups ----------------
    const int grp = warp >> 2, row = tid & 127, w4 = warp & 3;
    const uint32_t lane_base = static_cast<uint32_t>(w4 * 32) << 16;
    uint8_t* myP = sP + grp * C::kPBytes;
    const int box_shift = 31 - __clz(p.box);
    int t = 0, mine = 0;                   // tiles of the CTA so far, of this group
    Walk w = w0;
    while (w.left > 0) {
      // ---- one segment ----
      const int seg = w.seg, par = seg & 1, t0 = w.t, n = min(w.left, w.tiles - t0), len = w.len;
      const int slice = p.slices == 1 ? 0 : w.r % p.slices, G = min(NP, p.group - slice * NP);
      float qf = p.scale_log2, qs[NP];     // e4m3: a factor per head undoes the query's scale
      if constexpr (kF8) {
        const int slot = seg % kQSlots;
        mbar_wait(bQfull + slot, (seg / kQSlots) & 1, abort_flag, kSiteDecodeTc);
#pragma unroll
        for (int h = 0; h < NP; ++h) qs[h] = s_qinv[slot * NP + h] * p.scale_log2;
        bar_sync_named(1 + grp, 128);
        if (row == 0) mbar_arrive(bQfree + slot);
      }
      float m[NP], l[NP];
#pragma unroll
      for (int h = 0; h < NP; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
      }
      for (int i = 0; i < n; ++i, ++t) {
        if ((t & 1) != grp) continue;
        const int stage = t % NS, buf = t & 3;
        mbar_wait(bSf + buf, (t >> 2) & 1, abort_flag, kSiteDecodeTc);
        mbar_wait(bFull + stage, (t / NS) & 1, abort_flag, kSiteDecodeTc);
        __syncwarp();
        tc_fence_after();
        const bool valid = (t0 + i) * BT + row < len && !((s_bad[stage] >> (row >> box_shift)) & 1u);
        float s[NP];
        {
          uint32_t raw[kQParts][NP];
#pragma unroll
          for (int k = 0; k < kQParts; ++k) tmem_ld16(tmem + lane_base + buf * C::kSCols + k * NP, raw[k]);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < kQParts; ++k) reg_fence(raw[k]);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bSfree + buf);
#pragma unroll
          for (int h = 0; h < NP; ++h) {
            float x = __uint_as_float(raw[0][h]);
            if constexpr (kQParts > 1) x += __uint_as_float(raw[1][h]);
            if constexpr (kQParts > 2) x += __uint_as_float(raw[2][h]);
            s[h] = valid ? x * (kF8 ? qs[h] : qf) : -INFINITY;
          }
        }
        const bool fresh = i < kGroups;    // the group's first tile of the segment
        bool up = false;
        if (!fresh) {
#pragma unroll
          for (int h = 0; h < NP; ++h) up |= h < G && s[h] > m[h] + (C::kShift + C::kRescale);
        }
        if (fresh || bar_any_named(1 + grp, 128, up)) {
          // the tile's maximum of each head over its 128 rows (the buffer
          // alternates: a slow thread may still read the previous one)
          float* gmax = s_max + (grp * 2 + (mine & 1)) * 4 * NP;
          const float wm = reduce16<true>(s, lane);
          if ((lane & 1) == 0) gmax[w4 * NP + (lane >> 1)] = wm;
          bar_sync_named(1 + grp, 128);
          float alpha[NP];
#pragma unroll
          for (int h0 = 0; h0 < NP; h0 += 4) {
            if (h0 >= G) break;
            float4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const float4*>(gmax + k * NP + h0);
            const float tm[4] = {fmaxf(fmaxf(x[0].x, x[1].x), fmaxf(x[2].x, x[3].x)), fmaxf(fmaxf(x[0].y, x[1].y), fmaxf(x[2].y, x[3].y)),
                                 fmaxf(fmaxf(x[0].z, x[1].z), fmaxf(x[2].z, x[3].z)), fmaxf(fmaxf(x[0].w, x[1].w), fmaxf(x[2].w, x[3].w))};
#pragma unroll
            for (int h = h0; h < h0 + 4; ++h) {
              // the same decision in every thread of the group
              const float mx = tm[h - h0], to = mx - C::kShift;
              if (fresh) {
                m[h] = to;
              } else {
                const bool move = mx > m[h] + (C::kShift + C::kRescale);
                alpha[h] = !move ? 1.f : m[h] == -INFINITY ? 0.f : ex2(m[h] - to);
                m[h] = move ? to : m[h];
                l[h] *= alpha[h];
              }
            }
          }
          if (!fresh) {                    // the accumulator holds earlier tiles of this segment
#pragma unroll
            for (int h = 0; h < NP; ++h)
              if (h >= (G + 3) / 4 * 4) alpha[h] = 1.f;
            mbar_wait(bPv + grp, (mine - 1) & 1, abort_flag, kSiteDecodeTc);
            __syncwarp();
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < kPParts; ++k) {
              uint32_t ov[NP];
              const uint32_t at = tmem + lane_base + C::kColO + (par * kGroups + grp) * C::kOCols + k * NP;
              tmem_ld16(at, ov);
              tmem_wait_ld();
              reg_fence(ov);
#pragma unroll
              for (int h = 0; h < NP; ++h) ov[h] = __float_as_uint(__uint_as_float(ov[h]) * alpha[h]);
              tmem_st16(at, ov);
            }
            tmem_wait_st();
          }
        }
        if (!valid) {
          // rows past the length or not loaded: zero V, so that P = 0 times them is 0
          uint8_t* vrow = sKV + stage * 2 * kTile + row * 128;
#pragma unroll
          for (int cb = 0; cb < C::kBlocks; ++cb)
#pragma unroll
            for (int c = 0; c < 8; ++c) reinterpret_cast<uint4*>(vrow + cb * BT * 128)[c] = make_uint4(0u, 0u, 0u, 0u);
        }
        // the group's previous P V product has read its P
        if (mine > 0) mbar_wait(bPv + grp, (mine - 1) & 1, abort_flag, kSiteDecodeTc);
        // Heads are taken four at a time: a branch for each would put their
        // chains of instructions one behind the other.
        float pr[NP];
#pragma unroll
        for (int h0 = 0; h0 < NP; h0 += 4) {
          if (h0 >= G) break;
#pragma unroll
          for (int h = h0; h < h0 + 4; ++h) {
            pr[h] = s[h] == -INFINITY ? 0.f : ex2(s[h] - m[h]);
            l[h] += pr[h];
          }
          if constexpr (kF8) {
            // byte `row` of P's rows h, of each part
            uint8_t* pb = myP + (row & 15);
            const int chunk = row >> 4;
#pragma unroll
            for (int h = h0; h < h0 + 4; h += 2) {
              uint16_t part[kPParts];
              split_e4m3<true>(pr[h], pr[h + 1], part);
              const int o0 = h * 128 + ((chunk ^ (h & 7)) << 4), o1 = (h + 1) * 128 + ((chunk ^ ((h + 1) & 7)) << 4);
#pragma unroll
              for (int k = 0; k < kPParts; ++k) {
                pb[k * C::kQBlock + o0] = (uint8_t)(part[k] & 0xff);
                pb[k * C::kQBlock + o1] = (uint8_t)(part[k] >> 8);
              }
            }
          } else {
            // column `row` of P: block row / 64, 16-byte chunk (row / 8) & 7
            uint8_t* pb = myP + (row >> 6) * C::kQBlock + (row & 7) * 2;
            const int chunk = (row >> 3) & 7;
#pragma unroll
            for (int h = h0; h < h0 + 4; ++h) *reinterpret_cast<uint16_t*>(pb + h * 128 + ((chunk ^ (h & 7)) << 4)) = to16<T>(pr[h]);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(bPf + grp);
        ++mine;
        __syncwarp();
      }

      // ---- the group's maxima and sums of the segment ----
      if (seg > 1) mbar_wait(bOfree + par, ((seg >> 1) - 1) & 1, abort_flag, kSiteDecodeTc);
      const float ls = reduce16<false>(l, lane);
      if ((lane & 1) == 0) s_l[((par * kGroups + grp) * 4 + w4) * NP + (lane >> 1)] = ls;
      if (row == 0) {
#pragma unroll
        for (int h = 0; h < NP; ++h) s_m[(par * kGroups + grp) * NP + h] = m[h];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bSums + par);
      w.next(n);
    }
  } else {
    reg_dealloc<kEndRegs>();
    // ---------------- ends of segments ----------------
    const int row = tid & 127, w4 = warp & 3;
    const uint32_t lane_base = static_cast<uint32_t>(w4 * 32) << 16;
    int t = 0;                             // the segment's first tile
    for (Walk w = w0; w.left > 0;) {
      const int seg = w.seg, par = seg & 1, b = w.b, r = w.r, tiles = w.tiles, n = min(w.left, tiles - w.t);
      const int slice = p.slices == 1 ? 0 : r % p.slices, G = min(NP, p.group - slice * NP);
      const float* pm = s_m + par * kGroups * NP;
      const float* pl = s_l + par * kGroups * 4 * NP;
      mbar_wait(bSums + par, (seg >> 1) & 1, abort_flag, kSiteDecodeTc);
      mbar_wait(bOdone + par, (seg >> 1) & 1, abort_flag, kSiteDecodeTc);
      __syncwarp();
      tc_fence_after();
      // Lane h of every warp: maximum and sum of head h over both groups and
      // the factors of their accumulators, passed on through shared memory
      // (each thread working out 16 heads' took longer than two tiles).
      const bool whole = n == tiles;       // every tile of the item is this CTA's
      const int hl = lane & (NP - 1);
      const float m0 = pm[hl], m1 = pm[NP + hl], M = fmaxf(m0, m1);
      const float a0 = m0 == -INFINITY ? 0.f : ex2(m0 - M), a1 = m1 == -INFINITY ? 0.f : ex2(m1 - M);
      const float* x0 = pl + hl;
      const float* x1 = pl + 4 * NP + hl;
      const float L = fmaf(a0, (x0[0] + x0[NP]) + (x0[2 * NP] + x0[3 * NP]), a1 * ((x1[0] + x1[NP]) + (x1[2 * NP] + x1[3 * NP])));
      const float f = !whole ? p.o_scale : L == 0.f ? 0.f : __fdividef(p.o_scale, L);
      float* fac = s_fac + w4 * 2 * NP;
      fac[lane] = (lane < NP ? a0 : a1) * f;
      __syncwarp();
      float oa[NP];                        // thread `row`: column row of o
#pragma unroll
      for (int h = 0; h < NP; ++h) oa[h] = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        // a group has an accumulator iff it took a tile
        if (!(n > 1 || (t & 1) == g)) continue;
        float wk = 1.f;
#pragma unroll
        for (int k = 0; k < kPParts; ++k, wk *= 1.f / kPartScale) {
          uint32_t ov[NP];
          tmem_ld16(tmem + lane_base + C::kColO + (par * kGroups + g) * C::kOCols + k * NP, ov);
          tmem_wait_ld();
          reg_fence(ov);
#pragma unroll
          for (int h = 0; h < NP; h += 4) {
            const float4 y = *reinterpret_cast<const float4*>(fac + g * NP + h);
            oa[h] = fmaf(__uint_as_float(ov[h]) * wk, y.x, oa[h]);
            oa[h + 1] = fmaf(__uint_as_float(ov[h + 1]) * wk, y.y, oa[h + 1]);
            oa[h + 2] = fmaf(__uint_as_float(ov[h + 2]) * wk, y.z, oa[h + 2]);
            oa[h + 3] = fmaf(__uint_as_float(ov[h + 3]) * wk, y.w, oa[h + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();                        // the factors have been read
      mbar_arrive(bOfree + par);

      // ---- result or record ----
      const size_t bh0 = (size_t)b * p.H + (size_t)(p.slices == 1 ? r : r / p.slices) * p.group + slice * NP;
      if (whole) {
        __nv_bfloat16* o = p.o + bh0 * D + row;
#pragma unroll
        for (int h0 = 0; h0 < NP; h0 += 4) {
          if (h0 >= G) break;
#pragma unroll
          for (int h = h0; h < h0 + 4; ++h)
            if (row < D && h < G) o[h * D] = __float2bfloat16_rn(oa[h]);
        }
        if (p.lse != nullptr && row < G) p.lse[bh0 + row] = L == 0.f ? -INFINITY : (M + lg2(L)) * kLn2;
      } else {
        // unit of the item's first tile, and the CTAs that hold its tiles
        const long long i0 = item0 + (long long)r * (tiles + w0.cost) + w0.cost, i1 = i0 + tiles;
        auto holder = [&](long long x) {   // an estimate in fp64 (x is exact there), then its neighbour if it is off
          long long c = x < rem * (q + 1) ? (long long)((double)x / (double)(q + 1)) : (long long)((double)(x - rem) / (double)q);
          if (part(c) > x) --c;
          else if (part(c + 1) <= x) ++c;
          return c;
        };
        const long long c0 = i0 >= first ? (long long)blockIdx.x : holder(i0);
        const long long c1 = i1 <= end ? (long long)blockIdx.x : holder(i1 - 1);
        // this CTA's record: 0 where the item is the first of its part, else 1
        const int which = seg == 0 ? 0 : 1;
        float* rec = p.rec + ((size_t)blockIdx.x * 2 + which) * NP * (D + kHead);
#pragma unroll
        for (int h = 0; h < NP; ++h) {
          if (row < D && h < G) __stcg(rec + h * (D + kHead) + kHead + row, oa[h]);
        }
        if (row < G) __stcg(reinterpret_cast<float2*>(rec + row * (D + kHead)), make_float2(M, L));
        bar_sync_named(3, 128);
        if (row == 0) {
          // the barrier orders every thread's record before this release, and
          // what the others released before the loads below
          int before;
          asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.count + c0) : "memory");
          *s_last = before == (int)(c1 - c0);
        }
        bar_sync_named(3, 128);
        if (*s_last) {
          // the last CTA of the item joins its records: a warp per head, lane
          // i the i-th record's weight and columns 4 i .. 4 i + 3; weights and
          // columns are asked for together (one L2 round trip per 8 records)
          const int nrec = (int)(c1 - c0) + 1;
          // the first CTA's record is its second unless the item begins its part
          const int w_first = part(c0) < i0 - w0.cost ? 1 : 0;
          for (int h = w4; h < G; h += 4) {
            const float* recs = p.rec + ((size_t)c0 * 2 * NP + h) * (D + kHead);
            constexpr size_t kStep = (size_t)2 * NP * (D + kHead), kSecond = (size_t)NP * (D + kHead);
            float Mx = -INFINITY, Ls = 0.f, o4[4] = {0.f, 0.f, 0.f, 0.f};
            constexpr int kAhead = 8;
            for (int base = 0; base < nrec; base += kAhead) {
              const int many = min(kAhead, nrec - base);
              float2 ml = make_float2(-INFINITY, 0.f);
              if (lane < many)
                ml = __ldcg(reinterpret_cast<const float2*>(recs + (base + lane) * kStep + (base + lane == 0 ? w_first : 0) * kSecond));
              float4 x[kAhead];
#pragma unroll
              for (int u = 0; u < kAhead; ++u) {
                x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (u < many && lane * 4 < D)
                  x[u] = __ldcg(reinterpret_cast<const float4*>(recs + (base + u) * kStep + (base + u == 0 ? w_first : 0) * kSecond + kHead) + lane);
              }
              float bm = fmaxf(ml.x, Mx);
#pragma unroll
              for (int off = 16; off > 0; off >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, off));
              const float keep = Mx == -INFINITY ? 0.f : ex2(Mx - bm);
              const float wt = ml.x == -INFINITY ? 0.f : ex2(ml.x - bm);
              float lw = wt * ml.y;
#pragma unroll
              for (int off = 16; off > 0; off >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, off);
              Ls = fmaf(Ls, keep, lw);
              Mx = bm;
#pragma unroll
              for (int c = 0; c < 4; ++c) o4[c] *= keep;
#pragma unroll
              for (int u = 0; u < kAhead; ++u) {
                const float wu = __shfl_sync(0xffffffffu, wt, u);   // 0 behind the last record
                o4[0] = fmaf(wu, x[u].x, o4[0]);
                o4[1] = fmaf(wu, x[u].y, o4[1]);
                o4[2] = fmaf(wu, x[u].z, o4[2]);
                o4[3] = fmaf(wu, x[u].w, o4[3]);
              }
            }
            const float inv = Ls == 0.f ? 0.f : 1.f / Ls;
            if (lane * 4 < D) {
              uint2 out;
              out.x = pack_bf16x2(o4[0] * inv, o4[1] * inv);
              out.y = pack_bf16x2(o4[2] * inv, o4[3] * inv);
              reinterpret_cast<uint2*>(p.o + (bh0 + h) * D)[lane] = out;
            }
            if (lane == 0 && p.lse != nullptr) p.lse[bh0 + h] = Ls == 0.f ? -INFINITY : (Mx + lg2(Ls)) * kLn2;
          }
          if (row == 0) p.count[c0] = 0;     // left zeroed for the next call
        }
      }
      // on to the next segment; a new sequence begins behind this one's items
      t += n;
      w.next(n);
      if (w.left > 0 && w.b != b) item0 += (long long)w.inner * (tiles + w.cost);
    }
    // sequences that hold nothing
    for (int b = blockIdx.x; b < p.B; b += (int)gridDim.x) {
      if (w0.len_of(b) > 0) continue;
      for (int i = row; i < p.H * D / 2; i += 128)
        reinterpret_cast<uint32_t*>(p.o + (size_t)b * p.H * D)[i] = 0u;
      if (p.lse != nullptr)
        for (int i = row; i < p.H; i += 128) p.lse[(size_t)b * p.H + i] = -INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kScoreWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

inline bool eligible(long long H, long long H_kv, long long D, int q_dtype, int kv_dtype) {
  if (q_dtype != PU_DTYPE_F16 && q_dtype != PU_DTYPE_BF16) return false;
  if (kv_dtype == PU_DTYPE_FP8_E4M3) return D == 128;
  return (D == 64 || D == 128) && q_dtype == kv_dtype && H / H_kv >= 2;
}

inline size_t workspace_bytes(long long D) {
  return kCountBytes + round_up((size_t)sm_count() * 2 * NP * (D + kHead) * sizeof(float), 256);
}

template <typename T, typename KVT, int D>
int launch_as(const CUtensorMap& tk, const CUtensorMap& tv, const Params& prm, cudaStream_t st) {
  constexpr int smem = Cfg<T, KVT, D>::kSmem;
  const int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(paged_tc_kernel<T, KVT, D>), smem,
                                      "paged grouped-head decode shared memory");
  if (rc) return rc;
  return check_cuda(launch_pdl(paged_tc_kernel<T, KVT, D>, dim3((unsigned)sm_count()), dim3(kCtaThreads), smem, st, tk, tv, prm),
                    "paged grouped-head decode launch");
}

inline int launch(const Params& prm, const void* k, const void* v, int q_dtype, int kv_dtype, int D, cudaStream_t st) {
  const bool f8 = kv_dtype == PU_DTYPE_FP8_E4M3;
  const uint64_t rows = 1ull << prm.page_shift, outer = (uint64_t)prm.num_pages * prm.H_kv;
  CUtensorMap tk, tv;
  int rc = f8 ? make_tmap_u8_3d(&tk, k, D, rows, outer, 128, prm.box, true)
              : make_tmap_bf16_3d(&tk, k, D, rows, outer, 64, prm.box, true);
  if (!rc)
    rc = f8 ? make_tmap_u8_3d(&tv, v, D, rows, outer, 128, prm.box, true)
            : make_tmap_bf16_3d(&tv, v, D, rows, outer, 64, prm.box, true);
  if (rc) return rc;
  const bool h = q_dtype == PU_DTYPE_F16;
  if (f8)
    return h ? launch_as<__half, __nv_fp8_e4m3, 128>(tk, tv, prm, st)
             : launch_as<__nv_bfloat16, __nv_fp8_e4m3, 128>(tk, tv, prm, st);
  if (D == 128)
    return h ? launch_as<__half, __half, 128>(tk, tv, prm, st) : launch_as<__nv_bfloat16, __nv_bfloat16, 128>(tk, tv, prm, st);
  return h ? launch_as<__half, __half, 64>(tk, tv, prm, st) : launch_as<__nv_bfloat16, __nv_bfloat16, 64>(tk, tv, prm, st);
}

}  // namespace ptc
}  // namespace decode
}  // namespace pu

extern "C" {

size_t pu_decode_paged_gqa_workspace_size(int64_t B, int64_t H, int64_t H_kv, int64_t max_pages_per_seq,
                                          int64_t page_size, int64_t D) {
  using namespace pu::decode;
  if (B <= 0 || H <= 0 || H_kv <= 0 || H % H_kv || max_pages_per_seq <= 0 || page_size <= 0 || D <= 0) return 0;
  if (B > kMaxBH / H) return ptc::workspace_bytes(D);      // the tensor-core kernel's alone
  return std::max(ptc::workspace_bytes(D), pu_decode_paged_workspace_size(B, H, max_pages_per_seq, page_size, D));
}

int pu_decode_paged_gqa(const void* q, int q_dtype, const void* k_pool, const void* v_pool, int kv_dtype,
                        const int32_t* page_table, int64_t max_pages_per_seq, int64_t num_pages, int64_t page_size,
                        const int32_t* kv_lens, void* o, float* lse, void* workspace, size_t workspace_bytes, int64_t B,
                        int64_t H, int64_t H_kv, int64_t D, float sm_scale, float k_scale, float v_scale, void* stream) {
  using namespace pu::decode;
  int shift = 0;
  int rc = pu::paged::check_pages(page_table, max_pages_per_seq, num_pages, page_size, &shift);
  if (rc) return rc;
  const long long n_cap = max_pages_per_seq * page_size;
  rc = check_args(q, q_dtype, k_pool, v_pool, kv_dtype, B, H, n_cap, D, true, false);
  if (rc) return rc;
  if (!o || !kv_lens) return pu::set_error(PU_ERR_INVALID_ARGUMENT, "null output or lengths");
  if (!pu::aligned16(o) || !pu::aligned16(workspace))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "the output and the workspace must be 16-byte aligned");
  if (H_kv <= 0 || H % H_kv != 0)
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "H = %lld is not a multiple of H_kv = %lld", (long long)H, (long long)H_kv);
  if (num_pages > 2147483647ll / H_kv) return pu::set_error(PU_ERR_UNSUPPORTED, "page pool too large");
  if (!(k_scale > 0.f) || !(v_scale > 0.f) || !isfinite(k_scale) || !isfinite(v_scale))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "k_scale and v_scale must be positive and finite");
  const bool tensor = ptc::eligible(H, H_kv, D, q_dtype, kv_dtype);
  // the query-head kernel has a counter and a grid row for each (b, h), the
  // tensor-core kernel a counter for each CTA
  if (H > kMaxBH || (B > kMaxBH / H && (!tensor || B > ptc::kMaxB)))
    return pu::set_error(PU_ERR_UNSUPPORTED, "paged decode of %lld sequences with %lld heads (B * H up to %d, or on the tensor core B up to %d)",
                         (long long)B, (long long)H, kMaxBH, ptc::kMaxB);
  Plan pl{};
  if (!tensor) pl = make_plan(B * H, n_cap, D, pu::sm_count(), true, page_size);
  const size_t need = tensor ? ptc::workspace_bytes(D) : pl.total_bytes;
  if (!workspace || workspace_bytes < need)
    return pu::set_error(PU_ERR_WORKSPACE, "paged decode workspace needs %zu bytes, got %zu", need, workspace_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const float scale_log2 = sm_scale * k_scale * kLog2e;
  if (tensor) {
    ptc::Params prm{};
    prm.q = q;
    prm.table = page_table;
    prm.lens = kv_lens;
    prm.o = static_cast<__nv_bfloat16*>(o);
    prm.lse = lse;
    prm.count = static_cast<int*>(workspace);
    prm.rec = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCountBytes);
    prm.B = (int)B;
    prm.H = (int)H;
    prm.H_kv = (int)H_kv;
    prm.group = (int)(H / H_kv);
    prm.slices = (prm.group + ptc::NP - 1) / ptc::NP;
    prm.max_pages = (int)max_pages_per_seq;
    prm.num_pages = (int)num_pages;
    prm.page_shift = shift;
    prm.box = (int)std::min<long long>(page_size, ptc::BT);
    prm.scale_log2 = scale_log2;
    prm.o_scale = v_scale;
    return ptc::launch(prm, k_pool, v_pool, q_dtype, kv_dtype, (int)D, st);
  }
  // q and cache of different 16-bit types, one query head per K/V head, and
  // e4m3 caches with D = 64: the query-head kernel reading K/V head h / G
  Params prm{};
  prm.q = q;
  prm.k = k_pool;
  prm.v = v_pool;
  prm.lens = kv_lens;
  prm.kv_offset = 0;
  prm.n_local = (int)n_cap;
  prm.H = (int)H;
  prm.group = (int)(H / H_kv);
  prm.o_scale = v_scale;
  prm.splits = pl.splits;
  prm.chunk = pl.chunk;
  prm.scale_log2 = scale_log2;
  prm.ws_rec = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.rec_off);
  prm.ws_count = static_cast<int*>(workspace);
  prm.o = static_cast<__nv_bfloat16*>(o);
  prm.lse = lse;
  prm.page_table = page_table;
  prm.max_pages = (int)max_pages_per_seq;
  prm.num_pages = (int)num_pages;
  prm.page_shift = shift;
  return launch<true, true>(prm, q_dtype, kv_dtype, (int)D, (int)(B * H), st);
}

}  // extern "C"
