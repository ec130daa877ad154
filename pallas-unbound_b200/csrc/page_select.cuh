// page_select.cuh — which pages of a cache a query attends: bounds of each
// page's keys, kept up to date as tokens are written, and the choice of pages
// by an upper bound of their scores.
//
// No counterpart in the reference (its decode reads every token of a dense
// cache, src/pallas_flash/kernels/decoding.py:86-103).
//
// Bounds.  lo_p and hi_p are the elementwise minimum and maximum of page p's
// keys, for each K/V head: bounds [num_pages][H_kv][2][D] in the pool's 16-bit
// type, or f16 for an e4m3 pool (which holds every e4m3 value).  A minimum is a
// choice, not a sum: no rounding, and the same bits in any order.
//
// Choice.  For query heads h of one K/V head and any key k of page p
//   sum_h q_h k <= sum_h sum_d max(q_hd lo_pd, q_hd hi_pd)
//                = sum_d hi_pd a_d + lo_pd b_d,  a_d = sum_h max(q_hd, 0), b_d = sum_h min(q_hd, 0),
// since lo <= hi: one dot product of 2 D values a page however many heads share
// it, and bound by reading the bounds once.  The sums are held in 64 bits: the
// page kept and the page dropped at the border differ by little, and fp32 sums
// would choose by their rounding.
#pragma once

#include "paged.cuh"

namespace pu {
namespace choose {

// ---------------------------------------------------------------------------
// bounds
// ---------------------------------------------------------------------------
constexpr int kBoundThreads = 256;
constexpr int kChunk = 32;               // most rows of the packed batch a CTA looks at

struct BoundParams {
  const void* k_pool;          // [num_pages][H_kv][page][D]
  const int32_t* slots;        // [T]
  void* bounds;                // [num_pages][H_kv][2][D]
  int H_kv, num_pages, page_shift;
  int chunk;                   // rows of the packed batch a CTA looks at: 8 or 32
  int heads;                   // K/V heads it takes
  long long T;
};

// Minimum or maximum of pairs; a NaN stays one.
template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using V = __half2;
  static constexpr uint32_t kInf = 0x7c007c00u, kMinusInf = 0xfc00fc00u;
};
template <>
struct Pair<__nv_bfloat16> {
  using V = __nv_bfloat162;
  static constexpr uint32_t kInf = 0x7f807f80u, kMinusInf = 0xff80ff80u;
};

template <typename T>
__device__ __forceinline__ uint32_t pair_min(uint32_t a, uint32_t b) {
  using V = typename Pair<T>::V;
  const V r = __hmin2_nan(*reinterpret_cast<const V*>(&a), *reinterpret_cast<const V*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {
  using V = typename Pair<T>::V;
  const V r = __hmax2_nan(*reinterpret_cast<const V*>(&a), *reinterpret_cast<const V*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// A CTA looks at 8 or 32 rows of the packed batch and some of the K/V heads.  The rows of a page stand
// together, in order: the first of such a run is its leader, and the CTA that holds the leader takes the
// whole run, wherever it ends, so that one CTA reads and writes the page's bounds.  A warp takes a
// (leader, head); where there are fewer of them than warps, warps share one.
template <typename KVT, int D>
__global__ void __launch_bounds__(kBoundThreads, 3) bounds_kernel(const BoundParams p) {
  constexpr bool kF8 = sizeof(KVT) == 1;
  using B = typename std::conditional<kF8, __half, KVT>::type;     // type of the bounds
  constexpr int kLanes = D * (int)sizeof(KVT) / 16;                // lanes of a row, 16 bytes each
  constexpr int kRows = 32 / kLanes;                               // rows a warp reads at once
  constexpr int kWords = kF8 ? 8 : 4;                              // pairs a lane holds
  constexpr int kVecs = kWords / 4;                                // 16-byte vectors of them
  constexpr int kAhead = 8;                                        // reads in flight
  __shared__ int s_slot[kChunk], s_at[kChunk], s_rows[kChunk], s_count;
  __shared__ uint4 s_part[kBoundThreads / 32][2][D / 8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int page = 1 << p.page_shift, head0 = blockIdx.y * p.heads, heads = min(p.heads, p.H_kv - head0);
  const long long places = (long long)p.num_pages << p.page_shift;
  grid_dep_wait();
  grid_dep_launch_dependents();
  const long long t0 = (long long)blockIdx.x * p.chunk;
  if (warp == 0) {
    const long long t = t0 + lane;
    int slot = lane < p.chunk && t < p.T ? p.slots[t] : -1;
    int before = lane == 0 && t0 > 0 ? p.slots[t0 - 1] : -1;
    const int up = __shfl_up_sync(0xffffffffu, slot, 1);
    if (lane > 0) before = up;
    if (slot >= places) {
      if (head0 == 0) record_device_error(PU_ERR_INVALID_ARGUMENT, kSitePageBounds);
      slot = -1;
    }
    const bool follows = slot >= 0 && before == slot - 1 && (slot & (page - 1)) != 0, leads = slot >= 0 && !follows;
    const unsigned first = __ballot_sync(0xffffffffu, leads), rest = __ballot_sync(0xffffffffu, follows);
    if (leads) {
      const int k = __popc(first & ((1u << lane) - 1)), n = __ffs(~((rest >> lane) >> 1));     // 1 and those that follow
      s_slot[k] = slot;
      s_at[k] = lane;
      s_rows[k] = n;
    }
    if (lane == 0) s_count = __popc(first);
  }
  __syncthreads();
  const int n = s_count * heads;
  // warps that share a unit: 8 where there is one, 1 from eight units on
  const int team = n <= 1 ? 8 : n <= 2 ? 4 : n <= 4 ? 2 : 1, teams = 8 / team;
  const int sub = lane / kLanes, vec = lane % kLanes;
  for (int i0 = 0; i0 < n; i0 += teams) {
    const int i = i0 + warp / team, part = warp % team;
    uint32_t lo[kWords], hi[kWords];
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      lo[w] = Pair<B>::kInf;
      hi[w] = Pair<B>::kMinusInf;
    }
    uint4* out = nullptr;
    auto fold = [&](int w, const uint4& a, const uint4& b) {
      const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo[w + j] = pair_min<B>(lo[w + j], x[j]);
        hi[w + j] = pair_max<B>(hi[w + j], y[j]);
      }
    };
    if (i < n) {
      const int k = i / heads, head = head0 + i % heads, slot = s_slot[k], row = slot & (page - 1);
      const size_t at = (size_t)(slot >> p.page_shift) * p.H_kv + head;
      out = reinterpret_cast<uint4*>(p.bounds) + at * (2 * D / 8) + vec * kVecs;
      // what the page's bounds were, where rows of it were written before
      const bool old = row != 0 && part == 0 && sub == 0;
      uint4 old_lo[kVecs], old_hi[kVecs];
#pragma unroll
      for (int w = 0; w < kVecs; ++w) {
        old_lo[w] = make_uint4(0u, 0u, 0u, 0u);
        old_hi[w] = old_lo[w];
        if (old) {
          old_lo[w] = out[w];
          old_hi[w] = out[D / 8 + w];
        }
      }
      // a run that reaches the end of the CTA's rows may go on: as long as the next slot is the next row of the page
      int rows = s_rows[k];
      if (s_at[k] + rows == p.chunk) {
        const long long t = t0 + s_at[k];
        const int most = (int)min((long long)(page - row), p.T - t);
        for (int r = rows; r < most; r += 32) {
          const bool more = r + lane < most && p.slots[t + r + lane] == slot + r + lane;
          const unsigned gap = ~__ballot_sync(0xffffffffu, more);
          rows = gap ? r + __ffs(gap) - 1 : r + 32;
          if (gap) break;
        }
      }
      const uint4* src = reinterpret_cast<const uint4*>(p.k_pool) + ((at << p.page_shift) + row) * kLanes + vec;
      for (int r0 = part * kRows + sub; r0 < rows; r0 += kAhead * team * kRows) {
        uint4 x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          // past the end the first row again, which changes nothing
          const int r = r0 + u * team * kRows;
          x[u] = decode::ld_stream(src + (size_t)(r < rows ? r : r0) * kLanes);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const uint32_t w4[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            uint32_t v = w4[w >> (kF8 ? 1 : 0)];
            if constexpr (kF8) {
              const __half2 h(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v >> (16 * (w & 1))), __NV_E4M3));
              v = *reinterpret_cast<const uint32_t*>(&h);
            }
            lo[w] = pair_min<B>(lo[w], v);
            hi[w] = pair_max<B>(hi[w], v);
          }
        }
      }
      // over the warp's rows
#pragma unroll
      for (int off = kLanes; off < 32; off <<= 1) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          lo[w] = pair_min<B>(lo[w], __shfl_xor_sync(0xffffffffu, lo[w], off));
          hi[w] = pair_max<B>(hi[w], __shfl_xor_sync(0xffffffffu, hi[w], off));
        }
      }
#pragma unroll
      for (int w = 0; w < kVecs; ++w) {
        if (old) fold(4 * w, old_lo[w], old_hi[w]);
        if (team > 1 && sub == 0) {
          s_part[warp][0][vec * kVecs + w] = make_uint4(lo[4 * w], lo[4 * w + 1], lo[4 * w + 2], lo[4 * w + 3]);
          s_part[warp][1][vec * kVecs + w] = make_uint4(hi[4 * w], hi[4 * w + 1], hi[4 * w + 2], hi[4 * w + 3]);
        }
      }
    }
    if (team > 1) __syncthreads();
    if (i < n && part == 0 && sub == 0) {
#pragma unroll
      for (int w = 0; w < kVecs; ++w) {
        for (int o = 1; o < team; ++o) fold(4 * w, s_part[warp + o][0][vec * kVecs + w], s_part[warp + o][1][vec * kVecs + w]);
        out[w] = make_uint4(lo[4 * w], lo[4 * w + 1], lo[4 * w + 2], lo[4 * w + 3]);
        out[D / 8 + w] = make_uint4(hi[4 * w], hi[4 * w + 1], hi[4 * w + 2], hi[4 * w + 3]);
      }
    }
    if (team > 1) __syncthreads();       // before the parts are written again
  }
}

// ---------------------------------------------------------------------------
// choice
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kRank = kThreads;          // as many candidates are ranked against each other
constexpr int kMaxPages = 24576;         // scores of a sequence that one CTA's shared memory holds
constexpr int kMaxCtas = 8;              // of a cluster
// Stages of a warp's copies, eight pages each.  Six, where a warp has many steps, leave one CTA an SM: 24 sequences
// of 131072 tokens, heads of 64, pages of 16 take 131 us instead of 84, three of them 22 instead of 18 (lengths
// from 0 to 131072: 67 instead of 73).  With heads of 128 they make no difference (52.5 to 53, 98.6 to 99.7).
constexpr int kStages = 3;
constexpr float kBig = 0x1p125f;         // fp32 sums from here on are not used
constexpr uint32_t kOutside = 0x10000u;  // a warp has seen a table entry outside the pool

struct Params {
  const void* q;               // [B][H][D]
  const void* bounds;          // [num_pages][H_kv][2][D]
  const int32_t* table;        // [B][max_pages]
  const int32_t* lens;         // [B]
  int32_t* pages;              // [B][H_kv][count]
  int32_t* out_lens;           // [B][H_kv]
  int H, H_kv, group;
  int max_pages, num_pages, page_shift;
  int count, first, last;
  int ctas;                    // of a cluster
  int by_length;               // the longest sequences are placed first
  int ring;                    // first byte of the copies, behind the scores
  int stages;                  // kStages, as an argument: known to the compiler, its order of the scoring loop takes 104.5 us
                               // instead of 98.8 (24 sequences of 131072 tokens, heads of 128), 88 instead of 84 (64)
  int B;
};

// A 16-bit value as fp64 times a power of two (2^-896 for bf16, 2^-1008 for f16): its sign,
// exponent and mantissa bits moved to their places, which is exact for subnormals as well.
// Infinities and NaN become values beyond the largest.
template <typename T>
__device__ __forceinline__ double wide(uint32_t high_half) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const int x = (int)high_half >> (kBf16 ? 3 : 6);
  return __hiloint2double(x & (kBf16 ? 0x8fffe000 : 0x81fffc00), 0);
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// A pair of 16-bit values as packed fp32.
template <typename T>
__device__ __forceinline__ uint64_t pair_to_f2(uint32_t w);
template <>
__device__ __forceinline__ uint64_t pair_to_f2<__nv_bfloat16>(uint32_t w) {
  return f2_pack(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ uint64_t pair_to_f2<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return f2_pack(f.x, f.y);
}

// 16 bytes from global to shared memory, zeros unless `ok`.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Shared memory of the choice.
struct Room {
  double cand[kRank];          // scores summed again
  double red[2][kWarps];
  double cut;
  int bins[kBins];
  int list[kRank];
  float near[kRank];           // their fp32 sums
  int sum[kWarps], tie[kWarps], scan[kWarps];
  int found[4];                // border bin, members above it, its members, members listed
  float edge;
};

// Sum over the block (every thread gets it).
__device__ __forceinline__ int block_sum(int x, Room& s, int warp, int lane) {
  x = __reduce_add_sync(0xffffffffu, x);
  if (lane == 0) s.sum[warp] = x;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all += s.sum[w];
  __syncthreads();
  return all;
}

// Calls f(i, score[i]) for this thread's part of [from, to): four reads at a time, which a loop with
// atomics or stores between its reads would take one after the other.
template <typename S, typename F>
__device__ __forceinline__ void each(const S* score, int from, int to, F f) {
  constexpr int kAhead = 4;
  int i = from + (int)threadIdx.x;
  for (; i + (kAhead - 1) * kThreads < to; i += kAhead * kThreads) {
    S x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) x[u] = score[i + u * kThreads];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) f(i + u * kThreads, x[u]);
  }
#pragma unroll 1
  for (; i < to; i += kThreads) f(i, score[i]);
}

// Smallest and largest of all threads' lo and hi.
template <typename S>
__device__ __forceinline__ void block_range(S& lo, S& hi, Room& s, int warp, int lane) {
  S(&red)[2][kWarps] = reinterpret_cast<S(&)[2][kWarps]>(s.red);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  if (lane == 0) {
    red[0][warp] = lo;
    red[1][warp] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    lo = min(lo, red[0][w]);
    hi = max(hi, red[1][w]);
  }
}

// Counts the scores in [lo, hi] (lo < hi) in kBins bins of equal width and finds the one that holds the
// want-th largest: s.found = {bin, members of the bins above, its members, 0}.  The map to bins is
// monotone, so no rounding of it orders two scores wrongly.
template <typename S>
struct Bins {
  S lo, scale;
  // (hi - lo is neither 0 nor infinite, so hi is never in lo's bin)
  __device__ __forceinline__ Bins(S lo_, S hi) : lo(lo_), scale((S)(kBins - 1) / (hi - lo_)) {}
  __device__ __forceinline__ int of(S x) const { return min(kBins - 1, (int)((x - lo) * scale)); }
};

template <typename S>
__device__ __forceinline__ void find_bin(const S* score, int from, int to, S lo, S hi, const Bins<S>& bins, int want, Room& s) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
  __syncthreads();
  each(score, from, to, [&](int, S x) {
    if (x >= lo && x <= hi) atomicAdd(s.bins + bins.of(x), 1);
  });
  __syncthreads();
  // a thread's four bins, counted from the top
  constexpr int kPer = kBins / kThreads;
  const int top = kBins - 1 - tid * kPer;
  int c[kPer], mine = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    c[k] = s.bins[top - k];
    mine += c[k];
  }
  int before = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += y;
  }
  if (lane == 31) s.scan[warp] = before;
  if (tid == 0) s.found[3] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) before += w < warp ? s.scan[w] : 0;
  before -= mine;                        // candidates in the bins above this thread's
  if (before < want && before + mine >= want) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (before < want && before + c[k] >= want) {
        s.found[0] = top - k;
        s.found[1] = before;
        s.found[2] = c[k];
      }
      before += c[k];
    }
  }
  __syncthreads();
}

// The want-th largest (want >= 1) of the finite scores in [from, to), of which there are more than `want`,
// and how many that equal it are among the first `want`.  Bins, then the border bin's members are ranked
// against each other; where they are more than 256 the same is done again between their own smallest and
// largest.
__device__ __forceinline__ void border(const double* score, int from, int to, int want, Room& s, double* cut, int* ties) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  double lo = INFINITY, hi = -INFINITY;
  each(score, from, to, [&](int, double x) {
    if (!isinf(x)) {
      lo = min(lo, x);
      hi = max(hi, x);
    }
  });
  while (true) {
    block_range(lo, hi, s, warp, lane);
    if (lo == hi) {                      // equal scores: the first of them
      *cut = lo;
      *ties = want;
      break;
    }
    const Bins<double> bins(lo, hi);
    find_bin(score, from, to, lo, hi, bins, want, s);
    const int at = s.found[0], members = s.found[2];
    want -= s.found[1];
    __syncthreads();
    if (members <= kRank) {
      each(score, from, to, [&](int, double x) {
        if (x >= lo && x <= hi && bins.of(x) == at) s.cand[atomicAdd(s.found + 3, 1)] = x;
      });
      __syncthreads();
      if (tid < members) {
        // fewer than `want` above it, at least `want` with its equals
        const double x = s.cand[tid];
        int above = 0, same = 0;
        for (int i = 0; i < members; ++i) {
          above += s.cand[i] > x;
          same += s.cand[i] == x;
        }
        if (above < want && above + same >= want) {
          s.cut = x;
          s.found[1] = want - above;     // equal threads write equal values
        }
      }
      __syncthreads();
      *cut = s.cut;
      *ties = s.found[1];
      break;
    }
    // again among the border's members
    double lo2 = INFINITY, hi2 = -INFINITY;
    each(score, from, to, [&](int, double x) {
      if (x >= lo && x <= hi && bins.of(x) == at) {
        lo2 = min(lo2, x);
        hi2 = max(hi2, x);
      }
    });
    lo = lo2;
    hi = hi2;
    __syncthreads();
  }
  __syncthreads();                       // the room is free again
}

// The list, in the sequence's order: pages above `cut`, and the first `ties` equal to it (a cut of -inf has
// none).  A run of pages a warp, counted and then written.
template <typename S>
__device__ __forceinline__ void write_list(const Params& p, const int32_t* table, const S* score, S cut, int ties, int live, int len, size_t row,
                                           Room& s) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int run = ((live + kWarps - 1) / kWarps + 31) & ~31, begin = warp * run, end = min(live, begin + run);
  constexpr int kAhead = 4;              // reads of 32 scores at a time
  S x[kAhead];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) x[u] = base + u * 32 + lane < end ? score[base + u * 32 + lane] : (S)-INFINITY;
  };
  int above = 0, same = 0;
  for (int base = begin; base < end; base += kAhead * 32) {
    load(base);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      above += __popc(__ballot_sync(0xffffffffu, x[u] > cut));
      if (ties > 0) same += __popc(__ballot_sync(0xffffffffu, x[u] == cut));
    }
  }
  if (lane == 0) {
    s.sum[warp] = above;
    s.tie[warp] = same;
  }
  __syncthreads();
  int a0 = 0, t0 = 0, a1 = 0, t1 = 0;    // before this warp, and in all
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      a0 += s.sum[w];
      t0 += s.tie[w];
    }
    a1 += s.sum[w];
    t1 += s.tie[w];
  }
  const int chosen = min(p.count, a1 + min(ties, t1));
  int32_t* out = p.pages + row * p.count;
  for (int base = begin; base < end; base += kAhead * 32) {
    if (run > kAhead * 32) load(base);   // otherwise they are still there
    int32_t entry[kAhead];
    int place[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const unsigned up = __ballot_sync(0xffffffffu, x[u] > cut), eq = ties > 0 ? __ballot_sync(0xffffffffu, x[u] == cut) : 0u;
      const unsigned below = (1u << lane) - 1;
      const int nth = t0 + __popc(eq & below);           // ties before this page
      const bool in = ((up >> lane) & 1u) || (((eq >> lane) & 1u) && nth < ties);
      place[u] = in ? a0 + __popc(up & below) + min(ties, nth) : p.count;
      entry[u] = place[u] < p.count ? table[base + u * 32 + lane] : 0;
      a0 += __popc(up);
      t0 += __popc(eq);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (place[u] < p.count) out[place[u]] = entry[u];
  }
  for (int i = chosen + tid; i < p.count; i += kThreads) out[i] = -1;
  if (tid == 0) {
    // only the sequence's last page may hold fewer tokens than a page; it is last in the list
    int tokens = chosen << p.page_shift;
    if (live > 0) {
      const S y = score[live - 1];
      if (y > cut || (y == cut && t1 - 1 < ties)) tokens -= (live << p.page_shift) - len;
    }
    p.out_lens[row] = tokens;
  }
}

// One cluster a (sequence, K/V head): its CTAs score the pages between them and leave the scores in
// the first one's shared memory, which chooses.
//
// Scores are first summed in fp32, with a bound of what they are off by:
//   e = 2^-19 max |x| sum_d |c_d|  (x the bounds, c the heads' sums; 16 + 4 roundings of 2^-24 each, and c's)
// The k-th largest of the true scores then lies within e of the k-th largest v of these, so pages above
// v + 2 e are chosen, pages below v - 2 e are not, and only pages between, if there are more than places
// left, are summed again in fp64 from their bounds: nearly always none.
//
// A page's bounds of one head are 4 D bytes in one piece.  Eight lanes take a page, and each lane copies
// the chunks that it will read itself into shared memory, eight pages a step and two steps ahead: copies
// in flight need no registers and no barrier.
template <typename QT, typename BT, int D>
__global__ void __launch_bounds__(kThreads, 2) select_kernel(const Params p) {
  constexpr int kChunks = 2 * D / 64;    // 16-byte chunks a lane reads of a page
  extern __shared__ __align__(16) uint8_t dyn[];
  float* s_score = reinterpret_cast<float*>(dyn);        // [max_pages], in the first CTA
  __shared__ float s_coef[2][D];         // sums of the heads' negative and positive parts
  __shared__ double s_wide[2][D];        // the same in fp64, times 2^800
  __shared__ double s_abs[kWarps];       // parts of the sum of their magnitudes
  __shared__ uint32_t s_top[kMaxCtas * kWarps];    // largest magnitude of a bound that a warp saw, as bits
  __shared__ int s_b;
  __shared__ Room s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, l8 = lane & 7, sub = lane >> 3;
  const int ctas = p.ctas, rank = (int)(blockIdx.x % (unsigned)ctas), item = (int)(blockIdx.x / (unsigned)ctas);
  const int head = item % p.H_kv;
  int b = item / p.H_kv;
  grid_dep_wait();
  grid_dep_launch_dependents();
  if (p.by_length) {
    // the longest sequences first: they get an SM each while there are any, the short ones the rest
    int* lens = s.bins;
    for (int i = tid; i < p.B; i += kThreads) lens[i] = p.lens[i];
    __syncthreads();
    for (int i = tid; i < p.B; i += kThreads) {
      const int n = lens[i];
      int before = 0;
      for (int j = 0; j < p.B; ++j) before += lens[j] > n || (lens[j] == n && j < i);
      if (before == b) s_b = i;
    }
    __syncthreads();
    b = s_b;
  }
  const int page = 1 << p.page_shift;
  const int len = max(0, min(p.lens[b], p.max_pages << p.page_shift));
  const int live = (len + page - 1) >> p.page_shift;
  const int32_t* table = p.table + (size_t)b * p.max_pages;
  const bool all = live <= p.count;      // nothing to choose
  if (all && rank != 0) return;
  const int from = p.first, to = live - p.last;      // candidates between the pages that are always kept
  const uint4* bounds = static_cast<const uint4*>(p.bounds);
  uint32_t top = 0;

  if (!all) {
    cluster_arrive();                    // every CTA runs before another writes to its shared memory
    // ---- scores: a run of pages a warp ----
    const int workers = ctas * kWarps, per = ((to - from + workers - 1) / workers + 7) & ~7;
    const int begin = from + (rank * kWarps + warp) * per, end = min(to, begin + per);
    const int steps = max(0, (end - begin + 7) >> 3);
    uint8_t* ring = dyn + p.ring + (warp * p.stages * 2 * kChunks * 32 + lane) * 16;
    // table entries of 32 pages at a time, the next 32 on their way
    auto look_up = [&](int i) { return i + lane < end ? table[i + lane] : 0; };
    int entry = look_up(begin), ahead = look_up(begin + 32);
    int row = -1;                        // of an entry for each lane: its bounds' place; negative: not in the pool
    bool outside = false;                // the warp has seen such an entry
    int to_stage = 0, from_stage = 0;
    auto begin_step = [&](int k) {       // copies of pages begin + 8 k + 4 u + sub
      if ((k & 3) == 0) {
        const int i = begin + 8 * k + lane;
        const bool bad = i < end && (unsigned)entry >= (unsigned)p.num_pages;
        row = bad || i >= end ? -1 : entry * p.H_kv + head;
        entry = ahead;
        ahead = look_up(begin + 8 * k + 64);
        if (__any_sync(0xffffffffu, bad)) {
          if (bad) record_device_error(PU_ERR_INVALID_ARGUMENT, kSiteSelectPage);
          outside = true;
        }
      }
      const uint32_t dst = smem_u32(ring + to_stage * 2 * kChunks * 512);
      to_stage = to_stage + 1 == p.stages ? 0 : to_stage + 1;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = __shfl_sync(0xffffffffu, row, (8 * k + 4 * u + sub) & 31);
        const uint4* src = bounds + (size_t)max(at, 0) * (2 * D / 8) + l8;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) cp_async_16(dst + (u * kChunks + c) * 512, src + c * 8, at >= 0);
      }
    };
    for (int k = 0; k < p.stages - 1; ++k) {
      if (k < steps) begin_step(k);
      cp_async_commit();
    }
    // ---- the heads' parts, while the first bounds arrive ----
    double sum = 0.;
    for (int i = tid; i < D; i += kThreads) {
      const QT* q = static_cast<const QT*>(p.q) + ((size_t)b * p.H + (size_t)head * p.group) * D + i;
      double neg = 0., pos = 0.;
      for (int h0 = 0; h0 < p.group; h0 += 8) {
        QT x[8];
#pragma unroll
        for (int h = 0; h < 8; ++h) x[h] = q[(size_t)min(h0 + h, p.group - 1) * D];
#pragma unroll
        for (int h = 0; h < 8; ++h) {
          const float y = h0 + h < p.group ? to_float(x[h]) : 0.f;
          neg += (double)fminf(y, 0.f);
          pos += (double)fmaxf(y, 0.f);
        }
      }
      s_coef[0][i] = (float)neg;
      s_coef[1][i] = (float)pos;
      // with the bounds as they are (wide) every product stays a normal number
      s_wide[0][i] = neg * 0x1p800;
      s_wide[1][i] = pos * 0x1p800;
      sum += pos - neg;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) s_abs[warp] = sum;
    __syncthreads();
    uint64_t coef[kChunks][4];           // of this lane's chunks
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = (c * 8 + l8) * 8 + 2 * e;          // element of the page's 2 D
        coef[c][e] = *reinterpret_cast<const uint64_t*>(&s_coef[i / D][i % D]);
      }
    const uint32_t dst = mapa_shared(s_score, 0);
    cluster_wait();
    uint32_t least = 0u, most = 0u;      // of the minima and the maxima, pair by pair
    bool usable = true;
    for (int k = 0; k < steps; ++k) {
      if (k + p.stages - 1 < steps) begin_step(k + p.stages - 1);
      cp_async_commit();
      cp_async_wait<kStages - 1>();
      const uint8_t* src = ring + from_stage * 2 * kChunks * 512;
      from_stage = from_stage + 1 == p.stages ? 0 : from_stage + 1;
      float x[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint64_t s2 = 0ull;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint4 v = *reinterpret_cast<const uint4*>(src + (u * kChunks + c) * 512);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s2 = f2_fma(pair_to_f2<BT>(w[e]), coef[c][e], s2);
            // chunks of minima, then of maxima: no bound is larger than the largest of these two
            if (c < kChunks / 2) least = pair_min<BT>(least, w[e]);
            else most = pair_max<BT>(most, w[e]);
          }
        }
        float y;
        f2_unpack(s2, x[u], y);
        x[u] += y;
      }
      // over the eight lanes: the upper four go on with the second page
      const bool up = l8 & 4;
      float y = up ? x[1] : x[0];
      y += __shfl_xor_sync(0xffffffffu, up ? x[0] : x[1], 4);
      y += __shfl_xor_sync(0xffffffffu, y, 2);
      y += __shfl_xor_sync(0xffffffffu, y, 1);
      // a sum that is too large, or NaN, is summed again below
      const int i = begin + 8 * k + (up ? 4 : 0) + sub;
      const bool fits = fabsf(y) < kBig;
      usable = usable && fits;
      if ((l8 & 3) == 0 && i < end) st_cluster_f32(dst + 4u * (uint32_t)i, fits ? y : kBig);
    }
    // as bits of a 16-bit magnitude, which order like it; a NaN is the largest
    least &= 0x7fff7fffu;
    most &= 0x7fff7fffu;
    top = usable ? max(max(least >> 16, least & 0xffffu), max(most >> 16, most & 0xffffu)) : 0x7fffu;
    top = __reduce_max_sync(0xffffffffu, top & 0x7fffu) | (outside ? kOutside : 0u);
    if (lane == 0) st_cluster_u32(mapa_shared(s_top + rank * kWarps + warp, 0), top);
    cluster_sync();
    if (rank != 0) return;
    top = lane < workers ? s_top[lane] : 0u;
    const uint32_t more = lane + 32 < workers ? s_top[lane + 32] : 0u;
    if (__any_sync(0xffffffffu, (top | more) & kOutside)) {
      // -inf marks an entry outside the pool
      for (int i = from + tid; i < to; i += kThreads)
        if ((unsigned)table[i] >= (unsigned)p.num_pages) s_score[i] = -INFINITY;
      __syncthreads();
    }
    top = __reduce_max_sync(0xffffffffu, max(top & 0x7fffu, more & 0x7fffu));
  }

  // ---- pages that are always kept (all of them where nothing is chosen), and candidates ----
  int counts = 0;                        // kept, and candidates times 2^16
  float lo = INFINITY, hi = -INFINITY;   // of the candidates
  for (int i = tid; i < live - (all ? 0 : to - from); i += kThreads) {
    const int at = all || i < from ? i : i + (to - from);
    const bool good = (unsigned)table[at] < (unsigned)p.num_pages;
    if (!good) record_device_error(PU_ERR_INVALID_ARGUMENT, kSiteSelectPage);
    s_score[at] = good ? INFINITY : -INFINITY;
    counts += good;
  }
  if (!all) {
    each(s_score, from, to, [&](int, float x) {
      if (x != -INFINITY) {
        counts += 1 << 16;
        lo = min(lo, x);
        hi = max(hi, x);
      }
    });
  }
  counts = __reduce_add_sync(0xffffffffu, counts);
  if (lane == 0) s.sum[warp] = counts;
  block_range(lo, hi, s, warp, lane);    // and the scores are visible to all
  counts = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) counts += s.sum[w];

  const size_t out_row = (size_t)b * p.H_kv + head;
  int want = p.count - (counts & 0xffff);            // of the candidates
  if (all || counts >> 16 <= want) {
    __syncthreads();                     // s.sum has been read
    write_list<float>(p, table, s_score, -INFINITY, 0, live, len, out_row, s);
    return;
  }
  if (want <= 0) {
    __syncthreads();
    write_list<float>(p, table, s_score, 0x1p126f, 0, live, len, out_row, s);    // none but those always kept
    return;
  }
  // what the fp32 sums are off by; 2^-140: sums of subnormals
  double sum_abs = 0.;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum_abs += s_abs[w];
  const float big = to_float(*reinterpret_cast<const BT*>(&top));
  const double e = isfinite(big) && sum_abs < 0x1p1000 ? fma(sum_abs * (double)big, 0x1p-19, 0x1p-140) : INFINITY;
  // a page in fp64, by a warp
  auto again = [&](int i) -> double {
    const uint4* src = bounds + ((size_t)table[i] * p.H_kv + head) * (2 * D / 8);
    double x = 0.;
    for (int c = lane; c < 2 * D / 8; c += 32) {
      const uint4 v = src[c];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      const double* f = &s_wide[0][0] + c * 8;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x = fma(wide<BT>(w[j] << 16), f[2 * j], x);
        x = fma(wide<BT>(w[j]), f[2 * j + 1], x);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
    // finite, also for queries that are not
    return x != x ? 0x1p1000 : fmin(fmax(x, -0x1p1000), 0x1p1000);
  };

  // ---- the border: bins, until those within 2 e of the border's are few enough to be ranked ----
  while (lo < hi) {
    const Bins<float> bins(lo, hi);
    find_bin(s_score, from, to, lo, hi, bins, want, s);
    const int at = s.found[0], reach = (int)fmin(2. * e * (double)bins.scale, 64.) + 1;
    if (reach > 32) break;
    const int first = max(0, at - reach), last = min(kBins - 1, at + reach);
    int above = s.found[1], members = s.found[2];
    for (int i = at + 1; i <= last; ++i) above -= s.bins[i];
    for (int i = first; i <= last; ++i) members += i == at ? 0 : s.bins[i];
    want -= above;
    if (members <= kRank) {
      // ---- ranked, the near ones of the border by fp64 sums ----
      each(s_score, from, to, [&](int i, float x) {
        const int c = bins.of(x);
        if (x >= lo && x <= hi && c >= first && c <= last) {
          const int k = atomicAdd(s.found + 3, 1);
          s.list[k] = i;
          s.near[k] = x;
        }
      });
      __syncthreads();
      const float x = tid < members ? s.near[tid] : 0.f;
      const int mine = tid < members ? s.list[tid] : 0;
      int before = 0;
      if (tid < members) {
        for (int j = 0; j < members; ++j) before += s.near[j] > x || (s.near[j] == x && s.list[j] < mine);
        if (before == want - 1) s.edge = x;
      }
      __syncthreads();
      const float edge = s.edge;
      const bool near = tid < members && fabs((double)x - (double)edge) <= 2. * e;
      bool in = before < want;
      if (__syncthreads_count(near) > 1) {
        const int sure = __syncthreads_count(tid < members && !near && x > edge);
        for (int k = warp; k < members; k += kWarps) {
          if (!(fabs((double)s.near[k] - (double)edge) <= 2. * e)) continue;
          const double y = again(s.list[k]);
          if (lane == 0) s.cand[k] = y;
        }
        __syncthreads();
        if (near) {
          const double y = s.cand[tid];
          int ahead = sure;
          for (int j = 0; j < members; ++j) {
            if (!(fabs((double)s.near[j] - (double)edge) <= 2. * e)) continue;
            ahead += s.cand[j] > y || (s.cand[j] == y && s.list[j] < mine);
          }
          in = ahead < want;
        } else {
          in = x > edge;
        }
      }
      if (tid < members) s_score[mine] = in ? INFINITY : -INFINITY;
      __syncthreads();
      write_list<float>(p, table, s_score, edge, 0, live, len, out_row, s);
      return;
    }
    // again between the smallest and the largest of them
    float lo2 = INFINITY, hi2 = -INFINITY;
    each(s_score, from, to, [&](int, float x) {
      const int c = bins.of(x);
      if (x >= lo && x <= hi && c >= first && c <= last) {
        lo2 = min(lo2, x);
        hi2 = max(hi2, x);
      }
    });
    block_range(lo2, hi2, s, warp, lane);
    __syncthreads();
    if (lo2 == lo && hi2 == hi) break;
    lo = lo2;
    hi = hi2;
  }

  // ---- more pages than can be ranked are as close as the fp32 sums tell (equal pages, say): those in [lo, hi]
  // and within 2 e of it in fp64, all scores as fp64 in the same place, which has room for them once the copies
  // are over ----
  const double least = (double)lo - 2. * e, most = (double)hi + 2. * e;
  double* fine = reinterpret_cast<double*>(dyn);
  for (int base = (live - 1) / kThreads * kThreads; base >= 0; base -= kThreads) {
    const int i = base + tid;
    const float x = i < live ? s_score[i] : 0.f;
    __syncthreads();
    if (i < live) fine[i] = x;
    __syncthreads();
  }
  want = p.count;                        // less those that are sure
  counts = 0;
  for (int i = tid; i < live; i += kThreads) {
    const double x = fine[i];
    if (x > most || x == INFINITY) {
      ++counts;
      fine[i] = INFINITY;
    } else if (x < least) {
      fine[i] = -INFINITY;
    }
  }
  want -= block_sum(counts, s, warp, lane);
  for (int i = from + warp; i < to; i += kWarps) {
    if (isinf(fine[i])) continue;
    const double x = again(i);
    if (lane == 0) fine[i] = x;
  }
  __syncthreads();
  double cut = 0x1p1010;
  int ties = 0;
  if (want > 0) border(fine, from, to, want, s, &cut, &ties);
  write_list<double>(p, table, fine, cut, ties, live, len, out_row, s);
}

// CTAs of a cluster: as many as leave the grid at two CTAs an SM, but no more than one for 64 pages of a full
// table row.  Each CTA pays about 3 us before its first score, and the first one as much for the choice.
inline int cluster_size(long long max_pages, long long items) {
  int c = 1;
  while (c < kMaxCtas && max_pages > 64ll * c && 2 * c * items <= 2ll * sm_count()) c *= 2;
  return c;
}

template <typename QT, typename BT, int D>
int launch_select(Params p, long long items, cudaStream_t st) {
  const auto f = select_kernel<QT, BT, D>;
  // scores, and behind them the copies (eight pages of 4 D bytes a warp and stage) or as much as lets the scores
  // be held in fp64
  constexpr int kStage = kWarps * 32 * D;
  p.ring = (p.max_pages * (int)sizeof(float) + 15) / 16 * 16;
  p.stages = kStages;
  const int ring = std::max(kStages * kStage, p.ring);
  const int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(f), 2 * kMaxPages * (int)sizeof(float) + 16, "page choice shared memory");
  if (rc) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(items * p.ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)(p.ring + ring);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return check_cuda(cudaLaunchKernelEx(&cfg, f, static_cast<const Params>(p)), "page choice launch");
}

template <typename KVT, int D>
int launch_bounds(const BoundParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)((p.T + p.chunk - 1) / p.chunk), (unsigned)((p.H_kv + p.heads - 1) / p.heads));
  return check_cuda(decode::launch_pdl(bounds_kernel<KVT, D>, grid, dim3(kBoundThreads), 0, st, p), "page bounds launch");
}

}  // namespace choose
}  // namespace pu

extern "C" int pu_page_bounds(const void* k_pool, int kv_dtype, const int32_t* slots, void* bounds, int64_t num_pages,
                              int64_t page_size, int64_t H_kv, int64_t D, int64_t num_tokens, void* stream) {
  using namespace pu::choose;
  if (!k_pool || !bounds || (num_tokens > 0 && !slots)) return pu::set_error(PU_ERR_INVALID_ARGUMENT, "page bounds: null pointer");
  if (!pu::aligned16(k_pool) || !pu::aligned16(bounds))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "page bounds: the pool and the bounds must be 16-byte aligned");
  if (kv_dtype != PU_DTYPE_F16 && kv_dtype != PU_DTYPE_BF16 && kv_dtype != PU_DTYPE_FP8_E4M3)
    return pu::set_error(PU_ERR_UNSUPPORTED, "page bounds: pools are f16, bf16 or e4m3");
  if (D != 64 && D != 128) return pu::set_error(PU_ERR_UNSUPPORTED, "page bounds: head size %lld (64 or 128)", (long long)D);
  if (H_kv <= 0 || H_kv > 65535) return pu::set_error(PU_ERR_UNSUPPORTED, "page bounds: %lld K/V heads", (long long)H_kv);
  if (num_tokens < 0 || num_tokens > 2147483647ll)
    return pu::set_error(PU_ERR_UNSUPPORTED, "page bounds: %lld tokens", (long long)num_tokens);
  int shift = 0;
  const int rc = pu::paged::check_pool(num_pages, page_size, &shift);
  if (rc || num_tokens == 0) return rc;
  BoundParams p{};
  p.k_pool = k_pool;
  p.slots = slots;
  p.bounds = bounds;
  p.H_kv = (int)H_kv;
  p.num_pages = (int)num_pages;
  p.page_shift = shift;
  p.T = num_tokens;
  // Small batches are spread out: eight single tokens and one head a CTA are a warp's row each.
  // Larger ones share the reads of the slots over as many heads as leave three CTAs an SM, which start at once (10000
  // tokens, 2 heads: 3.5 us, with one CTA more for each chunk 5.7; 14100 e4m3 tokens, 4 heads: 5.0, 8.5).  From
  // three chunks an SM on, 14208 tokens, the rest wait for a place: 14800 tokens 6.8 us, 64000 18.8.
  const long long room = 3ll * pu::sm_count();
  p.chunk = (num_tokens + 7) / 8 * H_kv <= room ? 8 : 32;
  const long long chunks = (num_tokens + p.chunk - 1) / p.chunk, parts = std::min<long long>(H_kv, std::max<long long>(1, room / chunks));
  p.heads = (int)((H_kv + parts - 1) / parts);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (kv_dtype == PU_DTYPE_FP8_E4M3)
    return D == 128 ? launch_bounds<__nv_fp8_e4m3, 128>(p, st) : launch_bounds<__nv_fp8_e4m3, 64>(p, st);
  if (kv_dtype == PU_DTYPE_F16) return D == 128 ? launch_bounds<__half, 128>(p, st) : launch_bounds<__half, 64>(p, st);
  return D == 128 ? launch_bounds<__nv_bfloat16, 128>(p, st) : launch_bounds<__nv_bfloat16, 64>(p, st);
}

extern "C" int pu_select_pages(const void* q, int q_dtype, const void* bounds, int bounds_dtype, const int32_t* page_table,
                               int64_t max_pages_per_seq, int64_t num_pages, int64_t page_size, const int32_t* kv_lens,
                               int32_t* pages, int32_t* lens, int64_t count, int64_t first, int64_t last, int64_t B,
                               int64_t H, int64_t H_kv, int64_t D, void* stream) {
  using namespace pu::choose;
  if (!q || !bounds || !kv_lens || !pages || !lens) return pu::set_error(PU_ERR_INVALID_ARGUMENT, "page choice: null pointer");
  if (!pu::aligned16(bounds)) return pu::set_error(PU_ERR_INVALID_ARGUMENT, "page choice: the bounds must be 16-byte aligned");
  if ((q_dtype != PU_DTYPE_F16 && q_dtype != PU_DTYPE_BF16) || (bounds_dtype != PU_DTYPE_F16 && bounds_dtype != PU_DTYPE_BF16))
    return pu::set_error(PU_ERR_UNSUPPORTED, "page choice: queries and bounds are f16 or bf16");
  if (D != 64 && D != 128) return pu::set_error(PU_ERR_UNSUPPORTED, "page choice: head size %lld (64 or 128)", (long long)D);
  if (B <= 0 || H <= 0 || H_kv <= 0 || H % H_kv)
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "page choice: %lld sequences, %lld heads over %lld", (long long)B, (long long)H, (long long)H_kv);
  if (first < 0 || last < 0 || count < 1 || first > count || last > count - first)
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "page choice: %lld first and %lld last of %lld pages", (long long)first, (long long)last,
                         (long long)count);
  int shift = 0;
  int rc = pu::paged::check_pages(page_table, max_pages_per_seq, num_pages, page_size, &shift);
  if (rc) return rc;
  if (max_pages_per_seq > kMaxPages)
    return pu::set_error(PU_ERR_UNSUPPORTED, "page choice: %lld pages per sequence (up to %d)", (long long)max_pages_per_seq, kMaxPages);
  if (num_pages > 2147483647ll / H_kv) return pu::set_error(PU_ERR_UNSUPPORTED, "page pool too large");
  if (count > (1ll << 30) / page_size) return pu::set_error(PU_ERR_UNSUPPORTED, "page choice: %lld pages chosen", (long long)count);
  Params p{};
  p.ctas = cluster_size(max_pages_per_seq, B * H_kv);
  if (H > 2147483647ll || B > 2147483647ll / p.ctas / H) return pu::set_error(PU_ERR_UNSUPPORTED, "page choice: batch too large");
  p.q = q;
  p.bounds = bounds;
  p.table = page_table;
  p.lens = kv_lens;
  p.pages = pages;
  p.out_lens = lens;
  p.H = (int)H;
  p.H_kv = (int)H_kv;
  p.group = (int)(H / H_kv);
  p.max_pages = (int)max_pages_per_seq;
  p.num_pages = (int)num_pages;
  p.page_shift = shift;
  p.B = (int)B;
  // Where SMs take two CTAs, and while ranking the lengths, which every CTA does, costs less than it gives: 24
  // sequences of up to 131072 tokens, 8 K/V heads of 128: 52 us with it, 63 without; 40 of them 74.5, 85; 64 of up to
  // 32768, heads of 64: 22, 25; but 64 of up to 65536, heads of 128: 74, 68; 64 of up to 4000, 4 K/V heads: 11.4, 10.3.
  // From 65 on it is left out: 65 of up to 32768: 22.7, 26; 128: 34.8, 35; of up to 4000 20, 17.5; 256: 72, 59.
  p.by_length = B > 1 && B <= 64 && B * H_kv * p.ctas > pu::sm_count();
  p.count = (int)count;
  p.first = (int)first;
  p.last = (int)last;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long items = B * H_kv;
  const bool qh = q_dtype == PU_DTYPE_F16, bh = bounds_dtype == PU_DTYPE_F16;
  if (D == 128) {
    if (bh) return qh ? launch_select<__half, __half, 128>(p, items, st) : launch_select<__nv_bfloat16, __half, 128>(p, items, st);
    return qh ? launch_select<__half, __nv_bfloat16, 128>(p, items, st) : launch_select<__nv_bfloat16, __nv_bfloat16, 128>(p, items, st);
  }
  if (bh) return qh ? launch_select<__half, __half, 64>(p, items, st) : launch_select<__nv_bfloat16, __half, 64>(p, items, st);
  return qh ? launch_select<__half, __nv_bfloat16, 64>(p, items, st) : launch_select<__nv_bfloat16, __nv_bfloat16, 64>(p, items, st);
}
