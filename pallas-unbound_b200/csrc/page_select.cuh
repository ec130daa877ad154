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

// A CTA looks at 8 or 32 rows of the packed batch for one K/V head.  The rows of a
// page stand together, in order: the first of such a run is its leader, and the
// CTA that holds the leader takes the whole run, wherever it ends, so that one
// CTA reads and writes the page's bounds.  Few leaders (prompts) share the
// eight warps out, many (a step of single tokens) take one warp each.
template <typename KVT, int D>
__global__ void __launch_bounds__(kBoundThreads) bounds_kernel(const BoundParams p) {
  constexpr bool kF8 = sizeof(KVT) == 1;
  using B = typename std::conditional<kF8, __half, KVT>::type;     // type of the bounds
  constexpr int kLanes = D * (int)sizeof(KVT) / 16;                // lanes of a row, 16 bytes each
  constexpr int kRows = 32 / kLanes;                               // rows a warp reads at once
  constexpr int kWords = kF8 ? 8 : 4;                              // pairs a lane holds
  constexpr int kAhead = 4;                                        // reads in flight
  __shared__ int s_leader[kChunk], s_count;
  __shared__ uint4 s_part[kBoundThreads / 32][2][D / 8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, head = blockIdx.y;
  const int page = 1 << p.page_shift;
  const long long places = (long long)p.num_pages << p.page_shift;
  grid_dep_wait();
  grid_dep_launch_dependents();
  const long long t0 = (long long)blockIdx.x * p.chunk;
  if (warp == 0) {
    const long long t = t0 + lane;
    const int slot = lane < p.chunk && t < p.T ? p.slots[t] : -1;
    int before = __shfl_up_sync(0xffffffffu, slot, 1);
    if (lane == 0) before = t0 > 0 ? p.slots[t0 - 1] : -1;
    if (slot >= places && head == 0) record_device_error(PU_ERR_INVALID_ARGUMENT, kSitePageBounds);
    const bool leads = slot >= 0 && slot < places && (before < 0 || before != slot - 1 || (slot & (page - 1)) == 0);
    const unsigned all = __ballot_sync(0xffffffffu, leads);
    if (leads) s_leader[__popc(all & ((1u << lane) - 1))] = lane;
    if (lane == 0) s_count = __popc(all);
  }
  __syncthreads();
  const int n = s_count;
  // warps that share a leader: 8 where there is one, 1 from eight leaders on
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
    int slot = 0;
    if (i < n) {
      const long long t = t0 + s_leader[i];
      slot = p.slots[t];
      // rows of the run: as long as the next slot is the next row of this page
      const int most = (int)min((long long)(page - (slot & (page - 1))), p.T - t);
      int rows = most;
      for (int r = 0; r < most; r += 32) {
        const bool more = r + lane < most && p.slots[t + r + lane] == slot + r + lane;
        const unsigned gap = ~__ballot_sync(0xffffffffu, more);
        if (gap) {
          rows = min(most, r + __ffs(gap) - 1);
          break;
        }
      }
      const uint4* at = reinterpret_cast<const uint4*>(p.k_pool) +
                        (((((size_t)(slot >> p.page_shift) * p.H_kv + head) << p.page_shift) + (slot & (page - 1))) * kLanes + vec);
      for (int r0 = part * kRows + sub; r0 < rows; r0 += kAhead * team * kRows) {
        uint4 x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          // past the end the first row again, which changes nothing
          const int r = r0 + u * team * kRows;
          x[u] = decode::ld_stream(at + (size_t)(r < rows ? r : r0) * kLanes);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const uint32_t w4[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
          if constexpr (kF8) {
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
              const __half2 h(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w4[w >> 1] >> (16 * (w & 1))), __NV_E4M3));
              const uint32_t v = *reinterpret_cast<const uint32_t*>(&h);
              lo[w] = pair_min<B>(lo[w], v);
              hi[w] = pair_max<B>(hi[w], v);
            }
          } else {
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
              lo[w] = pair_min<B>(lo[w], w4[w]);
              hi[w] = pair_max<B>(hi[w], w4[w]);
            }
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
      if (team > 1 && sub == 0) {
#pragma unroll
        for (int w = 0; w < kWords; w += 4) {
          s_part[warp][0][vec * (kWords / 4) + w / 4] = make_uint4(lo[w], lo[w + 1], lo[w + 2], lo[w + 3]);
          s_part[warp][1][vec * (kWords / 4) + w / 4] = make_uint4(hi[w], hi[w + 1], hi[w + 2], hi[w + 3]);
        }
      }
    }
    if (team > 1) __syncthreads();
    if (i < n && part == 0 && sub == 0) {
      uint4* out = reinterpret_cast<uint4*>(p.bounds) + ((size_t)(slot >> p.page_shift) * p.H_kv + head) * (2 * D / 8);
      const bool begun = (slot & (page - 1)) != 0;      // rows of the page were written before
#pragma unroll
      for (int w = 0; w < kWords; w += 4) {
        const int c = vec * (kWords / 4) + w / 4;
        auto fold = [&](const uint4& a, const uint4& b) {
          const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            lo[w + j] = pair_min<B>(lo[w + j], x[j]);
            hi[w + j] = pair_max<B>(hi[w + j], y[j]);
          }
        };
        for (int o = 1; o < team; ++o) fold(s_part[warp + o][0][c], s_part[warp + o][1][c]);
        if (begun) fold(out[c], out[D / 8 + c]);
        out[c] = make_uint4(lo[w], lo[w + 1], lo[w + 2], lo[w + 3]);
        out[D / 8 + c] = make_uint4(hi[w], hi[w + 1], hi[w + 2], hi[w + 3]);
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
};

// A 16-bit value as fp64 times a power of two (2^-896 for bf16, 2^-1008 for f16): its sign,
// exponent and mantissa bits moved to their places, which is exact for subnormals as well, in two
// or three integer instructions where the conversion unit takes 16 values a clock.  Infinities
// and NaN become values beyond the largest.
template <typename T>
__device__ __forceinline__ double wide(uint32_t high_half) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const int x = (int)high_half >> (kBf16 ? 3 : 6);
  return __hiloint2double(x & (kBf16 ? 0x8fffe000 : 0x81fffc00), 0);
}

template <typename T>
__device__ __forceinline__ double to_double(T x);
template <>
__device__ __forceinline__ double to_double<__half>(__half x) { return (double)__half2float(x); }
template <>
__device__ __forceinline__ double to_double<__nv_bfloat16>(__nv_bfloat16 x) { return (double)__bfloat162float(x); }

__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

// Sums over the block (every thread gets them); s: kWarps values of shared memory.
__device__ __forceinline__ int block_sum(int x, int* s, int warp, int lane) {
  x = __reduce_add_sync(0xffffffffu, x);
  if (lane == 0) s[warp] = x;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all += s[w];
  __syncthreads();
  return all;
}

// One cluster a (sequence, K/V head): its CTAs score the pages between them
// and leave the scores in the first one's shared memory, which chooses.
//
// The choice: scores lie in kBins bins of equal width between the smallest and
// the largest candidate (a monotone map, so no rounding of it can order two
// scores wrongly), bins are counted from the top until the one that holds the
// border, and its members are ranked against each other; where they are more
// than 256 the same is done again between their own smallest and largest.
template <typename QT, typename BT, int D>
__global__ void __launch_bounds__(kThreads) select_kernel(const Params p) {
  constexpr int kChunks = 2 * D / 64;    // 16-byte chunks a lane reads of a page: eight lanes a page
  extern __shared__ __align__(16) uint8_t dyn[];
  double* s_score = reinterpret_cast<double*>(dyn);                     // [max_pages], in the first CTA
  __shared__ double s_coef[2][D];        // sums of the heads' negative and positive parts
  __shared__ double s_red[2][kWarps];
  __shared__ int s_bins[kBins];
  __shared__ int s_sum[kWarps], s_tie[kWarps], s_warp[kWarps];
  __shared__ double s_cand[kRank];
  __shared__ int s_found[4];             // border bin, members above it, its members, members listed
  __shared__ double s_cut;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ctas = p.ctas, rank = (int)(blockIdx.x % (unsigned)ctas), item = (int)(blockIdx.x / (unsigned)ctas);
  const int b = item / p.H_kv, head = item % p.H_kv;
  grid_dep_wait();
  grid_dep_launch_dependents();
  const int page = 1 << p.page_shift;
  const int len = max(0, min(p.lens[b], p.max_pages << p.page_shift));
  const int live = (len + page - 1) >> p.page_shift;
  const int32_t* table = p.table + (size_t)b * p.max_pages;
  const bool all = live <= p.count;      // nothing to choose
  if (all && rank != 0) return;
  const int from = p.first, to = live - p.last;      // candidates between the pages that are always kept

  if (!all) {
    cluster_arrive();                    // every CTA runs before another writes to its shared memory
    // ---- the heads' parts ----
    for (int i = tid; i < D; i += kThreads) {
      const QT* q = static_cast<const QT*>(p.q) + ((size_t)b * p.H + (size_t)head * p.group) * D + i;
      double neg = 0., pos = 0.;
      for (int h = 0; h < p.group; ++h) {
        const double x = to_double(q[(size_t)h * D]);
        neg += fmin(x, 0.);
        pos += fmax(x, 0.);
      }
      // with the bounds as they are (wide) every product stays a normal number
      s_coef[0][i] = neg * 0x1p800;
      s_coef[1][i] = pos * 0x1p800;
    }
    __syncthreads();
    const int l8 = lane & 7, sub = lane >> 3;
    double coef[kChunks][8];             // of this lane's chunks
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = (c * 8 + l8) * 8 + e;             // element of the page's 2 D
        coef[c][e] = s_coef[at / D][at % D];
      }
    // ---- scores: a run of pages a warp, 32 table entries at a time, four pages a read ----
    const int workers = ctas * kWarps, per = ((to - from + workers - 1) / workers + 3) & ~3;
    const int begin = from + (rank * kWarps + warp) * per, end = min(to, begin + per);
    const uint4* bounds = static_cast<const uint4*>(p.bounds);
    const uint32_t dst = mapa_shared(s_score, 0);
    cluster_wait();
    for (int base = begin; base < end; base += 32) {
      const int pg = base + lane < end ? table[base + lane] : -1;
      const bool bad = base + lane < end && (unsigned)pg >= (unsigned)p.num_pages;
      if (bad) record_device_error(PU_ERR_INVALID_ARGUMENT, kSiteSelectPage);
      const int n = min(32, end - base);
      for (int j = 0; j < n; j += 8) {
        uint4 x[2][kChunks];
        bool ok[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int k = j + u * 4 + sub, entry = __shfl_sync(0xffffffffu, pg, k & 31);
          ok[u] = k < n && (unsigned)entry < (unsigned)p.num_pages;
          const uint4* at = bounds + ((size_t)(ok[u] ? entry : 0) * p.H_kv + head) * (2 * D / 8) + l8;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) x[u][c] = decode::ld_stream_if(at + c * 8, ok[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          double s0 = 0., s1 = 0.;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const uint32_t w[4] = {x[u][c].x, x[u][c].y, x[u][c].z, x[u][c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s0 = fma(wide<BT>(w[e] << 16), coef[c][2 * e], s0);
              s1 = fma(wide<BT>(w[e]), coef[c][2 * e + 1], s1);
            }
          }
          double s = s0 + s1;
#pragma unroll
          for (int off = 4; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
          // finite for what follows (queries that are not finite); -inf marks an entry outside the pool
          s = s != s ? 0x1p1000 : fmin(fmax(s, -0x1p1000), 0x1p1000);
          if (l8 == 0 && j + u * 4 + sub < n) st_cluster_f64(dst + 8u * (uint32_t)(base + j + u * 4 + sub), ok[u] ? s : -INFINITY);
        }
      }
    }
    cluster_sync();
    if (rank != 0) return;
  }

  // ---- pages that are always kept, and all of them where nothing is chosen ----
  int kept = 0;
  for (int i = tid; i < live; i += kThreads) {
    if (!all && i >= from && i < to) continue;
    const bool good = (unsigned)table[i] < (unsigned)p.num_pages;
    if (!good) record_device_error(PU_ERR_INVALID_ARGUMENT, kSiteSelectPage);
    s_score[i] = good ? INFINITY : -INFINITY;
    kept += good;
  }
  kept = block_sum(kept, s_sum, warp, lane);       // and the scores are visible to all

  // ---- the border: every score above `cut` is kept, and the first `ties` equal to it ----
  double cut = -INFINITY;
  int ties = 0;
  if (!all) {
    int want = p.count - kept;           // of the candidates
    double lo = INFINITY, hi = -INFINITY;
    int cands = 0;
    for (int i = from + tid; i < to; i += kThreads) {
      const double s = s_score[i];
      if (s == -INFINITY) continue;
      ++cands;
      lo = fmin(lo, s);
      hi = fmax(hi, s);
    }
    cands = block_sum(cands, s_sum, warp, lane);
    if (want <= 0) {
      cut = 0x1p1010;                    // none but those always kept
    } else if (cands > want) {
      while (true) {
        // smallest and largest candidate, of all threads
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
          lo = fmin(lo, __shfl_xor_sync(0xffffffffu, lo, off));
          hi = fmax(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        }
        if (lane == 0) {
          s_red[0][warp] = lo;
          s_red[1][warp] = hi;
        }
        for (int i = tid; i < kBins; i += kThreads) s_bins[i] = 0;
        if (tid < 4) s_found[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          lo = fmin(lo, s_red[0][w]);
          hi = fmax(hi, s_red[1][w]);
        }
        if (lo == hi) {                  // equal scores: the first of them
          cut = lo;
          ties = want;
          break;
        }
        const double scale = (double)(kBins - 1) / (hi - lo);
        auto bin_of = [&](double s) { return min(kBins - 1, (int)((s - lo) * scale)); };
        for (int i = from + tid; i < to; i += kThreads) {
          const double s = s_score[i];
          if (s >= lo && s <= hi) atomicAdd(s_bins + bin_of(s), 1);
        }
        __syncthreads();
        // a thread's four bins, counted from the top
        constexpr int kPer = kBins / kThreads;
        const int top = kBins - 1 - tid * kPer;
        int mine = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) mine += s_bins[top - k];
        int before = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, before, off);
          if (lane >= off) before += y;
        }
        if (lane == 31) s_warp[warp] = before;
        __syncthreads();
        for (int w = 0; w < warp; ++w) before += s_warp[w];
        before -= mine;                  // candidates in the bins above this thread's
        if (before < want && before + mine >= want) {
          int at = before;
#pragma unroll
          for (int k = 0; k < kPer; ++k) {
            const int c = s_bins[top - k];
            if (at < want && at + c >= want) {
              s_found[0] = top - k;
              s_found[1] = at;
              s_found[2] = c;
            }
            at += c;
          }
        }
        __syncthreads();
        const int border = s_found[0], members = s_found[2];
        want -= s_found[1];
        if (members <= kRank) {
          for (int i = from + tid; i < to; i += kThreads) {
            const double s = s_score[i];
            if (s >= lo && s <= hi && bin_of(s) == border) s_cand[atomicAdd(s_found + 3, 1)] = s;
          }
          __syncthreads();
          if (tid < members) {
            // the want-th largest: fewer than `want` above it, at least `want` with its equals
            const double s = s_cand[tid];
            int above = 0, same = 0;
            for (int i = 0; i < members; ++i) {
              above += s_cand[i] > s;
              same += s_cand[i] == s;
            }
            if (above < want && above + same >= want) {
              s_cut = s;
              s_found[1] = want - above; // equal threads write equal values
            }
          }
          __syncthreads();
          cut = s_cut;
          ties = s_found[1];
          break;
        }
        // again among the border's members
        double lo2 = INFINITY, hi2 = -INFINITY;
        for (int i = from + tid; i < to; i += kThreads) {
          const double s = s_score[i];
          if (s >= lo && s <= hi && bin_of(s) == border) {
            lo2 = fmin(lo2, s);
            hi2 = fmax(hi2, s);
          }
        }
        lo = lo2;
        hi = hi2;
        __syncthreads();
      }
    }
  }

  // ---- the list, in the sequence's order: a run of pages a warp, counted and then written ----
  const int run = ((live + kWarps - 1) / kWarps + 31) & ~31, begin = warp * run, end = min(live, begin + run);
  int above = 0, same = 0;
  for (int i = begin; i < end; i += 32) {
    const double s = i + lane < end ? s_score[i + lane] : -INFINITY;
    above += __popc(__ballot_sync(0xffffffffu, s > cut));
    same += __popc(__ballot_sync(0xffffffffu, s == cut && s != -INFINITY));
  }
  if (lane == 0) {
    s_sum[warp] = above;
    s_tie[warp] = same;
  }
  __syncthreads();
  int a0 = 0, t0 = 0, a1 = 0, t1 = 0;    // before this warp, and in all
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      a0 += s_sum[w];
      t0 += s_tie[w];
    }
    a1 += s_sum[w];
    t1 += s_tie[w];
  }
  const int chosen = min(p.count, a1 + min(ties, t1));
  int32_t* out = p.pages + (size_t)item * p.count;
  for (int i = begin; i < end; i += 32) {
    const double s = i + lane < end ? s_score[i + lane] : -INFINITY;
    const unsigned up = __ballot_sync(0xffffffffu, s > cut), eq = __ballot_sync(0xffffffffu, s == cut && s != -INFINITY);
    const unsigned below = (1u << lane) - 1;
    const int nth = t0 + __popc(eq & below);             // ties before this page
    const int place = a0 + __popc(up & below) + min(ties, nth);
    if ((((up >> lane) & 1u) || (((eq >> lane) & 1u) && nth < ties)) && place < p.count) out[place] = table[i + lane];
    a0 += __popc(up);
    t0 += __popc(eq);
  }
  for (int i = chosen + tid; i < p.count; i += kThreads) out[i] = -1;
  if (tid == 0) {
    // only the sequence's last page may hold fewer tokens than a page; it is last in the list
    int tokens = chosen << p.page_shift;
    if (live > 0) {
      const double s = s_score[live - 1];
      const bool in = s > cut || (s == cut && s != -INFINITY && t1 - 1 < ties);
      if (in) tokens -= (live << p.page_shift) - len;
    }
    p.out_lens[item] = tokens;
  }
}

// CTAs of a cluster: one for 64 pages of a full table row, up to the portable eight
inline int cluster_size(long long max_pages) {
  int c = 1;
  while (c < 8 && max_pages > 64ll * c) c *= 2;
  return c;
}

template <typename QT, typename BT, int D>
int launch_select(const Params& p, long long items, cudaStream_t st) {
  const auto f = select_kernel<QT, BT, D>;
  int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(f), kMaxPages * (int)sizeof(double), "page choice shared memory");
  if (rc) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(items * p.ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)p.max_pages * sizeof(double);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return check_cuda(cudaLaunchKernelEx(&cfg, f, p), "page choice launch");
}

template <typename KVT, int D>
int launch_bounds(const BoundParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)((p.T + p.chunk - 1) / p.chunk), (unsigned)p.H_kv);
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
  p.chunk = 32;
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
  if (count > (1ll << 30) / page_size) return pu::set_error(PU_ERR_UNSUPPORTED, "page choice: %lld pages chosen", (long long)count);
  Params p{};
  p.ctas = cluster_size(max_pages_per_seq);
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
