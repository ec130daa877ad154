// rope.cuh — norms of queries and keys for each head with the position
// rotation in the same pass: forward, backward, and the serving form that
// writes keys and values into their places of a paged cache.
//
// No counterpart in the reference (its attention takes q, k, v as they are,
// src/pallas_flash/ops/interface.py:20-27).  For one row x of D values (one
// head of one token), weight w, frequencies f_p of R/2 pairs:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w
//   (a, b) = pair p of n  ->  (a cos t - b sin t, b cos t + a sin t),
//   t = position f_p
// and, with h the output gradient rotated back by -t and u = x r,
//   dx = r (h w - u mean(h w u)),   dw = sum over rows of h u.
// Pair p is (p, p + R/2) or, interleaved, (2p, 2p + 1); the values behind R
// are normed and not rotated.
//
// Everything is computed in fp32 from one read of each row and rounded once.
// The angle is exact to the last fp32 bit at any position: f_p / 2 pi is
// held as a 64-bit fixed-point fraction of a turn, so position * f_p modulo
// one turn is one wrapping integer product (its error, position * 2^-54
// turns of the double product it comes from, stays under 2^-23 up to 2^31).
//
// A row is spread over D/16 lanes (a group of 4 or 8): each lane holds two
// 16-byte vectors (8 elements each, for fp32 two loads per vector) which are
// partners, 8p.. and R/2 + 8p.., so the rotation needs no exchange between
// lanes and the group reads whole 128-byte lines.  cos and sin are made once
// per token by the warp, pass through shared memory into registers, and
// serve all heads of the token that the warp takes.
// Both kernels are bound by HBM: forward 2, backward 3 passes over the rows.
#pragma once

#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace pu {
namespace rope {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 128;
constexpr int kMaxPairs = kMaxDim / 2;
constexpr int kMaxAxes = 4;

// Rows of one tensor: element (b, h, n, d) at b sB + h sH + n sN + d.
struct Rows {
  void* p;
  long long sB, sH, sN;
};

struct Angles {
  const void* freq;       // [R/2] radians per position, fp64 or fp32
  int freq64;
  const void* pos;        // int32 / int64, or nullptr: the token's index n
  int pos64;
  long long pA, pB, pN;   // strides of axis, sequence and token
  int pair_end[kMaxAxes]; // pairs [pair_end[a-1], pair_end[a]) turn with axis a
};

// One kind of head: queries (0), keys (1), values (2, append only).
struct Side {
  Rows x, y;              // forward: input, output; backward: input, its gradient
  Rows g;                 // backward: the output's gradient
  const void* w;          // [D] norm weight, or nullptr: no norm
  int w_dtype;
  int heads;
  int ctas;               // backward: CTAs that work on this kind
  float* dw_part;         // backward: [ctas][D] partial weight gradients, or nullptr
  void* dw;               // backward: [D] weight gradient in w_dtype
  float unit;             // append: the stored value is the value / unit
};

struct Params {
  Side side[3];
  Angles ang;
  long long N;            // tokens per sequence
  long long T;            // tokens in all
  int D, R;
  float eps;
  int chunk;              // forward: passes per warp
  int chunks;             // warps per token (backward: of either kind)
  // append
  const int32_t* slots;   // [T] page * page_size + row, negative: none
  int pool_dtype;
  int page_shift;
  long long num_slots;
};

// 8 elements: 16 bytes (16-bit types) or 32 (fp32).
template <typename T>
struct Vec8 {
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = decode::ld_stream(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void zero() { w = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float (&f)[8]) const { decode::unpack8<T>(w, f); }
};
template <>
struct Vec8<float> {
  uint4 w[2];
  __device__ __forceinline__ void load(const float* p) {
    w[0] = decode::ld_stream(reinterpret_cast<const uint4*>(p));
    w[1] = decode::ld_stream(reinterpret_cast<const uint4*>(p) + 1);
  }
  __device__ __forceinline__ void zero() { w[0] = w[1] = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i] = __uint_as_float(w[i].x);
      f[4 * i + 1] = __uint_as_float(w[i].y);
      f[4 * i + 2] = __uint_as_float(w[i].z);
      f[4 * i + 3] = __uint_as_float(w[i].w);
    }
  }
};

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  uint4 w;
  if constexpr (std::is_same<T, __half>::value)
    w = make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7]));
  else
    w = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  *reinterpret_cast<uint4*>(p) = w;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// 8 values into a pool row of pool_dtype (saturating e4m3, or 16-bit).
__device__ __forceinline__ void store8_pool(void* pool, size_t at, int dtype, const float (&f)[8]) {
  if (dtype == PU_DTYPE_BF16) {
    store8(static_cast<__nv_bfloat16*>(pool) + at, f);
  } else if (dtype == PU_DTYPE_F16) {
    store8(static_cast<__half*>(pool) + at, f);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | (hi << 16);
    }
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + at) = make_uint2(w[0], w[1]);
  }
}

__device__ __forceinline__ float load_weight(const void* w, int dtype, int i) {
  if (dtype == PU_DTYPE_F32) return static_cast<const float*>(w)[i];
  if (dtype == PU_DTYPE_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// cos and sin of every pair of one token into the warp's shared row.
__device__ __forceinline__ void make_angles(const Angles& a, int pairs, long long b, long long n, int lane, float2* out) {
  for (int p = lane; p < pairs; p += 32) {
    const double f = a.freq64 ? static_cast<const double*>(a.freq)[p] : (double)static_cast<const float*>(a.freq)[p];
    double turns = f * 0.15915494309189533577;               // per position: 1 / 2 pi
    turns -= floor(turns);
    const unsigned long long step = (unsigned long long)(turns * 18446744073709551616.0);   // * 2^64, below it
    long long pos = n;
    if (a.pos != nullptr) {
      int axis = 0;
#pragma unroll
      for (int i = 0; i + 1 < kMaxAxes; ++i) axis += p >= a.pair_end[i];
      const long long at = axis * a.pA + b * a.pB + n * a.pN;
      pos = a.pos64 ? static_cast<const long long*>(a.pos)[at] : (long long)static_cast<const int32_t*>(a.pos)[at];
    }
    const int turn = (int)((step * (unsigned long long)pos) >> 32);     // signed: half turns of 2^31
    float s, c;
    sincospif((float)turn * 4.6566128730773926e-10f, &s, &c);           // 2^-31
    out[p] = make_float2(c, s);
  }
}

// What a lane of a row group holds: its two vectors' places in the row.
struct Place {
  int o0, o1;
  bool in, rot;
};

template <bool kInter>
__device__ __forceinline__ Place make_place(int sub, int D, int R) {
  Place pl;
  pl.in = sub * 16 < D;
  pl.rot = sub * 16 < R;
  pl.o0 = kInter || !pl.rot ? sub * 16 : sub * 8;
  pl.o1 = kInter || !pl.rot ? sub * 16 + 8 : R / 2 + sub * 8;
  return pl;
}

// Rotates the lane's 8 pairs by (c, s); with s negated, back.
template <bool kInter>
__device__ __forceinline__ void rotate(float (&a)[8], float (&b)[8], const float (&c)[8], const float (&s)[8]) {
  if constexpr (kInter) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x0 = a[2 * i], x1 = a[2 * i + 1], y0 = b[2 * i], y1 = b[2 * i + 1];
      a[2 * i] = fmaf(x0, c[i], -x1 * s[i]);
      a[2 * i + 1] = fmaf(x1, c[i], x0 * s[i]);
      b[2 * i] = fmaf(y0, c[4 + i], -y1 * s[4 + i]);
      b[2 * i + 1] = fmaf(y1, c[4 + i], y0 * s[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = fmaf(x, c[i], -y * s[i]);
      b[i] = fmaf(y, c[i], x * s[i]);
    }
  }
}

template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// The lane's cos and sin (pairs 8 sub ..) from the warp's shared row.
__device__ __forceinline__ void take_angles(const float2* row, const Place& pl, int sub, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = pl.rot ? row[sub * 8 + i] : make_float2(1.f, 0.f);
    c[i] = v.x;
    s[i] = v.y;
  }
}

__device__ __forceinline__ void take_weight(const Side& sd, const Place& pl, float (&wa)[8], float (&wb)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool use = sd.w != nullptr && pl.in;
    wa[i] = use ? load_weight(sd.w, sd.w_dtype, pl.o0 + i) : 1.f;
    wb[i] = use ? load_weight(sd.w, sd.w_dtype, pl.o1 + i) : 1.f;
  }
}

// A pass is 32 / kLanes rows (heads) of one token; queries' passes come
// first, then keys', then values'.  Each warp takes `chunk` consecutive passes
// of one token, kBatch of them loaded before the first is used.
template <typename T, int kLanes, bool kInter, bool kAppend>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const __grid_constant__ Params p) {
  constexpr int kRows = 32 / kLanes;
  constexpr int kBatch = sizeof(T) == 4 ? 2 : 4;
  __shared__ float2 s_ang[kWarps][kMaxPairs];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % kLanes, row = lane / kLanes;
  const long long unit = (long long)blockIdx.x * kWarps + warp;
  const long long t = unit / p.chunks;
  grid_dep_wait();
  grid_dep_launch_dependents();
  if (t >= p.T) return;
  const long long b = t / p.N, n = t - b * p.N;
  const Place pl = make_place<kInter>(sub, p.D, p.R);
  make_angles(p.ang, p.R / 2, b, n, lane, s_ang[warp]);
  __syncwarp();
  float c[8], s[8];
  take_angles(s_ang[warp], pl, sub, c, s);

  size_t pool_row = 0;      // append: page and row of this token
  bool put = true;
  if constexpr (kAppend) {
    const long long slot = p.slots[t];
    put = slot >= 0 && slot < p.num_slots;
    if (slot >= p.num_slots && lane == 0) record_device_error(PU_ERR_INVALID_ARGUMENT, kSiteAppendSlot);
    pool_row = put ? (size_t)slot : 0;
  }
  const int first = (int)(unit - t * p.chunks) * p.chunk, last = first + p.chunk;
  int begin = 0;
#pragma unroll
  for (int kind = 0; kind < (kAppend ? 3 : 2); ++kind) {
    const Side& sd = p.side[kind];
    const int end = begin + (sd.heads + kRows - 1) / kRows;
    const int lo = max(first, begin), hi = min(last, end);
    if (lo < hi) {
      const T* x0 = static_cast<const T*>(sd.x.p) + b * sd.x.sB + n * sd.x.sN;
      float wa[8], wb[8];
      if (kind < 2) take_weight(sd, pl, wa, wb);
      for (int pass = lo; pass < hi; pass += kBatch) {
        Vec8<T> va[kBatch], vb[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int h = (pass + u - begin) * kRows + row;
          va[u].zero();
          vb[u].zero();
          if (pass + u < hi && h < sd.heads && pl.in) {
            const T* x = x0 + h * sd.x.sH;
            va[u].load(x + pl.o0);
            vb[u].load(x + pl.o1);
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int h = (pass + u - begin) * kRows + row;
          if (pass + u >= hi) break;
          float a[8], bb[8];
          va[u].get(a);
          vb[u].get(bb);
          if (kind < 2) {
            if (sd.w != nullptr) {
              float ss = 0.f;
#pragma unroll
              for (int i = 0; i < 8; ++i) ss = fmaf(a[i], a[i], fmaf(bb[i], bb[i], ss));
              const float r = rsqrtf(group_sum<kLanes>(ss) / (float)p.D + p.eps);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                a[i] *= r * wa[i];
                bb[i] *= r * wb[i];
              }
            }
            if (pl.rot) rotate<kInter>(a, bb, c, s);
          }
          if (h >= sd.heads || !pl.in) continue;
          if (kAppend && kind > 0) {
            if (!put) continue;
            if (sd.unit != 1.f) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                a[i] = a[i] / sd.unit;
                bb[i] = bb[i] / sd.unit;
              }
            }
            const size_t mask = ((size_t)1 << p.page_shift) - 1;
            const size_t at = ((((pool_row >> p.page_shift) * sd.heads + h) << p.page_shift) + (pool_row & mask)) * p.D;
            store8_pool(sd.y.p, at + pl.o0, p.pool_dtype, a);
            store8_pool(sd.y.p, at + pl.o1, p.pool_dtype, bb);
          } else {
            T* y = static_cast<T*>(sd.y.p) + b * sd.y.sB + h * sd.y.sH + n * sd.y.sN;
            store8(y + pl.o0, a);
            store8(y + pl.o1, bb);
          }
        }
      }
    }
    begin = end;
  }
}

// CTAs [0, side[0].ctas) take the queries, the rest the keys; a warp walks
// units (token, chunk of passes) of its kind and keeps the weight gradient of
// its rows in registers; each CTA writes one partial row, summed in a fixed
// order by dw_kernel (no atomics: the same bits every time).
template <typename T, int kLanes, bool kInter>
__global__ void __launch_bounds__(kThreads) bwd_kernel(const __grid_constant__ Params p) {
  constexpr int kRows = 32 / kLanes;
  constexpr int kBatch = sizeof(T) == 4 ? 1 : 2;
  __shared__ float2 s_ang[kWarps][kMaxPairs];
  __shared__ float s_dw[kWarps][kMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % kLanes, row = lane / kLanes;
  const int kind = (int)blockIdx.x < p.side[0].ctas ? 0 : 1;
  const int cta = (int)blockIdx.x - (kind ? p.side[0].ctas : 0);
  const Side& sd = p.side[kind];
  const Place pl = make_place<kInter>(sub, p.D, p.R);
  grid_dep_wait();
  grid_dep_launch_dependents();
  const bool norm = sd.w != nullptr;
  float wa[8], wb[8], da[8], db[8];
  take_weight(sd, pl, wa, wb);
#pragma unroll
  for (int i = 0; i < 8; ++i) da[i] = db[i] = 0.f;
  const int passes = (sd.heads + kRows - 1) / kRows;
  const int chunk = (passes + p.chunks - 1) / p.chunks;
  const float inv_d = 1.f / (float)p.D;
  const long long units = p.T * p.chunks, stride = (long long)sd.ctas * kWarps;
  for (long long unit = (long long)cta * kWarps + warp; unit < units; unit += stride) {
    const long long t = unit / p.chunks;
    const long long b = t / p.N, n = t - b * p.N;
    const int lo = (int)(unit - t * p.chunks) * chunk, hi = min(lo + chunk, passes);
    __syncwarp();
    make_angles(p.ang, p.R / 2, b, n, lane, s_ang[warp]);
    __syncwarp();
    float c[8], s[8];
    take_angles(s_ang[warp], pl, sub, c, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = -s[i];
    const T* x0 = static_cast<const T*>(sd.x.p) + b * sd.x.sB + n * sd.x.sN;
    const T* g0 = static_cast<const T*>(sd.g.p) + b * sd.g.sB + n * sd.g.sN;
    T* y0 = static_cast<T*>(sd.y.p) + b * sd.y.sB + n * sd.y.sN;
    for (int pass = lo; pass < hi; pass += kBatch) {
      Vec8<T> xa[kBatch], xb[kBatch], ga[kBatch], gb[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int h = (pass + u) * kRows + row;
        xa[u].zero();
        xb[u].zero();
        ga[u].zero();
        gb[u].zero();
        if (pass + u < hi && h < sd.heads && pl.in) {
          const T* g = g0 + h * sd.g.sH;
          ga[u].load(g + pl.o0);
          gb[u].load(g + pl.o1);
          if (norm) {
            const T* x = x0 + h * sd.x.sH;
            xa[u].load(x + pl.o0);
            xb[u].load(x + pl.o1);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int h = (pass + u) * kRows + row;
        if (pass + u >= hi) break;
        float ha[8], hb[8];
        ga[u].get(ha);
        gb[u].get(hb);
        if (pl.rot) rotate<kInter>(ha, hb, c, s);
        if (norm) {
          float x[8], y[8];
          xa[u].get(x);
          xb[u].get(y);
          float ss = 0.f, dot = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
            dot = fmaf(ha[i] * wa[i], x[i], fmaf(hb[i] * wb[i], y[i], dot));
          }
          ss = group_sum<kLanes>(ss);
          dot = group_sum<kLanes>(dot);
          const float r = rsqrtf(ss * inv_d + p.eps);
          const float k = dot * inv_d * r * r * r;        // dx = r (h w) - x k
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            da[i] = fmaf(ha[i] * r, x[i], da[i]);
            db[i] = fmaf(hb[i] * r, y[i], db[i]);
            ha[i] = fmaf(ha[i] * wa[i], r, -x[i] * k);
            hb[i] = fmaf(hb[i] * wb[i], r, -y[i] * k);
          }
        }
        if (h >= sd.heads || !pl.in) continue;
        T* y = y0 + h * sd.y.sH;
        store8(y + pl.o0, ha);
        store8(y + pl.o1, hb);
      }
    }
  }
  if (sd.dw_part == nullptr) return;
  // rows of the warp, then the warps
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int off = kLanes; off < 32; off <<= 1) {
      da[i] += __shfl_xor_sync(0xffffffffu, da[i], off);
      db[i] += __shfl_xor_sync(0xffffffffu, db[i], off);
    }
  }
  if (row == 0 && pl.in) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s_dw[warp][pl.o0 + i] = da[i];
      s_dw[warp][pl.o1 + i] = db[i];
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < p.D) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += s_dw[w][threadIdx.x];
    sd.dw_part[(size_t)cta * p.D + threadIdx.x] = v;
  }
}

// Weight gradient of kind blockIdx.x: column d's partials, summed by
// kDwParts threads each and then in thread order.
constexpr int kDwParts = 8;
__global__ void __launch_bounds__(kMaxDim * kDwParts) dw_kernel(const __grid_constant__ Params p) {
  __shared__ float s[kDwParts][kMaxDim];
  const Side& sd = p.side[blockIdx.x];
  const int d = threadIdx.x % kMaxDim, part = threadIdx.x / kMaxDim;
  grid_dep_wait();
  grid_dep_launch_dependents();
  if (sd.dw == nullptr) return;
  float v = 0.f;
  if (d < p.D) {
#pragma unroll 8
    for (int c = part; c < sd.ctas; c += kDwParts) v += __ldcg(sd.dw_part + (size_t)c * p.D + d);
  }
  s[part][d] = v;
  __syncthreads();
  if (part == 0 && d < p.D) {
#pragma unroll
    for (int i = 1; i < kDwParts; ++i) v += s[i][d];
    if (sd.w_dtype == PU_DTYPE_F32) static_cast<float*>(sd.dw)[d] = v;
    else if (sd.w_dtype == PU_DTYPE_F16) static_cast<__half*>(sd.dw)[d] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(sd.dw)[d] = __float2bfloat16_rn(v);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr int kCtasPerSm = 2;        // resident CTAs the backward's grid asks for

inline bool type_ok(int64_t t) { return t == PU_DTYPE_BF16 || t == PU_DTYPE_F16 || t == PU_DTYPE_F32; }

// Every row a kernel reads or writes in 16-byte vectors starts on a 16-byte
// boundary: the base, and each stride of a dimension longer than one.
inline bool rows_aligned(const void* p, const int64_t* st, int64_t B, int64_t H, int64_t N, int64_t unit) {
  return aligned16(p) && (B <= 1 || st[0] % unit == 0) && (H <= 1 || st[1] % unit == 0) && (N <= 1 || st[2] % unit == 0);
}

// Checks what all three entry points share and fills the angles.
inline int check(const pu_qk_rope_desc* d, const char* who, Params* p) {
  if (!d) return set_error(PU_ERR_INVALID_ARGUMENT, "%s: null description", who);
  if (d->B <= 0 || d->N <= 0 || d->H <= 0 || d->H_kv <= 0)
    return set_error(PU_ERR_INVALID_ARGUMENT, "%s: B, N, H and H_kv must be positive", who);
  if (d->N > (1ll << 31) || d->B > (1ll << 31) / d->N || d->H > 65536 || d->H_kv > 65536)
    return set_error(PU_ERR_UNSUPPORTED, "%s: more than 2^31 tokens or 65536 heads", who);
  if (d->D < 16 || d->D > kMaxDim || d->D % 16)
    return set_error(PU_ERR_UNSUPPORTED, "%s: head size %lld (a multiple of 16 up to %d)", who, (long long)d->D, kMaxDim);
  if (d->rotary_dim < 16 || d->rotary_dim > d->D || d->rotary_dim % 16)
    return set_error(PU_ERR_UNSUPPORTED, "%s: rotary size %lld (a multiple of 16 up to the head size)", who,
                     (long long)d->rotary_dim);
  if (!type_ok(d->dtype)) return set_error(PU_ERR_UNSUPPORTED, "%s: dtype must be bf16, f16 or f32", who);
  if (!d->inv_freq) return set_error(PU_ERR_INVALID_ARGUMENT, "%s: null frequencies", who);
  if ((d->q_weight && !type_ok(d->q_weight_dtype)) || (d->k_weight && !type_ok(d->k_weight_dtype)))
    return set_error(PU_ERR_UNSUPPORTED, "%s: norm weights must be bf16, f16 or f32", who);
  if (!(d->eps >= 0.0) || !(d->eps < 1e30)) return set_error(PU_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", who);
  if (d->axes < 1 || d->axes > kMaxAxes) return set_error(PU_ERR_UNSUPPORTED, "%s: %lld position axes (1 to %d)", who, (long long)d->axes, kMaxAxes);
  if (d->axes > 1 && !d->positions) return set_error(PU_ERR_INVALID_ARGUMENT, "%s: several axes need positions", who);
  int64_t sum = 0;
  for (int a = 0; a < kMaxAxes; ++a) {
    const int64_t n = a < d->axes ? d->sections[a] : 0;
    if (n < 0 || n > d->rotary_dim / 2) return set_error(PU_ERR_INVALID_ARGUMENT, "%s: bad section size", who);
    sum += n;
    p->ang.pair_end[a] = (int)sum;
  }
  if (sum != d->rotary_dim / 2)
    return set_error(PU_ERR_INVALID_ARGUMENT, "%s: the sections hold %lld pairs, the rotation %lld", who, (long long)sum,
                     (long long)(d->rotary_dim / 2));
  p->ang.freq = d->inv_freq;
  p->ang.freq64 = d->freq_is_f64 != 0;
  p->ang.pos = d->positions;
  p->ang.pos64 = d->pos_is_i64 != 0;
  p->ang.pA = d->pos_stride[0];
  p->ang.pB = d->pos_stride[1];
  p->ang.pN = d->pos_stride[2];
  p->N = d->N;
  p->T = d->B * d->N;
  p->D = (int)d->D;
  p->R = (int)d->rotary_dim;
  p->eps = (float)d->eps;
  p->side[0].heads = (int)d->H;
  p->side[1].heads = p->side[2].heads = (int)d->H_kv;
  p->side[0].w = d->q_weight;
  p->side[0].w_dtype = (int)d->q_weight_dtype;
  p->side[1].w = d->k_weight;
  p->side[1].w_dtype = (int)d->k_weight_dtype;
  return PU_OK;
}

inline Rows rows_of(const void* p, const int64_t* st) { return Rows{const_cast<void*>(p), st[0], st[1], st[2]}; }

// Lanes of a row, rows of a pass.
inline int lanes_of(int D) { return D <= 64 ? 4 : 8; }
inline int passes_of(int heads, int D) { return (heads + 32 / lanes_of(D) - 1) / (32 / lanes_of(D)); }

template <typename T, bool kAppend>
int launch_fwd(Params& p, bool inter, cudaStream_t st) {
  int passes = 0;
  for (int k = 0; k < (kAppend ? 3 : 2); ++k) passes += passes_of(p.side[k].heads, p.D);
  // A warp takes all passes of its token, so that the angles are made once,
  // unless that leaves SMs without work (32 warps on each are wanted).
  const long long want = (long long)sm_count() * 32;
  p.chunk = (int)std::max<long long>(1, std::min<long long>(passes, p.T * passes / want));
  p.chunks = (passes + p.chunk - 1) / p.chunk;
  const long long grid = (p.T * p.chunks + kWarps - 1) / kWarps;
  if (grid > 2147483647ll) return set_error(PU_ERR_UNSUPPORTED, "too many rows for one launch");
  const bool wide = lanes_of(p.D) == 8;
  auto* k = wide ? (inter ? fwd_kernel<T, 8, true, kAppend> : fwd_kernel<T, 8, false, kAppend>)
                 : (inter ? fwd_kernel<T, 4, true, kAppend> : fwd_kernel<T, 4, false, kAppend>);
  return check_cuda(decode::launch_pdl(k, dim3((unsigned)grid), dim3(kThreads), 0, st, p), "norm and rotation launch");
}

template <bool kAppend>
int launch_fwd(Params& p, int64_t dtype, bool inter, cudaStream_t st) {
  if (dtype == PU_DTYPE_F32) return launch_fwd<float, kAppend>(p, inter, st);
  return dtype == PU_DTYPE_F16 ? launch_fwd<__half, kAppend>(p, inter, st) : launch_fwd<__nv_bfloat16, kAppend>(p, inter, st);
}

template <typename T>
int launch_bwd(const Params& p, bool inter, int grid, cudaStream_t st) {
  const bool wide = lanes_of(p.D) == 8;
  auto* k = wide ? (inter ? bwd_kernel<T, 8, true> : bwd_kernel<T, 8, false>)
                 : (inter ? bwd_kernel<T, 4, true> : bwd_kernel<T, 4, false>);
  return check_cuda(decode::launch_pdl(k, dim3((unsigned)grid), dim3(kThreads), 0, st, p), "norm and rotation backward launch");
}

inline long long bwd_ctas() { return (long long)sm_count() * kCtasPerSm; }

}  // namespace rope
}  // namespace pu

extern "C" {

int pu_qk_norm_rope_fwd(const pu_qk_rope_desc* d, const void* q, const void* k, void* q_out, void* k_out, void* stream) {
  using namespace pu::rope;
  Params p{};
  const int rc = check(d, "pu_qk_norm_rope_fwd", &p);
  if (rc) return rc;
  if (!q || !k || !q_out || !k_out) return pu::set_error(PU_ERR_INVALID_ARGUMENT, "null q/k pointer");
  const int64_t unit = d->dtype == PU_DTYPE_F32 ? 4 : 8;
  if (!rows_aligned(q, d->q_stride, d->B, d->H, d->N, unit) || !rows_aligned(k, d->k_stride, d->B, d->H_kv, d->N, unit) ||
      !pu::aligned16(q_out) || !pu::aligned16(k_out))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "rows of q, k and the outputs must start on 16-byte boundaries");
  p.side[0].x = rows_of(q, d->q_stride);
  p.side[1].x = rows_of(k, d->k_stride);
  p.side[0].y = Rows{q_out, d->H * d->N * d->D, d->N * d->D, d->D};
  p.side[1].y = Rows{k_out, d->H_kv * d->N * d->D, d->N * d->D, d->D};
  return launch_fwd<false>(p, d->dtype, d->interleaved != 0, static_cast<cudaStream_t>(stream));
}

int pu_qk_norm_rope_append(const pu_qk_rope_desc* d, const void* q, const void* k, const void* v, void* q_out,
                           const int32_t* slots, void* k_pool, void* v_pool, int pool_dtype, int64_t num_pages,
                           int64_t page_size, float k_scale, float v_scale, void* stream) {
  using namespace pu::rope;
  Params p{};
  int rc = check(d, "pu_qk_norm_rope_append", &p);
  if (rc) return rc;
  if (!q || !k || !v || !q_out || !slots || !k_pool || !v_pool)
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "null q/k/v, slots or pool pointer");
  if (d->B != 1) return pu::set_error(PU_ERR_INVALID_ARGUMENT, "appended tokens are packed: B must be 1");
  if (pool_dtype != PU_DTYPE_BF16 && pool_dtype != PU_DTYPE_F16 && pool_dtype != PU_DTYPE_FP8_E4M3)
    return pu::set_error(PU_ERR_UNSUPPORTED, "pool dtype must be bf16, f16 or e4m3");
  if (!(k_scale > 0.f) || !(v_scale > 0.f) || !std::isfinite(k_scale) || !std::isfinite(v_scale))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "k_scale and v_scale must be positive and finite");
  int shift = 0;
  rc = pu::paged::check_pool(num_pages, page_size, &shift);
  if (rc) return rc;
  const int64_t unit = d->dtype == PU_DTYPE_F32 ? 4 : 8;
  if (!rows_aligned(q, d->q_stride, 1, d->H, d->N, unit) || !rows_aligned(k, d->k_stride, 1, d->H_kv, d->N, unit) ||
      !rows_aligned(v, d->v_stride, 1, d->H_kv, d->N, unit) || !pu::aligned16(q_out) || !pu::aligned16(k_pool) ||
      !pu::aligned16(v_pool))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "rows of q, k, v and the pools must start on 16-byte boundaries");
  p.side[0].x = rows_of(q, d->q_stride);
  p.side[1].x = rows_of(k, d->k_stride);
  p.side[2].x = rows_of(v, d->v_stride);
  p.side[0].y = Rows{q_out, 0, d->D, d->H * d->D};       // [T, H, D]
  p.side[1].y = Rows{k_pool, 0, 0, 0};
  p.side[2].y = Rows{v_pool, 0, 0, 0};
  p.side[1].unit = k_scale;
  p.side[2].unit = v_scale;
  p.slots = slots;
  p.pool_dtype = pool_dtype;
  p.page_shift = shift;
  p.num_slots = num_pages * page_size;
  return launch_fwd<true>(p, d->dtype, d->interleaved != 0, static_cast<cudaStream_t>(stream));
}

size_t pu_qk_norm_rope_bwd_workspace_size(int64_t D) {
  if (D <= 0 || D > pu::rope::kMaxDim) return 0;
  return (size_t)pu::rope::bwd_ctas() * D * sizeof(float);
}

int pu_qk_norm_rope_bwd(const pu_qk_rope_desc* d, const void* q, const void* k, const void* gq, const void* gk, void* dq,
                        void* dk, void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pu::rope;
  Params p{};
  int rc = check(d, "pu_qk_norm_rope_bwd", &p);
  if (rc) return rc;
  if ((!dq && !dk) || (dq && (!q || !gq)) || (dk && (!k || !gk)))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "null q/k, gradient or output pointer");
  if ((dq_weight && (!dq || !d->q_weight)) || (dk_weight && (!dk || !d->k_weight)))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "a weight gradient needs its weight and its row gradient");
  const int64_t unit = d->dtype == PU_DTYPE_F32 ? 4 : 8;
  if ((dq && (!rows_aligned(q, d->q_stride, d->B, d->H, d->N, unit) || !rows_aligned(gq, d->gq_stride, d->B, d->H, d->N, unit) ||
              !rows_aligned(dq, d->dq_stride, d->B, d->H, d->N, unit))) ||
      (dk && (!rows_aligned(k, d->k_stride, d->B, d->H_kv, d->N, unit) ||
              !rows_aligned(gk, d->gk_stride, d->B, d->H_kv, d->N, unit) ||
              !rows_aligned(dk, d->dk_stride, d->B, d->H_kv, d->N, unit))))
    return pu::set_error(PU_ERR_INVALID_ARGUMENT, "rows of q, k and their gradients must start on 16-byte boundaries");
  const size_t need = pu_qk_norm_rope_bwd_workspace_size(d->D);
  if ((dq_weight || dk_weight) && (!workspace || workspace_bytes < need || !pu::aligned16(workspace)))
    return pu::set_error(PU_ERR_WORKSPACE, "norm and rotation backward needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  // warps for the rows of either kind in proportion, each with whole tokens
  // unless there are fewer tokens than warps
  const int pq = dq ? passes_of(p.side[0].heads, p.D) : 0, pk = dk ? passes_of(p.side[1].heads, p.D) : 0;
  const long long most = bwd_ctas();
  p.chunks = (int)std::max<long long>(1, std::min<long long>(std::max(pq, pk), most * kWarps / p.T));
  const long long per_kind = (p.T * p.chunks + kWarps - 1) / kWarps;
  long long nq = pq ? std::max<long long>(1, most * pq / (pq + pk)) : 0;
  nq = std::min(nq, pk ? most - 1 : most);
  long long nk = pk ? most - nq : 0;
  nq = std::min(nq, per_kind);
  nk = std::min(nk, per_kind);
  p.side[0].ctas = (int)nq;
  p.side[1].ctas = (int)nk;
  p.side[0].x = rows_of(q, d->q_stride);
  p.side[1].x = rows_of(k, d->k_stride);
  p.side[0].g = rows_of(gq, d->gq_stride);
  p.side[1].g = rows_of(gk, d->gk_stride);
  p.side[0].y = rows_of(dq, d->dq_stride);
  p.side[1].y = rows_of(dk, d->dk_stride);
  float* part = static_cast<float*>(workspace);
  p.side[0].dw_part = dq_weight ? part : nullptr;
  p.side[1].dw_part = dk_weight ? part + (size_t)nq * d->D : nullptr;
  p.side[0].dw = dq_weight;
  p.side[1].dw = dk_weight;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool inter = d->interleaved != 0;
  const int grid = (int)(nq + nk);
  rc = d->dtype == PU_DTYPE_F32 ? launch_bwd<float>(p, inter, grid, st)
       : d->dtype == PU_DTYPE_F16 ? launch_bwd<__half>(p, inter, grid, st)
                                  : launch_bwd<__nv_bfloat16>(p, inter, grid, st);
  if (rc || (!dq_weight && !dk_weight)) return rc;
  return pu::check_cuda(pu::decode::launch_pdl(dw_kernel, dim3(2), dim3(kMaxDim * kDwParts), 0, st, p),
                        "norm weight gradient launch");
}

}  // extern "C"
