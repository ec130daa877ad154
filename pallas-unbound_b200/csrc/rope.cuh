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
// f_p / 2 pi is held as a 64-bit fixed-point fraction of a turn, rounded from twice a
// double's precision, so position * f_p modulo one turn is one wrapping integer
// product, off by |position| 2^-64 of a turn (2^-33 at any int32 position).
//
// A row is spread over D/16 lanes (a group of 4 or 8): each lane holds two
// vectors of 8 elements which are partners, 8p.. and R/2 + 8p.., so the rotation
// needs no exchange between lanes and the group reads whole 128-byte lines.
// cos and sin are made once per token by the warp, pass through shared memory
// and serve all heads of the token that the warp takes.  Arithmetic is on
// packed fp32 pairs; rows reach the warps through a ring in shared memory, asked
// for two to three passes ahead over the borders of heads and tokens, and the
// next token's positions before the angles of this one.
//
// Both directions read and write each row once: forward 2, backward 3 passes
// over the rows.  Measured (calls back to back; copy rate 6.4 TB/s): 4 x 4096
// tokens, 32 + 8 heads of 128, bf16: forward 336 MB in 58 us (5.8 TB/s, 91 %),
// backward 503 MB in 109 us (4.6 TB/s, 72 %: neither issue slots, 56 %, nor DRAM
// full, but the chains of a pass and its lane sums at 16 warps an SM); with
// neighbouring pairs 83 to 87 and 176 (the exchange inside each packed pair); fp32
// 671 MB in 165 us (4.1 TB/s) and 1.0 GB in 265 (3.8 TB/s: ring and sums leave one CTA
// an SM, and the grid's other half runs behind the first).  128 registers and 16
// warps an SM measured best in bf16: 24 warps forward 65 us, 20 warps 64.  17 packed
// prompts of 15 thousand tokens into a cache, 184 MB, 44 us, into e4m3 pages 52 (a
// division for each element).  64 tokens appended 5.2 us.
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
constexpr int kCtasPerSm = 2;        // resident CTAs the grids ask for

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
  float* dw_part;         // backward: [CTAs][D] partial weight gradients, or nullptr
  void* dw;               // backward: [D] weight gradient in w_dtype
  float unit;             // append: the stored value is the value / unit
};

struct Params {
  Side side[3];
  Angles ang;
  long long N;            // tokens per sequence
  long long T;            // tokens in all
  int D, R;
  float eps, inv_d;
  unsigned whole;         // units below: a token each; the other tokens are cut into parts
  unsigned units;
  unsigned step_b, step_n;   // sequences and tokens from a warp's unit to its next
  int passes;             // of a token
  int chunk;              // passes of a part
  int chunks;             // parts of a token
  int ctas;               // backward: CTAs, each with a partial weight gradient
  // append
  const int32_t* slots;   // [T] page * page_size + row, negative: none
  int pool_dtype;
  int page_shift;
  long long num_slots;
};

// 8 elements: 16 bytes (16-bit types) or 32 (fp32), as four packed fp32 pairs.
template <typename T>
struct Vec8 {
  uint4 w;
  __device__ __forceinline__ void set(int, uint4 x) { w = x; }
  __device__ __forceinline__ void get(uint64_t (&f)[4]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        f[i] = f2_pack(x.x, x.y);
      } else {
        f[i] = f2_pack(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
      }
    }
  }
};
template <>
struct Vec8<float> {
  uint4 w[2];
  __device__ __forceinline__ void set(int c, uint4 x) { w[c] = x; }
  __device__ __forceinline__ void get(uint64_t (&f)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[2 * i] = f2_pack(__uint_as_float(w[i].x), __uint_as_float(w[i].y));
      f[2 * i + 1] = f2_pack(__uint_as_float(w[i].z), __uint_as_float(w[i].w));
    }
  }
};

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const uint64_t (&f)[4]) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_unpack(f[i], x[2 * i], x[2 * i + 1]);
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else if constexpr (std::is_same<T, __half>::value) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(x[4], x[5]),
                                              pack_f16x2(x[6], x[7]));
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                              pack_bf16x2(x[6], x[7]));
  }
}

// 8 values / unit into a pool row of pool_dtype (saturating e4m3, or 16-bit).
__device__ __forceinline__ void store8_pool(void* pool, size_t at, int dtype, float unit, uint64_t (&f)[4]) {
  if (unit != 1.f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      f2_unpack(f[i], a, b);
      f[i] = f2_pack(a / unit, b / unit);
    }
  }
  if (dtype == PU_DTYPE_BF16) {
    store8(static_cast<__nv_bfloat16*>(pool) + at, f);
  } else if (dtype == PU_DTYPE_F16) {
    store8(static_cast<__half*>(pool) + at, f);
  } else {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 x;
      f2_unpack(f[i], x.x, x.y);
      h[i] = __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
    }
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + at) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
  }
}

__device__ __forceinline__ float load_weight(const void* w, int dtype, int i) {
  if (dtype == PU_DTYPE_F32) return static_cast<const float*>(w)[i];
  if (dtype == PU_DTYPE_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// What a CTA keeps in shared memory: the weights as fp32 (1 without a norm)
// and, per warp, cos and sin of a token's pairs.
struct Shared {
  float w[2][kMaxDim];
  unsigned long long step[kMaxPairs];    // turn per position, as a 64-bit fraction
  float cs[kWarps][4][kMaxPairs];        // forward: cos, sin; backward: see back_angles
};

__device__ __forceinline__ void fill_shared(const Params& p, Shared& sh) {
  for (int i = threadIdx.x; i < 2 * p.D; i += kThreads) {
    const int k = i >= p.D, d = i - k * p.D;
    sh.w[k][d] = p.side[k].w != nullptr ? load_weight(p.side[k].w, p.side[k].w_dtype, d) : 1.f;
  }
  for (int i = threadIdx.x; i < p.R / 2; i += kThreads) {
    const double f = p.ang.freq64 ? static_cast<const double*>(p.ang.freq)[i] : (double)static_cast<const float*>(p.ang.freq)[i];
    // f / 2 pi as the sum of two doubles (1 / 2 pi is one, too), whole turns taken off,
    // in 2^-64ths of a turn
    const double inv = 0.15915494309189535, inv_lo = -9.839338337591243e-18;
    const double turns = f * inv, rest = fma(f, inv, -turns) + f * inv_lo;
    sh.step[i] = (unsigned long long)__double2ll_rn((turns - rint(turns)) * 18446744073709551616.0) +
                 (unsigned long long)__double2ll_rn(rest * 18446744073709551616.0);
  }
  __syncthreads();
}

// Sine and cosine of 2 pi turn / 2^64.  The nearest quarter turn comes off in
// 64-bit integers, so what is left, at most pi / 4, is rounded to fp32 relative to
// itself and small angles keep their precision; then the Taylor series up to x^9 and
// x^8 (the terms left out are below 2 10^-9 and 3 10^-8).  In all under 3.2 roundings
// of 2^-24: of the sine itself near 0, of 1 for the cosine.
__device__ __forceinline__ void sin_cos(unsigned long long turn, float& s, float& c) {
  const unsigned quarter = (unsigned)((turn + 0x2000000000000000ull) >> 62);
  const float x = (float)(long long)(turn - ((unsigned long long)quarter << 62)) * 3.4061215800865545e-19f;   // 2 pi / 2^64
  const float z = x * x;
  float ps = fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
  ps = fmaf(z, ps, 1.f / 120.f);
  ps = fmaf(z, ps, -1.f / 6.f);
  ps = fmaf(x * z, ps, x);
  float pc = fmaf(z, 1.f / 40320.f, -1.f / 720.f);
  pc = fmaf(z, pc, 1.f / 24.f);
  pc = fmaf(z, pc, -0.5f);
  pc = fmaf(z, pc, 1.f);
  const float a = quarter & 1 ? pc : ps, b = quarter & 1 ? ps : pc;
  s = __uint_as_float(__float_as_uint(a) ^ ((quarter & 2) << 30));
  c = __uint_as_float(__float_as_uint(b) ^ (((quarter + 1) & 2) << 30));
}

// A lane's share of a token's angles: pairs `lane` and `lane + 32`.
struct Turner {
  int axis[2];                  // of the pair; -1: no such pair
  long long pos[2];             // of the token that comes next

  __device__ __forceinline__ void start(const Params& p, int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int pair = lane + 32 * i;
      axis[i] = 0;
      pos[i] = 0;
#pragma unroll
      for (int a = 0; a + 1 < kMaxAxes; ++a) axis[i] += pair >= p.ang.pair_end[a];
      if (pair >= p.R / 2) axis[i] = -1;
    }
  }
  // asks for a token's positions (used by the next turn)
  __device__ __forceinline__ void fetch(const Angles& a, unsigned b, unsigned n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (axis[i] < 0) continue;
      if (a.pos == nullptr) {
        pos[i] = n;
      } else {
        const long long at = axis[i] * a.pA + b * a.pB + n * a.pN;
        pos[i] = a.pos64 ? static_cast<const long long*>(a.pos)[at] : (long long)static_cast<const int32_t*>(a.pos)[at];
      }
    }
  }
  // sine and cosine of pair lane + 32 i at its fetched position
  __device__ __forceinline__ void turn(const Shared& sh, int lane, int i, float& s, float& c) const {
    sin_cos(sh.step[lane + 32 * i] * (unsigned long long)pos[i], s, c);
  }
  // of all pairs, into the warp's shared rows
  __device__ __forceinline__ void make(const Shared& sh, int lane, float* cs, float* sn) const {
    __syncwarp();                        // the previous token's have been read
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (axis[i] >= 0) turn(sh, lane, i, sn[lane + 32 * i], cs[lane + 32 * i]);
    __syncwarp();
  }
};

// The units of a warp: a token each, or one part of a token's passes.
struct Unit {
  unsigned id, b, n;          // the token's sequence and index in it
  int first, last;            // its passes

  __device__ __forceinline__ void cut(const Params& p) {
    const unsigned v = id - p.whole, part = v / (unsigned)p.chunks, t = p.whole + part;
    first = (int)(v - part * p.chunks) * p.chunk;
    last = first + p.chunk;
    b = t / (unsigned)p.N;
    n = t - b * (unsigned)p.N;
  }
  __device__ __forceinline__ void start(const Params& p, unsigned warp) {
    id = warp;
    first = 0;
    last = p.passes;
    b = id / (unsigned)p.N;
    n = id - b * (unsigned)p.N;
    if (id >= p.whole) cut(p);
  }
  __device__ __forceinline__ void next(const Params& p, unsigned warps) {
    id += warps;
    n += p.step_n;                       // whole tokens: no division
    b += p.step_b;
    if (n >= (unsigned)p.N) {
      n -= (unsigned)p.N;
      ++b;
    }
    if (id >= p.whole) cut(p);
  }
};

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

template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

__device__ __forceinline__ uint64_t f2_swap(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return f2_pack(b, a);
}

// Row coefficients: with a, b the lane's two vectors (four pairs of values
// each), the rotated norm is, up to 1 / rms,
//   a' = a k0 + x k1,  b' = b k2 + y k3,  (x, y) = (b, a), or interleaved the
//   vectors' own values with neighbours swapped
// so the weight, the rotation and its signs cost one product and one fma per
// two values.  They are made once for a token and kind, k_i by the i-th row's lanes, and
// lie in shared memory as 16-byte pieces [k0 .. k3][2][lane of the row].  (In
// registers, made by every lane: 17 prompts into a cache 46 us instead of 44.)
template <bool kInter, int kLanes>
__device__ __forceinline__ void put_coef(const float* cs, const float* sn, const float* w, const Place& pl, int lane, float4* out) {
  const int sub = lane % kLanes, which = lane / kLanes;
  if (which >= 4) return;
  const bool far = kInter ? which >= 2 : which == 1 || which == 2, sine = which & 1;
  float4 w0 = make_float4(1.f, 1.f, 1.f, 1.f), w1 = w0;
  if (pl.in) {
    const float4* from = reinterpret_cast<const float4*>(w + (far ? pl.o1 : pl.o0));
    w0 = from[0], w1 = from[1];
  }
  const float other = sine ? 0.f : 1.f;
  float4 t0 = make_float4(other, other, other, other), t1 = t0;
  if (pl.rot) {
    const float4* from = reinterpret_cast<const float4*>((sine ? sn : cs) + sub * 8);
    if constexpr (kInter) {
      t0 = from[far];
    } else {
      t0 = from[0], t1 = from[1];
    }
  }
  if constexpr (kInter) {
    if (sine) {
      w0 = make_float4(-w0.y, w0.x, -w0.w, w0.z);
      w1 = make_float4(-w1.y, w1.x, -w1.w, w1.z);
    }
    t1 = make_float4(t0.z, t0.z, t0.w, t0.w);
    t0 = make_float4(t0.x, t0.x, t0.y, t0.y);
  } else if (which == 1) {
    w0 = make_float4(-w0.x, -w0.y, -w0.z, -w0.w);
    w1 = make_float4(-w1.x, -w1.y, -w1.z, -w1.w);
  }
  out[(2 * which) * kLanes + sub] = make_float4(w0.x * t0.x, w0.y * t0.y, w0.z * t0.z, w0.w * t0.w);
  out[(2 * which + 1) * kLanes + sub] = make_float4(w1.x * t1.x, w1.y * t1.y, w1.z * t1.z, w1.w * t1.w);
}

// a, b -> a', b' of kU rows.  Lanes behind R take no cross term (theirs would be 0 times
// a value that need not be finite).
template <bool kInter, int kLanes, int kU>
__device__ __forceinline__ void apply_coef(const float4* k, int sub, bool partial, bool rot, uint64_t (&a)[kU][4], uint64_t (&b)[kU][4]) {
  auto two = [&](int c) { return *reinterpret_cast<const ulonglong2*>(k + c * kLanes + sub); };
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const ulonglong2 k0 = two(half), k2 = two(4 + half);
    if (partial && !rot) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        a[u][2 * half] = f2_mul(a[u][2 * half], k0.x);
        a[u][2 * half + 1] = f2_mul(a[u][2 * half + 1], k0.y);
        b[u][2 * half] = f2_mul(b[u][2 * half], k2.x);
        b[u][2 * half + 1] = f2_mul(b[u][2 * half + 1], k2.y);
      }
    } else {
      const ulonglong2 k1 = two(2 + half), k3 = two(6 + half);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint64_t p = a[u][2 * half + i], q = b[u][2 * half + i];
          a[u][2 * half + i] = f2_fma(kInter ? f2_swap(p) : q, i ? k1.y : k1.x, f2_mul(p, i ? k0.y : k0.x));
          b[u][2 * half + i] = f2_fma(kInter ? f2_swap(q) : p, i ? k3.y : k3.x, f2_mul(q, i ? k2.y : k2.x));
        }
      }
    }
  }
}

// The rotation back, straight from shared memory (its coefficients would take
// the registers that hold rows in flight).  The warp's 256 floats: for halves
// c, s, -s of each pair; interleaved (c, c) and (s, -s) of each.
template <bool kInter>
__device__ __forceinline__ void back_angles(const Turner& t, const Shared& sh, int lane, float* m) {
  __syncwarp();                          // the previous token's have been read
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (t.axis[i] < 0) continue;
    const int pair = lane + 32 * i;
    float s, c;
    t.turn(sh, lane, i, s, c);
    if constexpr (kInter) {
      reinterpret_cast<float2*>(m)[pair] = make_float2(c, c);
      reinterpret_cast<float2*>(m + 2 * kMaxPairs)[pair] = make_float2(s, -s);
    } else {
      m[pair] = c;
      m[kMaxPairs + pair] = s;
      m[2 * kMaxPairs + pair] = -s;
    }
  }
  __syncwarp();
}

template <bool kInter>
__device__ __forceinline__ void turn_back(const float* m, int sub, uint64_t (&a)[4], uint64_t (&b)[4]) {
  auto two = [](const float* p) { return *reinterpret_cast<const ulonglong2*>(p); };
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    if constexpr (kInter) {
      const float* c = m + sub * 16 + 2 * i;
      const ulonglong2 ca = two(c), sa = two(c + 2 * kMaxPairs), cb = two(c + 8), sb = two(c + 8 + 2 * kMaxPairs);
      a[i] = f2_fma(f2_swap(a[i]), sa.x, f2_mul(a[i], ca.x));
      a[i + 1] = f2_fma(f2_swap(a[i + 1]), sa.y, f2_mul(a[i + 1], ca.y));
      b[i] = f2_fma(f2_swap(b[i]), sb.x, f2_mul(b[i], cb.x));
      b[i + 1] = f2_fma(f2_swap(b[i + 1]), sb.y, f2_mul(b[i + 1], cb.y));
    } else {
      const float* c = m + sub * 8 + 2 * i;
      const ulonglong2 cc = two(c), ss = two(c + kMaxPairs), ns = two(c + 2 * kMaxPairs);
      const uint64_t a0 = a[i], a1 = a[i + 1];
      a[i] = f2_fma(b[i], ss.x, f2_mul(a0, cc.x));
      a[i + 1] = f2_fma(b[i + 1], ss.y, f2_mul(a1, cc.y));
      b[i] = f2_fma(a0, ns.x, f2_mul(b[i], cc.x));
      b[i + 1] = f2_fma(a1, ns.y, f2_mul(b[i + 1], cc.y));
    }
  }
}

__device__ __forceinline__ float f2_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

// A pass is 32 / kLanes rows (heads) of one token; queries' passes come
// first, then keys', then values'.  A warp walks units, whole tokens or parts
// of one; a run is a unit's passes of one kind.
//
// Rows come through a ring in shared memory: each lane copies its own
// vectors of the passes to come (cp.async) into places of its own, kSlots - 2
// passes ahead, over the borders of runs and tokens.  Nobody else reads them, so a
// lane waits for its own copies and for no other thread.  (Loads into registers
// run ahead inside a run only: forward 61 us instead of 58, backward 114 instead of
// 109, 17 prompts into a cache 48 instead of 44.)
// kVecs: vectors of 8 a lane copies for a pass, two of the row and, backward, two of its gradient.
template <typename T, int kLanes, int kKinds, int kVecs>
struct Feed {
  static constexpr int kRows = 32 / kLanes;
  static constexpr int kSlots = sizeof(T) == 4 || kVecs == 4 ? 4 : 5;   // forward, 16-bit: 4 58.9 us, 5 57.8, 6 59.9
  static constexpr int kChunks = (int)sizeof(T) / 2;        // 16-byte pieces of a vector
  static constexpr int kSlotBytes = kVecs * kChunks * 512;
  static constexpr int kBytes = kWarps * kSlots * kSlotBytes;
  static_assert(kSlots >= 4, "two passes in use, two on their way");
  Unit unit;
  unsigned warps;
  uint32_t base, fill;        // the lane's place in slot 0; byte offset of the slot to fill
  int gap;                    // bytes between the lane's two vectors
  int kind, begin;
  int left, h, heads;         // of the run: passes to ask for; the lane's head, and below which it copies
  const uint8_t *x, *g;       // the lane's first vector of the next row
  const uint8_t* safe;        // a row's address for copies that read nothing
  long long xs, gs;
  bool norm;

  // to the next run, of this unit or a later one; heads = 0 behind the last
  __device__ __forceinline__ void run(const Params& p, const Place& pl, int row) {
    for (; unit.id < p.units; unit.next(p, warps), kind = -1, begin = 0) {
      while (++kind < kKinds) {
        const Side& sd = p.side[kind];
        const int passes = (sd.heads + kRows - 1) / kRows;
        const int lo = max(unit.first - begin, 0), hi = min(unit.last - begin, passes);
        begin += passes;
        if (lo >= hi) continue;
        left = hi - lo;
        heads = pl.in ? sd.heads : 0;
        h = lo * kRows + row;
        xs = sd.x.sH * (long long)sizeof(T);
        x = static_cast<const uint8_t*>(sd.x.p) +
            (unit.b * sd.x.sB + unit.n * sd.x.sN + pl.o0) * (long long)sizeof(T) + h * xs;
        xs *= kRows;
        if constexpr (kVecs == 4) {
          norm = sd.w != nullptr;
          gs = sd.g.sH * (long long)sizeof(T);
          g = static_cast<const uint8_t*>(sd.g.p) +
              (unit.b * sd.g.sB + unit.n * sd.g.sN + pl.o0) * (long long)sizeof(T) + h * gs;
          gs *= kRows;
        }
        return;
      }
    }
    h = heads = 0;                       // (a warp may come here before its first run)
    left = 1 << 30;
  }
  // Asks for one pass; zeros where the lane has no row or no place in it.
  __device__ __forceinline__ void ask(const Params& p, const Place& pl, int row) {
    const uint32_t to = base + fill;
    const bool use = h < heads;
    auto copy = [&](int v, const uint8_t* from, bool read) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + (v * kChunks + c) * 512), "l"(from + c * 16),
                     "r"(read ? 16 : 0)
                     : "memory");
    };
    const int far = use ? gap : 0;
    const uint8_t* from = use ? x : safe;
    copy(0, from, use && (kVecs == 2 || norm));
    copy(1, from + far, use && (kVecs == 2 || norm));
    if constexpr (kVecs == 4) {
      const uint8_t* grad = use ? g : safe;
      copy(2, grad, use);
      copy(3, grad + far, use);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    fill = fill + kSlotBytes == kSlots * kSlotBytes ? 0 : fill + kSlotBytes;
    h += kRows;
    x += xs;
    if constexpr (kVecs == 4) g += gs;
    if (--left == 0) run(p, pl, row);
  }
  __device__ __forceinline__ void start(const Params& p, uint8_t* smem, int warp, int lane, const Place& pl) {
    base = smem_u32(smem) + (uint32_t)(warp * kSlots * kSlotBytes + lane * 16);
    gap = (pl.o1 - pl.o0) * (int)sizeof(T);
    warps = gridDim.x * kWarps;
    fill = 0;
    kind = -1;
    begin = 0;
    x = g = nullptr;
    xs = gs = 0;
    safe = static_cast<const uint8_t*>(p.side[p.side[0].heads > 0 ? 0 : 1].x.p);
    unit.start(p, blockIdx.x * kWarps + warp);
    run(p, pl, lane / kLanes);
    for (int i = 0; i + 2 < kSlots; ++i) ask(p, pl, lane / kLanes);
  }
  // Waits for the next kU passes (1 or 2) and returns the place of the first.
  template <int kU>
  __device__ __forceinline__ void wait() const {
    asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 2 - kU) : "memory");
  }
  __device__ __forceinline__ void get(int u, int v, uint64_t (&f)[4]) const {
    const uint32_t off = fill + (2 + u) * kSlotBytes, at = base + (off >= kSlots * kSlotBytes ? off - kSlots * kSlotBytes : off);
    Vec8<T> x;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      uint4 w;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                   : "r"(at + (v * kChunks + c) * 512)
                   : "memory");
      x.set(c, w);
    }
    x.get(f);
  }
  // The vectors of the next kU passes.  The slots that are refilled are those of
  // the two passes before, whose values have been used.
  template <int kU>
  __device__ __forceinline__ void take(const Params& p, const Place& pl, int row, uint64_t (&a)[kU][4], uint64_t (&c)[kU][4]) {
    wait<kU>();
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      get(u, 0, a[u]);
      get(u, 1, c[u]);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) ask(p, pl, row);
  }
};

template <typename T, int kLanes, bool kInter, bool kAppend>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) fwd_kernel(const __grid_constant__ Params p) {
  constexpr int kRows = 32 / kLanes;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) Shared sh;
  __shared__ float4 s_coef[kWarps][2][8 * kLanes];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % kLanes, row = lane / kLanes;
  grid_dep_wait();
  grid_dep_launch_dependents();
  const Place pl = make_place<kInter>(sub, p.D, p.R);
  Feed<T, kLanes, kAppend ? 3 : 2, 2> feed;
  feed.start(p, smem, warp, lane, pl);
  fill_shared(p, sh);
  const bool partial = p.R < p.D;
  Turner turner;
  turner.start(p, lane);
  int next_slot = -1;        // append: where the next unit's token goes
  Unit next;
  auto fetch = [&] {
    if (next.id >= p.units) return;
    turner.fetch(p.ang, next.b, next.n);
    if (kAppend) next_slot = p.slots[next.n];
  };
  next.start(p, blockIdx.x * kWarps + warp);
  fetch();
  while (next.id < p.units) {
    const Unit unit = next;
    const int first = unit.first, last = unit.last;
    const long long b = unit.b, n = unit.n;
    next.next(p, gridDim.x * kWarps);
    size_t pool_row = 0;    // append: page and row of this token
    bool put = true;
    if constexpr (kAppend) {
      const long long slot = next_slot;
      put = slot >= 0 && slot < p.num_slots;
      if (slot >= p.num_slots && lane == 0) record_device_error(PU_ERR_INVALID_ARGUMENT, kSiteAppendSlot);
      pool_row = put ? (size_t)slot : 0;
    }
    bool angles = false;
    int begin = 0;
#pragma unroll
    for (int kind = 0; kind < (kAppend ? 3 : 2); ++kind) {
      const Side& sd = p.side[kind];
      const int heads = sd.heads, end = begin + (heads + kRows - 1) / kRows;
      const int lo = max(first, begin), hi = min(last, end);
      if (lo < hi) {
        // the lane's rows of the kind: head h, then kRows heads further, ...
        int h = (lo - begin) * kRows + row;
        const bool norm = kind < 2 && sd.w != nullptr;
        constexpr bool kPool = kAppend;
        T* y = nullptr;
        size_t at = 0, ys = 0;
        if (kPool && kind > 0) {
          const size_t mask = ((size_t)1 << p.page_shift) - 1;
          at = ((((pool_row >> p.page_shift) * heads + h) << p.page_shift) + (pool_row & mask)) * p.D;
          ys = (size_t)p.D << p.page_shift;
        } else {
          ys = sd.y.sH;
          y = static_cast<T*>(sd.y.p) + b * sd.y.sB + n * sd.y.sN + h * ys;
        }
        if (kind < 2 && !angles) {
          turner.make(sh, lane, sh.cs[warp][0], sh.cs[warp][1]);
          put_coef<kInter, kLanes>(sh.cs[warp][0], sh.cs[warp][1], sh.w[0], pl, lane, s_coef[warp][0]);
          put_coef<kInter, kLanes>(sh.cs[warp][0], sh.cs[warp][1], sh.w[1], pl, lane, s_coef[warp][1]);
          __syncwarp();
          fetch();
          angles = true;
        }
        // kU passes, their chains of sums and shuffles side by side
        auto passes = [&](auto count) {
          constexpr int kU = decltype(count)::value;
          uint64_t a[kU][4], bb[kU][4];
          feed.take(p, pl, row, a, bb);
          if (kind < 2) {
            uint64_t rr[kU];
            if (norm) {
              float ss[kU];
#pragma unroll
              for (int u = 0; u < kU; ++u) {
                uint64_t s0 = 0ull, s1 = 0ull;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  s0 = f2_fma(a[u][i], a[u][i], s0);
                  s1 = f2_fma(bb[u][i], bb[u][i], s1);
                }
                ss[u] = f2_sum(f2_add(s0, s1));
              }
#pragma unroll
              for (int off = kLanes / 2; off > 0; off >>= 1)
#pragma unroll
                for (int u = 0; u < kU; ++u) ss[u] += __shfl_xor_sync(0xffffffffu, ss[u], off);
#pragma unroll
              for (int u = 0; u < kU; ++u) {
                const float r = rsqrtf(ss[u] * p.inv_d + p.eps);
                rr[u] = f2_pack(r, r);
              }
            }
            apply_coef<kInter, kLanes>(s_coef[warp][kind & 1], sub, partial, pl.rot, a, bb);
            if (norm) {
#pragma unroll
              for (int u = 0; u < kU; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  a[u][i] = f2_mul(a[u][i], rr[u]);
                  bb[u][i] = f2_mul(bb[u][i], rr[u]);
                }
            }
          }
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            if (h + u * kRows < heads && pl.in) {
              if (kPool && kind > 0) {
                if (put) {
                  store8_pool(sd.y.p, at + u * kRows * ys + pl.o0, p.pool_dtype, sd.unit, a[u]);
                  store8_pool(sd.y.p, at + u * kRows * ys + pl.o1, p.pool_dtype, sd.unit, bb[u]);
                }
              } else {
                store8(y + u * kRows * ys + pl.o0, a[u]);
                store8(y + u * kRows * ys + pl.o1, bb[u]);
              }
            }
          }
          h += kU * kRows;
          y += kU * kRows * ys;
          at += kU * kRows * ys;
        };
        int pass = lo;
#pragma unroll 1
        for (; pass + 1 < hi; pass += 2) passes(std::integral_constant<int, 2>());
        if (pass < hi) passes(std::integral_constant<int, 1>());
      }
      begin = end;
    }
    if (!angles) fetch();   // a unit of values alone
  }
}

// As the forward: a warp walks units of passes, queries' first, then keys'.
// The weight gradients of a unit's rows go from registers into sums of the
// lane in shared memory; each CTA writes one partial row of either kind, summed
// in a fixed order by dw_kernel (no atomics: the same bits every time).
constexpr int kDwStride = 18;   // floats a lane: 16 sums, and 2 that keep lanes on different banks
template <typename T, int kLanes, bool kInter>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) bwd_kernel(const __grid_constant__ Params p) {
  constexpr int kRows = 32 / kLanes;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) Shared sh;
  __shared__ __align__(16) float s_dw[2][kWarps][32][kDwStride];   // sums by lane, queries' and keys'
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % kLanes, row = lane / kLanes;
  const Place pl = make_place<kInter>(sub, p.D, p.R);
  grid_dep_wait();
  grid_dep_launch_dependents();
  Feed<T, kLanes, 2, 4> feed;
  feed.start(p, smem, warp, lane, pl);
  fill_shared(p, sh);
#pragma unroll
  for (int kind = 0; kind < 2; ++kind)
#pragma unroll
    for (int i = 0; i < 16; ++i) s_dw[kind][warp][lane][i] = 0.f;
  Turner turner;
  turner.start(p, lane);
  Unit next;
  auto fetch = [&] {
    if (next.id < p.units) turner.fetch(p.ang, next.b, next.n);
  };
  next.start(p, blockIdx.x * kWarps + warp);
  fetch();
  while (next.id < p.units) {
    const Unit unit = next;
    const int first = unit.first, last = unit.last;
    const long long b = unit.b, n = unit.n;
    next.next(p, gridDim.x * kWarps);
    bool angles = false;
    int begin = 0;
#pragma unroll 1
    for (int kind = 0; kind < 2; ++kind) {
      const Side& sd = p.side[kind];
      const int heads = sd.heads, end = begin + (heads + kRows - 1) / kRows;   // heads: 0 where no gradient is asked for
      const int lo = max(first, begin), hi = min(last, end);
      if (lo < hi) {
        const bool norm = sd.w != nullptr;
        const float* wa = sh.w[kind] + (pl.in ? pl.o0 : 0);   // lanes without a place hold zeros
        const float* wb = sh.w[kind] + (pl.in ? pl.o1 : 8);
        const long long ys = sd.y.sH;
        int h = (lo - begin) * kRows + row;
        T* yp = static_cast<T*>(sd.y.p) + b * sd.y.sB + n * sd.y.sN + h * ys;
        uint64_t da[4], db[4];               // weight gradient of the unit's rows
#pragma unroll
        for (int i = 0; i < 4; ++i) da[i] = db[i] = 0ull;
        if (!angles) {
          back_angles<kInter>(turner, sh, lane, sh.cs[warp][0]);
          fetch();
          angles = true;
        }
#pragma unroll 1
        for (int pass = lo; pass < hi; ++pass) {
          const bool use = h < heads && pl.in;
          uint64_t x[4], y[4], ha[4], hb[4];
          feed.template wait<1>();
          feed.get(0, 2, ha);
          feed.get(0, 3, hb);
          feed.get(0, 0, x);
          feed.get(0, 1, y);
          feed.ask(p, pl, row);
          if (pl.rot) turn_back<kInter>(sh.cs[warp][0], sub, ha, hb);   // others: no coefficients of theirs are there
          if (norm) {
            uint64_t s0 = 0ull, s1 = 0ull, t0 = 0ull, t1 = 0ull, va[4], vb[4];
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const ulonglong2 w0 = *reinterpret_cast<const ulonglong2*>(wa + 2 * i), w1 = *reinterpret_cast<const ulonglong2*>(wb + 2 * i);
              va[i] = f2_mul(ha[i], w0.x);
              va[i + 1] = f2_mul(ha[i + 1], w0.y);
              vb[i] = f2_mul(hb[i], w1.x);
              vb[i + 1] = f2_mul(hb[i + 1], w1.y);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              s0 = f2_fma(x[i], x[i], s0);
              s1 = f2_fma(y[i], y[i], s1);
              t0 = f2_fma(va[i], x[i], t0);
              t1 = f2_fma(vb[i], y[i], t1);
            }
            const float ss = group_sum<kLanes>(f2_sum(f2_add(s0, s1)));
            const float dot = group_sum<kLanes>(f2_sum(f2_add(t0, t1)));
            const float r = use ? rsqrtf(ss * p.inv_d + p.eps) : 0.f;   // no row: 0 times 0, also where eps is 0
            const float q = -dot * p.inv_d * r * r * r;      // dx = r (h w) + x q
            const uint64_t rr = f2_pack(r, r), qq = f2_pack(q, q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              da[i] = f2_fma(ha[i], f2_mul(x[i], rr), da[i]);
              db[i] = f2_fma(hb[i], f2_mul(y[i], rr), db[i]);
              ha[i] = f2_fma(va[i], rr, f2_mul(x[i], qq));
              hb[i] = f2_fma(vb[i], rr, f2_mul(y[i], qq));
            }
          }
          if (use) {
            store8(yp + pl.o0, ha);
            store8(yp + pl.o1, hb);
          }
          h += kRows;
          yp += kRows * ys;
        }
        if (sd.dw_part != nullptr) {
          float* mine = s_dw[kind][warp][lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint64_t* a = reinterpret_cast<uint64_t*>(mine + 2 * i);
            uint64_t* c = reinterpret_cast<uint64_t*>(mine + 8 + 2 * i);
            *a = f2_add(*a, da[i]);
            *c = f2_add(*c, db[i]);
          }
        }
      }
      begin = end;
    }
  }
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    const Side& sd = p.side[kind];
    if (sd.dw_part == nullptr) continue;
    // rows of the warp, then the warps
    float v[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* mine = s_dw[kind][warp][lane];
      v[2 * i] = mine[2 * i], v[2 * i + 1] = mine[2 * i + 1];
      v[8 + 2 * i] = mine[8 + 2 * i], v[8 + 2 * i + 1] = mine[8 + 2 * i + 1];
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
#pragma unroll
      for (int off = kLanes; off < 32; off <<= 1) v[j] += __shfl_xor_sync(0xffffffffu, v[j], off);
    }
    __syncthreads();                       // the other kind's sums have been read
    float* sums = sh.cs[warp][0];          // no more angles
    if (row == 0 && pl.in) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sums[pl.o0 + j] = v[j];
        sums[pl.o1 + j] = v[8 + j];
      }
    }
    __syncthreads();
    if ((int)threadIdx.x < p.D) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) sum += (&sh.cs[i][0][0])[threadIdx.x];
      sd.dw_part[(size_t)blockIdx.x * p.D + threadIdx.x] = sum;
    }
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
    for (int c = part; c < p.ctas; c += kDwParts) v += __ldcg(sd.dw_part + (size_t)c * p.D + d);
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
  p->inv_d = 1.f / (float)d->D;
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

// Cuts the tokens' passes into units; returns the CTAs.  A warp takes all
// passes of a token, so that the angles are made once; the tokens left over
// after the last full round of the warps are cut into parts while that leaves
// no warp a second one (17 prompts of 15 thousand
// tokens: 6.3 rounds, the last one then a third of a token long).
inline int share_out(Params& p, int kinds, int ctas_per_sm) {
  p.passes = 0;
  for (int k = 0; k < kinds; ++k) p.passes += p.side[k].heads ? passes_of(p.side[k].heads, p.D) : 0;
  const long long ctas = (long long)sm_count() * ctas_per_sm, warps = ctas * kWarps, rest = p.T % warps;
  p.chunks = rest ? (int)std::min<long long>(p.passes, std::max<long long>(1, warps / rest)) : 1;
  p.chunk = (p.passes + p.chunks - 1) / p.chunks;
  p.chunks = (p.passes + p.chunk - 1) / p.chunk;
  p.whole = (unsigned)(p.T - rest);
  p.units = (unsigned)(p.whole + rest * p.chunks);
  p.step_b = (unsigned)(warps / p.N);
  p.step_n = (unsigned)(warps % p.N);
  return (int)std::min<long long>((p.units + kWarps - 1ll) / kWarps, ctas);
}

template <typename T, bool kAppend>
int launch_fwd(Params& p, bool inter, cudaStream_t st) {
  const int grid = share_out(p, kAppend ? 3 : 2, kCtasPerSm);
  const bool wide = lanes_of(p.D) == 8;
  auto* k = wide ? (inter ? fwd_kernel<T, 8, true, kAppend> : fwd_kernel<T, 8, false, kAppend>)
                 : (inter ? fwd_kernel<T, 4, true, kAppend> : fwd_kernel<T, 4, false, kAppend>);
  const int smem = wide ? Feed<T, 8, 2, 2>::kBytes : Feed<T, 4, 2, 2>::kBytes;
  const int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(k), smem, "norm and rotation shared memory");
  if (rc) return rc;
  return check_cuda(decode::launch_pdl(k, dim3(grid), dim3(kThreads), smem, st, p), "norm and rotation launch");
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
  const int smem = wide ? Feed<T, 8, 2, 4>::kBytes : Feed<T, 4, 2, 4>::kBytes;
  const int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(k), smem, "norm and rotation backward shared memory");
  if (rc) return rc;
  return check_cuda(decode::launch_pdl(k, dim3((unsigned)grid), dim3(kThreads), smem, st, p), "norm and rotation backward launch");
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
  return (size_t)pu::rope::bwd_ctas() * 2 * D * sizeof(float);
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
  if (!dq) p.side[0].heads = 0;
  if (!dk) p.side[1].heads = 0;
  p.ctas = share_out(p, 2, kCtasPerSm);
  p.side[0].x = rows_of(q, d->q_stride);
  p.side[1].x = rows_of(k, d->k_stride);
  p.side[0].g = rows_of(gq, d->gq_stride);
  p.side[1].g = rows_of(gk, d->gk_stride);
  p.side[0].y = rows_of(dq, d->dq_stride);
  p.side[1].y = rows_of(dk, d->dk_stride);
  float* part = static_cast<float*>(workspace);
  p.side[0].dw_part = dq_weight ? part : nullptr;
  p.side[1].dw_part = dk_weight ? part + (size_t)bwd_ctas() * d->D : nullptr;
  p.side[0].dw = dq_weight;
  p.side[1].dw = dk_weight;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool inter = d->interleaved != 0;
  const int grid = p.ctas;
  rc = d->dtype == PU_DTYPE_F32 ? launch_bwd<float>(p, inter, grid, st)
       : d->dtype == PU_DTYPE_F16 ? launch_bwd<__half>(p, inter, grid, st)
                                  : launch_bwd<__nv_bfloat16>(p, inter, grid, st);
  if (rc || (!dq_weight && !dk_weight)) return rc;
  return pu::check_cuda(pu::decode::launch_pdl(dw_kernel, dim3(2), dim3(kMaxDim * kDwParts), 0, st, p),
                        "norm weight gradient launch");
}

}  // extern "C"
