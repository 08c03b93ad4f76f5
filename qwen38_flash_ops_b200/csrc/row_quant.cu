// Rows in eight bits with a scale each: of a root-mean-square norm, with the residual stream's addition; of a gated activation; of
// the rows themselves.
//
//   norm    h = x + residual, rounded to its type and kept; y_i = h_i (offset + weight_i) rsqrt(mean(h^2) + eps)
//   act     y_i = x_i / (1 + exp(-x_i)) u_i, or x_i
//   scale = max(max_i |y_i|, 2^-100) / top, q_i = y_i / scale rounded to the nearest (ties to even), top = 127 (INT8) or 448 (E4M3)
//
// All of it in FP32 until the one rounding to eight bits.  One pass over memory: the largest |h_i (offset + weight_i)| is found
// beside the sum of squares, because the norm's factor is the same for the whole row, and leaves q_i altogether, so a row needs one reduction and its
// values wait in registers.  Rows longer than the registers of a block hold (18432 values, 19968 of many rows through the ring, 16384 that lie anywhere) are
// read again.  A row whose sum of squares or largest value is no finite FP32 number has scale NaN and q 0.
//
// What bounds it, on one B200 (a copy's 6.55 TB/s is the floor, in brackets).  Few rows: the launch, one trip to memory and the reduction, 2.4 us in a graph for
// 1 x 5120, 3.7 for 4 x 17408 gated; a call takes longer on the host (4.5 to 5.8).  Many rows: memory, 4096 x 5120 with residual 24 to 27 us (22.4), as they are 12
// (9.6); instructions, 16 an element of which four are the exponential and the quotient, 2048 x 17408 gated 33 to 34 (27.2); a norm alone the latency of its two
// reductions, 4096 x 5120 16 (9.6).  Rows that lie off 16 bytes go element by element, 4096 x 5119 67 as they are, 75 a norm, 96 with residual, 83 gated: loads of
// two bytes and stores of one take the load unit as long as wide ones.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "qfg_internal.h"
#include "stream_order.cuh"
#include "tc_ptx.cuh"

namespace qfg {
namespace {

enum RowKind : int { kRows = 0, kSwish = 1, kNorm = 2, kNormAdd = 3 };
constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100

struct RowParams {
  const void *x, *second, *weight;  // second: u, or the residual
  void* h;
  uint8_t* q;
  float* scale;
  long long ldx, ld2, rows;
  int n, warps, rows_per_block;  // warps of a row
  int stages, stage_bytes;       // of the ring
  bool trigger;                  // release the next kernel behind the wait
  bool give_up;                  // testing: no row reaches the ring
  bool fp8, weight_f32;
  float offset, eps, inv_n;
};

template <typename T>
__device__ __forceinline__ float ToFloat(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T FromFloat(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
}
// C consecutive elements as they are stored, of 16 bytes or one
template <typename T, int C>
struct alignas(C == 1 ? sizeof(T) : 16) Piece {
  T v[C];
};
template <typename T, int C>
__device__ __forceinline__ Piece<T, C> Load(const T* p) {
  Piece<T, C> r;
  if constexpr (C == 1) {
    r.v[0] = *p;
  } else {
    static_assert(sizeof(r) % 16 == 0, "");
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  return r;
}
template <typename T, int C>
__device__ __forceinline__ void Store(T* p, const Piece<T, C>& v) {
  if constexpr (C == 1) {
    *p = v.v[0];
  } else {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(v) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&v)[i];
  }
}

// Two FP32 operations in one instruction.
__device__ __forceinline__ float2 Mul2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 Fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{ .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 Add2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 Both(float v) { return make_float2(v, v); }

// x + residual in their type.  In 16 bits the packed addition rounds once, as an FP32 addition rounded to 16 bits does here: a sum that is
// inexact in FP32 has an addend below a quarter of an ulp of the other.
__device__ __forceinline__ float Add(float a, float b) { return a + b; }
__device__ __forceinline__ __half Add(__half a, __half b) { return __float2half_rn(__half2float(a) + __half2float(b)); }
__device__ __forceinline__ __nv_bfloat16 Add(__nv_bfloat16 a, __nv_bfloat16 b) { return __float2bfloat16_rn(__bfloat162float(a) + __bfloat162float(b)); }
template <typename T, int C>
__device__ __forceinline__ Piece<T, C> AddPieces(const Piece<T, C>& a, const Piece<T, C>& b) {
  Piece<T, C> r;
  if constexpr (C == 1 || sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < C; ++e) r.v[e] = Add(a.v[e], b.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < C / 2; ++e) {
      uint32_t &o = reinterpret_cast<uint32_t*>(&r)[e];
      const uint32_t u = reinterpret_cast<const uint32_t*>(&a)[e], v = reinterpret_cast<const uint32_t*>(&b)[e];
      if constexpr (std::is_same_v<T, __half>) {
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(o) : "r"(u), "r"(v));
      } else {
        asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(o) : "r"(u), "r"(v));
      }
    }
  }
  return r;
}
// elements 2 e and 2 e + 1 (C = 1: the one, and nothing)
template <typename T, int C>
__device__ __forceinline__ float2 Two(const Piece<T, C>& p, int e) {
  if constexpr (C == 1) {
    return make_float2(ToFloat(p.v[0]), 0.f);
  } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(&p)[e];
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  } else if constexpr (std::is_same_v<T, __half>) {
    return __half22float2(reinterpret_cast<const __half2*>(&p)[e]);
  } else {
    return make_float2(ToFloat(p.v[2 * e]), ToFloat(p.v[2 * e + 1]));
  }
}

template <int C>
constexpr int kPairs = C == 1 ? 1 : C / 2;
// What the largest value of a row gives the others: top / largest, and what that quotient's rounding left of it.
struct Factor {
  float hi, lo;
};
// The values f[i] top / largest in eight bits.  INT8: adding 1.5 * 2^23 leaves the integer nearest to a value of at most 2^22 in the low
// bits; |f| <= largest keeps it within [-127, 127].  The quotient is rounded to FP32 once, the factor's own rounding carried along, so that one that lies half
// way, as half of the largest does, is rounded to even and not as the factor was.  (A value that lands on the other side is a step in one of the sums of
// the product that follows; with the rounded factor alone one in ten calls had such rows, 8 x 5120.)
template <int C>
__device__ __forceinline__ void StoreQuantised(uint8_t* p, const float2 (&f)[kPairs<C>], const Factor& by, bool fp8) {
  uint32_t two[kPairs<C>];  // a pair in the lower 16 bits
  auto value = [&](int e) { return Fma2(f[e], Both(by.hi), Mul2(f[e], Both(by.lo))); };
  if (fp8) {
#pragma unroll
    for (int e = 0; e < kPairs<C>; ++e) two[e] = __nv_cvt_float2_to_fp8x2(value(e), __NV_SATFINITE, __NV_E4M3);
  } else {
#pragma unroll
    for (int e = 0; e < kPairs<C>; ++e) {
      const float2 v = Add2(value(e), Both(12582912.f));
      two[e] = __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x0040);
    }
  }
  if constexpr (C == 1) {
    *p = static_cast<uint8_t>(two[0]);
  } else if constexpr (C == 4) {
    *reinterpret_cast<uint32_t*>(p) = __byte_perm(two[0], two[1], 0x5410);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(__byte_perm(two[0], two[1], 0x5410), __byte_perm(two[2], two[3], 0x5410));
  }
}
// The part of a row's factor that StoreQuantised does not apply, where there is one.
template <int KIND, int C>
__device__ __forceinline__ void TakeUp(float2 (&f)[kPairs<C>], float first) {
  if constexpr (KIND >= kNorm) {
    if (first != 1.f) {
#pragma unroll
      for (int e = 0; e < kPairs<C>; ++e) f[e] = Mul2(f[e], Both(first));
    }
  }
}
template <int C>
__device__ __forceinline__ void StoreZeros(uint8_t* p) {
  if constexpr (C == 1) {
    *p = 0;
  } else if constexpr (C == 4) {
    *reinterpret_cast<uint32_t*>(p) = 0;
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(0, 0);
  }
}

// a / (1 + exp(-a)), to 2^-21: exp(-a) is 2^hi (1 + lo ln 2) with hi + lo = -a log2 e.  With the rounded product alone for the exponent the
// result would be off by 2^-24 |a|, 2^-18 at 60.  A BF16 value times the upper 16 bits of log2 e is exact, and lo the rest; else hi is the rounded
// product and lo what the rounding left, for which values that overflow it (FP32 alone) are kept within bounds.  A reciprocal below 2^-126 is
// flushed, so that from a = -87.3 down, where a result is below 1.1e-36, it is zero before u multiplies it.
template <typename T>
__device__ __forceinline__ float2 Swish2(float2 a) {
  float2 hi, t;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    hi = Mul2(a, Both(-47274.f / 32768.f));
    t = Fma2(a, Both(-4.888495e-06f), Both(1.0f));  // 7.052608e-6 ln 2
  } else {
    const float2 b = std::is_same_v<T, float> ? make_float2(fmaxf(fminf(a.x, 1e38f), -200.f), fmaxf(fminf(a.y, 1e38f), -200.f)) : a;
    hi = Mul2(b, Both(-1.44269504f));
    const float2 lo = Fma2(b, Both(-1.92596299e-8f), Fma2(b, Both(-1.44269504f), make_float2(-hi.x, -hi.y)));
    t = Fma2(lo, Both(0.693147181f), Both(1.0f));
  }
  float2 e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(hi.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(hi.y));
  const float2 d = Fma2(e, t, Both(1.0f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  return Mul2(a, r);
}

// The largest magnitude of three, or a NaN.
__device__ __forceinline__ float MaxMagnitude(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The part of a row's values that follows from the elements themselves, what they add to the row's sum of squares, and the
// largest magnitude so far.  The sum of the residual stream is stored to h.
template <int KIND, typename T, int C>
__device__ __forceinline__ void Values(float2 (&f)[kPairs<C>], const Piece<T, C>& x, const Piece<T, C>& second, const RowParams& p, const void* weight,
                                       const Piece<T, C>* held, int i, T* h, float2& squares, float& largest) {
  Piece<T, C> v = x;
  if constexpr (KIND == kNormAdd) {
    v = AddPieces<T, C>(x, second);
    Store<T, C>(h, v);
  }
#pragma unroll
  for (int e = 0; e < kPairs<C>; ++e) f[e] = Two<T, C>(v, e);
  if constexpr (KIND == kSwish) {
#pragma unroll
    for (int e = 0; e < kPairs<C>; ++e) f[e] = Mul2(Swish2<T>(f[e]), Two<T, C>(second, e));
  }
  if constexpr (KIND >= kNorm) {
#pragma unroll
    for (int e = 0; e < kPairs<C>; ++e) squares = Fma2(f[e], f[e], squares);
    if (p.weight_f32) {
      const Piece<float, C> w = Load<float, C>(static_cast<const float*>(weight) + i);
#pragma unroll
      for (int e = 0; e < kPairs<C>; ++e) f[e] = Mul2(f[e], Add2(Two<float, C>(w, e), Both(p.offset)));
    } else {
      const Piece<T, C> w = held != nullptr ? *held : Load<T, C>(static_cast<const T*>(weight) + i);
#pragma unroll
      for (int e = 0; e < kPairs<C>; ++e) f[e] = Mul2(f[e], Add2(Two<T, C>(w, e), Both(p.offset)));
    }
  }
#pragma unroll
  for (int e = 0; e < kPairs<C>; ++e) largest = MaxMagnitude(largest, f[e].x, f[e].y);  // C = 1: y is 0
}

// The row's sum of squares and largest magnitude, for every thread of it.  Magnitudes are compared as the integers their bits are,
// in which a NaN is larger than any number.
struct RowSums {
  float squares;
  uint32_t largest;
};
// Of up to 32 warps.
struct Partial {
  float sums[32];
  uint32_t tops[32];
};
template <bool SUM>
__device__ __forceinline__ RowSums Reduce(float2 squares2, float largest_f, int warps, int warp_of_row, Partial& part) {
  float squares = squares2.x + squares2.y;
  uint32_t largest = __reduce_max_sync(0xffffffffu, __float_as_uint(largest_f) & 0x7FFFFFFFu);
#pragma unroll
  for (int d = 16; SUM && d > 0; d >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, d);
  if (warps == 1) {
    __syncwarp();
    return {squares, largest};
  }
  if ((threadIdx.x & 31) == 0) {
    if (SUM) part.sums[warp_of_row] = squares;
    part.tops[warp_of_row] = largest;
  }
  __syncthreads();
  // every warp adds the warps' sums in the same order
  const int lane = threadIdx.x & 31;
  largest = __reduce_max_sync(0xffffffffu, lane < warps ? part.tops[lane] : 0u);
  if (SUM) {
    squares = lane < warps ? part.sums[lane] : 0.f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, d);
  }
  return {squares, largest};
}

struct Scaling {
  Factor by;
  float first;  // a factor ahead of `by`, of rows whose one factor FP32 might not hold; else 1
  float most;   // the largest magnitude behind the norm, at least `tiny`
  bool bad;
};
// The quotient by the rounded reciprocal, corrected by what it leaves: rounded as a division is (Markstein's theorem, of a reciprocal rounded to nearest), without
// the cases of a division that cannot come up here.
__device__ __forceinline__ float ScaleOf(const Scaling& s, bool fp8) {
  const float top = fp8 ? 448.f : 127.f, part = fp8 ? 1.f / 448.f : 1.f / 127.f, q = s.most * part;
  return s.bad ? __uint_as_float(0x7FFFFFFFu) : fmaf(fmaf(-q, top, s.most), part, q);
}
template <int KIND>
__device__ __forceinline__ Scaling ScalingOf(const RowSums& r, const RowParams& p) {
  const float top = p.fp8 ? 448.f : 127.f;
  Scaling s;
  float root = 1.f;
  if constexpr (KIND >= kNorm) root = rsqrtf(fmaf(r.squares, p.inv_n, p.eps));
  // (f root) / (max(largest root, tiny) / top).  The norm's factor leaves the quotient but for rows of tiny values, where f root is at most `tiny` and
  // root (top / tiny) alone may be past FP32.  So may top / largest be where a small eps makes much of little: such values are taken up by a power of two.
  const float largest = __uint_as_float(r.largest), most = largest * root;
  // An infinite root (zeros without eps have no norm) leaves an infinity or, of zeros, a NaN; a sum of squares past FP32 leaves a root of zero.
  s.bad = !(most <= 3.4028234e38f) || (KIND >= kNorm && !(r.squares <= 3.4028234e38f));
  s.first = 1.f;
  if (most > kTiny) {
    float by = largest;
    if (KIND >= kNorm && largest < kTiny) {
      s.first = 1.8446744073709552e19f;  // 2^64
      by *= s.first;
    }
    s.by.hi = top / by;
    s.by.lo = fmaf(-by, s.by.hi, top) * (s.by.hi * (p.fp8 ? 1.f / 448.f : 1.f / 127.f));
  } else {
    s.first = root;
    s.by.hi = top / kTiny;
    s.by.lo = 0.f;
  }
  s.most = fmaxf(most, kTiny);
  return s;
}

// Threads a block may have with so many elements of a row in each one's registers.
constexpr int MostThreads(int elements) { return elements <= 16 ? 1024 : elements <= 24 ? 768 : elements <= 32 ? 576 : 416; }
constexpr int kMostOfRow = 24 * MostThreads(24);  // of pieces of 16 bytes: the longest row in 24 elements a thread, and in 32

// Rows straight into registers, V pieces of C elements a thread.  C > 1: pieces of 16 bytes; C = 1: rows that lie anywhere.  V = 0: rows
// read twice.
template <int KIND, typename T, int C, int V>
__global__ void __launch_bounds__(MostThreads(C * V)) RowQuantKernel(const RowParams p) {
  __shared__ Partial parts[4];
  constexpr bool kTwo = KIND == kSwish || KIND == kNormAdd;
  GridDependencyWait();
  if (p.trigger) GridLaunchDependents();
  const T *const x = BehindWait(static_cast<const T*>(p.x)), *const second = BehindWait(static_cast<const T*>(p.second));
  const char* const weight = BehindWait(static_cast<const char*>(p.weight));
  const int warp = static_cast<int>(threadIdx.x) >> 5, row_of_block = warp / p.warps, warp_of_row = warp - row_of_block * p.warps;
  const int step = p.warps * 32 * C, first = (warp_of_row * 32 + (static_cast<int>(threadIdx.x) & 31)) * C;
  const long long row = static_cast<long long>(blockIdx.x) * p.rows_per_block + row_of_block;
  const int n = row < p.rows ? p.n : 0;
  const T* const xr = x + row * p.ldx;
  const T* const sr = second + row * p.ld2;
  T* const hr = static_cast<T*>(p.h) + row * p.n;
  uint8_t* const qr = p.q + row * p.n;
  float2 squares = make_float2(0.f, 0.f);
  float largest = 0.f;
  if constexpr (V > 0) {
    Piece<T, C> a[V], b[V];
    float2 f[V][kPairs<C>];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (first + j * step < n) {
        a[j] = Load<T, C>(xr + first + j * step);
        if constexpr (kTwo) b[j] = Load<T, C>(sr + first + j * step);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (first + j * step < n) Values<KIND, T, C>(f[j], a[j], b[j], p, weight, nullptr, first + j * step, hr + first + j * step, squares, largest);
    }
    const RowSums r = Reduce<(KIND >= kNorm)>(squares, largest, p.warps, warp_of_row, parts[row_of_block]);
    const Scaling s = ScalingOf<KIND>(r, p);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (first + j * step >= n) break;
      if (s.bad) {
        StoreZeros<C>(qr + first + j * step);
      } else {
        TakeUp<KIND, C>(f[j], s.first);
        StoreQuantised<C>(qr + first + j * step, f[j], s.by, p.fp8);
      }
    }
    if (first == 0 && n > 0) p.scale[row] = ScaleOf(s, p.fp8);
  } else {
    float2 f[kPairs<C>];
    for (int i = first; i < n; i += step) {
      const Piece<T, C> a = Load<T, C>(xr + i);
      Values<KIND, T, C>(f, a, kTwo ? Load<T, C>(sr + i) : a, p, weight, nullptr, i, hr + i, squares, largest);
    }
    const RowSums r = Reduce<(KIND >= kNorm)>(squares, largest, p.warps, warp_of_row, parts[row_of_block]);
    const Scaling s = ScalingOf<KIND>(r, p);
    for (int i = first; i < n; i += step) {
      // of the residual stream, the sums that this thread has stored
      const Piece<T, C> a = Load<T, C>(KIND == kNormAdd ? hr + i : xr + i);
      Values<KIND == kNormAdd ? kNorm : KIND, T, C>(f, a, KIND == kSwish ? Load<T, C>(sr + i) : a, p, weight, nullptr, i, hr + i, squares, largest);
      if (s.bad) {
        StoreZeros<C>(qr + i);
      } else {
        TakeUp<KIND, C>(f, s.first);
        StoreQuantised<C>(qr + i, f, s.by, p.fp8);
      }
    }
    if (first == 0 && n > 0) p.scale[row] = ScaleOf(s, p.fp8);
  }
}

// Many rows on 16 bytes: blocks that stay walk over them, and bulk copies bring the next rows into a ring in shared memory meanwhile.  A thread
// holds its V pieces of a row as FP32 between the row's sums and its eight bits.  Nothing but the barrier of those sums says that a row
// has left the ring: the block's first thread then asks for the row that takes its place.  The weight waits in registers, as it is stored.
// Every wait is bounded.  A block that gives up on one marks the rows that it has left, as rows without a finite value are, and asks for no more.
constexpr int kMaxRowStages = 8, kRingRoom = 210 * 1024, kRingBlocks = 8;
struct RowCtl {
  unsigned long long full[kMaxRowStages];
  volatile uint32_t fault;
};
template <int KIND, typename T, int V>
__global__ void __launch_bounds__(MostThreads(16 / sizeof(T) * V)) RowRingKernel(const RowParams p) {
  constexpr int C = 16 / sizeof(T);
  constexpr bool kTwo = KIND == kSwish || KIND == kNormAdd;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ RowCtl ctl;
  __shared__ Partial parts[2];
  const uint32_t full0 = Smem(ctl.full), ring0 = Smem(ring);
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) BarInit(full0 + i * 8, 1);
    ctl.fault = p.give_up ? 1u : 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  GridDependencyWait();
  if (p.trigger) GridLaunchDependents();
  __syncthreads();
  const T *const x = BehindWait(static_cast<const T*>(p.x)), *const second = BehindWait(static_cast<const T*>(p.second));
  const char* const weight = BehindWait(static_cast<const char*>(p.weight));
  const uint32_t row_bytes = static_cast<uint32_t>(p.n * sizeof(T)), stage_bytes = static_cast<uint32_t>(p.stage_bytes);
  auto fetch = [&](long long row, int stage) {
    const uint32_t bar = full0 + stage * 8, dst = ring0 + static_cast<uint32_t>(stage) * stage_bytes;
    BarExpect(bar, kTwo ? 2 * row_bytes : row_bytes);
    BulkLoad(dst, x + row * p.ldx, row_bytes, bar);
    if constexpr (kTwo) BulkLoad(dst + stage_bytes / 2, second + row * p.ld2, row_bytes, bar);
  };
  if (threadIdx.x == 0 && !p.give_up) {
    for (int i = 0; i < p.stages; ++i) {
      const long long row = blockIdx.x + static_cast<long long>(i) * gridDim.x;
      if (row < p.rows) fetch(row, i);
    }
  }
  const int warp = static_cast<int>(threadIdx.x) >> 5, step = p.warps * 32 * C, first = static_cast<int>(threadIdx.x) * C, own = (p.n - first + step - 1) / step;
  Piece<T, C> w[KIND >= kNorm ? V : 1];
#pragma unroll
  for (int j = 0; KIND >= kNorm && j < V; ++j) {
    if (!p.weight_f32 && j < own) w[j] = Load<T, C>(reinterpret_cast<const T*>(weight) + first + j * step);
  }
  const uint8_t* const from = ring + threadIdx.x * 16;
  T* hr = static_cast<T*>(p.h) + blockIdx.x * static_cast<long long>(p.n) + first;
  uint8_t* qr = p.q + blockIdx.x * static_cast<long long>(p.n) + first;
  const long long stride = static_cast<long long>(gridDim.x) * p.n;
  int stage = 0, turn = 0;
  uint32_t parity = 0;
  bool good = true;  // of this thread: false from its first wait that ran out.  What it adds to the sums marks this row and all that the block has left
#pragma unroll 1
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1, hr += stride, qr += stride) {
    float2 f[V][kPairs<C>], squares = make_float2(0.f, 0.f);
    good &= BarWait(full0 + stage * 8, parity, ctl);
    float largest = good ? 0.f : __uint_as_float(0x7FFFFFFFu);
    const int come = KIND == kNormAdd && !good ? 0 : own;  // else what is read where nothing came goes nowhere
    const T* const at = reinterpret_cast<const T*>(from + static_cast<uint32_t>(stage) * stage_bytes);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (j < come) {
        const Piece<T, C> a = Load<T, C>(at + j * step);
        Values<KIND, T, C>(f[j], a, kTwo ? Load<T, C>(at + j * step + stage_bytes / 2 / sizeof(T)) : a, p, weight, KIND >= kNorm ? &w[j] : nullptr, first + j * step, hr + j * step,
                           squares, largest);
      }
    }
    const RowSums r = Reduce<(KIND >= kNorm)>(squares, largest, p.warps, warp, parts[turn]);
    const long long next = row + static_cast<long long>(p.stages) * gridDim.x;
    if (threadIdx.x == 0 && good && next < p.rows) fetch(next, stage);  // what was there has come, and all have read it
    const Scaling s = ScalingOf<KIND>(r, p);
    if (!s.bad) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (j < own) {
          TakeUp<KIND, C>(f[j], s.first);
          StoreQuantised<C>(qr + j * step, f[j], s.by, p.fp8);
        }
      }
    } else {
      for (int j = 0; j < own; ++j) StoreZeros<C>(qr + j * step);
    }
    if (threadIdx.x == 0) p.scale[row] = ScaleOf(s, p.fp8);
    if (++stage == p.stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
  for (int i = 0; i < 16 && !good; ++i) __nanosleep(1000000);  // copies may still be landing in what the block leaves
}

// ------------------------------------------------------------------------------ host
template <int KIND, typename T, int C, int V>
cudaError_t Launch(const RowParams& p, unsigned blocks, unsigned threads, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {OverlapAttribute()};
  cfg.attrs = attr;
  cfg.numAttrs = MayOverlapPredecessor(stream) ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, RowQuantKernel<KIND, T, C, V>, p);
}

template <int KIND, typename T>
int RingBytes(int n) {  // of a row, or the two that it is made of
  return (n * static_cast<int>(sizeof(T)) + 127) / 128 * 128 * (KIND == kSwish || KIND == kNormAdd ? 2 : 1);
}
// Warps of a row whose threads take `v` pieces each.
int WarpsOf(int pieces, int v) { return (pieces + 32 * v - 1) / (32 * v); }

template <int KIND, typename T, int V>
cudaError_t LaunchRing(RowParams& p, int sms, cudaStream_t stream) {
  constexpr int C = 16 / sizeof(T);
  constexpr bool kTwo = KIND == kSwish || KIND == kNormAdd;
  // set up once per device: the limit of shared memory belongs to one
  static std::atomic<uint64_t> raised{0};
  static std::atomic<int> registers{0};
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err == cudaSuccess && (device > 63 || !(raised.load(std::memory_order_acquire) >> device & 1))) {
    cudaFuncAttributes attr;
    err = cudaFuncGetAttributes(&attr, RowRingKernel<KIND, T, V>);
    if (err == cudaSuccess) err = cudaFuncSetAttribute(RowRingKernel<KIND, T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingRoom);
    if (err == cudaSuccess) {
      registers.store((attr.numRegs + 7) / 8 * 8, std::memory_order_relaxed);
      if (device <= 63) raised.fetch_or(1ull << device, std::memory_order_release);
    }
  }
  if (err != cudaSuccess) return err;
  p.warps = WarpsOf(p.n / C, V);
  const int threads = 32 * p.warps;
  // as many blocks as the registers allow, of three rows in flight each where a row is not too long for that
  int blocks = std::max(1, std::min({kRingBlocks, 65536 / (std::max(registers.load(std::memory_order_relaxed), 24) * threads), 2048 / threads}));
  p.stage_bytes = RingBytes<KIND, T>(p.n);
  while (blocks > 1 && kRingRoom / blocks < 3 * p.stage_bytes) --blocks;
  p.stages = std::min(kMaxRowStages, kRingRoom / blocks / p.stage_bytes);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<long long>(p.rows, static_cast<long long>(sms) * blocks)));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(p.stages) * p.stage_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {OverlapAttribute()};
  cfg.attrs = attr;
  cfg.numAttrs = MayOverlapPredecessor(stream) ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, RowRingKernel<KIND, T, V>, p);
}

template <int KIND, typename T, int C>
cudaError_t LaunchShape(RowParams& p, cudaStream_t stream) {
  const int sms = DeviceSmCount(), pieces = (p.n + C - 1) / C;
  constexpr int kOne = C == 1 ? 4 : 8 / C;  // pieces: four elements of a row that lies anywhere, or eight
  const bool few = p.rows <= 2 * sms;
  if constexpr (C > 1) {
    // Many rows of a kilobyte or more, two of which fit the ring.  24 elements a thread, 32 for a norm alone, whose reduction takes the longest for
    // what it reads: rows of up to 18432 either way.  Longer rows 48, where two of them fit at all.  Rows of 5120, 4096 of them, 16 / 24 / 32 / 48 a thread, us: norm
    // 19.5 / 18.9 / 16.3 / 17.3, with residual 24.3 / 24.4 / 24.3 / 27.0, gated 20.5 / 20.9 / 21.3 / 21.4.
    constexpr int kElements = KIND == kNorm ? 32 : 24, kBytes = static_cast<int>(sizeof(T)) * (KIND == kSwish || KIND == kNormAdd ? 2 : 1);
    static_assert(kElements * MostThreads(kElements) == kMostOfRow, "");
    if (!few && p.n * sizeof(T) >= 1024 && 2 * RingBytes<KIND, T>(p.n) <= kRingRoom) {
      if (p.n <= kMostOfRow) return LaunchRing<KIND, T, kElements / C>(p, sms, stream);
      if constexpr (2 * kBytes * kMostOfRow < kRingRoom) {
        if (p.n <= 48 * MostThreads(48)) return LaunchRing<KIND, T, 48 / C>(p, sms, stream);
      }
    }
  }
  // Few rows: as many threads a row as it has pieces.  Many: more pieces a thread, so that the blocks of other rows hide a row's reduction.  32 elements a thread
  // hold no longer a row than 24 do.  Rows that are read twice: 18 warps, three blocks an SM (2000 x 33000, norm alone, 69 us; of 24 warps 93).
  constexpr int kMost = C > 1 ? 3 : 4;
  int e = few ? 1 : 2, warps = 0, most = 1;
  for (;; ++e) {
    warps = WarpsOf(pieces, e * kOne);
    most = MostThreads(C * e * kOne) / 32;
    if (warps <= most || e == kMost) break;
  }
  const bool again = warps > most;
  p.warps = again && C > 1 ? 18 : std::min(warps, most);
  p.rows_per_block = few ? 1 : std::max(1, 4 / p.warps);
  const unsigned threads = static_cast<unsigned>(32 * p.warps * p.rows_per_block);
  const long long blocks = (p.rows + p.rows_per_block - 1) / p.rows_per_block;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  if (again) return Launch<KIND, T, C, 0>(p, static_cast<unsigned>(blocks), threads, stream);
  if (e == 1) return Launch<KIND, T, C, kOne>(p, static_cast<unsigned>(blocks), threads, stream);
  if (e == 2) return Launch<KIND, T, C, 2 * kOne>(p, static_cast<unsigned>(blocks), threads, stream);
  if (e == 3) return Launch<KIND, T, C, 3 * kOne>(p, static_cast<unsigned>(blocks), threads, stream);
  return Launch<KIND, T, C, kMost * kOne>(p, static_cast<unsigned>(blocks), threads, stream);
}

bool On(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <int KIND, typename T>
cudaError_t LaunchTyped(const RowQuantCall& c, RowParams& p, cudaStream_t stream) {
  constexpr int C = 16 / sizeof(T);  // elements of 16 bytes, as many bytes of q
  const bool aligned = On(c.x, 16) && p.ldx % C == 0 && p.n % C == 0 && On(c.q, C) && On(p.second, 16) && p.ld2 % C == 0 && On(c.weight, 16) && On(c.h, 16);
  return aligned ? LaunchShape<KIND, T, C>(p, stream) : LaunchShape<KIND, T, 1>(p, stream);
}

template <typename T>
cudaError_t LaunchKind(const RowQuantCall& c, RowParams& p, cudaStream_t stream) {
  if (!c.norm) return c.u != nullptr ? LaunchTyped<kSwish, T>(c, p, stream) : LaunchTyped<kRows, T>(c, p, stream);
  return c.residual != nullptr ? LaunchTyped<kNormAdd, T>(c, p, stream) : LaunchTyped<kNorm, T>(c, p, stream);
}

}  // namespace

cudaError_t LaunchRowQuant(const RowQuantCall& c, cudaStream_t stream) {
  if (c.rows == 0) return cudaSuccess;
  RowParams p = {};
  p.x = c.x;
  p.second = c.norm ? c.residual : c.u;
  p.weight = c.weight;
  p.h = c.h;
  p.q = c.q;
  p.scale = c.scale;
  p.ldx = c.ldx;
  p.ld2 = p.second == nullptr ? 0 : c.norm ? c.ldr : c.ldu;
  p.weight_f32 = c.weight_dtype == QFG_FLOAT;
  p.fp8 = c.fp8;
  p.trigger = c.trigger;
  p.give_up = c.give_up;
  p.rows = c.rows;
  p.n = static_cast<int>(c.n);
  p.offset = c.weight_offset;
  p.eps = c.eps;
  p.inv_n = 1.0f / static_cast<float>(c.n);
  cudaError_t err;
  switch (c.dtype) {
    case QFG_BFLOAT16: err = LaunchKind<__nv_bfloat16>(c, p, stream); break;
    case QFG_FLOAT16: err = LaunchKind<__half>(c, p, stream); break;
    case QFG_FLOAT: err = LaunchKind<float>(c, p, stream); break;
    default: return cudaErrorInvalidValue;
  }
  const cudaError_t last = cudaGetLastError();
  return err == cudaSuccess ? last : err;
}

}  // namespace qfg
