// Rows in eight bits with a scale each: of a root-mean-square norm, with the residual stream's addition; of a gated activation; of
// the rows themselves.
//
//   norm    h = x + residual, rounded to its type and kept; y_i = h_i rsqrt(mean(h^2) + eps) (offset + weight_i)
//   act     y_i = x_i / (1 + exp(-x_i)) u_i, or x_i
//   scale = max(max_i |y_i|, 2^-100) / top, q_i = y_i / scale rounded to the nearest (ties to even), top = 127 (INT8) or 448 (E4M3)
//
// All of it in FP32 until the one rounding to eight bits.  One pass over memory: the largest |h_i (offset + weight_i)| is found
// beside the sum of squares, because the norm's factor is the same for the whole row, and leaves q_i altogether, so a row needs one reduction and its
// values wait in registers.  Rows longer than the registers of a block of 1024 threads hold are read again.  A row whose sum of squares or largest
// value is no finite FP32 number has scale NaN and q 0.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "qfg_internal.h"
#include "stream_order.cuh"

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

// Four products f[i] * inv in eight bits.  INT8: adding 1.5 * 2^23 leaves the integer nearest to a product of at most 2^22 in the low
// bits, rounded once; |f| <= largest and inv = top / largest to within two ulp keep it within [-127, 127].
__device__ __forceinline__ uint32_t Quantise4(const float (&f)[4], float inv, bool fp8) {
  if (fp8) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0] * inv, f[1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2] * inv, f[3] * inv), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(fmaf(f[i], inv, 12582912.f));
  return __byte_perm(__byte_perm(v[0], v[1], 0x0040), __byte_perm(v[2], v[3], 0x0040), 0x5410);
}
template <int C>
__device__ __forceinline__ void StoreQuantised(uint8_t* p, const float (&f)[C], float inv, bool fp8, bool bad) {
  if constexpr (C == 1) {
    const float four[4] = {f[0], 0.f, 0.f, 0.f};
    *p = bad ? 0 : static_cast<uint8_t>(Quantise4(four, inv, fp8));
  } else {
    uint32_t w[C / 4];
#pragma unroll
    for (int i = 0; i < C / 4; ++i) {
      const float four[4] = {f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]};
      w[i] = bad ? 0u : Quantise4(four, inv, fp8);
    }
    if constexpr (C == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    }
  }
}

// a / (1 + exp(-a)), to 2^-21: exp(-a) as 2^hi (1 + lo ln 2), where hi + lo is -a log2 e to 2^-40 or so.  With the one rounded product
// hi for the exponent, the result is off by 2^-24 |a|, 2^-18 at 60.  Past 2^127 the quotient is zero.
__device__ __forceinline__ float Swish(float a) {
  const float b = fminf(fmaxf(a, -200.f), 200.f), hi = b * -1.44269504f, lo = fmaf(b, -1.44269504f, -hi) + b * -1.92596299e-8f;  // log2 e in two parts
  float e, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(hi));
  e *= fmaf(lo, 0.693147181f, 1.0f);
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return a * r;
}

// The part of a row's values that follows from the elements themselves, and what they add to the row's sum of squares.  With
// `keep`, the sum of the residual stream is stored to h.
template <int KIND, typename T, int C>
__device__ __forceinline__ void Values(float (&f)[C], const Piece<T, C>& x, const Piece<T, C>& second, const RowParams& p, const void* weight, int i, T* h,
                                       float& squares) {
#pragma unroll
  for (int e = 0; e < C; ++e) f[e] = ToFloat(x.v[e]);
  if constexpr (KIND == kSwish) {
#pragma unroll
    for (int e = 0; e < C; ++e) f[e] = Swish(f[e]) * ToFloat(second.v[e]);
  }
  if constexpr (KIND == kNormAdd) {
    Piece<T, C> sum;
#pragma unroll
    for (int e = 0; e < C; ++e) {
      sum.v[e] = FromFloat<T>(f[e] + ToFloat(second.v[e]));
      f[e] = ToFloat(sum.v[e]);
    }
    Store<T, C>(h + i, sum);
  }
  if constexpr (KIND >= kNorm) {
#pragma unroll
    for (int e = 0; e < C; ++e) squares = fmaf(f[e], f[e], squares);
    if (p.weight_f32) {
      const Piece<float, C> w = Load<float, C>(static_cast<const float*>(weight) + i);
#pragma unroll
      for (int e = 0; e < C; ++e) f[e] *= p.offset + w.v[e];
    } else {
      const Piece<T, C> w = Load<T, C>(static_cast<const T*>(weight) + i);
#pragma unroll
      for (int e = 0; e < C; ++e) f[e] *= p.offset + ToFloat(w.v[e]);
    }
  }
}

// The row's sum of squares and largest magnitude, for every thread of it.  Magnitudes are compared as the integers their bits are,
// in which a NaN is larger than any number.
__device__ __forceinline__ void Reduce(float& squares, uint32_t& largest, int warps, int warp_of_row, float* sums, uint32_t* tops, bool need_sum) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    if (need_sum) squares += __shfl_xor_sync(0xffffffffu, squares, d);
  }
  largest = __reduce_max_sync(0xffffffffu, largest);
  if (warps == 1) return;
  const int lane = threadIdx.x & 31;
  if (lane == 0) {
    sums[warp_of_row] = squares;
    tops[warp_of_row] = largest;
  }
  __syncthreads();
  // every warp adds the warps' sums in the same order
  squares = lane < warps ? sums[lane] : 0.f;
  largest = lane < warps ? tops[lane] : 0u;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    if (need_sum) squares += __shfl_xor_sync(0xffffffffu, squares, d);
  }
  largest = __reduce_max_sync(0xffffffffu, largest);
}

struct Scaling {
  float inv, scale;
  bool bad;
};
template <int KIND>
__device__ __forceinline__ Scaling ScaleOf(float squares, uint32_t largest, const RowParams& p) {
  const float top = p.fp8 ? 448.f : 127.f;
  Scaling s;
  s.bad = largest >= 0x7F800000u;
  float root = 1.f;
  if constexpr (KIND >= kNorm) {
    s.bad = s.bad || !(squares <= 3.4028234e38f);
    root = 1.f / sqrtf(fmaf(squares, p.inv_n, p.eps));
  }
  // (f root) / (max(largest root, tiny) / top) without rounding f root first
  const float most = fmaxf(__uint_as_float(largest) * root, kTiny);
  s.inv = root * (top / most);
  s.scale = s.bad ? __uint_as_float(0x7FFFFFFFu) : most / top;
  return s;
}

// V pieces of C elements a thread.  C > 1: pieces of 16 bytes; C = 1: rows that lie anywhere.  V = 0: rows read twice.
template <int KIND, typename T, int C, int V>
__global__ void __launch_bounds__(1024) RowQuantKernel(const RowParams p) {
  __shared__ float sums[2][8][32];
  __shared__ uint32_t tops[2][8][32];
  constexpr bool kTwo = KIND == kSwish || KIND == kNormAdd;
  GridDependencyWait();
  const T *const x = BehindWait(static_cast<const T*>(p.x)), *const second = BehindWait(static_cast<const T*>(p.second));
  const char* const weight = BehindWait(static_cast<const char*>(p.weight));
  const int warp = static_cast<int>(threadIdx.x) >> 5, row_of_block = warp / p.warps, warp_of_row = warp - row_of_block * p.warps;
  const int step = p.warps * 32 * C, first = (warp_of_row * 32 + (static_cast<int>(threadIdx.x) & 31)) * C;
  int turn = 0;
  for (long long r0 = static_cast<long long>(blockIdx.x) * p.rows_per_block; r0 < p.rows; r0 += static_cast<long long>(gridDim.x) * p.rows_per_block, turn ^= 1) {
    const long long row = r0 + row_of_block;
    const int n = row < p.rows ? p.n : 0;
    const T* const xr = x + row * p.ldx;
    const T* const sr = second + row * p.ld2;
    T* const hr = static_cast<T*>(p.h) + row * p.n;
    uint8_t* const qr = p.q + row * p.n;
    float squares = 0.f;
    uint32_t largest = 0;
    auto look = [&](const float(&f)[C]) {
#pragma unroll
      for (int e = 0; e < C; ++e) largest = max(largest, __float_as_uint(f[e]) & 0x7FFFFFFFu);
    };
    if constexpr (V > 0) {
      Piece<T, C> a[V], b[V];
      float f[V][C];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (first + j * step < n) {
          a[j] = Load<T, C>(xr + first + j * step);
          if constexpr (kTwo) b[j] = Load<T, C>(sr + first + j * step);
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (first + j * step < n) {
          Values<KIND, T, C>(f[j], a[j], b[j], p, weight, first + j * step, hr, squares);
          look(f[j]);
        }
      }
      Reduce(squares, largest, p.warps, warp_of_row, sums[turn][row_of_block], tops[turn][row_of_block], KIND >= kNorm);
      const Scaling s = ScaleOf<KIND>(squares, largest, p);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (first + j * step < n) StoreQuantised<C>(qr + first + j * step, f[j], s.inv, p.fp8, s.bad);
      }
      if (first < n && first == 0) p.scale[row] = s.scale;
    } else {
      float f[C];
      for (int i = first; i < n; i += step) {
        const Piece<T, C> a = Load<T, C>(xr + i);
        Values<KIND, T, C>(f, a, kTwo ? Load<T, C>(sr + i) : a, p, weight, i, hr, squares);
        look(f);
      }
      Reduce(squares, largest, p.warps, warp_of_row, sums[turn][row_of_block], tops[turn][row_of_block], KIND >= kNorm);
      const Scaling s = ScaleOf<KIND>(squares, largest, p);
      for (int i = first; i < n; i += step) {
        if constexpr (KIND == kNormAdd) {  // the sums that this thread has stored
          const Piece<T, C> a = Load<T, C>(hr + i);
          Values<kNorm, T, C>(f, a, a, p, weight, i, hr, squares);
        } else {
          const Piece<T, C> a = Load<T, C>(xr + i);
          Values<KIND, T, C>(f, a, kTwo ? Load<T, C>(sr + i) : a, p, weight, i, hr, squares);
        }
        StoreQuantised<C>(qr + i, f, s.inv, p.fp8, s.bad);
      }
      if (first < n && first == 0) p.scale[row] = s.scale;
    }
  }
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

template <int KIND, typename T, int C>
cudaError_t LaunchShape(RowParams& p, cudaStream_t stream) {
  const int sms = DeviceSmCount();
  const int pieces = (p.n + C - 1) / C;
  constexpr int kMost = C == 1 ? 16 : C == 4 ? 8 : 4;  // pieces that a thread holds at most
  // Few rows: as many threads a row as it has pieces.  Many: a few pieces a thread, so that the blocks of other rows hide a row's reduction.
  const bool few = p.rows <= 2 * sms;
  int warps = few ? (pieces + 31) / 32 : (pieces + 32 * kMost - 1) / (32 * kMost);
  warps = std::min(32, std::max(1, warps));
  const int v = (pieces + 32 * warps - 1) / (32 * warps);
  p.warps = warps;
  p.rows_per_block = few ? 1 : std::max(1, 4 / warps);
  const unsigned threads = static_cast<unsigned>(32 * warps * p.rows_per_block);
  const long long want = (p.rows + p.rows_per_block - 1) / p.rows_per_block, most = static_cast<long long>(sms) * std::max(1u, 2048 / threads);
  const unsigned blocks = static_cast<unsigned>(std::min(want, most));
  if (v <= 1) return Launch<KIND, T, C, 1>(p, blocks, threads, stream);
  if (v <= kMost / 2) return Launch<KIND, T, C, kMost / 2>(p, blocks, threads, stream);
  if (v <= kMost) return Launch<KIND, T, C, kMost>(p, blocks, threads, stream);
  return Launch<KIND, T, C, 0>(p, blocks, threads, stream);
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
