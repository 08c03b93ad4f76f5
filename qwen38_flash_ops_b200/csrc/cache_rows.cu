// What stands between a block's q / k / v projection and its attention, a head's row of one token at a time: the norm of query and key heads
// with the rotation by position, the write of keys and values into a cache of eight or four bits, and the read back.
//
//   norm      y_i = x_i rsqrt(mean(x^2) + eps) (offset + weight_i)                  (FP32 from here on)
//   rotation  (y_a, y_b) -> (y_a cos t - y_b sin t, y_b cos t + y_a sin t), t = position * frequency of the pair, for the pairs (i, i + R/2) or (2 i, 2 i + 1) of
//             the first R channels; with several axes each pair has one of the positions
//   E4M3      scale = max(max_i |y_i| / 448, 2^-40), q_i = y_i 448 / max_i |y_i| (where the scale is 2^-40 y_i / scale)   one for each token and head
//   NVFP4     scale = max(E4M3(max_i |y_i| / (6 unit)), 2^-9), q_i = E2M1(y_i / (scale unit))   one for each 16 channels
//
// An angle is a product of 64-bit integers: a pair's frequency in turns, as a fraction of 2^64, times the position, modulo 2^64, is the fraction of the turn to 2^-44
// for positions of a million; the sine and cosine of its first 32 bits are right to 2^-23 wherever the position is.  A product in FP32 is off by 2^-8 there.
// Quotients are rounded once: their factor is carried in two parts, so that half-way values go to even.
//
// A row has D / 16 lanes of sixteen channels each: of a rotated part in halves, eight of the one and the eight that they are rotated with, so that nothing crosses lanes
// but the sum of squares and the largest value, and the lanes of a load or a store fill whole sectors (with sixteen beside one another, the write of 2048 tokens of 8 heads
// and the reading of 10007 took 23.7 us instead of 18.6).  A token's sines and cosines are made once and wait in shared memory for all of its heads; weights do, too.
//
// Rows are fetched by asynchronous copies into a ring of each warp's own, four of its runs at a time: no register waits for them, and they are on their way while the angles
// are made (from registers, one run ahead, 38.5 us for the 35.4 below, and 286 bytes of them spilt).
//
// What bounds them: one read and one write of every head.  4096 tokens of 64 + 8 + 8 heads of 128, BF16, with an E4M3 cache: 35.4 us for 160 MB, 4.5 TB/s; of the issue slots
// two thirds are taken (the norm and the rotation in FP32 of 64 + 8 heads, whose weights are read from shared memory for each; without the cache, keys out instead, 31 us).  Four blocks an SM of 64 registers hide more than five with shorter rings (47 us), and than
// three of 80 did.  Sines and cosines read from shared memory at every row: 46.  Eight tokens: 4.8 us, the launch and one trip to memory: a row for each warp.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "qfg_internal.h"
#include "stream_order.cuh"

namespace qfg {
namespace {

constexpr int kThreads = 256;
constexpr int kMostTokens = 8;  // of a block, one for each warp

struct Side {  // queries, keys or values
  const void* x;
  long long ld;  // elements from token to token
  void* out;     // contiguous rows, or null
  const void* weight;
  int heads;
};
struct HeadsParams {
  Side side[3];
  const void* positions;
  long long ld_positions;
  const RotaryPair* pairs;
  const long long* slots;
  KvCacheView cache;
  int tokens, log_tokens, rotary;  // 2^log_tokens tokens a block; rotary: channels
  float rotary_scale, eps, offset;
  bool weight_f32, positions_64, interleaved;
};

template <typename T>
struct alignas(16) Eight {
  T v[8];
};
template <typename T, bool VEC>
__device__ __forceinline__ Eight<T> LoadEight(const T* p) {
  Eight<T> e;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(e) / 16); ++i) reinterpret_cast<uint4*>(&e)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e.v[i] = p[i];
  }
  return e;
}
template <typename T>
__device__ __forceinline__ float ToFloat(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ void ToFloats(float* f, const Eight<T>& e) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(&e)[i];
      f[2 * i] = __uint_as_float(w << 16);
      f[2 * i + 1] = __uint_as_float(w & 0xFFFF0000u);
    } else if constexpr (std::is_same_v<T, __half>) {
      const float2 two = __half22float2(reinterpret_cast<const __half2*>(&e)[i]);
      f[2 * i] = two.x;
      f[2 * i + 1] = two.y;
    } else {
      f[2 * i] = e.v[2 * i];
      f[2 * i + 1] = e.v[2 * i + 1];
    }
  }
}
template <typename T>
__device__ __forceinline__ void StoreEight(T* p, const float* f) {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      reinterpret_cast<__nv_bfloat162*>(&e)[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    } else if constexpr (std::is_same_v<T, __half>) {
      reinterpret_cast<__half2*>(&e)[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    } else {
      reinterpret_cast<float2*>(&e)[i] = make_float2(f[2 * i], f[2 * i + 1]);
    }
  }
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(e) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&e)[i];
}

// The larger magnitude of all lanes of a row, as the integer that its bits are: a NaN is larger than any number.
template <int L>
__device__ __forceinline__ uint32_t RowMax(uint32_t v) {
#pragma unroll
  for (int d = L / 2; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
// of eight values, the same; a NaN is kept
__device__ __forceinline__ uint32_t Magnitude(const float* f) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(f[2 * i]), "f"(f[2 * i + 1]));
  return __float_as_uint(m) & 0x7FFFFFFFu;
}
constexpr uint32_t kInfinity = 0x7F800000u;
constexpr float kLeastScale = 9.094947017729282e-13f;  // 2^-40

// top / by in two parts: v top / by = v hi + v lo, rounded once by the addition
struct Quotient {
  float hi, lo;
  __device__ Quotient(float top, float by) : hi(top / by) { lo = fmaf(-by, hi, top) * (hi / top); }
  __device__ float operator()(float v) const { return fmaf(v, hi, v * lo); }
};
__device__ __forceinline__ uint2 EightE4m3(const float* f, const Quotient& r, bool bad) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(r(f[2 * i]), r(f[2 * i + 1])), __NV_SATFINITE, __NV_E4M3);
  return bad ? make_uint2(0, 0) : make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
}
__device__ __forceinline__ uint32_t EightE2m1(const float* f, const Quotient& r, bool bad) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(make_float2(r(f[2 * i]), r(f[2 * i + 1])), __NV_E2M1, cudaRoundNearest)) << (8 * i);
  }
  return bad ? 0u : w;
}

__device__ __forceinline__ void Turn(float& a, float& b, float cosine, float sine) {
  const float u = a, v = b;
  a = u * cosine - v * sine;
  b = v * cosine + u * sine;
}
// two at a time
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

// A row's sixteen values of this lane, at channels c0 and c1 of eight each, into the cache.
template <int L>
__device__ __forceinline__ void StoreCache(const float (&f)[16], int c0, int c1, bool blocks_shared, const KvCacheView& cache, bool values, long long row, int lane,
                                           bool write) {
  uint8_t* const codes = values ? cache.v : cache.k;
  const uint32_t m0 = Magnitude(f), m1 = Magnitude(f + 8);
  constexpr int D = 16 * L;
  if (cache.fp4) {
    // a block of sixteen channels is this lane's, or eight of it are and the others the neighbour's
    const float unit = values ? cache.v_unit : cache.k_unit;
    const uint32_t n0 = __shfl_xor_sync(0xffffffffu, m0, 1), n1 = __shfl_xor_sync(0xffffffffu, m1, 1);
    uint32_t most[2];
    most[0] = max(m0, blocks_shared ? n0 : m1);
    most[1] = max(m1, blocks_shared ? n1 : m0);
    uint8_t* const scales = static_cast<uint8_t*>(values ? cache.v_scale : cache.k_scale) + row * L;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool bad = most[h] >= kInfinity;
      const int c = h == 0 ? c0 : c1;
      const __nv_fp8_storage_t coded = __nv_cvt_float_to_fp8(__uint_as_float(most[h]) / (6.f * unit), __NV_SATFINITE, __NV_E4M3);
      const uint32_t s = bad ? 0x7Fu : max(1u, static_cast<uint32_t>(coded));
      const float scale = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(s), __NV_E4M3))) * unit;
      const uint32_t w = EightE2m1(f + 8 * h, Quotient(1.f, scale), bad);
      if (write) {
        *reinterpret_cast<uint32_t*>(codes + row * (D / 2) + c / 2) = w;
        if ((c & 15) == 0) scales[c >> 4] = static_cast<uint8_t>(s);
      }
    }
  } else {
    const uint32_t most = RowMax<L>(max(m0, m1));
    const bool bad = most >= kInfinity;
    const float scale = __uint_as_float(most) / 448.f;
    const bool small = scale < kLeastScale;
    const Quotient r(small ? 1.f : 448.f, small ? kLeastScale : __uint_as_float(most));
    const uint2 a = EightE4m3(f, r, bad), b = EightE4m3(f + 8, r, bad);
    if (write) {
      *reinterpret_cast<uint2*>(codes + row * D + c0) = a;
      *reinterpret_cast<uint2*>(codes + row * D + c1) = b;
      if (lane == 0) static_cast<float*>(values ? cache.v_scale : cache.k_scale)[row] = bad ? __uint_as_float(0x7FFFFFFFu) : fmaxf(scale, kLeastScale);
    }
  }
}

// This lane's channels of rows of a side: eight from c0 and eight from c1.  Where it may be, those are eight of either half of what is rotated or of the row, so that
// the lanes of a load or a store take whole sectors.
struct Channels {
  int c0, c1;
  bool turned, split;  // rotated; eight of either half
};
template <int L, int WHICH>  // 0: queries, 1: keys, 2: values, 3: keys as they are
__device__ __forceinline__ Channels ChannelsOf(const HeadsParams& p, int lane) {
  Channels c;
  c.turned = WHICH < 2 && 16 * lane < p.rotary;
  c.split = WHICH >= 2 || (c.turned && !p.interleaved);
  c.c0 = c.split ? 8 * lane : 16 * lane;
  c.c1 = c.split ? (WHICH < 2 ? p.rotary / 2 : 8 * L) + 8 * lane : c.c0 + 8;
  return c;
}
// Rows on their way: of each warp kStages runs, a lane's two pieces where only it looks for them.
template <typename T>
struct Ring {
  static constexpr int kStages = sizeof(T) == 4 ? 2 : 4, kLane = 16 * sizeof(T), kBytes = kStages * kLane * 32;  // of a warp
};
template <typename T, bool VEC>
__device__ __forceinline__ void Fetch(uint8_t* slot, const T* a, const T* b) {  // the k-th 16 bytes of a lane's part 512 k bytes on
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const T* const from = h == 0 ? a : b;
    constexpr int kPieces = sizeof(T) / 2;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(slot + 512 * (kPieces * h + i)))),
                     "l"(from + 16 / sizeof(T) * i)
                     : "memory");
    } else {
      const Eight<T> e = LoadEight<T, false>(from);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) *reinterpret_cast<uint4*>(slot + 512 * (kPieces * h + i)) = reinterpret_cast<const uint4*>(&e)[i];
    }
  }
}
template <typename T>
__device__ __forceinline__ void Fetched(float (&f)[16], const uint8_t* slot) {
  constexpr int kPieces = sizeof(T) / 2;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      uint4& to = reinterpret_cast<uint4*>(&e)[i];
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(to.x), "=r"(to.y), "=r"(to.z), "=r"(to.w)
                   : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(slot + 512 * (kPieces * h + i))))
                   : "memory");
    }
    ToFloats(f + 8 * h, e);
  }
}

// A row of the queries (0), keys (1), values (2) or keys as they are (3).  Every lane of the warp is here, as shuffles are of whole warps; rows from `heads` on are not written.
template <typename T, int L, int WHICH>
__device__ __forceinline__ void Row(const HeadsParams& p, float (&f)[16], const Channels& c, const float (&cosine)[8], const float (&sine)[8], const float* weight,
                                    long long token, long long place, int row) {
  constexpr int D = 16 * L;
  const Side& s = p.side[WHICH == 3 ? 1 : WHICH];
  if (WHICH < 2 && s.weight != nullptr) {
    float2 squares = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < 16; e += 2) squares = Fma2(make_float2(f[e], f[e + 1]), make_float2(f[e], f[e + 1]), squares);
    float all = squares.x + squares.y;
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
    // squares that FP32 does not hold: the row is NaN, not 0 (taken nearer to 1 and made again, even behind the loop, the call is 4 to 6 % longer)
    const float square = fmaf(all, 1.f / D, p.eps);
    float root = rsqrtf(square);
    if (square == INFINITY) root = __int_as_float(0x7FFFFFFF);
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float4 w = *reinterpret_cast<const float4*>(weight + (e < 8 ? c.c0 + e : c.c1 + e - 8));
      const float2 by[2] = {Mul2(make_float2(root, root), make_float2(w.x, w.y)), Mul2(make_float2(root, root), make_float2(w.z, w.w))};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 y = Mul2(make_float2(f[e + 2 * i], f[e + 2 * i + 1]), by[i]);
        f[e + 2 * i] = y.x;
        f[e + 2 * i + 1] = y.y;
      }
    }
  }
  if (WHICH < 2 && c.turned) {
    if (p.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; ++e) Turn(f[2 * e], f[2 * e + 1], cosine[e], sine[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 a = make_float2(f[e], f[e + 1]), b = make_float2(f[8 + e], f[9 + e]), by = make_float2(cosine[e], cosine[e + 1]), in = make_float2(sine[e], sine[e + 1]);
        const float2 u = Fma2(make_float2(-b.x, -b.y), in, Mul2(a, by)), v = Fma2(a, in, Mul2(b, by));
        f[e] = u.x, f[e + 1] = u.y;
        f[8 + e] = v.x, f[9 + e] = v.y;
      }
    }
  }
  if (WHICH < 2 && row < s.heads && s.out != nullptr) {
    T* const out = static_cast<T*>(s.out) + (token * s.heads + row) * D;
    StoreEight<T>(out + c.c0, f);
    StoreEight<T>(out + c.c1, f + 8);
  }
  if (WHICH > 0 && p.slots != nullptr)
    StoreCache<L>(f, c.c0, c.c1, c.split, p.cache, WHICH == 2, place + static_cast<long long>(row) * p.cache.page, static_cast<int>(threadIdx.x) % L, row < s.heads && place >= 0);
}

// L lanes a row, D = 16 L.  QUERIES: false where keys and values alone are written, without a norm or a rotation.
template <typename T, int L, bool QUERIES>
constexpr int kHeadsBlocks = QUERIES && (sizeof(T) == 4 || L == 16) ? 3 : 4;  // of an SM
template <typename T, int L, bool VEC, bool QUERIES>
__global__ void __launch_bounds__(kThreads, kHeadsBlocks<T, L, QUERIES>) HeadsKernel(const HeadsParams p) {
  using R = Ring<T>;
  constexpr int D = 16 * L, kRows = 32 / L, kKeys = QUERIES ? 1 : 3;
  __shared__ __align__(16) uint8_t rings[kThreads / 32 * R::kBytes];
  __shared__ __align__(16) float2 turn[QUERIES ? kMostTokens * D / 2 : 1];
  __shared__ __align__(16) float weight[2][D];
  GridDependencyWait();
  // a token's warps, a power of two, take turns at its runs of rows, of queries, keys and values one after another; or every warp has one run
  const int warp = static_cast<int>(threadIdx.x) / 32, warps = kThreads / 32 >> p.log_tokens, t = warp * (1 << p.log_tokens) / (kThreads / 32), sub = warp & (warps - 1);
  const long long token = (static_cast<long long>(blockIdx.x) << p.log_tokens) + t;
  const bool real = token < p.tokens, turns = gridDim.y == 1;
  const int in_warp = static_cast<int>(threadIdx.x) & 31, in_run = in_warp / L, lane = in_warp % L, half = p.rotary / 2;
  const int q_runs = (p.side[0].heads + kRows - 1) / kRows, k_runs = q_runs + (p.side[1].heads + kRows - 1) / kRows, runs = k_runs + (p.side[2].heads + kRows - 1) / kRows;
  const int step = turns ? warps : 1 << 24;
  int run = turns ? sub : static_cast<int>(blockIdx.y) * (kThreads / 32) + warp;
  const Channels c = ChannelsOf<L, kKeys>(p, lane), as_they_are = ChannelsOf<L, 2>(p, lane);
  uint8_t* const ring = rings + warp * R::kBytes + in_warp * 16;
  const auto issue = [&](int of, int stage) {
    if (of < runs && real) {
      const int which = of < q_runs ? 0 : of < k_runs ? 1 : 2, row = (of - (which == 0 ? 0 : which == 1 ? q_runs : k_runs)) * kRows + in_run;
      const Side& s = p.side[which];
      const Channels& at = which == 2 ? as_they_are : c;
      const T* const x = static_cast<const T*>(s.x) + token * s.ld + row * D;
      if (row < s.heads) Fetch<T, VEC>(ring + stage * (R::kLane * 32), x + at.c0, x + at.c1);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < R::kStages; ++i) issue(run + i * step, i);

  for (int i = threadIdx.x; QUERIES && i < 2 * D; i += kThreads) {
    const void* const w = p.side[i / D].weight;
    if (w != nullptr) weight[i / D][i % D] = p.offset + (p.weight_f32 ? static_cast<const float*>(w)[i % D] : ToFloat(static_cast<const T*>(w)[i % D]));
  }
  float2* const by = turn + t * half;
  long long to = -1;  // (page, row of it) as page * kv_heads * page size + row; < 0: not written
  if (real) {
    for (int j = sub * 32 + in_warp; QUERIES && j < half; j += 32 * warps) {
      const RotaryPair pair = p.pairs[j];
      const long long at = token + pair.axis * p.ld_positions;
      const long long position = p.positions_64 ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
      const unsigned long long part = static_cast<unsigned long long>(position) * pair.turns;
      float s, c;
      sincospif(static_cast<float>(static_cast<int>(part >> 32)) * 4.656612873077393e-10f, &s, &c);  // 2^-31
      by[j] = make_float2(c * p.rotary_scale, s * p.rotary_scale);
    }
    if (p.slots != nullptr) {
      const long long slot = p.slots[token], page = slot >> 32 ? slot / p.cache.page : static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.cache.page);
      to = slot >= 0 && page < p.cache.pages ? page * p.cache.heads * p.cache.page + (slot - page * p.cache.page) : -1;
    }
  }
  if constexpr (QUERIES) __syncthreads();
  if (!real) return;
  float cosine[8], sine[8];  // of this lane's eight pairs
  if (c.turned) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float4 two = *reinterpret_cast<const float4*>(by + 8 * lane + e);
      cosine[e] = two.x, sine[e] = two.y;
      cosine[e + 1] = two.z, sine[e + 1] = two.w;
    }
  }
  int stage = 0;
#pragma unroll 1
  for (; run < runs; run += step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(R::kStages - 1) : "memory");
    float f[16];
    Fetched<T>(f, ring + stage * (R::kLane * 32));
    issue(run + R::kStages * step, stage);
    if (++stage == R::kStages) stage = 0;
    if (QUERIES && run < q_runs) {
      Row<T, L, 0>(p, f, c, cosine, sine, weight[0], token, to, run * kRows + in_run);
    } else if (run < k_runs) {
      Row<T, L, kKeys>(p, f, c, cosine, sine, weight[1], token, to, (run - q_runs) * kRows + in_run);
    } else {
      Row<T, L, 2>(p, f, as_they_are, cosine, sine, nullptr, token, to, (run - k_runs) * kRows + in_run);
    }
  }
}

template <typename T, int L>
cudaError_t LaunchHeads(HeadsParams& p, bool vec, cudaStream_t stream) {
  // Few tokens: one a block, its rows over as many blocks as leave every warp one run of them.  More: as few tokens a block as let the GPU hold all blocks at once, but two
  // where warps would have nothing else; of more tokens than that up to eight, as long as a warp has no more than sixteen runs.  64 + 8 + 8 heads of 128, us of 1, 2, 4, 8
  // tokens a block: 1024 of them - / 12.5 / 12.8 / 16.8, 2048 - / - / 20.2 / 21.5; 24 + 4 + 4 of 256, 1024 of them - / 13.3 / 11.2 / 13.6.
  constexpr int kRows = 32 / L, kWarps = kThreads / 32;
  int runs = 0;
  for (const Side& s : p.side) runs += (s.heads + kRows - 1) / kRows;
  const int sms = DeviceSmCount();
  const bool few = p.tokens <= 2 * sms;
  p.log_tokens = 0;
  const int slots = sms * (p.side[0].heads > 0 ? kHeadsBlocks<T, L, true> : kHeadsBlocks<T, L, false>);
  const auto blocks = [&](int log) { return (p.tokens - 1 >> log) + 1; };
  while (!few && 1 << p.log_tokens < kMostTokens &&
         ((blocks(p.log_tokens) > slots && runs << p.log_tokens < 16 * kWarps) || (runs << p.log_tokens < kWarps && blocks(p.log_tokens + 1) >= sms))) {
    ++p.log_tokens;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks(p.log_tokens)), static_cast<unsigned>(few ? (runs + kWarps - 1) / kWarps : 1));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {OverlapAttribute()};
  cfg.attrs = attr;
  cfg.numAttrs = MayOverlapPredecessor(stream) ? 1 : 0;
  if (p.side[0].heads > 0) return vec ? cudaLaunchKernelEx(&cfg, HeadsKernel<T, L, true, true>, p) : cudaLaunchKernelEx(&cfg, HeadsKernel<T, L, false, true>, p);
  return vec ? cudaLaunchKernelEx(&cfg, HeadsKernel<T, L, true, false>, p) : cudaLaunchKernelEx(&cfg, HeadsKernel<T, L, false, false>, p);
}

template <typename T>
cudaError_t LaunchHeadsOf(int dim, HeadsParams& p, bool vec, cudaStream_t stream) {
  switch (dim) {
    case 64: return LaunchHeads<T, 4>(p, vec, stream);
    case 128: return LaunchHeads<T, 8>(p, vec, stream);
    case 256: return LaunchHeads<T, 16>(p, vec, stream);
    default: return cudaErrorInvalidValue;
  }
}

// ------------------------------------------------------------------------------ the way back
struct ReadParams {
  KvCacheView cache;
  const int* table;
  const int* offsets;
  void *k_out, *v_out;
  long long ld_table, rows;
  int seqs, most_pages;
};
// Tokens of a block.  10007 tokens of 8 heads of 128, NVFP4 to BF16 (53 MB, a floor of 8.1 us): 10 of the 17.4 us with a write ahead of it; with blocks of 32 tokens 3 more.
constexpr int kReadRows = 16;

template <typename T, int L, bool FP4>
__global__ void __launch_bounds__(kThreads) CacheReadKernel(const ReadParams p) {
  constexpr int D = 16 * L;
  __shared__ long long place[kReadRows];  // -2: a row of no sequence; -1: one that no page holds
  GridDependencyWait();
  const long long row0 = static_cast<long long>(blockIdx.x) * kReadRows;
  if (threadIdx.x < kReadRows) {
    const long long row = row0 + threadIdx.x;
    long long at = -2;
    if (row < p.rows && row >= p.offsets[0] && row < p.offsets[p.seqs]) {
      int lo = 0, hi = p.seqs;  // the last sequence that begins at this row or ahead of it
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        (p.offsets[mid] <= row ? lo : hi) = mid;
      }
      const long long in = row - p.offsets[lo], room = static_cast<long long>(p.most_pages) * p.cache.page;  // an offset may be as far below 0 as an integer can
      at = -1;
      if (in < room) {  // and so within 32 bits
        const int page = static_cast<int>(in) / p.cache.page, id = p.table[lo * p.ld_table + page];
        if (id >= 0 && id < p.cache.pages) at = static_cast<long long>(id) * p.cache.heads * p.cache.page + (static_cast<int>(in) - page * p.cache.page);
      }
    }
    place[threadIdx.x] = at;
  }
  __syncthreads();
  // A warp takes a head's keys, or values: rows that lie beside one another in the cache, L lanes each, all of whose codes are on their way together.
  constexpr int kAtOnce = 32 / L, kSteps = kReadRows / kAtOnce, kAhead = kSteps < 4 ? kSteps : 4;
  const int warp = static_cast<int>(threadIdx.x) / 32, in_warp = static_cast<int>(threadIdx.x) & 31, lane = in_warp % L;
  for (int side = warp; side < 2 * p.cache.heads; side += kThreads / 32) {
    const bool values = side >= p.cache.heads;
    const int head = values ? side - p.cache.heads : side;
    const long long base = static_cast<long long>(head) * p.cache.page;
    const uint8_t* const codes = values ? p.cache.v : p.cache.k;
    const uint8_t* const scales = static_cast<const uint8_t*>(values ? p.cache.v_scale : p.cache.k_scale);
    const float unit = values ? p.cache.v_unit : p.cache.k_unit;
    // eight channels of either half of the row, so that the lanes of a store fill whole sectors
    T* const out = static_cast<T*>(values ? p.v_out : p.k_out) + (row0 * p.cache.heads + head) * D + lane * 8;
#pragma unroll
    for (int first = 0; first < kSteps; first += kAhead) {
      uint4 w[kAhead];
      float scale[kAhead][2];
      long long at[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        at[i] = place[(first + i) * kAtOnce + in_warp / L];
        w[i] = make_uint4(0, 0, 0, 0);
        scale[i][0] = scale[i][1] = 0.f;
        if (at[i] < 0) continue;
        const long long row = at[i] + base;
        if constexpr (FP4) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            (h == 0 ? w[i].x : w[i].z) = *reinterpret_cast<const uint32_t*>(codes + row * (D / 2) + h * (D / 4) + lane * 4);
            scale[i][h] = __half2float(__half(__nv_cvt_fp8_to_halfraw(scales[row * L + h * (L / 2) + lane / 2], __NV_E4M3))) * unit;
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint2 two = *reinterpret_cast<const uint2*>(codes + row * D + h * (D / 2) + lane * 8);
            (h == 0 ? w[i].x : w[i].z) = two.x, (h == 0 ? w[i].y : w[i].w) = two.y;
          }
          scale[i][0] = scale[i][1] = reinterpret_cast<const float*>(scales)[row];
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (at[i] == -2) continue;
        float f[16];
        const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          __half2_raw h;
          if constexpr (FP4) {
            h = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(words[e >> 2 << 1] >> (8 * (e & 3))), __NV_E2M1);
          } else {
            h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(words[e >> 1] >> (16 * (e & 1))), __NV_E4M3);
          }
          const float2 v = __half22float2(__half2(h));
          f[2 * e] = v.x * scale[i][e >> 2];
          f[2 * e + 1] = v.y * scale[i][e >> 2];
        }
        T* const to = out + static_cast<long long>((first + i) * kAtOnce + in_warp / L) * p.cache.heads * D;
        StoreEight<T>(to, f);
        StoreEight<T>(to + D / 2, f + 8);
      }
    }
  }
}

template <typename T>
cudaError_t LaunchReadOf(int dim, const ReadParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.rows + kReadRows - 1) / kReadRows));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {OverlapAttribute()};
  cfg.attrs = attr;
  cfg.numAttrs = MayOverlapPredecessor(stream) ? 1 : 0;
  switch (dim) {
    case 64: return p.cache.fp4 ? cudaLaunchKernelEx(&cfg, CacheReadKernel<T, 4, true>, p) : cudaLaunchKernelEx(&cfg, CacheReadKernel<T, 4, false>, p);
    case 128: return p.cache.fp4 ? cudaLaunchKernelEx(&cfg, CacheReadKernel<T, 8, true>, p) : cudaLaunchKernelEx(&cfg, CacheReadKernel<T, 8, false>, p);
    case 256: return p.cache.fp4 ? cudaLaunchKernelEx(&cfg, CacheReadKernel<T, 16, true>, p) : cudaLaunchKernelEx(&cfg, CacheReadKernel<T, 16, false>, p);
    default: return cudaErrorInvalidValue;
  }
}

size_t BytesOf(int dtype) { return dtype == QFG_FLOAT ? 4 : 2; }
bool Vectors(const void* x, long long ld, int dtype) { return reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld * BytesOf(dtype) % 16 == 0; }

cudaError_t Ended(cudaError_t err) {
  const cudaError_t last = cudaGetLastError();
  return err == cudaSuccess ? last : err;
}

}  // namespace

cudaError_t LaunchHeadRows(const HeadsCall& c, cudaStream_t stream) {
  if (c.tokens == 0) return cudaSuccess;
  HeadsParams p = {};
  p.side[0] = {c.q, c.ldq, c.q_out, c.q_weight, c.q != nullptr ? c.q_heads : 0};
  p.side[1] = {c.k, c.ldk, c.k_out, c.k_weight, c.kv_heads};
  p.side[2] = {c.v, c.ldv, nullptr, nullptr, c.slots != nullptr ? c.kv_heads : 0};
  bool vec = true;  // everything on 16 bytes
  for (const Side& s : p.side) vec = vec && Vectors(s.x, s.ld, c.dtype) && Vectors(s.weight, 0, c.dtype);
  p.positions = c.positions;
  p.ld_positions = c.ld_positions;
  p.positions_64 = c.positions_64;
  p.pairs = c.pairs;
  p.rotary = 2 * c.n_pairs;
  p.interleaved = c.interleaved;
  p.rotary_scale = c.rotary_scale;
  p.eps = c.eps;
  p.offset = c.weight_offset;
  p.weight_f32 = c.weight_dtype == QFG_FLOAT;
  p.slots = reinterpret_cast<const long long*>(c.slots);
  p.cache = c.cache;
  p.tokens = static_cast<int>(c.tokens);
  cudaError_t err;
  switch (c.dtype) {
    case QFG_BFLOAT16: err = LaunchHeadsOf<__nv_bfloat16>(c.dim, p, vec, stream); break;
    case QFG_FLOAT16: err = LaunchHeadsOf<__half>(c.dim, p, vec, stream); break;
    case QFG_FLOAT: err = LaunchHeadsOf<float>(c.dim, p, vec, stream); break;
    default: return cudaErrorInvalidValue;
  }
  return Ended(err);
}

cudaError_t LaunchCacheRead(const CacheReadCall& c, cudaStream_t stream) {
  if (c.rows == 0 || c.seqs == 0) return cudaSuccess;
  ReadParams p = {};
  p.cache = c.cache;
  p.table = c.table;
  p.ld_table = c.ld_table;
  p.offsets = c.offsets;
  p.seqs = c.seqs;
  p.most_pages = c.most_pages;
  p.rows = c.rows;
  p.k_out = c.k_out;
  p.v_out = c.v_out;
  cudaError_t err;
  switch (c.dtype) {
    case QFG_BFLOAT16: err = LaunchReadOf<__nv_bfloat16>(c.cache.dim, p, stream); break;
    case QFG_FLOAT16: err = LaunchReadOf<__half>(c.cache.dim, p, stream); break;
    case QFG_FLOAT: err = LaunchReadOf<float>(c.cache.dim, p, stream); break;
    default: return cudaErrorInvalidValue;
  }
  return Ended(err);
}

}  // namespace qfg
