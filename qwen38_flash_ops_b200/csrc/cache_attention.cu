// Attention of the last few tokens of each sequence over a paged cache of four or eight bits.
//
//   s_rt = scale q_r . k_t,  t < length - tokens + 1 + (token of r);   y_r = sum_t exp(s_rt - m_r) v_t / sum_t exp(s_rt - m_r)
//
// The rows of one key head (its query heads, times the tokens) share every key and value that is read, so what bounds the kernel is the cache's bytes, 9/16 of one a
// value in four bits, and then the instructions that unpack them.  Products are warp matrix instructions with the cache as the large operand, sixteen tokens (keys) or
// sixteen channels (values) by eight rows: unpacked codes go from registers straight into them, each once for eight rows, and a tile of rows that is not full wastes
// nothing of the unpacking.
//
//   keys     S^T = K q^T.  A lane holds a quarter of the channels of two tokens; channels are taken in the order in which they lie in memory, by q as well.
//   values   O^T = V^T P^T.  A lane holds D / 8 channels of four tokens of each sixteen; pairs of tokens are made by byte permutations.  P^T is S^T's layout transposed.
//   scales   four bits: the product of an E2M1 value and an E4M3 scale has at most six significant bits and is exact in FP16.  Eight bits: the keys' scale multiplies the
//            score, the values' the weight.
//   q        as FP16, each row times the power of two that takes its largest value to 2^9, so that only what is 2^-23 of that is rounded.
//
// Softmax runs along: m is taken up only when a score passes it by 8 (in powers of two), so that sums and weights stay within 2^8 of what they would be and the outputs
// are seldom scaled again.  Statistics and sums are FP32, weights FP16 (2^-11 of themselves, as the values are exact).
//
// A warp has its own ring of tiles in shared memory, which it fills by bulk copies, and its own sums; no warp waits for another before the end of a unit.  A unit is a run
// of tiles of one sequence for one key head; sequences are cut so that units are of nearly one size, by their lengths, which only the device knows.  A second kernel joins
// the parts of the sequences that were cut, in their order, so that results do not depend on which block is first.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "qfg_internal.h"
#include "stream_order.cuh"
#include "tc_ptx.cuh"

namespace qfg {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kLeastTiles = kWarps;  // of a unit: a tile a warp

struct AttendParams {
  KvCacheView cache;
  const void* q;
  const int *table, *lengths;
  float* partial;
  void* out;
  float* lse;
  long long ld_seq, ld_token, ld_table;
  int seqs, tokens, q_heads, group, most_pages, row_blocks, target_units;
  float scale;  // of scores, in powers of two, with the keys' unit
  bool bf16, give_up;
};

template <int D, bool FP4>
struct Geometry {
  static constexpr int kCodes = FP4 ? D / 2 : D, kScales = FP4 ? D / 16 : 4;  // bytes of a row
  static constexpr int kTile = (kCodes + kScales) * 64 <= 9000 ? 32 : 16;     // tokens
  static constexpr int kPart = kTile * (kCodes + kScales);                    // keys or values of a tile
  static constexpr int kStage = 2 * kPart;
  static constexpr int kStages = std::min(8, 220 * 1024 / 2 / (kWarps * kStage) >= 2 ? 220 * 1024 / 2 / (kWarps * kStage) : 220 * 1024 / (kWarps * kStage));
  static constexpr int kBytes = kWarps * kStages * kStage;
};

struct AttendCtl {
  unsigned long long full[kWarps][8];
  float most[kWarps][16], sum[kWarps][16];
  int scan[kWarps];
  long long total[kWarps];
  volatile uint32_t fault;
};

// How the sequences are cut: into pieces of `tiles` tiles; `first` is the number of pieces of the sequences ahead.
struct Cut {
  int seq, first, tiles, pieces;
};
__device__ __forceinline__ int TilesOf(const AttendParams& p, int seq, int tile, int* length) {
  const long long room = static_cast<long long>(p.most_pages) * p.cache.page;
  *length = static_cast<int>(min(static_cast<long long>(max(p.lengths[seq], 0)), room));
  return (*length + tile - 1) / tile;
}
// Of the sequence that holds piece `piece` (or of sequence `seq`, where it is not negative), for every thread of the block; seq is -1 where there is none.
template <int THREADS>
__device__ Cut FindCut(const AttendParams& p, int tile, int piece, int seq) {
  constexpr int kW = THREADS / 32;
  __shared__ long long total[kW];
  __shared__ int sums[kW];
  __shared__ Cut found;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int length;
  long long mine = 0;
  for (int i = threadIdx.x; i < p.seqs; i += THREADS) mine += TilesOf(p, i, tile, &length);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  if (lane == 0) total[warp] = mine;
  if (threadIdx.x == 0) found = {-1, 0, 0, 0};
  __syncthreads();
  long long all = 0;
#pragma unroll
  for (int i = 0; i < kW; ++i) all += total[i];
  const long long units = all * p.cache.heads * p.row_blocks;
  const int most = static_cast<int>(max(static_cast<long long>(kLeastTiles), (units + p.target_units - 1) / p.target_units));
  int before = 0;
  for (int base = 0; base < p.seqs; base += THREADS) {
    const int i = base + static_cast<int>(threadIdx.x);
    const int tiles = i < p.seqs ? TilesOf(p, i, tile, &length) : 0;
    const int pieces = i < p.seqs ? max(1, (tiles + most - 1) / most) : 0;
    int upto = pieces;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int ahead = before;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      if (w < warp) ahead += sums[w];
      before += sums[w];
    }
    const int begin = ahead + upto - pieces;
    // pieces of one sequence are of one size, to a tile
    if (i < p.seqs && (seq >= 0 ? i == seq : piece >= begin && piece < begin + pieces)) found = {i, begin, (tiles + pieces - 1) / pieces, pieces};
  }
  __syncthreads();
  return found;
}

__device__ __forceinline__ void Mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t Transposed(uint32_t v) {  // 8 x 8 of 16 bits
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float Exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float Log2(float v) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ uint32_t Mul16(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t Pack16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// eight E2M1 values, two of a byte in a register
__device__ __forceinline__ void FromE2m1(uint32_t c, uint32_t* r) {
  asm("{ .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %4;\n cvt.rn.f16x2.e2m1x2 %0, b0;\n cvt.rn.f16x2.e2m1x2 %1, b1;\n"
      " cvt.rn.f16x2.e2m1x2 %2, b2;\n cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(c));
}
// four E4M3 values
__device__ __forceinline__ void FromE4m3(uint32_t c, uint32_t* r) {
  asm("{ .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %2;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n cvt.rn.f16x2.e4m3x2 %1, hi;\n}" : "=r"(r[0]), "=r"(r[1]) : "r"(c));
}
template <int BYTES>
__device__ __forceinline__ void LoadShared(uint32_t a, uint32_t* v) {
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[4 * i]), "=r"(v[4 * i + 1]), "=r"(v[4 * i + 2]), "=r"(v[4 * i + 3]) : "r"(a + 16 * i));
  } else if constexpr (BYTES == 8) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a));
  } else if constexpr (BYTES == 4) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(a));
  } else if constexpr (BYTES == 2) {
    uint16_t h;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(a));
    v[0] = h;
  } else {
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v[0]) : "r"(a));
  }
}

// NT tiles of eight rows.
template <int D, bool FP4, int NT>
__global__ void __launch_bounds__(kThreads, D * NT <= 128 ? 2 : 1) CacheAttentionKernel(const AttendParams p) {
  using G = Geometry<D, FP4>;
  constexpr int kRows = 8 * NT, kSteps = D / 16, kGroups = G::kTile / 16;
  constexpr int kKeyBytes = G::kCodes / 4, kValueBytes = G::kCodes / 8;  // of a lane's part of a row
  constexpr int kKeyScales = FP4 ? D / 64 : 1;                           // E4M3 scales of that part
  constexpr int kValueChannels = D / 8, kTilesOfO = D / 16;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ AttendCtl ctl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < G::kStages; ++i) BarInit(Smem(&ctl.full[warp][i]), 1);
    if (warp == 0) ctl.fault = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  GridDependencyWait();
  const int heads = p.cache.heads, per_piece = heads * p.row_blocks;
  const Cut cut = FindCut<kThreads>(p, G::kTile, static_cast<int>(blockIdx.x) / per_piece, -1);  // its barriers: the ring's exist for all
  if (cut.seq < 0) return;
  const int in_piece = static_cast<int>(blockIdx.x) % per_piece, head = in_piece / p.row_blocks, row0 = in_piece % p.row_blocks * kRows;
  const int piece = static_cast<int>(blockIdx.x) / per_piece - cut.first, rows = min(kRows, p.tokens * p.group - row0);
  int length;
  const int tiles = TilesOf(p, cut.seq, G::kTile, &length);
  const int tile0 = piece * cut.tiles, tile1 = min(tiles, tile0 + cut.tiles);

  // q, and the factor from a row's products to its scores
  uint32_t q[NT][kSteps][2];
  float factor[NT][2];
  int sees[NT][2];  // tokens that a row may look at
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = row0 + 8 * n + g, token = row / p.group, of = head * p.group + row - token * p.group;
    const bool real = 8 * n + g < rows;
    const uint16_t* const at = static_cast<const uint16_t*>(p.q) + (real ? cut.seq * p.ld_seq + token * p.ld_token + static_cast<long long>(of) * D + c * (D / 4) : 0);
    uint32_t raw[kSteps][2];
    float most = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint2 w = real ? *reinterpret_cast<const uint2*>(at + 4 * s) : make_uint2(0, 0);
      raw[s][0] = w.x, raw[s][1] = w.y;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 v = p.bf16 ? make_float2(__uint_as_float(raw[s][e] << 16), __uint_as_float(raw[s][e] & 0xFFFF0000u)) : __half22float2(*reinterpret_cast<__half2*>(&raw[s][e]));
        most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^(9 - exponent) and its inverse; the exponent is kept where both are ordinary numbers
    const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23), 20), 240);
    const float up = __uint_as_float(static_cast<uint32_t>(263 - e) << 23), down = __uint_as_float(static_cast<uint32_t>(e - 9) << 23);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 v = p.bf16 ? make_float2(__uint_as_float(raw[s][h] << 16), __uint_as_float(raw[s][h] & 0xFFFF0000u)) : __half22float2(*reinterpret_cast<__half2*>(&raw[s][h]));
        q[n][s][h] = Pack16(v.x * up, v.y * up);
      }
    }
    const int see = length - p.tokens + 1 + token;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      factor[n][h] = __shfl_sync(0xffffffffu, down, (2 * c + h) * 4) * p.scale;
      sees[n][h] = __shfl_sync(0xffffffffu, see, (2 * c + h) * 4);
    }
  }
  const int least_seen = length - p.tokens + 1;

  // ---- this warp's tiles: tile0 + warp, kWarps further, ...
  const int count = tile0 + warp < tile1 ? (tile1 - tile0 - warp + kWarps - 1) / kWarps : 0;
  const uint32_t ring = Smem(smem) + static_cast<uint32_t>(warp * G::kStages * G::kStage), bars = Smem(&ctl.full[warp][0]);
  const int* const table = p.table + cut.seq * p.ld_table;
  int ids = 0;              // lane i: the page of tile (i mod 32) of this warp
  uint32_t present = 0;     // bit i mod 32: that page is one of the cache
  bool good = !p.give_up;
  auto issue = [&](int i) {
    const int at = tile0 + warp + i * kWarps;  // of the sequence
    if ((i & 31) == 0) {
      const int mine = at + lane * kWarps;
      ids = mine < tile1 ? table[static_cast<long long>(mine) * G::kTile / p.cache.page] : 0;
    }
    const int id = __shfl_sync(0xffffffffu, ids, i & 31);
    const bool is = id >= 0 && id < p.cache.pages;
    present = (present & ~(1u << (i & 31))) | (is ? 1u << (i & 31) : 0u);
    if (lane == 0) {
      const long long row = (static_cast<long long>(is ? id : 0) * heads + head) * p.cache.page + at * G::kTile % p.cache.page;
      const uint32_t to = ring + static_cast<uint32_t>(i % G::kStages * G::kStage), bar = bars + i % G::kStages * 8;
      BarExpect(bar, G::kStage);
      BulkLoad(to, p.cache.k + row * G::kCodes, G::kTile * G::kCodes, bar);
      BulkLoad(to + G::kTile * G::kCodes, static_cast<const uint8_t*>(p.cache.k_scale) + row * G::kScales, G::kTile * G::kScales, bar);
      BulkLoad(to + G::kPart, p.cache.v + row * G::kCodes, G::kTile * G::kCodes, bar);
      BulkLoad(to + G::kPart + G::kTile * G::kCodes, static_cast<const uint8_t*>(p.cache.v_scale) + row * G::kScales, G::kTile * G::kScales, bar);
    }
  };
  if (good) {
    for (int i = 0; i < min(count, G::kStages); ++i) issue(i);
  }

  float o[NT][kTilesOfO][4];
  float most[NT][2], sum[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) most[n][h] = -INFINITY, sum[n][h] = 0.f;
#pragma unroll
    for (int m = 0; m < kTilesOfO; ++m) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][m][e] = 0.f;
    }
  }

  for (int i = 0; i < count && good; ++i) {
    const uint32_t at = ring + static_cast<uint32_t>(i % G::kStages * G::kStage);
    if (!BarWait(bars + i % G::kStages * 8, static_cast<uint32_t>(i / G::kStages & 1), ctl)) {
      good = false;
      break;
    }
    const int token0 = (tile0 + warp + i * kWarps) * G::kTile;
    const bool absent = !(present >> (i & 31) & 1);
    const bool whole = token0 + G::kTile <= least_seen && !absent;  // no row leaves any token of it out
    // ---- scores
    float s[kGroups][NT][4];
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][n][e] = 0.f;
      }
      uint32_t raw[2][kKeyBytes / 4], scale[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t token = static_cast<uint32_t>(16 * u + 8 * h + g);
        LoadShared<kKeyBytes>(at + token * G::kCodes + c * kKeyBytes, raw[h]);
        if constexpr (FP4) LoadShared<kKeyScales>(at + G::kTile * G::kCodes + token * G::kScales + c * kKeyScales, &scale[h]);
      }
      if constexpr (FP4) {
        uint32_t by[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) FromE4m3(scale[h], by[h]);  // pairs of scales; four at most
#pragma unroll
        for (int j = 0; j < kKeyBytes / 4; ++j) {
          uint32_t v[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int b = j / 2;  // the block of sixteen channels
            const uint32_t both = __byte_perm(by[h][b >> 1], 0, b & 1 ? 0x3232 : 0x1010);
            FromE2m1(raw[h][j], v[h]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[h][e] = Mul16(v[h][e], both);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a[4] = {v[0][2 * e], v[1][2 * e], v[0][2 * e + 1], v[1][2 * e + 1]};
#pragma unroll
            for (int n = 0; n < NT; ++n) Mma(s[u][n], a, q[n][2 * j + e][0], q[n][2 * j + e][1]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kKeyBytes / 4; ++j) {
          uint32_t v[2][2];
#pragma unroll
          for (int h = 0; h < 2; ++h) FromE4m3(raw[h][j], v[h]);
          const uint32_t a[4] = {v[0][0], v[1][0], v[0][1], v[1][1]};
#pragma unroll
          for (int n = 0; n < NT; ++n) Mma(s[u][n], a, q[n][j][0], q[n][j][1]);
        }
      }
    }
    // ---- weights.  s[u][n][2 h + r] is token 16 u + 8 h + g, row 8 n + 2 c + r.
    float value_scale[kGroups][2];
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t token = static_cast<uint32_t>(16 * u + 8 * h + g);
        float key_scale = 1.f;
        value_scale[u][h] = 1.f;
        if constexpr (!FP4) {
          LoadShared<4>(at + G::kTile * G::kCodes + token * 4, reinterpret_cast<uint32_t*>(&key_scale));
          LoadShared<4>(at + G::kPart + G::kTile * G::kCodes + token * 4, reinterpret_cast<uint32_t*>(&value_scale[u][h]));
          if (token0 + static_cast<int>(token) >= length || absent) value_scale[u][h] = 1.f;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float& v = s[u][n][2 * h + r];
            v *= FP4 ? factor[n][r] : factor[n][r] * key_scale;
            if (!whole && (token0 + static_cast<int>(token) >= sees[n][r] || absent)) v = -INFINITY;
          }
        }
      }
    }
    // what a score may be at most without its weight, times the value's scale, passing 2^8
    bool higher = false;
    float upto[NT][2];
    float log_scale[kGroups][2];
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) log_scale[u][h] = FP4 ? 0.f : fminf(fmaxf(Log2(value_scale[u][h]), -60.f), 60.f);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float m = s[0][n][r] + log_scale[0][0];
#pragma unroll
        for (int u = 0; u < kGroups; ++u) {
#pragma unroll
          for (int h = 0; h < 2; ++h) m = fmaxf(m, s[u][n][2 * h + r] + log_scale[u][h]);
        }
        upto[n][r] = m;
        higher = higher || m > most[n][r] + 8.f;
      }
    }
    if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float m = upto[n][r];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          m = fmaxf(m, most[n][r]);
          const float by = m == -INFINITY ? 1.f : Exp2(most[n][r] - m);
          most[n][r] = m;
          sum[n][r] *= by;
#pragma unroll
          for (int t = 0; t < kTilesOfO; ++t) {
            o[n][t][r] *= by;
            o[n][t][2 + r] *= by;
          }
        }
      }
    }
    uint32_t weights[kGroups][NT][2];  // tokens 2 c, 2 c + 1 (and eight on) of the sixteen, row 8 n + g
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float from = most[n][e & 1];
          const float v = Exp2(s[u][n][e] - (from == -INFINITY ? 0.f : from));
          sum[n][e & 1] += v;
          w[e] = FP4 ? v : v * value_scale[u][e >> 1];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) weights[u][n][h] = Transposed(Pack16(w[2 * h], w[2 * h + 1]));
      }
    }
    // ---- values
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
      uint32_t raw[4][(kValueBytes + 3) / 4], scale[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t token = static_cast<uint32_t>(16 * u + 8 * (t >> 1) + 2 * c + (t & 1));
        LoadShared<kValueBytes>(at + G::kPart + token * G::kCodes + g * kValueBytes, raw[t]);
        if constexpr (FP4) {
          constexpr int kScalesOfLane = D == 256 ? 2 : 1;
          LoadShared<kScalesOfLane>(at + G::kPart + G::kTile * G::kCodes + token * G::kScales + g * kValueChannels / 16, &scale[t]);
        }
        if (!whole && (token0 + static_cast<int>(token) >= length || absent)) {  // nothing that may lie there takes part
#pragma unroll
          for (int e = 0; e < (kValueBytes + 3) / 4; ++e) raw[t][e] = 0;
          scale[t] = 0;
        }
      }
      if constexpr (FP4) {
        uint32_t by[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          uint32_t two[2];
          FromE4m3(scale[t], two);
          by[t] = two[0];
        }
#pragma unroll
        for (int j = 0; j < kValueBytes / 4; ++j) {
          uint32_t v[4][4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            FromE2m1(raw[t][j], v[t]);
            const uint32_t both = __byte_perm(by[t], 0, j / 2 ? 0x3232 : 0x1010);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[t][e] = Mul16(v[t][e], both);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t a[4] = {__byte_perm(v[0][e], v[1][e], 0x5410), __byte_perm(v[0][e], v[1][e], 0x7632), __byte_perm(v[2][e], v[3][e], 0x5410),
                                   __byte_perm(v[2][e], v[3][e], 0x7632)};
#pragma unroll
            for (int n = 0; n < NT; ++n) Mma(o[n][4 * j + e], a, weights[u][n][0], weights[u][n][1]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kValueBytes / 4; ++j) {
          uint32_t v[4][2];
#pragma unroll
          for (int t = 0; t < 4; ++t) FromE4m3(raw[t][j], v[t]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a[4] = {__byte_perm(v[0][e], v[1][e], 0x5410), __byte_perm(v[0][e], v[1][e], 0x7632), __byte_perm(v[2][e], v[3][e], 0x5410),
                                   __byte_perm(v[2][e], v[3][e], 0x7632)};
#pragma unroll
            for (int n = 0; n < NT; ++n) Mma(o[n][2 * j + e], a, weights[u][n][0], weights[u][n][1]);
          }
        }
      }
    }
    __syncwarp();  // every lane has read the tile
    if (i + G::kStages < count) issue(i + G::kStages);
  }

  // ---- the warps' sums.  o[n][t][2 h + r] is channel g D / 8 + 2 t + h, row 8 n + 2 c + r.
  if (!good) {
    ctl.fault = 1;
    for (int i = 0; i < 16; ++i) __nanosleep(1000000);  // copies may still be landing
  }
  __syncthreads();  // no warp reads the ring any more
  const bool failed = ctl.fault != 0;
  float* const parts = reinterpret_cast<float*>(smem);  // [warp][row][D]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum[n][r] += __shfl_xor_sync(0xffffffffu, sum[n][r], d);
      const int row = 8 * n + 2 * c + r;
      if (g == 0) {
        ctl.most[warp][row] = most[n][r];
        ctl.sum[warp][row] = sum[n][r];
      }
      float* const to = parts + (warp * kRows + row) * D + g * kValueChannels;
#pragma unroll
      for (int t = 0; t < kTilesOfO; ++t) *reinterpret_cast<float2*>(to + 2 * t) = make_float2(o[n][t][r], o[n][t][2 + r]);
    }
  }
  __syncthreads();
  float* const partial = p.partial + static_cast<long long>(blockIdx.x) * kRows * (D + 2);
  for (int i = threadIdx.x; i < rows * (D / 2); i += kThreads) {
    const int row = i / (D / 2), channel = i % (D / 2) * 2;
    float all = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all = fmaxf(all, ctl.most[w][row]);
    float2 y = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float by = all == -INFINITY ? 0.f : Exp2(ctl.most[w][row] - all);
      const float2 v = *reinterpret_cast<const float2*>(parts + (w * kRows + row) * D + channel);
      total = fmaf(by, ctl.sum[w][row], total);
      y.x = fmaf(by, v.x, y.x);
      y.y = fmaf(by, v.y, y.y);
    }
    if (failed) total = __uint_as_float(0x7FFFFFFFu);
    if (cut.pieces > 1) {
      *reinterpret_cast<float2*>(partial + row * D + channel) = y;
      if (channel == 0) *reinterpret_cast<float2*>(partial + kRows * D + 2 * row) = make_float2(all, total);
    } else {
      const float by = total == 0.f ? 0.f : p.cache.v_unit / total;
      const int token = (row0 + row) / p.group, of = head * p.group + (row0 + row) % p.group;
      const long long to = (static_cast<long long>(cut.seq) * p.tokens + token) * p.q_heads + of;
      if (p.bf16) {
        *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p.out) + to * D + channel) = __floats2bfloat162_rn(y.x * by, y.y * by);
      } else {
        *reinterpret_cast<__half2*>(static_cast<__half*>(p.out) + to * D + channel) = __floats2half2_rn(y.x * by, y.y * by);
      }
      if (p.lse != nullptr && channel == 0) p.lse[to] = total == 0.f ? -INFINITY : (all + Log2(total)) * 0.693147181f;
    }
  }
}

// The pieces of the sequences that were cut.  A block: eight or sixteen rows of one key head of one sequence.
template <int D, int NT>
__global__ void __launch_bounds__(kThreads) JoinKernel(const AttendParams p, int tile) {
  constexpr int kRows = 8 * NT;
  GridDependencyWait();
  const int per_seq = p.cache.heads * p.row_blocks, seq = static_cast<int>(blockIdx.x) / per_seq, unit = static_cast<int>(blockIdx.x) % per_seq;
  const Cut cut = FindCut<kThreads>(p, tile, -1, seq);
  if (cut.pieces < 2) return;
  const int head = unit / p.row_blocks, row0 = unit % p.row_blocks * kRows, rows = min(kRows, p.tokens * p.group - row0);
  const float* const first = p.partial + (static_cast<long long>(cut.first) * per_seq + unit) * kRows * (D + 2);
  const long long step = static_cast<long long>(per_seq) * kRows * (D + 2);
  for (int i = threadIdx.x; i < rows * (D / 2); i += kThreads) {
    const int row = i / (D / 2), channel = i % (D / 2) * 2;
    float all = -INFINITY, total = 0.f;
    for (int k = 0; k < cut.pieces; ++k) all = fmaxf(all, first[k * step + kRows * D + 2 * row]);
    float2 y = make_float2(0.f, 0.f);
    for (int k = 0; k < cut.pieces; ++k) {
      const float* const part = first + k * step;
      const float2 ms = *reinterpret_cast<const float2*>(part + kRows * D + 2 * row), v = *reinterpret_cast<const float2*>(part + row * D + channel);
      const float by = all == -INFINITY ? 0.f : Exp2(ms.x - all);
      total = fmaf(by, ms.y, total);
      y.x = fmaf(by, v.x, y.x);
      y.y = fmaf(by, v.y, y.y);
    }
    const float by = total == 0.f ? 0.f : p.cache.v_unit / total;
    const int token = (row0 + row) / p.group, of = head * p.group + (row0 + row) % p.group;
    const long long to = (static_cast<long long>(seq) * p.tokens + token) * p.q_heads + of;
    if (p.bf16) {
      *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p.out) + to * D + channel) = __floats2bfloat162_rn(y.x * by, y.y * by);
    } else {
      *reinterpret_cast<__half2*>(static_cast<__half*>(p.out) + to * D + channel) = __floats2half2_rn(y.x * by, y.y * by);
    }
    if (p.lse != nullptr && channel == 0) p.lse[to] = total == 0.f ? -INFINITY : (all + Log2(total)) * 0.693147181f;
  }
}

struct Shape {
  int nt, row_blocks, target, tile;
  long long units;  // no more than that many
  bool cuts;        // sequences may be cut
};
Shape ShapeOf(const CacheAttentionCall& c) {
  Shape s;
  const int rows = c.tokens * (c.q_heads / c.cache.heads);
  s.nt = rows > 8 && c.cache.dim < 256 ? 2 : 1;
  s.row_blocks = (rows + 8 * s.nt - 1) / (8 * s.nt);
  const int codes = c.cache.fp4 ? c.cache.dim / 2 : c.cache.dim, scales = c.cache.fp4 ? c.cache.dim / 16 : 4;
  s.tile = (codes + scales) * 64 <= 9000 ? 32 : 16;
  // Pieces for four rounds of two blocks an SM: enough that the last ones to end are short, few enough that a block's start is.
  s.target = 8 * DeviceSmCount();
  const long long per_piece = static_cast<long long>(c.cache.heads) * s.row_blocks;
  const long long tiles = (static_cast<long long>(c.most_pages) * c.cache.page + s.tile - 1) / s.tile;
  s.cuts = tiles > kLeastTiles;
  const long long most_pieces = std::max(1LL, (tiles + kLeastTiles - 1) / kLeastTiles);  // of a sequence
  s.units = per_piece * std::min(c.seqs * most_pieces, c.seqs + s.target / per_piece + 1);
  return s;
}

template <int D, bool FP4, int NT>
cudaError_t Launch(const AttendParams& p, const Shape& s, cudaStream_t stream) {
  using G = Geometry<D, FP4>;
  static_assert(G::kBytes >= kWarps * 8 * NT * D * 4, "the warps' sums take the ring's place");
  static_assert(G::kStages >= 1 && G::kStages <= 8 && G::kBytes + 4096 <= 227 * 1024, "");
  const cudaError_t set = cudaFuncSetAttribute(CacheAttentionKernel<D, FP4, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kBytes);
  if (set != cudaSuccess) return set;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(s.units));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = G::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {OverlapAttribute()};
  cfg.attrs = attr;
  cfg.numAttrs = MayOverlapPredecessor(stream) ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, CacheAttentionKernel<D, FP4, NT>, p);
  if (err != cudaSuccess || !s.cuts) return err;
  cfg.gridDim = dim3(static_cast<unsigned>(p.seqs * p.cache.heads * p.row_blocks));
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, JoinKernel<D, NT>, p, s.tile);
}

template <bool FP4>
cudaError_t LaunchOf(const AttendParams& p, const Shape& s, cudaStream_t stream) {
  switch (p.cache.dim) {
    case 64: return s.nt == 1 ? Launch<64, FP4, 1>(p, s, stream) : Launch<64, FP4, 2>(p, s, stream);
    case 128: return s.nt == 1 ? Launch<128, FP4, 1>(p, s, stream) : Launch<128, FP4, 2>(p, s, stream);
    case 256: return Launch<256, FP4, 1>(p, s, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

size_t CacheAttentionWorkspace(const CacheAttentionCall& c) {
  const Shape s = ShapeOf(c);
  return s.cuts ? static_cast<size_t>(s.units) * 8 * s.nt * (c.cache.dim + 2) * sizeof(float) : 0;
}

cudaError_t LaunchCacheAttention(const CacheAttentionCall& c, cudaStream_t stream) {
  if (c.seqs == 0 || c.tokens == 0) return cudaSuccess;
  const Shape s = ShapeOf(c);
  if (s.units > INT_MAX) return cudaErrorInvalidValue;
  AttendParams p = {};
  p.cache = c.cache;
  p.q = c.q;
  p.ld_seq = c.ld_seq;
  p.ld_token = c.ld_token;
  p.table = c.table;
  p.ld_table = c.ld_table;
  p.most_pages = c.most_pages;
  p.lengths = c.lengths;
  p.seqs = c.seqs;
  p.tokens = c.tokens;
  p.q_heads = c.q_heads;
  p.group = c.q_heads / c.cache.heads;
  p.row_blocks = s.row_blocks;
  p.target_units = s.target;
  p.scale = c.scale * 1.44269504f * (c.cache.fp4 ? c.cache.k_unit : 1.f);
  if (!c.cache.fp4) p.cache.v_unit = 1.f;
  p.partial = static_cast<float*>(c.workspace);
  p.out = c.out;
  p.lse = c.lse;
  p.bf16 = c.dtype == QFG_BFLOAT16;
  p.give_up = c.give_up;
  const cudaError_t err = c.cache.fp4 ? LaunchOf<true>(p, s, stream) : LaunchOf<false>(p, s, stream);
  const cudaError_t last = cudaGetLastError();
  return err == cudaSuccess ? last : err;
}

}  // namespace qfg
