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
//            score, the values' the weight; scores then count from where score + log2(the value's scale) is largest, so that the product is within FP16 for values of any
//            size (of scores past 2^20 FP32 loses the logarithm, and small scales bits of their weight with it).
//   q        as FP16, each row times the power of two that takes its largest value to 2^9, so that only what is 2^-23 of that is rounded.
//
// Softmax runs along: m is taken up only when a score passes it by 8 (in powers of two), so that sums and weights stay within 2^8 of what they would be and the outputs
// are seldom scaled again.  Statistics and sums are FP32, weights FP16 (2^-11 of themselves, as the values are exact).
//
// A block runs through an equal share of all tiles (of one sequence and key head after another, in that order), its warps taking turns; each warp has its own ring of
// tiles in shared memory, which it fills by asynchronous copies ahead of itself, across the borders of sequences and heads too.  Where a sequence and head ends the warps add up
// their sums.  Shares begin and end anywhere; a second kernel joins those parts that share a sequence and head, in their order, so that results do not depend on which
// block is first.  Lengths are on the device only: where the shares lie is worked out there.
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

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kLeastTiles = kWarps;  // of a block's share: a tile a warp

// All tiles, in equal shares: share i begins at tile size i + min(i, more).
struct Shares {
  long long size;
  int more, count;
  __device__ __forceinline__ long long begin(int i) const { return size * i + min(i, more); }
};
struct alignas(16) ShareInfo {  // what the second kernel needs to know of a share: where it begins
  int seq, unit, tile, tiles;
};
struct AttendParams {
  KvCacheView cache;
  const void* q;
  const int *table, *lengths;
  Shares* shares;
  ShareInfo* share;   // [blocks]
  float* partial;     // [blocks][2][rows (D + 2)]: of a share that begins within a unit, and of its last unit where that goes on
  void* out;
  float* lse;
  long long ld_seq, ld_token, ld_table;
  int seqs, tokens, q_heads, group, most_pages, row_blocks;
  float scale;  // of scores, in powers of two, with the keys' unit
  bool bf16;
};

constexpr int TileOf(int dim, bool fp4) { return (fp4 ? dim / 2 + dim / 16 : dim + 4) * 64 <= 9300 && (fp4 || dim == 64) ? 32 : 16; }
template <int D, bool FP4, int NT>
struct Geometry {
  static constexpr int kCodes = FP4 ? D / 2 : D, kScales = FP4 ? D / 16 : 4;  // bytes of a row
  static constexpr int kTile = TileOf(D, FP4);                                // tokens
  static constexpr int kPart = kTile * (kCodes + kScales);                    // keys or values of a tile
  static constexpr int kStage = 2 * kPart;
  static constexpr int kBlocks = D * NT <= 128 ? 2 : 1;                       // of an SM
  static constexpr int kSums = kWarps * 8 * NT * D * 4;                       // the warps' sums
  static constexpr int kRoom = (kBlocks == 2 ? 111 : 222) * 1024 - kSums;
  static constexpr int kStages = std::min(8, kRoom / (kWarps * kStage));
  static constexpr int kBytes = kWarps * kStages * kStage + kSums;
};

__device__ __forceinline__ int TilesOf(const AttendParams& p, int seq, int tile, int* length) {
  const long long room = static_cast<long long>(p.most_pages) * p.cache.page;
  *length = static_cast<int>(min(static_cast<long long>(max(p.lengths[seq], 0)), room));
  return (*length + tile - 1) / tile;
}
// This block's share, `from` to `to`, and the sequence that holds `from`, with the number of tiles ahead of it.  A sequence's tiles count once for each key head and
// block of rows.
struct Share {
  Shares all;
  long long from, to, ahead;
  int seq, tiles, length;  // seq is -1 where there is no share
};
__device__ __forceinline__ Share FindShare(const AttendParams& p, int tile) {
  __shared__ int sums[kWarps];
  __shared__ long long total[kWarps];
  __shared__ Share found;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per_seq = p.cache.heads * p.row_blocks;
  int length = 0;
  long long all = 0;
  if (p.seqs > kThreads) {
    for (int i = threadIdx.x; i < p.seqs; i += kThreads) all += TilesOf(p, i, tile, &length);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
    if (lane == 0) total[warp] = all;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all += total[w];
  }
  Share s;
  s.seq = -1;
  long long before = 0;
  for (int base = 0; base < p.seqs; base += kThreads) {
    const int i = base + static_cast<int>(threadIdx.x);
    const int tiles = i < p.seqs ? TilesOf(p, i, tile, &length) : 0;
    int upto = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    if (base > 0) __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    long long ahead = before;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) ahead += sums[w];
      before += sums[w];
    }
    if (base == 0) {
      if (p.seqs <= kThreads) all = before;
      all *= per_seq;
      s.all.count = static_cast<int>(min(static_cast<long long>(gridDim.x), (all + kLeastTiles - 1) / kLeastTiles));
      if (static_cast<int>(blockIdx.x) >= s.all.count) return s;
      s.all.size = all >> 32 ? all / s.all.count : static_cast<uint32_t>(all) / static_cast<uint32_t>(s.all.count);
      s.all.more = static_cast<int>(all - s.all.size * s.all.count);
      s.from = s.all.begin(blockIdx.x);
      s.to = s.all.begin(blockIdx.x + 1);
    }
    const long long begin = (ahead + upto - tiles) * per_seq, end = (ahead + upto) * per_seq;
    if (s.from >= begin && s.from < end) {
      found = s;
      found.ahead = begin;
      found.seq = i;
      found.tiles = tiles;
      found.length = length;
    }
  }
  __syncthreads();
  return found;
}
// A run of tiles of one unit: a key head of a sequence, and a block of its rows.
struct Segment {
  int seq, unit, tile, tiles, length;  // tile: the first; tiles: of the whole unit
  int begin, end;                      // in the share
};
__device__ __forceinline__ Segment FirstSegment(const Share& s) {
  Segment g;
  g.seq = s.seq;
  g.tiles = s.tiles;
  g.length = s.length;
  const long long into = s.from - s.ahead;
  const int in = static_cast<int>(into >> 32 ? into / g.tiles : static_cast<uint32_t>(into) / static_cast<uint32_t>(g.tiles));
  g.unit = in;
  g.tile = static_cast<int>(s.from - s.ahead - static_cast<long long>(in) * g.tiles);
  g.begin = 0;
  g.end = static_cast<int>(min(s.to - s.from, static_cast<long long>(g.tiles - g.tile)));
  return g;
}
__device__ __forceinline__ void NextSegment(const AttendParams& p, int count, int tile, Segment* g) {  // while g->end < count
  g->begin = g->end;
  g->tile = 0;
  if (++g->unit == p.cache.heads * p.row_blocks) {
    g->unit = 0;
    do g->tiles = TilesOf(p, ++g->seq, tile, &g->length);
    while (g->tiles == 0);
  }
  g->end = g->begin + min(count - g->begin, g->tiles);
}

__device__ __forceinline__ void CopyAsync(uint32_t to, const uint8_t* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ uint32_t Smem(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
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
// a half of a pair, twice: the multiplication takes it so
__device__ __forceinline__ uint32_t Lower(uint32_t v) {
  uint32_t r;
  asm("{ .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n mov.b32 %0, {l, l};\n}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t Upper(uint32_t v) {
  uint32_t r;
  asm("{ .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n mov.b32 %0, {h, h};\n}" : "=r"(r) : "r"(v));
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

template <int D>
__device__ __forceinline__ void StoreRow(const AttendParams& p, int seq, int unit, int row, int channel, float2 y, float most, float total) {
  const int head = unit / p.row_blocks, token = row / p.group, of = head * p.group + row - token * p.group;
  const long long to = (static_cast<long long>(seq) * p.tokens + token) * p.q_heads + of;
  const float by = total == 0.f ? 0.f : p.cache.v_unit / total;
  if (p.bf16) {
    *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p.out) + to * D + channel) = __floats2bfloat162_rn(y.x * by, y.y * by);
  } else {
    *reinterpret_cast<__half2*>(static_cast<__half*>(p.out) + to * D + channel) = __floats2half2_rn(y.x * by, y.y * by);
  }
  if (p.lse != nullptr && channel == 0) p.lse[to] = total == 0.f ? -INFINITY : (most + Log2(total)) * 0.693147181f;
}

// NT tiles of eight rows.
template <int D, bool FP4, int NT>
__global__ void __launch_bounds__(kThreads, Geometry<D, FP4, NT>::kBlocks) CacheAttentionKernel(const AttendParams p) {
  using G = Geometry<D, FP4, NT>;
  constexpr int kRows = 8 * NT, kSteps = D / 16, kGroups = G::kTile / 16;
  constexpr int kKeyBytes = G::kCodes / 4, kValueBytes = G::kCodes / 8;  // of a lane's part of a row
  constexpr int kKeyScales = FP4 ? D / 64 : 1;                           // E4M3 scales of that part
  constexpr int kValueChannels = D / 8, kTilesOfO = D / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float row_most[kWarps][kRows], row_sum[kWarps][kRows];
  __shared__ __align__(16) uint16_t q_rows[kRows][D + 8];
  __shared__ float q_factor[kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  GridDependencyWait();
  GridLaunchDependents();  // the second kernel, which waits for all of this one
  const Share share = FindShare(p, G::kTile);
  for (int seq = blockIdx.x; seq < p.seqs; seq += gridDim.x) {
    int length;
    if (TilesOf(p, seq, G::kTile, &length) > 0) continue;
    for (int unit = 0; unit < p.cache.heads * p.row_blocks; ++unit) {
      const int row0 = unit % p.row_blocks * kRows, rows = min(kRows, p.tokens * p.group - row0);
      for (int i = threadIdx.x; i < rows * (D / 2); i += kThreads) StoreRow<D>(p, seq, unit, row0 + i / (D / 2), i % (D / 2) * 2, make_float2(0.f, 0.f), 0.f, 0.f);
    }
  }
  if (share.seq < 0) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.shares != nullptr) *p.shares = {0, 0, 0};
    return;
  }
  Segment at = FirstSegment(share);
  if (threadIdx.x == 0 && p.shares != nullptr) {
    p.share[blockIdx.x] = {at.seq, at.unit, at.tile, at.tiles};
    if (blockIdx.x == 0) *p.shares = share.all;
  }
  const int count = static_cast<int>(share.to - share.from);

  // q of a segment's rows, as FP16, for all warps: row w (and w + 8) by warp w
  auto make_q = [&](const Segment& of) {
    const int head = of.unit / p.row_blocks, row0 = (of.unit - head * p.row_blocks) * kRows;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 8 * n + warp, token = (row0 + r) / p.group;
      uint32_t w[D / 64] = {};
      if (row0 + r < p.tokens * p.group) {
        const uint16_t* const from = static_cast<const uint16_t*>(p.q) + of.seq * p.ld_seq + token * p.ld_token +
                                     static_cast<long long>(head * p.group + row0 + r - token * p.group) * D + lane * (D / 32);
        if constexpr (D == 64) w[0] = *reinterpret_cast<const uint32_t*>(from);
        if constexpr (D == 128) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(from);
        if constexpr (D == 256) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(from);
      }
      float2 v[D / 64];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        v[i] = p.bf16 ? make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u)) : __half22float2(*reinterpret_cast<__half2*>(&w[i]));
        top = max(top, max(__float_as_uint(v[i].x) & 0x7FFFFFFFu, __float_as_uint(v[i].y) & 0x7FFFFFFFu));
      }
      // 2^(9 - exponent) of the largest and its inverse; the exponent is kept where both are ordinary numbers
      const int e = min(max(static_cast<int>(__reduce_max_sync(0xffffffffu, top) >> 23), 20), 240);
      const float up = __uint_as_float(static_cast<uint32_t>(263 - e) << 23);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) *reinterpret_cast<uint32_t*>(&q_rows[r][lane * (D / 32) + 2 * i]) = Pack16(v[i].x * up, v[i].y * up);
      if (lane == 0) q_factor[r] = __uint_as_float(static_cast<uint32_t>(e - 9) << 23) * p.scale;
    }
  };

  // ---- this warp's tiles: warp, warp + kWarps, ... of the share
  const uint32_t ring = Smem(smem) + G::kSums + static_cast<uint32_t>(warp * G::kStages * G::kStage);
  Segment ahead = at;
  int next = warp, batch = 0, issued = 0;  // the tile that is copied next; the first one that `row` is of
  bool known = false;
  long long row = 0;     // lane i: where tile batch + i kWarps lies in the cache, or -1: in no page of it
  uint32_t present = 0;  // of the stages
  const int tiles_of_page = p.cache.page / G::kTile;
  auto copy = [&](uint32_t to, const uint8_t* from, auto bytes) {
    constexpr int kBytes = decltype(bytes)::value;
#pragma unroll
    for (int i = 0; i < kBytes; i += 512) {
      if (i + 512 <= kBytes || 16 * lane < kBytes - i) CopyAsync(to + i + 16 * lane, from + i + 16 * lane);
    }
  };
  auto issue = [&] {
    if (next < count) {
      while (next >= ahead.end) {
        NextSegment(p, count, G::kTile, &ahead);
        known = false;
      }
      if (!known || next - batch >= 32 * kWarps) {
        batch = next;
        known = true;
        const int mine = next + lane * kWarps;
        row = -1;
        if (mine < ahead.end) {
          const int tile = ahead.tile + mine - ahead.begin, page = tile / tiles_of_page, id = p.table[ahead.seq * p.ld_table + page];
          if (id >= 0 && id < p.cache.pages)
            row = (static_cast<long long>(id) * p.cache.heads + ahead.unit / p.row_blocks) * p.cache.page + (tile - page * tiles_of_page) * G::kTile;
        }
      }
      const long long from = __shfl_sync(0xffffffffu, row, (next - batch) / kWarps), r = max(from, 0LL);
      present = (present & ~(1u << issued)) | (from >= 0 ? 1u << issued : 0u);
      const uint32_t to = ring + static_cast<uint32_t>(issued * G::kStage);
      copy(to, p.cache.k + r * G::kCodes, std::integral_constant<int, G::kTile * G::kCodes>());
      copy(to + G::kTile * G::kCodes, static_cast<const uint8_t*>(p.cache.k_scale) + r * G::kScales, std::integral_constant<int, G::kTile * G::kScales>());
      copy(to + G::kPart, p.cache.v + r * G::kCodes, std::integral_constant<int, G::kTile * G::kCodes>());
      copy(to + G::kPart + G::kTile * G::kCodes, static_cast<const uint8_t*>(p.cache.v_scale) + r * G::kScales, std::integral_constant<int, G::kTile * G::kScales>());
      issued = issued + 1 == G::kStages ? 0 : issued + 1;
      next += kWarps;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // one a tile, of nothing behind the last
  };
#pragma unroll 1
  for (int i = 0; i < G::kStages; ++i) issue();
  make_q(at);
  __syncthreads();

  int x = warp, stage = 0;
#pragma unroll 1
  for (;;) {  // segments
    const int head = at.unit / p.row_blocks, row0 = (at.unit - head * p.row_blocks) * kRows, rows = min(kRows, p.tokens * p.group - row0);
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
    const bool any = x < at.end;
    if (any) {
      uint32_t q[NT][kSteps][2];
      float factor[NT][2];  // from a row's products to its scores
      int sees[NT][2];      // tokens that a row may look at
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const uint2 w = *reinterpret_cast<const uint2*>(&q_rows[8 * n + g][c * (D / 4) + 4 * i]);
          q[n][i][0] = w.x, q[n][i][1] = w.y;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          factor[n][h] = q_factor[8 * n + 2 * c + h];
          sees[n][h] = at.length - p.tokens + 1 + (row0 + 8 * n + 2 * c + h) / p.group;
        }
      }
      const int least_seen = at.length - p.tokens + 1;

#pragma unroll 1
      for (; x < at.end; x += kWarps) {
        const uint32_t tile = ring + static_cast<uint32_t>(stage * G::kStage);
        asm volatile("cp.async.wait_group %0;" ::"n"(G::kStages - 1) : "memory");
        __syncwarp();
        const int token0 = (at.tile + x - at.begin) * G::kTile;
        const bool absent = !(present >> stage & 1);
        const bool whole = token0 + G::kTile <= least_seen && !absent;  // no row leaves any token of it out
        // ---- scores: s[u][n][2 h + r] is token 16 u + 8 h + g, row 8 n + 2 c + r
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
            LoadShared<kKeyBytes>(tile + token * G::kCodes + c * kKeyBytes, raw[h]);
            if constexpr (FP4) LoadShared<kKeyScales>(tile + G::kTile * G::kCodes + token * G::kScales + c * kKeyScales, &scale[h]);
          }
          if constexpr (FP4) {
            uint32_t by[2][2];  // pairs of scales
#pragma unroll
            for (int h = 0; h < 2; ++h) FromE4m3(scale[h], by[h]);
#pragma unroll
            for (int j = 0; j < kKeyBytes / 4; ++j) {
              uint32_t v[2][4];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t both = j & 2 ? Upper(by[h][j / 4]) : Lower(by[h][j / 4]);  // block j / 2 of sixteen channels
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
        // eight bits: the scales of keys and values; a value's moves the point from which a weight is measured, so that the product of both stays within FP16
        float value_scale[kGroups][2], log_scale[kGroups][2];
        if constexpr (!FP4) {
#pragma unroll
          for (int u = 0; u < kGroups; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t token = static_cast<uint32_t>(16 * u + 8 * h + g);
              float key_scale;
              LoadShared<4>(tile + G::kTile * G::kCodes + token * 4, reinterpret_cast<uint32_t*>(&key_scale));
              LoadShared<4>(tile + G::kPart + G::kTile * G::kCodes + token * 4, reinterpret_cast<uint32_t*>(&value_scale[u][h]));
              if (!whole && (token0 + static_cast<int>(token) >= at.length || absent)) value_scale[u][h] = 1.f;
              log_scale[u][h] = fminf(fmaxf(Log2(value_scale[u][h]), -60.f), 60.f);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int r = 0; r < 2; ++r) s[u][n][2 * h + r] *= key_scale * factor[n][r];
              }
            }
          }
        }
        if constexpr (FP4) {
#pragma unroll
          for (int u = 0; u < kGroups; ++u) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
              for (int e = 0; e < 4; ++e) s[u][n][e] *= factor[n][e & 1];
            }
          }
        }
        if (!whole) {
#pragma unroll
          for (int u = 0; u < kGroups; ++u) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (token0 + 16 * u + 8 * (e >> 1) + g >= sees[n][e & 1] || absent) s[u][n][e] = -INFINITY;
              }
            }
          }
        }
        // m is taken up where a score passes it by 8
        bool higher = false;
        float upto[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float m = -INFINITY;
#pragma unroll
            for (int u = 0; u < kGroups; ++u) {
#pragma unroll
              for (int h = 0; h < 2; ++h) m = fmaxf(m, FP4 ? s[u][n][2 * h + r] : s[u][n][2 * h + r] + log_scale[u][h]);
            }
            upto[n][r] = m;
            higher = higher || upto[n][r] > most[n][r] + 8.f;
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
        for (int n = 0; n < NT; ++n) {
          float off[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) off[r] = most[n][r] == -INFINITY ? 0.f : most[n][r];
#pragma unroll
          for (int u = 0; u < kGroups; ++u) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = Exp2(s[u][n][e] - off[e & 1]);  // of a rounded score: 0 at the maximum, however large that is
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
          uint32_t raw[4][kValueBytes / 4], scale[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t token = static_cast<uint32_t>(16 * u + 8 * (t >> 1) + 2 * c + (t & 1));
            LoadShared<kValueBytes>(tile + G::kPart + token * G::kCodes + g * kValueBytes, raw[t]);
            if constexpr (FP4) LoadShared<(D == 256 ? 2 : 1)>(tile + G::kPart + G::kTile * G::kCodes + token * G::kScales + g * kValueChannels / 16, &scale[t]);
          }
          if (!whole) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              if (token0 + 16 * u + 8 * (t >> 1) + 2 * c + (t & 1) >= at.length || absent) {  // nothing that may lie there takes part
#pragma unroll
                for (int e = 0; e < kValueBytes / 4; ++e) raw[t][e] = 0;
                scale[t] = 0;
              }
            }
          }
          if constexpr (FP4) {
            // codes of the same channel of two tokens side by side in a byte, and their scales in a pair
            uint32_t by[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              FromE4m3(D == 256 ? __byte_perm(scale[2 * h], scale[2 * h + 1], 0x5140) : __byte_perm(scale[2 * h], scale[2 * h + 1], 0x0040), by[h]);
            }
#pragma unroll
            for (int j = 0; j < kValueBytes / 4; ++j) {
              uint32_t v[2][2][4];  // [tokens][even, odd channels][pairs of channels]
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t a = raw[2 * h][j], b = raw[2 * h + 1][j];
                FromE2m1((a & 0x0F0F0F0Fu) | (b << 4 & 0xF0F0F0F0u), v[h][0]);
                FromE2m1((a >> 4 & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u), v[h][1]);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[h][e / 4][e % 4] = Mul16(v[h][e / 4][e % 4], by[h][j / 2]);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t a[4] = {v[0][0][e], v[0][1][e], v[1][0][e], v[1][1][e]};
#pragma unroll
                for (int n = 0; n < NT; ++n) Mma(o[n][4 * j + e], a, weights[u][n][0], weights[u][n][1]);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < kValueBytes / 4; ++j) {
              uint32_t v[2][2][2];  // [tokens][channels 0 and 1, 2 and 3 of four][as codes: of one channel and the next]
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                // (token, next token) of channel 0, 1 | 2, 3
                FromE4m3(__byte_perm(raw[2 * h][j], raw[2 * h + 1][j], 0x5140), v[h][0]);
                FromE4m3(__byte_perm(raw[2 * h][j], raw[2 * h + 1][j], 0x7362), v[h][1]);
              }
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t a[4] = {v[0][e][0], v[0][e][1], v[1][e][0], v[1][e][1]};
#pragma unroll
                for (int n = 0; n < NT; ++n) Mma(o[n][2 * j + e], a, weights[u][n][0], weights[u][n][1]);
              }
            }
          }
        }
        __syncwarp();  // every lane has read the tile
        issue();
        if (++stage == G::kStages) stage = 0;
      }
    }

    // ---- the warps' sums.  o[n][t][2 h + r] is channel g D / 8 + 2 t + h, row 8 n + 2 c + r.
    float* const parts = reinterpret_cast<float*>(smem);  // [warp][row][D]
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int to_row = 8 * n + 2 * c + r;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum[n][r] += __shfl_xor_sync(0xffffffffu, sum[n][r], d);
        if (g == 0) {
          row_most[warp][to_row] = most[n][r];
          row_sum[warp][to_row] = sum[n][r];
        }
        if (any) {
          float* const to = parts + (warp * kRows + to_row) * D + g * kValueChannels;
#pragma unroll
          for (int t = 0; t < kTilesOfO; ++t) *reinterpret_cast<float2*>(to + 2 * t) = make_float2(o[n][t][r], o[n][t][2 + r]);
        }
      }
    }
    __syncthreads();
    const bool whole_unit = at.tile == 0 && at.end - at.begin == at.tiles;
    float* const partial = p.partial + (static_cast<long long>(blockIdx.x) * 2 + (at.tile > 0 ? 0 : 1)) * kRows * (D + 2);
    for (int i = threadIdx.x; i < rows * (D / 2); i += kThreads) {
      const int of = i / (D / 2), channel = i % (D / 2) * 2;
      float all = -INFINITY, total = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) all = fmaxf(all, row_most[w][of]);
      float2 y = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float m = row_most[w][of];
        if (m == -INFINITY) {
          total += row_sum[w][of];  // 0, or of a row that saw nothing but NaN
          continue;
        }
        const float by = Exp2(m - all);
        const float2 v = *reinterpret_cast<const float2*>(parts + (w * kRows + of) * D + channel);
        total = fmaf(by, row_sum[w][of], total);
        y.x = fmaf(by, v.x, y.x);
        y.y = fmaf(by, v.y, y.y);
      }
      if (whole_unit) {
        StoreRow<D>(p, at.seq, at.unit, row0 + of, channel, y, all, total);
      } else {
        *reinterpret_cast<float2*>(partial + of * D + channel) = y;
        if (channel == 0) *reinterpret_cast<float2*>(partial + kRows * D + 2 * of) = make_float2(all, total);
      }
    }
    if (at.end == count) break;
    NextSegment(p, count, G::kTile, &at);
    make_q(at);
    __syncthreads();  // the sums have been read, and q is there
  }
}

// The units that lie in several shares.  Block b looks after the unit that share b + 1 begins within, where no earlier share does.
template <int D, int NT>
__global__ void __launch_bounds__(kThreads) JoinKernel(const AttendParams p) {
  constexpr int kRows = 8 * NT, kRow = D + 2, kSlot = kRows * kRow, kBatch = 64;
  __shared__ float2 stats[kBatch][kRows];
  GridDependencyWait();
  const int b = static_cast<int>(blockIdx.x) + 1;
  const Shares shares = *p.shares;
  const ShareInfo at = p.share[b];
  if (b >= shares.count) return;
  const long long first = shares.begin(b) - at.tile, end = first + at.tiles;
  if (at.tile == 0 || first < shares.begin(b - 1)) return;
  const int row0 = at.unit % p.row_blocks * kRows, rows = min(kRows, p.tokens * p.group - row0);
  int pieces = 2;  // of shares b - 1 (its second slot), b, ...
  while (b - 1 + pieces < shares.count && shares.begin(b - 1 + pieces) < end) ++pieces;
  const auto slot = [&](int k) { return p.partial + (static_cast<long long>(b - 1 + k) * 2 + (k == 0 ? 1 : 0)) * kSlot; };
  constexpr int kMine = (kRows * D / 2 + kThreads - 1) / kThreads;
  float most[kMine], total[kMine];
  float2 y[kMine];
#pragma unroll
  for (int j = 0; j < kMine; ++j) most[j] = -INFINITY, total[j] = 0.f, y[j] = make_float2(0.f, 0.f);
  for (int k0 = 0; k0 < pieces; k0 += kBatch) {
    const int n = min(kBatch, pieces - k0);
    __syncthreads();
    for (int i = threadIdx.x; i < n * kRows; i += kThreads) stats[i / kRows][i % kRows] = *reinterpret_cast<const float2*>(slot(k0 + i / kRows) + kRows * D + i % kRows * 2);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = static_cast<int>(threadIdx.x) + j * kThreads, of = i / (D / 2), channel = i % (D / 2) * 2;
      if (of >= rows) continue;
      float all = most[j];
      for (int k = 0; k < n; ++k) all = fmaxf(all, stats[k][of].x);
      const float again = all == -INFINITY ? 0.f : Exp2(most[j] - all);
      total[j] *= most[j] == -INFINITY ? 1.f : again;
      y[j].x *= again;
      y[j].y *= again;
      most[j] = all;
#pragma unroll 8
      for (int k = 0; k < n; ++k) {
        const float2 ms = stats[k][of], v = *reinterpret_cast<const float2*>(slot(k0 + k) + of * D + channel);
        const float by = ms.x == -INFINITY ? 0.f : Exp2(ms.x - all);
        total[j] += ms.x == -INFINITY ? ms.y : by * ms.y;
        y[j].x = fmaf(by, v.x, y[j].x);
        y[j].y = fmaf(by, v.y, y[j].y);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    const int i = static_cast<int>(threadIdx.x) + j * kThreads, of = i / (D / 2), channel = i % (D / 2) * 2;
    if (of < rows) StoreRow<D>(p, at.seq, at.unit, row0 + of, channel, y[j], most[j], total[j]);
  }
}

struct Shape {
  int nt, row_blocks, blocks;
};
Shape ShapeOf(const CacheAttentionCall& c) {
  Shape s;
  const int rows = c.tokens * (c.q_heads / c.cache.heads);
  s.nt = rows > 8 && c.cache.dim < 256 ? 2 : 1;
  s.row_blocks = (rows + 8 * s.nt - 1) / (8 * s.nt);
  const int tile = TileOf(c.cache.dim, c.cache.fp4);
  const long long room = static_cast<long long>(c.most_pages) * c.cache.page, tiles = (room + tile - 1) / tile * c.seqs * c.cache.heads * s.row_blocks;
  // as many as the GPU holds at once, and no more than have a tile for each warp
  const long long most = static_cast<long long>(DeviceSmCount()) * (c.cache.dim * s.nt <= 128 ? 2 : 1);
  s.blocks = static_cast<int>(std::max(1LL, std::min(most, (tiles + kLeastTiles - 1) / kLeastTiles)));
  return s;
}

template <int D, bool FP4, int NT>
cudaError_t Launch(const AttendParams& p, const Shape& s, cudaStream_t stream) {
  using G = Geometry<D, FP4, NT>;
  static_assert(G::kStages >= 2 && G::kBlocks * (G::kBytes + 6144) <= 227 * 1024, "");
  const cudaError_t set = cudaFuncSetAttribute(CacheAttentionKernel<D, FP4, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kBytes);
  if (set != cudaSuccess) return set;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(s.blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = G::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {OverlapAttribute()};
  cfg.attrs = attr;
  cfg.numAttrs = MayOverlapPredecessor(stream) ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, CacheAttentionKernel<D, FP4, NT>, p);
  if (err != cudaSuccess || s.blocks < 2) return err;
  cfg.gridDim = dim3(static_cast<unsigned>(s.blocks - 1));
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, JoinKernel<D, NT>, p);
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
  return s.blocks < 2 ? 0 : sizeof(Shares) + s.blocks * (sizeof(ShareInfo) + sizeof(float) * 2 * 8 * s.nt * (c.cache.dim + 2));
}

cudaError_t LaunchCacheAttention(const CacheAttentionCall& c, cudaStream_t stream) {
  if (c.seqs == 0 || c.tokens == 0) return cudaSuccess;
  const Shape s = ShapeOf(c);
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
  p.scale = c.scale * 1.44269504f * (c.cache.fp4 ? c.cache.k_unit : 1.f);
  if (!c.cache.fp4) p.cache.v_unit = 1.f;
  if (s.blocks > 1) {
    p.shares = static_cast<Shares*>(c.workspace);
    p.share = reinterpret_cast<ShareInfo*>(p.shares + 1);
    p.partial = reinterpret_cast<float*>(p.share + s.blocks);
  }
  p.out = c.out;
  p.lse = c.lse;
  p.bf16 = c.dtype == QFG_BFLOAT16;
  const cudaError_t err = c.cache.fp4 ? LaunchOf<true>(p, s, stream) : LaunchOf<false>(p, s, stream);
  const cudaError_t last = cudaGetLastError();
  return err == cudaSuccess ? last : err;
}

}  // namespace qfg
