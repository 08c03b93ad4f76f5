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
//            score, the values' the weight; scores then count from where score + log2(the value's scale) is largest, so that the product is within FP16 for scales up
//            to 2^107 (of scores past 2^20 FP32 loses the logarithm, and small scales bits of their weight with it).
//   q        as FP16, each row times the power of two that takes its largest value to 2^9, so that only what is 2^-23 of that is rounded.
//
// Softmax runs along: m is taken up only when a score has gone past it by some powers of two, so that the outputs are seldom scaled again.  Statistics and sums are FP32, weights
// FP16: off by 2^-11 of themselves, as the values are exact, and by 2^-25 below 2^-14.  So that long sequences whose weights are all small beside one do not lose them, in four
// bits m lies 7 below the largest score when it is taken up: FP16's smallest number is 2^-31 of that one's weight.  In eight bits it is 2^-24 of the largest product with a scale.
//
// A warp runs through an equal share of all tiles (of one sequence and key head after another, in that order) and has its own ring of tiles in shared memory, which it
// fills by asynchronous copies ahead of itself, across the borders of sequences and heads too; no warp waits for another.  Shares begin and end anywhere; a second kernel
// joins those parts that share a sequence and head, in their order, so that results do not depend on which warp is first.  Lengths are on the device only: where the
// shares lie is worked out there.
//
// Measured, 8 key heads of 128 channels.  Two sequences of up to 131072 tokens, E4M3, 64 query heads: 83 us for 400 MB, 4.8 TB/s; the first kernel takes 72 to 75 of them.  64 of up
// to 8192, NVFP4: 85 us for 335 MB, 3.9 TB/s; 61 % of the issue slots are taken, by conversions, multiplications by scales and the order of the values' codes, one warp in four
// waits for the result of the instruction ahead, one in five for the unit of its own.  Few tiles for each warp (16 of up to 4001 tokens, four tokens each: 7): 29.6 us where the
// bytes take 7; three trips to memory before the first tile, two warps a scheduler, and the join.  One sequence of 1000 tokens: 9.8 us, trips to memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "qfg_internal.h"
#include "stream_order.cuh"

namespace qfg {
namespace {

// Warps of a block.  One tile of eight rows leaves room for two blocks an SM, sixteen warps of 128 registers; two tiles, or heads of 256 channels, for one, eight warps of up to
// 255.  Twelve warps of 168 are slower there: 16 sequences of up to 4001 tokens, four tokens of 32 / 8 heads of 128 each, 31.7 -> 39.8 us; 32 of up to 8192, 24 / 4 heads of
// 256, NVFP4 50.7 -> 62.7, E4M3 69.3 -> 85.9.
constexpr int kWarps = 8, kThreads = 32 * kWarps;
// Eight bits: of a value's scale, 2^this is the most that moves the point from which weights are measured.  FP32 still holds the exponentials of 2^-26 of the largest there; FP16
// holds a weight's product with a scale of 2^7 more.
constexpr float kMostLogScale = 100.f;
// All tiles, in equal shares: share i begins at tile size i + min(i, more).
struct Shares {
  long long size;
  int more, count;
  __device__ __forceinline__ long long begin(int i) const { return size * i + min(i, more); }
};
struct AttendParams {
  KvCacheView cache;
  const void* q;
  const int *table, *lengths;
  int2* parts;     // [seqs][key heads][row blocks]: the first share of a unit, and how many have a part of it; (0, 0) where one has all of it
  float* partial;  // [shares][2][rows (D + 2)]: of a share that begins within a unit, and of its last unit where that goes on
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
  // Codes are kept with their pieces of 16 bytes exchanged within 128, by the place of those among the others, so that the lanes of a load, which read tokens that are two
  // apart (values) or lie beside one another (keys), meet in no bank.
  static __device__ __forceinline__ uint32_t Swizzled(uint32_t at) {
    constexpr int kShift = kCodes == 32 ? 32 : kCodes == 64 ? 2 : 3;  // of bits 7 to 9 down to bits 4 to 6; rows of 64 bytes: bits 7 and 8 to 5 and 6
    return kCodes == 32 ? at : at ^ (at >> kShift & (kCodes == 64 ? 0x60u : 0x70u));
  }
  static constexpr int kBlocks = D * NT <= 128 ? 2 : 1;                       // of an SM
  static constexpr int kStages = std::min(8, (kBlocks == 2 ? 110 : 220) * 1024 / (kWarps * kStage));
  static constexpr int kBytes = kWarps * kStages * kStage;
};

__device__ __forceinline__ int TilesOf(const AttendParams& p, int seq, int tile, int* length) {
  const long long room = static_cast<long long>(p.most_pages) * p.cache.page;
  *length = static_cast<int>(min(static_cast<long long>(max(p.lengths[seq], 0)), room));
  return (*length + tile - 1) / tile;
}
// This warp's share, `from` to `to`, and the sequence that holds `from`, with the number of tiles ahead of it.  A sequence's tiles count once for each key head and
// block of rows.
struct Share {
  Shares all;
  long long from, to, ahead;
  int seq, tiles, length;  // seq is -1 where there is no share
};
__device__ __forceinline__ Share FindShare(const AttendParams& p, int tile) {
  __shared__ int sums[kWarps];
  __shared__ long long total[kWarps];
  __shared__ Share found[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per_seq = p.cache.heads * p.row_blocks, first = static_cast<int>(blockIdx.x) * kWarps;
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
      // Few units: a part more costs the join about 9 ns, a tile more a share 1.5 us, so that of a unit of n tiles shares are best sqrt(n / 160) tiles or longer.  One sequence
      // of 131072 tokens and one key head, NVFP4: 47 us with shares of one or two tiles, 29 of five; 20000 tokens 17.9 and
      // 15.0 of two.
      const int least = static_cast<int>(sqrtf(static_cast<float>(all) / (160.f * p.seqs * per_seq)) + 0.5f);
      s.all.count = static_cast<int>(min(static_cast<long long>(gridDim.x) * kWarps, least > 1 ? (all + least - 1) / least : all));
      if (first >= s.all.count) return s;
      s.all.size = all >> 32 ? all / s.all.count : static_cast<uint32_t>(all) / static_cast<uint32_t>(s.all.count);
      s.all.more = static_cast<int>(all - s.all.size * s.all.count);
    }
    const long long begin = (ahead + upto - tiles) * per_seq, end = (ahead + upto) * per_seq;
#pragma unroll 1
    for (int w = 0; w < kWarps && first + w < s.all.count; ++w) {
      const long long from = s.all.begin(first + w);
      if (from >= begin && from < end) found[w] = {s.all, from, s.all.begin(first + w + 1), begin, i, tiles, length};
    }
  }
  __syncthreads();
  if (first + warp < s.all.count) s = found[warp];
  return s;
}
// The share that holds a tile.
__device__ __forceinline__ int ShareOf(const Shares& s, long long tile) {
  const long long larger = (s.size + 1) * s.more;  // tiles of the shares that have one more
  if (tile < larger) return static_cast<int>(tile >> 32 ? tile / (s.size + 1) : static_cast<uint32_t>(tile) / static_cast<uint32_t>(s.size + 1));
  return s.more + static_cast<int>((tile - larger) >> 32 ? (tile - larger) / s.size : static_cast<uint32_t>(tile - larger) / static_cast<uint32_t>(s.size));
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

// Where a row of a unit lies among the outputs.
__device__ __forceinline__ long long RowOf(const AttendParams& p, int seq, int unit, int row) {
  const int head = unit / p.row_blocks, token = row / p.group, of = head * p.group + row - token * p.group;
  return (static_cast<long long>(seq) * p.tokens + token) * p.q_heads + of;
}
__device__ __forceinline__ uint32_t Packed(bool bf16, float lo, float hi) {
  uint32_t r;
  if (bf16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    r = Pack16(lo, hi);
  }
  return r;
}
__device__ __forceinline__ float LogOfSum(float most, float total) { return total == 0.f ? -INFINITY : (most + Log2(total)) * 0.693147181f; }

// NT tiles of eight rows.
template <int D, bool FP4, int NT>
__global__ void __launch_bounds__(kThreads, Geometry<D, FP4, NT>::kBlocks) CacheAttentionKernel(const AttendParams p) {
  using G = Geometry<D, FP4, NT>;
  constexpr int kRows = 8 * NT, kSteps = D / 16, kGroups = G::kTile / 16;
  constexpr int kKeyBytes = G::kCodes / 4, kValueBytes = G::kCodes / 8;  // of a lane's part of a row
  constexpr int kKeyScales = FP4 ? D / 64 : 1;                           // E4M3 scales of that part
  constexpr int kValueChannels = D / 8, kTilesOfO = D / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, worker = static_cast<int>(blockIdx.x) * kWarps + warp;
  GridDependencyWait();
  if (p.parts != nullptr) GridLaunchDependents();  // the second kernel, which waits for all of this one; without it the caller's next one, which has no business here yet
  const Share share = FindShare(p, G::kTile);
  const int units = p.cache.heads * p.row_blocks;
  for (int seq = blockIdx.x; seq < p.seqs; seq += gridDim.x) {
    int length;
    if (TilesOf(p, seq, G::kTile, &length) > 0) continue;
    const long long rows = static_cast<long long>(p.tokens) * p.q_heads;
    uint4* const out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + seq * rows * D);
    for (long long i = threadIdx.x; i < rows * (D / 8); i += kThreads) out[i] = make_uint4(0, 0, 0, 0);
    for (long long i = threadIdx.x; p.lse != nullptr && i < rows; i += kThreads) p.lse[seq * rows + i] = -INFINITY;
    for (int i = threadIdx.x; p.parts != nullptr && i < units; i += kThreads) p.parts[static_cast<long long>(seq) * units + i] = make_int2(0, 0);
  }
  if (share.seq < 0) return;
  Segment at = FirstSegment(share);
  const int count = static_cast<int>(share.to - share.from);

  // ---- this warp's tiles
  const uint32_t ring = Smem(smem) + static_cast<uint32_t>(warp * G::kStages * G::kStage);
  Segment ahead = at;
  int next = 0, batch = 0, issued = 0;  // the tile that is copied next; the first one that `row` is of
  bool known = false;
  long long row = 0;     // lane i: where tile batch + i lies in the cache, or -1: in no page of it
  uint32_t present = 0;  // of the stages
  const int tiles_of_page = p.cache.page / G::kTile;
  auto copy = [&](uint32_t to, const uint8_t* from, auto bytes, auto swizzled) {
    constexpr int kBytes = decltype(bytes)::value;
#pragma unroll
    for (int i = 0; i < kBytes; i += 512) {
      const uint32_t at = static_cast<uint32_t>(i + 16 * lane);
      if (i + 512 <= kBytes || 16 * lane < kBytes - i) CopyAsync(to + (decltype(swizzled)::value ? G::Swizzled(at) : at), from + at);
    }
  };
  auto issue = [&] {
    if (next < count) {
      while (next >= ahead.end) {
        NextSegment(p, count, G::kTile, &ahead);
        known = false;
      }
      if (!known || next - batch >= 32) {
        batch = next;
        known = true;
        const int mine = next + lane;
        row = -1;
        if (mine < ahead.end) {
          const int tile = ahead.tile + mine - ahead.begin, page = tile / tiles_of_page, id = p.table[ahead.seq * p.ld_table + page];
          if (id >= 0 && id < p.cache.pages)
            row = (static_cast<long long>(id) * p.cache.heads + ahead.unit / p.row_blocks) * p.cache.page + (tile - page * tiles_of_page) * G::kTile;
        }
      }
      const long long from = __shfl_sync(0xffffffffu, row, next - batch), r = max(from, 0LL);
      present = (present & ~(1u << issued)) | (from >= 0 ? 1u << issued : 0u);
      const uint32_t to = ring + static_cast<uint32_t>(issued * G::kStage);
      copy(to, p.cache.k + r * G::kCodes, std::integral_constant<int, G::kTile * G::kCodes>(), std::true_type());
      copy(to + G::kTile * G::kCodes, static_cast<const uint8_t*>(p.cache.k_scale) + r * G::kScales, std::integral_constant<int, G::kTile * G::kScales>(), std::false_type());
      copy(to + G::kPart, p.cache.v + r * G::kCodes, std::integral_constant<int, G::kTile * G::kCodes>(), std::true_type());
      copy(to + G::kPart + G::kTile * G::kCodes, static_cast<const uint8_t*>(p.cache.v_scale) + r * G::kScales, std::integral_constant<int, G::kTile * G::kScales>(), std::false_type());
      issued = issued + 1 == G::kStages ? 0 : issued + 1;
      ++next;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // one a tile, of nothing behind the last
  };
#pragma unroll 1
  for (int i = 0; i < G::kStages; ++i) issue();

  // where this lane's parts of the tile's first tokens lie; sixteen, and eight, tokens on it is the same place
  constexpr int kKeyPieces = (kKeyBytes + 15) / 16, kValuePieces = (kValueBytes + 15) / 16;
  uint32_t key_at[kKeyPieces], value_at[2][kValuePieces];
#pragma unroll
  for (int i = 0; i < kKeyPieces; ++i) key_at[i] = G::Swizzled(static_cast<uint32_t>(g * G::kCodes + c * kKeyBytes + 16 * i));
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int i = 0; i < kValuePieces; ++i) {
      const uint32_t at_lane = static_cast<uint32_t>((2 * c + t) * G::kCodes + g * kValueBytes + 16 * i);
      value_at[t][i] = static_cast<uint32_t>(G::kPart) + (G::Swizzled(at_lane & ~15u) | (at_lane & 15u));
    }
  }

  int x = 0, stage = 0;
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
    {
      // q as FP16, and the factor from a row's products to its scores
      uint32_t q[NT][kSteps][2];
      float factor[NT][2];
      int sees[NT][2];  // tokens that a row may look at
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = row0 + 8 * n + g, token = r / p.group;
        const uint16_t* const from = static_cast<const uint16_t*>(p.q) + at.seq * p.ld_seq + token * p.ld_token + static_cast<long long>(head * p.group + r - token * p.group) * D;
        constexpr int kPieces = D / 32;  // of eight channels, this lane's part of the row
        uint4 raw[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) raw[i] = 8 * n + g < rows ? *reinterpret_cast<const uint4*>(from + c * (D / 4) + 8 * i) : make_uint4(0, 0, 0, 0);
        float v[D / 4];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(raw)[i];
          const float2 two = p.bf16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&w));
          v[2 * i] = two.x, v[2 * i + 1] = two.y;
          top = max(top, max(__float_as_uint(two.x) & 0x7FFFFFFFu, __float_as_uint(two.y) & 0x7FFFFFFFu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(9 - exponent) of the largest and its inverse; the exponent is kept where both are ordinary numbers
        const int e = min(max(static_cast<int>(top >> 23), 20), 254);  // 254: of the largest number there is
        const float up = __uint_as_float(static_cast<uint32_t>(263 - e) << 23);
        // of an infinity the scores may all be -infinity, which is not to pass for a row that sees nothing
        const float down = top >= 0x7F800000u ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(static_cast<uint32_t>(e - 9) << 23) * p.scale;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) q[n][i / 2][i % 2] = Pack16(v[2 * i] * up, v[2 * i + 1] * up);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          factor[n][h] = __shfl_sync(0xffffffffu, down, (2 * c + h) * 4);
          sees[n][h] = at.length - p.tokens + 1 + (row0 + 8 * n + 2 * c + h) / p.group;
        }
      }
      const int least_seen = at.length - p.tokens + 1;

#pragma unroll 1
      for (; x < at.end; ++x) {
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
#pragma unroll
            for (int i = 0; i < kKeyPieces; ++i) LoadShared<(kKeyBytes < 16 ? kKeyBytes : 16)>(tile + key_at[i] + static_cast<uint32_t>((16 * u + 8 * h) * G::kCodes), raw[h] + 4 * i);
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
              log_scale[u][h] = fminf(fmaxf(Log2(value_scale[u][h]), -60.f), kMostLogScale);
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
        // m is taken up where a weight is past 2^15, near FP16's largest (eight bits: past 2^8, as the sums of scores past 2^24 and logarithms are off by up to 2^8 themselves)
        constexpr float kBelow = FP4 ? 7.f : 0.f, kRoom = FP4 ? 15.f : 8.f;
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
            higher = higher || upto[n][r] - most[n][r] > kRoom;  // the difference is exact, however large they are
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
              m = fmaxf(m - kBelow, most[n][r]);
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
#pragma unroll
            for (int i = 0; i < kValuePieces; ++i)
              LoadShared<(kValueBytes < 16 ? kValueBytes : 16)>(tile + value_at[t & 1][i] + static_cast<uint32_t>((16 * u + 8 * (t >> 1)) * G::kCodes), raw[t] + 4 * i);
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

    // ---- the sums.  o[n][t][2 h + r] is channel g D / 8 + 2 t + h, row 8 n + 2 c + r.
    const bool whole_unit = at.tile == 0 && at.end - at.begin == at.tiles;
    float* const partial = p.partial + (static_cast<long long>(worker) * 2 + (at.tile > 0 ? 0 : 1)) * kRows * (D + 2);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float total = sum[n][r];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        const int of = 8 * n + 2 * c + r;
        if (of >= rows) continue;
        if (whole_unit) {
          const long long to = RowOf(p, at.seq, at.unit, row0 + of);
          const float by = total == 0.f ? 0.f : p.cache.v_unit / total;
          const uint32_t seen = total == 0.f ? 0u : ~0u;  // 0 times what a row does not see may be no number
          uint32_t w[kTilesOfO];
#pragma unroll
          for (int t = 0; t < kTilesOfO; ++t) w[t] = Packed(p.bf16, o[n][t][r] * by, o[n][t][2 + r] * by) & seen;
          uint4* const out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + to * D + g * kValueChannels);
#pragma unroll
          for (int t = 0; t < kTilesOfO / 4; ++t) out[t] = make_uint4(w[4 * t], w[4 * t + 1], w[4 * t + 2], w[4 * t + 3]);
          if (p.lse != nullptr && g == 0) p.lse[to] = LogOfSum(most[n][r], total);
        } else {
          float4* const out = reinterpret_cast<float4*>(partial + of * D + g * kValueChannels);
#pragma unroll
          for (int t = 0; t < kTilesOfO / 2; ++t) out[t] = make_float4(o[n][2 * t][r], o[n][2 * t][2 + r], o[n][2 * t + 1][r], o[n][2 * t + 1][2 + r]);
          if (g == 0) *reinterpret_cast<float2*>(partial + kRows * D + 2 * of) = make_float2(most[n][r], total);
        }
      }
    }
    if (at.tile == 0 && lane == 0 && p.parts != nullptr) {  // the first share of the unit says where the others are
      const long long last = share.from + at.begin + at.tiles - 1;
      p.parts[static_cast<long long>(at.seq) * units + at.unit] = whole_unit ? make_int2(0, 0) : make_int2(worker, ShareOf(share.all, last) - worker + 1);
    }
    if (at.end == count) break;
    NextSegment(p, count, G::kTile, &at);
  }
}

// The units that lie in several shares.  Of few parts, a row is a warp's; of many, a block's, whose warps each take every eighth.  Which of the two goes by the parts
// alone, so that the order of the sums does, too.  From how many on, us of both kernels: 4, 24, never.  16 sequences of 4000 tokens, four of them queries, 32 / 8 heads (10 parts a
// unit): 41.3, 34.3, 34.4; one of 1000, 64 / 8 heads (32 parts): 9.7, 9.7, 12.0; one of 131072, one key head: 28.8, 28.7, 94.
constexpr int kManyParts = 24;
template <int D>
__global__ void __launch_bounds__(kThreads) JoinKernel(const AttendParams p, int rows_of_unit) {
  constexpr int kMine = D / 32;  // channels of a lane
  __shared__ float sums[kWarps][D + 2];
  GridDependencyWait();
  const int units = p.cache.heads * p.row_blocks, warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const int2 parts = p.parts[blockIdx.x];
  const bool many = parts.y >= kManyParts;
  if (parts.y == 0) return;
  const int seq = static_cast<int>(blockIdx.x) / units, unit = static_cast<int>(blockIdx.x) - seq * units, row0 = unit % p.row_blocks * rows_of_unit;
  const int rows = min(rows_of_unit, p.tokens * p.group - row0);
  const long long slot = static_cast<long long>(rows_of_unit) * (D + 2);
  // the first part is of a share that goes on behind its unit's beginning, the others of shares that begin within the unit
  const auto part = [&](int k) { return p.partial + (static_cast<long long>(parts.x + k) * 2 + (k == 0 ? 1 : 0)) * slot; };
  const int rows_at_once = static_cast<int>(gridDim.y) * (many ? 1 : kWarps);
  for (int of = static_cast<int>(blockIdx.y) + (many ? 0 : static_cast<int>(gridDim.y) * warp); of < rows; of += rows_at_once) {
    // kAhead parts at a time, all of whose loads are on their way together
    constexpr int kAhead = D == 256 ? 4 : 8;
    const int step = many ? kWarps : 1;
    float all = -INFINITY, y[kMine] = {}, total = 0.f;
    for (int k0 = many ? warp : 0; k0 < parts.y; k0 += kAhead * step) {
      float2 ms[kAhead], v[kAhead][kMine / 2];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = k0 + i * step;
        ms[i] = make_float2(-INFINITY, 0.f);
        if (k < parts.y) {
          ms[i] = *reinterpret_cast<const float2*>(part(k) + rows_of_unit * D + 2 * of);
#pragma unroll
          for (int e = 0; e < kMine / 2; ++e) v[i][e] = *reinterpret_cast<const float2*>(part(k) + of * D + lane * kMine + 2 * e);
        }
      }
      float to = all;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) to = fmaxf(to, ms[i].x);
      const float again = to == -INFINITY ? 1.f : Exp2(all - to);
      total *= again;
#pragma unroll
      for (int e = 0; e < kMine; ++e) y[e] *= again;
      all = to;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (ms[i].x == -INFINITY) {
          total += ms[i].y;  // 0, or of a row that saw nothing but NaN
          continue;
        }
        const float by = Exp2(ms[i].x - all);
        total = fmaf(by, ms[i].y, total);
#pragma unroll
        for (int e = 0; e < kMine / 2; ++e) {
          y[2 * e] = fmaf(by, v[i][e].x, y[2 * e]);
          y[2 * e + 1] = fmaf(by, v[i][e].y, y[2 * e + 1]);
        }
      }
    }
    if (many) {
      __syncthreads();  // the row ahead has been read
#pragma unroll
      for (int e = 0; e < kMine; ++e) sums[warp][lane * kMine + e] = y[e];
      if (lane == 0) sums[warp][D] = total, sums[warp][D + 1] = all;
      __syncthreads();
      if (warp > 0) continue;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) all = fmaxf(all, sums[w][D + 1]);
#pragma unroll
      for (int e = 0; e < kMine; ++e) y[e] = 0.f;
      total = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float most = sums[w][D + 1], by = most == -INFINITY ? 1.f : Exp2(most - all);
        total = fmaf(by, sums[w][D], total);
#pragma unroll
        for (int e = 0; e < kMine; ++e) y[e] = fmaf(by, sums[w][lane * kMine + e], y[e]);
      }
    }
    const long long to = RowOf(p, seq, unit, row0 + of);
    const float by = total == 0.f ? 0.f : p.cache.v_unit / total;
    uint32_t* const out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + to * D + lane * kMine);
#pragma unroll
    for (int e = 0; e < kMine / 2; ++e) out[e] = Packed(p.bf16, y[2 * e] * by, y[2 * e + 1] * by);
    if (p.lse != nullptr && lane == 0) p.lse[to] = LogOfSum(all, total);
  }
}

struct Shape {
  int nt, row_blocks, blocks;
  bool cuts;  // shares may begin within a unit
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
  s.blocks = static_cast<int>(std::max(1LL, std::min(most, (tiles + kWarps - 1) / kWarps)));
  s.cuts = tiles > static_cast<long long>(c.seqs) * c.cache.heads * s.row_blocks;  // a unit may have more than one
  return s;
}

template <int D, bool FP4, int NT>
cudaError_t Launch(const AttendParams& p, const Shape& s, cudaStream_t stream) {
  using G = Geometry<D, FP4, NT>;
  static_assert(G::kStages >= 2 && G::kBlocks * (G::kBytes + 2048) <= 227 * 1024, "");
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
  if (err != cudaSuccess || !s.cuts) return err;
  // a block for each row of a unit, for those of many parts, as long as that makes no more blocks than run at once; else one for each eight rows (128 units of 16 rows, few
  // parts each: 31.9 us of both kernels with 2048 blocks, 29.6 with 256)
  const int units = p.seqs * p.cache.heads * p.row_blocks, rows = std::min(8 * NT, p.tokens * p.group);
  cfg.gridDim = dim3(static_cast<unsigned>(units), static_cast<unsigned>(std::clamp(2 * DeviceSmCount() / units, (rows + kWarps - 1) / kWarps, rows)));
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, JoinKernel<D>, p, 8 * NT);
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

// The parts of the units come first, on 16 bytes.
size_t PartsBytes(const CacheAttentionCall& c, const Shape& s) { return (sizeof(int2) * c.seqs * c.cache.heads * s.row_blocks + 15) / 16 * 16; }
size_t CacheAttentionWorkspace(const CacheAttentionCall& c) {
  const Shape s = ShapeOf(c);
  return !s.cuts ? 0 : PartsBytes(c, s) + sizeof(float) * s.blocks * kWarps * 2 * 8 * s.nt * (c.cache.dim + 2);
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
  if (static_cast<long long>(c.seqs) * c.cache.heads * s.row_blocks > INT_MAX) return cudaErrorInvalidValue;
  if (s.cuts) {
    p.parts = static_cast<int2*>(c.workspace);
    p.partial = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + PartsBytes(c, s));
  }
  p.out = c.out;
  p.lse = c.lse;
  p.bf16 = c.dtype == QFG_BFLOAT16;
  const cudaError_t err = c.cache.fp4 ? LaunchOf<true>(p, s, stream) : LaunchOf<false>(p, s, stream);
  const cudaError_t last = cudaGetLastError();
  return err == cudaSuccess ? last : err;
}

}  // namespace qfg
