// Attention of whole prompts: packed sequences of different lengths, causal or not, query heads in groups over key heads.
//
//   s_ij = scale q_i . k_j,  j within the sequence (causal: j <= i + keys - queries);   y_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)
//
// A block's item of work is one head's tiles of 128 queries, and the keys they see, 128 at a time: two tiles of heads of 128 channels, the block having the SM to itself, or one
// tile of heads of 64, two blocks an SM (packed prompts, one against two: 53 -> 44 us).  Both products are tcgen05.mma with FP32 sums in tensor memory: S = Q K^T from shared
// memory, and O += P V with P, in 16 bits, in tensor memory where S was.  A row of S belongs to one thread, so that the maximum and the sum of a row cross no lanes.  Two
// tiles take turns: while the tensor core works for the one, the other's four warps are at their exponentials.  Three quarters of the second product begin while the last
// quarter of P is made.
//
//   columns   S (of each tile) | O (of each), of 128 and D; P over the first half of its S
//   warps     0 products, 1 copies (and zeros in the place of values past the sequence's end), 2 and 3 idle, 4-7 softmax and output of the first tile, 8-11 of the second:
//             registers are shared out by four warps.  Two warpgroups for a tile, each half of a row's columns, were slower (1.1 to 1.4 ms), two warps for products no faster
//   ring      128 keys or 128 values a stage, by tensor copies; rows of 128 bytes, swizzled
//
// Where there are more blocks than the GPU holds, a block that is done takes on one that has not begun, and never will: the copies go on to its queries and keys while the last
// ones are worked on, and its first S is made while the rows ahead are written.  8192 tokens of 64 / 8 heads of 128: 871 us by itself without that, 813 with it; back to back, under
// the power cap, 890 and 840.  48 prompts of 256 tokens of 24 / 8 heads, back to back: 95 and 50.  Rows are written in runs of 64 bytes: a warp's 16 bytes of 32 rows at a time
// fill the queue of loads and stores, and waits and the next item's reading stand behind them.
//
// One pass: m is taken up only when a score passes it by 8 (in powers of two), and only then are O and the sum scaled again.  In FP16 weights are 2^7 times as large, up to 2^15: its
// smallest number is 2^-31 of the largest weight then, which keeps those of long sequences that are all small beside one.  S and the sums are FP32; P is rounded to the type of
// the inputs, as tensor cores take it (2^-8 or 2^-11 of each weight, before sums of many).
//
// Products and exponentials take the same time (a tile of 128 x 128 at D = 128: 1024 cycles of the tensor core, 1024 of the unit for exponentials at 16 a cycle), which is
// what bounds the kernel; a quarter of the exponentials goes to the FMA units for that reason.  No weight is made for tiles that the mask leaves out.  Causal, 8192 tokens of
// 64 / 8 heads of 128: 813 to 835 us by itself, 1.32 to 1.35 PFLOP/s, the tensor pipe busy for 72 % of the cycles; 830 to 940 back to back, by the power that the inputs take.
// Heads of 64: the softmax warps, two a scheduler, 650 instructions a tile each (S apart from P, so that the next is made meanwhile, changed nothing; 8192 tokens of 24 heads
// 260 us).
//
// Two tiles that take turns, a maximum that is seldom taken up, a part of the exponentials by a polynomial and P in the place of S are methods that have been published for
// attention on GPUs with tensor memory; sums that run along with a maximum are Milakov and Gimelshein's (2018).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstddef>
#include <type_traits>

#include "qfg_internal.h"
#include "stream_order.cuh"
#include "tc_ptx.cuh"
#include "tensor_map.h"

namespace qfg {
namespace {

constexpr int kTile = 128;
// Of sixteen pairs of weights those that the FMA units make, so that less waits for the unit for exponentials, which is an eighth as wide.  8192 tokens, us: of 24 heads of 64 none
// 280, two 267, four 263, six 277; of 64 heads of 128, by itself, none 848, four 829, and back to back, under the power cap, 863 to 874 and 860 to 870.
constexpr int kPolyOf16 = 4;
struct PromptParams {
  CUtensorMap q, k, v;
  const int *q_offsets, *k_offsets;
  void* out;
  float* lse;
  int seqs, q_rows, k_rows, q_heads, group;
  float scale, step;  // of scores, in powers of two; how far, before that, one may pass the highest ahead of it
  bool causal, waves, give_up;  // waves: there are more blocks than the GPU holds at once
};

// TILES: of queries, for a block.
template <int D, int TILES>
struct Geometry {
  static constexpr int kThreads = 128 + 128 * TILES, kBlocks = TILES == 1 ? 2 : 1;
  // Registers of a thread: the launch's for all are shared out, by four warps.  Two tiles: 168, 8 warps of 232 and 4 of 40 (together the 2016 that a lane of twelve warps
  // has).  One tile, two blocks an SM: 128, 4 warps of 208 and 4 of 48 (the 1024 of eight warps).
  static constexpr int kSoftmaxRegisters = TILES == 2 ? 232 : 208, kOtherRegisters = TILES == 2 ? 40 : 48;
  static_assert(TILES * 4 * kSoftmaxRegisters + 4 * kOtherRegisters <= (TILES == 2 ? 12 * 168 : 8 * 128), "");
  static constexpr int kColumns = TILES == 2 ? 512 : 256, kOutput = TILES * kTile;  // of tensor memory; where O begins
  static constexpr int kHeadTile = kTile * D * 2;                                   // bytes of 128 rows
  static constexpr int kStages = 5;
  static constexpr int kBytes = (TILES + kStages) * kHeadTile + 1024;
};

// Where a block's queries and keys lie.
struct Place {
  int q0, k0, queries, keys, first;  // first: the first of its queries, within the sequence; < 0: a block too many
};
// Work for all warps: a place, the head, and the tiles of keys that its tiles of queries look at.
struct Item {
  Place at;
  int head, tiles[2];
};
constexpr int kItems = 4;  // that the copies may be ahead
struct PromptCtl {
  uint4 next;  // the answer to this block's asking for another one's work
  unsigned long long q_full[2], q_empty[2], full[8], empty[8], fixed[8], s_full[2], o_full[2], item_full[kItems], next_full;  // of one arrival,
  unsigned long long p_most[2], p_ready[2], o_empty[2];                                                                      // of four warps',
  unsigned long long item_empty[kItems];                                                                                     // of all that take items
  Item item[kItems];
  int claimed;  // a block whose work is this one's, but not in `item` yet; -1: none
  uint32_t tmem;
  volatile uint32_t fault;
};

__device__ __forceinline__ void TmaLoad3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar),
               "r"(x), "r"(y), "r"(z)
               : "memory");
}
// The products of one k-step, 16 wide: operands OFF bytes (of tensor memory: columns) behind those that the lower words of the descriptors name, so that what differs
// from step to step takes no registers.  All operands in shared memory have rows of 128 bytes, swizzled, and 1024 bytes from eight rows to the next.
constexpr uint32_t kDescUpper = static_cast<uint32_t>(((1024ull >> 4) << 32 | 1ull << 46 | 2ull << 61) >> 32);
template <int OFF_A, int OFF_B>
__device__ __forceinline__ void MmaSsAt(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int add) {
  asm volatile("{ .reg .pred p;\n .reg .b32 x, y;\n .reg .b64 m, n;\n setp.ne.b32 p, %4, 0;\n add.u32 x, %1, %6;\n add.u32 y, %2, %7;\n mov.b64 m, {x, %5};\n"
               " mov.b64 n, {y, %5};\n tcgen05.mma.cta_group::1.kind::f16 [%0], m, n, %3, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(kDescUpper),
               "n"(OFF_A / 16), "n"(OFF_B / 16)
               : "memory");
}
template <int OFF_A, int OFF_B>
__device__ __forceinline__ void MmaTsAt(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int add) {
  asm volatile("{ .reg .pred p;\n .reg .b32 x, y;\n .reg .b64 n;\n setp.ne.b32 p, %4, 0;\n add.u32 x, %1, %6;\n add.u32 y, %2, %7;\n mov.b64 n, {y, %5};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], [x], n, %3, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(kDescUpper), "n"(OFF_A), "n"(OFF_B / 16)
               : "memory");
}
// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void LoadColumns(uint32_t a, float* f) {
  uint32_t* const v = reinterpret_cast<uint32_t*>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, "
      "%26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
        "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
        "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(a));
}
__device__ __forceinline__ void LoadColumns16(uint32_t a, float* f) {
  uint32_t* const v = reinterpret_cast<uint32_t*>(f);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                 "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(a));
}
__device__ __forceinline__ void StoreColumns16(uint32_t a, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(a), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
               "r"(v[14]), "r"(v[15])
               : "memory");
}
__device__ __forceinline__ void WaitLoads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void WaitStores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
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
__device__ __forceinline__ float2 Mul2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float MaxOrNan(float a, float b) {  // the larger one; NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^v for v <= 127 without the unit for exponentials: v = n + f with n whole and |f| <= 1/2, a polynomial for 2^f (the least relative error there: 7.5e-5 of degree 3, for
// weights in BF16; 2.6e-6 of degree 4, for FP16), and 2^n, whose exponent n is.  What is no number stays none: 2^n is a product's
// factor, as n added to the polynomial's exponent makes a number of a NaN.  From v = -126.5 down n is -127, for which the factor's bits are those of 0: a masked key weighs
// nothing, whatever its value.
template <bool BF16>
__device__ __forceinline__ float2 PolyExp2(float2 v) {
  const float2 round = make_float2(12582912.f, 12582912.f);  // 1.5 * 2^23
  v = make_float2(MaxOrNan(v.x, -127.f), MaxOrNan(v.y, -127.f));
  const float2 n = Add2(v, round), whole = Add2(n, make_float2(-12582912.f, -12582912.f)), f = Fma2(whole, make_float2(-1.f, -1.f), v);
  float2 r;
  if constexpr (BF16) {
    r = Fma2(f, make_float2(0.05517167f, 0.05517167f), make_float2(0.24261114f, 0.24261114f));
    r = Fma2(r, f, make_float2(0.69326097f, 0.69326097f));
    r = Fma2(r, f, make_float2(0.99992806f, 0.99992806f));
  } else {
    r = Fma2(f, make_float2(0.0095701022f, 0.0095701022f), make_float2(0.055917863f, 0.055917863f));
    r = Fma2(r, f, make_float2(0.24024744f, 0.24024744f));
    r = Fma2(r, f, make_float2(0.69312179f, 0.69312179f));
    r = Fma2(r, f, make_float2(0.99999928f, 0.99999928f));
  }
  const auto power = [](float whole) { return __int_as_float((__float_as_int(whole) << 23) + (127 << 23)); };
  return Mul2(r, make_float2(power(n.x), power(n.y)));
}
template <bool BF16>
__device__ __forceinline__ uint32_t Pack(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}

// BarWait without the pause of try_wait and in few instructions: for those that hold up the others.
__device__ __forceinline__ bool SpinWait(uint32_t a, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p;\n .reg .u32 n;\n mov.u32 n, 0;\n"
      "AGAIN:\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra.uni DONE;\n add.u32 n, n, 1;\n setp.lt.u32 p, n, %3;\n @p bra.uni AGAIN;\n"
      " setp.ne.u32 p, n, n;\nDONE:\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok) : "r"(a), "r"(parity), "n"(16 * kSpin) : "memory");
  return ok != 0;
}

// The same, until some warp of the block has given up.
__device__ __forceinline__ bool SpinWait(uint32_t a, uint32_t parity, const PromptCtl& c) {
  for (int i = 0; i < 16 * kSpin; ++i) {
    if (BarTest(a, parity)) return true;
    if ((i & 255) == 255 && c.fault) return false;
  }
  return false;
}

// Four pieces of 16 bytes of each lane's row: lane i of four gets piece i of their four rows instead, so that a store takes 64 bytes of a row and not 16.
__device__ __forceinline__ void Exchange(uint32_t (&w)[16], int lane) {
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    const bool upper = (lane & d) != 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i & 4 * d) continue;
      const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? w[i] : w[i + 4 * d], d);
      w[i] = upper ? got : w[i];
      w[i + 4 * d] = upper ? w[i + 4 * d] : got;
    }
  }
}

// A value that all lanes of the warp have, and the compiler knows it: what the instructions of the tensor core and their branches go by has to be so (else each product
// costs its issuing thread about 90 cycles, more than the tensor core takes for it).
template <typename T>
__device__ __forceinline__ T Uniform(T v) {
  return __shfl_sync(0xffffffffu, v, 0);
}

// Asks for a block of the grid that has not begun: it never will, and its work is this block's.  One asking at a time, and none behind the first that got nothing.
__device__ __forceinline__ void AskForBlock(uint4* answer, uint32_t bar) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  BarExpect(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(Smem(answer)), "r"(bar) : "memory");
}
__device__ __forceinline__ int BlockGot(const uint4* answer) {  // -1: none
  uint32_t block;
  asm volatile(
      "{ .reg .b128 r;\n .reg .pred p;\n ld.shared.b128 r, [%1];\n clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n mov.u32 %0, -1;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n}"
      : "=r"(block) : "r"(Smem(answer)) : "memory");
  return static_cast<int>(block);
}

// A sequence, and its blocks of ROWS queries.
template <int ROWS>
struct Sequence {
  int q0 = 0, queries = 0, k0 = 0, keys = 0, blocks = 0;
  __device__ __forceinline__ Sequence(const PromptParams& p, int i) {
    if (i < 0 || i >= p.seqs) return;
    const int q1 = p.q_offsets[i + 1], k1 = p.k_offsets[i + 1];
    q0 = min(max(p.q_offsets[i], 0), p.q_rows), k0 = min(max(p.k_offsets[i], 0), p.k_rows);
    queries = min(max(q1, q0), p.q_rows) - q0, keys = min(max(k1, k0), p.k_rows) - k0;
    blocks = (queries + ROWS - 1) / ROWS;
  }
  // its blocks whose last row sees more than `seen` keys: the last ones
  __device__ __forceinline__ int seeing(const PromptParams& p, int seen) const {
    if (seen < 0) return blocks;
    if (!p.causal) return keys > seen ? blocks : 0;
    // block i < blocks - 1 sees (i + 1) ROWS + keys - queries, the last one all
    return (keys > seen && blocks > 0 ? 1 : 0) + max(0, blocks - max(1, (seen + 1 - keys + queries + ROWS - 1) / ROWS));
  }
};
__device__ __forceinline__ int UpTo(int v, int lane) {  // the sum of this lane's and those ahead of it
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += u;
  }
  return v;
}
// The place of a block of the grid, by its rank among those of its head.  `from` is where the last search of many sequences ended, which is where the next one begins: ranks
// mostly rise (the last of 32 sequences, and the blocks ahead of them).  512 prompts of up to 300 tokens, 24 / 8 heads of 128: 745 us from the start, 458 so; 2000 of up to 30
// 4.0 and 1.08 ms.
struct Cursor {
  int base, before;
};
template <int ROWS>
__device__ __forceinline__ Place FindPlace(const PromptParams& p, int rank, Cursor* from) {
  const int lane = threadIdx.x & 31;
  // Where the GPU holds fewer blocks than there are, those with the most keys come first, so that none of them is the last to end; of up to 32 sequences, that is, which
  // a warp has at hand.  Of more, each one's last rows, which see the most keys, come ahead of its others.
  const bool sorted = p.waves && p.seqs > 1 && p.seqs <= 32;
  if (rank < from->before) *from = {p.seqs - 1, 0};
  int before = from->before;
  for (int base = from->base; base >= 0; base -= 32) {
    const Sequence<ROWS> s(p, base - lane);
    int mine = s.blocks, behind = 0;  // of this sequence's blocks: those that are counted, and those behind them, which come ahead of all that are
    if (sorted) {
      int lo = -1, hi = __reduce_max_sync(0xffffffffu, s.keys / kTile);  // the most tiles of keys that this block and those ahead of it look at are lo + 1
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (static_cast<int>(__reduce_add_sync(0xffffffffu, s.seeing(p, mid * kTile))) > rank) {
          lo = mid;
        } else {
          hi = mid - 1;
        }
      }
      behind = s.seeing(p, (lo + 1) * kTile);
      mine = s.seeing(p, lo < 0 ? -1 : lo * kTile) - behind;
      before = __reduce_add_sync(0xffffffffu, behind);
    }
    const int upto = UpTo(mine, lane);
    const uint32_t there = __ballot_sync(0xffffffffu, rank < before + upto);
    if (there != 0) {
      const int of = __ffs(there) - 1;
      const int back = behind + rank - before - (upto - mine);  // blocks of the sequence behind this one
      if (!sorted) *from = {base, before};
      return {__shfl_sync(0xffffffffu, s.q0, of), __shfl_sync(0xffffffffu, s.k0, of), __shfl_sync(0xffffffffu, s.queries, of), __shfl_sync(0xffffffffu, s.keys, of),
              __shfl_sync(0xffffffffu, (s.blocks - 1 - back) * ROWS, of)};
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return {0, 0, 0, 0, -1};
}
// The tiles of keys that 128 queries from `first` on look at.
__device__ __forceinline__ int KeyTiles(const PromptParams& p, const Place& at, int first) {
  if (first >= at.queries) return 0;
  const int last = min(at.queries, first + kTile) - 1;
  const int seen = p.causal ? min(at.keys, max(0, last + 1 + at.keys - at.queries)) : at.keys;
  return (seen + kTile - 1) / kTile;
}

template <int D, bool BF16, int TILES>
__global__ void __launch_bounds__(Geometry<D, TILES>::kThreads, Geometry<D, TILES>::kBlocks) PromptAttentionKernel(const __grid_constant__ PromptParams p) {
  using G = Geometry<D, TILES>;
  constexpr int kBoxes = D / 64, kBox = kTile * 128;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PromptCtl ctl;
  const int warp = Uniform(static_cast<int>(threadIdx.x) >> 5), lane = static_cast<int>(threadIdx.x) & 31;
  const uint32_t smem = (Smem(smem_raw) + 1023u) & ~1023u, ring = smem + TILES * G::kHeadTile;
  if (warp == 2) {
    constexpr int kFours = offsetof(PromptCtl, p_most), kItemEmpty = offsetof(PromptCtl, item_empty), kFirst = offsetof(PromptCtl, q_full);
    for (int at = kFirst + 8 * lane; at < kItemEmpty + 8 * kItems; at += 8 * 32) {
      BarInit(Smem(&ctl) + static_cast<uint32_t>(at), at < kFours ? 1 : at < kItemEmpty ? 4 : 4 * TILES + 1);
    }
    if (lane < kItems) ctl.item[lane].at.first = -1;
    if (lane == 0) {
      ctl.claimed = -1;
      ctl.fault = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Smem(&ctl.tmem)), "r"(G::kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 1 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.q) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.v) : "memory");
  }
  FenceBefore();
  GridDependencyWait();
  Place at = {0, 0, 0, 0, -1};
  Cursor cursor = {p.seqs - 1, 0};
  if (warp == 1) at = FindPlace<TILES * kTile>(p, static_cast<int>(blockIdx.x) / p.q_heads, &cursor);
  __syncthreads();
  FenceAfter();
  const uint32_t tmem = Uniform(ctl.tmem);
  // whether there is an n-th item, which is in `item` until this warp has done with it; a wait that runs out shows in `good`, which is the same for all lanes
  bool good = true;
  auto there = [&](int n) {
    good = __all_sync(0xffffffffu, SpinWait(Smem(&ctl.item_full[n % kItems]), static_cast<uint32_t>(n / kItems & 1), ctl)) != 0;
    return good && Uniform(ctl.item[n % kItems].at.first) >= 0;
  };
  auto done = [&](int n) {
    __syncwarp();
    if (lane == 0) BarArrive(Smem(&ctl.item_empty[n % kItems]));
  };

  if (warp >= 4) {
    // ---- softmax and output
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::kSoftmaxRegisters));
    const int t = (warp >> 2) - 1;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_at = tmem + lanes + static_cast<uint32_t>(t * kTile), o_at = tmem + lanes + static_cast<uint32_t>(G::kOutput + t * D);
    uint32_t s_parity = 0, o_parity = 0;
    const int in_block = t * kTile + (warp & 3) * 32 + lane;
#pragma unroll 1
    for (int n = 0; there(n); ++n) {
      const Item& item = ctl.item[n % kItems];
      const int keys = item.at.keys, count = item.tiles[t], over = keys - item.at.queries + 1 + item.at.first + in_block;  // what a causal row sees, if there is as much
      const int sees = p.causal ? min(keys, over) : keys, first_sees = p.causal ? min(keys, over - lane) : keys;          // first_sees: the warp's first row
      float limit = -INFINITY, offset = 0.f;  // a weight is 2^(scale s + offset), as long as no s is above the limit
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
      for (int j = 0; j < count; ++j) {
        good = __all_sync(0xffffffffu, BarWait(Smem(&ctl.s_full[t]), s_parity, ctl)) != 0;
        if (!good) break;
        s_parity ^= 1u;
        FenceAfter();
        float s[kTile];
#pragma unroll
        for (int i = 0; i < 4; ++i) LoadColumns(s_at + 32 * i, s + 32 * i);
        WaitLoads();
        if ((j + 1) * kTile > first_sees) {
          const int left = sees - j * kTile;
#pragma unroll
          for (int i = 0; i < kTile; ++i) s[i] = i < left ? s[i] : -INFINITY;
        }
        float m[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m[i] = fmaxf(s[i], s[i + 4]);
#pragma unroll
          for (int e = i + 8; e < kTile; e += 8) m[i] = fmaxf(fmaxf(m[i], s[e]), s[e + 4]);
        }
        const float highest = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        if (__any_sync(0xffffffffu, highest > limit)) {
          float by = 1.f;
          if (highest + p.step > limit) {
            // of scores past 2^23 the offset's rounding leaves FP16 no room for the 2^7; past 2^28 (BF16: 2^31) it may be that all weights are 0: the row is NaN
            const float most = highest * p.scale, bias = BF16 || !(fabsf(most) < 8388608.f) ? 0.f : 7.f;
            const float to = fabsf(most) < (BF16 ? 2147483648.f : 268435456.f) ? bias - most : __int_as_float(0x7FFFFFFF);
            by = limit == -INFINITY ? 0.f : Exp2(to - offset);
            limit = highest + p.step;
            offset = to;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) sum[i] = make_float2(sum[i].x * by, sum[i].y * by);
          if (j > 0) {  // the products of the tile ahead have ended: S, which was issued after them, has
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              float o[16];
              LoadColumns16(o_at + c, o);
              WaitLoads();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= by;
              StoreColumns16(o_at + c, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        const float2 scale2 = make_float2(p.scale, p.scale), offset2 = make_float2(offset, offset);
#pragma unroll
        for (int c = 0; c < kTile; c += 32) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 v = Fma2(make_float2(s[c + 2 * i], s[c + 2 * i + 1]), scale2, offset2);
            v = i * kPolyOf16 % 16 < kPolyOf16 ? PolyExp2<BF16>(v) : make_float2(Exp2(v.x), Exp2(v.y));
            sum[i & 1] = Add2(sum[i & 1], v);
            w[i] = Pack<BF16>(v.x, v.y);
          }
          StoreColumns16(s_at + c / 2, w);
          if (c >= kTile - 64) {  // three quarters of the product may begin while the last weights are made
            WaitStores();
            FenceBefore();
            __syncwarp();
            if (lane == 0) BarArrive(Smem(c == kTile - 64 ? &ctl.p_most[t] : &ctl.p_ready[t]));
          }
        }
      }
      if (count > 0 && good) good = __all_sync(0xffffffffu, BarWait(Smem(&ctl.o_full[t]), o_parity, ctl)) != 0;
      if (!good) break;
      FenceAfter();
      // 0: of a row that saw nothing; of keys whose scores are all -infinity nothing can be said
      const float all = (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y), total = limit == -INFINITY && sees > 0 ? __int_as_float(0x7FFFFFFF) : all;
      const float by = total == 0.f ? 0.f : 1.f / total;
      const int row = item.at.first + in_block;  // of the sequence
      const int rows = item.at.queries - (row & ~3);  // from the first of four lanes' on
      const long long to = (static_cast<long long>(item.at.q0) + row) * p.q_heads + item.head, step_of_row = static_cast<long long>(p.q_heads) * D;
      uint16_t* const out = static_cast<uint16_t*>(p.out) + to * D - (lane & 3) * step_of_row + (lane & 3) * 8;
      done(n);
#pragma unroll 1  // cold code
      for (int c = 0; c < D; c += 32) {
        uint32_t w[16] = {};
        if (count > 0) {
          float o[32];
          LoadColumns(o_at + c, o);
          WaitLoads();
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = total == 0.f ? 0u : Pack<BF16>(o[2 * i] * by, o[2 * i + 1] * by);  // 0 times what it does not see may be no number
          Exchange(w, lane);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i < rows) *reinterpret_cast<uint4*>(out + i * step_of_row + c) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
      }
      if (count > 0) {
        o_parity ^= 1u;
        FenceBefore();
        __syncwarp();
        if (lane == 0) BarArrive(Smem(&ctl.o_empty[t]));
      }
      if ((lane & 3) < rows && p.lse != nullptr) p.lse[to] = total == 0.f ? -INFINITY : (Log2(total) - offset) * 0.693147181f;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kOtherRegisters));
  }
  if (warp == 0) {
    // ---- products
    constexpr uint32_t kType = BF16 ? 1u << 7 | 1u << 10 : 0u;
    constexpr uint32_t kScores = 0x10u | kType | static_cast<uint32_t>(kTile >> 3) << 17 | 8u << 24;
    constexpr uint32_t kOutputs = 0x10u | kType | 1u << 16 | static_cast<uint32_t>(D >> 3) << 17 | 8u << 24;  // V: the columns of a row lie beside one another
    // descriptors' lower words: of Q, of the ring's first stage as keys and as values; they have one upper word
    const uint32_t q_desc = static_cast<uint32_t>(SmemDesc(smem, 16, 1024)), k_desc = static_cast<uint32_t>(SmemDesc(ring, 16, 1024)),
                   v_desc = static_cast<uint32_t>(SmemDesc(ring, kBox, 1024));
    constexpr uint32_t kStageStep = G::kHeadTile >> 4;
    auto wait = [&](uint32_t bar, uint32_t parity) {  // as every lane sees it: what follows is uniform to the compiler, too
      good = __all_sync(0xffffffffu, SpinWait(bar, parity)) != 0 && good;
    };
    // copies are waited for in their order: keys 0, values 0, keys 1, ..., ahead of what has to be waited for longer
    int next = 0;
    uint32_t parity = 0;
    auto arrived = [&] {
      const int stage = next;
      wait(Smem(&ctl.full[0]) + static_cast<uint32_t>(stage * 8), parity);
      if (++next == G::kStages) {
        next = 0;
        parity ^= 1u;
      }
      return stage;
    };
    auto release = [&](int stage) { MmaCommit<false>(Smem(&ctl.empty[0]) + static_cast<uint32_t>(stage * 8)); };
    uint32_t q_parity[2] = {0, 0}, p_parity[2] = {0, 0}, o_uses[2] = {0, 0}, fixes = 0;
    auto scores = [&](auto tile, int stage, bool last) {
      constexpr int t = decltype(tile)::value;
      const uint32_t a = q_desc + t * kStageStep, b = k_desc + static_cast<uint32_t>(stage) * kStageStep, d = tmem + t * kTile;
      MmaSsAt<0, 0>(d, a, b, kScores, 0);
      MmaSsAt<32, 32>(d, a, b, kScores, 1);
      MmaSsAt<64, 64>(d, a, b, kScores, 1);
      MmaSsAt<96, 96>(d, a, b, kScores, 1);
      if constexpr (D == 128) {
        MmaSsAt<kBox, kBox>(d, a, b, kScores, 1);
        MmaSsAt<kBox + 32, kBox + 32>(d, a, b, kScores, 1);
        MmaSsAt<kBox + 64, kBox + 64>(d, a, b, kScores, 1);
        MmaSsAt<kBox + 96, kBox + 96>(d, a, b, kScores, 1);
      }
      MmaCommit<false>(Smem(&ctl.s_full[t]));
      if (last) MmaCommit<false>(Smem(&ctl.q_empty[t]));
    };
    auto outputs = [&](auto tile, int j, int v, int k, int count) {  // of tile t, and its next scores
      constexpr int t = decltype(tile)::value;
      const uint32_t b = v_desc + static_cast<uint32_t>(v) * kStageStep, d = tmem + G::kOutput + t * D, a = tmem + t * kTile;
      if (j == 0 && o_uses[t]++ > 0) wait(Smem(&ctl.o_empty[t]), o_uses[t] & 1);  // the item ahead has been read
      wait(Smem(&ctl.p_most[t]), p_parity[t]);
      FenceAfter();
      if (good && ElectOne()) {
        MmaTsAt<0, 0>(d, a, b, kOutputs, j > 0);
        MmaTsAt<8, 2048>(d, a, b, kOutputs, 1);
        MmaTsAt<16, 4096>(d, a, b, kOutputs, 1);
        MmaTsAt<24, 6144>(d, a, b, kOutputs, 1);
        MmaTsAt<32, 8192>(d, a, b, kOutputs, 1);
        MmaTsAt<40, 10240>(d, a, b, kOutputs, 1);
      }
      __syncwarp();
      wait(Smem(&ctl.p_ready[t]), p_parity[t]);
      p_parity[t] ^= 1u;
      FenceAfter();
      if (good && ElectOne()) {
        MmaTsAt<48, 12288>(d, a, b, kOutputs, 1);
        MmaTsAt<56, 14336>(d, a, b, kOutputs, 1);
        if (j + 1 == count) {
          MmaCommit<false>(Smem(&ctl.o_full[t]));
        } else {
          scores(tile, k, j + 2 == count);
        }
      }
      __syncwarp();
    };
    const std::integral_constant<int, 0> first;
    const std::integral_constant<int, 1> second;
#pragma unroll 1
    for (int n = 0; good && there(n); ++n) {
      const Item& item = ctl.item[n % kItems];
      const int n0 = Uniform(item.tiles[0]), n1 = Uniform(item.tiles[1]), most = max(n0, n1);
      const bool fix = most * kTile > Uniform(item.at.keys);  // the last tile of values runs past the sequence's end
      done(n);
      if (most == 0) continue;
      if (n0 > 0) wait(Smem(&ctl.q_full[0]), q_parity[0]), q_parity[0] ^= 1u;
      if (TILES > 1 && n1 > 0) wait(Smem(&ctl.q_full[1]), q_parity[1]), q_parity[1] ^= 1u;
      const int k0 = arrived();
      FenceAfter();
      if (good && ElectOne()) {
        if (n0 > 0) scores(first, k0, n0 == 1);
        if constexpr (TILES > 1) {
          if (n1 > 0) scores(second, k0, n1 == 1);
        }
        release(k0);
      }
      __syncwarp();
#pragma unroll 1
      for (int j = 0; j < most && good; ++j) {
        const bool more = j + 1 < most;
        const int v = arrived(), k = more ? arrived() : 0;
        if (fix && !more) {
          wait(Smem(&ctl.fixed[0]) + static_cast<uint32_t>(v * 8), fixes >> v & 1);
          fixes ^= 1u << v;
        }
        if (j < n0) outputs(first, j, v, k, n0);
        if constexpr (TILES > 1) {
          if (j < n1) outputs(second, j, v, k, n1);
        }
        if (good && ElectOne()) {
          release(v);
          if (more) release(k);
        }
        __syncwarp();
      }
    }
    if (!good) ctl.fault = 1;
  } else if (warp == 1) {
    // ---- copies
    auto load = [&](uint32_t dst, const CUtensorMap* map, int of, int row, uint32_t bar) {
      if (ElectOne()) {
        BarExpect(bar, G::kHeadTile);
#pragma unroll
        for (int b = 0; b < kBoxes; ++b) TmaLoad3(dst + static_cast<uint32_t>(b * kBox), map, 64 * b, of, row, bar);
      }
      __syncwarp();
    };
    int stage = 0, items = 0, block = static_cast<int>(blockIdx.x);
    uint32_t parity = 1, q_uses[2] = {0, 0};  // a ring's first round waits for nothing: the phase ahead of the first has ended
    auto wait = [&](unsigned long long* bar, uint32_t of) { good = good && __all_sync(0xffffffffu, BarWait(Smem(bar), of, ctl)) != 0; };
    auto tell = [&](const Item& item) {  // all warps
      const int slot = items % kItems;
      wait(&ctl.item_empty[slot], static_cast<uint32_t>(items / kItems & 1) ^ 1u);
      if (lane == 0 && good) {
        ctl.item[slot] = item;
        ctl.claimed = -1;
        BarArrive(Smem(&ctl.item_full[slot]));
      }
      if (good) ++items;
      __syncwarp();
    };
    if (lane == 0) ctl.claimed = block;
    good = !p.give_up;
#pragma unroll 1
    for (uint32_t asked = 0; good; asked ^= 1u) {
      if (at.first >= 0) {
        const Item item = {at, block % p.q_heads, {KeyTiles(p, at, at.first), TILES == 1 ? 0 : KeyTiles(p, at, at.first + kTile)}};
        const int most = max(item.tiles[0], item.tiles[1]), of = item.head / p.group, keep = at.keys - (most - 1) * kTile;
        if (most == 0) tell(item);
        for (int position = 0; position < 2 * most && good; ++position) {
          wait(&ctl.empty[stage], parity);
          if (!good) break;
          const uint32_t to = ring + static_cast<uint32_t>(stage * G::kHeadTile);
          load(to, position & 1 ? &p.v : &p.k, of, at.k0 + (position >> 1) * kTile, Smem(&ctl.full[stage]));
          if (position == 0) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
              if (item.tiles[t] == 0) continue;
              wait(&ctl.q_empty[t], ++q_uses[t] & 1);
              if (good) load(smem + static_cast<uint32_t>(t * G::kHeadTile), &p.q, item.head, at.q0 + at.first + t * kTile, Smem(&ctl.q_full[t]));
            }
            tell(item);
          }
          if (position + 1 == 2 * most && keep < kTile) {
            // what lies past the sequence's end may be no number, and a weight of zero does not undo that
            wait(&ctl.full[stage], parity ^ 1u);
            const uint32_t zero[4] = {0, 0, 0, 0};
            for (int b = 0; b < kBoxes && good; ++b) {
              for (int i = lane; i < (kTile - keep) * 8; i += 32) Sts128(to + static_cast<uint32_t>(b * kBox + keep * 128 + i * 16), zero);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && good) BarArrive(Smem(&ctl.fixed[stage]));
          }
          if (++stage == G::kStages) {
            stage = 0;
            parity ^= 1u;
          }
        }
      }
      if (!good || !p.waves) break;
      if (lane == 0) AskForBlock(&ctl.next, Smem(&ctl.next_full));
      __syncwarp();
      // the answer comes in any case, and what it gives is this block's
      bool answered = false;
      for (int i = 0; i < kSpin && !answered; ++i) answered = BarTry(Smem(&ctl.next_full), asked);
      good = __all_sync(0xffffffffu, answered) != 0;
      block = answered ? BlockGot(&ctl.next) : -1;
      __syncwarp();
      if (block < 0) break;
      if (lane == 0) ctl.claimed = block;
      at = FindPlace<TILES * kTile>(p, block / p.q_heads, &cursor);
    }
    if (good) tell({{0, 0, 0, 0, -1}, 0, {0, 0}});
    if (!good) ctl.fault = 1;
  }
  if (ctl.fault != 0) {
    for (int i = 0; i < 16; ++i) __nanosleep(1000000);  // copies and products may still be under way
  }
  FenceBefore();
  __syncthreads();
  FenceAfter();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::kColumns) : "memory");
  if (ctl.fault != 0 && warp >= 4) {  // all rows of the last items, and of one that no warp has heard of
    const int thread = static_cast<int>(threadIdx.x) - 128;
    for (int i = 0; i <= kItems; ++i) {
      const int block = i < kItems ? -1 : ctl.claimed;
      const Place from = i < kItems ? ctl.item[i].at : block < 0 ? Place{0, 0, 0, 0, -1} : FindPlace<TILES * kTile>(p, block / p.q_heads, &cursor);
      const int head = i < kItems ? ctl.item[i].head : block % p.q_heads, rows = from.first < 0 ? 0 : min(TILES * kTile, from.queries - from.first);
      for (int e = thread; e < rows * (D / 8); e += 128 * TILES) {
        const long long to = (static_cast<long long>(from.q0) + from.first + e / (D / 8)) * p.q_heads + head;
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + to * D)[e % (D / 8)] = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
        if (p.lse != nullptr && e % (D / 8) == 0) p.lse[to] = __uint_as_float(0x7FFFFFFFu);
      }
    }
  }
}

bool EncodeHeads(CUtensorMap* map, const void* x, int dtype, int dim, int heads, int64_t rows, int64_t ld) {
  const TensorMapEncodeFn encode = TensorMapEncoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(dim) * 2, static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[3] = {64, 1, kTile}, one[3] = {1, 1, 1};
  return encode(map, dtype == QFG_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(x), dims, strides, box, one,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16, int TILES>
cudaError_t Launch(PromptParams p, cudaStream_t stream) {
  using G = Geometry<D, TILES>;
  static_assert(G::kBlocks * (G::kBytes + static_cast<int>(sizeof(PromptCtl)) + 1024) <= 228 * 1024, "");
  // sequences of any lengths that add up to the rows have no more tiles than this
  const long long blocks = (static_cast<long long>(p.q_rows) / (TILES * kTile) + std::min(p.seqs, p.q_rows)) * p.q_heads;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  p.waves = blocks > G::kBlocks * DeviceSmCount();
  const cudaError_t set = cudaFuncSetAttribute(PromptAttentionKernel<D, BF16, TILES>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kBytes);
  if (set != cudaSuccess) return set;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(G::kThreads);
  cfg.dynamicSmemBytes = G::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {OverlapAttribute()};
  cfg.attrs = attr;
  cfg.numAttrs = MayOverlapPredecessor(stream) ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, PromptAttentionKernel<D, BF16, TILES>, p);
}

}  // namespace

cudaError_t LaunchPromptAttention(const PromptCall& c, cudaStream_t stream) {
  PromptParams p = {};
  // without keys nothing is copied, and any map will do
  const bool keys = c.k_rows > 0;
  if (!EncodeHeads(&p.q, c.q, c.dtype, c.dim, c.q_heads, c.q_rows, c.ldq) ||
      !EncodeHeads(&p.k, keys ? c.k : c.q, c.dtype, c.dim, keys ? c.kv_heads : c.q_heads, keys ? c.k_rows : c.q_rows, keys ? c.ldk : c.ldq) ||
      !EncodeHeads(&p.v, keys ? c.v : c.q, c.dtype, c.dim, keys ? c.kv_heads : c.q_heads, keys ? c.k_rows : c.q_rows, keys ? c.ldv : c.ldq))
    return cudaErrorInvalidValue;
  p.q_offsets = c.q_offsets;
  p.k_offsets = c.k_offsets;
  p.out = c.out;
  p.lse = c.lse;
  p.seqs = c.seqs;
  p.q_rows = static_cast<int>(c.q_rows);
  p.k_rows = static_cast<int>(c.k_rows);
  p.q_heads = c.q_heads;
  p.group = c.q_heads / c.kv_heads;
  p.scale = c.scale * 1.44269504f;
  p.step = 8.f / p.scale;
  p.causal = c.causal;
  p.give_up = c.give_up;
  cudaError_t err;
  if (c.dtype == QFG_BFLOAT16) {
    err = c.dim == 64 ? Launch<64, true, 1>(p, stream) : Launch<128, true, 2>(p, stream);
  } else {
    err = c.dim == 64 ? Launch<64, false, 1>(p, stream) : Launch<128, false, 2>(p, stream);
  }
  const cudaError_t last = cudaGetLastError();
  return err == cudaSuccess ? last : err;
}

}  // namespace qfg
