// The product of eight-bit rows with an eight-bit weight: out[m, n] = sum_k x[m, k] w[k, n] * x_scale[m] * w_scale[n], INT8 summed
// in 32-bit integers (exact) or E4M3 in FP32, scaled in FP32 and rounded once.  The tensor core cuts an FP32 sum off to 24 bits, toward zero, at every
// instruction of 32 k: a choice that leaves sums of 17408 positive products 1.0e-5 too small, where a 16-bit output rounds by 2e-3 or 5e-4, and spares the
// epilogue's passes that adding in FP32 beside the tensor core would take.  Sums that K is split for lose less, each from zero (8 ways: 4.5e-7).
//
// A CTA computes tiles of 128 columns of w by `bm` rows of x (a multiple of 16, at most 256) with tcgen05.mma: the weight is the
// 128-row operand, so that one decoded token costs 16 columns of the instruction and not 128 rows; the rows of x are the bm-column
// operand.  Both come by tensor copies into 128-byte-swizzled shared memory, 128 bytes of k per stage, as they lie in memory: the
// weight with its columns contiguous (order n) is read MN-major, with k contiguous (order k) K-major.  Roles by warp:
//   0-3   epilogue: sums -> scaled -> the output; pairs have four more (6-9), since theirs took 4 us behind the last tile of 256 rows and takes 2
//   4     tensor copies of every stage; it makes the barriers too, and waits for nothing that the others set up
//   5     tensor memory; one lane issues the MMAs
//   6-21  LOADERS only: operands whose rows do not lie on 16 bytes, which a tensor copy cannot address; see CopyRole and ShiftRole
// SPLIT: the CTAs of a cluster share K, and add their sums through distributed shared memory in rank order.  PAIR: two CTAs work
// on 256 columns with cta_group::2, each with its own 128 columns of w and half of the rows of x.
//
// What bounds it, on one B200.  Few rows: the weights' way from memory.  1 x 5120 x 34816 30.0 us, 91 % of a copy's bandwidth, 1 x 5120 x 151936 117 to 120 (all of
// it); narrower weights have fewer CTAs than SMs hold, or ranks that meet: 8 x 5120 x 10240 12.1 us (8.0 at that bandwidth; 80 CTAs), 8 x 17408 x 5120 18.2 (13.6; 40 clusters),
// 1 x 5120 x 5120 7.0 (4.0; start, first trip to memory and the ranks' exchange are 3).  Many rows: the tensor pipe, 94 % of cycles at 4096 x 5120 x 34816, 420 us cold and
// 490 to 515 under the power cap (2.9 to 3.5 POP/s); fewer tiles than that the last wave, 509 x 5120 x 10240 32 us, tensor pipe 49 %.  Rows off 16 bytes: the
// instructions that move them, 1 us a stage of 208 rows (77 x 2561 x 5117 16.0 us).
//
// Every wait is bounded.  A CTA that gives up on one writes NaN to the rest of its tiles and leaves.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <map>
#include <mutex>
#include <new>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "qfg_internal.h"
#include "stream_order.cuh"
#include "tc_ptx.cuh"
#include "tensor_map.h"
#include "tile_walk.h"

namespace qfg {
namespace {

namespace cg = cooperative_groups;

constexpr int kTileN = 128;               // columns of w per CTA
constexpr int kTileK = 128;               // k per stage: one swizzled row of a K-major operand
constexpr int kWBytes = kTileN * kTileK;  // of a stage
constexpr int kRing = 12;                 // stages at most
constexpr int kCopyWarps = 8, kShiftWarps = 8;  // LOADERS; a warp copies the ninth pieces of 32 rows, so there are eight for tiles of 256
constexpr int kRawPitch = 144;            // bytes of a row as it is copied: 128 of them lie in nine aligned pieces of sixteen
constexpr int kRawMost = 4;               // stages of that at most
constexpr int kPitch = 80;                // bytes of a row of 32 columns in an epilogue warp's buffer: rows 16 bytes apart in the banks
constexpr int kWarpBuffer = 32 * kPitch + 256 * 4;  // that, and the warp's copy of its rows' scales
constexpr int kMostColumns = 512;           // of tensor memory
constexpr int kMaxSplit = 8;                // CTAs that share K
constexpr int kGroup = 8;                   // row blocks that the tiles go down before the next column block

struct QuantParams {
  CUtensorMap xmap, wmap;
  const uint8_t *x, *w;
  long long ldx, ldw, x_span, w_span;  // bytes from row to row; bytes from the first to the last
  const float *x_scale, *w_scale;
  void* out;
  long long ldo;
  int M, N, K, ksteps, bm, tiles, stages, sets, raw_stages;
  TileGrid grid;
  int order_k;           // the weight is stored [n][k]
  int x_loads, w_loads;  // LOADERS: which operands do not come by tensor copies
  int raw_at;            // where the rows of those are copied to, behind everything else
  int out_type;          // a qfg_dtype
  int out_vec;           // rows of the output lie on 16 bytes
  int early_weight;      // of a QuantCall; for single CTAs and tensor copies
  int give_up;           // testing: no stage comes
};

struct QuantCtl {
  unsigned long long full[kRing], empty[kRing], raw_full[kRawMost], raw_empty[kRawMost], acc_full[2], acc_empty[2];
  uint32_t tmem;
  volatile uint32_t fault;
};

template <bool FP8, bool PAIR>
__device__ __forceinline__ void MmaBytes(uint32_t d, unsigned long long a, unsigned long long b, uint32_t idesc, bool add) {
#define QFG_MMA(group, kind)                                                                                                                       \
  asm volatile("{ .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), \
               "l"(b), "r"(idesc), "r"(add ? 1 : 0)                                                                                                 \
               : "memory")
  if constexpr (FP8 && PAIR) {
    QFG_MMA("2", "f8f6f4");
  } else if constexpr (FP8) {
    QFG_MMA("1", "f8f6f4");
  } else if constexpr (PAIR) {
    QFG_MMA("2", "i8");
  } else {
    QFG_MMA("1", "i8");
  }
#undef QFG_MMA
}

// An accumulator as FP32: an integer sum is rounded to 24 bits here, the first of the result's roundings.
template <bool FP8>
__device__ __forceinline__ float Sum(uint32_t v) {
  return FP8 ? __uint_as_float(v) : __int2float_rn(static_cast<int>(v));
}
template <bool BF16>
__device__ __forceinline__ uint32_t Pack(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ void ClusterArrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void ClusterWait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// A pair shares a tile of twice the columns, and its second CTA has the upper half.
template <bool PAIR>
__device__ __forceinline__ At Locate(const QuantParams& p, int tile, int rank) {
  const At t = p.grid.Locate(tile);
  return {t.n0 + (PAIR ? rank * kTileN : 0), t.m0};
}

// ------------------------------------------------------------------------------ operands off 16 bytes
// Rows that tensor copies cannot address come in two steps.  Copying warps fetch the aligned pieces of sixteen bytes that hold a row's 128 into a ring of
// their own, asynchronously, and shifting warps move the rows from there to where the MMA reads them, sixteen bytes a lane.  Those have no copies of
// their own in flight: the proxy fence behind their stores would wait for them.  (One set of warps that loaded words and stored them took 2.8 us a
// stage of 208 rows, the two steps 1.)  No byte outside the tensor is read: the last piece is copied in part, and one that begins before the tensor byte by byte.
struct Unaligned {  // which rows a stage takes: the weight's, then those of x
  const uint8_t *x, *w;
  int w_rows, rows;
  __device__ __forceinline__ explicit Unaligned(const QuantParams& p)
      : x(BehindWait(p.x)), w(BehindWait(p.w)), w_rows(p.w_loads ? kTileK : 0), rows(w_rows + (p.x_loads ? p.bm : 0)) {}
};
struct StageRows {  // of an operand in one stage
  const uint8_t *row, *begin, *end;  // the first row's first byte; the tensor
  long long ld;
  int rows, valid;  // rows that the tensor has from there on, and bytes of each
};
__device__ __forceinline__ StageRows RowsOf(const QuantParams& p, const Unaligned& u, bool of_w, const At& t, int k0) {
  if (!of_w) return {u.x + t.m0 * p.ldx + k0, u.x, u.x + p.x_span, p.ldx, p.M - t.m0, min(kTileK, p.K - k0)};
  const int row = p.order_k ? t.n0 : k0, col = p.order_k ? k0 : t.n0;
  return {u.w + row * p.ldw + col, u.w, u.w + p.w_span, p.ldw, (p.order_k ? p.N : p.K) - row, min(kTileK, (p.order_k ? p.K : p.N) - col)};
}

// The first stage's copies are on their way before the barriers exist that later ones need, which `set_up` waits for.
template <typename F>
__device__ __forceinline__ void CopyRole(const QuantParams& p, QuantCtl& ctl, int warp, int lane, int kbeg, int kcount, int first_tile, int tile_step, uint32_t raw, F&& set_up) {
  const uint32_t full0 = Smem(&ctl.raw_full[0]), empty0 = Smem(&ctl.raw_empty[0]);
  const Unaligned u(p);
  const uint32_t slot_bytes = static_cast<uint32_t>(u.rows * kRawPitch);
  constexpr int kPass = 4 * kCopyWarps;
  const int sub = lane >> 3, piece = lane & 7, first = warp * 4 + sub;
  int slot = 0, round = 0;
  bool met = false;
  if (p.give_up) {
    set_up();
    return;
  }
  auto copy = [&](const StageRows& s, int stored, uint32_t to) {  // `stored`: rows that the stage has
    const int rows = min(s.rows, stored);
    const uint8_t* const last = s.row + (rows - 1) * s.ld + s.valid;
    if (rows > 0 && s.valid == kTileK && s.row - (reinterpret_cast<uintptr_t>(s.row) & 15) >= s.begin && last + 15 <= s.end) {
      // Whole rows, and no piece leaves the tensor: a warp takes eight pieces of four rows at a time, then the ninth of 32.
      const uint8_t* at = s.row + first * s.ld;
      const long long step = kPass * s.ld;
      uint32_t dst = to + static_cast<uint32_t>(first * kRawPitch + piece * 16);
#pragma unroll 4
      for (int r = first; r < rows; r += kPass) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(at - (reinterpret_cast<uintptr_t>(at) & 15) + 16 * piece) : "memory");
        at += step;
        dst += kPass * kRawPitch;
      }
      const int r = warp * 32 + lane;
      const uint8_t* const ninth = s.row + r * s.ld;
      const int off = static_cast<int>(reinterpret_cast<uintptr_t>(ninth) & 15);
      if (r < rows && off > 0) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + static_cast<uint32_t>(r * kRawPitch + 128)), "l"(ninth - off + 128) : "memory");
      return;
    }
    // Ends of rows or of the tensor: the same pieces, each as far as it goes.
    auto part = [&](int r, int c) {
      const uint8_t* const at = s.row + r * s.ld;
      const int off = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
      const uint8_t* const src = at + (16 * c - off);
      const uint32_t dst = to + static_cast<uint32_t>(r * kRawPitch + c * 16);
      if (r >= rows || 16 * c >= off + s.valid) return;
      if (src >= s.begin) {
        const long long left = s.end - src;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(static_cast<int>(left < 16 ? left : 16)) : "memory");
      } else {
        for (int e = 0; e < 16; ++e) {
          if (src + e >= s.begin && src + e < s.end) asm volatile("st.shared.u8 [%0], %1;" ::"r"(dst + e), "r"(static_cast<uint32_t>(src[e])) : "memory");
        }
        __threadfence_block();  // the arrival below is that of the copies
      }
    };
    for (int r = first; r < rows; r += kPass) part(r, piece);
    part(warp * 32 + lane, 8);
  };
  for (int tile = first_tile; tile < p.tiles; tile += tile_step) {
    const At t = Locate<false>(p, tile, 0);
    for (int k = 0; k < kcount; ++k) {
      if (round > 0 && !BarWait(empty0 + slot * 8, static_cast<uint32_t>((round - 1) & 1), ctl)) return;
      const uint32_t to = raw + static_cast<uint32_t>(slot) * slot_bytes;
      if (p.w_loads) copy(RowsOf(p, u, true, t, (kbeg + k) * kTileK), kTileK, to);
      if (p.x_loads) copy(RowsOf(p, u, false, t, (kbeg + k) * kTileK), p.bm, to + static_cast<uint32_t>(u.w_rows * kRawPitch));
      if (!met) set_up();
      met = true;
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full0 + slot * 8) : "memory");
      if (++slot == p.raw_stages) {
        slot = 0;
        ++round;
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");  // nothing lands behind the end of the block
}

__device__ __forceinline__ void ShiftRole(const QuantParams& p, QuantCtl& ctl, int warp, int lane, int kbeg, int kcount, int first_tile, int tile_step, uint32_t smem,
                                          uint32_t stage_bytes, uint32_t raw) {
  const uint32_t rfull0 = Smem(&ctl.raw_full[0]), rempty0 = Smem(&ctl.raw_empty[0]), full0 = Smem(&ctl.full[0]), empty0 = Smem(&ctl.empty[0]);
  const Unaligned u(p);
  const uint32_t slot_bytes = static_cast<uint32_t>(u.rows * kRawPitch);
  int slot = 0, stage = 0, round = 0;
  uint32_t raw_parity = 0;
  // A warp takes four rows at a time, sixteen bytes a lane, out of two aligned pieces: words apart, then bits.  (Five loads of words meet in the banks,
  // four lanes each.)  Its next rows are 32 on, at the same place in the swizzle.
  const int sub = lane >> 3, piece = lane & 7, first = warp * 4 + sub;
  const uint32_t swizzled = static_cast<uint32_t>(first * 128 + ((piece ^ (first & 7)) * 16));
  constexpr int kPass = 4 * kShiftWarps;
  auto shift = [&](const StageRows& s, int stored, bool zeros, uint32_t from, uint32_t to) {  // `zeros`: rows that the tensor does not have count
    const uint32_t low = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(s.row)), ld = static_cast<uint32_t>(s.ld);  // only the place in sixteen bytes counts
    const int rows = zeros ? s.rows : stored;
    const bool whole = s.valid == kTileK && rows >= stored;
    auto some = [&](int r0, auto steps) {  // rows r0, r0 + 32, ...
      constexpr int STEPS = decltype(steps)::value;
      uint32_t w[STEPS][8];
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        uint32_t lo[4], hi[4];
        const uint32_t at = from + static_cast<uint32_t>((r0 + j * kPass) * kRawPitch + 16 * piece);
        Lds128(at, lo);
        Lds128(at + 16, hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[j][i] = lo[i];
          w[j][4 + i] = hi[i];
        }
      }
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const int r = r0 + j * kPass;
        const uint32_t off = (low + static_cast<uint32_t>(r) * ld) & 15;
        uint32_t v[5];
#pragma unroll
        for (int i = 0; i < 6; ++i) w[j][i] = off & 8 ? w[j][i + 2] : w[j][i];
#pragma unroll
        for (int i = 0; i < 5; ++i) v[i] = off & 4 ? w[j][i + 1] : w[j][i];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __funnelshift_r(v[i], v[i + 1], (off & 3) * 8);
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int left = r < rows ? s.valid - 16 * piece - 4 * i : 0;
            if (left < 4) v[i] = left <= 0 ? 0u : v[i] & (0xFFFFFFFFu >> (32 - 8 * left));
          }
        }
        Sts128(to + static_cast<uint32_t>((r - first) * 128), v);
      }
    };
    int r = first;  // of a warp, all four rows exist or none: a stage has a multiple of sixteen
    for (; r - sub + 3 * kPass < stored; r += 4 * kPass) some(r, std::integral_constant<int, 4>());
    for (; r - sub < stored; r += kPass) some(r, std::integral_constant<int, 1>());
  };
  for (int tile = first_tile; tile < p.tiles; tile += tile_step) {
    const At t = Locate<false>(p, tile, 0);
    for (int k = 0; k < kcount; ++k) {
      if (round > 0 && !BarWait(empty0 + stage * 8, static_cast<uint32_t>((round - 1) & 1), ctl)) return;
      if (!BarWait(rfull0 + slot * 8, raw_parity, ctl)) return;
      const uint32_t from = raw + static_cast<uint32_t>(slot) * slot_bytes, to = smem + static_cast<uint32_t>(stage) * stage_bytes + swizzled;
      if (p.w_loads) shift(RowsOf(p, u, true, t, (kbeg + k) * kTileK), kTileK, !p.order_k, from, to);  // k past the end
      if (p.x_loads) shift(RowsOf(p, u, false, t, (kbeg + k) * kTileK), p.bm, false, from + static_cast<uint32_t>(u.w_rows * kRawPitch), to + kWBytes);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        BarArrive(full0 + stage * 8);
        BarArrive(rempty0 + slot * 8);
      }
      if (++stage == p.stages) {
        stage = 0;
        ++round;
      }
      if (++slot == p.raw_stages) {
        slot = 0;
        raw_parity ^= 1u;
      }
    }
  }
}

// ------------------------------------------------------------------------------ the kernel
template <bool PAIR, bool LOADERS>
constexpr int kThreads = 32 * (6 + (PAIR ? 4 : 0) + (LOADERS ? kCopyWarps + kShiftWarps : 0));

// SPLIT: one tile per cluster.  PAIR and the others never together.
template <bool FP8, bool PAIR, bool SPLIT, bool LOADERS>
__global__ void __launch_bounds__(kThreads<PAIR, LOADERS>, 1) QuantGemmKernel(const __grid_constant__ QuantParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ QuantCtl ctl;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t smem = (Smem(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem_ptr = smem_raw + (smem - Smem(smem_raw));
  const int csize = (PAIR || SPLIT) ? static_cast<int>(cg::this_cluster().num_blocks()) : 1;
  const int rank = (PAIR || SPLIT) ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
  const int first_tile = static_cast<int>(blockIdx.x) / csize, tile_step = static_cast<int>(gridDim.x) / csize;
  const int kbeg = SPLIT ? rank * p.ksteps / csize : 0;
  const int kcount = SPLIT ? (rank + 1) * p.ksteps / csize - kbeg : p.ksteps;
  const int xrows = PAIR ? p.bm / 2 : p.bm;
  const uint32_t stage_bytes = static_cast<uint32_t>(kWBytes + xrows * kTileK);
  const uint32_t full0 = Smem(&ctl.full[0]), empty0 = Smem(&ctl.empty[0]), accf0 = Smem(&ctl.acc_full[0]), acce0 = Smem(&ctl.acc_empty[0]);
  const bool load_w = !LOADERS || !p.w_loads, load_x = !LOADERS || !p.x_loads;
  constexpr int kEpilogueWarps = PAIR ? 8 : 4;
  int acc_cols = 32;
  while (acc_cols < p.sets * p.bm) acc_cols *= 2;
  // SPLIT: the rows of the tile that this rank finishes
  const int tile_rows = SPLIT ? min(p.bm, p.M - Locate<false>(p, first_tile, 0).m0) : 0, share = (p.bm + csize - 1) / csize;
  const int my_rows = max(0, min(share, tile_rows - rank * share));

  // The copying warp makes the barriers itself, so that its first copies are on their way while the other warps set up.
  StageWalk at(p.grid, first_tile);
  const uint32_t mine = static_cast<uint32_t>((load_w ? kWBytes : 0) + (load_x ? xrows * kTileK : 0));
  auto copy_stage = [&](bool w, bool x) {
    const uint32_t bar = PAIR ? MapRank(full0 + at.stage * 8, 0) : full0 + at.stage * 8;
    const uint32_t dst = smem + static_cast<uint32_t>(at.stage) * stage_bytes;
    const int k0 = (kbeg + at.k) * kTileK, n0 = at.at.n0 + (PAIR ? rank * kTileN : 0);
    if (ElectOne()) {
      if (w && (rank == 0 || !PAIR)) BarExpect(full0 + at.stage * 8, PAIR ? 2 * mine : mine);
      if (w && load_w) TmaLoad<PAIR>(dst, &p.wmap, p.order_k ? k0 : n0, p.order_k ? n0 : k0, bar);
      if (x && load_x) TmaLoad<PAIR>(dst + kWBytes, &p.xmap, k0, at.at.m0 + (PAIR ? rank * xrows : 0), bar);
    }
    __syncwarp();
    at.Next(p.grid, p.tiles, tile_step, kcount, p.stages);
  };
  const bool copies = p.give_up == 0 && (load_w || load_x), early = !PAIR && !LOADERS && p.early_weight != 0 && copies;
  if (warp == 4) {
    if (lane == 0) {
      if (load_x) asm volatile("prefetch.tensormap [%0];" ::"l"(&p.xmap) : "memory");
      if (load_w) asm volatile("prefetch.tensormap [%0];" ::"l"(&p.wmap) : "memory");
      for (int i = 0; i < p.stages; ++i) {
        BarInit(full0 + i * 8, (load_w || load_x ? 1 : 0) + (LOADERS ? kShiftWarps : 0));
        BarInit(empty0 + i * 8, 1);
      }
      for (int i = 0; i < 2; ++i) {
        BarInit(accf0 + i * 8, 1);
        BarInit(acce0 + i * 8, kEpilogueWarps * (PAIR ? 2 : 1));
      }
      for (int i = 0; LOADERS && i < p.raw_stages; ++i) {
        BarInit(Smem(&ctl.raw_full[i]), kCopyWarps * 32);
        BarInit(Smem(&ctl.raw_empty[i]), kShiftWarps);
      }
      ctl.fault = static_cast<uint32_t>(p.give_up);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  } else if (warp == 5) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Smem(&ctl.tmem)), "r"(acc_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Smem(&ctl.tmem)), "r"(acc_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  FenceBefore();
  const bool copier = LOADERS && warp >= 6 && warp < 6 + kCopyWarps;  // these come to the barrier with their first copies on their way
  if (copier) {
    GridDependencyWait();
  } else if (PAIR || warp != 4) {
    GridDependencyWait();
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads<PAIR, LOADERS>) : "memory");
  } else {  // this warp waits for nothing that the others set up, only they for its barriers
    asm volatile("bar.arrive 1, %0;" ::"n"(kThreads<PAIR, LOADERS>) : "memory");
    if (early) {  // a stage is full when its rows of x have come as well
      while (at.tile < p.tiles && at.round == 0) copy_stage(true, false);
      at = StageWalk(p.grid, first_tile);
    }
    GridDependencyWait();
  }
  if constexpr (PAIR) cg::this_cluster().sync();  // the leader's barriers exist before the peer arrives on them
  FenceAfter();
  const uint32_t tmem = PAIR || (warp != 4 && !copier) ? ctl.tmem : 0;

  if (warp < 4 || (PAIR && warp >= 6)) {
    // ---- epilogue; a warp reaches the 32 columns of w that its number says.  Of a pair's eight, two share them and take the rows by 32 in turn.
    const float* const x_scale = BehindWait(p.x_scale);
    const int quarter = warp & 3, half = warp >= 6 ? 1 : 0;
    uint8_t* const bufs = smem_ptr + static_cast<size_t>(p.stages) * stage_bytes + (quarter + 4 * half) * kWarpBuffer;
    const uint32_t buf = Smem(bufs);
    float* const xs = reinterpret_cast<float*>(bufs + 32 * kPitch);
    int it = 0;
    bool good = true;  // false from the first wait that ran out: the tiles that are left become NaN
    for (int tile = first_tile; tile < p.tiles; tile += tile_step, ++it) {
      const int b = p.sets == 2 ? it & 1 : 0, turn = p.sets == 2 ? it >> 1 : it;
      const At t = Locate<PAIR>(p, tile, rank);
      const int n = t.n0 + 32 * quarter;  // the warp's first column
      if constexpr (!SPLIT) {
        for (int i = lane; i < p.bm; i += 32) xs[i] = t.m0 + i < p.M ? x_scale[t.m0 + i] : 0.f;
        __syncwarp();
      }
      // asked for ahead of the wait: a trip to memory
      float ws[2][2] = {{1.f, 1.f}, {1.f, 1.f}};
      if (!SPLIT && p.w_scale != nullptr) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int col = p.out_type == QFG_FLOAT ? n + lane : n + 8 * h + (lane >> 2);
          if (col < p.N) ws[h >> 1][h & 1] = p.w_scale[col];
        }
      }
      good = good && BarWait(accf0 + b * 8, static_cast<uint32_t>(turn & 1), ctl);
      __syncwarp();
      FenceAfter();
      const uint32_t src = tmem + (static_cast<uint32_t>(32 * quarter) << 16) + static_cast<uint32_t>(b * p.bm);
      if (SPLIT || p.out_type == QFG_FLOAT) {
        // a lane is a column, a register a row
        // where the stages were: after a wait that ran out, copies may still be landing there
        for (int i = 0; SPLIT && i < 16 && !good; ++i) __nanosleep(1000000);
        for (int c = 16 * half; c < (SPLIT ? tile_rows : p.bm); c += PAIR ? 32 : 16) {
          uint32_t v[16];
          asm volatile(
              "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
              : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
              : "r"(src + static_cast<uint32_t>(c)));
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          if constexpr (SPLIT) {
            uint32_t* const part = reinterpret_cast<uint32_t*>(smem_ptr) + c * kTileN + 32 * quarter + lane;
#pragma unroll
            for (int i = 0; i < 16; ++i) part[i * kTileN] = v[i];
          } else if (n + lane < p.N) {
            float* const out = static_cast<float*>(p.out) + static_cast<long long>(t.m0 + c) * p.ldo + n + lane;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (t.m0 + c + i < p.M) out[i * p.ldo] = good ? Sum<FP8>(v[i]) * xs[c + i] * ws[0][0] : __uint_as_float(0x7FFFFFFFu);
            }
          }
        }
      } else {
        // 8 x 8 fragments, columns of w down and rows of x across, transposed through shared memory for stores of 16 bytes
        const int t2 = (lane & 3) * 2, row = lane >> 2, chunk = lane & 3;
        const int rows = min(p.bm, p.M - t.m0), cols = p.N - n;
        uint16_t* const out = static_cast<uint16_t*>(p.out) + static_cast<long long>(t.m0) * p.ldo + n;
        const uint32_t st = buf + static_cast<uint32_t>((((lane >> 4) & 1) * 8 + (lane & 7)) * kPitch + ((lane >> 3) & 1) * 16);
        const uint32_t ld = buf + static_cast<uint32_t>(row * kPitch + chunk * 16);
        auto finish = [&](auto type) {
          for (int c = 32 * half; c < p.bm; c += PAIR ? 64 : 32) {
            uint32_t v[2][2][8];  // [lower, upper 16 columns][16 rows][fragments]
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                if (k == 0 || c + 16 < p.bm) {
                  uint32_t(&f)[8] = v[h][k];
                  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                               : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]), "=r"(f[4]), "=r"(f[5]), "=r"(f[6]), "=r"(f[7])
                               : "r"(src + (static_cast<uint32_t>(16 * h) << 16) + static_cast<uint32_t>(c + 16 * k)));
                }
              }
            }
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            __syncwarp();  // the rows before have been read
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if (k == 0 || c + 16 < p.bm) {
                const float2 s0 = *reinterpret_cast<const float2*>(xs + c + 16 * k + t2), s1 = *reinterpret_cast<const float2*>(xs + c + 16 * k + 8 + t2);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  uint32_t w[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const float2 s = i < 2 ? s0 : s1;
                    const float lo = Sum<FP8>(v[h][k][2 * i]) * s.x * ws[h][i & 1], hi = Sum<FP8>(v[h][k][2 * i + 1]) * s.y * ws[h][i & 1];
                    w[i] = good ? Pack<decltype(type)::value>(lo, hi) : 0x7FFF7FFFu;
                  }
                  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(st + k * (16 * kPitch) + h * 32), "r"(w[0]),
                               "r"(w[1]), "r"(w[2]), "r"(w[3])
                               : "memory");
                }
              }
            }
            __syncwarp();
            if (p.out_vec && cols >= 32) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = c + 8 * i + row;
                if (r < rows) {
                  uint32_t o[4];
                  Lds128(ld + i * (8 * kPitch), o);
                  *reinterpret_cast<uint4*>(out + static_cast<long long>(r) * p.ldo + 8 * chunk) = make_uint4(o[0], o[1], o[2], o[3]);
                }
              }
            } else {
              const uint16_t* const from = reinterpret_cast<const uint16_t*>(bufs) + lane;
              const int last = min(32, rows - c);
              for (int r = 0; r < last; ++r) {
                if (lane < cols) out[static_cast<long long>(c + r) * p.ldo + lane] = from[r * (kPitch / 2)];
              }
            }
          }
        };
        if (p.out_type == QFG_BFLOAT16) {
          finish(std::true_type());
        } else {
          finish(std::false_type());
        }
      }
      FenceBefore();
      __syncwarp();
      if (lane == 0 && good) BarArriveLeader<PAIR>(acce0 + b * 8);
    }
  } else if (warp == 4) {
    // ---- tensor copies
    while (copies && at.tile < p.tiles && (at.round == 0 || BarWait(empty0 + at.stage * 8, static_cast<uint32_t>((at.round - 1) & 1), ctl)))
      copy_stage(!early || at.round > 0, true);
  } else if (warp == 5) {
    // ---- MMAs (the leader's, for both CTAs of a pair)
    if (!PAIR || rank == 0) {
      // sums in FP32 (1) or integers (2), operands E4M3 (0) or signed bytes (1), the weight MN-major in order n, N = bm, M = 128 (256 across a pair)
      const uint32_t idesc = (FP8 ? 1u << 4 : (2u << 4) | (1u << 7) | (1u << 10)) | (p.order_k ? 0u : 1u << 15) | (static_cast<uint32_t>(p.bm >> 3) << 17) |
                             (static_cast<uint32_t>(PAIR ? 16 : 8) << 24);
      const unsigned long long a0 = SmemDesc(smem, kWBytes, 1024), b0 = SmemDesc(smem + kWBytes, 16, 1024);
      const uint32_t a_step = p.order_k ? 32 >> 4 : 4096 >> 4;  // 32 k on
      int stage = 0, it = 0;
      uint32_t parity = 0;
      bool good = true, ready = false;
      for (int tile = first_tile; tile < p.tiles && good; tile += tile_step, ++it) {
        const int b = p.sets == 2 ? it & 1 : 0, turn = p.sets == 2 ? it >> 1 : it;
        if (turn > 0 && !BarWait(acce0 + b * 8, static_cast<uint32_t>((turn - 1) & 1), ctl)) break;
        FenceAfter();
        const uint32_t d = tmem + static_cast<uint32_t>(b * p.bm);
        for (int k = 0; k < kcount; ++k) {
          if (!ready && !BarWait(full0 + stage * 8, parity, ctl)) {
            good = false;
            break;
          }
          FenceAfter();
          const uint32_t off = static_cast<uint32_t>(stage) * stage_bytes >> 4, done = empty0 + stage * 8;
          if (++stage == p.stages) {
            stage = 0;
            parity ^= 1u;
          }
          ready = BarTest(full0 + stage * 8, parity);  // asked before the MMAs are issued, needed after
          if (ElectOne()) {
#pragma unroll
            for (int i = 0; i < kTileK / 32; ++i) MmaBytes<FP8, PAIR>(d, a0 + off + i * a_step, b0 + off + i * (32 >> 4), idesc, k > 0 || i > 0);
            MmaCommit<PAIR>(done);
            if (k == kcount - 1) MmaCommit<PAIR>(accf0 + b * 8);
          }
          __syncwarp();
        }
      }
    }
  } else if constexpr (LOADERS) {
    const uint32_t raw = smem + static_cast<uint32_t>(p.raw_at);
    if (copier) {
      CopyRole(p, ctl, warp - 6, lane, kbeg, kcount, first_tile, tile_step, raw,
               [] { asm volatile("bar.sync 1, %0;" ::"n"(kThreads<PAIR, LOADERS>) : "memory"); });
    } else {
      ShiftRole(p, ctl, warp - 6 - kCopyWarps, lane, kbeg, kcount, first_tile, tile_step, smem, stage_bytes, raw);
    }
  }

  if constexpr (SPLIT) {
    // The ranks' sums meet: rank r finishes rows [r share, (r + 1) share) of the tile, adding in rank order.  (Sums sent ahead to the rank that adds them,
    // which spares one of the two times that the ranks meet, were no faster: 8 x 5120 x 10240 in threes 13.3 us, read from where they are 13.0.)
    cg::cluster_group cluster = cg::this_cluster();
    const At t = Locate<false>(p, first_tile, 0);
    const float* const x_scale = BehindWait(p.x_scale);
    const int c = lane * 4, n = t.n0 + c, cols = p.N - n, m_first = t.m0 + rank * share;
    const int warps = static_cast<int>(blockDim.x) / 32;
    // asked for ahead of the waits: trips to memory
    float ws[4], x_first = warp < my_rows ? x_scale[m_first + warp] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ws[e] = p.w_scale != nullptr && e < cols ? p.w_scale[n + e] : 1.f;
    FenceBefore();
    ClusterArrive();
    ClusterWait();
    bool bad = false;  // a rank gave up
#pragma unroll
    for (int r = 0; r < kMaxSplit; ++r) {
      if (r < csize) bad |= *cluster.map_shared_rank(const_cast<const uint32_t*>(&ctl.fault), r) != 0;
    }
    // ROWS rows a warp at a time, so that the loads of all of them and of all ranks are on their way together
    auto add_up = [&](auto rows_tag, auto ranks_tag) {
      constexpr int ROWS = decltype(rows_tag)::value, RANKS = decltype(ranks_tag)::value;
      for (int m0 = warp; m0 < my_rows; m0 += warps * ROWS) {
        uint4 v[ROWS][RANKS];
        float xs[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int m = m0 + i * warps;
          xs[i] = m == warp ? x_first : m < my_rows ? x_scale[m_first + m] : 0.f;
#pragma unroll
          for (int r = 0; r < RANKS; ++r) {
            if (r < csize && m < my_rows) {
              v[i][r] = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(reinterpret_cast<const uint32_t*>(smem_ptr), r) + (rank * share + m) * kTileN + c);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int m = m0 + i * warps;
          if (m >= my_rows) break;
          uint32_t s[4] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w};
#pragma unroll
          for (int r = 1; r < RANKS; ++r) {
            if (r < csize) {
              const uint32_t a[4] = {v[i][r].x, v[i][r].y, v[i][r].z, v[i][r].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) s[e] = FP8 ? __float_as_uint(__uint_as_float(s[e]) + __uint_as_float(a[e])) : s[e] + a[e];
            }
          }
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = bad ? __uint_as_float(0x7FFFFFFFu) : Sum<FP8>(s[e]) * xs[i] * ws[e];
          const long long at = static_cast<long long>(m_first + m) * p.ldo + n;
          if (p.out_type == QFG_FLOAT) {
            float* const dst = static_cast<float*>(p.out) + at;
            if (p.out_vec && cols >= 4) {
              *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (e < cols) dst[e] = y[e];
              }
            }
          } else {
            uint16_t* const dst = static_cast<uint16_t*>(p.out) + at;
            const uint2 o = p.out_type == QFG_BFLOAT16 ? make_uint2(Pack<true>(y[0], y[1]), Pack<true>(y[2], y[3]))
                                                       : make_uint2(Pack<false>(y[0], y[1]), Pack<false>(y[2], y[3]));
            if (p.out_vec && cols >= 4) {
              *reinterpret_cast<uint2*>(dst) = o;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (e < cols) dst[e] = static_cast<uint16_t>((e < 2 ? o.x : o.y) >> (16 * (e & 1)));
              }
            }
          }
        }
      }
    };
    if (csize <= 2) {
      add_up(std::integral_constant<int, 4>(), std::integral_constant<int, 2>());
    } else if (csize <= 4) {
      add_up(std::integral_constant<int, LOADERS ? 2 : 4>(), std::integral_constant<int, 4>());
    } else {
      add_up(std::integral_constant<int, LOADERS ? 1 : 2>(), std::integral_constant<int, kMaxSplit>());
    }
  }
  if constexpr (SPLIT) ClusterArrive();  // nothing more is read from the others
  if (ctl.fault) __nanosleep(100000);  // copies of a CTA that gave up may still be landing
  FenceBefore();
  __syncthreads();
  if constexpr (PAIR) cg::this_cluster().sync();  // no CTA leaves while its peer's MMAs still read its shared memory
  if constexpr (SPLIT) ClusterWait();
  if (warp == 5) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(acc_cols) : "memory");
    } else {
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(acc_cols) : "memory");
    }
  }
}

// ------------------------------------------------------------------------------ host
constexpr int kSmemPerSm = 233472;                                      // of an SM; a CTA takes 1 KB of it beside its own
constexpr int kStatic = (static_cast<int>(sizeof(QuantCtl)) + 127) / 128 * 128;
// bytes beside the stages
int Fixed(const QuantPlan& plan) {
  return 1024 + (plan.pair ? 8 : 4) * kWarpBuffer;
}

int SmemLimit(int per_sm) { return kSmemPerSm / per_sm - 1024 - kStatic; }

bool EncodeRows(CUtensorMap* map, const uint8_t* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)}, step[2] = {1, 1};
  const TensorMapEncodeFn fn = TensorMapEncoder();
  return fn != nullptr && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool FP8, bool PAIR, bool SPLIT, bool LOADERS>
cudaError_t LaunchAs(const QuantParams& p, int ctas, int cluster, size_t smem, bool overlap, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(kThreads<PAIR, LOADERS>));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (cluster > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (overlap) attr[cfg.numAttrs++] = OverlapAttribute();
  return cudaLaunchKernelEx(&cfg, QuantGemmKernel<FP8, PAIR, SPLIT, LOADERS>, p);
}

// ------------------------------------------------------------------------------ set-up, once per device
struct QuantSetup {
  int device, sms;
  int slots[3][kMaxSplit + 1];  // [CTAs an SM holds][cluster size]: clusters that are resident at once
};
std::mutex g_quant_mu;
std::map<int, QuantSetup> g_quant;
std::atomic<const QuantSetup*> g_quant_last{nullptr};

template <bool FP8>
cudaError_t RaiseLimits() {
  cudaError_t err = cudaSuccess;
  auto raise = [&](auto* kernel) {
    if (err == cudaSuccess) err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SmemLimit(1));
  };
  raise(QuantGemmKernel<FP8, true, false, false>);
  raise(QuantGemmKernel<FP8, false, false, false>);
  raise(QuantGemmKernel<FP8, false, true, false>);
  raise(QuantGemmKernel<FP8, false, false, true>);
  raise(QuantGemmKernel<FP8, false, true, true>);
  return err;
}

int ResidentClusters(int per_sm, int cluster, int sms) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(cluster));
  cfg.blockDim = dim3(static_cast<unsigned>(kThreads<false, false>));
  cfg.dynamicSmemBytes = static_cast<size_t>(SmemLimit(per_sm));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, QuantGemmKernel<false, false, true, false>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = std::max(1, per_sm * sms * 8 / (10 * cluster));
  }
  return n;
}

cudaError_t SetUpQuant(const QuantSetup** out) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  *out = g_quant_last.load(std::memory_order_acquire);
  if (*out != nullptr && (*out)->device == dev) return cudaSuccess;
  std::lock_guard<std::mutex> lock(g_quant_mu);
  auto it = g_quant.find(dev);
  if (it == g_quant.end()) {
    QuantSetup s = {dev, 0, {}};
    err = cudaDeviceGetAttribute(&s.sms, cudaDevAttrMultiProcessorCount, dev);
    if (err == cudaSuccess) err = RaiseLimits<false>();
    if (err == cudaSuccess) err = RaiseLimits<true>();
    if (err != cudaSuccess) return err;
    for (int per_sm = 1; per_sm <= 2; ++per_sm) {
      for (int c = 1; c <= kMaxSplit; ++c) s.slots[per_sm][c] = c == 1 ? per_sm * s.sms : ResidentClusters(per_sm, c, s.sms);
    }
    it = g_quant.emplace(dev, s).first;
  }
  *out = &it->second;
  g_quant_last.store(*out, std::memory_order_release);
  return cudaSuccess;
}

bool OnSixteen(const void* base, int64_t pitch) { return reinterpret_cast<uintptr_t>(base) % 16 == 0 && pitch % 16 == 0; }

}  // namespace

cudaError_t ConfigureQuantKernels() {
  const QuantSetup* setup = nullptr;
  return SetUpQuant(&setup);
}

// Launch shape: rows per tile, CTAs that split K, pairs, CTAs per SM.  The cheapest by a model of a call's time in us, fitted to calls in graphs on one
// B200: 413 random shapes (1 to 2048 rows, K 256 to 17408, N 256 to 152000), up to 131 launch shapes each, kept in profiles/quant_gemm_launch_shapes.csv; the shape
// chosen takes 1.8 % longer than the best one on average (the worst: 197 x 13840 x 2880 27 us against 19 in other rows per tile).  Rows off 16 bytes have a fit of
// their own (142 shapes, 0.6 %).
//   blocks of 128 k in turn, `waves` times; or what the CTAs fetch through L2; or memory: the longest, and a part of the shorter
//   around that what a call takes anyway, with the last tile's epilogue, and where K is split, the ranks' exchange
// More row tiles than needed are tried because they can fill the last wave better (509 x 5120 x 10240: three of 192 28 us, two of 256 32).
struct QuantCost {
  double step_least, step_row;   // of a block: at least, and for each row of the tile
  double call, call_row, wave;   // around the blocks; of a further wave
  double join, join_row, join_rank;
  double memory, l2;             // bytes a us
  double rest;                   // of the shorter of the two
};
constexpr double kAny = 1e30;
constexpr QuantCost kSingle = {0.125, 0.0019, 2.6, 0.0149, 0.3, 0.565, 0.0216, 0.027, 11.5e6, 16.8e6, 0.1};
constexpr QuantCost kPair = {0.102, 0.00134, 3.9, 0.0054, 0.73, 0, 0, 0, 11.5e6, 16.8e6, 0.1};
constexpr QuantCost kUnaligned = {0.22, 0.00104, 0.6, 0.001, 2.6, 0.31, 0.0028, 0.027, 5.4e6, kAny, 0.41};
constexpr double kShared = 1.17;  // a block of two CTAs on an SM, in the sum of what it takes at least and for its rows

QuantPlan ChooseQuantPlan(const QuantCall& c) {
  const QuantSetup* setup = nullptr;
  if (SetUpQuant(&setup) != cudaSuccess) throw std::runtime_error("QuantGemm: the kernels could not be set up on this device");
  const bool loads = !OnSixteen(c.x, c.ldx) || !OnSixteen(c.w, c.ldw);
  const int64_t blocks = (c.k + kTileK - 1) / kTileK, least = (c.m + 255) / 256;
  const double bytes = static_cast<double>(c.k) * c.n + static_cast<double>(c.m) * c.k + 2.0 * c.m * c.n;
  QuantPlan best;
  double best_cost = kAny;
  auto consider = [&](const QuantPlan& plan) {
    const QuantCost& q = loads ? kUnaligned : plan.pair ? kPair : kSingle;
    const int64_t tiles = ((c.m + plan.bm - 1) / plan.bm) * ((c.n + (plan.pair ? 2 * kTileN : kTileN) - 1) / (plan.pair ? 2 * kTileN : kTileN));
    const int64_t slots = plan.pair ? setup->sms / 2 : setup->slots[plan.per_sm][plan.split];
    if (slots < 1) return;
    const int64_t waves = (tiles + slots - 1) / slots, each = (blocks + plan.split - 1) / plan.split;
    const int64_t ctas = tiles * plan.split * (plan.pair ? 2 : 1);
    double step = std::max(q.step_least, q.step_row * plan.bm);
    if (plan.per_sm == 2 && std::min(ctas, slots * plan.split) > setup->sms) step = std::max(step, kShared * (q.step_least + q.step_row * plan.bm));
    const double walk = static_cast<double>(waves * each) * step + q.wave * static_cast<double>(waves - 1);
    const double l2 = static_cast<double>(ctas * each) * (kTileN + (plan.pair ? plan.bm / 2 : plan.bm)) * kTileK / q.l2;
    const double fetch = std::max(l2, bytes / q.memory);
    const double join = plan.split == 1 ? 0.0 : q.join + q.join_row * plan.bm * (plan.split - 1) / plan.split + q.join_rank * (plan.split - 1);
    const double cost = std::max(walk, fetch) + q.rest * std::min(walk, fetch) + q.call + q.call_row * plan.bm + join;
    if (cost < best_cost) {
      best_cost = cost;
      best = plan;
    }
  };
  // from the tallest tiles on, each height once: the next is that of the first count of row tiles that allows a lower one
  for (int64_t mt = least; mt <= 2 * least + 2 && mt <= c.m;) {
    QuantPlan plan;
    plan.bm = static_cast<int>(((c.m + mt - 1) / mt + 15) / 16 * 16);
    mt = plan.bm > 16 ? (c.m + plan.bm - 17) / (plan.bm - 16) : c.m + 1;
    for (plan.per_sm = 1; plan.per_sm <= (loads ? 1 : 2); ++plan.per_sm) {
      for (plan.split = 1; plan.split <= std::min<int64_t>(kMaxSplit, blocks); ++plan.split) consider(plan);
    }
    if (!loads) consider({(plan.bm + 31) / 32 * 32, 1, 1, 1});
  }
  return best;
}

struct Ready {
  QuantParams p;
  cudaError_t (*launch)(const QuantParams&, int ctas, int cluster, size_t smem, bool overlap, cudaStream_t);
  int ctas, cluster;
  size_t smem;
  bool overlap;
};
static_assert(sizeof(Ready) <= sizeof(QuantReady) && alignof(Ready) <= alignof(QuantReady) && std::is_trivially_copyable_v<Ready>, "");

bool PrepareQuantGemm(const QuantCall& c, const QuantPlan& asked, cudaStream_t stream, QuantReady* out) {
  QuantPlan plan = asked;
  const QuantSetup* setup = nullptr;
  cudaError_t err = SetUpQuant(&setup);
  if (err != cudaSuccess) throw std::runtime_error(std::string("QuantGemm: ") + cudaGetErrorString(err));
  const bool x_loads = !OnSixteen(c.x, c.ldx), w_loads = !OnSixteen(c.w, c.ldw), loads = x_loads || w_loads;
  if (plan.bm < 16 || plan.bm > 256 || plan.bm % 16 != 0 || plan.split < 1 || plan.split > kMaxSplit || plan.per_sm < 1 || plan.per_sm > 2 ||
      (plan.pair && (plan.split != 1 || plan.bm % 32 != 0 || plan.per_sm != 1 || loads)))
    throw std::runtime_error("QuantGemm: bad launch shape");
  if (loads) plan.per_sm = 1;  // the registers of its warps, and the second ring
  Ready& ready = *new (out) Ready();
  QuantParams& p = ready.p;
  p.x = c.x;
  p.w = c.w;
  p.ldx = c.ldx;
  p.ldw = c.ldw;
  p.order_k = c.order_k;
  const int64_t w_rows = c.order_k ? c.n : c.k, w_cols = c.order_k ? c.k : c.n;
  p.x_span = (c.m - 1) * c.ldx + c.k;
  p.w_span = (w_rows - 1) * c.ldw + w_cols;
  p.x_scale = c.x_scale;
  p.w_scale = c.w_scale;
  p.out = c.out;
  p.ldo = c.ldo;
  p.out_type = c.out_type;
  p.out_vec = reinterpret_cast<uintptr_t>(c.out) % 16 == 0 && c.ldo * (c.out_type == QFG_FLOAT ? 4 : 2) % 16 == 0;
  p.M = static_cast<int>(c.m);
  p.N = static_cast<int>(c.n);
  p.K = static_cast<int>(c.k);
  p.give_up = c.give_up;
  ready.overlap = MayOverlapPredecessor(stream);
  p.early_weight = c.early_weight && ready.overlap;  // all weights ahead of all rows of x cost 0.8 us where there is nothing to wait for
  p.x_loads = x_loads;
  p.w_loads = w_loads;
  p.bm = plan.bm;
  p.ksteps = static_cast<int>((c.k + kTileK - 1) / kTileK);
  const int m_tiles = static_cast<int>((c.m + p.bm - 1) / p.bm);
  const int width = plan.pair ? 2 * kTileN : kTileN;
  const int64_t tiles = (c.n + width - 1) / width * m_tiles;
  if (tiles > INT_MAX / 16) throw std::runtime_error("QuantGemm: too many tiles");
  p.tiles = static_cast<int>(tiles);
  p.grid = {m_tiles, p.tiles / m_tiles, std::min(m_tiles, kGroup), p.bm, width};
  const int cluster = plan.pair ? 2 : std::min(plan.split, p.ksteps);
  const int xrows = plan.pair ? p.bm / 2 : p.bm, stage = kWBytes + xrows * kTileK;
  if (!x_loads && !EncodeRows(&p.xmap, c.x, c.m, c.k, c.ldx, xrows)) return false;
  if (!w_loads && !EncodeRows(&p.wmap, c.w, w_rows, w_cols, c.ldw, 128)) return false;
  // half of the room, or less, for the rows as they are copied: they wait for memory, those behind them only for the MMA
  const int room = SmemLimit(plan.per_sm) - Fixed(plan), raw_stage = ((w_loads ? kTileK : 0) + (x_loads ? p.bm : 0)) * kRawPitch;
  p.raw_stages = loads ? std::max(1, std::min(kRawMost, room * 5 / 9 / raw_stage)) : 0;
  p.stages = std::min(kRing, (room - p.raw_stages * raw_stage) / stage);
  const bool split = cluster > 1 && !plan.pair;
  const int resident = plan.pair ? setup->sms / 2 : plan.per_sm * setup->sms;
  const int walkers = split ? p.tiles : std::min(p.tiles, resident);  // clusters that walk over the tiles
  p.sets = walkers < p.tiles ? 2 : 1;
  if (p.sets * p.bm * plan.per_sm > kMostColumns) p.sets = 1;
  p.raw_at = (Fixed(plan) - 1024 + p.stages * stage + 15) / 16 * 16;
  size_t smem = static_cast<size_t>(1024 + p.raw_at + p.raw_stages * raw_stage);
  if (split) smem = std::max(smem, static_cast<size_t>(1024 + p.bm * kTileN * 4));
  if (p.stages < 2 || smem > static_cast<size_t>(SmemLimit(1))) throw std::runtime_error("QuantGemm: bad launch shape");
  ready.ctas = walkers * cluster;
  ready.cluster = cluster;
  ready.smem = smem;
  auto pick = [&](auto fp8) {
    constexpr bool FP8 = decltype(fp8)::value;
    return plan.pair       ? LaunchAs<FP8, true, false, false>
           : split && loads ? LaunchAs<FP8, false, true, true>
           : split          ? LaunchAs<FP8, false, true, false>
           : loads          ? LaunchAs<FP8, false, false, true>
                            : LaunchAs<FP8, false, false, false>;
  };
  ready.launch = c.fp8 ? pick(std::true_type()) : pick(std::false_type());
  return true;
}

cudaError_t LaunchQuantGemm(const QuantReady& prepared, cudaStream_t stream) {
  const Ready& ready = reinterpret_cast<const Ready&>(prepared);
  const cudaError_t err = ready.launch(ready.p, ready.ctas, ready.cluster, ready.smem, ready.overlap, stream), last = cudaGetLastError();
  return err == cudaSuccess ? last : err;
}

}  // namespace qfg
