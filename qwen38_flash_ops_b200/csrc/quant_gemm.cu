// The product of eight-bit rows with an eight-bit weight: out[m, n] = sum_k x[m, k] w[k, n] * x_scale[m] * w_scale[n], INT8 summed
// in 32-bit integers (exact) or E4M3 in FP32, scaled in FP32 and rounded once.
//
// A CTA computes tiles of 128 columns of w by `bm` rows of x (a multiple of 16, at most 256) with tcgen05.mma: the weight is the
// 128-row operand, so that one decoded token costs 16 columns of the instruction and not 128 rows; the rows of x are the bm-column
// operand.  Both come by tensor copies into 128-byte-swizzled shared memory, 128 bytes of k per stage, as they lie in memory: the
// weight with its columns contiguous (order n) is read MN-major, with k contiguous (order k) K-major.  Roles by warp:
//   0-3   epilogue: sums -> scaled -> the output
//   4     tensor copies of every stage
//   5     tensor memory; one lane issues the MMAs
//   6-13  LOADERS only: operands whose rows do not lie on 16 bytes, which a tensor copy cannot address, come by these warps'
//         32-bit loads, shifted into place
// SPLIT: the CTAs of a cluster share K, and add their sums through distributed shared memory in rank order.  PAIR: two CTAs work
// on 256 columns with cta_group::2, each with its own 128 columns of w and half of the rows of x.
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
#include <stdexcept>
#include <string>
#include <type_traits>

#include "qfg_internal.h"
#include "stream_order.cuh"
#include "tc_ptx.cuh"
#include "tensor_map.h"

namespace qfg {
namespace {

namespace cg = cooperative_groups;

constexpr int kTileN = 128;               // columns of w per CTA
constexpr int kTileK = 128;               // k per stage: one swizzled row of a K-major operand
constexpr int kWBytes = kTileN * kTileK;  // of a stage
constexpr int kRing = 12;                 // stages at most
constexpr int kLoaderWarps = 8;
constexpr int kBatch = 4;                 // 16-byte pieces a loading thread has in hand
constexpr int kPitch = 80;                // bytes of a row of 32 columns in an epilogue warp's buffer: rows 16 bytes apart in the banks
constexpr int kOutBuffers = 4 * 32 * kPitch;
constexpr int kScaleBuffers = 4 * 256 * 4;  // each epilogue warp's copy of its rows' scales
constexpr int kMostColumns = 512;           // of tensor memory
constexpr int kMaxSplit = 8;                // CTAs that share K

struct QuantParams {
  CUtensorMap xmap, wmap;
  const uint8_t *x, *w;
  long long ldx, ldw, x_span, w_span;  // bytes from row to row; bytes from the first to the last
  const float *x_scale, *w_scale;
  void* out;
  long long ldo;
  int M, N, K, ksteps, bm, m_tiles, tiles, stages, sets;
  int order_k;           // the weight is stored [n][k]
  int x_loads, w_loads;  // LOADERS: which operands do not come by tensor copies
  int out_type;          // a qfg_dtype
  int out_vec;           // rows of the output lie on 16 bytes
  int give_up;           // testing: no stage comes
};

struct QuantCtl {
  unsigned long long full[kRing], empty[kRing], acc_full[2], acc_empty[2];
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
__device__ __forceinline__ uint32_t Pack(int type, float lo, float hi) {
  if (type == QFG_BFLOAT16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

struct At {
  int n0, m0;
};
// the tiles of one block of columns follow one another, so the SMs share its weights in L2
template <bool PAIR>
__device__ __forceinline__ At Locate(const QuantParams& p, int tile, int rank) {
  const int nt = tile / p.m_tiles;
  return {nt * (PAIR ? 2 * kTileN : kTileN) + (PAIR ? rank * kTileN : 0), (tile - nt * p.m_tiles) * p.bm};
}

// ------------------------------------------------------------------------------ loading warps
// The words that hold `valid` bytes from `pos` on, of a tensor of `span` bytes that begins anywhere.  A word that the tensor only
// begins or ends in is put together of the tensor's own bytes.
__device__ __forceinline__ void LoadWords(const uint8_t* base, long long pos, int valid, long long span, uint32_t (&w)[5]) {
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(base) + static_cast<uintptr_t>(pos)) & 3);
  const long long first = pos - shift;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const long long at = first + 4 * i;
    w[i] = 0;
    if (valid > 0 && 4 * i < shift + valid) {
      if (at >= 0 && at + 4 <= span) {
        w[i] = *reinterpret_cast<const uint32_t*>(base + at);
      } else {
        for (int b = 0; b < 4; ++b) {
          if (at + b >= 0 && at + b < span) w[i] |= static_cast<uint32_t>(base[at + b]) << (8 * b);
        }
      }
    }
  }
}

// Fills every stage's share of the operands that tensor copies cannot address.  A piece is 16 bytes of a row of either operand;
// a thread's next pieces are asked for before those in hand are stored.
__device__ __forceinline__ void LoaderRole(const QuantParams& p, QuantCtl& ctl, int thread, int kbeg, int kcount, int first_tile, int tile_step, uint32_t smem,
                                           uint32_t stage_bytes) {
  const uint32_t full0 = Smem(&ctl.full[0]), empty0 = Smem(&ctl.empty[0]);
  const uint8_t *const x = BehindWait(p.x), *const w = BehindWait(p.w);
  const int w_rows = p.w_loads ? kTileK : 0, pieces = (w_rows + (p.x_loads ? p.bm : 0)) * 8;
  const int batches = (pieces + kLoaderWarps * 32 * kBatch - 1) / (kLoaderWarps * 32 * kBatch);
  const int mine = ((p.tiles - first_tile + tile_step - 1) / tile_step) * kcount;  // stages in all
  if (p.give_up) return;
  uint32_t next[kBatch][5], words[kBatch][5];
  int next_valid[kBatch], valid[kBatch], next_shift[kBatch], shift[kBatch];
  auto load = [&](int stage_index, int batch) {
    const int turn = stage_index / kcount, k0 = (kbeg + stage_index - turn * kcount) * kTileK;
    const At t = Locate<false>(p, first_tile + turn * tile_step, 0);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int piece = (batch * kBatch + j) * (kLoaderWarps * 32) + thread, r = piece >> 3, c = (piece & 7) * 16;
      const bool of_w = r < w_rows;
      // rows and bytes of a row, of the operand as it is stored
      const int row = of_w ? (p.order_k ? t.n0 : k0) + r : t.m0 + r - w_rows, rows = of_w ? (p.order_k ? p.N : p.K) : p.M;
      const int col = (of_w && !p.order_k ? t.n0 : k0) + c, cols = of_w && !p.order_k ? p.N : p.K;
      const uint8_t* const base = of_w ? w : x;
      const long long pos = static_cast<long long>(row) * (of_w ? p.ldw : p.ldx) + col;
      next_valid[j] = piece < pieces && row < rows ? min(16, cols - col) : 0;
      next_shift[j] = static_cast<int>((reinterpret_cast<uintptr_t>(base) + static_cast<uintptr_t>(pos)) & 3) * 8;
      LoadWords(base, pos, next_valid[j], of_w ? p.w_span : p.x_span, next[j]);
    }
  };
  load(0, 0);
  int stage = 0;
  uint32_t parity = 1;
#pragma unroll 1
  for (int s = 0; s < mine; ++s) {
#pragma unroll 1
    for (int b = 0; b < batches; ++b) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        valid[j] = next_valid[j];
        shift[j] = next_shift[j];
#pragma unroll
        for (int i = 0; i < 5; ++i) words[j][i] = next[j][i];
      }
      if (b + 1 < batches) {
        load(s, b + 1);
      } else if (s + 1 < mine) {
        load(s + 1, 0);
      }
      if (b == 0 && s >= p.stages && !BarWait(empty0 + stage * 8, parity, ctl)) return;
      const uint32_t dst = smem + static_cast<uint32_t>(stage) * stage_bytes;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int piece = (b * kBatch + j) * (kLoaderWarps * 32) + thread, r = piece >> 3, c = piece & 7;
        if (piece >= pieces) continue;
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = __funnelshift_r(words[j][i], words[j][i + 1], shift[j]);
          const int left = valid[j] - 4 * i;
          if (left < 4) v[i] = left <= 0 ? 0u : v[i] & (0xFFFFFFFFu >> (32 - 8 * left));
        }
        const int row = r < w_rows ? r : r - w_rows;
        Sts128(dst + (r < w_rows ? 0u : static_cast<uint32_t>(kWBytes)) + static_cast<uint32_t>(row * 128 + ((c ^ (row & 7)) * 16)), v);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if ((thread & 31) == 0) BarArrive(full0 + stage * 8);
    if (++stage == p.stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
}

// ------------------------------------------------------------------------------ the kernel
template <bool LOADERS>
constexpr int QuantThreads() {
  return 32 * (6 + (LOADERS ? kLoaderWarps : 0));
}

// SPLIT: one tile per cluster.  PAIR and the others never together.
template <bool FP8, bool PAIR, bool SPLIT, bool LOADERS>
__global__ void __launch_bounds__(QuantThreads<LOADERS>(), 1) QuantGemmKernel(const __grid_constant__ QuantParams p) {
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
  const bool copies = !LOADERS || !p.x_loads || !p.w_loads;
  int acc_cols = 32;
  while (acc_cols < p.sets * p.bm) acc_cols *= 2;

  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      BarInit(full0 + i * 8, (copies ? 1 : 0) + (LOADERS ? kLoaderWarps : 0));
      BarInit(empty0 + i * 8, 1);
    }
    for (int i = 0; i < 2; ++i) {
      BarInit(accf0 + i * 8, 1);
      BarInit(acce0 + i * 8, 4 * (PAIR ? 2 : 1));
    }
    ctl.fault = static_cast<uint32_t>(p.give_up);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 && lane == 0) {
    if (!LOADERS || !p.x_loads) asm volatile("prefetch.tensormap [%0];" ::"l"(&p.xmap) : "memory");
    if (!LOADERS || !p.w_loads) asm volatile("prefetch.tensormap [%0];" ::"l"(&p.wmap) : "memory");
  }
  if (warp == 5) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Smem(&ctl.tmem)), "r"(acc_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Smem(&ctl.tmem)), "r"(acc_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  FenceBefore();
  GridDependencyWait();
  __syncthreads();
  if constexpr (PAIR) cg::this_cluster().sync();  // the leader's barriers exist before the peer arrives on them
  FenceAfter();
  const uint32_t tmem = ctl.tmem;

  if (warp < 4) {
    // ---- epilogue
    const float* const x_scale = BehindWait(p.x_scale);
    uint8_t* const bufs = smem_ptr + static_cast<size_t>(p.stages) * stage_bytes;
    const uint32_t buf = Smem(bufs) + static_cast<uint32_t>(warp * 32 * kPitch);
    float* const xs = reinterpret_cast<float*>(bufs + kOutBuffers) + warp * 256;
    int it = 0;
    bool good = true;  // false from the first wait that ran out: the tiles that are left become NaN
    for (int tile = first_tile; tile < p.tiles; tile += tile_step, ++it) {
      const int b = p.sets == 2 ? it & 1 : 0, turn = p.sets == 2 ? it >> 1 : it;
      const At t = Locate<PAIR>(p, tile, rank);
      const int n = t.n0 + 32 * warp;  // the warp's first column
      if constexpr (!SPLIT) {
        for (int i = lane; i < p.bm; i += 32) xs[i] = t.m0 + i < p.M ? x_scale[t.m0 + i] : 0.f;
        __syncwarp();
      }
      good = good && BarWait(accf0 + b * 8, static_cast<uint32_t>(turn & 1), ctl);
      __syncwarp();
      FenceAfter();
      const uint32_t src = tmem + (static_cast<uint32_t>(32 * warp) << 16) + static_cast<uint32_t>(b * p.bm);
      if (SPLIT || p.out_type == QFG_FLOAT) {
        // a lane is a column, a register a row
        const float ws = !SPLIT && p.w_scale != nullptr && n + lane < p.N ? p.w_scale[n + lane] : 1.f;
        // where the stages were: after a wait that ran out, copies may still be landing there
        for (int i = 0; SPLIT && i < 16 && !good; ++i) __nanosleep(1000000);
        for (int c = 0; c < p.bm; c += 16) {
          uint32_t v[16];
          asm volatile(
              "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
              : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
              : "r"(src + static_cast<uint32_t>(c)));
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          if constexpr (SPLIT) {
            uint32_t* const part = reinterpret_cast<uint32_t*>(smem_ptr) + c * kTileN + 32 * warp + lane;
#pragma unroll
            for (int i = 0; i < 16; ++i) part[i * kTileN] = v[i];
          } else if (n + lane < p.N) {
            float* const out = static_cast<float*>(p.out) + static_cast<long long>(t.m0 + c) * p.ldo + n + lane;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (t.m0 + c + i < p.M) out[i * p.ldo] = good ? Sum<FP8>(v[i]) * xs[c + i] * ws : __uint_as_float(0x7FFFFFFFu);
            }
          }
        }
      } else {
        // 8 x 8 fragments, columns of w down and rows of x across, transposed through shared memory for stores of 16 bytes
        const int g = lane >> 2, t2 = (lane & 3) * 2, row = lane >> 2, chunk = lane & 3;
        float ws[2][2];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int col = n + 8 * h + g;
          ws[h >> 1][h & 1] = p.w_scale != nullptr && col < p.N ? p.w_scale[col] : 1.f;
        }
        const int rows = min(p.bm, p.M - t.m0), cols = p.N - n;
        uint16_t* const out = static_cast<uint16_t*>(p.out) + static_cast<long long>(t.m0) * p.ldo + n;
        const uint32_t st = buf + static_cast<uint32_t>((((lane >> 4) & 1) * 8 + (lane & 7)) * kPitch + ((lane >> 3) & 1) * 16);
        const uint32_t ld = buf + static_cast<uint32_t>(row * kPitch + chunk * 16);
        for (int c = 0; c < p.bm; c += 32) {
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
                  w[i] = good ? Pack(p.out_type, lo, hi) : 0x7FFF7FFFu;
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
            const uint16_t* const from = reinterpret_cast<const uint16_t*>(bufs + warp * 32 * kPitch) + lane;
            const int last = min(32, rows - c);
            for (int r = 0; r < last; ++r) {
              if (lane < cols) out[static_cast<long long>(c + r) * p.ldo + lane] = from[r * (kPitch / 2)];
            }
          }
        }
      }
      FenceBefore();
      __syncwarp();
      if (lane == 0 && good) BarArriveLeader<PAIR>(acce0 + b * 8);
    }
  } else if (warp == 4) {
    // ---- tensor copies
    int stage = 0, round = 0;
    bool good = p.give_up == 0 && copies;
    const bool load_w = !LOADERS || !p.w_loads, load_x = !LOADERS || !p.x_loads;
    const uint32_t mine = static_cast<uint32_t>((load_w ? kWBytes : 0) + (load_x ? xrows * kTileK : 0));
    for (int tile = first_tile; tile < p.tiles && good; tile += tile_step) {
      const At t = Locate<PAIR>(p, tile, rank);
      for (int k = 0; k < kcount; ++k) {
        if (round > 0 && !BarWait(empty0 + stage * 8, static_cast<uint32_t>((round - 1) & 1), ctl)) {
          good = false;
          break;
        }
        const uint32_t bar = PAIR ? MapRank(full0 + stage * 8, 0) : full0 + stage * 8;
        const uint32_t dst = smem + static_cast<uint32_t>(stage) * stage_bytes;
        const int k0 = (kbeg + k) * kTileK;
        if (ElectOne()) {
          if (rank == 0 || !PAIR) BarExpect(full0 + stage * 8, PAIR ? 2 * mine : mine);
          if (load_w) TmaLoad<PAIR>(dst, &p.wmap, p.order_k ? k0 : t.n0, p.order_k ? t.n0 : k0, bar);
          if (load_x) TmaLoad<PAIR>(dst + kWBytes, &p.xmap, k0, t.m0 + (PAIR ? rank * xrows : 0), bar);
        }
        __syncwarp();
        if (++stage == p.stages) {
          stage = 0;
          ++round;
        }
      }
    }
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
    LoaderRole(p, ctl, tid - 6 * 32, kbeg, kcount, first_tile, tile_step, smem, stage_bytes);
  }

  if constexpr (SPLIT) {
    // the ranks' sums meet: rank r finishes rows [r bm / C, (r + 1) bm / C) of the tile, adding in rank order
    cg::cluster_group cluster = cg::this_cluster();
    FenceBefore();
    cluster.sync();
    const At t = Locate<false>(p, first_tile, 0);
    const uint32_t* const part = reinterpret_cast<const uint32_t*>(smem_ptr);
    const float* const x_scale = BehindWait(p.x_scale);
    const int r0 = rank * p.bm / csize, r1 = (rank + 1) * p.bm / csize;
    const int c = lane * 4, n = t.n0 + c, cols = p.N - n;
    const int rows = min(r1, p.M - t.m0), warps = static_cast<int>(blockDim.x) / 32;
    float ws[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ws[e] = p.w_scale != nullptr && e < cols ? p.w_scale[n + e] : 1.f;
    uint32_t bad = 0;  // a rank gave up
#pragma unroll
    for (int r = 0; r < kMaxSplit; ++r) {
      if (r < csize) bad |= *cluster.map_shared_rank(const_cast<const uint32_t*>(&ctl.fault), r);
    }
    // ROWS rows a warp at a time, so that the loads of all of them and of all ranks are on their way together
    auto add_up = [&](auto rows_tag, auto ranks_tag) {
      constexpr int ROWS = decltype(rows_tag)::value, RANKS = decltype(ranks_tag)::value;
      for (int m0 = r0 + warp; m0 < rows; m0 += warps * ROWS) {
        uint4 v[ROWS][RANKS];
        float xs[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int m = m0 + i * warps;
          xs[i] = m < rows ? x_scale[t.m0 + m] : 0.f;
#pragma unroll
          for (int r = 0; r < RANKS; ++r) {
            if (r < csize && m < rows) v[i][r] = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(part, r) + m * kTileN + c);
          }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int m = m0 + i * warps;
          if (m >= rows) break;
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
          const long long at = static_cast<long long>(t.m0 + m) * p.ldo + n;
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
            const uint2 o = make_uint2(Pack(p.out_type, y[0], y[1]), Pack(p.out_type, y[2], y[3]));
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
      add_up(std::integral_constant<int, 3>(), std::integral_constant<int, 4>());
    } else {
      add_up(std::integral_constant<int, 1>(), std::integral_constant<int, 8>());
    }
  }
  if (ctl.fault) __nanosleep(100000);  // copies of a CTA that gave up may still be landing
  FenceBefore();
  __syncthreads();
  if constexpr (PAIR || SPLIT) cg::this_cluster().sync();  // no CTA leaves while a peer still reads its shared memory
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
constexpr int kFixed = 1024 + kOutBuffers + kScaleBuffers;              // beside the stages

int SmemLimit(int per_sm) { return kSmemPerSm / per_sm - 1024 - kStatic; }

bool EncodeRows(CUtensorMap* map, const uint8_t* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)}, step[2] = {1, 1};
  const TensorMapEncodeFn fn = TensorMapEncoder();
  return fn != nullptr && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool FP8, bool PAIR, bool SPLIT, bool LOADERS>
cudaError_t LaunchAs(const QuantParams& p, int ctas, int cluster, size_t smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(QuantThreads<LOADERS>()));
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
  if (MayOverlapPredecessor(stream)) attr[cfg.numAttrs++] = OverlapAttribute();
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
  cfg.blockDim = dim3(static_cast<unsigned>(QuantThreads<false>()));
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

QuantPlan ChooseQuantPlan(const QuantCall& c) {
  const QuantSetup* setup = nullptr;
  if (SetUpQuant(&setup) != cudaSuccess) throw std::runtime_error("QuantGemm: the kernels could not be set up on this device");
  QuantPlan best;
  const bool loads = !OnSixteen(c.x, c.ldx) || !OnSixteen(c.w, c.ldw);
  const int64_t blocks = (c.k + kTileK - 1) / kTileK;
  const int64_t n_tiles = (c.n + kTileN - 1) / kTileN;
  if (!loads && c.m > 256) {
    best.pair = 1;
    best.bm = 256;
    best.per_sm = 1;
    return best;
  }
  const int64_t mt = (c.m + 255) / 256;
  best.bm = static_cast<int>(((c.m + mt - 1) / mt + 15) / 16 * 16);
  best.per_sm = loads || best.bm > 128 ? 1 : 2;
  const int64_t tiles = n_tiles * mt;
  for (int s = 2; s <= kMaxSplit && s <= blocks; ++s) {
    if (tiles <= setup->slots[best.per_sm][s]) best.split = s;
  }
  return best;
}

bool LaunchQuantGemm(const QuantCall& c, const QuantPlan& plan, cudaStream_t stream) {
  const QuantSetup* setup = nullptr;
  cudaError_t err = SetUpQuant(&setup);
  if (err != cudaSuccess) throw std::runtime_error(std::string("QuantGemm: ") + cudaGetErrorString(err));
  const bool x_loads = !OnSixteen(c.x, c.ldx), w_loads = !OnSixteen(c.w, c.ldw), loads = x_loads || w_loads;
  if (plan.bm < 16 || plan.bm > 256 || plan.bm % 16 != 0 || plan.split < 1 || plan.split > kMaxSplit || plan.per_sm < 1 || plan.per_sm > 2 ||
      (plan.pair && (plan.split != 1 || plan.bm % 32 != 0 || plan.per_sm != 1 || loads)))
    throw std::runtime_error("QuantGemm: bad launch shape");
  QuantParams p = {};
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
  p.x_loads = x_loads;
  p.w_loads = w_loads;
  p.bm = plan.bm;
  p.ksteps = static_cast<int>((c.k + kTileK - 1) / kTileK);
  p.m_tiles = static_cast<int>((c.m + p.bm - 1) / p.bm);
  const int width = plan.pair ? 2 * kTileN : kTileN;
  const int64_t tiles = (c.n + width - 1) / width * p.m_tiles;
  if (tiles > INT_MAX / 16) throw std::runtime_error("QuantGemm: too many tiles");
  p.tiles = static_cast<int>(tiles);
  const int cluster = plan.pair ? 2 : std::min(plan.split, p.ksteps);
  const int xrows = plan.pair ? p.bm / 2 : p.bm, stage = kWBytes + xrows * kTileK;
  if (!x_loads && !EncodeRows(&p.xmap, c.x, c.m, c.k, c.ldx, xrows)) return false;
  if (!w_loads && !EncodeRows(&p.wmap, c.w, w_rows, w_cols, c.ldw, 128)) return false;
  p.stages = std::min(kRing, (SmemLimit(plan.per_sm) - kFixed) / stage);
  const bool split = cluster > 1 && !plan.pair;
  const int resident = plan.pair ? setup->sms / 2 : plan.per_sm * setup->sms;
  const int walkers = split ? p.tiles : std::min(p.tiles, resident);  // clusters that walk over the tiles
  p.sets = walkers < p.tiles ? 2 : 1;
  if (p.sets * p.bm * plan.per_sm > kMostColumns) p.sets = 1;
  size_t smem = static_cast<size_t>(kFixed) + static_cast<size_t>(p.stages) * stage;
  if (split) smem = std::max(smem, static_cast<size_t>(1024 + p.bm * kTileN * 4));
  if (p.stages < 2 || smem > static_cast<size_t>(SmemLimit(1))) throw std::runtime_error("QuantGemm: bad launch shape");
  const int ctas = walkers * cluster;
  if (plan.pair) {
    err = c.fp8 ? LaunchAs<true, true, false, false>(p, ctas, 2, smem, stream) : LaunchAs<false, true, false, false>(p, ctas, 2, smem, stream);
  } else if (split && loads) {
    err = c.fp8 ? LaunchAs<true, false, true, true>(p, ctas, cluster, smem, stream) : LaunchAs<false, false, true, true>(p, ctas, cluster, smem, stream);
  } else if (split) {
    err = c.fp8 ? LaunchAs<true, false, true, false>(p, ctas, cluster, smem, stream) : LaunchAs<false, false, true, false>(p, ctas, cluster, smem, stream);
  } else if (loads) {
    err = c.fp8 ? LaunchAs<true, false, false, true>(p, ctas, 1, smem, stream) : LaunchAs<false, false, false, true>(p, ctas, 1, smem, stream);
  } else {
    err = c.fp8 ? LaunchAs<true, false, false, false>(p, ctas, 1, smem, stream) : LaunchAs<false, false, false, false>(p, ctas, 1, smem, stream);
  }
  if (err == cudaSuccess) err = cudaGetLastError();
  if (err != cudaSuccess) throw std::runtime_error(std::string("QuantGemm: ") + cudaGetErrorString(err));
  return true;
}

}  // namespace qfg
