// The instructions around tcgen05.mma that the kernels on tensor memory share: barriers in shared memory with bounded waits, tensor
// copies, the products with both operands in shared memory, and their descriptors.
#pragma once

#include <cuda.h>

#include <cstdint>

namespace qfg {
namespace {

constexpr int kSpin = 1 << 20;  // tries of a wait, after which a CTA gives up; a CTA's control block has a `fault` that says so

__device__ __forceinline__ uint32_t Smem(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void BarInit(uint32_t a, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(a), "r"(n) : "memory"); }
__device__ __forceinline__ void BarArrive(uint32_t a) {
  asm volatile("{ .reg .b64 st; mbarrier.arrive.shared::cta.b64 st, [%0]; }" ::"r"(a) : "memory");
}
__device__ __forceinline__ uint32_t MapRank(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ void BarExpect(uint32_t a, uint32_t bytes) {
  asm volatile("{ .reg .b64 st; mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1; }" ::"r"(a), "r"(bytes) : "memory");
}
// arrives on the barrier of this CTA, or of the leader of its pair
template <bool PAIR>
__device__ __forceinline__ void BarArriveLeader(uint32_t a) {
  if constexpr (PAIR) {
    asm volatile("{ .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, 0;\n mbarrier.arrive.shared::cluster.b64 _, [r];\n}" ::"r"(a) : "memory");
  } else {
    BarArrive(a);
  }
}
__device__ __forceinline__ bool BarTry(uint32_t a, uint32_t parity) {
  uint32_t ok;
  asm volatile("{ .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(a), "r"(parity) : "memory");
  return ok != 0;
}
// the same without the pause of up to a microsecond that try_wait may take where the phase is still open
__device__ __forceinline__ bool BarTest(uint32_t a, uint32_t parity) {
  uint32_t ok;
  asm volatile("{ .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(a), "r"(parity) : "memory");
  return ok != 0;
}
// false once a wait of this CTA ran out
template <typename C>
__device__ __forceinline__ bool BarWait(uint32_t a, uint32_t parity, C& c) {
  for (int i = 0; i < kSpin; ++i) {
    if (BarTry(a, parity)) return true;
    if ((i & 255) == 255 && c.fault) return false;
  }
  c.fault = 1;
  return false;
}
// the same where what is waited for was written by another CTA of the cluster
template <typename C>
__device__ __forceinline__ bool BarWaitCluster(uint32_t a, uint32_t parity, C& c) {
  for (int i = 0; i < kSpin; ++i) {
    uint32_t ok;
    asm volatile("{ .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(a), "r"(parity) : "memory");
    if (ok) return true;
    if ((i & 255) == 255 && c.fault) return false;
  }
  c.fault = 1;
  return false;
}
template <bool PAIR>
__device__ __forceinline__ void TmaLoad(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (PAIR) {  // the barrier may be the leader's
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y)
                 : "memory");
  } else {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map),
                 "r"(bar), "r"(x), "r"(y)
                 : "memory");
  }
}
// bytes that lie beside one another, from and to 16-byte boundaries, a multiple of 16 of them
__device__ __forceinline__ void BulkLoad(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// one lane of a converged warp; unlike a test of the lane number it leaves the compiler's view of the operands uniform,
// which the MMA's descriptors need (a lane test cost 80 cycles per MMA and 350 per wait)
__device__ __forceinline__ bool ElectOne() {
  uint32_t yes;
  asm volatile("{ .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes)::"memory");
  return yes != 0;
}
template <bool PAIR>
__device__ __forceinline__ void MmaSs(uint32_t d, unsigned long long a, unsigned long long b, uint32_t idesc, bool add) {
  if constexpr (PAIR) {
    asm volatile("{ .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(add ? 1 : 0)
                 : "memory");
  } else {
    asm volatile("{ .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(add ? 1 : 0)
                 : "memory");
  }
}
// arrives on the barrier (of both CTAs of a pair) when the MMAs issued so far have completed
template <bool PAIR>
__device__ __forceinline__ void MmaCommit(uint32_t bar) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
  } else {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  }
}
__device__ __forceinline__ void FenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void FenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 128-byte swizzle; `lbo`: distance of the 64-element groups of an MN-major operand (unused K-major), `sbo`: of the
// groups of eight rows
__device__ __forceinline__ unsigned long long SmemDesc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return static_cast<unsigned long long>((addr >> 4) & 0x3FFF) | (static_cast<unsigned long long>(lbo >> 4) << 16) |
         (static_cast<unsigned long long>(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void Lds128(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
}
__device__ __forceinline__ void Sts128(uint32_t a, const uint32_t* v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

}  // namespace
}  // namespace qfg
