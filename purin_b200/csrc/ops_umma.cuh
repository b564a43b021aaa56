// Warp-level building blocks of the tcgen05 matrix products: mbarriers with bounded waits,
// TMA loads, matrix descriptors, tensor memory.
//
// kGroup is the CTA pair's size (cta_group::1 or ::2).  With 2, the CTAs of a cluster of
// two share one product of 256 rows: each loads its 128 rows of A and its half of B, CTA 0
// issues the instructions for both, and each finds its 128 rows in its own tensor memory.
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace purin {
namespace ops {
namespace umma {

constexpr unsigned long long kWaitNs = 4000000000ull;  // a wait that lasts longer has failed

__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address of the same shared-memory place in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t in_cta(uint32_t address, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Arrives at a barrier of this or another CTA of the cluster (an address from in_cta).
__device__ __forceinline__ void barrier_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// False if the phase has not completed within kWaitNs.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
  if (barrier_try(bar, parity)) return true;
  const unsigned long long start = now_ns();
  while (!barrier_try(bar, parity))
    if (now_ns() - start > kWaitNs) return false;
  return true;
}

// Loads a box of a 3-dimensional tensor; x * element size is a multiple of 16 bytes.  With
// a CTA pair the bytes may be counted at the other CTA's barrier.
template <int kGroup>
__device__ __forceinline__ void tma_load(uint32_t to, const CUtensorMap* map, uint32_t bar, int x,
                                         int y, int z) {
  if constexpr (kGroup == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(to), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(to), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Operand tiles in shared memory have 64 elements of 2 bytes in a 128-byte row, with the
// 128-byte swizzle that TMA writes; groups of 8 rows are 1024 bytes apart.
//   K-major:  a row is one line of the operand, 64 values along K; a step of 16 along K is
//             32 bytes further into the rows.
//   MN-major: a row is one K index, 64 lines of the operand; 64 K rows make a block of
//             8192 bytes, the next 64 lines are the next block (the leading offset); a
//             step of 16 along K is 16 rows, 2048 bytes.
constexpr uint32_t kKStepMajor = 32, kMnStepMajor = 2048;

__device__ __forceinline__ uint64_t descriptor(uint32_t address, bool mn_major) {
  uint64_t d = (address & 0x3ffff) >> 4;
  d |= uint64_t(mn_major ? 8192 >> 4 : 1) << 16;  // leading offset (unused if K-major)
  d |= uint64_t(1024 >> 4) << 32;                 // stride between groups of 8 rows
  d |= uint64_t(1) << 46;                         // descriptor version of sm_100
  d |= uint64_t(2) << 61;                         // 128-byte swizzle
  return d;
}
// bf16 x bf16 -> f32, m x n.
__host__ __device__ constexpr uint32_t instruction(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

template <int kGroup>
__device__ __forceinline__ void mma(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if constexpr (kGroup == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
}
// Arrives at `bar` (in both CTAs of a pair) when this thread's products so far are done.
template <int kGroup>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (kGroup == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"(uint16_t(3)) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 ::"r"(bar) : "memory");
}
template <int kGroup>
__device__ __forceinline__ void tmem_alloc(uint32_t to, uint32_t columns) {
  if constexpr (kGroup == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <int kGroup>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
  if constexpr (kGroup == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes: value j is column j of the lane's row.  The load and the wait
// for it are one statement: between two the compiler could use the registers before they are filled.
__device__ __forceinline__ void tmem_load32(uint32_t from, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(from)
      : "memory");
}

// ---- 32-byte accesses and pairs of 32-bit operations ----------------------------------
// A lane's row is far from its neighbours': 32 bytes, a whole sector, per access.
__device__ __forceinline__ void store32(void* to, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "l"(to)
               : "memory");
}
__device__ __forceinline__ void load32(const void* from, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(from) : "memory");
}
struct Pair {
  unsigned long long bits;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(bits)); }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace umma
}  // namespace ops
}  // namespace purin
