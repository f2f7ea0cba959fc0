// Barriers, bulk copies and cluster addressing of the products with packed weights.
#pragma once

#include <atomic>

#include "stored.cuh"

namespace hi2 {
namespace stored {

// Lets a kernel have as much shared memory as there is; asked of the driver once per device.
constexpr int MAX_SMEM = 227 * 1024;
template <auto KERNEL>
bool reserve_smem() {
  static std::atomic<bool> done[64];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  if (device < 64 && done[device].load(std::memory_order_relaxed)) return true;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM) != cudaSuccess) return false;
  if (device < 64) done[device].store(true, std::memory_order_relaxed);
  return true;
}

constexpr long long WAIT_CYCLES = 2000000000LL;  // about one second

__device__ __forceinline__ uint32_t s32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(unsigned long long* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(b)), "r"(n));
}
__device__ __forceinline__ void bar_expect(unsigned long long* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(s32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(unsigned long long* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(b)) : "memory");
}
// Sleeps up to 20 us for the phase.
__device__ __forceinline__ bool bar_try(unsigned long long* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(s32(b)), "r"(parity), "r"(20000u) : "memory");
  return ok != 0;
}
// False when the limit ran out or another role of this block gave up.
__device__ __forceinline__ bool bar_wait(unsigned long long* b, uint32_t parity, volatile uint32_t* abort, int32_t* status) {
  if (bar_try(b, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (bar_try(b, parity)) return true;
    if (*abort) return false;
    if (clock64() - t0 > WAIT_CYCLES) {
      *abort = 1;
      atomicExch(status, HI2_ERR_TIMEOUT);
      return false;
    }
  }
}
// Copies that a block which gave up has already issued still land in its shared memory: time for them.
__device__ __forceinline__ void let_copies_land() {
  const long long t0 = clock64();
  while (clock64() - t0 < 2000000LL) {
  }
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, unsigned long long* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(s32(dst)), "l"(src), "r"(bytes), "r"(s32(bar)) : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ uint32_t in_rank(uint32_t local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

}  // namespace stored
}  // namespace hi2
