// Messages between the blocks of a thread-block cluster: a few floats stored into another
// block's shared memory (st.async), counted in bytes on a barrier there, and the bounded wait
// for them.  Unlike a cluster-wide barrier they order nothing else and stall no one but the
// receiver.
#pragma once

#include "tc_ptx.cuh"

namespace dp {
namespace ptx {

// The address of this block's shared-memory object p in block `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(const void *p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void cluster_send(uint32_t dst, uint32_t bar, float a, float b) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];\n" ::"r"(dst),
               "f"(a), "f"(b), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void cluster_send(uint32_t dst, uint32_t bar, float2 a, float2 b) {
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];\n" ::"r"(dst),
      "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "r"(bar)
      : "memory");
}
// Waits for the messages of a phase; false after kWaitNs (which cannot pass unless a block of
// the cluster died): the caller records it in the device error word and waits no more.
constexpr uint64_t kWaitNs = 2000000000ull;
__device__ __forceinline__ bool cluster_wait(uint64_t *bar, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if (globaltimer() - t0 > kWaitNs) return false;
  }
}

}  // namespace ptx
}  // namespace dp
