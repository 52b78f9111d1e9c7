// serve_tma.cuh — bounded waits on mbarriers and boxes of the 16-bit cache by TMA (sm_100a).
#pragma once

#include <cuda.h>
#include <cstdint>

namespace b200 {
namespace srv {

constexpr uint32_t WAIT_POLLS = 1u << 18;     // a poll that finds nothing takes 7800 clocks: a second

__device__ __forceinline__ void mbar_init(uint32_t bar, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(n) : "memory"); }
__device__ __forceinline__ void mbar_init_done() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory"); }
// the phase of this parity; where it does not come within `polls` the caller is dead and waits for nothing more
__device__ __forceinline__ void mbar_wait(uint32_t bar, uint32_t parity, uint32_t polls, bool & dead) {
    for (uint32_t spins = 0; !dead; spins++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) break;
        if (spins >= polls) dead = true;
    }
}
// 64 dims of the box's tokens of a KV head of a page, keys then values: the map is [pages][2][heads][page_tokens][head_dim]
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap * map, uint32_t bar, int dim, int token, int head, int page) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
                 :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(dim), "r"(token), "r"(head), "r"(0), "r"(page) : "memory");
}

}  // namespace srv
}  // namespace b200
