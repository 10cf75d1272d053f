// 5th-generation tensor core helpers (tcgen05, sm_100a) for CTA pairs: tensor
// memory, matrix descriptors, the pair's multiply, commits and TMA loads whose
// completion goes to the leader CTA's barrier.
#pragma once

#include <stdint.h>

namespace mms {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// 512 columns of tensor memory in both CTAs of the pair (one whole warp of
// each executes it); the address is written to shared memory.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(dst) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t addr) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(addr));
}

__device__ __forceinline__ void umma_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void umma_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }

// Shared-memory matrix descriptor of a 128-byte swizzled tile. Strides in
// bytes: `lead` between 64-element blocks of the row dimension (tiles whose
// rows are contiguous; unused where the summed dimension is), `stride`
// between groups of 8 lines of 128 bytes.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(lead >> 4) << 16 |
           (uint64_t)(stride >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// Instruction descriptor: fp16 x fp16 or bf16 x bf16 -> fp32, M = 256 over the
// pair, N = n; at / bt: the factor's rows (not the summed dimension) are contiguous.
__device__ __forceinline__ uint32_t umma_idesc(int n, bool fp16, bool at, bool bt) {
    return 1u << 4 | (fp16 ? 0u : 1u << 7 | 1u << 10) | (at ? 1u << 15 : 0u) | (bt ? 1u << 16 : 0u) |
           (uint32_t)(n >> 3) << 17 | (uint32_t)(256 >> 4) << 24;
}

// d (+)= a b over 16 summed elements, by one thread of the leader CTA.
__device__ __forceinline__ void umma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}

// Arrive on the barrier at this offset in both CTAs once every multiply issued
// so far by this thread is done.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
                 " [%0], %1;\n" ::"r"(bar), "h"((uint16_t)3) : "memory");
}

// Shared-memory address of this offset in the pair's leader (rank 0).
__device__ __forceinline__ uint32_t leader_addr(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}

// TMA tile load into this CTA's shared memory that completes on the leader's
// barrier (`bar`: a leader_addr).
__device__ __forceinline__ void tma3_pair(uint32_t dst, const CUtensorMap *m, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%2, %3, %4}], [%5];\n"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
                 : "memory");
}

// 32 columns of this warp's 32 lanes of tensor memory; complete after tmem_wait.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32"
                 " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
                 " %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                   "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
// The loads so far are complete. `v` goes through, so that nothing reads the
// registers of a load before this.
__device__ __forceinline__ void tmem_wait(float (&v)[32]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}

}  // namespace mms
