// kc_tcgen05.cuh -- the 5th-generation tensor core's plumbing shared by the
// batched GEMM (batched.cu) and the paged attention (paged_chunk.cu; the loads
// also paged_decode.cu): matrix instructions, shared-memory descriptors, 2D and
// 3D TMA loads and bounded mbarrier waits.
#pragma once

#include <cuda.h>

#include "kc_common.cuh"

namespace kc {

// Instruction descriptor, kind::f16: fp32 accumulator, f16 (0) or bf16 (1)
// operands, A K-major, B K-major or MN-major (bit 16), N >> 3 at bit 17,
// M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t umma_idesc(bool bf16, int m, int n, bool b_mn_major) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn_major ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// D (tensor memory) (+)= A (shared memory) B (shared memory)
__device__ __forceinline__ void umma_bf16(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(acc));
}
// A operand from tensor memory (one row per lane, two 16-bit values per 32-bit column)
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc,
                                             uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// True in one lane of a converged warp, the same one each time.  The compiler
// knows that a branch on it has one thread, so matrix instructions inside it are
// issued from uniform registers one after the other: 64 clocks for one of 128 x
// 128 x 16, as fast as they run.  Behind a test of the lane's number, or with it
// as their predicate, each takes 92, whatever its size.
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// try_wait: wakes when the phase completes, gives up after 2^17 tries (one that
// fails takes about 3000 clocks: 0.2 s in all) or as soon as another thread of the
// CTA has given up (abort flag), so a protocol error ends the kernel instead of
// hanging the GPU.  (No suspend-time hint: with one of 1 us a wait that is met at
// once takes 240 clocks, without it about 180, and one that gives up 0.5 s; batched
// decode of 16, 32 and 64 sequences 3.58, 3.41 and 4.04 ms a step, without it 3.54,
// 3.36 and 3.97.)
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                         bool honour_abort = true, uint32_t tries = 1u << 17) {
    for (uint32_t i = 0; i < tries; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if (honour_abort && *abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
}
// Shared-memory matrix descriptor, K-major with the 128-byte swizzle (the
// layout TMA writes with CU_TENSOR_MAP_SWIZZLE_128B): rows 128 B apart, 8-row
// groups 1024 B apart (SBO), LBO unused (1), version 1, layout type 2.  A K
// step of 16 16-bit values advances the start address by 32 B inside the swizzle atom.
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t saddr) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) |
           (2ull << 61);
}
// The same tile read MN-major (the 64 values of a 128-byte row lie along M or
// N, rows along K): 8-row groups 1024 B apart (SBO), the next 64 values of M or
// N `lbo` bytes further.  A K step of 16 rows advances the start by 2048 B.
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t saddr, uint32_t lbo) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lbo >> 4) << 16) | (64ull << 32) |
           (1ull << 46) | (2ull << 61);
}

}  // namespace kc
