// tcgen05.mma: descriptors of operands in shared memory (128-byte swizzle), the instruction, its completion.
#pragma once

#include "common.cuh"

namespace reskv {

// Shared-memory matrix descriptor, 128-byte swizzle, address bits [4, 18), leading / stride byte offsets.
__device__ __forceinline__ uint64_t umma_desc(uint32_t saddr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lbo_bytes >> 4) << 16) |
           (static_cast<uint64_t>(sbo_bytes >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// FP16 x FP16 (bf16: BF16 x BF16) -> FP32, M = 128, N = n; a_mn / b_mn: the operand is MN-major (its tile read transposed).
__host__ __device__ constexpr uint32_t umma_idesc(int n, bool a_mn, bool b_mn = false, bool bf16 = false) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? (1u << 15) : 0u) | (b_mn ? (1u << 16) : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
}

__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Descriptors in halves, for the compiler to add to the low one only: the address (in units of 16 bytes) is in its low bits.
struct UmmaDesc {
    uint32_t low, high;
};
__device__ __forceinline__ UmmaDesc umma_desc_halves(uint32_t saddr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
    const uint64_t d = umma_desc(saddr, lbo_bytes, sbo_bytes);
    return {static_cast<uint32_t>(d), static_cast<uint32_t>(d >> 32)};
}
template <bool ACCUMULATE>
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t high, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_low), "r"(b_low), "r"(high), "r"(idesc), "n"(ACCUMULATE ? 1 : 0)
        : "memory");
}

// The same with A in tensor memory: row r in lane r, two 16-bit elements of a row in a column.
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t b_high, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_low), "r"(b_high), "r"(idesc), "r"(accumulate)
        : "memory");
}

// One arrival on `bar` once every MMA issued so far by the calling thread has completed.
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// True in one lane of the (converged) warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t chosen;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
    return chosen != 0;
}

}  // namespace reskv
