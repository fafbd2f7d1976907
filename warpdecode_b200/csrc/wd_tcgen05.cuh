// Tensor memory and the fifth-generation tensor core (tcgen05), as the kernels that use them share it.
#pragma once

#include "wd_device.cuh"

namespace wd {

// ---- tensor memory and the tensor core -----------------------------------------------------------------------------------
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// a warp's 32 lanes x N columns, N a multiple of 4; the values are there after tc_wait_ld
__device__ __forceinline__ void tc_ld4(uint32_t a, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void tc_ld8(uint32_t a, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t a, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(a)
                 : "memory");
}
// The wait for a read into v, and nothing that uses v is moved in front of it (there is no form without v: the read's own output does not
// tie its uses to the wait).
template <int N>
__device__ __forceinline__ void tc_wait_ld(uint32_t (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i])::"memory");
}
template <int N>
__device__ __forceinline__ void tc_ld(uint32_t a, uint32_t (&v)[N]) {
    static_assert(N % 4 == 0 && N <= 32, "columns of one read");
#pragma unroll
    for (int i = 0; i + 16 <= N; i += 16) tc_ld16(a + i, v + i);
    if constexpr (N % 16 >= 8) tc_ld8(a + N / 16 * 16, v + N / 16 * 16);
    if constexpr (N % 8 == 4) tc_ld4(a + N - 4, v + N - 4);
}
__device__ __forceinline__ void tc_st4(uint32_t a, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t a, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
template <int N>
__device__ __forceinline__ void tc_st(uint32_t a, const uint32_t (&v)[N]) {
#pragma unroll
    for (int i = 0; i + 8 <= N; i += 8) tc_st8(a + i, v + i);
    if constexpr (N % 8 == 4) tc_st4(a + N - 4, v + N - 4);
}
// Descriptor of a K-major operand without swizzle: 16-byte rows of 8 x 16 B matrices, `k_step` bytes from one to the next in K and 128 in N.
__device__ __forceinline__ uint64_t tc_smem_desc(uint32_t addr, uint32_t k_step) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | static_cast<uint64_t>((k_step >> 4) & 0x3fffu) << 16 | static_cast<uint64_t>(128u >> 4) << 32 |
           1ull << 46;
}
// D[128][N] (s32, tensor memory) = A[128][32] (s8, tensor memory) * B[N][32] (s8, shared memory); by one thread
__device__ __forceinline__ void tc_mma_s8(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(0u)
                 : "memory");
}
// D[128][N] (f32, tensor memory) (+)= A[128][16] * B[N][16] of f16, A in shared memory or in tensor memory (two elements a column). By a whole warp with
// the same arguments in every lane, of which one issues it: so the descriptors stay in uniform registers. (From one lane's branch a product took 100 cycles
// to issue.)
__device__ __forceinline__ void tc_mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n .reg .pred p, e;\n .reg .b32 r;\n elect.sync r|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add)
                 : "memory");
}
__device__ __forceinline__ void tc_mma_f16_t(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n .reg .pred p, e;\n .reg .b32 r;\n elect.sync r|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add)
                 : "memory");
}
// as tc_commit, by a whole warp
__device__ __forceinline__ void tc_commit_warp(uint64_t *bar) {
    asm volatile("{\n .reg .pred e;\n .reg .b32 r;\n elect.sync r|e, 0xffffffff;\n"
                 " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t *bar) {      // the barrier takes an arrival when the MMAs issued so far are done
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Bounded wait of this kernel's pipeline: by a count of polls, inline; a poll suspends the thread for 1.3 us, so that the limit is 1.4 s, or 0.3 ms
// when another wait of the pass has run out. (These waits stand between the stages of the warps that compute: a limit by the timer takes 2 to 3 %
// of the kernel, a flag in shared memory or a fence behind the loop 5 to 15.)
__device__ __forceinline__ bool tc_wait(uint64_t *bar, uint32_t parity, unsigned *status) {
#pragma unroll 1
    for (unsigned i = 0; i < kSpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255u) == 255u && *reinterpret_cast<volatile unsigned *>(status) != 0u) break;
    }
    atomicOr(status, kErrCopyTimeout);
    return false;
}
// What is under way ends before the CTA's memory is given back, whether a wait has run out or not.
__device__ __forceinline__ void tc_drain(uint64_t *bar, uint32_t parity) {
#pragma unroll 1
    for (unsigned i = 0; i < kSpinLimit && !mbar_try_wait(bar, parity); ++i) {
    }
}

}  // namespace wd
