// sk_tcgen05.cuh -- 5th-generation tensor core instructions (sm_100a PTX):
// tensor memory, matrix descriptors, tcgen05.mma / commit / ld.
#pragma once

#include <stdint.h>

#include "sk_tma.cuh"

namespace sk {

// Shared-memory matrix descriptor of a 128-byte swizzled operand of 16-bit
// elements. K-major (the contraction dimension contiguous): rows of 64 elements
// (128 bytes), 8 rows to a 1024-byte atom, `sbo` bytes from atom to atom.
// MN-major: 64 consecutive elements of the M or N dimension to a 128-byte row,
// 8 contraction indexes to an atom, `sbo` bytes to the next 8, `lbo` bytes to
// the next 64 elements.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(lbo >> 4) << 16 |
           (uint64_t)(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// Instruction descriptor of kind::f16: fp32 accumulators, both operands bf16 or
// both fp16, M x N.
__host__ __device__ constexpr uint32_t mma_idesc(bool bf16, bool a_mn, bool b_mn, int M, int N) {
    return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (a_mn ? 1u : 0u) << 15 |
           (b_mn ? 1u : 0u) << 16 | (uint32_t)(N >> 3) << 17 | (uint32_t)(M >> 4) << 24;
}

// cta_group::2: the two CTAs of a cluster of two work on one tile. Allocation
// and release are joint (a warp of each CTA calls them); the CTA of even rank
// issues the MMAs, which read both CTAs' shared memory at the same offsets and
// write both CTAs' tensor memory (each holds its 128 of the 256 lanes).
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* out, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(out)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_free_pair(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr),
                 "r"(columns)
                 : "memory");
}

__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                             bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// tma_load_3d of a CTA of a pair into its own shared memory, completing on a
// barrier of either CTA of the pair (a shared::cluster address).
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, int x, int y,
                                                 int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// Arrive at `bar` of both CTAs once the MMAs this thread has issued are done.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster"
        ".b64 [%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(on));
    return on != 0;
}

__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 32 lanes (the warp's quarter) x 32 columns of fp32 from tensor memory: lane l
// gets row l, register c column c. Complete after tmem_ld_wait().
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
          "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
          "=r"(v[31])
        : "r"(addr));
}
// 16 lanes x 32 columns as four 16 x 8 fragments: of fragment i, thread t gets in
// v[4i], v[4i+1] row t / 4, columns 2 (t % 4) and the next, in v[4i+2], v[4i+3]
// the same columns of row t / 4 + 8.
__device__ __forceinline__ void tmem_ld16x32(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
          "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
// Four 8 x 8 matrices of 16-bit elements (fragments as above, two columns to a
// register) to shared memory, transposed: lane l gives the address of row l % 8
// -- the matrix's column -- of matrix l / 8, 16 bytes each.
__device__ __forceinline__ void st_matrix4_trans(uint32_t addr, uint32_t a, uint32_t b,
                                                 uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr),
                 "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

}  // namespace sk
