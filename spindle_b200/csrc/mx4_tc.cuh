// mx4_tc.cuh — what the tensor-core kernels on microscaled 4-bit matrices have in common: operand,
// scale and instruction descriptors, tcgen05 in inline PTX (G: CTAs that work on a tile, 1 or 2).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx4.cuh"
#include "tiled_block.cuh"

namespace sg {
namespace mx4 {

// K-major operand, 128-byte swizzle: groups of 8 rows 1024 bytes apart, version 1 (bits 46-47), layout 2 (61-63).
__device__ __forceinline__ uint64_t desc_operand(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Scales, no swizzle: groups of 8 rows of 16 bytes, 128 bytes apart.
__device__ __forceinline__ uint64_t desc_scales(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128u >> 4) << 32) | (1ull << 46);
}
// kind::mxf4: E2M1 x E2M1 (bits 7-9, 10-12 = 1), N >> 3 at bit 17, scales UE8M0 (bit 23), M >> 4 at bit 24; the half of a
// scale word's four bytes at bits 29-30 (A) and 4-5 (B).
__device__ __forceinline__ uint32_t idesc(uint32_t m, uint32_t n, uint32_t half) {
    return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24) | ((2 * half) << 29) | ((2 * half) << 4);
}
template <int G>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sa, uint32_t sb, uint32_t add) {
    if constexpr (G == 1)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(id), "r"(sa), "r"(sb), "r"(add)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(id), "r"(sa), "r"(sb), "r"(add)
            : "memory");
}
// 32 rows of 16 bytes to four columns of all 128 lanes (of a pair: each CTA's own)
template <int G>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
    if constexpr (G == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// The barrier (of a pair: of both CTAs) is arrived at when everything issued before is done.
template <int G>
__device__ __forceinline__ void commit(uint64_t *bar) {
    if constexpr (G == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                     "h"((uint16_t)3)
                     : "memory");
}
template <int G>
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t cols) {  // a whole warp (of a pair: one of each CTA)
    if constexpr (G == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int G>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
    if constexpr (G == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 columns of this thread's lane, waited for in the same statement
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
// 32 lanes from the address's on, 16 columns: of each eight columns b and 16 lanes h a thread gets two of the lane (thread / 4)
// in v[8 h + 4 b] and the next, columns 8 b + 2 (thread % 4) on, and the same of the lane 8 further in v[8 h + 4 b + 2] and the
// next.  They are there after tmem_wait of the same registers (which are its operands, so that no use of them can move in
// between).
__device__ __forceinline__ void tmem_ld32x16(uint32_t addr, float *v) {
#pragma unroll
    for (uint32_t h = 0; h < 2; h++, v += 8)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                     : "r"(addr + ((16 * h) << 16))
                     : "memory");
}
__device__ __forceinline__ void tmem_wait(float *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                   "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :
                 : "memory");
}

// One lane of a converged warp.  (Copies, products and arrivals under this cost their warp half of what they cost under
// lane == 0: about 20 ns instead of 44 a bulk copy.)
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}

// silu(g) * u, by E = exp(-|g|), at most 1: the logistic function of g is 1 or E (of a negative g) over 1 + E.  The exponent
// |g| log2(e) is taken with its rest, so that E of a far g is off by little more than ex2's 2 units (|g| 1.3e-8 of it); below
// 2^-126 it is 0.  13 instructions, two of them on the unit that has 16 lanes an SM (with expf and a division 60: a tile's
// gates took three times as long as its products).
__device__ __forceinline__ float silu_times(float g, float u) {
    const float a = fminf(fabsf(g), 200.0f), t = a * -1.44269504f, rest = fmaf(a, -1.44269504f, -t);
    float e, q;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    e = fmaf(e, rest * 0.693147181f, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.0f + e));
    return (g < 0.0f ? e : 1.0f) * (q * (g * u));
}

}  // namespace mx4
}  // namespace sg
