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
// The same for 32 and for 64 columns, a piece of 16 of them after the other in v.  (Four pieces one by one take 450 ns a tile,
// which the next tile's products wait for where there is one buffer of sums.)
__device__ __forceinline__ void tmem_ld32x32(uint32_t addr, float *v) {
#pragma unroll
    for (uint32_t h = 0; h < 2; h++, v += 8)
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
              "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23])
            : "r"(addr + ((16 * h) << 16))
            : "memory");
}
__device__ __forceinline__ void tmem_ld32x64(uint32_t addr, float *v) {
#pragma unroll
    for (uint32_t h = 0; h < 2; h++, v += 8)
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
            "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
              "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
              "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
              "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55])
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
// 2^-126 (g under -87.3) it is 0, and so is the result.  The function multiplies g before u does: g u alone can pass f32's
// range where the result is small.  13 instructions, two of them on the unit that has 16 lanes an SM (with expf and a division
// 60: a tile's gates took three times as long as its products).
__device__ __forceinline__ float silu_times(float g, float u) {
    const float a = fminf(fabsf(g), 200.0f), t = a * -1.44269504f, rest = fmaf(a, -1.44269504f, -t);
    float e, q;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    e = fmaf(e, rest * 0.693147181f, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.0f + e));
    return (g < 0.0f ? e : 1.0f) * g * q * u;
}

// ---- what the kernels have in common ----

constexpr uint32_t MAX_E = MOE_SORT_MAX_EXPERTS;
constexpr uint32_t OUT_ROW = MX4_ROWS * 2 + 16;   // 16-bit results of a token in shared memory, and padding
constexpr uint32_t OUT_BYTES = 2 * 16 * OUT_ROW;  // two pieces of 16 tokens, or one of f32
static_assert(OUT_BYTES >= 16 * (MX4_ROWS * 4 + 16), "a piece of f32");

__device__ __forceinline__ bool try_wait_cluster(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// By a whole warp, which goes on together.  Bounded: a wait that does not end is recorded, and everybody goes home.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity) {
    for (int i = 0; i < 16; i++)
        if (__all_sync(0xffffffffu, try_wait_cluster(bar, parity))) return true;
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
        for (int i = 0; i < 64; i++)
            if (__all_sync(0xffffffffu, try_wait_cluster(bar, parity))) return true;
        if (__any_sync(0xffffffffu, globaltimer_ns() - t0 > WAIT_LIMIT_NS)) return false;
    }
}
// Of each expert: how many tiles end with it and its first sorted place (a lookup from global memory took
// every role 0.7 us a tile).
struct Experts {
    uint32_t upto[MAX_E], first[MAX_E], n_rows;
};
constexpr uint32_t EXPERTS_BYTES = 2 * 4 * MAX_E + 1024;

// A tile: up to NT rows of x, a tile of it, those of one expert, to rows of the output from row0 on.
struct Tile {
    uint32_t e, x_tile, rows;
    uint64_t row0;
};

// The experts' lookups for tiles of nt tokens, by one warp.  (Of a plan that was filled anew, by a replayed graph, for more
// tokens than the host counts and has room for, there are no tiles.  Bounds on every place cost experts of 464 tokens, 480 to
// 672, 2 %; this does not.)
__device__ __forceinline__ void find_experts(const Mx4GemmArgs &a, Experts &ex, uint32_t nt, uint32_t lane) {
    uint32_t before = 0;
    for (uint32_t base = 0; base < a.n_expert; base += 128) {  // four experts a lane
        uint32_t f[5], n[4], upto = 0;
#pragma unroll
        for (uint32_t k = 0; k < 5; k++) f[k] = (uint32_t)__ldg(a.first + min(base + 4 * lane + k, a.n_expert));
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) upto += n[k] = (f[k + 1] - f[k] + nt - 1) / nt;
        const uint32_t mine = upto;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += v;
        }
        uint32_t at = before + upto - mine;
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const uint32_t e = base + 4 * lane + k;
            at += n[k];
            if (e < a.n_expert) ex.upto[e] = at, ex.first[e] = f[k];
            if (e + 1 == a.n_expert) ex.n_rows = f[k + 1], ex.upto[e] = f[k + 1] > a.n_places ? 0 : at;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
}

// The tt-th tile of NT tokens (there has to be one), as x lies in memory; by a whole warp.
template <uint32_t NT>
__device__ __forceinline__ Tile tile_of(const Mx4GemmArgs &a, const Experts &ex, uint32_t tt) {
    Tile t;
    if (a.first) {
        // the first expert whose tiles reach past tt, 32 at a time
        uint32_t lo = 0;
        for (uint32_t base = 0; base < a.n_expert; base += 32) {
            const uint32_t i = base + (threadIdx.x & 31u), before = __ballot_sync(0xffffffffu, i < a.n_expert && ex.upto[i] <= tt);
            lo += __popc(before);
            if (before != 0xffffffffu) break;
        }
        const uint32_t r = (tt - (lo ? ex.upto[lo - 1] : 0)) * NT, f0 = ex.first[lo], n = (lo + 1 < a.n_expert ? ex.first[lo + 1] : ex.n_rows) - f0;
        t.e = lo;
        t.x_tile = tt;
        t.rows = min(n - r, NT);
        t.row0 = f0 + r;
    } else {
        t.e = 0;
        t.row0 = (uint64_t)tt * NT;
        t.x_tile = tt;
        t.rows = (uint32_t)(a.n_tok - t.row0 < NT ? a.n_tok - t.row0 : NT);
    }
    return t;
}

__device__ __forceinline__ uint32_t pack(__half, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack(__nv_bfloat16, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Where a thread's part of a tile's results goes, of a token 128 features from f0 on, from row `row` of the output on: 16
// bytes of every eighth token (of f32: fourth); where the rows do not allow such stores, whatever their size, the warp's
// lanes beside one another in every fourth token, words of 4 bytes or, for 16-bit rows that begin between words, values.
// (1586 rows of 8320 columns to 6971 in bf16: eight stores of a value a lane, lanes 16 bytes apart 81 us, so 49.)
// VEC: known to be so (1), not to be so (0), or found out (2).
template <typename T, int VEC>
struct Out {
    static constexpr uint32_t ROW = MX4_ROWS * sizeof(T) + 16, PER = MX4_ROWS * sizeof(T) / 16, ES = 16 / sizeof(T), STEP = 128 / PER;
    T *at;
    uint32_t left;  // features from there on
    static __device__ __forceinline__ bool vec(const Mx4GemmArgs &a) { return VEC == 2 ? a.vec : VEC == 1; }
    static __device__ __forceinline__ uint32_t token(const Mx4GemmArgs &a, uint32_t warp, uint32_t lane) { return vec(a) ? (32 * warp + lane) / PER : warp; }
    __device__ __forceinline__ Out(const Mx4GemmArgs &a, uint64_t row, uint32_t f0, uint32_t warp, uint32_t lane) {
        const uint32_t f = vec(a) ? (32 * warp + lane) % PER * ES : lane * (a.pairs ? 2 : 1);
        at = static_cast<T *>(a.out) + (row + token(a, warp, lane)) * a.ldo + f0 + f;
        left = f0 + f < a.feats ? a.feats - f0 - f : 0;
    }
};

// A piece of 16 tokens (n of them are there, the first of them the tile's `from`th) by 128 features, of which a warp has 32 in
// v as tmem_ld32x16 gives them, to the output by way of shared memory, where the four warps' features of a token come
// together.  16-bit results go there eight by eight, turned over on the way (stmatrix), to one of two places in turn, so that
// one barrier a piece will do.
template <typename T, int VEC>
__device__ __forceinline__ void put_piece(const Mx4GemmArgs &a, const Out<T, VEC> &o, uint8_t *buf, const float *v, uint32_t from, uint32_t n, uint32_t warp,
                                          uint32_t lane, uint32_t group) {
    using O = Out<T, VEC>;
    if constexpr (sizeof(T) == 2) {
        const uint32_t at = smem_u32(buf) + (lane & 7) * O::ROW + (32 * warp + 8 * (lane >> 3)) * 2;
#pragma unroll
        for (uint32_t b = 0; b < 2; b++) {
            const float *lo = v + 4 * b, *hi = v + 8 + 4 * b;
            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at + 8 * b * O::ROW), "r"(pack(T(), lo[0], lo[1])),
                         "r"(pack(T(), lo[2], lo[3])), "r"(pack(T(), hi[0], hi[1])), "r"(pack(T(), hi[2], hi[3]))
                         : "memory");
        }
    } else {
        asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");  // the piece before has been read
        float *at = reinterpret_cast<float *>(buf + 2 * (lane & 3) * O::ROW) + 32 * warp + (lane >> 2);
#pragma unroll
        for (uint32_t b = 0; b < 2; b++)
#pragma unroll
            for (uint32_t i = 0; i < 8; i++)  // (token 8 b + 2 (lane % 4) + i % 2, feature 8 (i / 2) + lane / 4 of the warp's)
                at[(8 * b + (i & 1)) * (O::ROW / 4) + 8 * (i >> 1)] = v[(i >> 2) * 8 + 4 * b + (i & 3)];
    }
    asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
    const uint32_t token = O::token(a, warp, lane);
    T *to = o.at + from * a.ldo;
    if (O::vec(a)) {
        const uint8_t *mine = buf + token * O::ROW + (32 * warp + lane) % O::PER * 16;
#pragma unroll
        for (uint32_t t = 0; t < 16; t += O::STEP, to += O::STEP * a.ldo) {
            if (token + t >= n) break;
            const uint4 w = *reinterpret_cast<const uint4 *>(mine + t * O::ROW);
            if (o.left >= O::ES) *reinterpret_cast<uint4 *>(to) = w;
            else {
                const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
                for (uint32_t j = 0; j < O::ES; j++)
                    if (j < o.left) to[j] = e[j];
            }
        }
    } else if (sizeof(T) == 2 && a.pairs) {
        const uint8_t *mine = buf + token * O::ROW + 4 * lane;
#pragma unroll
        for (uint32_t t = 0; t < 16; t += 4, to += 4 * a.ldo) {
            if (token + t >= n) break;
#pragma unroll
            for (uint32_t j = 0; j < 2; j++) {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(mine + t * O::ROW + 128 * j);
                if (o.left > 64 * j + 1) *reinterpret_cast<uint32_t *>(to + 64 * j) = w;
                else if (o.left > 64 * j) to[64 * j] = reinterpret_cast<const T *>(&w)[0];
            }
        }
    } else {
        const T *mine = reinterpret_cast<const T *>(buf + token * O::ROW) + lane;
#pragma unroll
        for (uint32_t t = 0; t < 16; t += 4, to += 4 * a.ldo) {
            if (token + t >= n) break;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (o.left > 32 * j) to[32 * j] = mine[t * (O::ROW / sizeof(T)) + 32 * j];
        }
    }
}

}  // namespace mx4
}  // namespace sg
