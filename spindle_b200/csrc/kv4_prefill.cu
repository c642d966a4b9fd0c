// kv4_prefill.cu — attention over the paged 4-bit KV cache for many query rows
// per KV head (prompt chunks, large verify batches), f16 and bf16: what bounds it
// is the tensor cores, so the products run on tcgen05 with the sums in TMEM.
//
// A CTA has NQ tiles of 128 query rows (a row is a (token, head of the group)
// pair) of one request and KV head, and goes over the positions NK at a time:
//   - 128 threads per tile: a thread per row takes its scores from TMEM, keeps the
//     running maximum and sum, and puts its weights, in f16, where the scores were;
//   - ND threads turn the codes into f16 operands in shared memory (K, and V twice or with its rest);
//   - one thread issues the tensor products, a tile's sums and its next scores when
//     its weights are there: the tensor cores work for one tile while the weights
//     of the other are made.
// The scores are as good as f32: with K values m + s c (16-bit s and m, a code c)
// s c goes in as its f16 rounding and the exact rest (down to f16's last bit, 2^-25 of
// a K value), and the minima as 16 more columns against the sums of the query's
// groups (f16 rounding and rest).  Weights are rounded to f16 once, without the rest
// that the streaming kernel keeps for f16: TMEM has no room for it.  V values are rounded
// to f16 once for bf16; for f16 they go in as rounding and rest, since V's rounding,
// the weights' and the result's together were 1.5 to 1.6 times the result's alone
// (3.1e-4 to 3.3e-4 against 2.1e-4 of it, root mean square; without V's 2.4e-4 to 2.9e-4).
//
// Two chunks of 1024 and 768 tokens against up to 8100 positions, 32 query and 4 KV heads of 128, bf16: 370 us, 500
// TFLOP/s of the 186 GFLOP that attention has (30 % of the measured matrix rate; with the rests of K and the minima
// the products are 1.56 times that).  A step of 128 positions takes a tile 6100 cycles, of which its own thread-per-row
// work is 3600 and the products of both tiles 3700; the last wave of CTAs is part empty (224 CTAs on 148 SMs).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "kv4.cuh"

namespace sg {

namespace {

constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;
constexpr float P_SHIFT = 6.0f, LAG = 8.0f;  // weights are held as 2^6 p, p below 2^8: inside f16's range

template <typename T, int D>
struct Pre {
    static constexpr int G = D / 32;
    static constexpr bool VREST = std::is_same<T, __half>::value;  // V as f16 rounding and rest
    // Products of 128 rows by 128 positions run at twice the rate of those by 64 (73 cycles against 59); what a head of
    // 256 leaves of the shared memory and of TMEM is one tile of rows and 64 positions.
    static constexpr int NQ = D == 256 ? 1 : 2, NK = D == 256 ? 64 : 128;
    static constexpr int ND = 256;                                  // threads that make operands
    // V's rest takes the place of V's second buffer where there is no room for both (heads of 128, 8000 positions, a wave
    // of CTAs: 274 us against 228 without a rest; with both and 96 positions a step 301).
    static constexpr uint32_t VBUFS = D >= 128 && VREST ? 1 : 2;
    // With one buffer of V the first of a thread's groups is made while the buffer is still read: heads of 128 274 us
    // against 291; heads of 256 397 against 385, so there it is not.
    static constexpr bool EARLY = VBUFS == 1 && D == 128;
    static constexpr int THREADS = 128 * NQ + ND + 32;
    static constexpr int GV = NK * G / ND;                          // groups of V that one of them makes
    static constexpr int KI = NK * 4 * (G == 8 ? 2 : 1) / ND;       // items of K: a position's part of four groups (two)
    static constexpr uint32_t SBO_Q = (D / 8 + 2) * 128, SBO_K = D / 8 * 128, SBO_M = 256, SBO_V = NK * 16 + 16;
    static constexpr uint32_t Q_BYTES = 16 * SBO_Q;                 // 128 rows
    static constexpr uint32_t K_BYTES = NK / 8 * SBO_K, M_BYTES = NK / 8 * SBO_M, V_BYTES = D / 8 * SBO_V, VBUF_BYTES = V_BYTES * (VREST ? 2 : 1);
    static constexpr uint32_t K_AT = NQ * Q_BYTES, M_AT = K_AT + 2 * K_BYTES, V_AT = M_AT + M_BYTES, BAR_AT = V_AT + VBUFS * VBUF_BYTES;
    static constexpr uint32_t SMEM = BAR_AT + 256;
    // TMEM columns: scores, whose place the weights take (two f16 a column), and sums
    static constexpr uint32_t S_COL = 0, O_COL = 256;
    static_assert(GV >= 1 && KI >= 1 && SMEM <= 227 * 1024, "shapes");
};

__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr, uint32_t sbo) {
    // K-major, no swizzle: core matrices of 8 rows x 16 bytes, 128 bytes apart along K, sbo apart along the rows
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128u >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46);
}
constexpr uint32_t idesc(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((128u >> 4) << 24); }  // f16 x f16 -> f32, M = 128

// d (+)= a b: the first product of a sum and the others
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool add) {
    if (add) asm volatile("{\n .reg .pred p;\n setp.eq.b32 p, 0, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(id) : "memory");
    else asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, 0, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(id) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b),
                 "r"(id), "r"(add)
                 : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }

// 32 columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t hneg2(uint32_t a) {
    uint32_t d;
    asm("neg.f16x2 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The exponents of two weights in base 2, (s - m) scale + shift: the difference to the reference m first, which is exact
// near the maximum, so that no weight passes its bound however large the scores.
__device__ __forceinline__ float2 exponents(float s0, float s1, float2 minus_m, float2 scale, float shift) {
    float2 d;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 y, {%6, %7};\n"
        " mov.b64 z, {%8, %8};\n fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(s0), "f"(s1), "f"(minus_m.x), "f"(minus_m.y), "f"(scale.x), "f"(scale.y), "f"(shift));
    return d;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (std::is_same<T, __half>::value) return kv4_f16(v);
    else return __float2bfloat16_rn(v);
}

template <int N>
__device__ __forceinline__ void ldg_words(uint32_t (&w)[N], const uint8_t *p) {
    if constexpr (N == 1) w[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
    else if constexpr (N == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = v.x, w[1] = v.y;
    } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
}

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(Pre<T, D>::THREADS, 1) kv4_prefill_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using L = Kv4Tile<D>;
    using C = Pre<T, D>;
    constexpr int G = C::G, NQ = C::NQ, NK = C::NK, ND = C::ND, GV = C::GV, KI = C::KI;
    constexpr bool VREST = C::VREST;
    constexpr uint32_t VBUFS = C::VBUFS;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *q_s = smem;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::BAR_AT);
    // operands made and free again (V by buffer); scores and weights there and sums done, by tile of rows
    uint64_t *k_full = bars, *k_free = bars + 1, *v_full = bars + 2, *v_free = bars + 4;
    uint64_t *s_full = bars + 6, *p_full = bars + 8, *pv_done = bars + 10, *drain = bars + 12;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 13);
    volatile uint32_t *dead = tmem_slot + 1;
    uint32_t *there_s = tmem_slot + 2;  // [4][2] of steps: a byte per 16 positions, 1 where they are there
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t req = blockIdx.z, head = blockIdx.y;

    // tokens of no request: zeros, and no sum
    if ((a.first || a.last) && req == 0) {
        const uint32_t lead = a.first ? min((uint32_t)max(a.cu[0], 0), a.n_tok) : 0;
        const uint32_t spare = a.last ? min((uint32_t)max(a.cu[a.n_req], 0), a.n_tok) : a.n_tok, all = (lead + a.n_tok - spare) * a.n_heads;
        for (uint32_t r = (blockIdx.y * gridDim.x + blockIdx.x) * (C::THREADS / 32) + warp; r < all; r += gridDim.x * gridDim.y * (C::THREADS / 32)) {
            const uint32_t i = r / a.n_heads;
            const uint64_t t = i < lead ? i : spare + i - lead, h = r % a.n_heads;
            for (uint32_t d = lane; d < D; d += 32) ((T *)a.out)[t * a.o_tok + h * a.o_head + d] = from_f32<T>(0.0f);
            if (a.lse && lane == 0) a.lse[t * a.n_heads + h] = -INFINITY;
        }
    }

    // this CTA's rows; the requests' last tiles, which see most, come first
    const int32_t tok0 = max(a.cu[req], 0), nq = max(min(a.cu[req + 1], (int32_t)a.n_tok) - tok0, 0);
    const uint32_t rows = (uint32_t)nq * a.group, tile = gridDim.x - 1 - blockIdx.x, row0 = tile * (128 * NQ);
    // rows of tokens past max_new, which no CTA has: not a number, rather than what was there before
    if (blockIdx.x == 0)
        for (uint32_t r = gridDim.x * (128 * NQ) + warp; r < rows; r += C::THREADS / 32) {
            const uint64_t t = (uint64_t)tok0 + r / a.group, hq = head * a.group + r % a.group;
            for (uint32_t d = lane; d < D; d += 32) ((T *)a.out)[t * a.o_tok + hq * a.o_head + d] = from_f32<T>(NAN);
            if (a.lse && lane == 0) a.lse[t * a.n_heads + hq] = NAN;
        }
    if (row0 >= rows) return;
    const uint32_t halves = min((uint32_t)NQ, (rows - row0 + 127) / 128);
    const int32_t seq = max(a.seq[req], 0);
    const int32_t end = (int32_t)min((int64_t)seq, (int64_t)a.width << a.c.page_shift);
    const uint32_t last_row = min(rows, row0 + 128 * NQ) - 1;
    const int64_t first_place = (int64_t)seq - nq + row0 / a.group, last_place = (int64_t)seq - nq + last_row / a.group;
    const int32_t see_lo = a.window && first_place + 1 > (int64_t)a.window ? (int32_t)(first_place + 1 - a.window) : 0;
    const int32_t see_hi = (int32_t)max((int64_t)0, min(last_place + 1, (int64_t)end));
    const int32_t k0 = min(see_lo, see_hi) / NK, k1 = (see_hi + NK - 1) / NK;
    const uint32_t n = (uint32_t)max(k1 - k0, 0);  // steps

    if (tid == 0) {
        mbar_init(k_full, ND);
        mbar_init(k_free, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&v_full[i], ND);
            mbar_init(&v_free[i], 1);
            mbar_init(&s_full[i], 2);  // the products' end, and the issuing lane's own word on what it saw
            mbar_init(&p_full[i], 128);
            mbar_init(&pv_done[i], 1);
        }
        for (int i = 0; i < 8; i++) there_s[i] = 0x01010101u;
        mbar_init(drain, 1);
        fence_mbar_init();
        *dead = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    // ---- the query rows, a thread each: scaled by a power of two, in the order of the K operand, and their groups' sums ----
    float cs = 0.0f;
    if (tid < 128 * NQ) {
        const uint32_t r = row0 + tid, rr = min(r, rows - 1), tok = rr / a.group, hq = head * a.group + rr % a.group;
        const T *q = (const T *)a.q + (uint64_t)(tok0 + tok) * a.q_tok + hq * a.q_head;
        auto load8 = [&](uint32_t c, float (&x)[8]) {
            alignas(16) T v[8];
            if (a.vec_q) {
                *reinterpret_cast<uint4 *>(v) = __ldg(reinterpret_cast<const uint4 *>(q + c * 8));
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = q[c * 8 + i];
            }
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = to_f32(v[i]);
        };
        float amax = 0.0f, x[8];
        for (int c = 0; c < D / 8; c++) {
            load8(c, x);
#pragma unroll
            for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[i]));
        }
        // q * 2^(6 - e) is below 2^7; the K operand is half of s c
        const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 116);
        const float up = copysignf(__uint_as_float((uint32_t)(127 + 6 - e) << 23), a.scale);
        // (above 0, so that a position that is not seen stays at minus infinity)
        cs = fmaxf(fabsf(a.scale) * LOG2E * 2.0f * __uint_as_float((uint32_t)(127 - 6 + e) << 23), 0x1p-126f);
        uint8_t *dst = q_s + tid / 128 * C::Q_BYTES + tid % 128 / 8 * C::SBO_Q + tid % 8 * 16;
        float sum[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
            sum[g] = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                load8(g * 4 + c, x);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] *= up, sum[g] += x[i];
                *reinterpret_cast<uint4 *>(dst + (g * 4 + c) * 128) = make_uint4(pack2(x[0], x[4]), pack2(x[1], x[5]), pack2(x[2], x[6]), pack2(x[3], x[7]));
            }
            sum[g] *= 0.5f;
        }
        // 16 columns: the sums' f16 roundings, what those left, zeros
        __half col[16];
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const float s = sum[k % G], h = __half2float(__float2half_rn(s));
            col[k] = __float2half_rn(k < G ? s : k < 2 * G ? s - h : 0.0f);
        }
        *reinterpret_cast<uint4 *>(dst + D / 8 * 128) = *reinterpret_cast<const uint4 *>(col);
        *reinterpret_cast<uint4 *>(dst + (D / 8 + 1) * 128) = *reinterpret_cast<const uint4 *>(col + 8);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (*dead) return;
        if (!mbar_wait_bounded(bar, parity, WAIT_LIMIT_NS)) {
            *dead = 1;
            atomicExch(&g_dev_status, (unsigned)DEV_TIMEOUT_TMA);
        }
    };

    if (warp == (128 * NQ + ND) / 32) {
        // ---- the tensor products: the warp goes together, one lane issues ----
        const uint32_t base = smem_u32(smem), tm = __shfl_sync(~0u, tmem, 0);
        const uint64_t q_desc = smem_desc(base, C::SBO_Q), k_desc = smem_desc(base + C::K_AT, C::SBO_K),
                       m_desc = smem_desc(base + C::M_AT, C::SBO_M), v_desc = smem_desc(base + C::V_AT, C::SBO_V);
        // step i: for each tile of rows the sums of step i - 1, then the scores of step i in the weights' place
#pragma unroll 1
        for (uint32_t i = 0; i <= n && n; i++) {
            const uint32_t b = (i - 1) % VBUFS;
            if (i) wait(&v_full[b], (i - 1) / VBUFS & 1);
#pragma unroll 1
            for (uint32_t h = 0; h < halves; h++) {
                if (i) {
                    wait(&p_full[h], (i - 1) & 1);
                    __syncwarp();
                    fence_after();
                    if (elect_one() && !*dead) {
                        const uint32_t d = tm + C::O_COL + h * D, p = tm + C::S_COL + h * NK;
                        const uint64_t vd = v_desc + b * (C::VBUF_BYTES >> 4);
#pragma unroll
                        for (uint32_t c = 0; c < NK / 16; c++) mma_ts(d, p + c * 8, vd + c * 16, idesc(D), c ? 1u : i - 1);
                        if constexpr (VREST) {
#pragma unroll
                            for (uint32_t c = 0; c < NK / 16; c++) mma_ts(d, p + c * 8, vd + (C::V_BYTES >> 4) + c * 16, idesc(D), 1u);
                        }
                        if (h + 1 == halves) commit(&v_free[b]);
                        commit(&pv_done[h]);
                    }
                    __syncwarp();
                }
                if (i < n) {
                    if (i) wait(&pv_done[h], (i - 1) & 1);  // the weights are read
                    if (h == 0) wait(k_full, i & 1);
                    __syncwarp();
                    fence_after();
                    if (elect_one() && !*dead) {
                        const uint32_t d = tm + C::S_COL + h * NK;
                        const uint64_t qd = q_desc + h * (C::Q_BYTES >> 4);
#pragma unroll
                        for (uint32_t c = 0; c < D / 8; c += 2) {
                            mma_ss(d, qd + c * 8, k_desc + c * 8, idesc(NK), c != 0);
                            mma_ss(d, qd + c * 8, k_desc + (C::K_BYTES >> 4) + c * 8, idesc(NK), true);
                        }
                        mma_ss(d, qd + D, m_desc, idesc(NK), true);
                        commit(&s_full[h]);
                        arrive(&s_full[h]);
                        if (h + 1 == halves) commit(k_free);
                    }
                    __syncwarp();
                }
            }
        }
        if (*dead && lane == 0) {  // what is still running must end before its memory goes
            commit(drain);
            mbar_wait_bounded(drain, 0, WAIT_LIMIT_NS / 10);
        }
        __syncwarp();
    } else if (tid >= 128 * NQ) {
        // ---- the operands of a step from the cache: its codes are read a step ahead, its table entries two ----
        const Kv4Codes codes;
        const uint32_t dt = tid - 128 * NQ, dw = dt >> 5, x8 = lane & 7, y4 = lane >> 3;
        // K: item j of this thread is word part y4 of the groups from 4 ka(j) on, at position kpos(j); V: the eight
        // positions tb, word part x8, groups from gq * GV on
        auto kpos = [&](int j) { return (uint32_t)(j * (ND / 32) + dw) % (NK / 8) * 8 + x8; };
        auto ka = [&](int j) { return (uint32_t)(j * (ND / 32) + dw) / (NK / 8); };
        const uint32_t vi = dw * 4 + y4, tb = vi % (NK / 8), gq = vi / (NK / 8);
        const int32_t *table = a.tables + (uint64_t)req * a.ld_tables;
        const uint32_t shift = a.c.page_shift;
        auto entry = [&](int32_t pos) { return pos < end ? __ldg(table + (pos >> shift)) : -1; };
        auto tile_of = [&](int32_t blk, int32_t pos) {
            return a.c.data + (uint32_t)blk * a.block_bytes + ((((uint64_t)head << (shift - 4)) + ((pos & ((1 << shift) - 1)) >> 4)) * L::BYTES);
        };
        constexpr int KG = G < 4 ? G : 4;  // groups of a K item
        int32_t kb[KI], vb;
        uint32_t kr[KI][KG], ks[KI][KG], km[KI][KG / 2], vr[4][GV], vs[4][GV], vm[4][GV];
        bool k_ok[KI], v_ok;
        auto entries_k = [&](uint32_t i) {
#pragma unroll
            for (int j = 0; j < KI; j++) kb[j] = entry((k0 + (int32_t)i) * NK + kpos(j));
        };
        auto entries_v = [&](uint32_t i) { vb = entry((k0 + (int32_t)i) * NK + tb * 8); };
        auto load_k = [&](uint32_t i) {
            const int32_t t = (k0 + (int32_t)i) * NK;
#pragma unroll
            for (int j = 0; j < KI; j++) {
                const int32_t pos = t + kpos(j);
                const uint32_t p = pos & 15;
                k_ok[j] = pos < end && (uint32_t)kb[j] < a.c.n_blocks;
                if (k_ok[j]) {
                    const uint8_t *tl = tile_of(kb[j], pos);
                    ldg_words<KG>(kr[j], tl + p * L::KROW + (G < 4 ? y4 * G : (ka(j) * 4 + y4) * 4) * 4);
                    ldg_words<KG>(ks[j], tl + L::KS + (p >> 1) * (G * 4) + ka(j) * 16);
                    ldg_words<KG / 2>(km[j], tl + L::KM + p * (G * 2) + ka(j) * 8);
                }
            }
        };
        auto load_v = [&](uint32_t i) {
            const int32_t pos = (k0 + (int32_t)i) * NK + tb * 8;
            v_ok = pos < end && (uint32_t)vb < a.c.n_blocks;
            if (v_ok) {
                const uint8_t *tl = tile_of(vb, pos);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t pair = ((pos & 15) >> 1) + q, g0 = gq * GV;
                    ldg_words<GV>(vr[q], tl + L::VC + pair * L::VROW + kv4_word(x8, g0, 8, G) * 4);
                    ldg_words<GV>(vs[q], tl + L::VS + (pair * G + g0) * 4);
                    ldg_words<GV>(vm[q], tl + L::VM + (pair * G + g0) * 4);
                }
            }
        };
        if (n) {
            entries_k(0), entries_v(0);
            load_k(0), load_v(0);
            if (n > 1) entries_k(1), entries_v(1);
        }
        for (uint32_t i = 0; i < n; i++) {
            const uint32_t b = i % VBUFS;
            wait(k_free, (i & 1) ^ 1);
            uint8_t *k_hi = smem + C::K_AT, *k_lo = k_hi + C::K_BYTES, *k_m = smem + C::M_AT, *v_t = smem + C::V_AT + b * C::VBUF_BYTES;
            const int32_t t = (k0 + (int32_t)i) * NK;
#pragma unroll
            for (int j = 0; j < KI; j++) {
                const uint32_t pos = kpos(j);
                uint8_t *hi = k_hi + (pos >> 3) * C::SBO_K + (pos & 7) * 16, *lo = k_lo + (pos >> 3) * C::SBO_K + (pos & 7) * 16;
#pragma unroll
                for (int g = 0; g < KG; g++) {
                    uint32_t c[4], h[4], l[4];
                    // the position's scale twice, halved
                    uint32_t s = k_ok[j] ? __byte_perm(ks[j][g], 0, pos & 1 ? 0x3232 : 0x1010) : 0u;
                    s = hmul2(s, 0x38003800u);
                    codes.get<0>(k_ok[j] ? kr[j][g] : 0u, c);
#pragma unroll
                    for (int k = 0; k < 4; k++) h[k] = hmul2(c[k], s), l[k] = hfma2(c[k], s, hneg2(h[k]));
                    const uint32_t chunk = ((G < 4 ? g : ka(j) * 4 + g) * 4 + y4) * 128;
                    *reinterpret_cast<uint4 *>(hi + chunk) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(lo + chunk) = make_uint4(l[0], l[1], l[2], l[3]);
                }
                if (y4 == 0) {
                    // the minima: groups 0..G-1 and again, against the sums' roundings and rests
                    uint8_t *m = k_m + (pos >> 3) * C::SBO_M + (pos & 7) * 16;
                    uint32_t w[KG / 2];
#pragma unroll
                    for (int g = 0; g < KG / 2; g++) w[g] = k_ok[j] ? km[j][g] : 0u;
                    if constexpr (G == 2) {
                        *reinterpret_cast<uint4 *>(m) = make_uint4(w[0], w[0], 0u, 0u);
                        *reinterpret_cast<uint4 *>(m + 128) = make_uint4(0u, 0u, 0u, 0u);
                    } else if constexpr (G == 4) {
                        *reinterpret_cast<uint4 *>(m) = make_uint4(w[0], w[1], w[0], w[1]);
                        *reinterpret_cast<uint4 *>(m + 128) = make_uint4(0u, 0u, 0u, 0u);
                    } else {
                        *reinterpret_cast<uint2 *>(m + ka(j) * 8) = make_uint2(w[0], w[1]);
                        *reinterpret_cast<uint2 *>(m + 128 + ka(j) * 8) = make_uint2(w[0], w[1]);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            if (y4 == 0) {
#pragma unroll
                for (int j = 0; j < KI; j++)
                    if ((kpos(j) & 15) == 0 && ka(j) == 0) reinterpret_cast<uint8_t *>(there_s + (i & 3) * 2)[kpos(j) / 16] = k_ok[j];
            }
            arrive(k_full);
            if (i + 1 < n) {
                load_k(i + 1);
                if (i + 2 < n) entries_k(i + 2);
            }
            if (!C::EARLY) wait(&v_free[b], (i / VBUFS & 1) ^ 1);
#pragma unroll
            for (int g = 0; g < GV; g++) {
                uint32_t val[4][4], low[VREST ? 4 : 1][4];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int32_t p = t + (int32_t)tb * 8 + 2 * q;
                    const uint32_t mask = !v_ok || p >= end ? 0u : p + 1 >= end ? 0xFFFFu : 0xFFFFFFFFu;
                    const uint32_t s = vs[q][g] & mask, m = vm[q][g] & mask;
                    uint32_t c[4];
                    codes.get<0>(vr[q][g], c);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if constexpr (VREST) {
                            const float2 cf = unpack2(c[k]), sf = unpack2(s), mf = unpack2(m);
                            const float v0 = fmaf(cf.x, sf.x, mf.x), v1 = fmaf(cf.y, sf.y, mf.y);
                            val[k][q] = pack2(v0, v1);
                            const float2 h = unpack2(val[k][q]);
                            low[k][q] = pack2(v0 - h.x, v1 - h.y);
                        } else {
                            val[k][q] = hfma2(c[k], s, m);
                        }
                    }
                }
                if (C::EARLY && g == 0) wait(&v_free[b], (i / VBUFS & 1) ^ 1);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t d = 32 * (gq * GV + g) + 4 * x8 + k;
                    uint4 *at = reinterpret_cast<uint4 *>(v_t + (d >> 3) * C::SBO_V + tb * 128 + (d & 7) * 16);
                    *at = make_uint4(val[k][0], val[k][1], val[k][2], val[k][3]);
                    if constexpr (VREST) at[C::V_BYTES / 16] = make_uint4(low[k][0], low[k][1], low[k][2], low[k][3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(&v_full[b]);
            if (i + 1 < n) {
                load_v(i + 1);
                if (i + 2 < n) entries_v(i + 2);
            }
        }
    } else if (tid < 128 * halves) {
        // ---- the weights: a thread per row ----
        const uint32_t h = tid >> 7, row = row0 + tid, rr = min(row, rows - 1);
        const bool live = row < rows;
        const uint32_t mine = tmem + ((warp & 3) << 21);  // this warp's 32 lanes
        const int64_t place = (int64_t)seq - nq + rr / a.group;
        const int32_t hi_t = live ? (int32_t)max((int64_t)0, min(place + 1, (int64_t)end)) : 0;
        const int32_t lo_t = a.window && place + 1 > (int64_t)a.window ? (int32_t)(place + 1 - a.window) : 0;
        const uint32_t s_at = mine + C::S_COL + h * NK, o_at = mine + C::O_COL + h * D;
        float m = -INFINITY, l = 0.0f;
        for (uint32_t i = 0; i < n; i++) {
            const int32_t t0 = (k0 + (int32_t)i) * NK;
            wait(&s_full[h], i & 1);  // and the sums of the step before are done
            __syncwarp();
            fence_after();
            const uint2 there = *reinterpret_cast<const uint2 *>(there_s + (i & 3) * 2);
            const bool whole = t0 >= lo_t && t0 + NK <= hi_t && (there.x & there.y) == 0x01010101u;
            auto masked = [&](uint32_t (&s)[32], int c) {
                if (whole) return;
#pragma unroll
                for (int k = 0; k < 32; k++) {
                    const int32_t t = c + k;
                    if (t0 + t < lo_t || t0 + t >= hi_t || !((t < 64 ? there.x : there.y) >> (t / 16 % 4 * 8) & 1)) s[k] = 0xFF800000u;
                }
            };
            // 32 scores at a time, twice: for the maximum, and for the weights
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < NK; c += 32) {
                uint32_t s[32];
                __syncwarp();
                tmem_ld32(s_at + c, s);
                masked(s, c);
                float t1 = __uint_as_float(s[0]), t2 = __uint_as_float(s[1]);
#pragma unroll
                for (int k = 2; k < 32; k += 2) t1 = fmaxf(t1, __uint_as_float(s[k])), t2 = fmaxf(t2, __uint_as_float(s[k + 1]));
                top = fmaxf(top, fmaxf(t1, t2));
            }
            // the reference of the weights follows the maximum when that is 2^LAG above it
            const bool up = (top - m) * cs > LAG;
            if (__any_sync(~0u, up)) {
                const float f = up ? ex2((m - top) * cs) : 1.0f;
                if (up) m = top, l *= f;
                if (i) {
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        __syncwarp();
                        tmem_ld32(o_at + c, o);
#pragma unroll
                        for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                        tmem_st16(o_at + c, o);
                        tmem_st16(o_at + c + 16, o + 16);
                    }
                }
            }
            const float nm = m == -INFINITY ? 0.0f : -m;
            float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
            for (int c = 0; c < NK; c += 32) {
                uint32_t s[32], p[16];
                __syncwarp();
                tmem_ld32(s_at + c, s);
                masked(s, c);
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float2 t = exponents(__uint_as_float(s[k]), __uint_as_float(s[k + 1]), make_float2(nm, nm), make_float2(cs, cs), P_SHIFT);
                    const float p0 = ex2(t.x), p1 = ex2(t.y);
                    l0 += p0, l1 += p1;
                    p[k / 2] = pack2(p0, p1);
                }
                __syncwarp();
                tmem_st16(s_at + c / 2, p);  // over scores that are taken
            }
            l += l0 + l1;
            tmem_st_wait();
            fence_before();
            arrive(&p_full[h]);
        }
        // ---- the results ----
        if (n) {
            wait(&pv_done[h], (n - 1) & 1);
            __syncwarp();
            fence_after();
        }
        const uint32_t tok = rr / a.group, hq = head * a.group + rr % a.group;
        const uint64_t t = (uint64_t)tok0 + tok;
        T *out = (T *)a.out + t * a.o_tok + hq * a.o_head;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            __syncwarp();
            if (n) tmem_ld32(mine + C::O_COL + h * D + c, o);
            if (live) {
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    alignas(16) T y[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) y[j] = from_f32<T>(l == 0.0f ? 0.0f : __uint_as_float(o[k + j]) * inv);
                    if (a.vec_out) {
                        *reinterpret_cast<uint4 *>(out + c + k) = *reinterpret_cast<const uint4 *>(y);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++) out[c + k + j] = y[j];
                    }
                }
            }
        }
        if (live && a.lse) a.lse[t * a.n_heads + hq] = l == 0.0f ? -INFINITY : (m * cs - P_SHIFT + log2f(l)) * LN2;
    }
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

namespace {

template <typename T, int D>
cudaError_t launch(const Kv4AttnArgs &a, cudaStream_t s) {
    using C = Pre<T, D>;
    auto fn = kv4_prefill_kernel<T, D>;
    static bool ready[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!ready[dev & 63]) {
        if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess) return e;
        ready[dev & 63] = true;
    }
    const uint32_t tiles = (uint32_t)(((uint64_t)a.max_new * a.group + 128 * C::NQ - 1) / (128 * C::NQ));
    for (uint32_t r0 = 0; r0 < a.n_req; r0 += 32768) {
        Kv4AttnArgs b = a;
        b.n_req = a.n_req - r0 < 32768 ? a.n_req - r0 : 32768;
        b.first = r0 == 0, b.last = r0 + b.n_req == a.n_req;
        b.cu += r0, b.seq += r0, b.tables += (uint64_t)r0 * a.ld_tables;
        fn<<<dim3(tiles, a.c.heads, b.n_req), C::THREADS, C::SMEM, s>>>(b);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t kv4_prefill_launch(const Kv4AttnArgs &a, int32_t type, uint32_t d, cudaStream_t s) {
    if (type == SG_F16) return d == 64 ? launch<__half, 64>(a, s) : d == 128 ? launch<__half, 128>(a, s) : launch<__half, 256>(a, s);
    return d == 64 ? launch<__nv_bfloat16, 64>(a, s) : d == 128 ? launch<__nv_bfloat16, 128>(a, s) : launch<__nv_bfloat16, 256>(a, s);
}

bool kv4_prefill_pays(const Kv4AttnArgs &a, int32_t type, uint32_t d, int sms) {
    if (type == SG_F32 || a.n_req == 0) return false;
    // Rows (of all heads and requests) a wave of its CTAs from which this kernel is the faster one.  One request of 2000
    // positions, 4 KV heads, groups of 8, streaming kernel / this one in us, bf16 (f16): heads of 128 at 5632 rows 63 / 73
    // (66 / 85), at 6656 72 / 74 (77 / 86), at 8192 85 / 74 (91 / 86); of 8000 positions 190 / 228 (205 / 276), 221 / 228
    // (238 / 277), 270 / 226 (291 / 275).  Heads of 64: 6656 rows 48 / 58 (49 / 60), 8192 57 / 58 (58 / 62), 13312 84 / 58
    // (88 / 62).  Heads of 256, whose tiles are half as tall: 4096 rows 91 / 101 (93 / 111), 5632 119 / 100 (121 / 112).
    // Over 260 shapes in both types (1 to 9 requests, 256 to 8000 positions, pages of 16 to 128, with and without a window)
    // the kernel that these limits choose is 0.9 % (64), 0.2 % and 0 % slower than the faster of the two in the mean, at
    // worst 19 %, 19 % and 0 %.
    const uint64_t per = d == 256 ? 128 : 256, rows = (uint64_t)a.n_tok * a.group;
    const uint64_t ctas = (rows / per + a.n_req) * a.c.heads, waves = (ctas + sms - 1) / sms;
    return rows * a.c.heads > waves * (d == 64 ? 7700 : d == 128 ? 6850 : 4900);
}

}  // namespace sg
