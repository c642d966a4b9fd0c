// kv4_attn.cu — attention over the paged 4-bit KV cache for few query rows per
// KV head (decode, verify batches): what bounds it is reading the cache once.
//
// Work.  A segment is eight query rows (a row is a (token, head of the group)
// pair) of one request against one KV head; it is cut into steps of STEP
// positions, and the steps of all segments, in order, are dealt to the warps of
// the device in equal contiguous stretches, so that ragged batches and a single
// long request are spread alike.  Each warp streams its steps' tiles through its
// own ring in shared memory (one bulk copy a step where the page allows it) and
// never waits for another warp.  Segments that end up whole in a warp are written
// by it; the others' partial results (running maximum m, sum l, unnormalised
// rows) meet in shared memory at the end of the CTA, and those that span CTAs in
// scratch, where the last CTA to arrive joins them, always in position order.
//
// Arithmetic.  All products are m16n8k16 f16 tensor operations with f32 sums,
// and the cache's codes go into them as they are: a code c masked out of its
// word is the f16 number c * 2^-24 (or c * 2^-20), exact, so a pair of values
// costs one AND.  With a value m + s c, per group g of 32 values
//   q.k   = sum_g s_g (q_g . c_g) + sum_g m_g sum(q_g)
//   sum_t p_t v_t = sum_t (p_t s_tg) c_t + sum_t p_t m_tg
// where the scales s_g are applied in f32 to the small results on the K side and
// to p on the V side.  The sixteen rows of an operand hold the eight query rows
// twice: the f16 rounding of a number above, the f16 rounding of what that left
// below (about 22 bits together), for p, p s and an f32 q.  A 16-bit q is exact
// after scaling by a power of two.  So every product is as good as one in f32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace sg {

namespace {

template <typename T>
struct Act;
template <>
struct Act<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Act<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Act<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// N words of shared memory (8- or 16-byte aligned).
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], const uint8_t *p) {
    if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p + i * 4);
            w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
        }
    }
}
// The code words of all groups of lane part j out of J (kv4_word).
template <int G, int J>
__device__ __forceinline__ void lds_codes(uint32_t (&w)[G], const uint8_t *row, uint32_t j) {
    if constexpr (G == 2) {
        lds_words<2>(w, row + j * 8);
    } else {
#pragma unroll
        for (int a = 0; a < G / 4; a++) {
            const uint4 v = *reinterpret_cast<const uint4 *>(row + (a * J + j) * 16);
            w[4 * a] = v.x, w[4 * a + 1] = v.y, w[4 * a + 2] = v.z, w[4 * a + 3] = v.w;
        }
    }
}

constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;
constexpr float P_SHIFT = 10.0f;  // weights are held as 2^10 p: small ones keep their bits in f16
constexpr int ROWS = 8;
constexpr uint32_t MAX_REQ = 2048;  // requests of one launch (their prefix sums are in shared memory)
constexpr uint32_t MAX_CTAS = 320;

template <int D>
struct Cfg {
    // D = 256 holds 128 sums a lane: 8 warps of at most 255 registers, steps of one tile
    static constexpr int WARPS = D == 256 ? 8 : 12;
    static constexpr int TILES = D == 256 ? 1 : 2;
    static constexpr int STAGES = D == 256 ? 3 : 2;
    static constexpr int STEP = TILES * 16;
    static constexpr uint32_t STAGE_BYTES = TILES * Kv4Tile<D>::BYTES;
    static constexpr uint32_t PART_BYTES = ROWS * D * 4 + 2 * ROWS * 4;  // rows, m, l
    static constexpr uint32_t RING = WARPS * STAGES * STAGE_BYTES;
    static constexpr uint32_t SMEM = RING + WARPS * PART_BYTES + (MAX_REQ + 1) * 8 + WARPS * STAGES * 8 + 1024;
    static_assert(STAGES * STAGE_BYTES >= PART_BYTES, "a warp's last partial result lies in its ring");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};
constexpr uint32_t PART_MAX = Cfg<256>::PART_BYTES;
static_assert(4096 + (uint64_t)MAX_CTAS * 2 * PART_MAX <= KV4_SCRATCH_BYTES, "scratch");

// The steps of one request, the same for each of its heads and row tiles.
struct Req {
    int32_t tok0, nq, seq;      // first packed token, new tokens, positions
    uint32_t s0, steps, tiles;  // first step, steps (at least one where there are rows), row tiles
};

template <int STEP>
__device__ __forceinline__ Req req_of(const Kv4AttnArgs &a, uint32_t i) {
    Req r;
    r.tok0 = max(a.cu[i], 0);
    r.nq = max(min(a.cu[i + 1], (int32_t)a.n_tok) - r.tok0, 0);
    const int64_t cap = (int64_t)a.width << a.c.page_shift;
    const int32_t seq = max(a.seq[i], 0);
    r.seq = seq < cap ? seq : (int32_t)cap;
    int32_t lo = 0;
    if (a.window && seq - r.nq + 1 > (int64_t)a.window) lo = seq - r.nq + 1 - (int32_t)a.window;
    r.s0 = min(lo, r.seq) / STEP;
    const uint32_t s1 = (r.seq + STEP - 1) / STEP;
    r.steps = r.nq ? max(1u, s1 - min(s1, r.s0)) : 0;
    r.tiles = (uint32_t)(((uint64_t)r.nq * a.group + ROWS - 1) / ROWS);
    return r;
}

struct Seg {
    Req r;
    uint32_t req, head, tile;
    uint64_t begin;  // its first step among all steps
};

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::WARPS * 32, 1) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using L = Kv4Tile<D>;
    using C = Cfg<D>;
    constexpr int G = L::G, TILES = C::TILES, STAGES = C::STAGES, STEP = C::STEP, WARPS = C::WARPS;
    constexpr bool Q32 = sizeof(T) == 4;
    constexpr int QR = Q32 ? 4 : 2;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring_all = smem;
    float *first_all = reinterpret_cast<float *>(smem + C::RING);
    uint64_t *pre = reinterpret_cast<uint64_t *>(smem + C::RING + WARPS * C::PART_BYTES);  // [n_req + 1] steps before each request
    uint64_t *bars = pre + MAX_REQ + 1;
    uint64_t *seg_begin = bars + WARPS * STAGES;                      // [2 * WARPS] the partials' segments, ~0: none
    uint64_t *scan_s = seg_begin + 2 * WARPS;                         // [WARPS + 1]
    uint32_t *flag_s = reinterpret_cast<uint32_t *>(scan_s + WARPS + 1);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, quad = lane & 3;

    if (lane == 0)
        for (int s = 0; s < STAGES; s++) mbar_init(&bars[warp * STAGES + s], 1);
    fence_mbar_init();
    if (tid < 2 * WARPS) seg_begin[tid] = ~0ull;

    // steps before each request
    uint64_t total = 0;
    for (uint32_t r0 = 0; r0 < a.n_req; r0 += WARPS * 32) {
        uint64_t v = 0;
        if (r0 + tid < a.n_req) {
            const Req r = req_of<STEP>(a, r0 + tid);
            v = (uint64_t)r.steps * r.tiles * a.c.heads;
        }
        uint64_t inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t u = __shfl_up_sync(~0u, inc, o);
            if (lane >= (uint32_t)o) inc += u;
        }
        if (lane == 31) scan_s[warp] = inc;
        __syncthreads();
        uint64_t base = total, all = 0;
        for (int w = 0; w < WARPS; w++) {
            if ((uint32_t)w < warp) base += scan_s[w];
            all += scan_s[w];
        }
        if (r0 + tid < a.n_req) pre[r0 + tid] = base + inc - v;
        total += all;
        __syncthreads();
    }
    if (tid == 0) pre[a.n_req] = total;
    __syncthreads();

    // tokens of no request
    {
        const uint32_t t0 = !a.last ? a.n_tok : a.n_req ? (uint32_t)max(a.cu[a.n_req], 0) : 0;
        const uint64_t n = t0 < a.n_tok ? (uint64_t)(a.n_tok - t0) * a.n_heads * D : 0;
        for (uint64_t e = (uint64_t)blockIdx.x * (WARPS * 32) + tid; e < n; e += (uint64_t)gridDim.x * (WARPS * 32)) {
            const uint64_t row = e / D, t = t0 + row / a.n_heads, h = row % a.n_heads;
            ((T *)a.out)[t * a.o_tok + h * a.o_head + e % D] = Act<T>::put(0.0f);
            if (a.lse && e % D == 0) a.lse[t * a.n_heads + h] = -INFINITY;
        }
    }

    // this warp's stretch [w0, w1) of the steps; fewer warps a CTA where there is little to do
    const uint64_t per_cta = (total + gridDim.x - 1) / gridDim.x;
    const uint32_t nw = (uint32_t)min((uint64_t)WARPS, max((uint64_t)1, per_cta));
    const uint64_t chunk = (per_cta + nw - 1) / nw, cta_chunk = chunk * nw;
    const uint64_t w0 = min(total, blockIdx.x * cta_chunk + (uint64_t)min(warp, nw) * chunk);
    const uint64_t w1 = warp < nw ? min(total, w0 + chunk) : w0;

    uint8_t *ring = ring_all + warp * (STAGES * C::STAGE_BYTES);
    uint64_t *bar = bars + warp * STAGES;

    auto seg_at = [&](uint64_t idx) {
        uint32_t x = 0, y = a.n_req;
        while (y - x > 1) {
            const uint32_t m = (x + y) >> 1;
            if (pre[m] <= idx) x = m;
            else y = m;
        }
        Seg s;
        s.req = x;
        s.r = req_of<STEP>(a, x);
        const uint64_t rem = idx - pre[x], k = rem / s.r.steps;
        s.head = (uint32_t)(k / s.r.tiles);
        s.tile = (uint32_t)(k % s.r.tiles);
        s.begin = pre[x] + k * s.r.steps;
        return s;
    };

    // ---- the copies: one step at a time, the table entries read a step ahead ----
    uint64_t p_idx = w0, p_end = w0;
    const int32_t *p_row = nullptr;
    uint32_t p_head = 0, p_step = 0;
    int32_t p_seq = 0, p_blk[TILES];
    bool dead = false;  // a wait ran out: no further copies
    auto fetch = [&]() {
        if (p_idx >= w1) return;
        if (p_idx >= p_end) {
            const Seg s = seg_at(p_idx);
            p_end = s.begin + s.r.steps;
            p_row = a.tables + (uint64_t)s.req * a.ld_tables;
            p_head = s.head;
            p_step = s.r.s0 + (uint32_t)(p_idx - s.begin);
            p_seq = s.r.seq;
        }
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const uint32_t t = p_step * STEP + i * 16;
            p_blk[i] = (int32_t)t < p_seq ? __ldg(p_row + (t >> a.c.page_shift)) : -1;
        }
    };
    // returns a bit per tile that is there
    auto issue = [&](uint32_t stage) -> uint32_t {
        if (p_idx >= w1) return 0;
        uint32_t there = 0;
#pragma unroll
        for (int i = 0; i < TILES; i++) there |= ((uint32_t)p_blk[i] < a.c.n_blocks) << i;
        if (lane == 0 && !dead) {
            mbar_arrive_expect_tx(&bar[stage], __popc(there) * L::BYTES);
            uint8_t *dst = ring + stage * C::STAGE_BYTES;
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                if (!(there >> i & 1)) continue;
                const uint32_t t = p_step * STEP + i * 16, at = (t & ((1u << a.c.page_shift) - 1)) >> 4;
                const uint8_t *src = a.c.data + ((((uint64_t)p_blk[i] * a.c.heads + p_head) << (a.c.page_shift - 4)) + at) * (uint64_t)L::BYTES;
                bulk_g2s(dst + i * L::BYTES, src, L::BYTES, &bar[stage]);
            }
        }
        p_idx++;
        p_step++;
        return there;
    };
    uint32_t there[STAGES];
#pragma unroll
    for (int s = 0; s < STAGES; s++) {
        fetch();
        there[s] = issue(s);
    }
    fetch();

    // ---- the steps ----
    uint32_t qa[2 * G][QR], qs[G == 8 ? 2 : 1];
    float o[4 * G][4], om[4];
    float m = -INFINITY, l = 0.0f, cs = 0.0f;
    int32_t lo_t = 0, hi_t = 0, full_lo = 0, full_hi = 0;
    int32_t kexp = 15;        // of group lane % G: V scales are multiplied by 2^kexp
    float vlim = -1.0f;       // and are at most this
    uint32_t kmul[G];         // f16x2 of each group's 2^kexp
    uint64_t seg_end = w0;
    Seg seg;
    uint32_t phase = 0, stage = 0;

    // the rows' sums in values: lane holds row gid, d = 32 g + 8 quad + 0..7 of each group in r[g]
    auto rows_of = [&](float (&r)[G][8]) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int k = __shfl_sync(~0u, kexp, g);
            const float f = __uint_as_float((uint32_t)(127 + 24 - k) << 23);
            const int src = (lane & 28) | (g >> 1);
            const float mn = (g & 1) ? __shfl_sync(~0u, om[1] + om[3], src) : __shfl_sync(~0u, om[0] + om[2], src);
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float fn = n & 1 ? f * 0.0625f : f;
                r[g][n] = fmaf(o[4 * g + n][0] + o[4 * g + n][2], fn, mn);
                r[g][4 + n] = fmaf(o[4 * g + n][1] + o[4 * g + n][3], fn, mn);
            }
        }
    };
    auto put_part = [&](float *part, const float (&r)[G][8]) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            float4 *p = reinterpret_cast<float4 *>(part + gid * D + g * 32 + quad * 8);
            p[0] = make_float4(r[g][0], r[g][1], r[g][2], r[g][3]);
            p[1] = make_float4(r[g][4], r[g][5], r[g][6], r[g][7]);
        }
        if (quad == 0) part[ROWS * D + gid] = m, part[ROWS * D + ROWS + gid] = l;
    };
    auto lse_of = [](float mm, float ll) { return ll == 0.0f ? -INFINITY : (mm - P_SHIFT + log2f(ll)) * LN2; };

    for (uint64_t idx = w0; idx < w1; idx++) {
        if (idx >= seg_end) {
            // a new segment: its query rows as operand registers
            seg = seg_at(idx);
            seg_end = seg.begin + seg.r.steps;
            const uint32_t row = seg.tile * ROWS + gid, tok = row / a.group, hq = seg.head * a.group + row % a.group;
            const bool live = tok < (uint32_t)seg.r.nq;
            const T *q = (const T *)a.q + (uint64_t)(seg.r.tok0 + (live ? tok : 0)) * a.q_tok + hq * a.q_head + quad * 8;
            float x[G][8], amax = 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int n = 0; n < 8; n++) {
                    x[g][n] = live ? Act<T>::get(q[g * 32 + n]) : 0.0f;
                    amax = fmaxf(amax, fabsf(x[g][n]));
                }
            amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
            // q * 2^(14 - e) is below 2^15 in f16; e is kept where 2^(14 - e) and 2^(e + 10) are f32 numbers
            const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 116);
            const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
            cs = a.scale * LOG2E * __uint_as_float((uint32_t)(127 + 10 + e) << 23);
            float sum[G];
#pragma unroll
            for (int g = 0; g < G; g++) {
                sum[g] = 0.0f;
#pragma unroll
                for (int n = 0; n < 8; n++) sum[g] += x[g][n];
                sum[g] += __shfl_xor_sync(~0u, sum[g], 1);
                sum[g] += __shfl_xor_sync(~0u, sum[g], 2);
                sum[g] *= up * 0.015625f;
                // nibbles (0, 4), (1, 5), (2, 6), (3, 7) make the four K registers; those of odd n are 16 c
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const float f = n & 1 ? up * 0.0625f : up, x0 = x[g][n] * f, x1 = x[g][n + 4] * f;
                    const uint32_t hi = pack_h2(x0, x1);
                    const int ks = 2 * g + (n >> 1), at = n & 1;
                    if constexpr (Q32) {
                        const float2 h = unpack_h2(hi);
                        qa[ks][2 * at] = hi;
                        qa[ks][2 * at + 1] = pack_h2(x0 - h.x, x1 - h.y);
                    } else {
                        qa[ks][at] = hi;
                    }
                }
            }
            // sums of the query's groups against the K minima: column k holds group k % G, first the f16
            // rounding, then what it left
            {
                constexpr int KK = G == 8 ? 16 : 8;
#pragma unroll
                for (int w = 0; w < KK / 8; w++) {
                    float v[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint32_t k = w * 8 + quad * 2 + i, part = k / G, gg = k % G;
                        float s = 0.0f;
#pragma unroll
                        for (int g = 0; g < G; g++) s = (uint32_t)g == gg ? sum[g] : s;
                        const float h = __half2float(__float2half_rn(s));
                        v[i] = part == 0 ? h : part == 1 ? s - h : 0.0f;
                    }
                    qs[w] = pack_h2(v[0], v[1]);
                }
            }
            // what this row sees, and what every row of the tile sees
            const int64_t place = (int64_t)a.seq[seg.req] - seg.r.nq + tok;
            hi_t = live ? (int32_t)min(place + 1, (int64_t)seg.r.seq) : 0;
            lo_t = a.window && place + 1 > (int64_t)a.window ? (int32_t)(place + 1 - a.window) : 0;
            full_hi = __reduce_min_sync(~0u, live ? hi_t : 0x7fffffff);
            full_lo = __reduce_max_sync(~0u, live ? lo_t : 0);
            m = -INFINITY, l = 0.0f, kexp = 15, vlim = -1.0f;
#pragma unroll
            for (int i = 0; i < 4 * G; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            om[0] = om[1] = om[2] = om[3] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++) kmul[g] = 0x78007800u;  // 2^15
        }

        if (!dead && !mbar_wait_bounded(&bar[stage], phase, WAIT_LIMIT_NS)) {
            dead = true;
            if (lane == 0) atomicExch(&g_dev_status, (unsigned)DEV_TIMEOUT_TMA);
        }
        dead = __any_sync(~0u, dead);
        const uint8_t *buf = ring + stage * C::STAGE_BYTES;
        const int32_t t0 = (int32_t)(seg.r.s0 + (uint32_t)(idx - seg.begin)) * STEP;
        const uint32_t here = there[0];
        // whole: every row sees every position of the step
        const bool whole = here == (1u << TILES) - 1 && t0 >= full_lo && t0 + STEP <= full_hi;

        // scores
        float s[TILES][4];
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const uint8_t *tile = buf + i * L::BYTES;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                uint32_t w[G], ks[G];
                lds_codes<G, 4>(w, tile + (8 * j + gid) * L::KROW, quad);
                lds_words<G>(ks, tile + L::KS + (4 * j + quad) * (G * 4));
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (G == 8) {
                    const uint32_t km = *reinterpret_cast<const uint32_t *>(tile + L::KM + ((8 * j + gid) * G + 2 * quad) * 2);
                    mma16(c, qs[0], 0, qs[1], 0, km, km);
                } else {
                    const uint32_t km = *reinterpret_cast<const uint32_t *>(tile + L::KM + ((8 * j + gid) * G + (G == 4 ? (quad & 1) * 2 : 0)) * 2);
                    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                        : "r"(qs[0]), "r"(0), "r"(km));
                }
                float s0 = c[0] * 0x1p-18f, s1 = c[1] * 0x1p-18f;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const uint32_t h = w[g] >> 8;
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (Q32) {
                        mma16(d, qa[2 * g][0], qa[2 * g][1], qa[2 * g][2], qa[2 * g][3], w[g] & 0x000F000Fu, w[g] & 0x00F000F0u);
                        mma16(d, qa[2 * g + 1][0], qa[2 * g + 1][1], qa[2 * g + 1][2], qa[2 * g + 1][3], h & 0x000F000Fu, h & 0x00F000F0u);
                        d[0] += d[2], d[1] += d[3];
                    } else {
                        mma16(d, qa[2 * g][0], 0, qa[2 * g][1], 0, w[g] & 0x000F000Fu, w[g] & 0x00F000F0u);
                        mma16(d, qa[2 * g + 1][0], 0, qa[2 * g + 1][1], 0, h & 0x000F000Fu, h & 0x00F000F0u);
                    }
                    const float2 sc = unpack_h2(ks[g]);
                    s0 = fmaf(d[0], sc.x, s0);
                    s1 = fmaf(d[1], sc.y, s1);
                }
                s[i][2 * j] = s0, s[i][2 * j + 1] = s1;
            }
        }
        // positions that a row does not see, and the running maximum
        float top = m;
#pragma unroll
        for (int i = 0; i < TILES; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[i][j] *= cs;
                if (!whole) {
                    const int32_t t = t0 + i * 16 + (j >> 1) * 8 + quad * 2 + (j & 1);
                    if (t < lo_t || t >= hi_t || !(here >> i & 1)) s[i][j] = -INFINITY;
                }
                top = fmaxf(top, s[i][j]);
            }
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
        if (__any_sync(~0u, top > m)) {
            const float f = m == top ? 1.0f : ex2(m - top);
            m = top;
            l *= f;
#pragma unroll
            for (int i = 0; i < 4 * G; i++) o[i][0] *= f, o[i][1] *= f, o[i][2] *= f, o[i][3] *= f;
            om[0] *= f, om[1] *= f, om[2] *= f, om[3] *= f;
        }
        const float shift = m == -INFINITY ? 0.0f : P_SHIFT - m;
#pragma unroll
        for (int i = 0; i < TILES; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[i][j] = ex2(s[i][j] + shift);
                l += s[i][j];
            }

        // values
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const uint8_t *tile = buf + i * L::BYTES;
            // positions of this tile that are held; the others' scales and minima may be anything
            const int32_t held = here >> i & 1 ? seg.r.seq - (t0 + i * 16) : 0;
            const bool part = held < 16;
            // a V scale larger than any before: the group's sums move to a new power of two
            float vmax = 0.0f;
            {
                constexpr int N = G * 8 / 32 ? G * 8 / 32 : 1;
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const uint32_t at = (lane + 32 * k) % (G * 8), pos = at / G * 2;
                    const float2 v = unpack_h2(*reinterpret_cast<const uint32_t *>(tile + L::VS + at * 4));
                    if ((int32_t)pos < held) vmax = fmaxf(vmax, v.x);
                    if ((int32_t)pos + 1 < held) vmax = fmaxf(vmax, v.y);
                }
            }
            if (__any_sync(~0u, vmax > vlim)) {
#pragma unroll
                for (int off = G; off < 32; off <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(~0u, vmax, off));
                if (vmax > vlim) {
                    // 2^kexp times the largest scale is below 2^5 (kexp at most 15, f16's largest power)
                    const int k = min(15, 4 - ((int)(__float_as_uint(vmax) >> 23) - 127));
                    vlim = __uint_as_float((uint32_t)(127 + 5 - k) << 23) * 0.99999994f;
                    const int old = kexp;
                    kexp = min(k, kexp);
                    vmax = __uint_as_float((uint32_t)(127 + kexp - old) << 23);
                } else {
                    vmax = 1.0f;
                }
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const float f = __shfl_sync(~0u, vmax, g);
                    const int k = __shfl_sync(~0u, kexp, g);
                    kmul[g] = (uint32_t)(15 + k) << 10 | (uint32_t)(15 + k) << 26;
#pragma unroll
                    for (int n = 0; n < 4; n++)
                        o[4 * g + n][0] *= f, o[4 * g + n][1] *= f, o[4 * g + n][2] *= f, o[4 * g + n][3] *= f;
                }
            }
            uint32_t vs[2][G], vm[2], v[2][G], ph[2], pl[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                lds_words<G>(vs[j], tile + L::VS + (4 * j + quad) * (G * 4));
                vm[j] = gid < G ? *reinterpret_cast<const uint32_t *>(tile + L::VM + ((4 * j + quad) * G + (G == 8 ? gid : gid % G)) * 4) : 0u;
                lds_codes<G, 8>(v[j], tile + L::VC + (4 * j + quad) * L::VROW, gid);
                if (part) {
                    const int32_t t = 8 * j + 2 * quad;
                    const uint32_t mask = t + 1 < held ? 0xffffffffu : t < held ? 0xffffu : 0u;
                    vm[j] &= mask;
#pragma unroll
                    for (int g = 0; g < G; g++) vs[j][g] &= mask;
                }
                ph[j] = pack_h2(s[i][2 * j], s[i][2 * j + 1]);
                const float2 h = unpack_h2(ph[j]);
                pl[j] = pack_h2(s[i][2 * j] - h.x, s[i][2 * j + 1] - h.y);
            }
            mma16(om, ph[0], pl[0], ph[1], pl[1], vm[0], vm[1]);
#pragma unroll
            for (int g = 0; g < G; g++) {
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float2 sc = unpack_h2(mul_h2(vs[j][g], kmul[g]));
                    hi[j] = pack_h2(s[i][2 * j] * sc.x, s[i][2 * j + 1] * sc.y);
                    const float2 h = unpack_h2(hi[j]);
                    lo[j] = pack_h2(fmaf(s[i][2 * j], sc.x, -h.x), fmaf(s[i][2 * j + 1], sc.y, -h.y));
                }
                const uint32_t w0_ = v[0][g], w1_ = v[1][g], h0 = w0_ >> 8, h1 = w1_ >> 8;
                mma16(o[4 * g], hi[0], lo[0], hi[1], lo[1], w0_ & 0x000F000Fu, w1_ & 0x000F000Fu);
                mma16(o[4 * g + 1], hi[0], lo[0], hi[1], lo[1], w0_ & 0x00F000F0u, w1_ & 0x00F000F0u);
                mma16(o[4 * g + 2], hi[0], lo[0], hi[1], lo[1], h0 & 0x000F000Fu, h1 & 0x000F000Fu);
                mma16(o[4 * g + 3], hi[0], lo[0], hi[1], lo[1], h0 & 0x00F000F0u, h1 & 0x00F000F0u);
            }
        }

        // the stage is read: the next copy into it
        __syncwarp();
#pragma unroll
        for (int k = 0; k + 1 < STAGES; k++) there[k] = there[k + 1];
        there[STAGES - 1] = issue(stage);
        fetch();
        if (++stage == STAGES) stage = 0, phase ^= 1;

        if (idx + 1 == seg_end || idx + 1 == w1) {
            // the end of the segment, or of this warp's part of it
            l += __shfl_xor_sync(~0u, l, 1);
            l += __shfl_xor_sync(~0u, l, 2);
            float r[G][8];
            rows_of(r);
            const bool begins = seg.begin >= w0, ends = seg_end <= w1;
            if (begins && ends) {
                const uint32_t row = seg.tile * ROWS + gid, tok = row / a.group, hq = seg.head * a.group + row % a.group;
                if (tok < (uint32_t)seg.r.nq) {
                    const uint64_t t = (uint64_t)seg.r.tok0 + tok;
                    T *out = (T *)a.out + t * a.o_tok + hq * a.o_head + quad * 8;
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        alignas(16) T y[8];
#pragma unroll
                        for (int n = 0; n < 8; n++) y[n] = Act<T>::put(r[g][n] * inv);
                        if (a.vec_out) {
#pragma unroll
                            for (int k = 0; k < (int)sizeof(T) / 2; k++)
                                reinterpret_cast<uint4 *>(out + g * 32)[k] = reinterpret_cast<const uint4 *>(y)[k];
                        } else {
#pragma unroll
                            for (int n = 0; n < 8; n++) out[g * 32 + n] = y[n];
                        }
                    }
                    if (a.lse && quad == 0) a.lse[t * a.n_heads + hq] = lse_of(m, l);
                }
            } else {
                // at most one part that began before this warp, and one that goes on after it
                const uint32_t k = begins ? 1 : 0;
                put_part(k ? reinterpret_cast<float *>(ring) : first_all + warp * (C::PART_BYTES / 4), r);
                if (lane == 0) seg_begin[2 * warp + k] = seg.begin;
            }
        }
    }
    if (dead) {  // copies still in flight must not land in memory that is used for something else
        for (int s = 0; s < STAGES; s++) mbar_wait_bounded(&bar[s], phase, WAIT_LIMIT_NS / 20);
    }
    __syncthreads();

    // ---- joining the CTA's partial results, segment by segment ----
    uint32_t *counters = reinterpret_cast<uint32_t *>(a.scratch);
    float *parts = reinterpret_cast<float *>(a.scratch + 4096);
    constexpr uint32_t PART = C::PART_BYTES / 4;
    auto slot = [&](uint32_t k) -> const float * {
        return k & 1 ? reinterpret_cast<const float *>(ring_all + (k >> 1) * (STAGES * C::STAGE_BYTES)) : first_all + (k >> 1) * PART;
    };
    const uint64_t c0 = min(total, blockIdx.x * cta_chunk), c1 = min(total, c0 + cta_chunk);
    for (uint32_t k0 = 0; k0 < 2 * WARPS;) {
        const uint64_t sb = seg_begin[k0];
        if (sb == ~0ull) {
            k0++;
            continue;
        }
        uint32_t k1 = k0 + 1;
        while (k1 < 2 * WARPS && (seg_begin[k1] == sb || seg_begin[k1] == ~0ull)) k1++;
        const Seg sg_ = seg_at(sb);
        const uint64_t se = sb + sg_.r.steps;
        const bool all_here = sb >= c0 && se <= c1;
        const uint32_t cb = (uint32_t)(sb / cta_chunk), ce = (uint32_t)((se - 1) / cta_chunk);
        // joins the rows of n partial results, a thread per value
        auto join_out = [&](uint32_t n, auto part, auto ld, bool final_, float *dst) {
            for (uint32_t e = tid; e < ROWS * D; e += WARPS * 32) {
                const uint32_t row = e / D, d = e % D;
                float mm = -INFINITY;
                for (uint32_t i = 0; i < n; i++) {
                    const float *p = part(i);
                    if (p) mm = fmaxf(mm, ld(p + ROWS * D + row));
                }
                float acc = 0.0f, ll = 0.0f;
                for (uint32_t i = 0; i < n; i++) {
                    const float *p = part(i);
                    if (!p) continue;
                    const float mi = ld(p + ROWS * D + row), w = mi == mm ? 1.0f : ex2(mi - mm);
                    acc = fmaf(w, ld(p + e), acc);
                    ll = fmaf(w, ld(p + ROWS * D + ROWS + row), ll);
                }
                if (!final_) {
                    dst[e] = acc;
                    if (d == 0) dst[ROWS * D + row] = mm, dst[ROWS * D + ROWS + row] = ll;
                    continue;
                }
                const uint32_t rr = sg_.tile * ROWS + row, tok = rr / a.group, hq = sg_.head * a.group + rr % a.group;
                if (tok >= (uint32_t)sg_.r.nq) continue;
                const uint64_t t = (uint64_t)sg_.r.tok0 + tok;
                ((T *)a.out)[t * a.o_tok + hq * a.o_head + d] = Act<T>::put(ll == 0.0f ? 0.0f : acc / ll);
                if (a.lse && d == 0) a.lse[t * a.n_heads + hq] = lse_of(mm, ll);
            }
        };
        auto in_smem = [&](uint32_t i) -> const float * { return seg_begin[k0 + i] == sb ? slot(k0 + i) : nullptr; };
        float *mine = parts + (uint64_t)(blockIdx.x * 2 + (sb < c0 ? 0 : 1)) * PART;
        join_out(k1 - k0, in_smem, [](const float *p) { return *p; }, all_here, mine);
        if (!all_here) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const uint32_t before = atomicAdd(&counters[cb], 1u);
                *flag_s = before == ce - cb;
                if (before == ce - cb) counters[cb] = 0;
            }
            __syncthreads();
            if (*flag_s) {
                __threadfence();
                auto in_scratch = [&](uint32_t i) -> const float * { return parts + (uint64_t)((cb + i) * 2 + (i ? 0 : 1)) * PART; };
                join_out(ce - cb + 1, in_scratch, [](const float *p) { return __ldcg(p); }, true, nullptr);
            }
            __syncthreads();
        }
        k0 = k1;
    }
}

namespace {

template <typename T, int D>
sg_status launch(const Kv4AttnArgs &a0, int sms, cudaStream_t s, cudaError_t *err) {
    auto fn = kv4_attn_kernel<T, D>;
    static bool ready[64];
    int dev = 0;
    if ((*err = cudaGetDevice(&dev)) != cudaSuccess) return SG_ERR_CUDA;
    if (!ready[dev & 63]) {
        if ((*err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM)) != cudaSuccess) return SG_ERR_CUDA;
        ready[dev & 63] = true;
    }
    const uint32_t grid = (uint32_t)sms < MAX_CTAS ? (uint32_t)sms : MAX_CTAS;
    // MAX_REQ requests a launch; the tokens of no request are those after the last one's
    for (uint32_t r0 = 0; r0 == 0 || r0 < a0.n_req; r0 += MAX_REQ) {
        Kv4AttnArgs a = a0;
        a.n_req = a0.n_req - r0 < MAX_REQ ? a0.n_req - r0 : MAX_REQ;
        if (r0) a.cu += r0, a.seq += r0, a.tables += (uint64_t)r0 * a.ld_tables;
        a.last = r0 + a.n_req == a0.n_req;
        fn<<<grid, Cfg<D>::WARPS * 32, Cfg<D>::SMEM, s>>>(a);
        if ((*err = cudaGetLastError()) != cudaSuccess) return SG_ERR_CUDA;
    }
    return SG_OK;
}

template <typename T>
sg_status pick(const Kv4AttnArgs &a, uint32_t d, int sms, cudaStream_t s, cudaError_t *err) {
    return d == 64 ? launch<T, 64>(a, sms, s, err) : d == 128 ? launch<T, 128>(a, sms, s, err) : launch<T, 256>(a, sms, s, err);
}

}  // namespace

sg_status kv4_attention_launch(const Kv4AttnArgs &a, int32_t type, uint32_t d, int sms, cudaStream_t s, cudaError_t *err) {
    return type == SG_F32 ? pick<float>(a, d, sms, s, err) : type == SG_F16 ? pick<__half>(a, d, sms, s, err) : pick<__nv_bfloat16>(a, d, sms, s, err);
}

}  // namespace sg
