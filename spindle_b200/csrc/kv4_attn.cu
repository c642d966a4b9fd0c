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
// to p on the V side.  The codes are the 16-row operand (16 positions for the
// scores, 16 values of a position for the sums), the eight query rows the 8-wide
// one; p, p s and an f32 q go in as the f16 rounding and, in a second product,
// the rounding of what that left (about 22 bits together).  A 16-bit q is exact
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

__device__ __forceinline__ uint32_t fma_h2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
// Any half of a larger than b's: both hold f16 numbers that are not negative.
__device__ __forceinline__ bool any_gt_h2(uint32_t a, uint32_t b) { return __vmaxu2(a, b) != b; }

// d = a b, d += a b
__device__ __forceinline__ void mma16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma8_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
}
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An 8 x 8 matrix of 16-bit numbers, a row per four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

// Four neighbouring values of an output row.
template <typename T>
__device__ __forceinline__ void put4(T *out, float x, float y, float z, float w, bool vec) {
    alignas(16) T v[4] = {Act<T>::put(x), Act<T>::put(y), Act<T>::put(z), Act<T>::put(w)};
    if (vec) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<const uint4 *>(v);
        else *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(v);
    } else {
        out[0] = v[0], out[1] = v[1], out[2] = v[2], out[3] = v[3];
    }
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
// Weights are held as 2^P_SHIFT p with p below 2^LAG; V scales are brought below 2^5, so that a product
// stays inside f16's range above and keeps 30 bits below its largest.
constexpr float P_SHIFT = 2.0f, LAG = 8.0f;
constexpr int ROWS = 8;
constexpr uint32_t MAX_REQ = 1024;  // requests of one launch (their steps are in shared memory)
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
    static constexpr uint32_t SMEM = RING + WARPS * PART_BYTES + (MAX_REQ + 1) * 8 + MAX_REQ * 16 + WARPS * STAGES * 8 + 1024 + (MAX_CTAS + 2) * ROWS * 4;
    static_assert(STAGES * STAGE_BYTES >= PART_BYTES, "a warp's last partial result lies in its ring");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};
constexpr uint32_t PART_MAX = Cfg<256>::PART_BYTES;
static_assert(4096 + (uint64_t)MAX_CTAS * 2 * PART_MAX <= KV4_SCRATCH_BYTES, "scratch");

// One request: its steps are the same for each of its heads and row tiles.
struct Req {
    int32_t tok0, nq, seq;  // first packed token, new tokens, positions (as given: seq - nq is the first new one's place)
    uint32_t s0;            // first step
};

template <int STEP>
__device__ __forceinline__ Req req_of(const Kv4AttnArgs &a, uint32_t i, uint32_t &steps) {
    Req r;
    r.tok0 = max(a.cu[i], 0);
    r.nq = max(min(a.cu[i + 1], (int32_t)a.n_tok) - r.tok0, 0);
    r.seq = max(a.seq[i], 0);
    const int64_t cap = (int64_t)a.width << a.c.page_shift;
    const int32_t end = r.seq < cap ? r.seq : (int32_t)cap;
    int32_t lo = 0;
    if (a.window && r.seq - r.nq + 1 > (int64_t)a.window) lo = r.seq - r.nq + 1 - (int32_t)a.window;
    const uint32_t s1 = (end + STEP - 1) / STEP;
    r.s0 = min((uint32_t)lo / STEP, s1);
    steps = r.nq ? max(1u, s1 - r.s0) : 0;  // at least one where there are rows to write
    return r;
}

struct Seg {
    Req r;
    int32_t end;  // positions that the table has room for
    uint32_t req, head, tile, steps;
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
    Req *reqs = reinterpret_cast<Req *>(pre + MAX_REQ + 1);
    uint64_t *bars = reinterpret_cast<uint64_t *>(reqs + MAX_REQ);
    uint64_t *seg_begin = bars + WARPS * STAGES;                      // [2 * WARPS] the partials' segments, ~0: none
    uint64_t *scan_s = seg_begin + 2 * WARPS;                         // [WARPS + 1]
    uint32_t *flag_s = reinterpret_cast<uint32_t *>(scan_s + WARPS + 1);
    float *weight_s = reinterpret_cast<float *>(flag_s + 2), *ml_s = weight_s + MAX_CTAS * ROWS;  // of the joins
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, quad = lane & 3;

    if (lane == 0)
        for (int s = 0; s < STAGES; s++) mbar_init(&bars[warp * STAGES + s], 1);
    fence_mbar_init();
    if (tid < 2 * WARPS) seg_begin[tid] = ~0ull;

    auto tiles_of = [&](const Req &r) { return ((uint32_t)r.nq * a.group + ROWS - 1) / ROWS; };

    // steps before each request
    uint64_t total = 0;
    for (uint32_t r0 = 0; r0 < a.n_req; r0 += WARPS * 32) {
        uint64_t v = 0;
        if (r0 + tid < a.n_req) {
            uint32_t steps;
            const Req r = req_of<STEP>(a, r0 + tid, steps);
            reqs[r0 + tid] = r;
            v = (uint64_t)steps * tiles_of(r) * a.c.heads;
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
        s.r = reqs[x];
        const uint32_t tiles = tiles_of(s.r);
        const uint64_t rem = idx - pre[x], all = pre[x + 1] - pre[x];
        s.end = (int32_t)min((int64_t)s.r.seq, (int64_t)a.width << a.c.page_shift);
        s.steps = max(1u, (uint32_t)(s.end + STEP - 1) / STEP - s.r.s0);
        uint64_t k;
        if (all >> 32) k = rem / s.steps;
        else k = (uint32_t)rem / s.steps;
        s.head = tiles == 1 ? (uint32_t)k : (uint32_t)(k / tiles);
        s.tile = (uint32_t)k - s.head * tiles;
        s.begin = pre[x] + k * s.steps;
        return s;
    };

    // ---- the copies: a step at a time, the table entries of 32 pages in the lanes ----
    const uint32_t n = (uint32_t)(w1 - w0);
    uint32_t p_i = 0, p_end = 0, p_t = 0, p_page = 0, p_req = 0, p_head = 0;
    int32_t p_blk = -1, p_seq = 0;
    bool dead = false;  // a wait ran out: no further copies
    auto pages = [&]() {
        p_page = p_t >> a.c.page_shift;
        const uint64_t page = (uint64_t)p_page + lane;
        p_blk = (int64_t)(page << a.c.page_shift) < p_seq ? __ldg(a.tables + (uint64_t)p_req * a.ld_tables + page) : -1;
    };
    // copies the next step into a stage; returns a bit per tile that is there
    auto issue = [&](uint32_t stage) -> uint32_t {
        if (p_i >= n) return 0;
        if (p_i == p_end) {
            const Seg s = seg_at(w0 + p_i);
            p_end = (uint32_t)min((uint64_t)n, s.begin + s.steps - w0);
            p_req = s.req, p_head = s.head, p_seq = s.end;
            p_t = (s.r.s0 + (uint32_t)(w0 + p_i - s.begin)) * STEP;
            pages();
        }
        uint8_t *dst = ring + stage * C::STAGE_BYTES;
        uint32_t there = 0;
        const uint32_t shift = a.c.page_shift;
        const uint64_t head_off = ((uint64_t)p_head << (shift - 4)) * L::BYTES;
        if ((1u << shift) >= STEP) {  // the step lies in one page
            if ((p_t >> shift) - p_page >= 32) pages();
            const uint32_t blk = (uint32_t)__shfl_sync(~0u, p_blk, (p_t >> shift) - p_page);
            there = blk < a.c.n_blocks ? (1u << TILES) - 1 : 0;
            if (lane == 0 && !dead) {
                mbar_arrive_expect_tx(&bar[stage], there ? C::STAGE_BYTES : 0);
                if (there)
                    bulk_g2s(dst, a.c.data + blk * a.block_bytes + head_off + ((p_t & ((1u << shift) - 1)) >> 4) * L::BYTES, C::STAGE_BYTES,
                             &bar[stage]);
            }
        } else {  // a page per tile
            uint32_t blk[TILES];
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                if ((p_t >> 4) + i - p_page >= 32) {
                    p_t += 16 * i;
                    pages();
                    p_t -= 16 * i;
                }
                blk[i] = (uint32_t)__shfl_sync(~0u, p_blk, (p_t >> 4) + i - p_page);
                there |= (blk[i] < a.c.n_blocks) << i;
            }
            if (lane == 0 && !dead) {
                mbar_arrive_expect_tx(&bar[stage], __popc(there) * L::BYTES);
#pragma unroll
                for (int i = 0; i < TILES; i++)
                    if (there >> i & 1) bulk_g2s(dst + i * L::BYTES, a.c.data + blk[i] * a.block_bytes + head_off, L::BYTES, &bar[stage]);
            }
        }
        p_i++;
        p_t += STEP;
        return there;
    };
    uint32_t there = 0;  // the bits of the steps in the ring, the next one's lowest
#pragma unroll
    for (int s = 0; s < STAGES; s++) there |= issue(s) << (s * TILES);

    // ---- the steps ----
    // Operands: scores are K codes (16 positions) times query rows (8), sums V codes (16 values) times weights
    // (8 rows), so that a lane of quad `quad` has rows 2 quad and 2 quad + 1 of every result.
    uint32_t qb[2 * G][QR], qs[G == 8 ? 2 : 1];
    float o[2 * G][4], om[4];
    float m[2], l[2], cs[2];
    int32_t lo_t[2], hi_t[2], full_lo = 0, full_hi = 0;  // positions [lo, hi) that a row sees; that all rows see
    int32_t kexp = 15;   // of group lane % G: V scales are multiplied by 2^kexp
    uint32_t vlim2 = 0;  // and are at most this (f16x2)
    uint32_t kmul[G];    // f16x2 of each group's 2^kexp
    uint32_t c_end = 0, phase = 0, stage = 0;
    int32_t t0 = 0, held_end = 0;  // the step's first position, the positions held
    const uint32_t half_sel = gid & 1 ? 0x7632u : 0x5410u;

    // the sums as values: rows 2 quad + i, d = 32 g + 4 gid + n in r[g][i][n]
    auto rows_of = [&](float (&r)[G][2][4]) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int k = __shfl_sync(~0u, kexp, g);
            const float f = __uint_as_float((uint32_t)(127 + 24 - k) << 23), f16 = f * 0.0625f;  // odd nibbles came in 16-fold
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float mn = __shfl_sync(~0u, om[i], 4 * g + quad);
                r[g][i][0] = fmaf(o[2 * g][i], f, mn);
                r[g][i][1] = fmaf(o[2 * g][2 + i], f16, mn);
                r[g][i][2] = fmaf(o[2 * g + 1][i], f, mn);
                r[g][i][3] = fmaf(o[2 * g + 1][2 + i], f16, mn);
            }
        }
    };
    auto lse_of = [](float mm, float ll) { return ll == 0.0f ? -INFINITY : (mm - P_SHIFT + log2f(ll)) * LN2; };

    for (uint32_t idx = 0; idx < n; idx++, t0 += STEP) {
        if (idx == c_end) {
            // a new segment: its query rows as operand registers
            const Seg seg = seg_at(w0 + idx);
            c_end = (uint32_t)min((uint64_t)n, seg.begin + seg.steps - w0);
            t0 = (int32_t)(seg.r.s0 + (uint32_t)(w0 + idx - seg.begin)) * STEP;
            held_end = seg.end;
            const uint32_t row = seg.tile * ROWS + gid, tok = row / a.group, hq = seg.head * a.group + row % a.group;
            const bool live = tok < (uint32_t)seg.r.nq;
            const T *q = (const T *)a.q + (uint64_t)(seg.r.tok0 + (live ? tok : 0)) * a.q_tok + hq * a.q_head + quad * 8;
            alignas(16) T raw[G][8];
            if (a.vec_q) {
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int k = 0; k < (int)sizeof(T) / 2; k++)
                        reinterpret_cast<uint4 *>(raw[g])[k] = __ldg(reinterpret_cast<const uint4 *>(q + g * 32) + k);
            } else {
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int k = 0; k < 8; k++) raw[g][k] = q[g * 32 + k];
            }
            float amax = 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int k = 0; k < 8; k++) amax = fmaxf(amax, live ? fabsf(Act<T>::get(raw[g][k])) : 0.0f);
            amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
            // q * 2^(14 - e) is below 2^15 in f16; e is kept where 2^(14 - e) and 2^(e + 10) are f32 numbers
            const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 116);
            const float up = copysignf(__uint_as_float((uint32_t)(127 + 14 - e) << 23), a.scale);
            const float cs_row = fabsf(a.scale) * LOG2E * __uint_as_float((uint32_t)(127 + 10 + e) << 23);
            float sum[G];
#pragma unroll
            for (int g = 0; g < G; g++) {
                float x[8];
                sum[g] = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    x[k] = live ? Act<T>::get(raw[g][k]) : 0.0f;
                    sum[g] += x[k];
                }
                sum[g] += __shfl_xor_sync(~0u, sum[g], 1);
                sum[g] += __shfl_xor_sync(~0u, sum[g], 2);
                sum[g] *= up * 0.015625f;
                // nibbles (0, 4), (1, 5), (2, 6), (3, 7) make the four K registers; those of odd ones are 16 c
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float f = k & 1 ? up * 0.0625f : up, x0 = x[k] * f, x1 = x[k + 4] * f;
                    const uint32_t hi = pack_h2(x0, x1);
                    qb[2 * g + (k >> 1)][k & 1] = hi;
                    if constexpr (Q32) {
                        const float2 h = unpack_h2(hi);
                        qb[2 * g + (k >> 1)][2 + (k & 1)] = pack_h2(x0 - h.x, x1 - h.y);
                    }
                }
            }
            // sums of the query's groups against the K minima: column k holds group k % G, first the f16
            // rounding, then what it left
#pragma unroll
            for (int w = 0; w < (G == 8 ? 2 : 1); w++) {
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
            // what this row sees, and what every row of the tile sees
            const int64_t place = (int64_t)seg.r.seq - seg.r.nq + tok;
            const int32_t hi_row = live ? (int32_t)max((int64_t)0, min(place + 1, (int64_t)seg.end)) : 0;
            const int32_t lo_row = a.window && place + 1 > (int64_t)a.window ? (int32_t)(place + 1 - a.window) : 0;
            full_hi = __reduce_min_sync(~0u, live ? hi_row : 0x7fffffff);
            full_lo = __reduce_max_sync(~0u, live ? lo_row : 0);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int src = (2 * quad + i) * 4;
                cs[i] = __shfl_sync(~0u, cs_row, src);
                hi_t[i] = __shfl_sync(~0u, hi_row, src);
                lo_t[i] = __shfl_sync(~0u, lo_row, src);
                m[i] = -INFINITY, l[i] = 0.0f;
            }
            kexp = 15, vlim2 = 0x13FF13FFu;  // the f16 below 2^-10
#pragma unroll
            for (int i = 0; i < 2 * G; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
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
        const uint32_t here = there & ((1u << TILES) - 1);
        // whole: every row sees every position of the step
        const bool whole = here == (1u << TILES) - 1 && t0 >= full_lo && t0 + STEP <= full_hi;

        // scores: s[i][2 p + r] of position 16 i + gid + 8 p and row 2 quad + r
        float s[TILES][4];
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const uint8_t *tile = buf + i * L::BYTES;
            uint32_t w0_[G], w1_[G], ks0[G], ks1[G];
            lds_codes<G, 4>(w0_, tile + gid * L::KROW, quad);
            lds_codes<G, 4>(w1_, tile + (gid + 8) * L::KROW, quad);
            lds_words<G>(ks0, tile + L::KS + (gid >> 1) * (G * 4));
            lds_words<G>(ks1, tile + L::KS + (4 + (gid >> 1)) * (G * 4));
            constexpr int KMW = G == 2 ? 0 : G == 4 ? 1 : 3;
            const uint32_t km0 = *reinterpret_cast<const uint32_t *>(tile + L::KM + gid * (G * 2) + (quad & KMW) * 4);
            const uint32_t km1 = *reinterpret_cast<const uint32_t *>(tile + L::KM + (gid + 8) * (G * 2) + (quad & KMW) * 4);
            float c[4];
            if constexpr (G == 8) mma16_first(c, km0, km1, km0, km1, qs[0], qs[1]);
            else mma8_first(c, km0, km1, qs[0]);
#pragma unroll
            for (int k = 0; k < 4; k++) s[i][k] = c[k] * 0x1p-18f;
#pragma unroll
            for (int g = 0; g < G; g++) {
                const uint32_t h0 = w0_[g] >> 8, h1 = w1_[g] >> 8;
                float d[4];
                mma16_first(d, w0_[g] & 0x000F000Fu, w1_[g] & 0x000F000Fu, w0_[g] & 0x00F000F0u, w1_[g] & 0x00F000F0u, qb[2 * g][0], qb[2 * g][1]);
                mma16(d, h0 & 0x000F000Fu, h1 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x00F000F0u, qb[2 * g + 1][0], qb[2 * g + 1][1]);
                if constexpr (Q32) {
                    mma16(d, w0_[g] & 0x000F000Fu, w1_[g] & 0x000F000Fu, w0_[g] & 0x00F000F0u, w1_[g] & 0x00F000F0u, qb[2 * g][2], qb[2 * g][3]);
                    mma16(d, h0 & 0x000F000Fu, h1 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x00F000F0u, qb[2 * g + 1][2], qb[2 * g + 1][3]);
                }
                // scales of positions gid (even or odd in its pair) for two groups in one register
                if (g % 2 == 0) {
                    ks0[g] = __byte_perm(ks0[g], ks0[g + 1], half_sel);
                    ks1[g] = __byte_perm(ks1[g], ks1[g + 1], half_sel);
                }
                const float2 sc0 = unpack_h2(ks0[g & ~1]), sc1 = unpack_h2(ks1[g & ~1]);
                const float a0 = g & 1 ? sc0.y : sc0.x, a1 = g & 1 ? sc1.y : sc1.x;
                s[i][0] = fmaf(d[0], a0, s[i][0]), s[i][1] = fmaf(d[1], a0, s[i][1]);
                s[i][2] = fmaf(d[2], a1, s[i][2]), s[i][3] = fmaf(d[3], a1, s[i][3]);
            }
        }
        // positions that a row does not see, and the reference of the weights: a running maximum that follows
        // the true one only when it is 2^LAG behind, so that the sums are seldom rescaled
        if (!whole) {
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int32_t t = t0 + i * 16 + gid + (k >> 1) * 8;
                    if (t < lo_t[k & 1] || t >= hi_t[k & 1] || !(here >> i & 1)) s[i][k] = -INFINITY;
                }
        }
        float top[2];
        bool behind = false;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            top[r] = fmaxf(s[0][r], s[0][2 + r]);
#pragma unroll
            for (int i = 1; i < TILES; i++) top[r] = fmaxf(top[r], fmaxf(s[i][r], s[i][2 + r]));
            top[r] *= cs[r];
            behind |= top[r] > m[r] + LAG;
        }
        if (__any_sync(~0u, behind)) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], off));
                const float mm = fmaxf(m[r], top[r]), f = m[r] == mm ? 1.0f : ex2(m[r] - mm);
                m[r] = mm;
                l[r] *= f;
#pragma unroll
                for (int i = 0; i < 2 * G; i++) o[i][r] *= f, o[i][2 + r] *= f;
                om[r] *= f;
            }
        }
        const float sh0 = m[0] == -INFINITY ? 0.0f : P_SHIFT - m[0], sh1 = m[1] == -INFINITY ? 0.0f : P_SHIFT - m[1];

        // values
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const uint8_t *tile = buf + i * L::BYTES;
            // the weights, and as f16 rounding and rest, turned so that a lane has positions 2 quad + (0, 1) + 8 j of row gid
            uint32_t ph[2], pl[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float p0 = ex2(fmaf(s[i][2 * j], cs[0], sh0)), p1 = ex2(fmaf(s[i][2 * j + 1], cs[1], sh1));
                l[0] += p0, l[1] += p1;
                ph[j] = pack_h2(p0, p1);
                const float2 h = unpack_h2(ph[j]);
                pl[j] = transpose8(pack_h2(p0 - h.x, p1 - h.y));
                ph[j] = transpose8(ph[j]);
            }
            // positions of this tile that are held; the others' scales and minima may be anything
            const int32_t held = here >> i & 1 ? held_end - (t0 + i * 16) : 0;
            const bool part = held < 16;
            // a V scale larger than any before: the group's sums move to a new power of two
            constexpr int N = G == 8 ? 2 : 1;  // the tile's 8 G words of scales, lane l's of group l % G
            uint32_t vw[N];
            bool above = false;
#pragma unroll
            for (int k = 0; k < N; k++) {
                const uint32_t at = (lane + 32 * k) % (G * 8);
                vw[k] = *reinterpret_cast<const uint32_t *>(tile + L::VS + at * 4);
                if (part) {
                    const int32_t t = (int32_t)(at / G) * 2;
                    vw[k] &= t + 1 < held ? 0xffffffffu : t < held ? 0xffffu : 0u;
                }
                above |= any_gt_h2(vw[k], vlim2);
            }
            if (__any_sync(~0u, above)) {
                float vmax = 0.0f;
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const float2 v = unpack_h2(vw[k]);
                    vmax = fmaxf(vmax, fmaxf(v.x, v.y));
                }
#pragma unroll
                for (int off = G; off < 32; off <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(~0u, vmax, off));
                // 2^kexp times the largest scale is below 2^5 (kexp at most 15, f16's largest power of two)
                const int k = min(kexp, 4 - ((int)(__float_as_uint(vmax) >> 23) - 127));
                vmax = __uint_as_float((uint32_t)(127 + k - kexp) << 23);
                kexp = k;
                vlim2 = (uint32_t)((15 + 5 - k) << 10) * 0x10001u - 0x10001u;  // the f16 below 2^(5 - k)
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const float f = __shfl_sync(~0u, vmax, g);
                    const int kg = __shfl_sync(~0u, kexp, g);
                    kmul[g] = (uint32_t)(15 + kg) << 10 | (uint32_t)(15 + kg) << 26;
#pragma unroll
                    for (int k2 = 0; k2 < 4; k2++) o[2 * g][k2] *= f, o[2 * g + 1][k2] *= f;
                }
            }
            uint32_t vs[2][G], vm[2], v[2][G];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                lds_words<G>(vs[j], tile + L::VS + (4 * j + quad) * (G * 4));
                vm[j] = *reinterpret_cast<const uint32_t *>(tile + L::VM + ((4 * j + quad) * G + gid % G) * 4);
                lds_codes<G, 8>(v[j], tile + L::VC + (4 * j + quad) * L::VROW, gid);
                if (part) {
                    const int32_t t = 8 * j + 2 * quad;
                    const uint32_t mask = t + 1 < held ? 0xffffffffu : t < held ? 0xffffu : 0u;
                    vm[j] &= mask;
#pragma unroll
                    for (int g = 0; g < G; g++) vs[j][g] &= mask;
                }
            }
            // row gid of the minima's product is group gid % G
            mma16(om, vm[0], 0, vm[1], 0, ph[0], ph[1]);
            mma16(om, vm[0], 0, vm[1], 0, pl[0], pl[1]);
#pragma unroll
            for (int g = 0; g < G; g++) {
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    // (ph + pl) sc as the f16 rounding of ph sc and the rest
                    const uint32_t sc = mul_h2(vs[j][g], kmul[g]);
                    hi[j] = mul_h2(ph[j], sc);
                    lo[j] = fma_h2(pl[j], sc, fma_h2(ph[j], sc, hi[j] ^ 0x80008000u));
                }
                const uint32_t h0 = v[0][g] >> 8, h1 = v[1][g] >> 8;
                mma16(o[2 * g], v[0][g] & 0x000F000Fu, v[0][g] & 0x00F000F0u, v[1][g] & 0x000F000Fu, v[1][g] & 0x00F000F0u, hi[0], hi[1]);
                mma16(o[2 * g], v[0][g] & 0x000F000Fu, v[0][g] & 0x00F000F0u, v[1][g] & 0x000F000Fu, v[1][g] & 0x00F000F0u, lo[0], lo[1]);
                mma16(o[2 * g + 1], h0 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x000F000Fu, h1 & 0x00F000F0u, hi[0], hi[1]);
                mma16(o[2 * g + 1], h0 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x000F000Fu, h1 & 0x00F000F0u, lo[0], lo[1]);
            }
        }

        // the stage is read: the next copy into it
        __syncwarp();
        there = there >> TILES | issue(stage) << ((STAGES - 1) * TILES);
        if (++stage == STAGES) stage = 0, phase ^= 1;

        if (idx + 1 == c_end) {
            // the end of the segment, or of this warp's part of it
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                l[0] += __shfl_xor_sync(~0u, l[0], off);
                l[1] += __shfl_xor_sync(~0u, l[1], off);
            }
            float r[G][2][4];
            rows_of(r);
            const Seg seg = seg_at(w0 + idx);
            const bool begins = seg.begin >= w0, ends = seg.begin + seg.steps <= w1;
            // a part that began before this warp (at most one) and one that goes on after it (at most one) are left for the joins
            float *part = begins ? reinterpret_cast<float *>(ring) : first_all + warp * (C::PART_BYTES / 4);
            if (lane == 0 && !(begins && ends)) seg_begin[2 * warp + begins] = seg.begin;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t tr = 2 * quad + i;
                if (!(begins && ends)) {
#pragma unroll
                    for (int g = 0; g < G; g++)
                        *reinterpret_cast<float4 *>(part + tr * D + g * 32 + gid * 4) = make_float4(r[g][i][0], r[g][i][1], r[g][i][2], r[g][i][3]);
                    if (gid == 0) part[ROWS * D + tr] = m[i], part[ROWS * D + ROWS + tr] = l[i];
                    continue;
                }
                const uint32_t row = seg.tile * ROWS + tr, tok = row / a.group, hq = seg.head * a.group + row % a.group;
                if (tok >= (uint32_t)seg.r.nq) continue;
                const uint64_t t = (uint64_t)seg.r.tok0 + tok;
                T *out = (T *)a.out + t * a.o_tok + hq * a.o_head + gid * 4;
                const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
#pragma unroll
                for (int g = 0; g < G; g++) put4(out + g * 32, r[g][i][0] * inv, r[g][i][1] * inv, r[g][i][2] * inv, r[g][i][3] * inv, a.vec_out);
                if (a.lse && gid == 0) a.lse[t * a.n_heads + hq] = lse_of(m[i], l[i]);
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
        const uint64_t se = sb + sg_.steps;
        const bool all_here = sb >= c0 && se <= c1;
        const uint32_t cb = (uint32_t)(sb / cta_chunk), ce = (uint32_t)((se - 1) / cta_chunk);
        // Joins the rows of n partial results: the weights of each row by a warp, then a thread per four values
        // with several of the parts' loads in flight.
        auto join_out = [&](uint32_t n, auto part, auto ld4, auto ld, bool final_, float *dst) {
            for (uint32_t row = warp; row < ROWS; row += WARPS) {
                float mm = -INFINITY;
                for (uint32_t i = lane; i < n; i += 32) {
                    const float *p = part(i);
                    const float v = p ? ld(p + ROWS * D + row) : -INFINITY;
                    weight_s[i * ROWS + row] = v;
                    mm = fmaxf(mm, v);
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, o));
                float ll = 0.0f;
                for (uint32_t i = lane; i < n; i += 32) {
                    const float *p = part(i);
                    const float mi = weight_s[i * ROWS + row], w = !p ? 0.0f : mi == mm ? 1.0f : ex2(mi - mm);
                    weight_s[i * ROWS + row] = w;
                    if (p) ll = fmaf(w, ld(p + ROWS * D + ROWS + row), ll);
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) ll += __shfl_xor_sync(~0u, ll, o);
                if (lane == 0) ml_s[row] = mm, ml_s[ROWS + row] = ll;
            }
            __syncthreads();
            for (uint32_t e = tid * 4; e < ROWS * D; e += WARPS * 128) {
                const uint32_t row = e / D, d = e % D;
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                for (uint32_t i = 0; i < n; i++) {
                    const float *p = part(i);
                    const float w = weight_s[i * ROWS + row];
                    const float4 v = p ? ld4(p + e) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    acc.x = fmaf(w, v.x, acc.x), acc.y = fmaf(w, v.y, acc.y), acc.z = fmaf(w, v.z, acc.z), acc.w = fmaf(w, v.w, acc.w);
                }
                const float mm = ml_s[row], ll = ml_s[ROWS + row];
                if (!final_) {
                    *reinterpret_cast<float4 *>(dst + e) = acc;
                    if (d == 0) dst[ROWS * D + row] = mm, dst[ROWS * D + ROWS + row] = ll;
                    continue;
                }
                const uint32_t rr = sg_.tile * ROWS + row, tok = rr / a.group, hq = sg_.head * a.group + rr % a.group;
                if (tok >= (uint32_t)sg_.r.nq) continue;
                const uint64_t t = (uint64_t)sg_.r.tok0 + tok;
                const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                put4((T *)a.out + t * a.o_tok + hq * a.o_head + d, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv, a.vec_out);
                if (a.lse && d == 0) a.lse[t * a.n_heads + hq] = lse_of(mm, ll);
            }
        };
        auto in_smem = [&](uint32_t i) -> const float * { return seg_begin[k0 + i] == sb ? slot(k0 + i) : nullptr; };
        float *mine = parts + (uint64_t)(blockIdx.x * 2 + (sb < c0 ? 0 : 1)) * PART;
        join_out(k1 - k0, in_smem, [](const float *p) { return *reinterpret_cast<const float4 *>(p); },
                 [](const float *p) { return *p; }, all_here, mine);
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
                join_out(ce - cb + 1, in_scratch, [](const float *p) { return __ldcg(reinterpret_cast<const float4 *>(p)); },
                         [](const float *p) { return __ldcg(p); }, true, nullptr);
            }
        }
        __syncthreads();
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
