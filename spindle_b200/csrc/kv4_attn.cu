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
// Measured (device time): one token each of 64 requests of 2048 to 8192 positions, 32 query and 4 KV heads of 128,
// bf16: 59 us, 3.6 TB/s (56 % of the measured copy rate); one request of 131071 positions, 32 and 8 heads, f16: 54
// us, 3.1 TB/s; 1037 positions: 13 us; 16 requests of 9 tokens at 2050 positions in f32: 36 us.  What bounds it is
// issuing instructions: by the counters 730 (bf16), 750 (f16) and 890 (f32) for 32 positions of eight rows, starts and
// joins included.  A call that has almost nothing to read (1037 positions) shows what starting and joining take.
//
// Arithmetic.  All products are m16n8k16 f16 tensor operations with f32 sums, the
// codes the 16-row operand (16 positions for the scores, 16 values of a position
// for the sums), the eight query rows the 8-wide one.  A code becomes an exact f16
// number with a mask into the mantissa of 1024 or 64 and a subtraction, two values
// at a time.  (Masked alone it is a subnormal number, exact too, but the tensor
// cores add such products with ten bits less.)  With a value m + s c, per group g of
// 32 values
//   q.k = sum_g s_g (q_g . c_g) + sum_g m_g sum(q_g)
// with the scales applied in f32 to the small results, and q and its sums as f16
// rounding and, in a second product, the rounding of what that left (about 22 bits
// together; a 16-bit q is exact after scaling by a power of two).  The weights p are
// held the same way (for bf16 without the rest), with as many bits as f16 has above
// 2^-24.  For 16-bit types the V values are made in f16, one rounding each.  For f32
//   sum_t p_t v_t = sum_t (p_t s_tg) (c_t - 8) + sum_t p_t (m_tg + 8 s_tg)
// with p s and m + 8 s in two f16 parts again: around the middle of the codes the
// long sums stay small, so that nothing of them cancels.  The tensor cores cut off
// what does not fit a sum's f32, always towards zero, which over a long stretch of
// small weights after a large one adds up to more than f32 has to lose (4.6e-5 after 4096 positions, 2.2e-6
// now): so f32 sums the products of 16 positions apart and adds them by rounded f32 additions
// (16 requests of 9 tokens: 36.7 -> 38.5 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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
    static __device__ __forceinline__ __half put(float v) { return kv4_f16(v); }
};
template <>
struct Act<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

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

// a b + c, a b - c
__device__ __forceinline__ uint32_t fma_h2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t fms_h2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("{\n .reg .b32 t;\n neg.f16x2 t, %3;\n fma.rn.f16x2 %0, %1, %2, t;\n}" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t add_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t sub_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
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

// c += d, rounded to nearest, two numbers an instruction.
__device__ __forceinline__ void add4(float (&c)[4], const float (&d)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k += 2)
        asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
            : "+f"(c[k]), "+f"(c[k + 1])
            : "f"(d[k]), "f"(d[k + 1]));
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
// Weights are held as 2^P p with p at most 2^LAG, as far up in f16's range as they fit: f16 ends at 2^-24 below, and of a
// weight 2^-k of the largest 25 + P - k bits are left (a long tail of small weights has one error, so it counts).
// 16-bit types: 2^(P + LAG) is f16's largest power of two.  f32: the V scales are brought below 2, and the sums are
// rescaled sooner for more bits below; a product of the two is below 2^15.
template <typename T>
struct Weights {
    static constexpr float P = sizeof(T) == 4 ? 12.0f : 7.0f, LAG = sizeof(T) == 4 ? 2.0f : 8.0f;
};
constexpr int V_TOP = 1;  // f32: V scales below 2^V_TOP
constexpr int ROWS = 8;
constexpr uint32_t MAX_REQ = 1024;  // requests of one launch (their steps are in shared memory)
constexpr uint32_t MAX_CTAS = 192;
// Warps that a CTA uses at least where the steps are few.  One token of 200, 600, 1037, 2000 and 4000 positions, 16 query
// and 8 KV heads of 128 in f16, device time: 7.6, 12.6, 12.7, 11.3, 15.8 us; with 4 of them 12.0, 12.0, 13.3, 15.2, 15.8;
// with 11 13.6, 13.5, 11.3, 14.2, 15.5.  (f32, heads of 64 and of 256, and four requests go the same way.)
constexpr uint32_t MIN_WARPS = 7;

template <typename T, int D>
struct Cfg {
    // As many warps as their sums and query registers leave room for (65536 registers), and one that copies
    static constexpr int WARPS = D == 256 ? 7 : D == 64 ? 15 : 11;
    static constexpr int THREADS = (WARPS + 1) * 32;
    static constexpr int TILES = D == 256 ? 1 : 2;
    static constexpr int STAGES = D == 256 ? 4 : D == 64 ? 4 : 3;
    static constexpr int STEP = TILES * 16;
    static constexpr uint32_t STAGE_BYTES = TILES * Kv4Tile<D>::BYTES;
    static constexpr uint32_t PART_BYTES = ROWS * D * 4 + 2 * ROWS * 4;  // rows, m, l
    static constexpr uint32_t RING = WARPS * STAGES * STAGE_BYTES;
    static constexpr int SEGS = STAGES + 1;
    static constexpr uint32_t SMEM = RING + (MAX_REQ + 1) * 4 + MAX_REQ * 16 + WARPS * (STAGES * 20 + 2 * 8 + (SEGS + 2) * 40 + 4) + 512;
    static_assert(WARPS <= 16, "a lane per partial result");
    static_assert(STAGES * STAGE_BYTES >= PART_BYTES, "a warp's last partial result lies in its ring");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};
// Scratch: arrival counters, two partial results a CTA for the segments that go over its ends, and one a warp for a
// segment that ends in the middle of the warp's work.
constexpr uint64_t PART_MAX = Cfg<float, 256>::PART_BYTES;
static_assert(4096 + MAX_CTAS * (2 + 8) * PART_MAX <= KV4_SCRATCH_BYTES, "scratch");
static_assert(4096 + (uint64_t)MAX_CTAS * (2 + 16) * Cfg<__half, 128>::PART_BYTES <= KV4_SCRATCH_BYTES, "scratch");

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
    uint32_t req, head, tile;
    uint32_t begin, steps;  // its first step among all steps, its steps
};

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<T, D>::THREADS, 1) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using L = Kv4Tile<D>;
    using C = Cfg<T, D>;
    constexpr int G = L::G, TILES = C::TILES, STAGES = C::STAGES, STEP = C::STEP, WARPS = C::WARPS, THREADS = C::THREADS;
    constexpr bool Q32 = sizeof(T) == 4;
    constexpr float P_SHIFT = Weights<T>::P, LAG = Weights<T>::LAG;
    constexpr int QR = Q32 ? 4 : 2;
    constexpr bool REST = !std::is_same<T, __nv_bfloat16>::value;  // what the weights' f16 rounding leaves is far below bf16
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring_all = smem;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::RING);
    uint64_t *frees = bars + WARPS * STAGES;                          // a stage's copy has landed; a stage may be written
    const float **part_at = reinterpret_cast<const float **>(frees + WARPS * STAGES);  // [2 * WARPS] the partial results
    Req *reqs = reinterpret_cast<Req *>(part_at + 2 * WARPS);         // [n_req]
    Seg *segs_all = reinterpret_cast<Seg *>(reqs + MAX_REQ);          // [WARPS][SEGS] the segments in a warp's ring
    Seg *part_seg = segs_all + WARPS * C::SEGS;                       // [2 * WARPS] the partial results' segments
    uint32_t *pre = reinterpret_cast<uint32_t *>(part_seg + 2 * WARPS);  // [n_req + 1] steps before each request
    uint32_t *seg_begin = pre + MAX_REQ + 1;                          // [32] the partials' segments, NONE: no partial
    uint32_t *scan_s = seg_begin + 32;                                // [WARPS + 1]
    uint32_t *flag_s = scan_s + WARPS + 1;                            // [2]
    uint32_t *there_s = flag_s + 2;                                   // [WARPS][STAGES] a bit per tile of a stage that is there
    constexpr uint32_t NONE = 0xffffffffu;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, quad = lane & 3;

    for (uint32_t i = tid; i < 2 * WARPS * STAGES; i += THREADS) mbar_init(&bars[i], 1);
    fence_mbar_init();
    if (tid < 32) seg_begin[tid] = NONE;

    auto tiles_of = [&](const Req &r) { return ((uint32_t)r.nq * a.group + ROWS - 1) / ROWS; };

    const uint32_t spare = !a.last ? a.n_tok : a.n_req ? min((uint32_t)max(a.cu[a.n_req], 0), a.n_tok) : 0;

    // steps before each request
    uint32_t total = 0;
    for (uint32_t r0 = 0; r0 < a.n_req; r0 += THREADS) {
        uint32_t v = 0;
        if (r0 + tid < a.n_req) {
            uint32_t steps;
            const Req r = req_of<STEP>(a, r0 + tid, steps);
            reqs[r0 + tid] = r;
            v = steps * tiles_of(r) * a.n_kv;
        }
        uint32_t inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(~0u, inc, o);
            if (lane >= (uint32_t)o) inc += u;
        }
        if (lane == 31) scan_s[warp] = inc;
        __syncthreads();
        const uint32_t w = lane <= WARPS ? scan_s[lane] : 0;
        const uint32_t base = __reduce_add_sync(~0u, lane < warp ? w : 0);
        if (r0 + tid < a.n_req) pre[r0 + tid] = total + base + inc - v;
        total += __reduce_add_sync(~0u, w);
        __syncthreads();
    }
    if (tid == 0) pre[a.n_req] = total;
    __syncthreads();

    // tokens of no request: those before `lead` and those from `spare` on
    const uint32_t lead = a.first && a.n_req ? min((uint32_t)reqs[0].tok0, a.n_tok) : 0;
    if (lead || spare < a.n_tok) {
        const uint32_t rows = (lead + a.n_tok - spare) * a.n_heads;
        for (uint32_t row = blockIdx.x * (WARPS + 1) + warp; row < rows; row += gridDim.x * (WARPS + 1)) {
            const uint32_t i = row / a.n_heads, h = row % a.n_heads, t = i < lead ? i : spare + i - lead;
            if (h / a.group - a.head0 >= a.n_kv) continue;
            for (uint32_t d = lane; d < D; d += 32) ((T *)a.out)[t * a.o_tok + h * a.o_head + d] = Act<T>::put(0.0f);
            if (a.lse && lane == 0) a.lse[(uint64_t)t * a.n_heads + h] = -INFINITY;
        }
    }

    // the CTA's stretch [c0, c1) of the steps, and a warp's, n from w0 on; fewer warps a CTA where there is little to do.
    // The copying warp's lanes stand for one warp each.
    const uint32_t per_cta = (total + gridDim.x - 1) / gridDim.x, nw = min((uint32_t)WARPS, max((uint32_t)MIN_WARPS, per_cta));
    const uint32_t chunk = (per_cta + nw - 1) / nw, cta_chunk = chunk * nw;
    const uint32_t c0 = min(total, blockIdx.x * cta_chunk), c1 = min(total, c0 + cta_chunk);
    const uint32_t who = warp < WARPS ? warp : min(lane, (uint32_t)WARPS - 1);
    const uint32_t w0 = min(c1, c0 + min(who, nw) * chunk), n = min(c1, w0 + chunk) - w0;

    uint8_t *ring = ring_all + who * (STAGES * C::STAGE_BYTES);
    uint64_t *bar = bars + who * STAGES, *free_bar = frees + who * STAGES;
    Seg *segs = segs_all + who * C::SEGS;

    // The segment of a step; steps * row tiles * heads of a request fit in 32 bits.
    auto seg_at = [&](uint32_t idx) {
        uint32_t x = 0, y = a.n_req;
        while (y - x > 1) {
            const uint32_t m = (x + y) >> 1;
            if (pre[m] <= idx) x = m;
            else y = m;
        }
        Seg s;
        s.req = x;
        s.r = reqs[x];
        const uint32_t tiles = max(1u, tiles_of(s.r));
        s.end = (int32_t)min((int64_t)s.r.seq, (int64_t)a.width << a.c.page_shift);
        s.steps = max(1u, (uint32_t)(s.end + STEP - 1) / STEP - s.r.s0);
        const uint32_t k = (idx - pre[x]) / s.steps, h = tiles == 1 ? k : k / tiles;
        s.head = a.head0 + min(h, a.n_kv - 1);
        s.tile = k - h * tiles;
        s.begin = pre[x] + k * s.steps;
        return s;
    };

    if (warp == WARPS) {
        // ---- the copies: every lane keeps one warp's ring full ----
        uint32_t left = lane < WARPS ? n : 0, end = 0, seg_at_ = 0, t = 0, stage = 0, phase = 1;
        const uint32_t shift = a.c.page_shift;
        const int32_t *row = nullptr;
        const uint8_t *base = nullptr;
        int32_t blk = -1, next = -1, held = 0;
        uint64_t since = 0;
        while (__any_sync(~0u, left)) {
            const bool go = left && mbar_try_wait(&free_bar[stage], phase);
            if (!__any_sync(~0u, go)) {
                // nobody took anything: the warps always come on, so that a long wait is an error
                if (!since) since = globaltimer_ns();
                else if (globaltimer_ns() - since > 2 * WAIT_LIMIT_NS) {
                    if (lane == 0) atomicExch(&g_dev_status, (unsigned)DEV_TIMEOUT_TMA);
                    break;
                }
                continue;
            }
            since = 0;
            if (!go) continue;
            if (end == 0) {  // a new segment
                const uint32_t idx = w0 + n - left;
                const Seg s = seg_at(idx);
                segs[seg_at_] = s;
                if (++seg_at_ == C::SEGS) seg_at_ = 0;
                end = min(left, s.begin + s.steps - idx);
                t = (s.r.s0 + (idx - s.begin)) * STEP;
                held = s.end;
                row = a.tables + (uint64_t)s.req * a.ld_tables;
                base = a.c.data + ((uint64_t)s.head << (shift - 4)) * L::BYTES;
                blk = (int32_t)t < held ? __ldg(row + (t >> shift)) : -1;
                const int64_t u = ((int64_t)(t >> shift) + 1) << shift;
                next = u < held ? __ldg(row + (t >> shift) + 1) : -1;
            }
            // the next table entry is read a page ahead
            auto turn_page = [&](uint32_t page) {
                blk = next;
                next = ((int64_t)page + 1) << shift < held ? __ldg(row + page + 1) : -1;
            };
            uint8_t *dst = ring + stage * C::STAGE_BYTES;
            const uint32_t at = (t & ((1u << shift) - 1)) >> 4;
            uint32_t there = (uint32_t)blk < a.c.n_blocks;
            const uint8_t *src = base + (uint32_t)blk * a.block_bytes + at * L::BYTES;
            if (TILES == 1 || shift > 4) {  // the step lies in one page
                if (there) there = (1u << TILES) - 1;
                there_s[who * STAGES + stage] = there;
                mbar_arrive_expect_tx(&bar[stage], there ? C::STAGE_BYTES : 0);
                if (there) bulk_g2s(dst, src, C::STAGE_BYTES, &bar[stage]);
            } else {  // a page per tile
                turn_page((t >> shift) + 1);
                there |= ((uint32_t)blk < a.c.n_blocks) << 1;
                there_s[who * STAGES + stage] = there;
                mbar_arrive_expect_tx(&bar[stage], __popc(there) * L::BYTES);
                if (there & 1) bulk_g2s(dst, src, L::BYTES, &bar[stage]);
                if (there & 2) bulk_g2s(dst + L::BYTES, base + (uint32_t)blk * a.block_bytes, L::BYTES, &bar[stage]);
            }
            t += STEP;
            if ((t & ((1u << shift) - 1)) == 0) turn_page(t >> shift);
            left--, end--;
            if (++stage == STAGES) stage = 0, phase ^= 1;
        }
    }

    uint32_t *counters = reinterpret_cast<uint32_t *>(a.scratch);
    float *parts = reinterpret_cast<float *>(a.scratch + 4096);
    constexpr uint32_t PART = C::PART_BYTES / 4;

    // ---- the steps ----
    const Kv4Codes codes;
    // Operands: scores are K codes (16 positions) times query rows (8), sums V codes (16 values) times weights
    // (8 rows), so that a lane of quad `quad` has rows 2 quad and 2 quad + 1 of every result.
    uint32_t qb[2 * G][QR], qs[G == 8 ? 2 : 1];
    float o[2 * G][4], om[4];
    float m[2], nm[2], cs[2];  // the weights' reference (a score), its negative (0 for none); what a score is multiplied by
    float l[2];
    int32_t lo_t[2], hi_t[2], full_lo = 0, full_hi = 0;  // positions [lo, hi) that a row sees; that all rows see
    int32_t kexp = 15;   // of group lane % G: V scales are multiplied by 2^kexp
    uint32_t vlim2 = 0;  // and are at most this (f16x2), the f16 below 2^(V_TOP - kexp)
    constexpr uint32_t VLIM15 = ((15 + V_TOP - 15) << 10) * 0x10001u - 0x10001u;
    uint32_t kmul[G];    // f16x2 of each group's 2^kexp
    uint32_t c_end = 0, c_seg = 0, phase = 0, stage = 0;
    int32_t t0 = 0, held_end = 0;  // the step's first position, the positions held
    const uint32_t half_sel = gid & 1 ? 0x7632u : 0x5410u;

    // the sums as values: rows 2 quad + i, d = 32 g + 4 gid + n in r[g][i][n]
    auto rows_of = [&](float (&r)[G][2][4]) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float f = Q32 ? __uint_as_float((uint32_t)(127 - __shfl_sync(~0u, kexp, g)) << 23) : 1.0f;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                // (the middles came in halved)
                const float mn = Q32 ? 2.0f * __shfl_sync(~0u, om[i] + om[2 + i], 4 * g + quad) : 0.0f;
                r[g][i][0] = fmaf(o[2 * g][i], f, mn);
                r[g][i][1] = fmaf(o[2 * g][2 + i], f, mn);
                r[g][i][2] = fmaf(o[2 * g + 1][i], f, mn);
                r[g][i][3] = fmaf(o[2 * g + 1][2 + i], f, mn);
            }
        }
    };
    auto lse_of = [](float mm, float ll) { return ll == 0.0f ? -INFINITY : (mm - P_SHIFT + log2f(ll)) * LN2; };

    bool dead = false;  // a wait ran out
    const uint32_t n_mine = warp < WARPS ? n : 0;
    auto landed = [&]() {
        if (!dead && !mbar_wait_bounded(&bar[stage], phase, WAIT_LIMIT_NS)) {
            dead = true;
            if (lane == 0) atomicExch(&g_dev_status, (unsigned)DEV_TIMEOUT_TMA);
        }
    };
    for (uint32_t idx = 0; idx < n_mine; idx++, t0 += STEP) {
        if (idx) landed();
        if (idx == c_end) {
            // a new segment: its query rows as operand registers; the first one's while its copies are on their way (the
            // others come with theirs)
            const Seg seg = idx ? segs[c_seg] : seg_at(w0);
            c_end = min(n, seg.begin + seg.steps - w0);
            t0 = (int32_t)(seg.r.s0 + (w0 + idx - seg.begin)) * STEP;
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
            // q * 2^(14 - e) is below 2^15 in f16; e is kept where that power and its inverse are f32 numbers.
            // A row that is no row stands in with the values of the first one.
            int e;
            if constexpr (Q32) {
                float amax = 0.0f;
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int k = 0; k < 8; k++) amax = fmaxf(amax, fabsf(raw[g][k]));
                amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
                e = (int)(__float_as_uint(amax) >> 23) - 127;
            } else {
                uint32_t amax = 0;  // the bits without the sign have the order of the values
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int k = 0; k < 4; k++) amax = __vmaxu2(amax, reinterpret_cast<const uint32_t *>(raw[g])[k] & 0x7FFF7FFFu);
                amax = __vmaxu2(amax, amax >> 16);
                amax = __vmaxu2(amax, __shfl_xor_sync(~0u, amax, 1));
                amax = __vmaxu2(amax, __shfl_xor_sync(~0u, amax, 2)) & 0x7FFFu;
                e = std::is_same<T, __half>::value ? (int)(amax >> 10) - 15 : (int)(amax >> 7) - 127;
            }
            e = min(max(e, -100), 116);
            const float up = copysignf(__uint_as_float((uint32_t)(127 + 14 - e) << 23), a.scale);
            // (above 0, so that a position that is not seen stays at minus infinity)
            const float cs_row = fmaxf(fabsf(a.scale) * LOG2E * __uint_as_float((uint32_t)(127 - 14 + e) << 23), 0x1p-126f);
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                // nibbles (0, 4), (1, 5), (2, 6), (3, 7) make the four K registers
                for (int k = 0; k < 4; k++) {
                    const float x0 = Act<T>::get(raw[g][k]) * up, x1 = Act<T>::get(raw[g][k + 4]) * up;
                    const uint32_t hi = pack_h2(x0, x1);
                    qb[2 * g + (k >> 1)][k & 1] = hi;
                    if constexpr (Q32) {
                        const float2 h = unpack_h2(hi);
                        qb[2 * g + (k >> 1)][2 + (k & 1)] = pack_h2(x0 - h.x, x1 - h.y);
                    }
                }
            // The sums of the query's groups, for the K minima: the product with ones.
            // Column k of the operand holds group k % G, first the f16 rounding, then what it left.
            {
                float sum[2] = {0.0f, 0.0f};
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int g = 0; g < G; g++) {
                    float d[4];
                    constexpr uint32_t ONE = 0x3C003C00u;
                    mma16_first(d, ONE, ONE, ONE, ONE, qb[2 * g][0], qb[2 * g][1]);
                    mma16(d, ONE, ONE, ONE, ONE, qb[2 * g + 1][0], qb[2 * g + 1][1]);
                    if constexpr (Q32) {
                        mma16(d, ONE, ONE, ONE, ONE, qb[2 * g][2], qb[2 * g][3]);
                        mma16(d, ONE, ONE, ONE, ONE, qb[2 * g + 1][2], qb[2 * g + 1][3]);
                    }
                    if ((int)(gid % G) == g) sum[0] = d[0], sum[1] = d[1];
                }
                const float f = 0x1p-6f;  // inside f16's range
                hi[0] = pack_h2(sum[0] * f, sum[1] * f);
                const float2 h = unpack_h2(hi[0]);
                lo[0] = pack_h2(fmaf(sum[0], f, -h.x), fmaf(sum[1], f, -h.y));
                if constexpr (G == 8) {
                    qs[0] = transpose8(hi[0]);
                    qs[1] = transpose8(lo[0]);
                } else {
                    qs[0] = transpose8(gid < G ? hi[0] : gid < 2 * G ? lo[0] : 0u);
                }
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
                m[i] = -INFINITY, nm[i] = 0.0f, l[i] = 0.0f;
            }
            kexp = 15, vlim2 = VLIM15;
#pragma unroll
            for (int i = 0; i < 2 * G; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            om[0] = om[1] = om[2] = om[3] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++) kmul[g] = 0x78007800u;  // 2^15
        }

        if (!idx) landed();
        uint8_t *buf = ring + stage * C::STAGE_BYTES;
        const uint32_t here = there_s[warp * STAGES + stage];
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
            for (int k = 0; k < 4; k++) s[i][k] = c[k] * 0x1p6f;
#pragma unroll
            for (int g = 0; g < G; g++) {
                uint32_t ca[4], cb[4];
                codes.get<0>(w0_[g], ca);
                codes.get<0>(w1_[g], cb);
                float d[4];
                mma16_first(d, ca[0], cb[0], ca[1], cb[1], qb[2 * g][0], qb[2 * g][1]);
                mma16(d, ca[2], cb[2], ca[3], cb[3], qb[2 * g + 1][0], qb[2 * g + 1][1]);
                if constexpr (Q32) {
                    mma16(d, ca[0], cb[0], ca[1], cb[1], qb[2 * g][2], qb[2 * g][3]);
                    mma16(d, ca[2], cb[2], ca[3], cb[3], qb[2 * g + 1][2], qb[2 * g + 1][3]);
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
            // the scales and minima of positions that are not held may be anything: zeros in their place
#pragma unroll 1
            for (int i = 0; i < TILES; i++) {
                const int32_t held = here >> i & 1 ? held_end - (t0 + i * 16) : 0;
                if (held >= 16) continue;
                for (uint32_t k = lane; k < 16 * G; k += 32) {
                    const int32_t t = (int32_t)(k % (8 * G) / G) * 2;
                    uint32_t *w = reinterpret_cast<uint32_t *>(buf + i * L::BYTES + L::VS) + k;  // V scales, then V minima
                    *w &= t + 1 < held ? 0xffffffffu : t < held ? 0xffffu : 0u;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into this stage
            __syncwarp();
        }
        float top[2];
        bool behind = false;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            top[r] = fmaxf(s[0][r], s[0][2 + r]);
#pragma unroll
            for (int i = 1; i < TILES; i++) top[r] = fmaxf(top[r], fmaxf(s[i][r], s[i][2 + r]));
            behind |= (top[r] - m[r]) * cs[r] > LAG;
        }
        if (__any_sync(~0u, behind)) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], off));
                const float mm = fmaxf(m[r], top[r]), f = m[r] == mm ? 1.0f : ex2((m[r] - mm) * cs[r]);
                m[r] = mm;
#pragma unroll
                for (int i = 0; i < 2 * G; i++) o[i][r] *= f, o[i][2 + r] *= f;
                om[r] *= f, om[2 + r] *= f;
                l[r] *= f;
                nm[r] = mm == -INFINITY ? 0.0f : -mm;
            }
        }

        // a V scale larger than any before: the group's sums move to a new power of two
        if constexpr (Q32) {
            constexpr int N = TILES * (G == 8 ? 2 : 1);  // the 8 G words of a tile's scales, lane l's of group l % G
            uint32_t vw[N], wmax = vlim2;
#pragma unroll
            for (int k = 0; k < N; k++) {
                vw[k] = *reinterpret_cast<const uint32_t *>(buf + (k % TILES) * L::BYTES + L::VS + (lane + 32 * (k / TILES)) % (G * 8) * 4);
                wmax = __vmaxu2(wmax, vw[k]);
            }
            if (__any_sync(~0u, wmax != vlim2)) {
                const float2 v = unpack_h2(wmax);  // at least the limit, which is below 2^(V_TOP - kexp)
                float vmax = fmaxf(v.x, v.y);
#pragma unroll
                for (int off = G; off < 32; off <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(~0u, vmax, off));
                // 2^kexp times the largest scale is below 2^V_TOP (kexp at most 15, f16's largest power of two)
                const int k = min(kexp, V_TOP - 1 - ((int)(__float_as_uint(vmax) >> 23) - 127));
                vmax = __uint_as_float((uint32_t)(127 + k - kexp) << 23);
                kexp = k;
                vlim2 = (uint32_t)((15 + V_TOP - k) << 10) * 0x10001u - 0x10001u;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const float f = __shfl_sync(~0u, vmax, g);
                    const int kg = __shfl_sync(~0u, kexp, g);
                    kmul[g] = (uint32_t)(15 + kg) << 10 | (uint32_t)(15 + kg) << 26;
#pragma unroll
                    for (int k2 = 0; k2 < 4; k2++) o[2 * g][k2] *= f, o[2 * g + 1][k2] *= f;
                }
            }
        }

        // values
        float ls[2];  // the step's weights: one rounding of the long sums a step
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const uint8_t *tile = buf + i * L::BYTES;
            // the weights, and as f16 rounding and rest, turned so that a lane has positions 2 quad + (0, 1) + 8 j of row gid
            uint32_t ph[2], pl[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                // the difference to the reference first: exact near the maximum, so that no weight passes its bound however
                // large the scores
                const float p0 = ex2(fmaf(s[i][2 * j] + nm[0], cs[0], P_SHIFT)), p1 = ex2(fmaf(s[i][2 * j + 1] + nm[1], cs[1], P_SHIFT));
                ls[0] = i + j ? ls[0] + p0 : p0, ls[1] = i + j ? ls[1] + p1 : p1;
                ph[j] = pack_h2(p0, p1);
                if constexpr (REST) {
                    const float2 h = unpack_h2(ph[j]);
                    pl[j] = transpose8(pack_h2(p0 - h.x, p1 - h.y));
                }
                ph[j] = transpose8(ph[j]);
            }
            uint32_t vs[2][G], vm[2][G], v[2][G];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                lds_words<G>(vs[j], tile + L::VS + (4 * j + quad) * (G * 4));
                if constexpr (!Q32) lds_words<G>(vm[j], tile + L::VM + (4 * j + quad) * (G * 4));
                lds_codes<G, 8>(v[j], tile + L::VC + (4 * j + quad) * L::VROW, gid);
            }
            if constexpr (Q32) {
                // row gid of this product is half the middle m + 8 s of group gid % G, row 8 + gid what its f16 rounding left
                uint32_t mid[2], rest[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t at = ((4 * j + quad) * G + gid % G) * 4;
                    const uint32_t x = mul_h2(*reinterpret_cast<const uint32_t *>(tile + L::VS + at), 0x44004400u);  // 4 s
                    const uint32_t y = mul_h2(*reinterpret_cast<const uint32_t *>(tile + L::VM + at), 0x38003800u);  // m / 2
                    mid[j] = add_h2(x, y);
                    const uint32_t yy = sub_h2(mid[j], x);
                    rest[j] = add_h2(sub_h2(x, sub_h2(mid[j], yy)), sub_h2(y, yy));  // exactly x + y - mid
                }
                float d[4];
                mma16_first(d, mid[0], rest[0], mid[1], rest[1], ph[0], ph[1]);
                mma16(d, mid[0], rest[0], mid[1], rest[1], pl[0], pl[1]);
                add4(om, d);
            }
#pragma unroll
            for (int g = 0; g < G; g++) {
                uint32_t c0[4], c1[4], bh[2], bl[2];
                if constexpr (Q32) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        // (ph + pl) sc as the f16 rounding of ph sc and the rest
                        const uint32_t sc = mul_h2(vs[j][g], kmul[g]);
                        bh[j] = mul_h2(ph[j], sc);
                        bl[j] = fma_h2(pl[j], sc, fms_h2(ph[j], sc, bh[j]));
                    }
                    codes.get<8>(v[0][g], c0);
                    codes.get<8>(v[1][g], c1);
                } else {
                    // the values themselves
                    codes.get<0>(v[0][g], c0);
                    codes.get<0>(v[1][g], c1);
#pragma unroll
                    for (int k = 0; k < 4; k++) c0[k] = fma_h2(c0[k], vs[0][g], vm[0][g]), c1[k] = fma_h2(c1[k], vs[1][g], vm[1][g]);
                    bh[0] = ph[0], bh[1] = ph[1];
                    if constexpr (REST) bl[0] = pl[0], bl[1] = pl[1];
                }
                if constexpr (Q32) {
                    float d[4];
                    mma16_first(d, c0[0], c0[1], c1[0], c1[1], bh[0], bh[1]);
                    mma16(d, c0[0], c0[1], c1[0], c1[1], bl[0], bl[1]);
                    add4(o[2 * g], d);
                    mma16_first(d, c0[2], c0[3], c1[2], c1[3], bh[0], bh[1]);
                    mma16(d, c0[2], c0[3], c1[2], c1[3], bl[0], bl[1]);
                    add4(o[2 * g + 1], d);
                } else {
                    mma16(o[2 * g], c0[0], c0[1], c1[0], c1[1], bh[0], bh[1]);
                    if constexpr (REST) mma16(o[2 * g], c0[0], c0[1], c1[0], c1[1], bl[0], bl[1]);
                    mma16(o[2 * g + 1], c0[2], c0[3], c1[2], c1[3], bh[0], bh[1]);
                    if constexpr (REST) mma16(o[2 * g + 1], c0[2], c0[3], c1[2], c1[3], bl[0], bl[1]);
                }
            }
        }

        l[0] += ls[0], l[1] += ls[1];

        // the stage is read: it may be written again
        __syncwarp();
        if (lane == 0) mbar_arrive(&free_bar[stage]);
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
            const Seg &seg = segs[c_seg];
            const bool begins = seg.begin >= w0, ends = seg.begin + seg.steps <= w0 + n;
            // a part that began before this warp (at most one) and one that goes on after it (at most one) are left for the joins
            float *part = idx + 1 == n ? reinterpret_cast<float *>(ring) : parts + (uint64_t)(2 * MAX_CTAS + blockIdx.x * WARPS + warp) * PART;
            if (lane == 0 && !(begins && ends)) {
                seg_begin[2 * warp + begins] = seg.begin;
                part_seg[2 * warp + begins] = seg;
                part_at[2 * warp + begins] = part;
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t tr = 2 * quad + i;
                if (!(begins && ends)) {
#pragma unroll
                    for (int g = 0; g < G; g++)
                        *reinterpret_cast<float4 *>(part + tr * D + g * 32 + gid * 4) = make_float4(r[g][i][0], r[g][i][1], r[g][i][2], r[g][i][3]);
                    if (gid == 0) part[ROWS * D + tr] = m[i] * cs[i], part[ROWS * D + ROWS + tr] = l[i];
                    continue;
                }
                const uint32_t row = seg.tile * ROWS + tr, tok = row / a.group, hq = seg.head * a.group + row % a.group;
                if (tok >= (uint32_t)seg.r.nq) continue;
                const uint64_t t = (uint64_t)seg.r.tok0 + tok;
                T *out = (T *)a.out + t * a.o_tok + hq * a.o_head + gid * 4;
                const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
#pragma unroll
                for (int g = 0; g < G; g++) put4(out + g * 32, r[g][i][0] * inv, r[g][i][1] * inv, r[g][i][2] * inv, r[g][i][3] * inv, a.vec_out);
                if (a.lse && gid == 0) a.lse[t * a.n_heads + hq] = lse_of(m[i] * cs[i], l[i]);
            }
            if (++c_seg == C::SEGS) c_seg = 0;
        }
    }
    if (dead) {  // copies still in flight must not land in memory that is used for something else
        for (int s = 0; s < STAGES; s++) mbar_wait_bounded(&bar[s], s < (int)stage ? phase ^ 1 : phase, WAIT_LIMIT_NS / 20);
    }
    __syncthreads();

    // ---- joining the CTA's partial results: a warp per (segment, row), a lane per part for the weights ----
    constexpr uint32_t V = D / 32;
    // The row's values in a lane: V of them, in twos (D = 64) or fours, 32 lanes apart.
    constexpr uint32_t W = V < 4 ? V : 4;
    auto at_of = [&](uint32_t k) { return k / W * (W * 32) + lane * W + k % W; };
    auto get_row = [&](float (&x)[V], const float *p) {
        if constexpr (W == 2) {
            const float2 y = *reinterpret_cast<const float2 *>(p + lane * 2);
            x[0] = y.x, x[1] = y.y;
        } else {
#pragma unroll
            for (int k = 0; k < (int)V; k += 4) {
                const float4 y = *reinterpret_cast<const float4 *>(p + k * 32 + lane * 4);
                x[k] = y.x, x[k + 1] = y.y, x[k + 2] = y.z, x[k + 3] = y.w;
            }
        }
    };
    auto warp_max = [](float v) {
#pragma unroll
        for (int off = 16; off; off >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, off));
        return v;
    };
    auto warp_sum = [](float v) {
#pragma unroll
        for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(~0u, v, off);
        return v;
    };
    const uint32_t mine = seg_begin[lane];  // the parts, in order; a segment's are neighbours
    const uint32_t valid = __ballot_sync(~0u, mine != NONE), before = valid & ((1u << lane) - 1);
    if (!valid) return;
    const uint32_t prev = __shfl_sync(~0u, mine, before ? 31 - __clz(before) : 0);
    const uint32_t leads = __ballot_sync(~0u, mine != NONE && (!before || prev != mine));
    // the segments that other CTAs have parts of too: the one that began before this CTA, the one that goes on after it
    const Seg &edge0 = part_seg[__ffs(valid) - 1], &edge1 = part_seg[31 - __clz(valid)];
    const bool has0 = edge0.begin < c0, has1 = edge1.begin >= c0 && edge1.begin + edge1.steps > c1;
    // First the parts in this CTA, segment by segment; then, in the CTA that comes last to a segment, those of all CTAs.
#pragma unroll 1
    for (uint32_t pass = 0; pass < 2; pass++) {
        if (pass) {
            if (!has0 && !has1) return;
            __threadfence();
            __syncthreads();
            if (tid < 2) {
                flag_s[tid] = 0;
                if (tid ? has1 : has0) {
                    const Seg &sg_ = tid ? edge1 : edge0;
                    const uint32_t cb = sg_.begin / cta_chunk, ce = (sg_.begin + sg_.steps - 1) / cta_chunk;
                    const uint32_t arrived = atomicAdd(&counters[cb], 1u);
                    flag_s[tid] = arrived == ce - cb;
                    if (arrived == ce - cb) counters[cb] = 0;  // nobody else comes: ready for the next call
                }
            }
            __syncthreads();
            __threadfence();
        }
        const uint32_t units = pass ? 2 * ROWS : __popc(leads) * ROWS;
#pragma unroll 1
        for (uint32_t u = warp; u < units; u += WARPS + 1) {
            const uint32_t row = u % ROWS;
            uint32_t at = 0, count, cb = 0;  // pass 0: the first part's slot; its first CTA
            const Seg *of;
            if (pass == 0) {
                uint32_t lead = leads;
                for (uint32_t k = u / ROWS; k; k--) lead &= lead - 1;
                const uint32_t rest = lead & (lead - 1), these = valid & (rest ? (rest & (0u - rest)) - 1 : ~0u) & ~((lead & (0u - lead)) - 1);
                at = __ffs(lead) - 1;
                of = part_seg + at;
                count = __popc(these);  // the first warp's slot, then the even slots of the warps after it
            } else {
                if (!flag_s[u / ROWS]) continue;
                of = u / ROWS ? &edge1 : &edge0;
                cb = of->begin / cta_chunk;
                count = (of->begin + of->steps - 1) / cta_chunk - cb + 1;
            }
            auto part = [&](uint32_t i) -> const float * {
                return pass ? parts + (uint64_t)((cb + i) * 2 + (i ? 0 : 1)) * PART : part_at[i ? (at & ~1u) + 2 * i : at];
            };
            // 32 parts at a time: a lane per part for maximum and sum, then their values, several loads in flight
            float mm = -INFINITY, ll = 0.0f, acc[V] = {};
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < count; i0 += 32) {
                const bool in = i0 + lane < count;
                const float *p = part(in ? i0 + lane : 0) + row * D;
                const float mi = in ? p[ROWS * D - row * D + row] : -INFINITY, li = p[ROWS * D + ROWS - row * D + row];
                const float top = fmaxf(mm, warp_max(mi)), f = mm == top ? 1.0f : ex2(mm - top), w = !in ? 0.0f : mi == top ? 1.0f : ex2(mi - top);
                mm = top;
                ll = fmaf(w, li, ll * f);
#pragma unroll
                for (int v = 0; v < (int)V; v++) acc[v] *= f;
                constexpr int N = V == 8 ? 4 : 8;
                const uint32_t m = min(32u, count - i0);
                for (uint32_t i = 0; i < m; i += N) {
                    float x[N][V], wq[N];
#pragma unroll
                    for (int k = 0; k < N; k++) {
                        const uint32_t src = min(i + k, m - 1);
                        wq[k] = i + k < m ? __shfl_sync(~0u, w, src) : 0.0f;
                        get_row(x[k], part(i0 + src) + row * D);
                    }
#pragma unroll
                    for (int k = 0; k < N; k++)
#pragma unroll
                        for (int v = 0; v < (int)V; v++) acc[v] = fmaf(wq[k], x[k][v], acc[v]);
                }
            }
            ll = warp_sum(ll);
            const Seg &sg_ = *of;
            if (pass == 0 && (sg_.begin < c0 || sg_.begin + sg_.steps > c1)) {
                float *dst = parts + (uint64_t)(blockIdx.x * 2 + (sg_.begin < c0 ? 0 : 1)) * PART;
#pragma unroll
                for (int k = 0; k < (int)V; k++) dst[row * D + at_of(k)] = acc[k];
                if (lane == 0) dst[ROWS * D + row] = mm, dst[ROWS * D + ROWS + row] = ll;
                continue;
            }
            const uint32_t rr = sg_.tile * ROWS + row, tok = rr / a.group, hq = sg_.head * a.group + rr % a.group;
            if (tok >= (uint32_t)sg_.r.nq) continue;
            const uint64_t t = (uint64_t)sg_.r.tok0 + tok;
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
            T *out = (T *)a.out + t * a.o_tok + hq * a.o_head;
#pragma unroll
            for (int k = 0; k < (int)V; k++) out[at_of(k)] = Act<T>::put(acc[k] * inv);
            if (a.lse && lane == 0) a.lse[t * a.n_heads + hq] = lse_of(mm, ll);
        }
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
        if ((*err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<T, D>::SMEM)) != cudaSuccess) return SG_ERR_CUDA;
        ready[dev & 63] = true;
    }
    const uint32_t grid = (uint32_t)sms < MAX_CTAS ? (uint32_t)sms : MAX_CTAS, all = a0.c.heads;
    // MAX_REQ requests a launch, and as many heads as keep the number of steps below 2^32
    const uint64_t rows = (uint64_t)a0.n_tok * a0.group / ROWS + a0.n_req, steps = (((uint64_t)a0.width << a0.c.page_shift) + Cfg<T, D>::STEP - 1) / Cfg<T, D>::STEP + 1;
    const uint64_t heads = (1ull << 31) / (rows ? rows * steps : 1);  // (no requests and a few tokens of none: no rows)
    if (heads == 0) return SG_ERR_SHAPE;
    for (uint32_t r0 = 0; r0 == 0 || r0 < a0.n_req; r0 += MAX_REQ)
        for (uint32_t h0 = 0; h0 < all; h0 += (uint32_t)(heads < all ? heads : all)) {
            Kv4AttnArgs a = a0;
            a.n_req = a0.n_req - r0 < MAX_REQ ? a0.n_req - r0 : MAX_REQ;
            if (r0) a.cu += r0, a.seq += r0, a.tables += (uint64_t)r0 * a.ld_tables;
            a.first = r0 == 0, a.last = r0 + a.n_req == a0.n_req;
            a.head0 = h0;
            a.n_kv = (uint32_t)(all - h0 < heads ? all - h0 : heads);
            fn<<<grid, Cfg<T, D>::THREADS, Cfg<T, D>::SMEM, s>>>(a);
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
    if (kv4_prefill_pays(a, type, d, sms)) {
        *err = kv4_prefill_launch(a, type, d, s);
        return *err == cudaSuccess ? SG_OK : SG_ERR_CUDA;
    }
    return type == SG_F32 ? pick<float>(a, d, sms, s, err) : type == SG_F16 ? pick<__half>(a, d, sms, s, err) : pick<__nv_bfloat16>(a, d, sms, s, err);
}

}  // namespace sg
