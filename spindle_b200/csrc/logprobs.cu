// logprobs.cu — log probabilities of given tokens with entropy, rank and the
// likeliest alternatives, in one pass over the logits.
//
//   m = max x, z = sum e^(x - m), logprob = x_tok - m - ln z,
//   entropy = ln z - sum (x - m) e^(x - m) / z,
//   rank = how many tokens come before the given one when sorted by falling
//   logit, equal ones by rising index; the alternatives are the first of that order.
//
// A row belongs to a cluster of CTAs (one where the rows alone fill the device),
// each with a stretch of it.  A thread reads 64 bytes at a time, takes their
// maximum, and adds to its running m, z and sum of (x - m) e^(x - m); what bounds
// it is reading the row.  The alternatives cost the pass nothing but keeping the
// maximum of each thread's UNITS stretches: with t the top-th largest of the maxima
// of 128 groups of four threads, every alternative is at least t (each of `top`
// groups has one that is), and only about top elements are; the few stretches that
// reach t are read again and their elements sorted by counting.  Where that
// collects too many (a row of equal logits, say) or a NaN is about, the exact
// top-th key comes from four passes of 8 bits each, and ties are taken in index
// order.  That is where rows come whose mask is a finite number and leaves fewer tokens
// than alternatives: 45 us against 13 (one row of 151936 in f32, 20 alternatives of 8
// allowed tokens), 99 against 17 (65 rows).
//
// 2048 x 151935 bf16 with one alternative: 167 us, 3.7 TB/s, 57 % of the measured copy rate; 65 x 151936 f32 with 20:
// 22 us, 1.8 TB/s; one row 10 us.  Many rows are bound by issuing instructions (about 10 a value: exponential, two
// sums, maximum, rank), one row by the latency of its few dependent steps.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "logprobs.cuh"

namespace sg {

namespace cg = cooperative_groups;

namespace {

constexpr uint32_t GROUPS = 128;  // of a CTA's threads, by their maxima
constexpr uint32_t LOADS = 4;    // 16-byte loads of a thread in flight
constexpr uint32_t UNITS = 8;    // stretches of a thread whose maxima are kept; one more for the row's ragged ends
constexpr uint32_t CAP = 1536;   // candidates that are sorted by counting
constexpr float LAG = 8.0f;
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;

template <typename T>
struct El;
template <>
struct El<float> {
    static constexpr uint32_t N = 4, NEG = 0xFF800000u;  // values of 16 bytes; minus infinities
    static __device__ __forceinline__ float2 two(const uint32_t *r, int i) { return make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])); }
    static __device__ __forceinline__ float get(float v) { return v; }
};
template <>
struct El<__half> {
    static constexpr uint32_t N = 8, NEG = 0xFC00FC00u;
    static __device__ __forceinline__ float2 two(const uint32_t *r, int i) { return __half22float2(reinterpret_cast<const __half2 *>(r)[i]); }
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half inf() { return __ushort_as_half(0x7C00); }
};
template <>
struct El<__nv_bfloat16> {
    static constexpr uint32_t N = 8, NEG = 0xFF80FF80u;
    static __device__ __forceinline__ float2 two(const uint32_t *r, int i) { return make_float2(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xFFFF0000u)); }
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 inf() { return __ushort_as_bfloat16(0x7F80); }
};

// The larger one, NaN if either is.
__device__ __forceinline__ float max_nan(float x, float y) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(x), "f"(y));
    return d;
}
// Of two pairs of 16-bit values: 1 where x > y, or x >= y, else 0; their sums.
template <typename T>
__device__ __forceinline__ uint32_t more2(uint32_t x, uint32_t y, bool equal_too) {
    uint32_t d;
    if constexpr (std::is_same<T, __half>::value) {
        if (equal_too) asm("set.ge.f16x2.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
        else asm("set.gt.f16x2.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
    } else {
        if (equal_too) asm("set.ge.bf16x2.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
        else asm("set.gt.bf16x2.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
    }
    return d;
}
template <typename T>
__device__ __forceinline__ uint32_t add2_16(uint32_t x, uint32_t y) {
    uint32_t d;
    if constexpr (std::is_same<T, __half>::value) asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
    else asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
    return d;
}

// The largest of a thread's values, NaN if one is.
template <typename T, int W>
__device__ __forceinline__ float max_of(const uint32_t (&r)[W]) {
    if constexpr (sizeof(T) == 4) {
        float m = __uint_as_float(r[0]);
#pragma unroll
        for (int i = 1; i < W; i++) m = max_nan(m, __uint_as_float(r[i]));
        return m;
    } else {
        uint32_t m = r[0];
#pragma unroll
        for (int i = 1; i < W; i++) {
            if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(r[i]));
            else asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(r[i]));
        }
        const float2 f = El<T>::two(&m, 0);
        return max_nan(f.x, f.y);
    }
}

// The smallest of a thread's 16-bit values (none of them a NaN).
template <typename T, int W>
__device__ __forceinline__ float least_of(const uint32_t (&r)[W]) {
    uint32_t m = r[0];
#pragma unroll
    for (int i = 1; i < W; i++) {
        if constexpr (std::is_same<T, __half>::value) asm("min.f16x2 %0, %0, %1;" : "+r"(m) : "r"(r[i]));
        else asm("min.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(r[i]));
    }
    const float2 f = El<T>::two(&m, 0);
    return fminf(f.x, f.y);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two f32 operations in one instruction.
__device__ __forceinline__ uint64_t two_f32(float x, float y) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ float2 two_of(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// Order of falling logits, equal ones by rising index, as one number (larger
// comes first).  NaN counts as larger than everything; the zeros are equal.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x == x ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0xfffffffeu;
}
constexpr uint32_t ORDER_NEG_INF = 0x007fffffu;
__device__ __forceinline__ float value_of(uint32_t o) {
    return o == 0xfffffffeu ? NAN : __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)order_of(x) << 32 | (uint32_t)~i; }

// A reference near the running maximum (or minus infinity), sum of 2^t and sum of t 2^t over t = (x - m) log2 e.
struct Sum {
    float m, z, zt;
};

// A sum that has nothing yet changes nothing, whatever its maximum.
__device__ __forceinline__ Sum join(Sum a, Sum b) {
    if (b.m > a.m) {
        const Sum t = a;
        a = b;
        b = t;
    }
    if (b.z == 0.0f) return a;
    const float d = b.m == a.m ? 0.0f : (b.m - a.m) * LOG2E, w = ex2(d);
    a.z = fmaf(b.z, w, a.z);
    a.zt += w == 0.0f ? 0.0f : (b.zt + d * b.z) * w;
    return a;
}

// The sums of N neighbouring lanes together.
template <int N>
__device__ __forceinline__ Sum join_lanes(Sum a) {
    float m = a.m;
#pragma unroll
    for (int o = 1; o < N; o <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const float d = a.m == m ? 0.0f : (a.m - m) * LOG2E, w = ex2(d);
    float z = a.z == 0.0f ? 0.0f : a.z * w, zt = a.z == 0.0f || w == 0.0f ? 0.0f : (a.zt + d * a.z) * w;
#pragma unroll
    for (int o = 1; o < N; o <<= 1) z += __shfl_xor_sync(~0u, z, o), zt += __shfl_xor_sync(~0u, zt, o);
    return {m, z, zt};
}

template <uint32_t THREADS>
struct Shared {
    static constexpr uint32_t WARPS = THREADS / 32;
    Sum sum[WARPS], all[8];
    uint32_t ahead[WARPS], all_ahead[8];
    uint32_t gmax[GROUPS];
    uint32_t count, threshold;
    uint32_t warp_count[WARPS];
    union {
        uint64_t cand[CAP];
        uint32_t hist[256];
    };
    uint64_t top[8 * LP_TOP_MAX];  // the CTAs' alternatives, in the first CTA
    float unit[UNITS + 1][THREADS];
};

// A row, or a CTA's part of it: `head` values up to the first 16-byte boundary, whole 16-byte words (this CTA's are
// v0..v1), the rest.
template <typename T, uint32_t THREADS>
struct Row {
    const T *x;
    uint32_t head, tail, v0, v1, turns;
    __device__ __forceinline__ Row(const LogprobsArgs &a, uint32_t row, uint32_t part, uint32_t parts) {
        constexpr uint32_t N = El<T>::N;
        x = (const T *)a.logits + (uint64_t)row * a.ld;
        head = min(a.vocab, (uint32_t)((16 - ((uintptr_t)x & 15)) & 15) / (uint32_t)sizeof(T));
        const uint32_t words = (a.vocab - head) / N;
        tail = a.vocab - head - words * N;
        v0 = (uint32_t)((uint64_t)words * part / parts), v1 = (uint32_t)((uint64_t)words * (part + 1) / parts);
        turns = (v1 - v0 + LOADS * THREADS - 1) / (LOADS * THREADS);
    }
    __device__ __forceinline__ const uint4 *words() const { return reinterpret_cast<const uint4 *>(x + head); }
};

template <typename T, uint32_t THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprobs_kernel(const LogprobsArgs a) {
    using Shared = Shared<THREADS>;
    constexpr uint32_t N = El<T>::N, WARPS = THREADS / 32, PER_GROUP = THREADS / GROUPS;
    extern __shared__ __align__(16) uint8_t smem[];
    Shared &s = *reinterpret_cast<Shared *>(smem);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t row0 = blockIdx.x / parts, rows_apart = gridDim.x / parts;

    if (parts > 1) cluster.sync();  // another CTA's memory may be written from here on

    for (uint32_t row = row0; row < a.rows; row += rows_apart) {
    const Row<T, THREADS> R(a, row, part, parts);
    const T *x = R.x;
    const uint4 *xv = R.words();
    const uint32_t head = R.head, tail = R.tail, v0 = R.v0, v1 = R.v1, turns = R.turns, per_unit = (turns + UNITS - 1) / UNITS;
    const int32_t tok = a.tokens ? a.tokens[row] : -1;
    const bool given = tok >= 0 && (uint32_t)tok < a.vocab;
    const float xt = given ? El<T>::get(x[tok]) : INFINITY;
    uint32_t xt2 = 0;  // twice, in the logits' type
    if constexpr (sizeof(T) == 2) {
        const T v = given ? x[tok] : El<T>::inf();
        xt2 = (uint32_t)*reinterpret_cast<const uint16_t *>(&v) * 0x10001u;
    }
    const uint32_t begin = part == 0 ? 0 : head + v0 * N, end = part + 1 == parts ? a.vocab : head + v1 * N;  // this CTA's values

    Sum sum = {-INFINITY, 0.0f, 0.0f};
    uint64_t z2 = 0, zt2 = 0;  // the pair of sums at sum.m
    uint32_t ahead = 0;
    float tmax = -INFINITY, umax = -INFINITY;
    uint32_t unit = 0, in_unit = 0;
    // one load's worth: W words of a thread that start at element `at` (words LOADS * THREADS apart)
    auto add = [&](const uint32_t (&r)[LOADS * 4], uint32_t v) {
        const float m = max_of<T>(r);
        umax = fmaxf(umax, m);
        // the reference follows the maximum when that is LAG above it
        if (m > sum.m + LAG) {
            const float d = (sum.m - m) * LOG2E, w = ex2(d);
            const float2 z = two_of(z2), zt = two_of(zt2);
            // (where w is 0, d and d z may be minus infinity: the first sum, or one over a mask's large finite numbers)
            zt2 = two_f32(w == 0.0f ? 0.0f : (zt.x + d * z.x) * w, w == 0.0f ? 0.0f : (zt.y + d * z.y) * w);
            z2 = two_f32(z.x * w, z.y * w);
            sum.m = m;
        }
        const float ref = sum.m == -INFINITY ? 0.0f : -sum.m;
        const uint64_t nm = two_f32(ref, ref), l2 = two_f32(LOG2E, LOG2E);
        // t of masked values is held at -200, whose 2^t is 0 in f32, so that its product with t is 0 too
        auto terms = [&](bool masked) {
#pragma unroll
            for (int i = 0; i < (int)(LOADS * N / 2); i++) {
                const float2 f = El<T>::two(r, i);
                uint64_t t = mul2(add2(two_f32(f.x, f.y), nm), l2);
                float2 tt = two_of(t);
                if (masked) {
                    tt.x = fmaxf(tt.x, -200.0f), tt.y = fmaxf(tt.y, -200.0f);
                    t = two_f32(tt.x, tt.y);
                }
                const uint64_t e = two_f32(ex2(tt.x), ex2(tt.y));
                z2 = add2(z2, e);
                zt2 = fma2(e, t, zt2);
            }
        };
        if (m != m) z2 = two_f32(NAN, NAN);
        else if (m == -INFINITY) ;  // nothing to add
        else if (sizeof(T) == 4 || !(least_of<T>(r) - sum.m > -1e38f)) terms(true);  // (t inside f32's range)
        else terms(false);
        if (m >= xt) {
            // the values before the given token count when equal, those after it do not
            const uint32_t at0 = head + v * N, at1 = at0 + (LOADS - 1) * THREADS * N;
            if (v + (LOADS - 1) * THREADS < v1 && (at1 + N <= (uint32_t)tok || at0 > (uint32_t)tok)) {
                const bool equal_too = at0 < (uint32_t)tok;
                if constexpr (sizeof(T) == 4) {
                    if (equal_too) {
#pragma unroll
                        for (int i = 0; i < (int)(LOADS * 4); i++) ahead += __uint_as_float(r[i]) >= xt;
                    } else {
#pragma unroll
                        for (int i = 0; i < (int)(LOADS * 4); i++) ahead += __uint_as_float(r[i]) > xt;
                    }
                } else {
                    uint32_t n2 = 0;
                    if (equal_too) {
#pragma unroll
                        for (int i = 0; i < (int)(LOADS * 4); i++) n2 = add2_16<T>(n2, more2<T>(r[i], xt2, true));
                    } else {
#pragma unroll
                        for (int i = 0; i < (int)(LOADS * 4); i++) n2 = add2_16<T>(n2, more2<T>(r[i], xt2, false));
                    }
                    const float2 n = El<T>::two(&n2, 0);
                    ahead += (uint32_t)(n.x + n.y);
                }
            } else {
#pragma unroll
                for (int j = 0; j < (int)LOADS; j++) {
                    const uint32_t at = head + (v + j * THREADS) * N;
                    if (v + j * THREADS >= v1) continue;
#pragma unroll
                    for (int i = 0; i < (int)(N / 2); i++) {
                        const float2 f = El<T>::two(r + 4 * j, i);
                        ahead += f.x > xt || (f.x == xt && at + 2 * i < (uint32_t)tok);
                        ahead += f.y > xt || (f.y == xt && at + 2 * i + 1 < (uint32_t)tok);
                    }
                }
            }
        }
    };
    for (uint32_t turn = 0; turn < turns; turn++) {
        const uint32_t v = v0 + turn * LOADS * THREADS + tid;
        uint32_t r[LOADS * 4];
#pragma unroll
        for (int j = 0; j < (int)LOADS; j++) {
            const uint4 w = v + j * THREADS < v1 ? __ldg(xv + v + j * THREADS) : make_uint4(El<T>::NEG, El<T>::NEG, El<T>::NEG, El<T>::NEG);
            r[4 * j] = w.x, r[4 * j + 1] = w.y, r[4 * j + 2] = w.z, r[4 * j + 3] = w.w;
        }
        add(r, v);
        if (++in_unit == per_unit || turn + 1 == turns) {
            s.unit[unit][tid] = umax;
            tmax = fmaxf(tmax, umax);
            umax = -INFINITY;
            unit++, in_unit = 0;
        }
    }
    const uint32_t units = unit;
    // the ragged ends, a value per thread: the head in the first CTA, the tail in the last
    const uint32_t n_head = part == 0 ? head : 0, n_edge = n_head + (part + 1 == parts ? tail : 0);
    const uint32_t edge = tid < n_head ? tid : a.vocab - tail + (tid - n_head);
    if (tid < n_edge) {
        const float f = El<T>::get(x[edge]);
        const float2 z = two_of(z2), zt = two_of(zt2);
        const Sum one = {f, f == -INFINITY ? 0.0f : f - f + 1.0f, 0.0f};
        const Sum got = join(Sum{sum.m, z.x + z.y, zt.x + zt.y}, one);
        sum.m = got.m, z2 = two_f32(got.z, 0.0f), zt2 = two_f32(got.zt, 0.0f);
        ahead += f > xt || (f == xt && edge < (uint32_t)tok);
        umax = f;
        tmax = fmaxf(tmax, f);
    }
    s.unit[UNITS][tid] = umax;
    {
        const float2 z = two_of(z2), zt = two_of(zt2);
        sum.z = z.x + z.y, sum.zt = zt.x + zt.y;
    }

    // the CTA's sums
    sum = join_lanes<32>(sum);
    ahead = __reduce_add_sync(~0u, ahead);
    if (lane == 0) s.sum[warp] = sum, s.ahead[warp] = ahead;
    if (tid == 0) s.count = 0, s.threshold = 0;
    if (a.top) {
        float g = tmax;
#pragma unroll
        for (int o = 1; o < (int)PER_GROUP; o <<= 1) g = fmaxf(g, __shfl_xor_sync(~0u, g, o));
        if (tid % PER_GROUP == 0) s.gmax[tid / PER_GROUP] = order_of(g);
    }
    __syncthreads();
    sum = join_lanes<WARPS>(s.sum[lane % WARPS]);
    ahead = __reduce_add_sync(~0u, lane < WARPS ? s.ahead[lane] : 0u);
    const bool odd = sum.z != sum.z;  // a NaN, or infinities that cancel

    if (odd && given) {  // the comparisons above saw no NaN: count again by keys
        const uint64_t kt = key_of(xt, (uint32_t)tok);
        uint32_t n = 0;
        for (uint32_t i = begin + tid; i < end; i += THREADS) n += key_of(El<T>::get(x[i]), i) > kt;
        n = __reduce_add_sync(~0u, n);
        __syncthreads();
        if (lane == 0) s.ahead[warp] = n;
        __syncthreads();
        ahead = 0;
        for (uint32_t w = 0; w < WARPS; w++) ahead += s.ahead[w];
    }
    if (tid == 0) {
        Shared &first = *cluster.map_shared_rank(&s, 0);
        first.all[part] = sum;
        first.all_ahead[part] = ahead;
    }

    // ---- the alternatives in this CTA's stretch: at most `want`, into the first CTA's list ----
    const uint32_t k = a.top, want = min(k, end - begin);
    if (k) {
        uint64_t *list = cluster.map_shared_rank(&s.top[0], 0) + part * k;
        bool exact = odd;
        uint32_t n = 0;
        if (!odd) {
            // the top-th largest of the groups' maxima
            {
                const uint32_t mine = s.gmax[tid / PER_GROUP];
                uint32_t more = 0, same = 0;
#pragma unroll
                for (uint32_t g = 0; g < GROUPS; g += 4 * PER_GROUP) {  // the group's threads share the others
                    const uint4 o = *reinterpret_cast<const uint4 *>(&s.gmax[tid % PER_GROUP * 4 + g]);
                    more += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
                    same += (o.x == mine) + (o.y == mine) + (o.z == mine) + (o.w == mine);
                }
#pragma unroll
                for (int o = 1; o < (int)PER_GROUP; o <<= 1) more += __shfl_xor_sync(~0u, more, o), same += __shfl_xor_sync(~0u, same, o);
                if (more < k && more + same >= k) s.threshold = mine;
            }
            __syncthreads();
            // a threshold of minus infinity: all that is larger, and below as many of those that are not as can be needed
            const uint32_t t = s.threshold, least = t <= ORDER_NEG_INF ? ORDER_NEG_INF + 1 : t;
            const float floor_x = value_of(least);
            auto push = [&](float f, uint32_t i) {
                if (!(f >= floor_x)) return;
                const uint32_t c = atomicAdd(&s.count, 1u);
                if (c < CAP) s.cand[c] = key_of(f, i);
            };
            if (tmax >= floor_x) {
                for (uint32_t u = 0; u < units; u++) {
                    if (s.unit[u][tid] < floor_x) continue;
                    for (uint32_t turn = u * per_unit; turn < min(turns, (u + 1) * per_unit); turn++)
                        for (uint32_t j = 0; j < LOADS; j++) {
                            const uint32_t v = v0 + (turn * LOADS + j) * THREADS + tid;
                            if (v >= v1) break;
                            const uint4 w = xv[v];
                            const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int i = 0; i < (int)(N / 2); i++) {
                                const float2 f = El<T>::two(r, i);
                                push(f.x, head + v * N + 2 * i);
                                push(f.y, head + v * N + 2 * i + 1);
                            }
                        }
                }
                if (tid < n_edge) push(s.unit[UNITS][tid], edge);
            }
            __syncthreads();
            n = s.count;
            if (t <= ORDER_NEG_INF) {
                __syncthreads();  // every thread has read the count before one adds to it: all go the same way
                if (n < want) {
                    // of the first n + want values of the stretch at least want are minus infinities, or all of them are there
                    for (uint32_t i = begin + tid; i < min(end, begin + n + want); i += THREADS) {
                        const float f = El<T>::get(x[i]);
                        if (f != -INFINITY) continue;
                        const uint32_t c = atomicAdd(&s.count, 1u);
                        if (c < CAP) s.cand[c] = key_of(f, i);
                    }
                    __syncthreads();
                    n = s.count;
                }
            }
            exact = n > CAP;
        }
        if (exact) {
            // the want-th largest order, 8 bits at a time
            uint32_t prefix = 0, need = want;
            for (int shift = 24; shift >= 0; shift -= 8) {
                __syncthreads();
                for (uint32_t i = tid; i < 256; i += THREADS) s.hist[i] = 0;
                __syncthreads();
                for (uint32_t i = begin + tid; i < end; i += THREADS) {
                    const uint32_t o = order_of(El<T>::get(x[i]));
                    if (shift == 24 || (o >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s.hist[(o >> shift) & 255], 1u);
                }
                __syncthreads();
                if (tid == 0) {
                    uint32_t left = need;
                    int b = 255;
                    while (b > 0 && s.hist[b] < left) left -= s.hist[b--];
                    s.threshold = prefix | (uint32_t)b << shift;
                    s.count = left;
                }
                __syncthreads();
                prefix = s.threshold, need = s.count;
            }
            // the larger ones in any order; of the equal ones the first `need`
            __syncthreads();
            if (tid == 0) s.count = 0;
            __syncthreads();
            uint32_t taken = 0;
            for (uint32_t i0 = begin; i0 < end; i0 += THREADS) {
                const uint32_t i = i0 + tid;
                const float f = i < end ? El<T>::get(x[i]) : -INFINITY;
                const uint32_t o = order_of(f);
                if (i < end && o > prefix) s.cand[atomicAdd(&s.count, 1u)] = key_of(f, i);  // fewer than want
                if (taken >= need) continue;
                const uint32_t same = __ballot_sync(~0u, i < end && o == prefix);
                __syncthreads();
                if (lane == 0) s.warp_count[warp] = __popc(same);
                __syncthreads();
                uint32_t at = taken, all = 0;
                for (uint32_t w = 0; w < WARPS; w++) at += w < warp ? s.warp_count[w] : 0, all += s.warp_count[w];
                at += __popc(same & ((1u << lane) - 1));
                if (same >> lane & 1 && at < need) s.cand[atomicAdd(&s.count, 1u)] = key_of(f, i);
                taken += all;
            }
            __syncthreads();
            n = s.count;
        }
        // the best of the candidates, each at its place (any number of them is at least want)
        for (uint32_t c = tid; c < n; c += THREADS) {
            const uint64_t mine = s.cand[c];
            uint32_t before = 0;
            for (uint32_t j = 0; j < n; j++) before += s.cand[j] > mine;
            if (before < want) list[before] = mine;
        }
        if (tid >= want && tid < k) list[tid] = 0;
    }
    if (parts > 1) {
        cluster.sync();
        if (part) return;  // a cluster has one row
    } else {
        __syncthreads();
    }

    // ---- the row's results, in the first CTA ----
    sum = s.all[0], ahead = s.all_ahead[0];
    for (uint32_t p = 1; p < parts; p++) sum = join(sum, s.all[p]), ahead += s.all_ahead[p];
    const bool none = sum.m == -INFINITY && sum.z == 0.0f;          // a row whose mask leaves nothing
    const float lz = sum.m == INFINITY ? NAN : log2f(sum.z) * LN2;  // an infinite logit leaves no probabilities
    auto logprob_of = [&](float v) { return none ? -INFINITY : v - sum.m - lz; };
    if (tid == 0) {
        a.logprob[row] = given ? logprob_of(xt) : NAN;
        a.entropy[row] = none ? 0.0f : lz - sum.zt / sum.z * LN2;
        a.rank[row] = given ? (int32_t)ahead : -1;
    }
    for (uint32_t c = tid; c < parts * k; c += THREADS) {
        const uint64_t mine = s.top[c];
        uint32_t before = parts == 1 ? c : 0;
        if (parts > 1)
            for (uint32_t j = 0; j < parts * k; j++) before += s.top[j] > mine;
        if (mine && before < k) {
            a.top_ids[(uint64_t)row * k + before] = (int32_t)~(uint32_t)mine;
            a.top_logprobs[(uint64_t)row * k + before] = logprob_of(value_of((uint32_t)(mine >> 32)));
        }
    }
    __syncthreads();
    }
}

template <typename T, uint32_t THREADS>
cudaError_t launch_as(const LogprobsArgs &a, uint32_t parts, uint32_t grid, cudaStream_t s) {
    auto fn = logprobs_kernel<T, THREADS>;
    constexpr size_t smem = sizeof(Shared<THREADS>);
    static bool ready[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!ready[dev & 63]) {
        if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
        ready[dev & 63] = true;
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {parts, 1, 1};
    c.attrs = at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, fn, a);
}

template <typename T>
cudaError_t launch(const LogprobsArgs &a, int sms, cudaStream_t s) {
    // Many rows: four CTAs of 256 threads an SM, so that the steps at the end of a row, which wait for one another,
    // run beside the others' reading (2048 x 151935 bf16: 170 us against 195 with 512 threads, 1000 x 32000 f32: 49
    // against 59).  Fewer: CTAs of 512, two an SM (600 x 151936 f32: 108 against 122, 296: 49 against 70), and as many
    // of them a row as the device has room for, at most 8, while each has a turn of loads (one row: 10 us with 8, 23
    // with one; 65 rows: 22 against 38).
    if (a.rows >= (uint32_t)sms * 5) return launch_as<T, 256>(a, 1, a.rows < (uint32_t)sms * 4 ? a.rows : sms * 4, s);
    uint32_t parts = 1;
    while (parts < 8 && a.rows * parts <= (uint32_t)sms && a.vocab >= 2 * parts * 512 * El<T>::N) parts *= 2;
    return launch_as<T, 512>(a, parts, a.rows * parts, s);
}

}  // namespace

sg_status logprobs_launch(const LogprobsArgs &a, int32_t type, int sms, cudaStream_t s, cudaError_t *err) {
    *err = type == SG_F32 ? launch<float>(a, sms, s) : type == SG_F16 ? launch<__half>(a, sms, s) : launch<__nv_bfloat16>(a, sms, s);
    return *err == cudaSuccess ? SG_OK : SG_ERR_CUDA;
}

}  // namespace sg
