// moe_sort.cu — tokens sorted by expert and back: the choice of each token's experts from the
// router's logits, the stable sort of the (token, choice) pairs by expert, and the weighted sum
// of the experts' results.
//
// The sort is a counting sort: a CTA per stretch of tokens counts its experts, a second launch
// adds up the counts of the stretches before its own (all of them, for the places of the experts)
// and gives each pair its place by counting the bits of the pairs before it with the same expert.
// What bounds it: a step of a few tokens, the chain of dependent steps in one CTA; a prompt,
// the logits' bytes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx4.cuh"

namespace sg {

namespace {

constexpr uint32_t THREADS = 512, WARPS = THREADS / 32;

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A key that rises with the logit: 0 for minus infinity, NaN above everything; both zeros alike.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    if (b == 0xFF800000u) return 0;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k == 0xFFFFFFFFu ? 0x7FC00000u : k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The n_used likeliest experts of a token, by a warp: up to 32 * R experts.  Lane j < n_used returns the j-th (-1: none).
template <typename T, int R>
__device__ __forceinline__ int32_t choose(const MoeSortArgs &a, uint32_t t, uint32_t lane, float &weight) {
    const T *x = static_cast<const T *>(a.logits) + (uint64_t)t * a.ld;
    uint32_t key[R];
#pragma unroll
    for (int i = 0; i < R; i++) key[i] = lane + 32 * i < a.n_expert ? key_of(widen(x[lane + 32 * i])) : 0;
    float top = 0.0f, mine = 0.0f, all = 0.0f;
    int32_t id = -1;
    uint32_t found = 0;
    for (uint32_t j = 0; j < a.n_used; j++) {
        uint32_t best = key[0], at = 0;
#pragma unroll
        for (int i = 1; i < R; i++)
            if (key[i] > best) best = key[i], at = i;
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0) break;
        // equal ones: the lowest number
        const uint32_t e = __reduce_min_sync(0xffffffffu, best == most ? lane + 32 * at : 0xFFFFFFFFu);
        if (j == 0) {
            top = value_of(most);
            if (!a.norm) {
#pragma unroll
                for (int i = 0; i < R; i++)
                    if (key[i]) all += expf(value_of(key[i]) - top);
                all = warp_sum(all);
            }
        }
        if (lane == j) id = (int32_t)e, mine = expf(value_of(most) - top);
#pragma unroll
        for (int i = 0; i < R; i++)
            if (lane + 32 * i == e) key[i] = 0;
        found++;
    }
    // pruning, as the framework's one-token layer does it
    uint32_t keep = found;
    if (a.prune > 0.0f && found > 2) {
        const uint32_t least = found / 2 > 2 ? found / 2 : 2;
        if (a.prune >= 1.0f) {
            const uint32_t p = a.prune >= 1024.0f ? 1024u : (uint32_t)a.prune;
            keep = p < least ? least : p < found ? p : found;
        } else {
            const float target = warp_sum(mine) * (1.0f - a.prune);
            float sum = 0.0f;
            uint32_t n = 0;
            while (n < found && (n < least || sum < target)) sum += __shfl_sync(0xffffffffu, mine, n++);
            keep = n;
        }
    }
    if (lane >= keep) id = -1, mine = 0.0f;
    const float total = a.norm ? warp_sum(mine) : all;
    weight = id < 0 ? 0.0f : mine / total;
    return id;
}

struct Stretch {
    uint32_t t0, t1;
};
__device__ __forceinline__ Stretch stretch(const MoeSortArgs &a, uint32_t cta) {
    const uint32_t groups = (a.n_tok + MOE_SORT_TOKENS - 1) / MOE_SORT_TOKENS;
    const uint32_t g0 = (uint32_t)((uint64_t)groups * cta / a.ctas), g1 = (uint32_t)((uint64_t)groups * (cta + 1) / a.ctas);
    return {g0 * MOE_SORT_TOKENS, min(g1 * MOE_SORT_TOKENS, a.n_tok)};
}

// Inclusive sum over the CTA of one value a thread (sums: WARPS words).
__device__ __forceinline__ uint32_t cta_scan(uint32_t v, uint32_t *sums) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= (uint32_t)o) v += u;
    }
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    uint32_t w = lane < WARPS ? sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < (int)WARPS; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= (uint32_t)o) w += u;
    }
    const uint32_t before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
    __syncthreads();
    return v + (warp ? before : 0);
}

// Places of the pairs of this CTA's tokens.  at: the first place of each expert here, on entry its counts in the stretches
// before; total: the counts of all.  mask: zeroed, n_expert rows of n_used * 2 words.
__device__ __forceinline__ void place_pairs(const MoeSortArgs &a, uint32_t cta, uint32_t *at, const uint32_t *total, uint32_t *mask, uint32_t *sums) {
    const uint32_t tid = threadIdx.x, E = a.n_expert;
    // thread i has experts 2 i and 2 i + 1
    const uint32_t e0 = 2 * tid, c0 = e0 < E ? total[e0] : 0, c1 = e0 + 1 < E ? total[e0 + 1] : 0;
    const uint32_t upto = cta_scan(c0 + c1, sums);
    if (e0 < E) at[e0] += upto - c1 - c0;
    if (e0 + 1 < E) at[e0 + 1] += upto - c1;
    if (cta == 0) {
        if (e0 < E) a.first[e0] = (int32_t)(upto - c1 - c0);
        if (e0 + 1 < E) a.first[e0 + 1] = (int32_t)(upto - c1);
        if (tid == THREADS - 1) a.first[E] = (int32_t)upto;
#pragma unroll
        for (uint32_t k = 0; k < 3; k++) {
            const uint32_t r = (32u << k) - 1, n0 = (c0 + r) >> (5 + k), n1 = (c1 + r) >> (5 + k);
            const uint32_t u = cta_scan(n0 + n1, sums);
            int32_t *tiles = a.tiles + (uint64_t)k * (E + 1);
            if (e0 < E) tiles[e0] = (int32_t)(u - n1 - n0);
            if (e0 + 1 < E) tiles[e0 + 1] = (int32_t)(u - n1);
            if (tid == THREADS - 1) tiles[E] = (int32_t)u;
        }
    }
    if (tid == THREADS - 1) sums[WARPS] = upto;
    __syncthreads();
    const uint64_t pairs = (uint64_t)a.n_tok * a.n_used;
    for (uint64_t s = sums[WARPS] + (uint64_t)cta * THREADS + tid; s < pairs; s += (uint64_t)a.ctas * THREADS) a.order[s] = -1;
    const uint32_t words = MOE_SORT_TOKENS * a.n_used / 32;
    const Stretch st = stretch(a, cta);
    for (uint32_t t = st.t0; t < st.t1; t += MOE_SORT_TOKENS) {
        const uint32_t n = min(MOE_SORT_TOKENS, st.t1 - t) * a.n_used;  // pairs, at most 1024
        const uint64_t p0 = (uint64_t)t * a.n_used;
        int32_t e[2] = {-1, -1};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t p = tid + THREADS * i;
            if (p < n) e[i] = a.ids[p0 + p];
            if (e[i] >= 0) atomicOr(&mask[e[i] * words + p / 32], 1u << (p & 31));
        }
        __syncthreads();
        uint32_t rank[2] = {}, count[2] = {};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t p = tid + THREADS * i;
            if (e[i] >= 0) {
                const uint32_t *m = mask + e[i] * words;
                for (uint32_t w = 0; w < words; w++) {
                    const uint32_t b = m[w];
                    count[i] += __popc(b);
                    rank[i] += __popc(w < p / 32 ? b : w == p / 32 ? b & ((1u << (p & 31)) - 1) : 0);
                }
                const uint32_t s = at[e[i]] + rank[i];
                a.order[s] = (int32_t)(p0 + p);
                a.place[p0 + p] = (int32_t)s;
            } else if (p < n) a.place[p0 + p] = -1;
        }
        if (t + MOE_SORT_TOKENS < st.t1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (e[i] >= 0) {
                    if (rank[i] == 0) at[e[i]] += count[i];
                    mask[e[i] * words + (tid + THREADS * i) / 32] = 0;
                }
            __syncthreads();
        }
    }
}

__host__ __device__ constexpr uint32_t sort_smem(uint32_t experts, uint32_t used) {
    return (2 * experts + WARPS + 1 + experts * (MOE_SORT_TOKENS * used / 32)) * 4;
}

// Choices (or the given ones, those outside 0..n_expert - 1 as none) and the counts of this stretch; a single CTA goes on to the places.
template <typename T, int R>
__global__ void __launch_bounds__(THREADS) moe_choose_kernel(const __grid_constant__ MoeSortArgs a) {
    extern __shared__ uint32_t sm[];
    uint32_t *at = sm, *count = sm + a.n_expert, *sums = count + a.n_expert, *mask = sums + WARPS + 1;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t clear = a.ctas == 1 ? sort_smem(a.n_expert, a.n_used) / 4 : 2 * a.n_expert;
    for (uint32_t i = tid; i < clear; i += THREADS) sm[i] = 0;
    __syncthreads();
    const Stretch st = stretch(a, blockIdx.x);
    if (a.logits) {
        for (uint32_t t = st.t0 + warp; t < st.t1; t += WARPS) {
            float w;
            const int32_t id = choose<T, R>(a, t, lane, w);
            if (lane < a.n_used) {
                a.ids[(uint64_t)t * a.n_used + lane] = id;
                a.weights[(uint64_t)t * a.n_used + lane] = w;
                if (id >= 0) atomicAdd(&count[id], 1u);
            }
        }
    } else {
        const uint64_t p1 = (uint64_t)st.t1 * a.n_used;
        for (uint64_t p = (uint64_t)st.t0 * a.n_used + tid; p < p1; p += THREADS) {
            const int32_t id = a.ids[p];
            if (id >= 0 && (uint32_t)id < a.n_expert) atomicAdd(&count[id], 1u);
            else a.ids[p] = -1, a.weights[p] = 0.0f;
        }
    }
    __syncthreads();
    if (a.ctas == 1) place_pairs(a, 0, at, count, mask, sums);
    else
        for (uint32_t e = tid; e < a.n_expert; e += THREADS) a.counts[(uint64_t)blockIdx.x * a.n_expert + e] = (int32_t)count[e];
}

__global__ void __launch_bounds__(THREADS) moe_place_kernel(const __grid_constant__ MoeSortArgs a) {
    extern __shared__ uint32_t sm[];
    uint32_t *at = sm, *total = sm + a.n_expert, *sums = total + a.n_expert, *mask = sums + WARPS + 1;
    const uint32_t tid = threadIdx.x;
    for (uint32_t i = tid; i < sort_smem(a.n_expert, a.n_used) / 4; i += THREADS) sm[i] = 0;
    __syncthreads();
    // the stretches in as many shares as the threads allow, an expert a thread
    const uint32_t shares = max(1u, THREADS / a.n_expert), share = tid / a.n_expert;
    if (share < shares)
        for (uint32_t e = tid - share * a.n_expert; e < a.n_expert; e += THREADS) {
            uint32_t all = 0, before = 0;
#pragma unroll 8
            for (uint32_t c = share; c < a.ctas; c += shares) {
                const uint32_t n = (uint32_t)__ldg(a.counts + (uint64_t)c * a.n_expert + e);
                all += n;
                before += c < blockIdx.x ? n : 0;
            }
            atomicAdd(&total[e], all);
            atomicAdd(&at[e], before);
        }
    __syncthreads();
    place_pairs(a, blockIdx.x, at, total, mask, sums);
}

// out[t] = sum over j of weights[t, j] y[place[t, j]], in the order of j, in f32.  A thread has eight columns of a token and
// its loads of up to eight experts' rows in flight.  What bounds it: reading y.
template <typename T, typename O, bool VEC>
__global__ void __launch_bounds__(256) moe_combine_kernel(const __grid_constant__ MoeCombineArgs a) {
    const uint32_t per = (a.dim + 7) / 8;
    const uint64_t items = a.n_tok * per, step = (uint64_t)gridDim.x * 256;
    for (uint64_t it = (uint64_t)blockIdx.x * 256 + threadIdx.x; it < items; it += step) {
        const uint64_t t = it / per;
        const uint32_t col = (uint32_t)(it - t * per) * 8, n = min(8u, a.dim - col);
        float sum[8] = {};
        for (uint32_t j0 = 0; j0 < a.n_used; j0 += 8) {
            constexpr int N = 16 / sizeof(T);
            uint4 v[8][8 / N];
            float w[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                w[j] = 0.0f;
                int32_t p = -1;
                if (j0 + j < a.n_used) p = __ldg(a.place + t * a.n_used + j0 + j);
                const bool there = p >= 0 && (uint32_t)p < a.n_places;
                if (there) w[j] = __ldg(a.weights + t * a.n_used + j0 + j);
                const T *y = static_cast<const T *>(a.y) + (uint64_t)(there ? p : 0) * a.ldy + col;
                if constexpr (VEC) {
#pragma unroll
                    for (int i = 0; i < 8 / N; i++) v[j][i] = there ? __ldg(reinterpret_cast<const uint4 *>(y) + i) : make_uint4(0, 0, 0, 0);
                } else {
                    T *to = reinterpret_cast<T *>(v[j]);
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) to[i] = there && i < n ? y[i] : narrow<T>(0.0f);
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const T *y = reinterpret_cast<const T *>(v[j]);
#pragma unroll
                for (int i = 0; i < 8; i++) sum[i] = fmaf(w[j], widen(y[i]), sum[i]);
            }
        }
        O *o = static_cast<O *>(a.out) + t * a.ldo + col;
        if constexpr (VEC) {
            O r[8];
#pragma unroll
            for (int i = 0; i < 8; i++) r[i] = narrow<O>(sum[i]);
#pragma unroll
            for (uint32_t i = 0; i < 8 * sizeof(O) / 16; i++) reinterpret_cast<uint4 *>(o)[i] = reinterpret_cast<const uint4 *>(r)[i];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8; i++)
                if (i < n) o[i] = narrow<O>(sum[i]);
        }
    }
}

template <typename F>
cudaError_t big_smem(F fn, uint32_t bytes, bool (&ready)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || bytes <= 48 * 1024 || ready[dev & 63]) return e;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, sort_smem(MOE_SORT_MAX_EXPERTS, MOE_SORT_MAX_USED));
    if (e == cudaSuccess) ready[dev & 63] = true;
    return e;
}

template <typename T, int R>
cudaError_t choose_as(const MoeSortArgs &a, uint32_t smem, cudaStream_t s) {
    static bool ready[64];
    cudaError_t e = big_smem(moe_choose_kernel<T, R>, smem, ready);
    if (e != cudaSuccess) return e;
    moe_choose_kernel<T, R><<<a.ctas, THREADS, smem, s>>>(a);
    return cudaGetLastError();
}
template <typename T>
cudaError_t choose_of(const MoeSortArgs &a, uint32_t smem, cudaStream_t s) {
    return a.n_expert <= 128 ? choose_as<T, 4>(a, smem, s) : a.n_expert <= 256 ? choose_as<T, 8>(a, smem, s) : choose_as<T, 32>(a, smem, s);
}

template <typename T, typename O>
cudaError_t combine_as(const MoeCombineArgs &a, int sms, cudaStream_t s) {
    const uint64_t want = (a.n_tok * ((a.dim + 7) / 8) + 255) / 256;
    const uint32_t grid = (uint32_t)(want < (uint64_t)sms * 32 ? want : (uint64_t)sms * 32);
    if (a.vec) moe_combine_kernel<T, O, true><<<grid, 256, 0, s>>>(a);
    else moe_combine_kernel<T, O, false><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}
template <typename T>
cudaError_t combine_from(const MoeCombineArgs &a, int32_t o, int sms, cudaStream_t s) {
    return o == SG_F32 ? combine_as<T, float>(a, sms, s) : o == SG_F16 ? combine_as<T, __half>(a, sms, s) : combine_as<T, __nv_bfloat16>(a, sms, s);
}

}  // namespace

cudaError_t moe_sort_launch(const MoeSortArgs &a, int32_t type, cudaStream_t s) {
    const uint32_t smem = sort_smem(a.n_expert, a.n_used), first = a.ctas == 1 ? smem : 2 * a.n_expert * 4;
    cudaError_t e = type == SG_F32 ? choose_of<float>(a, first, s) : type == SG_F16 ? choose_of<__half>(a, first, s) : choose_of<__nv_bfloat16>(a, first, s);
    if (e != cudaSuccess || a.ctas == 1) return e;
    static bool ready[64];
    if ((e = big_smem(moe_place_kernel, smem, ready)) != cudaSuccess) return e;
    moe_place_kernel<<<a.ctas, THREADS, smem, s>>>(a);
    return cudaGetLastError();
}

cudaError_t moe_combine_launch(const MoeCombineArgs &a, int32_t type, int32_t out_type, int sms, cudaStream_t s) {
    return type == SG_F32 ? combine_from<float>(a, out_type, sms, s) : type == SG_F16 ? combine_from<__half>(a, out_type, sms, s) : combine_from<__nv_bfloat16>(a, out_type, sms, s);
}

}  // namespace sg
