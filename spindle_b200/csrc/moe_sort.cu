// moe_sort.cu — tokens sorted by expert and back: the choice of each token's experts from the
// router's logits, the stable sort of the (token, choice) pairs by expert, and the weighted sum
// of the experts' results.
//
// The sort is a counting sort: a CTA per stretch of tokens (one a warp) chooses and counts their
// experts, four of them together make a row of counts; a second launch adds up the rows before its
// own (all of them, for the places of the experts) and gives each pair its place by counting the
// bits of the pairs before it with the same expert.  A step of up to 64 tokens is one CTA's work.
// What bounds it: the chain of dependent steps, launches among them (16 tokens, 8 of 128: 5.6 us in a
// graph); of a prompt the choice's instructions, 670 a token (8191 tokens: 12 us and 6 for the places).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx4.cuh"
#include "tiled_block.cuh"

namespace cg = cooperative_groups;

namespace sg {
using namespace tiled;

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
    uint32_t mine_key = 0, top_key = 0, found = 0;
    int32_t id = -1;
    for (; found < a.n_used; found++) {
        uint32_t best = key[0], at = 0;
#pragma unroll
        for (int i = 1; i < R; i++)
            if (key[i] > best) best = key[i], at = i;
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0) break;
        // equal ones: the lowest number
        const uint32_t e = __reduce_min_sync(0xffffffffu, best == most ? lane + 32 * at : 0xFFFFFFFFu);
        if (found == 0) top_key = most;
        if (lane == found) id = (int32_t)e, mine_key = most;
#pragma unroll
        for (int i = 0; i < R; i++)
            if (lane + 32 * i == e) key[i] = 0;
    }
    const float top = found ? value_of(top_key) : 0.0f;
    float mine = id < 0 ? 0.0f : expf(value_of(mine_key) - top), all = 0.0f;
    if (!a.norm) {  // the sum over the others too
#pragma unroll
        for (int i = 0; i < R; i++)
            if (key[i]) all += expf(value_of(key[i]) - top);
        all = warp_sum(all + mine);
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

// Exclusive sums of f(e) over the experts, by one warp: put(e, sum before e), and the sum of all.
template <typename F, typename P>
__device__ __forceinline__ uint32_t warp_sums(uint32_t n, uint32_t lane, F f, P put) {
    uint32_t before = 0;
    for (uint32_t base = 0; base < n; base += 128) {  // four experts a lane
        uint32_t v[4], sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t e = base + 4 * lane + i;
            v[i] = e < n ? f(e) : 0;
            sum += v[i];
        }
        uint32_t upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += u;
        }
        uint32_t at = before + upto - sum;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t e = base + 4 * lane + i;
            if (e < n) put(e, at);
            at += v[i];
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return before;
}

// Shared memory: the first place of each expert for the pairs here, the counts of all, bits of a group's pairs, all pairs.
struct Tables {
    uint32_t *at, *total, *mask, *all;
};
// (a word more than the bits need: rows that begin in different banks)
__host__ __device__ constexpr uint32_t mask_words(uint32_t used) { return MOE_SORT_GROUP * used / 32 + 1; }
__host__ __device__ constexpr uint32_t sort_smem(uint32_t experts, uint32_t used) { return (2 * experts + experts * mask_words(used) + 1) * 4; }
__device__ __forceinline__ Tables tables(const MoeSortArgs &a, uint32_t *sm) { return {sm, sm + a.n_expert, sm + 2 * a.n_expert, sm + sort_smem(a.n_expert, a.n_used) / 4 - 1}; }

// Places of the pairs of the tokens t0 .. t1.  at: on entry the experts' counts in the tokens before; total: those of all.
// mask: zeroed.  first: this CTA writes what all have in common.
__device__ __forceinline__ void place_pairs(const MoeSortArgs &a, const Tables &m, uint32_t t0, uint32_t t1, bool first) {
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, E = a.n_expert;
    const uint32_t *total = m.total;
    if (warp == 0) {
        const uint32_t all = warp_sums(E, lane, [&](uint32_t e) { return total[e]; }, [&](uint32_t e, uint32_t v) {
            m.at[e] += v;
            if (first) a.first[e] = (int32_t)v;
        });
        if (lane == 0) *m.all = all;
        if (first && lane == 0) a.first[E] = (int32_t)all;
    } else if (warp < 5 && first) {  // tiles of 32, 128, 192 and 256 rows
        const uint32_t rows = warp == 1 ? 32 : warp == 2 ? 128 : warp == 3 ? 192 : 256;
        int32_t *tiles = a.tiles + (uint64_t)(warp - 1) * (E + 1);
        const uint32_t all = warp_sums(E, lane, [&](uint32_t e) { return (total[e] + rows - 1) / rows; }, [&](uint32_t e, uint32_t v) { tiles[e] = (int32_t)v; });
        if (lane == 0) tiles[E] = (int32_t)all;
    }
    __syncthreads();
    // places that no pair has
    const uint64_t pairs = (uint64_t)a.n_tok * a.n_used, ctas = (a.stretches + MOE_SORT_JOIN - 1) / MOE_SORT_JOIN;
    for (uint64_t s = *m.all + (uint64_t)blockIdx.x * THREADS + tid; s < pairs; s += ctas * THREADS) a.order[s] = -1;
    const uint32_t words = mask_words(a.n_used);
    for (uint32_t t = t0; t < t1; t += MOE_SORT_GROUP) {
        const uint32_t n = min(MOE_SORT_GROUP, t1 - t) * a.n_used;  // pairs, at most 1024
        const uint64_t p0 = (uint64_t)t * a.n_used;
        int32_t e[2] = {-1, -1};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t p = tid + THREADS * i;
            if (p < n) e[i] = a.ids[p0 + p];
            if (e[i] >= 0) atomicOr(&m.mask[e[i] * words + p / 32], 1u << (p & 31));
        }
        __syncthreads();
        uint32_t rank[2] = {}, count[2] = {};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t p = tid + THREADS * i;
            if (e[i] >= 0) {
                const uint32_t *w = m.mask + e[i] * words;
                for (uint32_t k = 0; k < words - 1; k++) {
                    const uint32_t b = w[k];
                    count[i] += __popc(b);
                    rank[i] += __popc(k < p / 32 ? b : k == p / 32 ? b & ((1u << (p & 31)) - 1) : 0);
                }
                const uint32_t s = m.at[e[i]] + rank[i];
                a.order[s] = (int32_t)(p0 + p);
                a.place[p0 + p] = (int32_t)s;
            } else if (p < n) a.place[p0 + p] = -1;
        }
        if (t + MOE_SORT_GROUP < t1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (e[i] >= 0) {
                    if (rank[i] == 0) m.at[e[i]] += count[i];
                    m.mask[e[i] * words + (tid + THREADS * i) / 32] = 0;
                }
            __syncthreads();
        }
    }
}

// Choices (or the given ones, those outside 0..n_expert - 1 as none) of a.stretch tokens, and their counts; a single CTA goes
// on to the places.
template <typename T, int R>
__global__ void __launch_bounds__(THREADS, R <= 8 ? 4 : 2) moe_choose_kernel(const __grid_constant__ MoeSortArgs a) {
    extern __shared__ uint32_t sm[];
    const Tables m = tables(a, sm);
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const bool alone = gridDim.x == 1;
    const uint32_t clear = alone ? sort_smem(a.n_expert, a.n_used) / 4 : 2 * a.n_expert;
    for (uint32_t i = tid; i < clear; i += THREADS) sm[i] = 0;
    __syncthreads();
    if (!alone) grid_launch_dependents();  // (the next launch clears its memory meanwhile)
    const uint32_t t0 = (uint32_t)min((uint64_t)blockIdx.x * a.stretch, (uint64_t)a.n_tok), t1 = min(t0 + a.stretch, a.n_tok);
    if (a.logits) {
        for (uint32_t t = t0 + warp; t < t1; t += WARPS) {
            float w;
            const int32_t id = choose<T, R>(a, t, lane, w);
            if (lane < a.n_used) {
                a.ids[(uint64_t)t * a.n_used + lane] = id;
                a.weights[(uint64_t)t * a.n_used + lane] = w;
                if (id >= 0) atomicAdd(&m.total[id], 1u);
            }
        }
    } else {
        const uint64_t p1 = (uint64_t)t1 * a.n_used;
        for (uint64_t p = (uint64_t)t0 * a.n_used + tid; p < p1; p += THREADS) {
            const int32_t id = a.ids[p];
            if (id >= 0 && (uint32_t)id < a.n_expert) atomicAdd(&m.total[id], 1u);
            else a.ids[p] = -1, a.weights[p] = 0.0f;
        }
    }
    if (alone) {
        __syncthreads();
        place_pairs(a, m, t0, t1, true);
        return;
    }
    // the counts of a cluster's stretches are one row
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const uint32_t rank = cluster.block_rank();
    for (uint32_t e = rank + MOE_SORT_JOIN * tid; e < a.counts_ld; e += MOE_SORT_JOIN * THREADS) {
        uint32_t n = 0;
        if (e < a.n_expert)
#pragma unroll
            for (uint32_t r = 0; r < MOE_SORT_JOIN; r++) n += *cluster.map_shared_rank(m.total + e, r);
        a.counts[(uint64_t)(blockIdx.x / MOE_SORT_JOIN) * a.counts_ld + e] = (int32_t)n;
    }
    cluster.sync();
}

// A CTA places the pairs of MOE_SORT_JOIN stretches, a row of counts: first the sums of all rows, and of those before its own.
__global__ void __launch_bounds__(THREADS) moe_place_kernel(const __grid_constant__ MoeSortArgs a) {
    extern __shared__ uint32_t sm[];
    const Tables m = tables(a, sm);
    const uint32_t tid = threadIdx.x;
    for (uint32_t i = tid; i < sort_smem(a.n_expert, a.n_used) / 4; i += THREADS) sm[i] = 0;
    __syncthreads();
    grid_dependency_wait();
    // four experts a thread, as many rows at once as the threads allow, eight loads in flight
    const uint32_t per = a.counts_ld / 4, shares = THREADS / per, share = tid / per, c = tid - share * per, rows = gridDim.x;
    if (share < shares) {
        uint32_t all[4] = {}, before[4] = {};
        for (uint32_t i0 = share; i0 < rows; i0 += 8 * shares) {
            int4 v[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; k++)
                v[k] = i0 + k * shares < rows ? *(reinterpret_cast<const int4 *>(a.counts + (uint64_t)(i0 + k * shares) * a.counts_ld) + c) : make_int4(0, 0, 0, 0);
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) {
                const bool b = i0 + k * shares < blockIdx.x;
                const uint32_t n[4] = {(uint32_t)v[k].x, (uint32_t)v[k].y, (uint32_t)v[k].z, (uint32_t)v[k].w};
#pragma unroll
                for (int j = 0; j < 4; j++) all[j] += n[j], before[j] += b ? n[j] : 0;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
            if (4 * c + k < a.n_expert) {
                if (all[k]) atomicAdd(&m.total[4 * c + k], all[k]);
                if (before[k]) atomicAdd(&m.at[4 * c + k], before[k]);
            }
    }
    __syncthreads();
    const uint64_t t0 = (uint64_t)blockIdx.x * MOE_SORT_JOIN * a.stretch, n = a.n_tok;
    place_pairs(a, m, (uint32_t)min(t0, n), (uint32_t)min(t0 + MOE_SORT_JOIN * a.stretch, n), blockIdx.x == 0);
}

// out[t] = sum over j of weights[t, j] y[place[t, j]], in the order of j, in f32.  A thread takes eight columns of a token, an
// item, with its loads of J experts' rows in flight.  With one slot or two, two items at a time (52592 rows of 1192 bf16, a row a
// token: eight slots, one item 125 us; one slot, one item 64, two 54, four 66; with four slots two are slower, 30.1 against 29.1).
// What bounds it: reading y (8191 x 8 rows of 2048 bf16: 50 us, 6.0 TB/s; x 4: 29 us, 5.8 TB/s; rows that do not begin on 16
// bytes, value by value: 98 us).
constexpr int combine_items(bool vec, int slots) { return vec && slots <= 2 ? 2 : 1; }

template <typename T, typename O, bool VEC, int J>
__global__ void __launch_bounds__(256) moe_combine_kernel(const __grid_constant__ MoeCombineArgs a) {
    constexpr int ITEMS = combine_items(VEC, J), N = 16 / sizeof(T);
    const uint32_t per = (a.dim + 7) / 8;
    const uint64_t items = a.n_tok * per, step = (uint64_t)gridDim.x * (256 * ITEMS);
    for (uint64_t first = (uint64_t)blockIdx.x * (256 * ITEMS) + threadIdx.x; first < items; first += step) {
        uint64_t t[ITEMS];
        uint32_t col[ITEMS], n[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const uint64_t it = first + i * 256;
            t[i] = it / per;
            col[i] = (uint32_t)(it - t[i] * per) * 8;
            n[i] = it < items ? min(8u, a.dim - col[i]) : 0;
        }
        float sum[ITEMS][8] = {};
        for (uint32_t j0 = 0; j0 < a.n_used; j0 += J) {
            uint4 v[ITEMS][J][8 / N];
            float w[ITEMS][J];
#pragma unroll
            for (int i = 0; i < ITEMS; i++)
#pragma unroll
                for (uint32_t j = 0; j < J; j++) {
                    w[i][j] = 0.0f;
                    int32_t p = -1;
                    if (n[i] && j0 + j < a.n_used) p = __ldg(a.place + t[i] * a.n_used + j0 + j);
                    const bool there = p >= 0 && (uint32_t)p < a.n_places;
                    if (there) w[i][j] = __ldg(a.weights + t[i] * a.n_used + j0 + j);
                    const T *y = static_cast<const T *>(a.y) + (uint64_t)(there ? p : 0) * a.ldy + col[i];
                    if constexpr (VEC) {
#pragma unroll
                        for (int c = 0; c < 8 / N; c++) v[i][j][c] = there ? __ldg(reinterpret_cast<const uint4 *>(y) + c) : make_uint4(0, 0, 0, 0);
                    } else {
                        T *to = reinterpret_cast<T *>(v[i][j]);
#pragma unroll
                        for (uint32_t c = 0; c < 8; c++) to[c] = there && c < n[i] ? y[c] : narrow<T>(0.0f);
                    }
                }
#pragma unroll
            for (int i = 0; i < ITEMS; i++)
#pragma unroll
                for (uint32_t j = 0; j < J; j++) {
                    const T *y = reinterpret_cast<const T *>(v[i][j]);
#pragma unroll
                    for (int c = 0; c < 8; c++) sum[i][c] = fmaf(w[i][j], widen(y[c]), sum[i][c]);
                }
        }
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            if (!n[i]) break;
            O *o = static_cast<O *>(a.out) + t[i] * a.ldo + col[i];
            if constexpr (VEC) {
                O r[8];
#pragma unroll
                for (int c = 0; c < 8; c++) r[c] = narrow<O>(sum[i][c]);
#pragma unroll
                for (uint32_t c = 0; c < 8 * sizeof(O) / 16; c++) reinterpret_cast<uint4 *>(o)[c] = reinterpret_cast<const uint4 *>(r)[c];
            } else {
#pragma unroll
                for (uint32_t c = 0; c < 8; c++)
                    if (c < n[i]) o[c] = narrow<O>(sum[i][c]);
            }
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
    cudaLaunchConfig_t c = {};
    const uint32_t cluster = a.stretches == 1 ? 1 : MOE_SORT_JOIN;
    c.gridDim = dim3((a.stretches + cluster - 1) / cluster * cluster);
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {cluster, 1, 1};
    c.attrs = at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, moe_choose_kernel<T, R>, a);
}
template <typename T>
cudaError_t choose_of(const MoeSortArgs &a, uint32_t smem, cudaStream_t s) {
    return a.n_expert <= 128 ? choose_as<T, 4>(a, smem, s) : a.n_expert <= 256 ? choose_as<T, 8>(a, smem, s) : choose_as<T, 32>(a, smem, s);
}

template <typename T, typename O, bool VEC, int J>
cudaError_t combine_slots(const MoeCombineArgs &a, int sms, cudaStream_t s) {
    constexpr int PER = 256 * combine_items(VEC, J);
    const uint64_t want = (a.n_tok * ((a.dim + 7) / 8) + PER - 1) / PER;
    const uint32_t grid = (uint32_t)(want < (uint64_t)sms * 32 ? want : (uint64_t)sms * 32);
    moe_combine_kernel<T, O, VEC, J><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}
template <typename T, typename O, bool VEC>
cudaError_t combine_vec(const MoeCombineArgs &a, int sms, cudaStream_t s) {
    return a.n_used == 1   ? combine_slots<T, O, VEC, 1>(a, sms, s)
           : a.n_used == 2 ? combine_slots<T, O, VEC, 2>(a, sms, s)
           : a.n_used <= 4 ? combine_slots<T, O, VEC, 4>(a, sms, s)
                           : combine_slots<T, O, VEC, 8>(a, sms, s);
}
template <typename T, typename O>
cudaError_t combine_as(const MoeCombineArgs &a, int sms, cudaStream_t s) {
    return a.vec ? combine_vec<T, O, true>(a, sms, s) : combine_vec<T, O, false>(a, sms, s);
}
template <typename T>
cudaError_t combine_from(const MoeCombineArgs &a, int32_t o, int sms, cudaStream_t s) {
    return o == SG_F32 ? combine_as<T, float>(a, sms, s) : o == SG_F16 ? combine_as<T, __half>(a, sms, s) : combine_as<T, __nv_bfloat16>(a, sms, s);
}

}  // namespace

cudaError_t moe_sort_launch(const MoeSortArgs &a, int32_t type, cudaStream_t s) {
    const uint32_t smem = sort_smem(a.n_expert, a.n_used), first = a.stretches == 1 ? smem : 2 * a.n_expert * 4;
    cudaError_t e = type == SG_F32 ? choose_of<float>(a, first, s) : type == SG_F16 ? choose_of<__half>(a, first, s) : choose_of<__nv_bfloat16>(a, first, s);
    if (e != cudaSuccess || a.stretches == 1) return e;
    static bool ready[64];
    if ((e = big_smem(moe_place_kernel, smem, ready)) != cudaSuccess) return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((a.stretches + MOE_SORT_JOIN - 1) / MOE_SORT_JOIN);
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, moe_place_kernel, a);
}

cudaError_t moe_combine_launch(const MoeCombineArgs &a, int32_t type, int32_t out_type, int sms, cudaStream_t s) {
    return type == SG_F32 ? combine_from<float>(a, out_type, sms, s) : type == SG_F16 ? combine_from<__half>(a, out_type, sms, s) : combine_from<__nv_bfloat16>(a, out_type, sms, s);
}

}  // namespace sg
