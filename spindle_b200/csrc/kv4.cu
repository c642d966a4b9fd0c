// kv4.cu — bookkeeping and rows of the paged 4-bit KV cache: block tables and
// slot maps from request lengths, rows quantized into the cache, rows read back.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace sg {

namespace {

template <typename T>
struct Conv;
template <>
struct Conv<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Conv<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Conv<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

__device__ __forceinline__ uint32_t warp_scan(uint32_t v, uint32_t lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= (uint32_t)o) v += u;
    }
    return v;
}

}  // namespace

// ---- plan -------------------------------------------------------------------
//
// Every CTA scans all requests (1024 at a time: new positions, blocks wanted,
// blocks given back), so one launch does without a grid-wide step, and fills its
// own stretch of the new positions: the request of a position by a binary search
// of the scan in shared memory.  A new block of a request starts exactly at the
// one new position that is a multiple of the page, so the thread of that
// position writes the table entry, and everyone else computes the block from the
// ring without reading it back.
__global__ void __launch_bounds__(KV4_PLAN_THREADS) kv4_plan_kernel(const __grid_constant__ Kv4PlanArgs a) {
    __shared__ uint32_t cu_s[KV4_PLAN_THREADS + 1], want_s[KV4_PLAN_THREADS];
    __shared__ int32_t ctx_s[KV4_PLAN_THREADS];
    __shared__ uint32_t warp_s[3][32], total_s[3];
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const uint32_t page = 1u << a.page_shift;
    const uint32_t head = (uint32_t)a.cursor[0], tail = (uint32_t)a.cursor[1], free_blocks = tail - head;
    const uint32_t per = (a.max_tok + gridDim.x - 1) / gridDim.x;
    const uint32_t t0 = min(a.max_tok, blockIdx.x * per), t1 = min(a.max_tok, t0 + per);
    uint32_t base_come = 0, base_want = 0, base_back = 0;

    for (uint32_t r0 = 0; r0 < a.n_req; r0 += KV4_PLAN_THREADS) {
        const uint32_t r = r0 + tid, n = min((uint32_t)KV4_PLAN_THREADS, a.n_req - r0);
        uint32_t ctx = 0, come = 0, want = 0, kept = 0, back = 0;
        bool ends = false;
        if (r < a.n_req) {
            const int32_t add = a.add[r];
            ctx = (uint32_t)max(a.ctx[r], 0);
            ends = add < 0;
            come = (uint32_t)max(add, 0);
            const uint32_t have = min((ctx + page - 1) >> a.page_shift, a.width);
            const uint32_t need = min((ctx + come + page - 1) >> a.page_shift, a.width);
            want = ends ? 0 : need - have;
            kept = ends ? have : 0;
        }
        // what a request that ends gives back: its entries that are blocks, counted a warp per request
        for (uint32_t todo = __ballot_sync(0xffffffffu, kept > 0); todo; todo &= todo - 1) {
            const int src = __ffs(todo) - 1;
            const uint32_t cnt = __shfl_sync(0xffffffffu, kept, src);
            const int32_t *row = a.tables + (uint64_t)(r0 + wid * 32 + src) * a.ld_tables;
            uint32_t valid = 0;
            for (uint32_t j = lane; j < cnt; j += 32) valid += (uint32_t)row[j] < a.n_blocks;
            valid = __reduce_add_sync(0xffffffffu, valid);
            if (lane == (uint32_t)src) back = valid;
        }
        const uint32_t s0 = warp_scan(come, lane), s1 = warp_scan(want, lane), s2 = warp_scan(back, lane);
        if (lane == 31) warp_s[0][wid] = s0, warp_s[1][wid] = s1, warp_s[2][wid] = s2;
        __syncthreads();
        if (wid < 3) {
            const uint32_t v = warp_s[wid][lane], inc = warp_scan(v, lane);
            warp_s[wid][lane] = inc - v;
            if (lane == 31) total_s[wid] = inc;
        }
        __syncthreads();
        const uint32_t c0 = base_come + warp_s[0][wid] + s0 - come;
        cu_s[tid] = c0;
        want_s[tid] = base_want + warp_s[1][wid] + s1 - want;
        ctx_s[tid] = (int32_t)ctx;
        const uint32_t back_at = base_back + warp_s[2][wid] + s2 - back;
        if (tid == 0) cu_s[KV4_PLAN_THREADS] = base_come + total_s[0];
        if (blockIdx.x == 0 && r < a.n_req) {
            a.cu[r] = (int32_t)c0;
            a.seq[r] = ends ? 0 : (int32_t)(ctx + come);
        }
        __syncthreads();
        // the blocks of the requests that end go back to the ring's tail, in table order, a warp per request
        for (uint32_t todo = __ballot_sync(0xffffffffu, back > 0 && (r % gridDim.x) == blockIdx.x); todo; todo &= todo - 1) {
            const int src = __ffs(todo) - 1;
            const uint32_t cnt = __shfl_sync(0xffffffffu, kept, src);
            uint32_t at = tail + __shfl_sync(0xffffffffu, back_at, src);
            const int32_t *row = a.tables + (uint64_t)(r0 + wid * 32 + src) * a.ld_tables;
            for (uint32_t j0 = 0; j0 < cnt; j0 += 32) {
                const int32_t block = j0 + lane < cnt ? row[j0 + lane] : -1;
                const uint32_t is = __ballot_sync(0xffffffffu, (uint32_t)block < a.n_blocks);
                if ((uint32_t)block < a.n_blocks) a.ring[(at + __popc(is & ((1u << lane) - 1))) % a.n_blocks] = block;
                at += __popc(is);
            }
        }
        // this CTA's new positions among these requests
        const uint32_t lo = max(t0, base_come), hi = min(t1, base_come + total_s[0]);
        for (uint32_t t = lo + tid; t < hi; t += KV4_PLAN_THREADS) {
            uint32_t x = 0, y = n;  // the last request with cu <= t
            while (y - x > 1) {
                const uint32_t m = (x + y) >> 1;
                if (cu_s[m] <= t) x = m;
                else y = m;
            }
            const uint32_t c = (uint32_t)ctx_s[x], pos = c + (t - cu_s[x]);
            const uint32_t have = min((c + page - 1) >> a.page_shift, a.width), j = pos >> a.page_shift;
            int32_t *row = a.tables + (uint64_t)(r0 + x) * a.ld_tables;
            int32_t block = -1;
            if (j >= a.width) {
            } else if (j < have) {
                block = row[j];
            } else {
                const uint32_t k = want_s[x] + j - have;
                if (k < free_blocks) block = a.ring[(head + k) % a.n_blocks];
                if ((pos & (page - 1)) == 0) row[j] = block;
            }
            a.pos[t] = (int32_t)pos;
            a.slots[t] = (uint32_t)block < a.n_blocks ? block * (int32_t)page + (int32_t)(pos & (page - 1)) : -1;
        }
        base_come += total_s[0];
        base_want += total_s[1];
        base_back += total_s[2];
        __syncthreads();
    }
    for (uint32_t t = max(t0, min(base_come, t1)) + tid; t < t1; t += KV4_PLAN_THREADS) a.pos[t] = a.slots[t] = -1;
    if (blockIdx.x == 0 && tid == 0) {
        const uint32_t taken = min(base_want, free_blocks);
        a.cu[a.n_req] = (int32_t)base_come;
        const uint32_t turn = (head + taken) / a.n_blocks * a.n_blocks;  // the head stays inside the ring
        a.info[0] = (int32_t)(head + taken - turn);
        a.info[1] = (int32_t)(tail + base_back - turn);
        a.info[2] = (int32_t)base_come;
        a.info[3] = (int32_t)(base_want - taken);
    }
}

// ---- append -------------------------------------------------------------------
//
// Four lanes per group of 32 values, eight values each: lane j's eight are the
// K word (j, g), and the two V half words (2j, g) and (2j + 1, g).
//   m = f16(min), s = f16((max - m) * f32(1/15)), c = rint(clamp((x - m) * (1 / s), 0, 15))
// with x clamped to f16's finite range and NaN counted as 0, so that the cache
// holds finite numbers only; groups that had such a value are counted.  Every
// step is one rounded f32 operation, so the codes can be reproduced bit for bit.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(KV4_ROW_THREADS) kv4_append_kernel(const __grid_constant__ Kv4RowArgs a) {
    using L = Kv4Tile<D>;
    constexpr uint32_t G = L::G;
    const uint64_t n = (uint64_t)a.n_tok * a.c.heads * G * 2;  // groups: K's and V's of a row side by side
    for (uint64_t i0 = ((uint64_t)blockIdx.x * KV4_ROW_THREADS + threadIdx.x) >> 2; i0 < ((n + 7) & ~7ull);
         i0 += (uint64_t)gridDim.x * KV4_ROW_THREADS >> 2) {
        const bool live = i0 < n;
        const uint64_t i = live ? i0 : n - 1;
        const uint32_t j = threadIdx.x & 3, g = (uint32_t)(i % G), is_v = (uint32_t)(i / G) & 1;
        const uint64_t row = i / (2 * G);
        const uint32_t h = (uint32_t)(row % a.c.heads);
        const uint64_t t = row / a.c.heads;
        const int32_t slot = a.slots[t];
        const T *src = (const T *)(is_v ? a.v : a.k) + t * (is_v ? a.v_tok : a.k_tok) + h * (is_v ? a.v_head : a.k_head) +
                       g * 32 + j * 8;
        float x[8];
        if (VEC) {
            alignas(16) T raw[8];
            constexpr int W = sizeof(T) * 8 / 16;
#pragma unroll
            for (int w = 0; w < W; w++) reinterpret_cast<uint4 *>(raw)[w] = __ldg(reinterpret_cast<const uint4 *>(src) + w);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = Conv<T>::get(raw[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = Conv<T>::get(src[e]);
        }
        float lo = x[0], hi = x[0], odd = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) odd = fmaf(x[e], 0.0f, odd);  // NaN when a value is not finite
        bool bad = !(odd == 0.0f);
        if (bad) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = x[e] == x[e] ? x[e] : 0.0f;
            lo = hi = x[0];
        }
#pragma unroll
        for (int e = 1; e < 8; e++) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        lo = fminf(fmaxf(lo, -65504.0f), 65504.0f);
        hi = fminf(fmaxf(hi, -65504.0f), 65504.0f);
        const __half mh = __float2half_rn(lo + 0.0f);  // + 0: no negative zero
        const float m = __half2float(mh);
        const __half sh = __float2half_rn(__fmul_rn(fmaxf(hi - m, 0.0f), 1.0f / 15.0f));
        const float s = __half2float(sh), r = s > 0.0f ? __frcp_rn(s) : 0.0f;
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float y = fminf(fmaxf(x[e], -65504.0f), 65504.0f);
            const float c = fminf(fmaxf(__fmul_rn(__fsub_rn(y, m), r), 0.0f), 15.0f);
            word |= (uint32_t)__float2int_rn(c) << (4 * e);
        }
        const unsigned any = __ballot_sync(0xffffffffu, bad && live) >> (threadIdx.x & 28) & 0xf;
        if (!live || slot < 0 || (uint32_t)(slot >> a.c.page_shift) >= a.c.n_blocks) continue;
        if (any && j == 0 && a.nonfinite) atomicAdd(a.nonfinite, 1);
        const uint32_t at = (uint32_t)slot & ((1u << a.c.page_shift) - 1), p = at & 15;
        uint8_t *tile = a.c.data + ((((uint64_t)(slot >> a.c.page_shift) * a.c.heads + h) << (a.c.page_shift - 4)) + (at >> 4)) *
                                       (uint64_t)L::BYTES;
        const uint32_t pair = ((p >> 1) * G + g) * 2 + (p & 1);
        if (is_v) {
            uint8_t *v = tile + L::VC + (p >> 1) * L::VROW + (p & 1) * 2;
            *reinterpret_cast<uint16_t *>(v + kv4_word(2 * j, g, 8, G) * 4) = (uint16_t)word;
            *reinterpret_cast<uint16_t *>(v + kv4_word(2 * j + 1, g, 8, G) * 4) = (uint16_t)(word >> 16);
            if (j == 0) {
                reinterpret_cast<__half *>(tile + L::VS)[pair] = sh;
                reinterpret_cast<__half *>(tile + L::VM)[pair] = mh;
            }
        } else {
            *reinterpret_cast<uint32_t *>(tile + p * L::KROW + kv4_word(j, g, 4, G) * 4) = word;
            if (j == 0) {
                reinterpret_cast<__half *>(tile + L::KS)[pair] = sh;
                reinterpret_cast<__half *>(tile + L::KM)[p * G + g] = mh;
            }
        }
    }
}

// ---- read ---------------------------------------------------------------------
// The values of given slots, m + s * c rounded once; a slot that is no slot reads as zeros.
template <typename T, int D>
__global__ void __launch_bounds__(KV4_ROW_THREADS) kv4_read_kernel(const __grid_constant__ Kv4RowArgs a) {
    using L = Kv4Tile<D>;
    constexpr uint32_t G = L::G;
    const uint64_t n = (uint64_t)a.n_tok * a.c.heads * G * 8;  // 8 values each: 4 lanes of K, 4 of V per group
    for (uint64_t i = (uint64_t)blockIdx.x * KV4_ROW_THREADS + threadIdx.x; i < n; i += (uint64_t)gridDim.x * KV4_ROW_THREADS) {
        const uint32_t j = (uint32_t)i & 3, g = (uint32_t)(i / 4 % G), is_v = (uint32_t)(i / (4 * G)) & 1;
        const uint64_t row = i / (8 * G), t = row / a.c.heads;
        const uint32_t h = (uint32_t)(row % a.c.heads);
        const int32_t slot = a.slots[t];
        alignas(16) T y[8];
        if (slot < 0 || (uint32_t)(slot >> a.c.page_shift) >= a.c.n_blocks) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = Conv<T>::put(0.0f);
        } else {
            const uint32_t at = (uint32_t)slot & ((1u << a.c.page_shift) - 1), p = at & 15;
            const uint8_t *tile = a.c.data + ((((uint64_t)(slot >> a.c.page_shift) * a.c.heads + h) << (a.c.page_shift - 4)) + (at >> 4)) *
                                                 (uint64_t)L::BYTES;
            const uint32_t pair = ((p >> 1) * G + g) * 2 + (p & 1);
            uint32_t word;
            float s, m;
            if (is_v) {
                const uint8_t *v = tile + L::VC + (p >> 1) * L::VROW + (p & 1) * 2;
                word = *reinterpret_cast<const uint16_t *>(v + kv4_word(2 * j, g, 8, G) * 4) |
                       (uint32_t) * reinterpret_cast<const uint16_t *>(v + kv4_word(2 * j + 1, g, 8, G) * 4) << 16;
                s = __half2float(reinterpret_cast<const __half *>(tile + L::VS)[pair]);
                m = __half2float(reinterpret_cast<const __half *>(tile + L::VM)[pair]);
            } else {
                word = *reinterpret_cast<const uint32_t *>(tile + p * L::KROW + kv4_word(j, g, 4, G) * 4);
                s = __half2float(reinterpret_cast<const __half *>(tile + L::KS)[pair]);
                m = __half2float(reinterpret_cast<const __half *>(tile + L::KM)[p * G + g]);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = Conv<T>::put(fmaf(s, (float)(word >> (4 * e) & 15u), m));
        }
        uint4 *dst = reinterpret_cast<uint4 *>((T *)(is_v ? a.v_out : a.k_out) + row * D + g * 32 + j * 8);
        constexpr int W = sizeof(T) * 8 / 16;
#pragma unroll
        for (int w = 0; w < W; w++) dst[w] = reinterpret_cast<const uint4 *>(y)[w];
    }
}

namespace {
template <typename T, bool VEC>
kv4_row_fn pick_append(uint32_t d) {
    return d == 64 ? kv4_append_kernel<T, 64, VEC> : d == 128 ? kv4_append_kernel<T, 128, VEC> : kv4_append_kernel<T, 256, VEC>;
}
template <typename T>
kv4_row_fn pick_read(uint32_t d) {
    return d == 64 ? kv4_read_kernel<T, 64> : d == 128 ? kv4_read_kernel<T, 128> : kv4_read_kernel<T, 256>;
}
}  // namespace

kv4_row_fn kv4_append_kernel_for(int32_t type, uint32_t d, bool vec) {
    if (type == SG_F32) return vec ? pick_append<float, true>(d) : pick_append<float, false>(d);
    if (type == SG_F16) return vec ? pick_append<__half, true>(d) : pick_append<__half, false>(d);
    return vec ? pick_append<__nv_bfloat16, true>(d) : pick_append<__nv_bfloat16, false>(d);
}

kv4_row_fn kv4_read_kernel_for(int32_t type, uint32_t d) {
    return type == SG_F32 ? pick_read<float>(d) : type == SG_F16 ? pick_read<__half>(d) : pick_read<__nv_bfloat16>(d);
}

}  // namespace sg
