// kv4_attn.cu — attention over the paged 4-bit KV cache.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace sg {

namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The simplest form: a warp per (token, query head), a position at a time with
// the running maximum and sum of the softmax; lane l holds the values l + 32 i.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using L = Kv4Tile<D>;
    constexpr uint32_t G = L::G;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t w = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const uint32_t tok = (uint32_t)(w / a.n_heads), hq = (uint32_t)(w % a.n_heads);
    if (tok >= a.n_tok) return;
    const uint32_t h = hq / a.group;
    uint32_t x = 0, y = a.n_req;
    while (y - x > 1) {
        const uint32_t m = (x + y) / 2;
        if (a.cu[m] <= (int32_t)tok) x = m;
        else y = m;
    }
    float q[G], o[G], m = -INFINITY, l = 0.0f;
    for (uint32_t i = 0; i < G; i++) {
        q[i] = to_f32(((const T *)a.q)[tok * a.q_tok + hq * a.q_head + lane + 32 * i]);
        o[i] = 0.0f;
    }
    int32_t pos = -1;
    if (a.cu[x] <= (int32_t)tok && (int32_t)tok < a.cu[x + 1]) pos = a.seq[x] - a.cu[x + 1] + (int32_t)tok;
    const int32_t page = 1 << a.c.page_shift;
    const int32_t end = min(min(pos + 1, a.seq[x]), (int32_t)a.width * page);
    const int32_t begin = a.window && pos + 1 > (int32_t)a.window ? pos + 1 - (int32_t)a.window : 0;
    for (int32_t t = begin; t < end; t++) {
        const int32_t block = a.tables[x * a.ld_tables + (t >> a.c.page_shift)];
        if ((uint32_t)block >= a.c.n_blocks) continue;
        const uint32_t at = t & (page - 1), p = at & 15;
        const uint8_t *tile = a.c.data + ((((uint64_t)block * a.c.heads + h) << (a.c.page_shift - 4)) + (at >> 4)) * (uint64_t)L::BYTES;
        float s = 0.0f;
        for (uint32_t g = 0; g < G; g++) {
            const uint32_t word = *(const uint32_t *)(tile + p * L::KROW + kv4_word(lane / 8, g, 4, G) * 4);
            const float sc = __half2float(((const __half *)(tile + L::KS))[((p >> 1) * G + g) * 2 + (p & 1)]);
            const float mn = __half2float(((const __half *)(tile + L::KM))[p * G + g]);
            s += q[g] * fmaf(sc, (float)(word >> (lane % 8 * 4) & 15), mn);
        }
        for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(~0u, s, off);
        s *= a.scale;
        const float mm = fmaxf(m, s), f = m == mm ? 1.0f : expf(m - mm), e = s == mm ? 1.0f : expf(s - mm);
        m = mm;
        l = l * f + e;
        for (uint32_t g = 0; g < G; g++) {
            const uint16_t word = *(const uint16_t *)(tile + L::VC + (p >> 1) * L::VROW + kv4_word(lane / 4, g, 8, G) * 4 + (p & 1) * 2);
            const uint32_t pair = ((p >> 1) * G + g) * 2 + (p & 1);
            const float sc = __half2float(((const __half *)(tile + L::VS))[pair]), mn = __half2float(((const __half *)(tile + L::VM))[pair]);
            o[g] = o[g] * f + e * fmaf(sc, (float)(word >> (lane % 4 * 4) & 15), mn);
        }
    }
    for (uint32_t g = 0; g < G; g++)
        ((T *)a.out)[tok * a.o_tok + hq * a.o_head + lane + 32 * g] = from_f32<T>(l > 0.0f || l != l ? o[g] / l : 0.0f);
    if (a.lse && lane == 0) a.lse[(uint64_t)tok * a.n_heads + hq] = l > 0.0f || l != l ? m + logf(l) : -INFINITY;
}

template <typename T>
void launch(const Kv4AttnArgs &a, uint32_t d, cudaStream_t s) {
    const uint32_t grid = (uint32_t)(((uint64_t)a.n_tok * a.n_heads + 3) / 4);
    if (d == 64) kv4_attn_kernel<T, 64><<<grid, 128, 0, s>>>(a);
    else if (d == 128) kv4_attn_kernel<T, 128><<<grid, 128, 0, s>>>(a);
    else kv4_attn_kernel<T, 256><<<grid, 128, 0, s>>>(a);
}

}  // namespace

sg_status kv4_attention_launch(const Kv4AttnArgs &a, int32_t type, uint32_t d, int sms, cudaStream_t s, cudaError_t *err) {
    if (type == SG_F32) launch<float>(a, d, s);
    else if (type == SG_F16) launch<__half>(a, d, s);
    else launch<__nv_bfloat16>(a, d, s);
    *err = cudaGetLastError();
    return *err == cudaSuccess ? SG_OK : SG_ERR_CUDA;
}

}  // namespace sg
