// logprobs.cu — log probabilities of given tokens with entropy, rank and the
// likeliest alternatives, one CTA per row.
//
//   m = max x, z = sum e^(x - m), logprob = x_tok - m - ln z,
//   entropy = ln z - sum (x - m) e^(x - m) / z,
//   rank = how many tokens come before the given one when sorted by falling
//   logit, equal ones by rising index; the alternatives are the first of that order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "logprobs.cuh"

namespace sg {

namespace {

constexpr int THREADS = 1024;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// Order of falling logits, equal ones by rising index, as one number (larger
// comes first).  NaN counts as larger than everything; the zeros are equal.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x == x ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0xfffffffeu;
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)order_of(x) << 32 | (uint32_t)~i; }

struct Sum {
    float m, z, zx;  // running max, sum e^(x-m), sum (x-m) e^(x-m)
};

// A term whose weight is zero counts nothing, whatever its distance.
__device__ __forceinline__ Sum join(Sum a, Sum b) {
    if (b.m > a.m) {
        const Sum t = a;
        a = b;
        b = t;
    }
    if (b.z == 0.0f && b.m == b.m) return a;
    const float d = b.m - a.m, w = d == 0.0f ? 1.0f : expf(d);  // equal infinities: no difference
    a.z += b.z * w;
    a.zx += w == 0.0f ? 0.0f : (b.zx + d * b.z) * w;
    return a;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) logprobs_kernel(const LogprobsArgs a) {
    __shared__ Sum sum_s[32];
    __shared__ uint64_t key_s[32];
    __shared__ uint32_t cnt_s[32];
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.logits + (uint64_t)row * a.ld;
        const int32_t tok = a.tokens ? a.tokens[row] : -1;
        const bool given = tok >= 0 && (uint32_t)tok < a.vocab;
        const uint64_t kt = given ? key_of(to_f32(x[tok]), tok) : ~0ull;
        Sum s = {-INFINITY, 0.0f, 0.0f};
        uint32_t ahead = 0;
        for (uint32_t i = tid; i < a.vocab; i += THREADS) {
            const float v = to_f32(x[i]);
            ahead += key_of(v, i) > kt;
            s = join(s, Sum{v, v == -INFINITY ? 0.0f : 1.0f, 0.0f});
        }
        for (int o = 16; o; o >>= 1) {
            s = join(s, Sum{__shfl_xor_sync(~0u, s.m, o), __shfl_xor_sync(~0u, s.z, o), __shfl_xor_sync(~0u, s.zx, o)});
            ahead += __shfl_xor_sync(~0u, ahead, o);
        }
        if (lane == 0) sum_s[wid] = s, cnt_s[wid] = ahead;
        __syncthreads();
        s = sum_s[0], ahead = cnt_s[0];
        for (int w = 1; w < 32; w++) s = join(s, sum_s[w]), ahead += cnt_s[w];
        const bool none = s.m == -INFINITY && s.z == 0.0f;  // a row whose mask leaves nothing
        const float lz = s.m == INFINITY ? NAN : logf(s.z);  // an infinite logit leaves no probabilities
        if (tid == 0) {
            a.logprob[row] = !given ? NAN : none ? -INFINITY : to_f32(x[tok]) - s.m - lz;
            a.entropy[row] = none ? 0.0f : lz - s.zx / s.z;
            a.rank[row] = given ? (int32_t)ahead : -1;
        }
        uint64_t last = ~0ull;
        for (uint32_t k = 0; k < a.top; k++) {
            uint64_t best = 0;
            for (uint32_t i = tid; i < a.vocab; i += THREADS) {
                const uint64_t q = key_of(to_f32(x[i]), i);
                if (q < last && q > best) best = q;
            }
            for (int o = 16; o; o >>= 1) {
                const uint64_t q = __shfl_xor_sync(~0u, best, o);
                best = q > best ? q : best;
            }
            __syncthreads();
            if (lane == 0) key_s[wid] = best;
            __syncthreads();
            for (int w = 0; w < 32; w++) best = key_s[w] > best ? key_s[w] : best;
            last = best;
            if (tid == 0) {
                const uint32_t id = ~(uint32_t)best;
                a.top_ids[(uint64_t)row * a.top + k] = (int32_t)id;
                a.top_logprobs[(uint64_t)row * a.top + k] = none ? -INFINITY : to_f32(x[id]) - s.m - lz;
            }
        }
        __syncthreads();
    }
}

}  // namespace

sg_status logprobs_launch(const LogprobsArgs &a, int32_t type, int sms, cudaStream_t s, cudaError_t *err) {
    const uint32_t grid = a.rows < (uint32_t)sms * 2 ? a.rows : (uint32_t)sms * 2;
    if (type == SG_F32) logprobs_kernel<float><<<grid, THREADS, 0, s>>>(a);
    else if (type == SG_F16) logprobs_kernel<__half><<<grid, THREADS, 0, s>>>(a);
    else logprobs_kernel<__nv_bfloat16><<<grid, THREADS, 0, s>>>(a);
    *err = cudaGetLastError();
    return *err == cudaSuccess ? SG_OK : SG_ERR_CUDA;
}

}  // namespace sg
