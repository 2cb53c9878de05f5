// The final RMSNorm's arithmetic for one row per CTA of kNormThreads threads
// (rms_norm_kernel, qwen_model.cuh:125-177): per-thread fma chains over bf16
// pairs, a cub block sum, mul = rsqrtf(fma(sum, 1/D, eps)), y = bf16((x * mul) * w).
#pragma once
#include <cuda_bf16.h>

#include <cub/block/block_reduce.cuh>

namespace qs {

constexpr int kNormThreads = 256;
constexpr float kNormEps = 1e-6f;

// The factor of a row of 2 * half values; the same for every thread.
__device__ __forceinline__ float rms_factor(const __nv_bfloat162* in, int half, float inv_d, float eps) {
    float lsum = 0.0f;
    for (int i = threadIdx.x; i < half; i += kNormThreads) {
        const float2 v = __bfloat1622float2(in[i]);
        lsum = __fmaf_rn(v.x, v.x, lsum);
        lsum = __fmaf_rn(v.y, v.y, lsum);
    }
    using BlockReduce = cub::BlockReduce<float, kNormThreads>;
    __shared__ typename BlockReduce::TempStorage tmp;
    const float total = BlockReduce(tmp).Sum(lsum);
    __shared__ float mul;
    if (threadIdx.x == 0) mul = rsqrtf(__fmaf_rn(total, inv_d, eps));
    __syncthreads();
    return mul;
}

__device__ __forceinline__ __nv_bfloat162 rms_scaled(__nv_bfloat162 x, float m, const __nv_bfloat162* w, int i) {
    float2 v = __bfloat1622float2(x);
    const float2 g = w ? __bfloat1622float2(w[i]) : make_float2(1.0f, 1.0f);
    v.x = __fmul_rn(__fmul_rn(v.x, m), g.x);
    v.y = __fmul_rn(__fmul_rn(v.y, m), g.y);
    return __float22bfloat162_rn(v);
}

}  // namespace qs
