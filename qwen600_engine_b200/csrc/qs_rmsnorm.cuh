// The final RMSNorm's arithmetic for one row per CTA of kNormThreads threads
// (rms_norm_kernel, qwen_model.cuh:125-177): per-thread fma chains over bf16
// pairs, a cub block sum, mul = rsqrtf(fma(sum, 1/D, eps)), y = bf16((x * mul) * w).
#pragma once
#include <cuda_bf16.h>

#include <cub/block/block_reduce.cuh>

namespace qs {

constexpr int kNormThreads = 256;
constexpr float kNormEps = 1e-6f;

// A thread's chain over its pairs threadIdx.x, + kNormThreads, ...
__device__ __forceinline__ float rms_add(float lsum, __nv_bfloat162 x) {
    const float2 v = __bfloat1622float2(x);
    return __fmaf_rn(v.y, v.y, __fmaf_rn(v.x, v.x, lsum));
}

// The row's factor from the threads' chains; the same for every thread.
__device__ __forceinline__ float rms_factor(float lsum, float inv_d, float eps) {
    using BlockReduce = cub::BlockReduce<float, kNormThreads>;
    __shared__ typename BlockReduce::TempStorage tmp;
    const float total = BlockReduce(tmp).Sum(lsum);
    __shared__ float mul;
    if (threadIdx.x == 0) mul = rsqrtf(__fmaf_rn(total, inv_d, eps));
    __syncthreads();
    return mul;
}

__device__ __forceinline__ __nv_bfloat162 rms_scaled(__nv_bfloat162 x, float m, float2 g) {
    float2 v = __bfloat1622float2(x);
    v.x = __fmul_rn(__fmul_rn(v.x, m), g.x);
    v.y = __fmul_rn(__fmul_rn(v.y, m), g.y);
    return __float22bfloat162_rn(v);
}

}  // namespace qs
