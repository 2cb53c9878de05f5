// The lm_head with 4-bit weights for few tokens: quantisation, the packed
// layout and the projection (include/qwen600_sampler.h gives the formulas).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "qs_common.cuh"
#include "qs_w4.h"

namespace qs {

__device__ __forceinline__ float scale_at(const void* s, size_t i, int dtype) {
    return dtype == QS_F16 ? __half2float(((const __half*)s)[i]) : __bfloat162float(((const __nv_bfloat16*)s)[i]);
}

// One thread per group of a row: the range that holds the group and zero, a
// bf16 scale of a fifteenth of it, codes rounded to nearest.
__global__ void w4_quantize_kernel(const __nv_bfloat16* __restrict__ w, int V, int K, int group,
                                   unsigned char* __restrict__ codes, __nv_bfloat16* __restrict__ scales,
                                   unsigned char* __restrict__ zeros) {
    const size_t g = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int per = K / group;
    if (g >= (size_t)V * per) return;
    const __nv_bfloat16* x = w + g * group;
    float lo = 0.0f, hi = 0.0f;
    for (int i = 0; i < group; i++) {
        const float v = __bfloat162float(x[i]);
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
    const __nv_bfloat16 sb = __float2bfloat16_rn((hi - lo) / 15.0f);
    const float s = __bfloat162float(sb);
    const float d = s > 0.0f ? s : 1.0f;  // a group of zeros: scale 0, codes 0
    const float z = fminf(fmaxf(rintf(-lo / d), 0.0f), 15.0f);
    for (int i = 0; i < group; i += 2) {
        const float a = fminf(fmaxf(rintf(__bfloat162float(x[i]) / d) + z, 0.0f), 15.0f);
        const float b = fminf(fmaxf(rintf(__bfloat162float(x[i + 1]) / d) + z, 0.0f), 15.0f);
        codes[(g * group + i) / 2] = (unsigned char)((int)a | ((int)b << 4));
    }
    scales[g] = sb;
    zeros[g] = (unsigned char)z;
}

cudaError_t launch_w4_quantize(const __nv_bfloat16* w, int V, int K, int group, unsigned char* codes,
                               __nv_bfloat16* scales, unsigned char* zeros, cudaStream_t st) {
    const size_t n = (size_t)V * (K / group);
    w4_quantize_kernel<<<(unsigned)((n + 127) / 128), 128, 0, st>>>(w, V, K, group, codes, scales, zeros);
    return cudaGetLastError();
}

size_t w4_codes_bytes(int V, int K) { return (size_t)V * K / 2; }
size_t w4_scales_bytes(int V, int K, int group) { return (size_t)V * (K / group) * 2; }
size_t w4_zeros_bytes(int V, int K, int group) { return (size_t)V * (K / group); }

cudaError_t launch_w4_pack(const unsigned char* codes, const void* scales, const unsigned char* zeros, int V, int K,
                           int group, unsigned char* pc, void* ps, unsigned char* pz, cudaStream_t st) {
    cudaError_t e = cudaMemcpyAsync(pc, codes, w4_codes_bytes(V, K), cudaMemcpyDeviceToDevice, st);
    if (e == cudaSuccess) e = cudaMemcpyAsync(ps, scales, w4_scales_bytes(V, K, group), cudaMemcpyDeviceToDevice, st);
    if (e == cudaSuccess && zeros)
        e = cudaMemcpyAsync(pz, zeros, w4_zeros_bytes(V, K, group), cudaMemcpyDeviceToDevice, st);
    return e;
}

// One warp per vocabulary row and token.
__global__ void __launch_bounds__(256)
lm_head_w4_kernel(const __nv_bfloat16* __restrict__ x, W4View w, __nv_bfloat16* __restrict__ out) {
    const int v = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, b = blockIdx.y;
    if (v >= w.vocab) return;
    const int per = w.hidden / w.group;
    float acc = 0.0f;
    for (int g = 0; g < per; g++) {
        float part = 0.0f;
        const float z = w.zeros ? (float)w.zeros[(size_t)v * per + g] : 8.0f;
        for (int i = lane; i < w.group; i += 32) {
            const int k = g * w.group + i;
            const int c = w.codes[((size_t)v * w.hidden + k) / 2];
            const float q = (float)((k & 1) ? c >> 4 : c & 15) - z;
            part = __fmaf_rn(q, __bfloat162float(x[(size_t)b * w.hidden + k]), part);
        }
        acc = __fmaf_rn(scale_at(w.scales, (size_t)v * per + g, w.scale_dtype), part, acc);
    }
    acc = warp_sum(acc);
    if (lane == 0) out[(size_t)b * w.vocab + v] = __float2bfloat16_rn(acc);
}

cudaError_t launch_lm_head_w4(const __nv_bfloat16* normed, const W4View& w, __nv_bfloat16* logits, int batch,
                              int num_sms, uint32_t* segk, int segk_stride, cudaStream_t st) {
    (void)num_sms; (void)segk; (void)segk_stride;
    for (int b = 0; b < batch; b += 65535) {
        const int n = batch - b < 65535 ? batch - b : 65535;
        lm_head_w4_kernel<<<dim3((w.vocab + 7) / 8, n), 256, 0, st>>>(normed + (size_t)b * w.hidden, w,
                                                                     logits + (size_t)b * w.vocab);
    }
    return cudaGetLastError();
}

}  // namespace qs
