// 4-bit lm_head weights: what qs_w4.cu offers to the C ABI.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "qwen600_sampler.h"

namespace qs {

constexpr int kW4MaxHidden = 8192;

struct W4View {
    const unsigned char* codes;
    const void* scales;
    const unsigned char* zeros;  // NULL: every zero point is 8
    int vocab, hidden, group, scale_dtype;
};

size_t w4_codes_bytes(int V, int K);
size_t w4_scales_bytes(int V, int K, int group);
size_t w4_zeros_bytes(int V, int K, int group);
cudaError_t launch_w4_quantize(const __nv_bfloat16* w, int V, int K, int group, unsigned char* codes,
                               __nv_bfloat16* scales, unsigned char* zeros, cudaStream_t st);
cudaError_t launch_w4_pack(const unsigned char* codes, const void* scales, const unsigned char* zeros, int V, int K,
                           int group, unsigned char* pc, void* ps, unsigned char* pz, cudaStream_t st);
// RMSNorm of the hidden rows into normed, and logits[batch, vocab] of them;
// with segk the epilogue also folds the rows' maxima of 256-column segments
// into it, as launch_lm_head does.  ws: w4_workspace bytes.
size_t w4_workspace(int batch, int K);
cudaError_t launch_lm_head_w4(const __nv_bfloat16* hidden, const __nv_bfloat16* norm_weight, const W4View& w, int batch,
                              __nv_bfloat16* normed, __nv_bfloat16* logits, unsigned char* ws, int num_sms,
                              uint32_t* segk, int segk_stride, cudaStream_t st);

}  // namespace qs
