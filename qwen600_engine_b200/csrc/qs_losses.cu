// Log-probabilities of chosen tokens, the clipped policy loss and the paired
// preference loss over them, with their gradients (include/qwen600_sampler.h
// gives the formulas).
//
// Everything rests on one row operation.  With m the row's maximum,
//   excess = sum_j exp((x[j] - m) / T) - 1      (the maximum's own term left out)
//   logprob = (x[t] - m) / T - log(1 + excess)
//   d logprob / d x[j] = ([j = t] - exp((x[j] - m) / T) / (1 + excess)) / T
// The maximum's own term is exactly 1; keeping it out of the fp32 sum lets a
// peaked row (log-probability near 0) keep its relative precision.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "qs_common.cuh"
#include "qwen600_sampler.h"

namespace qs {

int set_error(int code, const char* msg);  // qs_api.cu

constexpr int kLossThreads = 256;

// What a scored row leaves for the losses and the gradient.
struct RowScore {
    double logprob;  // 0 for a row that scores nothing
    float max;
    float excess;
    int scored;
    int pad;
};

template <typename T>
__device__ __forceinline__ float elem(const T* p, long long i) { return Elem<T>::widen(p[i]); }
__device__ __forceinline__ void put(float* p, long long i, float v) { p[i] = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, long long i, float v) { p[i] = __float2bfloat16_rn(v); }

__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Block-wide sum of one double per thread, in a fixed order.
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) s += red[w];
    return s;
}

template <typename T>
__global__ void __launch_bounds__(kLossThreads)
score_rows_kernel(const T* __restrict__ logits, int V, long long ld, const int* __restrict__ tokens,
                  const float* __restrict__ weights, double inv_t, RowScore* __restrict__ out,
                  float* __restrict__ logprobs, float* __restrict__ stats) {
    __shared__ float redf[32];
    __shared__ double redd[32];
    const int row = blockIdx.x, t = threadIdx.x;
    const int tok = tokens[row];
    const bool scored = tok >= 0 && tok < V && !(weights && weights[row] == 0.0f);
    RowScore r{0.0, 0.0f, 0.0f, 0, 0};
    if (scored) {
        const T* x = logits + (size_t)row * ld;
        float m = -INFINITY;
        for (int j = t; j < V; j += kLossThreads) m = fmaxf(m, elem(x, j));
        m = warp_max(m);
        if ((t & 31) == 0) redf[t >> 5] = m;
        __syncthreads();
        m = redf[0];
        for (int w = 1; w < kLossThreads / 32; w++) m = fmaxf(m, redf[w]);
        const float scale = (float)(inv_t * 1.4426950408889634);
        float s = 0.0f;
        int n = 0;
        for (int j = t; j < V; j += kLossThreads) {
            const float d = elem(x, j) - m;
            if (d == 0.0f) n++;
            else s += exp2_fast(d * scale);
        }
        const double others = block_sum((double)s, redd);
        const double at_max = block_sum((double)n, redd);
        r.scored = 1;
        r.max = m;
        const double excess = isinf(m) ? (double)NAN : others + (at_max - 1.0);
        r.excess = (float)excess;
        r.logprob = ((double)elem(x, tok) - (double)m) * inv_t - log1p(excess);
    }
    if (t == 0) {
        if (out) out[row] = r;
        if (logprobs) logprobs[row] = (float)r.logprob;
        if (stats) {
            stats[2 * (size_t)row] = r.max;
            stats[2 * (size_t)row + 1] = r.excess;
        }
    }
}

// grad = coef * ([j = t] - p_j) / T for one row per CTA.
template <typename T>
__global__ void __launch_bounds__(kLossThreads)
grad_rows_kernel(const T* logits, int V, long long ld, const int* __restrict__ tokens,
                 const float* __restrict__ stats, int stat_words, const float* __restrict__ coefs,
                 double inv_t, T* grad, long long gld) {
    const int row = blockIdx.x, t = threadIdx.x;
    const int tok = tokens[row];
    const float coef = coefs[row];
    const T* x = logits + (size_t)row * ld;
    T* g = grad + (size_t)row * gld;
    if (tok < 0 || tok >= V || coef == 0.0f) {
        for (int j = t; j < V; j += kLossThreads) put(g, j, 0.0f);
        return;
    }
    const float* st = reinterpret_cast<const float*>(reinterpret_cast<const char*>(stats) + (size_t)row * stat_words * 4);
    const float m = st[0];
    const double excess = st[1];
    const float scale = (float)(inv_t * 1.4426950408889634);
    const double c = (double)coef * inv_t;
    const float f = (float)(-c / (1.0 + excess));
    for (int j = t; j < V; j += kLossThreads) {
        const float v = elem(x, j);
        if (j == tok) {
            // 1 - p without cancellation where the token is the maximum
            const double q = v == m ? excess / (1.0 + excess) : 1.0 - exp(((double)v - (double)m) * inv_t) / (1.0 + excess);
            put(g, j, (float)(c * q));
        } else {
            put(g, j, f * exp2_fast((v - m) * scale));
        }
    }
}

// Per-row term of the policy loss: returns l, and its slope dl / dlogprob.
__device__ __forceinline__ double policy_term(double lp, double old_lp, double ref_lp, double adv, double lo,
                                              double hi, double kl, double* slope) {
    const double r = exp(lp - old_lp);
    const double clipped = r < lo ? lo : r > hi ? hi : r;
    const bool cut = (adv > 0.0 && r > hi) || (adv < 0.0 && r < lo);
    double l = -(cut ? clipped : r) * adv;
    double sl = cut ? 0.0 : -adv * r;
    if (kl > 0.0) {
        const double d = ref_lp - lp;
        const double e = expm1(d);
        l += kl * (e - d);
        sl -= kl * e;
    }
    *slope = sl;
    return l;
}

__global__ void __launch_bounds__(1024)
policy_rows_kernel(const RowScore* __restrict__ score, int rows, const float* __restrict__ old_lp,
                   const float* __restrict__ ref_lp, const float* __restrict__ adv,
                   const float* __restrict__ weights, qs_policy_params p, float* __restrict__ coefs,
                   float* __restrict__ loss) {
    __shared__ double red[32];
    double sum = 0.0;
    for (int i = threadIdx.x; i < rows; i += blockDim.x) {
        double c = 0.0;
        if (score[i].scored) {
            const double w = weights ? (double)weights[i] : 1.0 / rows;
            double slope;
            sum += w * policy_term(score[i].logprob, old_lp[i], p.kl_coef > 0.0 ? (double)ref_lp[i] : 0.0, adv[i],
                                   1.0 - p.clip_low, 1.0 + p.clip_high, p.kl_coef, &slope);
            c = w * slope;
        }
        coefs[i] = (float)c;
    }
    sum = block_sum(sum, red);
    if (threadIdx.x == 0) *loss = (float)sum;
}

// One warp per pair in turn: the two sequences' sums, the pair's loss and the
// coefficient of every row's gradient.
__global__ void __launch_bounds__(1024)
preference_pairs_kernel(const RowScore* __restrict__ score, int rows, const int* __restrict__ offsets, int pairs,
                        const float* __restrict__ ref, const float* __restrict__ weights,
                        qs_preference_params p, float* __restrict__ coefs, float* __restrict__ seq_lp,
                        float* __restrict__ loss) {
    __shared__ double red[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < rows; i += blockDim.x) coefs[i] = 0.0f;
    __syncthreads();
    double sum = 0.0;
    for (int q = warp; q < pairs; q += 32) {
        const int a[2] = {offsets[q], offsets[pairs + q]}, b[2] = {offsets[q + 1], offsets[pairs + q + 1]};
        const bool fine = a[0] >= 0 && a[0] <= b[0] && b[0] <= rows && a[1] >= 0 && a[1] <= b[1] && b[1] <= rows;
        double s[2] = {NAN, NAN};
        if (fine) {
            for (int k = 0; k < 2; k++) {
                double v = 0.0;
                for (int i = a[k] + lane; i < b[k]; i += 32) v += score[i].logprob;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                s[k] = v;
            }
        }
        const double z = p.beta * ((s[0] - (double)ref[q]) - (s[1] - (double)ref[pairs + q]));
        const double w = weights ? (double)weights[q] : 1.0 / pairs;
        const double e = p.label_smoothing;
        // -log sigmoid(z) = max(-z, 0) + log(1 + exp(-|z|)), and -log sigmoid(-z) = that + z
        const double low = fmax(-z, 0.0) + log1p(exp(-fabs(z)));
        const double slope =
            w == 0.0 ? 0.0 : -p.beta * w * ((1.0 - e) / (1.0 + exp(z)) - e / (1.0 + exp(-z)));
        if (lane == 0) {
            if (w != 0.0) sum += w * (low + (e > 0.0 ? e * z : 0.0));
            if (seq_lp) {
                seq_lp[q] = (float)s[0];
                seq_lp[pairs + q] = (float)s[1];
            }
        }
        if (fine)
            for (int k = 0; k < 2; k++)
                for (int i = a[k] + lane; i < b[k]; i += 32) coefs[i] = (float)(k ? -slope : slope);
    }
    sum = block_sum(sum, red);
    if (threadIdx.x == 0) *loss = (float)sum;
}

// --------------------------------------------------------------- host side
static int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return set_error(code, buf);
}

static int check_launch(const char* what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? QS_OK : fail(QS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

struct Rows {
    const void* logits;
    int dtype, rows, vocab;
    long long ld;
    const int* tokens;
    double inv_t;
    void* grad;
    long long gld;
    size_t esz() const { return dtype == QS_F32 ? 4 : 2; }
};

static int check_rows(const Rows& r, double temperature) {
    if (r.dtype != QS_F32 && r.dtype != QS_BF16) return fail(QS_ERR_INVALID, "unknown dtype %d", r.dtype);
    if (r.rows < 0) return fail(QS_ERR_INVALID, "rows %d < 0", r.rows);
    if (r.rows > 1 << 27) return fail(QS_ERR_UNSUPPORTED, "rows %d above 2^27", r.rows);
    if (r.vocab < 1 || r.vocab > kMaxVocab)
        return fail(QS_ERR_UNSUPPORTED, "vocab %d outside [1, %d]", r.vocab, kMaxVocab);
    if (!(temperature >= 1e-6) || isinf(temperature))
        return fail(QS_ERR_INVALID, "temperature %g is not a finite number of at least 1e-6", temperature);
    if (r.rows == 0) return QS_OK;
    if (!r.logits || !r.tokens) return fail(QS_ERR_INVALID, "NULL device pointer");
    if (((uintptr_t)r.logits | (uintptr_t)r.grad) % r.esz())
        return fail(QS_ERR_INVALID, "logits and gradient must be aligned to their element");
    if (r.rows > 1 && r.ld < r.vocab) return fail(QS_ERR_INVALID, "row_stride %lld < vocab %d", r.ld, r.vocab);
    if (r.grad) {
        if (r.rows > 1 && r.gld < r.vocab)
            return fail(QS_ERR_INVALID, "grad_row_stride %lld < vocab %d", r.gld, r.vocab);
        const uintptr_t a = (uintptr_t)r.logits, g = (uintptr_t)r.grad;
        const size_t an = ((size_t)(r.rows - 1) * r.ld + r.vocab) * r.esz();
        const size_t gn = ((size_t)(r.rows - 1) * r.gld + r.vocab) * r.esz();
        if (a < g + gn && g < a + an && !(a == g && (r.ld == r.gld || r.rows == 1)))
            return fail(QS_ERR_INVALID, "the gradient overlaps the logits without being their own buffer");
    }
    return QS_OK;
}

static int score(const Rows& r, const float* weights, RowScore* out, float* logprobs, float* stats,
                 cudaStream_t st) {
    if (r.dtype == QS_F32)
        score_rows_kernel<float><<<r.rows, kLossThreads, 0, st>>>((const float*)r.logits, r.vocab, r.ld, r.tokens,
                                                                 weights, r.inv_t, out, logprobs, stats);
    else
        score_rows_kernel<__nv_bfloat16><<<r.rows, kLossThreads, 0, st>>>(
            (const __nv_bfloat16*)r.logits, r.vocab, r.ld, r.tokens, weights, r.inv_t, out, logprobs, stats);
    return check_launch("score_rows_kernel");
}

static int grad(const Rows& r, const float* stats, int stat_words, const float* coefs, cudaStream_t st) {
    if (r.dtype == QS_F32)
        grad_rows_kernel<float><<<r.rows, kLossThreads, 0, st>>>((const float*)r.logits, r.vocab, r.ld, r.tokens,
                                                                stats, stat_words, coefs, r.inv_t, (float*)r.grad,
                                                                r.gld);
    else
        grad_rows_kernel<__nv_bfloat16><<<r.rows, kLossThreads, 0, st>>>(
            (const __nv_bfloat16*)r.logits, r.vocab, r.ld, r.tokens, stats, stat_words, coefs, r.inv_t,
            (__nv_bfloat16*)r.grad, r.gld);
    return check_launch("grad_rows_kernel");
}

static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace qs

using namespace qs;

extern "C" {

int qs_token_logprobs(const void* d_logits, int dtype, int rows, int vocab, long long row_stride,
                      const int* d_tokens, double temperature, float* d_logprobs, float* d_stats,
                      void* stream) {
    set_error(QS_OK, "");
    const Rows r{d_logits, dtype, rows, vocab, row_stride, d_tokens, 1.0 / temperature, nullptr, 0};
    const int rc = check_rows(r, temperature);
    if (rc || rows == 0) return rc;
    if (!d_logprobs || !d_stats) return fail(QS_ERR_INVALID, "NULL output buffer");
    return score(r, nullptr, nullptr, d_logprobs, d_stats, (cudaStream_t)stream);
}

int qs_token_logprobs_backward(const void* d_logits, int dtype, int rows, int vocab, long long row_stride,
                               const int* d_tokens, const float* d_stats, const float* d_grad_logprobs,
                               double temperature, void* d_grad, long long grad_row_stride, void* stream) {
    set_error(QS_OK, "");
    const Rows r{d_logits, dtype, rows, vocab, row_stride, d_tokens, 1.0 / temperature, d_grad, grad_row_stride};
    const int rc = check_rows(r, temperature);
    if (rc || rows == 0) return rc;
    if (!d_stats || !d_grad_logprobs) return fail(QS_ERR_INVALID, "NULL device pointer");
    if (!d_grad) return fail(QS_ERR_INVALID, "NULL output buffer");
    return grad(r, d_stats, 2, d_grad_logprobs, (cudaStream_t)stream);
}

size_t qs_policy_loss_workspace(int rows) {
    const size_t n = rows > 0 ? (size_t)rows : 1;
    return round256(n * sizeof(RowScore)) + round256(n * sizeof(float));
}

int qs_policy_loss(const void* d_logits, int dtype, int rows, int vocab, long long row_stride,
                   const int* d_tokens, const float* d_old_logprobs, const float* d_ref_logprobs,
                   const float* d_advantages, const float* d_weights, const qs_policy_params* params,
                   float* d_loss, float* d_logprobs, void* d_grad, long long grad_row_stride,
                   void* d_workspace, size_t workspace_bytes, void* stream) {
    set_error(QS_OK, "");
    if (!params) return fail(QS_ERR_INVALID, "params is NULL");
    const qs_policy_params p = *params;
    const Rows r{d_logits, dtype, rows, vocab, row_stride, d_tokens, 1.0 / p.temperature, d_grad, grad_row_stride};
    const int rc = check_rows(r, p.temperature);
    if (rc) return rc;
    if (!(p.clip_low >= 0.0 && p.clip_low <= 1.0) || !(p.clip_high >= 0.0) || isinf(p.clip_high))
        return fail(QS_ERR_INVALID, "clip_low %g outside [0, 1] or clip_high %g not a finite number >= 0", p.clip_low, p.clip_high);
    if (!(p.kl_coef >= 0.0) || isinf(p.kl_coef)) return fail(QS_ERR_INVALID, "kl_coef %g is not a finite number >= 0", p.kl_coef);
    if (!d_loss) return fail(QS_ERR_INVALID, "NULL output buffer");
    const cudaStream_t st = (cudaStream_t)stream;
    if (rows > 0) {
        if (!d_old_logprobs || !d_advantages) return fail(QS_ERR_INVALID, "NULL device pointer");
        if (p.kl_coef > 0.0 && !d_ref_logprobs) return fail(QS_ERR_INVALID, "kl_coef %g needs ref_logprobs", p.kl_coef);
        if (!d_workspace || workspace_bytes < qs_policy_loss_workspace(rows) || ((uintptr_t)d_workspace & 15))
            return fail(QS_ERR_INVALID, "workspace is NULL, unaligned or below %zu bytes", qs_policy_loss_workspace(rows));
    }
    RowScore* sc = (RowScore*)d_workspace;
    float* coefs = (float*)((char*)d_workspace + round256((size_t)rows * sizeof(RowScore)));
    if (rows > 0) {
        const int e = score(r, d_weights, sc, d_logprobs, nullptr, st);
        if (e) return e;
    }
    policy_rows_kernel<<<1, 1024, 0, st>>>(sc, rows, d_old_logprobs, d_ref_logprobs, d_advantages, d_weights, p,
                                          coefs, d_loss);
    const int e = check_launch("policy_rows_kernel");
    if (e || rows == 0 || !d_grad) return e;
    return grad(r, &sc->max, sizeof(RowScore) / 4, coefs, st);
}

size_t qs_preference_loss_workspace(int rows, int pairs) {
    (void)pairs;
    const size_t n = rows > 0 ? (size_t)rows : 1;
    return round256(n * sizeof(RowScore)) + round256(n * sizeof(float));
}

int qs_preference_loss(const void* d_logits, int dtype, int rows, int vocab, long long row_stride,
                       const int* d_tokens, const int* d_seq_offsets, int pairs, const float* d_ref_logprobs,
                       const float* d_weights, const qs_preference_params* params, float* d_loss,
                       float* d_seq_logprobs, void* d_grad, long long grad_row_stride, void* d_workspace,
                       size_t workspace_bytes, void* stream) {
    set_error(QS_OK, "");
    if (!params) return fail(QS_ERR_INVALID, "params is NULL");
    const qs_preference_params p = *params;
    const Rows r{d_logits, dtype, rows, vocab, row_stride, d_tokens, 1.0, d_grad, grad_row_stride};
    const int rc = check_rows(r, 1.0);
    if (rc) return rc;
    if (pairs < 0 || pairs > 1 << 27) return fail(QS_ERR_INVALID, "pairs %d outside [0, 2^27]", pairs);
    if (!(p.beta > 0.0) || isinf(p.beta)) return fail(QS_ERR_INVALID, "beta %g is not a finite number > 0", p.beta);
    if (!(p.label_smoothing >= 0.0 && p.label_smoothing < 0.5))
        return fail(QS_ERR_INVALID, "label_smoothing %g outside [0, 0.5)", p.label_smoothing);
    if (!d_loss) return fail(QS_ERR_INVALID, "NULL output buffer");
    if (pairs > 0 && (!d_seq_offsets || !d_ref_logprobs)) return fail(QS_ERR_INVALID, "NULL device pointer");
    if (rows > 0 && (!d_workspace || workspace_bytes < qs_preference_loss_workspace(rows, pairs) || ((uintptr_t)d_workspace & 15)))
        return fail(QS_ERR_INVALID, "workspace is NULL, unaligned or below %zu bytes", qs_preference_loss_workspace(rows, pairs));
    const cudaStream_t st = (cudaStream_t)stream;
    RowScore* sc = (RowScore*)d_workspace;
    float* coefs = (float*)((char*)d_workspace + round256((size_t)rows * sizeof(RowScore)));
    if (rows > 0) {
        const int e = score(r, nullptr, sc, nullptr, nullptr, st);
        if (e) return e;
    }
    preference_pairs_kernel<<<1, 1024, 0, st>>>(sc, rows, d_seq_offsets, pairs, d_ref_logprobs, d_weights, p, coefs,
                                               d_seq_logprobs, d_loss);
    const int e = check_launch("preference_pairs_kernel");
    if (e || rows == 0 || !d_grad) return e;
    return grad(r, &sc->max, sizeof(RowScore) / 4, coefs, st);
}

}  // extern "C"
