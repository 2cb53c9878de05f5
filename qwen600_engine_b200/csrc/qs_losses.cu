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

#include <atomic>
#include <type_traits>

#include "qs_common.cuh"
#include "qs_f32x2.cuh"
#include "qs_pipe.cuh"
#include "qwen600_sampler.h"

namespace qs {

int set_error(int code, const char* msg);  // qs_api.cu

// What a scored row leaves for the losses and the gradient.
struct RowScore {
    double logprob;  // 0 for a row that scores nothing
    float max;
    float excess;
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

__device__ __forceinline__ f32x2 exp2_pair(f32x2 v) {
    const float2 t = unpair2(v);
    return pair2(exp2_fast(t.x), exp2_fast(t.y));
}

// A term 2^((x - ref) scale) in one multiply-add is 2^(x scale - bias), bias
// the rounded ref * scale; every term is then 2^slip too large, slip being what
// the rounding took, and 2^-slip sets a sum of them right.  Below 2^24 slip is
// at most 1/2.  It grows with bias: from 2^31 on it can pass 128, and 2^slip
// and 2^-slip are inf and 0, their product NaN (logits masked with -1e10 or
// -1e30).  Larger values subtract before they scale.
__device__ __forceinline__ bool one_step(float bias) { return fabsf(bias) < 16777216.0f; }

// Block-wide sum of one double per thread, in a fixed order; in warp 0.
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x >= 32) return 0.0;
    v = threadIdx.x < blockDim.x >> 5 ? red[threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Vectors of 16 bytes of a row, at any alignment of its first element: up to
// kN - 1 elements before the first aligned vector (head), whole vectors, up to
// kN - 1 elements behind the last (tail).
template <typename T>
struct RowShape {
    static constexpr int kN = 16 / (int)sizeof(T);
    int head, vecs, tail;
    __device__ __forceinline__ RowShape(const T* row, int V) {
        head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
        vecs = (V - head) / kN;
        tail = V - head - vecs * kN;
    }
    // The element outside the vectors that thread t of a row's first CTA takes, or -1.
    __device__ __forceinline__ int edge(int t, int V) const {
        return t < head ? t : t >= 8 && t < 8 + tail ? V - tail + t - 8 : -1;
    }
};

// Plain (coherent) loads that do not stay in L1: the same kernel may write the
// gradient over the logits, so the read-only path is not used.
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p)
                 : "memory");
    return v;
}
__device__ __forceinline__ void store16(void* p, const uint4& v) {
    asm volatile("st.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}

// The same for data that should not push others out of L2.
__device__ __forceinline__ void store16_past(void* p, const uint4& v) {
    asm volatile("st.global.cs.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}

// 16 bytes of logits as floats and back.
template <typename T>
struct Pack;
template <>
struct Pack<float> {
    static constexpr int kN = 4;
    __device__ __forceinline__ static uint4 lowest() {
        return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);
    }
    __device__ __forceinline__ static void widen(const uint4& v, float* o) {
        o[0] = __uint_as_float(v.x); o[1] = __uint_as_float(v.y);
        o[2] = __uint_as_float(v.z); o[3] = __uint_as_float(v.w);
    }
    __device__ __forceinline__ static void widen_word(uint32_t w, float* o) { o[0] = __uint_as_float(w); }
    __device__ __forceinline__ static uint4 narrow(const float* o) {
        return make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
    }
    __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
};
template <>
struct Pack<__nv_bfloat16> {
    static constexpr int kN = 8;
    __device__ __forceinline__ static uint4 lowest() {
        return make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u);
    }
    __device__ __forceinline__ static void widen_word(uint32_t w, float* o) {
        o[0] = __uint_as_float(w << 16);
        o[1] = __uint_as_float(w & 0xFFFF0000u);
    }
    __device__ __forceinline__ static void widen(const uint4& v, float* o) {
        widen_word(v.x, o);
        widen_word(v.y, o + 2);
        widen_word(v.z, o + 4);
        widen_word(v.w, o + 6);
    }
    __device__ __forceinline__ static uint4 narrow(const float* o) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
        const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                         *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

__device__ __forceinline__ void cluster_arrive_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive_release() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// One CTA's part of a row: its maximum, how many elements equal it, and the
// sum of the others' exponentials against it.
struct __align__(16) Part {
    float max;
    int at_max;
    double others;
};

// Writes p to *slot of the cluster's CTA `rank`.
__device__ __forceinline__ void push_part(Part* slot, int rank, const Part& p) {
    uint32_t addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(addr)
                 : "r"((uint32_t)__cvta_generic_to_shared(slot)), "r"(rank));
    const unsigned long long o = (unsigned long long)__double_as_longlong(p.others);
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(__float_as_uint(p.max)),
                 "r"((uint32_t)p.at_max), "r"((uint32_t)o), "r"((uint32_t)(o >> 32))
                 : "memory");
}

// Per-row term of the policy loss: returns l, and its slope dl / dlogprob.
__device__ __forceinline__ double policy_term(double lp, double old_lp, double ref_lp, double adv, double lo,
                                              double hi, double kl, double* slope) {
    const double r = exp(lp - old_lp);
    const bool cut = (adv > 0.0 && r > hi) || (adv < 0.0 && r < lo);
    double l = -(cut ? (r > hi ? hi : lo) : r) * adv;
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

// 1 - p of the target xt, without cancellation where it is the maximum.
__device__ __forceinline__ double beyond(float xt, float max, double excess, double inv_t) {
    return xt == max ? excess / (1.0 + excess) : 1.0 - exp(((double)xt - (double)max) * inv_t) / (1.0 + excess);
}

constexpr int kScoreThreads = 256;                        // at most, in a CTA
constexpr unsigned long long kLoadWaitNs = 2000000000ull;  // a copy that has not landed by then: NaN in the results

template <typename T>
struct ScoreArgs {
    const T* logits;
    int rows, V;
    long long ld;
    const int* tokens;
    float scale;  // log2(e) / T
    double inv_t;
    int log_c;    // 1 << log_c CTAs per row, one cluster
    RowScore* out;
    float* coefs;  // with out: set to 0
    float* logprobs;
    float* stats;
    // the policy loss
    const float* weights;
    const float* old_lp;
    const float* ref_lp;
    const float* adv;
    qs_policy_params p;
    double* row_loss;
    T* grad;
    long long gld;
};

// Scores one row per cluster of 1 to 8 CTAs; with kPolicy it also forms the
// row's policy loss and writes its gradient.  Each CTA brings a contiguous
// share of the row's 16-byte vectors to shared memory with one bulk copy.  So
// the row is read from memory once, its maximum is known before the first
// exponential (no sum is rescaled), and the gradient is formed from the same
// copy.  The CTAs exchange their parts, 16 bytes each, through distributed
// shared memory.
//
// Bound: memory, as long as enough rows are under way: from its copy to its
// last store a CTA of 38 KB (a bf16 row of 151,936 over 8) takes about 10 us
// with its neighbours, so an SM needs some 200 KB in flight.  Shared memory
// holds five such CTAs, 226 us for 2048 bf16 rows of 151,936 a quarter of which
// is left out (1089 MB, 4.8 TB/s); with the shares in registers (80 a thread of
// 256) it were three, 293 us.  Without the exchange it would take 207 us,
// without the exponentials 216.  Shares of 76 KB on 4 CTAs: 224 us; of 19 KB on
// 16: 282.
template <typename T, bool kPolicy>
__global__ void __launch_bounds__(kScoreThreads)
score_kernel(const __grid_constant__ ScoreArgs<T> a) {
    constexpr int kN = Pack<T>::kN;
    constexpr int kW = kScoreThreads / 32;
    extern __shared__ __align__(16) uint4 vecs[];
    __shared__ Part parts[8];
    __shared__ float red_max[kW], red_sum[kW];
    __shared__ int red_n[kW];
    __shared__ float factor_s, max_s, target_s;
    __shared__ unsigned long long loaded;
    __shared__ int gave_up;
    const int t = threadIdx.x, thr = blockDim.x, C = 1 << a.log_c;
    const int row = blockIdx.x >> a.log_c, rank = blockIdx.x & (C - 1);
    const int tok = a.tokens[row];
    const bool scored = tok >= 0 && tok < a.V && !(kPolicy && a.weights && a.weights[row] == 0.0f);
    const T* x = a.logits + (size_t)row * a.ld;
    T* g = kPolicy && a.grad ? a.grad + (size_t)row * a.gld : nullptr;
    dependents_may_start();
    if (!scored) {  // alike for the whole cluster
        if (rank == 0 && t == 0) {
            if (a.out) {
                a.out[row] = RowScore{0.0, 0.0f, 0.0f};
                a.coefs[row] = 0.0f;
            }
            if (a.logprobs) a.logprobs[row] = 0.0f;
            if (a.stats) a.stats[2 * (size_t)row] = a.stats[2 * (size_t)row + 1] = 0.0f;
            if (kPolicy) a.row_loss[row] = 0.0;
        }
        if (kPolicy && g) {
            const RowShape<T> gs(g, a.V);
            for (int i = rank * thr + t; i < gs.vecs; i += C * thr)
                store16(g + gs.head + (size_t)i * kN, make_uint4(0u, 0u, 0u, 0u));
            const int e = rank == 0 ? gs.edge(t, a.V) : -1;
            if (e >= 0) put(g, e, 0.0f);
        }
        return;
    }

    const RowShape<T> sh(x, a.V);
    const int per = (sh.vecs + C - 1) >> a.log_c;
    const int first = min(rank * per, sh.vecs), cnt = min(per, sh.vecs - first);
    if (t == 0) {
        gave_up = 0;
        mbar_init(&loaded, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_expect_tx(&loaded, (uint32_t)cnt * 16u);
        if (cnt > 0)
            asm volatile(
                "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                    smem_u32(vecs)),
                "l"(x + sh.head + (size_t)first * kN), "r"((uint32_t)cnt * 16u), "r"(smem_u32(&loaded))
                : "memory");
    }
    if (C > 1) cluster_arrive_relaxed();  // waited for before the first store into another CTA
    // what the row's term takes, requested before anything waits
    float w_row = 0.0f, old_lp = 0.0f, ref_lp = 0.0f, adv = 0.0f;
    if (kPolicy && t == 0) {
        if (a.weights) w_row = a.weights[row];
        old_lp = a.old_lp[row];
        adv = a.adv[row];
        if (a.p.kl_coef > 0.0) ref_lp = a.ref_lp[row];
    }
    const int edge = rank == 0 ? sh.edge(t, a.V) : -1;
    const float xe = edge >= 0 ? elem(x, edge) : -INFINITY;
    const float xt = elem(x, tok);
    __syncthreads();
    if (!mbar_wait(&loaded, 0, &gave_up, kLoadWaitNs))
        mbar_wait(&loaded, 0, &gave_up, kLoadWaitNs, false);  // the copy lands before the CTA leaves

    // the maximum of this CTA's part
    float own_max = xe;
    {
        uint4 u = Pack<T>::lowest();
#pragma unroll 4
        for (int k = t; k < cnt; k += thr) {
            const uint4 v = vecs[k];
            u.x = Pack<T>::max2(u.x, v.x);
            u.y = Pack<T>::max2(u.y, v.y);
            u.z = Pack<T>::max2(u.z, v.z);
            u.w = Pack<T>::max2(u.w, v.w);
        }
        float o[kN];
        Pack<T>::widen(u, o);
#pragma unroll
        for (int j = 0; j < kN; j++) own_max = fmaxf(own_max, o[j]);
    }
    float m = warp_max(own_max);
    if ((t & 31) == 0) red_max[t >> 5] = m;
    __syncthreads();
    m = red_max[0];
    for (int w = 1; w < thr / 32; w++) m = fmaxf(m, red_max[w]);
    const float ref = m == -INFINITY ? 0.0f : m;

    // The sum of exponentials against it.  The maximum's own terms (exactly 1
    // each) are counted apart, by the warps that hold one; they also subtract
    // before they scale.  The others scale and subtract in one instruction
    // where one_step allows it.
    const float bias = ref * a.scale;
    const bool apart = __any_sync(0xffffffffu, own_max == ref) || !one_step(bias);
    float s = 0.0f;
    int n = 0;
    if (apart) {
#pragma unroll 2
        for (int k = t; k < cnt; k += thr) {
            float o[kN];
            Pack<T>::widen(vecs[k], o);
#pragma unroll
            for (int j = 0; j < kN; j++) {
                const float d = o[j] - ref;
                const float e = exp2_fast(d * a.scale);
                n += d == 0.0f;
                s += d == 0.0f ? 0.0f : e;
            }
        }
        const float d = xe - ref;
        n += d == 0.0f;
        s += d == 0.0f ? 0.0f : exp2_fast(d * a.scale);
        n = warp_sum_int(n);
    } else {
        const f32x2 scale2 = pair2(a.scale, a.scale), bias2 = pair2(-bias, -bias);
        f32x2 s2 = pair2(exp2_fast(__fmaf_rn(xe, a.scale, -bias)), 0.0f);
#pragma unroll 2
        for (int k = t; k < cnt; k += thr) {
            float o[kN];
            Pack<T>::widen(vecs[k], o);
#pragma unroll
            for (int j = 0; j < kN; j += 2) s2 = add2(s2, exp2_pair(fma2(pair2(o[j], o[j + 1]), scale2, bias2)));
        }
        const float2 u = unpair2(s2);
        const float slip = __fmaf_rn(ref, a.scale, -bias);
        s = (u.x + u.y) * exp2_fast(-slip);
    }
    s = warp_sum(s);
    if ((t & 31) == 0) {
        red_sum[t >> 5] = s;
        red_n[t >> 5] = n;
    }
    __syncthreads();
    if (C > 1) cluster_wait();  // every CTA of the cluster runs
    if (t < C) {
        Part p{m, 0, *(volatile int*)&gave_up ? (double)NAN : 0.0};
        for (int w = 0; w < thr / 32; w++) {
            p.others += (double)red_sum[w];
            p.at_max += red_n[w];
        }
        if (C > 1) push_part(&parts[rank], t, p);
        else parts[0] = p;
    }
    if (C > 1) {  // only the warp that stored into the others has stores to release
        if (t < 32) cluster_arrive_release();
        else cluster_arrive_relaxed();
        cluster_wait();
    }
    if (!kPolicy && rank != 0) return;
    if (t < 32) {
        __syncwarp();
        const Part p = t < C ? parts[t] : Part{-INFINITY, 0, 0.0};
        const float M = warp_max(p.max);
        const bool top = p.max == M;
        int at_max = top ? p.at_max : 0;
        double others = top ? p.others : t < C ? (double)exp2_fast((p.max - M) * a.scale) * (p.others + p.at_max) : 0.0;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            others += __shfl_xor_sync(0xffffffffu, others, o);
            at_max += __shfl_xor_sync(0xffffffffu, at_max, o);
        }
        if (t == 0) {
            const double excess = isinf(M) ? (double)NAN : others + (double)(at_max - 1);
            const double lp = ((double)xt - (double)M) * a.inv_t - log1p(excess);
            if (rank == 0) {
                if (a.out) {
                    a.out[row] = RowScore{lp, M, (float)excess};
                    a.coefs[row] = 0.0f;
                }
                if (a.logprobs) a.logprobs[row] = (float)lp;
                if (a.stats) {
                    a.stats[2 * (size_t)row] = M;
                    a.stats[2 * (size_t)row + 1] = (float)excess;
                }
            }
            if (kPolicy) {
                const double w = a.weights ? (double)w_row : 1.0 / a.rows;
                double slope;
                const double l = policy_term(lp, old_lp, ref_lp, adv, 1.0 - a.p.clip_low, 1.0 + a.p.clip_high,
                                             a.p.kl_coef, &slope);
                if (rank == 0) a.row_loss[row] = w * l;
                const double c = w * slope * a.inv_t;
                factor_s = (float)(-c / (1.0 + excess));
                target_s = c == 0.0 ? 0.0f : (float)(c * beyond(xt, M, excess, a.inv_t));
                max_s = M;
            }
        }
    }
    if (!kPolicy || !g) return;
    __syncthreads();
    float f = factor_s;
    const float M = max_s, top = M * a.scale;
    const bool plain = one_step(top);
    if (plain) f *= exp2_fast(-__fmaf_rn(M, a.scale, -top));
    const auto grad_of = [&](float v) {
        return f == 0.0f ? 0.0f : f * exp2_fast(plain ? __fmaf_rn(v, a.scale, -top) : (v - M) * a.scale);
    };
    const f32x2 f2 = pair2(f, f), scale2 = pair2(a.scale, a.scale), top2 = pair2(-top, -top);
    const bool aligned = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
    T* gbody = g + sh.head + (size_t)first * kN;
#pragma unroll 2
    for (int k = t; k < cnt; k += thr) {
        float o[kN];
        Pack<T>::widen(vecs[k], o);
        if (plain && f != 0.0f) {
#pragma unroll
            for (int j = 0; j < kN; j += 2) {
                const float2 r = unpair2(mul2(f2, exp2_pair(fma2(pair2(o[j], o[j + 1]), scale2, top2))));
                o[j] = r.x;
                o[j + 1] = r.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < kN; j++) o[j] = grad_of(o[j]);
        }
        if (aligned) {
            store16(gbody + (size_t)k * kN, Pack<T>::narrow(o));
        } else {
#pragma unroll
            for (int j = 0; j < kN; j++) put(gbody, (long long)k * kN + j, o[j]);
        }
    }
    if (edge >= 0 && edge != tok) put(g, edge, grad_of(xe));
    // the target, by the thread that wrote its vector
    const int at = tok - sh.head;
    if (at < 0 || at >= sh.vecs * kN) {
        if (edge == tok) put(g, tok, target_s);
    } else {
        const int k = at / kN - first;
        if (k >= 0 && k < cnt && k % thr == t) put(g, tok, target_s);
    }
}

// ------------------------------------------------- scoring many rows
// Without a gradient a row need not stay on the chip, and a call of many rows
// is a stream: rows are cut into units of 256 vectors (4 KB), every warp of a
// persistent grid takes units in turn through its own ring of bulk copies and
// leaves each unit's maximum and sums, and a second kernel joins a row's units.
// The maximum's own term is left out of the fp32 sum as in score_kernel: where
// one lane holds the maximum, the warp takes that lane's 128 bytes once more,
// two elements a lane.  (Where several do, the row's sum is at least 2, and the
// 1 costs it less than the exponentials do.)  Warps never wait for one another,
// so copies keep running while others compute.  1024 bf16 rows of 151,936: 61 us
// (52 of them this kernel, 6.0 TB/s, its exponentials at 75% of the unit's
// rate), 78 with a cluster per row.  24 warps with rings of 2 units; 16 with 3
// were 16 us slower.
constexpr int kUnitVecs = 256;
constexpr int kStreamWarps = 24;
constexpr int kStreamStages = 2;

template <typename T>
struct StreamArgs {
    const T* logits;
    int rows, V;
    long long ld;
    const int* tokens;
    float scale;
    double inv_t;
    int units;     // per row
    float4* parts; // [rows][units]: maximum, sum of exponentials against it, how many 1s were left out of it
    RowScore* out;
    float* coefs;  // with out: set to 0
    float* logprobs;
    float* stats;
};

// Where a warp is in its units: it takes every stride-th one.
struct UnitAt {
    int row, unit;
    __device__ __forceinline__ void step(int rows, int units, int units_per_row) {
        row += rows;
        unit += units;
        if (unit >= units_per_row) {
            unit -= units_per_row;
            row++;
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(kStreamWarps * 32, 1)
stream_kernel(const __grid_constant__ StreamArgs<T> a) {
    constexpr int kN = Pack<T>::kN;
    extern __shared__ __align__(128) uint4 ring[];  // [warp][stage][kUnitVecs]
    __shared__ unsigned long long full[kStreamWarps][kStreamStages];
    __shared__ int gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint4* mine = ring + (size_t)warp * kStreamStages * kUnitVecs;
    if (threadIdx.x == 0) gave_up = 0;
    if (lane == 0) {
        for (int i = 0; i < kStreamStages; i++) mbar_init(&full[warp][i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    dependents_may_start();

    const long long stride = (long long)gridDim.x * kStreamWarps, begin = (long long)warp * gridDim.x + blockIdx.x;
    const int dr = (int)(stride / a.units), du = (int)(stride % a.units);
    UnitAt now{(int)(begin / a.units), (int)(begin % a.units)}, ahead = now;
    const auto scored = [&](int row) {
        if (row >= a.rows) return false;
        const int tok = a.tokens[row];
        return tok >= 0 && tok < a.V;
    };
    const auto request = [&](const UnitAt& u, int stage) {
        if (lane == 0) {
            const T* x = a.logits + (size_t)u.row * a.ld;
            const RowShape<T> sh(x, a.V);
            const int first = u.unit * kUnitVecs, cnt = max(0, min(kUnitVecs, sh.vecs - first));
            mbar_expect_tx(&full[warp][stage], (uint32_t)cnt * 16u);
            if (cnt > 0)
                asm volatile(
                    "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                        smem_u32(mine + stage * kUnitVecs)),
                    "l"(x + sh.head + (size_t)first * kN), "r"((uint32_t)cnt * 16u), "r"(smem_u32(&full[warp][stage]))
                    : "memory");
        }
    };
    uint32_t live = 0;    // stages with a copy under way
    uint32_t phases = 0;  // the parity each stage's next copy completes
#pragma unroll
    for (int i = 0; i < kStreamStages; i++) {
        if (scored(ahead.row)) {
            request(ahead, i);
            live |= 1u << i;
        }
        ahead.step(dr, du, a.units);
    }
    bool next = scored(ahead.row);  // looked up one unit before it is asked for
    bool dead = false;
    for (int stage = 0; now.row < a.rows; stage = stage + 1 == kStreamStages ? 0 : stage + 1) {
        if (live >> stage & 1) {
            const bool landed = !dead && mbar_wait(&full[warp][stage], phases >> stage & 1, &gave_up, kLoadWaitNs);
            if (!landed) {
                mbar_wait(&full[warp][stage], phases >> stage & 1, &gave_up, kLoadWaitNs, false);
                dead = true;
            }
            phases ^= 1u << stage;
            const T* x = a.logits + (size_t)now.row * a.ld;
            const RowShape<T> sh(x, a.V);
            const int cnt = max(0, min(kUnitVecs, sh.vecs - now.unit * kUnitVecs));
            const int edge = now.unit == 0 ? sh.edge(lane, a.V) : -1;
            const float xe = edge >= 0 ? elem(x, edge) : -INFINITY;
            uint4 v[kUnitVecs / 32];
            uint4 u = Pack<T>::lowest();
#pragma unroll
            for (int i = 0; i < kUnitVecs / 32; i++) {
                const int k = i * 32 + lane;
                v[i] = k < cnt ? mine[stage * kUnitVecs + k] : Pack<T>::lowest();
                u.x = Pack<T>::max2(u.x, v[i].x);
                u.y = Pack<T>::max2(u.y, v[i].y);
                u.z = Pack<T>::max2(u.z, v[i].z);
                u.w = Pack<T>::max2(u.w, v[i].w);
            }
            float o[kN];
            Pack<T>::widen(u, o);
            float own = xe;
#pragma unroll
            for (int j = 0; j < kN; j++) own = fmaxf(own, o[j]);
            const float m = warp_max(own);
            const uint32_t holders = __ballot_sync(0xffffffffu, own == m);
            const bool one = (holders & (holders - 1)) == 0;
            const int holder = __ffs(holders) - 1;
            float again = 0.0f;  // this lane's share of the holder's elements
            int at_max = 0;
            if (one) {
                const int k = (lane >> 2) * 32 + holder;
                const uint32_t word = k < cnt ? reinterpret_cast<const uint32_t*>(mine + stage * kUnitVecs + k)[lane & 3]
                                              : Pack<T>::lowest().x;
                float e[kN / 4];
                Pack<T>::widen_word(word, e);
#pragma unroll
                for (int j = 0; j < kN / 4; j++) {
                    const float d = e[j] - m;
                    at_max += __popc(__ballot_sync(0xffffffffu, d == 0.0f));
                    again += d == 0.0f ? 0.0f : exp2_fast(d * a.scale);
                }
            }
            __syncwarp();  // every lane has read the stage
            live &= ~(1u << stage);
            if (next && !dead) {
                request(ahead, stage);
                live |= 1u << stage;
            }
            const float ref = m == -INFINITY ? 0.0f : m;
            const float bias = ref * a.scale;
            float s;
            if (one_step(bias)) {
                const f32x2 scale2 = pair2(a.scale, a.scale), bias2 = pair2(-bias, -bias);
                f32x2 s2 = pair2(exp2_fast(__fmaf_rn(xe, a.scale, -bias)), 0.0f);
#pragma unroll
                for (int i = 0; i < kUnitVecs / 32; i++) {
                    Pack<T>::widen(v[i], o);
#pragma unroll
                    for (int j = 0; j < kN; j += 2) s2 = add2(s2, exp2_pair(fma2(pair2(o[j], o[j + 1]), scale2, bias2)));
                }
                const float2 r = unpair2(s2);
                s = (r.x + r.y) * exp2_fast(-__fmaf_rn(ref, a.scale, -bias));
            } else {  // 1024 bf16 rows of 151,936, nearly all of -1e30: 86 us; shorter with packed operations, but
                      // their code costs ordinary rows 1% and more
                s = exp2_fast((xe - ref) * a.scale);
#pragma unroll 1
                for (int i = 0; i < kUnitVecs / 32; i++) {
                    uint4 w = v[0];
#pragma unroll
                    for (int k = 1; k < kUnitVecs / 32; k++)
                        if (k == i) w = v[k];
                    Pack<T>::widen(w, o);
                    for (int j = 0; j < kN; j++) s += exp2_fast((o[j] - ref) * a.scale);
                }
            }
            if (one) {
                const float held = __shfl_sync(0xffffffffu, xe, holder) - m;  // the holder's element outside the vectors
                at_max += held == 0.0f;
                if (lane == holder) s = held == 0.0f ? 0.0f : exp2_fast(held * a.scale);
                s += again;
            }
            s = warp_sum(s);
            if (lane == 0)
                a.parts[(size_t)now.row * a.units + now.unit] = make_float4(m, dead ? NAN : s, (float)at_max, 0.0f);
        } else {
            if (lane == 0 && dead) a.parts[(size_t)now.row * a.units + now.unit] = make_float4(0.0f, NAN, 0.0f, 0.0f);
            if (next && !dead) {
                request(ahead, stage);
                live |= 1u << stage;
            }
        }
        now.step(dr, du, a.units);
        ahead.step(dr, du, a.units);
        next = scored(ahead.row);
    }
}

// Joins a row's units, one warp a row.
constexpr int kJoinRows = 4;                                    // a CTA: small enough to start beside the stream
constexpr int kMaxUnits = kMaxVocab / 4 / kUnitVecs;            // of a row
static_assert(kMaxUnits % 32 == 0, "units of a lane");

template <typename T>
__global__ void __launch_bounds__(kJoinRows * 32)
join_kernel(const __grid_constant__ StreamArgs<T> a) {
    constexpr int kMine = kMaxUnits / 32;
    const int row = blockIdx.x * kJoinRows + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    dependents_may_start();
    const int tok = row < a.rows ? a.tokens[row] : -1;
    const bool scored = tok >= 0 && tok < a.V;
    const T* x = a.logits + (size_t)row * a.ld;
    const float xt = scored ? elem(x, tok) : 0.0f;
    wait_for_previous();
    if (row >= a.rows) return;
    RowScore r{0.0, 0.0f, 0.0f};
    if (scored) {
        const float4* all = a.parts + (size_t)row * a.units;
        float4 p[kMine];
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            p[i] = i * 32 + lane < a.units ? all[i * 32 + lane] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
            M = fmaxf(M, p[i].x);
        }
        M = warp_max(M);
        double others = 0.0;
        int at_max = 0;
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            if (i * 32 + lane >= a.units) break;
            if (p[i].x == M) {
                others += (double)p[i].y;
                at_max += (int)p[i].z;
            } else {
                others += (double)(exp2_fast((p[i].x - M) * a.scale) * (p[i].y + p[i].z));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) others += __shfl_xor_sync(0xffffffffu, others, o);
        double excess = others + (double)(warp_sum_int(at_max) - 1);
        if (isinf(M)) excess = NAN;
        r.max = M;
        r.excess = (float)excess;
        if (lane == 0) r.logprob = ((double)xt - (double)M) * a.inv_t - log1p(excess);
    }
    if (lane == 0) {
        if (a.out) {
            a.out[row] = r;
            a.coefs[row] = 0.0f;
        }
        if (a.logprobs) a.logprobs[row] = (float)r.logprob;
        if (a.stats) {
            a.stats[2 * (size_t)row] = r.max;
            a.stats[2 * (size_t)row + 1] = r.excess;
        }
    }
}

// grad = coef * ([j = t] - p_j) / T.  Rows are cut into pieces of kGradThreads
// x kGradVpt vectors, one CTA each.  Rows are taken from the last to the
// first: the scoring before read them in the other order, so the ones it read
// last come from L2; the gradient is stored past it (241 to 228 us for 1900
// rows of 151,936 bf16, 20.5 to 18.8 us for 509 of 50,021).
constexpr int kGradThreads = 256;
constexpr int kGradVpt = 6;

template <typename T>
__global__ void __launch_bounds__(kGradThreads)
grad_kernel(const T* logits, int rows, int V, long long ld, const int* __restrict__ tokens, const float* stats,
            int stat_words, const float* coefs, float scale, double inv_t, T* grad, long long gld, int pieces) {
    constexpr int kN = Pack<T>::kN;
    const int t = threadIdx.x;
    const int row = rows - 1 - (int)(blockIdx.x / (unsigned)pieces), piece = blockIdx.x % (unsigned)pieces;
    const int tok = tokens[row];
    const T* x = logits + (size_t)row * ld;
    T* g = grad + (size_t)row * gld;
    const RowShape<T> sh(x, V);
    const int base = piece * kGradThreads * kGradVpt, end = min(base + kGradThreads * kGradVpt, sh.vecs);
    const T* body = x + sh.head;
    const bool scored = tok >= 0 && tok < V;
    wait_for_previous();
    const float coef = scored ? coefs[row] : 0.0f;
    if (coef == 0.0f) {
        const RowShape<T> gs(g, V);
        for (int k = piece * kGradThreads + t; k < gs.vecs; k += pieces * kGradThreads)
            store16_past(g + gs.head + (size_t)k * kN, make_uint4(0u, 0u, 0u, 0u));
        const int e = piece == 0 ? gs.edge(t, V) : -1;
        if (e >= 0) put(g, e, 0.0f);
        return;
    }
    uint4 v[kGradVpt];
#pragma unroll
    for (int i = 0; i < kGradVpt; i++) {
        const int k = base + i * kGradThreads + t;
        v[i] = k < end ? load16(body + (size_t)k * kN) : Pack<T>::lowest();
    }
    const float* st = stats + (size_t)row * stat_words;
    const float M = st[0];
    const double excess = st[1], c = (double)coef * inv_t;
    const float f = (float)-c / (float)(1.0 + excess);
    const bool aligned = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
    T* gbody = g + sh.head;
    const int edge = piece == 0 ? sh.edge(t, V) : -1;
    const float xe = edge >= 0 ? elem(x, edge) : 0.0f;
    // the target's thread: it reads the target before anything of it is overwritten
    const int at = tok - sh.head, kt = at / kN - base;
    const bool mine = at < 0 || at >= sh.vecs * kN ? edge == tok
                                                   : kt >= 0 && kt < end - base && kt % kGradThreads == t;
    const float target = mine ? (float)(c * beyond(elem(x, tok), M, excess, inv_t)) : 0.0f;
#pragma unroll
    for (int i = 0; i < kGradVpt; i++) {
        const int k = base + i * kGradThreads + t;
        float o[kN];
        Pack<T>::widen(v[i], o);
#pragma unroll
        for (int j = 0; j < kN; j++) o[j] = f * exp2_fast((o[j] - M) * scale);
        if (k < end) {
            if (aligned) {
                store16_past(gbody + (size_t)k * kN, Pack<T>::narrow(o));
            } else {
#pragma unroll
                for (int j = 0; j < kN; j++) put(gbody, (long long)k * kN + j, o[j]);
            }
        }
    }
    if (edge >= 0) put(g, edge, f * exp2_fast((xe - M) * scale));
    if (mine) put(g, tok, target);
}

// The policy loss: the rows' terms, added in a fixed order.
__global__ void __launch_bounds__(1024)
sum_rows_kernel(const double* row_loss, int rows, float* __restrict__ loss) {
    __shared__ double red[32];
    wait_for_previous();
    double sum = 0.0;
    for (int i = threadIdx.x; i < rows; i += blockDim.x) sum += row_loss[i];
    sum = block_sum(sum, red);
    if (threadIdx.x == 0) *loss = (float)sum;
}

// One warp per pair in turn: the two sequences' sums, the pair's loss and the
// coefficients of their rows' gradients (0 so far).  Sequences share no row
// unless an offset falls somewhere: then none counts, so that no two warps write
// a row's coefficient.
__global__ void __launch_bounds__(1024)
preference_pairs_kernel(const RowScore* score, int rows, const int* __restrict__ offsets, int pairs,
                        const float* __restrict__ ref, const float* __restrict__ weights,
                        qs_preference_params p, float* __restrict__ coefs, float* __restrict__ seq_lp,
                        float* __restrict__ loss) {
    __shared__ double red[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    dependents_may_start();
    int falls = 0;  // looked for while the rows are scored
    for (int q = threadIdx.x; q < 2 * pairs; q += blockDim.x) falls |= offsets[q] > offsets[q + 1];
    const bool ordered = !__syncthreads_or(falls);
    wait_for_previous();
    double sum = 0.0;
    for (int q = warp; q < pairs; q += blockDim.x >> 5) {
        const int a[2] = {offsets[q], offsets[pairs + q]}, b[2] = {offsets[q + 1], offsets[pairs + q + 1]};
        const bool fine = ordered && a[0] >= 0 && b[0] <= rows && a[1] >= 0 && b[1] <= rows;
        double s[2] = {NAN, NAN};
        if (fine) {
            s[0] = s[1] = 0.0;
            // both sequences at once, four rows of each under way
            for (int i = lane; i < max(b[0] - a[0], b[1] - a[1]); i += 128) {
                double v[2][4];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        v[k][j] = i + j * 32 < b[k] - a[k] ? score[a[k] + i + j * 32].logprob : 0.0;
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[k] += v[k][j];
            }
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
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

static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

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

static int check_workspace(const void* p, size_t bytes, size_t need) {
    if (need == 0 || (p && bytes >= need && ((uintptr_t)p & 15) == 0)) return QS_OK;
    return fail(QS_ERR_INVALID, "workspace is NULL, unaligned or below %zu bytes", need);
}

static int check_rows(const Rows& r, double temperature) {
    if (r.dtype != QS_F32 && r.dtype != QS_BF16) return fail(QS_ERR_INVALID, "unknown dtype %d", r.dtype);
    if (r.rows < 0) return fail(QS_ERR_INVALID, "rows %d < 0", r.rows);
    if (r.rows > 1 << 27) return fail(QS_ERR_UNSUPPORTED, "rows %d above 2^27", r.rows);
    if (r.vocab < 1 || r.vocab > kMaxVocab)
        return fail(QS_ERR_UNSUPPORTED, "vocab %d outside [1, %d]", r.vocab, kMaxVocab);
    if (!(temperature >= 1e-6 && temperature <= 1e6))
        return fail(QS_ERR_INVALID, "temperature %g outside [1e-6, 1e6]", temperature);
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

// Lets a kernel use `bytes` of dynamic shared memory, once on each device.
struct DeviceOnce {
    std::atomic<unsigned long long> done{0};
    int raise(const void* kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e == cudaSuccess && (dev >= 64 || !(done.load() >> dev & 1))) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev);
        }
        return e == cudaSuccess ? QS_OK : fail(QS_ERR_CUDA, "shared memory: %s", cudaGetErrorString(e));
    }
};

// Launches `kernel` in clusters of `cluster` CTAs; `after`: it may start while
// the kernel before it ends (it waits for it before it reads its results).
template <typename... P, typename... A>
static int launch(const char* name, void (*kernel)(P...), long long grid, int threads, int cluster, size_t smem,
                  bool after, cudaStream_t st, A... args) {
    if (grid > 0x7FFFFFFFll) return fail(QS_ERR_UNSUPPORTED, "%s: %lld CTAs", name, grid);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2] = {};
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        cfg.numAttrs++;
    }
    if (after) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs++;
    }
    cfg.attrs = attr;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    if (e == cudaSuccess) return QS_OK;
    return fail(QS_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

// How a row is spread: CTAs per row (a power of two up to 8), doubled while a
// share is above 40 KB, and while the rows alone would leave some of the 148 SMs
// idle and a share keeps 4 KB.  Rows above 320 KB keep 8 with larger shares, up
// to 128 KB: fp32 rows of 151,936 (76 KB, two CTAs an SM) take 240 us for 1024
// rows of the policy loss with its gradient (5.2 TB/s), those of 262,144 have
// one CTA an SM.
template <typename T, bool kPolicy>
static int score_launch(ScoreArgs<T>& a, cudaStream_t st) {
    const int vecs = a.V / Pack<T>::kN;
    int log_c = 0;
    const auto share = [&] { return (vecs + (1 << log_c) - 1) >> log_c; };
    while (log_c < 3 && (share() > 2560 || ((long long)a.rows << log_c) < 148 && share() > 256)) log_c++;
    a.log_c = log_c;
    const int threads = share() > 128 ? 256 : 128;
    const size_t smem = (size_t)share() * 16;
    static DeviceOnce once;
    const int rc = once.raise((const void*)score_kernel<T, kPolicy>, 200 * 1024);
    if (rc) return rc;
    return launch("score_kernel", score_kernel<T, kPolicy>, (long long)a.rows << log_c, threads, 1 << log_c, smem, false,
                  st, a);
}

template <typename T>
static ScoreArgs<T> score_args(const Rows& r) {
    ScoreArgs<T> a = {};
    a.logits = (const T*)r.logits;
    a.rows = r.rows;
    a.V = r.vocab;
    a.ld = r.ld;
    a.tokens = r.tokens;
    a.scale = (float)(r.inv_t * 1.4426950408889634);
    a.inv_t = r.inv_t;
    a.grad = (T*)r.grad;
    a.gld = r.gld;
    return a;
}

static int row_units(int dtype, int vocab) {
    const int vecs = vocab / (dtype == QS_F32 ? 4 : 8);
    return vecs > kUnitVecs ? (vecs + kUnitVecs - 1) / kUnitVecs : 1;
}
// Large calls stream; smaller ones take a cluster per row, in one launch.  Long
// bf16 rows from 72 MB (22.0 us against 22.4 at 72 MB, 30.4 against 33.2 at
// 120), fp32 rows and rows of less than a CTA's 40 KB from 24 MB (at 32 MB fp32
// of 151,936: 9.7 against 12.3 us, bf16 of 4,099: 13.3 against 16.9; at 16 MB
// 7.2 against 7.0 and 9.5 against 9.9).
static bool streams(int dtype, int rows, int vocab) {
    const size_t row = (size_t)vocab * (dtype == QS_F32 ? 4 : 2);
    return rows * row >= (size_t)(dtype == QS_BF16 && row >= 40 * 1024 ? 72 : 24) << 20;
}
static size_t score_workspace(int dtype, int rows, int vocab) {
    return streams(dtype, rows, vocab) ? round256((size_t)rows * row_units(dtype, vocab) * sizeof(float4)) : 0;
}

template <typename T>
static int score(const Rows& r, RowScore* out, float* coefs, float* logprobs, float* stats, float4* parts,
                 cudaStream_t st) {
    if (!streams(r.dtype, r.rows, r.vocab)) {
        ScoreArgs<T> a = score_args<T>(r);
        a.out = out;
        a.coefs = coefs;
        a.logprobs = logprobs;
        a.stats = stats;
        return score_launch<T, false>(a, st);
    }
    StreamArgs<T> a = {};
    a.logits = (const T*)r.logits;
    a.rows = r.rows;
    a.V = r.vocab;
    a.ld = r.ld;
    a.tokens = r.tokens;
    a.scale = (float)(r.inv_t * 1.4426950408889634);
    a.inv_t = r.inv_t;
    a.units = row_units(r.dtype, r.vocab);
    a.parts = parts;
    a.out = out;
    a.coefs = coefs;
    a.logprobs = logprobs;
    a.stats = stats;
    const size_t smem = (size_t)kStreamWarps * kStreamStages * kUnitVecs * 16;
    static DeviceOnce once;
    int rc = once.raise((const void*)stream_kernel<T>, (int)smem);
    if (rc) return rc;
    int dev = 0, sms = 148;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail(QS_ERR_CUDA, "device: %s", cudaGetErrorString(e));
    rc = launch("stream_kernel", stream_kernel<T>, sms, kStreamWarps * 32, 1, smem, false, st, a);
    if (rc) return rc;
    return launch("join_kernel", join_kernel<T>, (r.rows + kJoinRows - 1) / kJoinRows, kJoinRows * 32, 1, 0, true, st, a);
}

template <typename T>
static int grad(const Rows& r, const float* stats, int stat_words, const float* coefs, bool after, cudaStream_t st) {
    const int vecs = r.vocab / Pack<T>::kN;
    const int pieces = max(1, (vecs + kGradThreads * kGradVpt - 1) / (kGradThreads * kGradVpt));
    return launch("grad_kernel", grad_kernel<T>, (long long)r.rows * pieces, kGradThreads, 1, 0, after, st,
                  (const T*)r.logits, r.rows, r.vocab, r.ld, r.tokens, stats, stat_words, coefs,
                  (float)(r.inv_t * 1.4426950408889634), r.inv_t, (T*)r.grad, r.gld, pieces);
}

}  // namespace qs

using namespace qs;

extern "C" {

size_t qs_token_logprobs_workspace(int dtype, int rows, int vocab) {
    return dtype != QS_F32 && dtype != QS_BF16 || rows < 1 || vocab < 1 || vocab > kMaxVocab ? 0
                                                                                             : score_workspace(dtype, rows, vocab);
}

int qs_token_logprobs(const void* d_logits, int dtype, int rows, int vocab, long long row_stride,
                      const int* d_tokens, double temperature, float* d_logprobs, float* d_stats,
                      void* d_workspace, size_t workspace_bytes, void* stream) {
    set_error(QS_OK, "");
    const Rows r{d_logits, dtype, rows, vocab, row_stride, d_tokens, 1.0 / temperature, nullptr, 0};
    int rc = check_rows(r, temperature);
    if (rc || rows == 0) return rc;
    if (!d_logprobs || !d_stats) return fail(QS_ERR_INVALID, "NULL output buffer");
    rc = check_workspace(d_workspace, workspace_bytes, score_workspace(dtype, rows, vocab));
    if (rc) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    return dtype == QS_F32 ? score<float>(r, nullptr, nullptr, d_logprobs, d_stats, (float4*)d_workspace, st)
                           : score<__nv_bfloat16>(r, nullptr, nullptr, d_logprobs, d_stats, (float4*)d_workspace, st);
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
    const cudaStream_t st = (cudaStream_t)stream;
    return dtype == QS_F32 ? grad<float>(r, d_stats, 2, d_grad_logprobs, false, st)
                           : grad<__nv_bfloat16>(r, d_stats, 2, d_grad_logprobs, false, st);
}

size_t qs_policy_loss_workspace(int rows) { return round256((rows > 0 ? (size_t)rows : 1) * sizeof(double)); }

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
        const int bad = check_workspace(d_workspace, workspace_bytes, qs_policy_loss_workspace(rows));
        if (bad) return bad;
    }
    double* row_loss = (double*)d_workspace;
    if (rows > 0) {
        const auto go = [&](auto a) {
            a.logprobs = d_logprobs;
            a.weights = d_weights;
            a.old_lp = d_old_logprobs;
            a.ref_lp = d_ref_logprobs;
            a.adv = d_advantages;
            a.p = p;
            a.row_loss = row_loss;
            return score_launch<std::remove_pointer_t<decltype(a.grad)>, true>(a, st);
        };
        const int e = dtype == QS_F32 ? go(score_args<float>(r)) : go(score_args<__nv_bfloat16>(r));
        if (e) return e;
    }
    return launch("sum_rows_kernel", sum_rows_kernel, 1, rows > 512 ? 1024 : 128, 1, 0, rows > 0, st, row_loss, rows, d_loss);
}

size_t qs_preference_loss_workspace(int dtype, int rows, int vocab) {
    if (rows < 1) return 0;
    return round256((size_t)rows * sizeof(RowScore)) + round256((size_t)rows * sizeof(float)) +
           qs_token_logprobs_workspace(dtype, rows, vocab);
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
    const int bad = check_workspace(d_workspace, workspace_bytes, qs_preference_loss_workspace(dtype, rows, vocab));
    if (bad) return bad;
    const cudaStream_t st = (cudaStream_t)stream;
    RowScore* sc = (RowScore*)d_workspace;
    float* coefs = (float*)((char*)d_workspace + round256((size_t)rows * sizeof(RowScore)));
    float4* parts = (float4*)((char*)coefs + round256((size_t)rows * sizeof(float)));
    if (rows > 0) {
        const int e = dtype == QS_F32 ? score<float>(r, sc, coefs, nullptr, nullptr, parts, st)
                                      : score<__nv_bfloat16>(r, sc, coefs, nullptr, nullptr, parts, st);
        if (e) return e;
    }
    const int e = launch("preference_pairs_kernel", preference_pairs_kernel, 1, pairs > 4 ? 1024 : 128, 1, 0, rows > 0, st, sc, rows,
                         d_seq_offsets, pairs, d_ref_logprobs, d_weights, p, coefs, d_seq_logprobs, d_loss);
    if (e || rows == 0 || !d_grad) return e;
    return dtype == QS_F32 ? grad<float>(r, &sc->max, sizeof(RowScore) / 4, coefs, true, st)
                           : grad<__nv_bfloat16>(r, &sc->max, sizeof(RowScore) / 4, coefs, true, st);
}

}  // extern "C"
