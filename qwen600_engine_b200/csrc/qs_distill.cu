// Divergence from a teacher known by the best tokens of each row, and the
// gradient of the logits (include/qwen600_sampler.h gives the formula).
//
// With m_r the maximum of the unlisted logits and m_l that of the listed ones,
//   S_r = sum over unlisted j of exp((x[j] - m_r) / T)     fp32, joined in 64 bits
//   S_l = sum over listed e of exp((x[e] - m_l) / T)       64 bits
// and S = S_l exp((m_l - m) / T) + S_r exp((m_r - m) / T), m the larger of the
// two.  The unlisted sum is taken by itself, against its own maximum: as what is
// left of 1 it would be nothing but rounding wherever the list holds nearly
// all, and p_r stands in a logarithm and a denominator.  The gradient is
//   listed    w / T (Q p[e] - q[e])                        64 bits
//   unlisted  f exp((x[j] - m_r) / T),  f = w / T (Q exp((m_r - m) / T) / S - r / S_r)
// so that one coefficient serves every token but the listed.
#include "qs_rows.cuh"

namespace qs {

constexpr int kDistillThreads = 256;
static_assert(QS_MAX_LISTED <= kDistillThreads, "one entry a thread");

template <typename T>
struct DistillArgs {
    const T* logits;
    int rows, V;
    long long ld;
    const int* tokens;
    const float* lps;
    int k;
    const float* weights;
    float scale;  // log2(e) / T
    double inv_t;
    int rest;
    int log_c;    // 1 << log_c CTAs per row, one cluster
    int buckets;  // of the table of listed tokens: a power of two, at least 2 k
    double* row_loss;
    float* row_losses;
    T* grad;
    long long gld;
};

// The slot of `tok` in the table of entries, or the first free one.
__device__ __forceinline__ int table_slot(const int* table, const int* listed, int mask, int tok) {
    int h = (int)((uint32_t)tok * 2654435769u >> 16) & mask;
    while (true) {
        const int e = *(const volatile int*)&table[h];
        if (e < 0 || listed[e] == tok) return h;
        h = (h + 1) & mask;
    }
}

// Sum of one double per thread over the CTA, in a fixed order, in every thread.
__device__ __forceinline__ double all_sum(double v, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kDistillThreads / 32; w++) v += red[w];
    __syncthreads();
    return v;
}
__device__ __forceinline__ float all_max(float v, float* red) {
    v = warp_max(v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < kDistillThreads / 32; w++) v = fmaxf(v, red[w]);
    __syncthreads();
    return v;
}

// One row per cluster of 1 to 8 CTAs, as the policy loss has it: each CTA brings
// a contiguous share of the row's 16-byte vectors to shared memory with one bulk
// copy, the row is read once and the gradient formed from the same copy.  The
// listed entries are read apart and their places in the shares overwritten with
// -inf, which takes them out of the maximum, the sum and the gradient's stream;
// every CTA does the small work on the list itself while its copy is under way.
template <typename T>
__global__ void __launch_bounds__(kDistillThreads)
distill_kernel(const __grid_constant__ DistillArgs<T> a, int share_vecs) {
    constexpr int kN = Pack<T>::kN;
    constexpr int kW = kDistillThreads / 32;
    extern __shared__ __align__(16) uint4 vecs[];
    int* listed = reinterpret_cast<int*>(vecs + share_vecs);  // [k] token, -1: no entry
    int* table = listed + a.k;                                // [buckets] entry, -1: none
    __shared__ Part parts[8];
    __shared__ double redd[kW];
    __shared__ float red_max[kW], red_sum[kW];
    __shared__ float factor_s, max_s;
    __shared__ double of_p_s, of_q_s, top_s;
    __shared__ unsigned long long loaded;
    __shared__ int gave_up;
    const int t = threadIdx.x, C = 1 << a.log_c;
    const int row = blockIdx.x >> a.log_c, rank = blockIdx.x & (C - 1);
    const T* x = a.logits + (size_t)row * a.ld;
    T* g = a.grad ? a.grad + (size_t)row * a.gld : nullptr;
    const float w_row = a.weights ? a.weights[row] : 1.0f;
    dependents_may_start();
    // what the row is when it adds nothing
    const auto nothing = [&] {
        if (rank == 0 && t == 0) {
            a.row_loss[row] = 0.0;
            if (a.row_losses) a.row_losses[row] = 0.0f;
        }
        if (g) {
            const RowShape<T> gs(g, a.V);
            for (int i = rank * kDistillThreads + t; i < gs.vecs; i += C * kDistillThreads)
                store16(g + gs.head + (size_t)i * kN, make_uint4(0u, 0u, 0u, 0u));
            const int e = rank == 0 ? gs.edge(t, a.V) : -1;
            if (e >= 0) put(g, e, 0.0f);
        }
    };
    if (w_row == 0.0f) {  // alike for the whole cluster
        nothing();
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

    // the list: one entry a thread, each token where it stands first
    int tok = -1;
    float lp = -INFINITY;
    if (t < a.k) {
        tok = a.tokens[(size_t)row * a.k + t];
        lp = a.lps[(size_t)row * a.k + t];
        if (tok < 0 || tok >= a.V) tok = -1;
        listed[t] = tok;
    }
    for (int i = t; i < a.buckets; i += kDistillThreads) table[i] = -1;
    const int edge = rank == 0 ? sh.edge(t, a.V) : -1;
    float xe = edge >= 0 ? elem(x, edge) : -INFINITY;
    const float xk = tok >= 0 ? elem(x, tok) : -INFINITY;
    __syncthreads();
    if (tok >= 0) {
        while (true) {
            const int h = table_slot(table, listed, a.buckets - 1, tok);
            const int e = atomicCAS(&table[h], -1, t);
            if (e < 0) break;
            if (listed[e] == tok) {
                atomicMin(&table[h], t);
                break;
            }
        }
    }
    __syncthreads();
    const bool entry = tok >= 0 && table[table_slot(table, listed, a.buckets - 1, tok)] == t;
    if (edge >= 0 && table[table_slot(table, listed, a.buckets - 1, edge)] >= 0) xe = -INFINITY;
    // the teacher's numbers; without a rest they count up to a common factor
    const float shift = a.rest ? 0.0f : all_max(entry ? lp : -INFINITY, red_max);
    const bool some = __syncthreads_or(entry && (a.rest || !(lp == -INFINITY)));
    const float ml = all_max(entry ? xk : -INFINITY, red_max);
    const double q = entry ? exp((double)lp - (double)shift) : 0.0;
    const double d = ((double)xk - (double)(ml == -INFINITY ? 0.0f : ml)) * a.inv_t;
    const double mass = all_sum(q, redd);                                                             // sum q
    const double cost = all_sum(q == 0.0 ? 0.0 : q * ((double)lp - (double)shift - d), redd);         // sum q (log q - d)
    const double sl = all_sum(entry ? exp(d) : 0.0, redd);
    if (!mbar_wait(&loaded, 0, &gave_up, kLoadWaitNs))
        mbar_wait(&loaded, 0, &gave_up, kLoadWaitNs, false);  // the copy lands before the CTA leaves
    if (!some) {
        if (C > 1) cluster_wait();
        nothing();
        return;
    }
    const int at = tok - sh.head - first * kN;  // in this CTA's share
    const bool held = entry && at >= 0 && at < cnt * kN;
    if (held) put(reinterpret_cast<T*>(vecs), at, -INFINITY);
    __syncthreads();

    // the maximum of this CTA's part
    float own_max = xe;
    {
        uint4 u = Pack<T>::lowest();
#pragma unroll 4
        for (int k = t; k < cnt; k += kDistillThreads) {
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
    const float m = all_max(own_max, red_max);
    const float ref = m == -INFINITY ? 0.0f : m;

    // the sum of exponentials against it: subtract and scale in one instruction where one_step allows it
    const float bias = ref * a.scale;
    float s;
    if (!one_step(bias)) {
        s = exp2_fast((xe - ref) * a.scale);
        for (int k = t; k < cnt; k += kDistillThreads) {
            float o[kN];
            Pack<T>::widen(vecs[k], o);
#pragma unroll
            for (int j = 0; j < kN; j++) s += exp2_fast((o[j] - ref) * a.scale);
        }
    } else {
        const f32x2 scale2 = pair2(a.scale, a.scale), bias2 = pair2(-bias, -bias);
        f32x2 s2 = pair2(exp2_fast(__fmaf_rn(xe, a.scale, -bias)), 0.0f);
#pragma unroll 2
        for (int k = t; k < cnt; k += kDistillThreads) {
            float o[kN];
            Pack<T>::widen(vecs[k], o);
#pragma unroll
            for (int j = 0; j < kN; j += 2) s2 = add2(s2, exp2_pair(fma2(pair2(o[j], o[j + 1]), scale2, bias2)));
        }
        const float2 u = unpair2(s2);
        s = (u.x + u.y) * exp2_fast(-__fmaf_rn(ref, a.scale, -bias));
    }
    s = warp_sum(s);
    if ((t & 31) == 0) red_sum[t >> 5] = s;
    __syncthreads();
    if (C > 1) cluster_wait();  // every CTA of the cluster runs
    if (t < C) {
        Part p{m, 0, *(volatile int*)&gave_up ? (double)NAN : 0.0};
        for (int w = 0; w < kW; w++) p.others += (double)red_sum[w];
        if (C > 1) push_part(&parts[rank], t, p);
        else parts[0] = p;
    }
    if (C > 1) {  // only the warp that stored into the others has stores to release
        if (t < 32) cluster_arrive_release();
        else cluster_arrive_relaxed();
        cluster_wait();
    }
    if (t < 32) {
        __syncwarp();
        const Part p = t < C ? parts[t] : Part{-INFINITY, 0, 0.0};
        const float mr = warp_max(p.max);
        double sr = p.max == mr ? p.others : t < C ? exp(((double)p.max - (double)mr) * a.inv_t) * p.others : 0.0;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) sr += __shfl_xor_sync(0xffffffffu, sr, o);
        if (t == 0) {
            const double top = fmax((double)mr, (double)ml);
            const double dr = mr == -INFINITY ? -(double)INFINITY : ((double)mr - top) * a.inv_t;
            const double dl = ml == -INFINITY ? -(double)INFINITY : ((double)ml - top) * a.inv_t;
            // an infinite maximum has no distribution; a NaN among the unlisted logits is in sr, one among the listed in sl
            const double total = isinf(top) ? (double)NAN : sl * exp(dl) + sr * exp(dr);
            const double log_total = log(total);
            double left = 0.0, l;
            if (a.rest) {
                if (mass < 1.0 && !(mr == -INFINITY && sr == 0.0)) left = 1.0 - mass;
                // the distance of d's reference from the row's, as log p has it: -inf - -inf where the logits mask the whole list
                l = cost + (mass == 0.0 ? 0.0 : mass * (log_total - (ml == -INFINITY ? -top * a.inv_t : dl)));
                if (left > 0.0) l += left * (log(left) - (dr + log(sr) - log_total));
            } else {
                l = cost / mass - log(mass) + log_total - (ml == -INFINITY ? -top * a.inv_t : dl);
            }
            const double w = a.weights ? (double)w_row : 1.0 / a.rows;
            if (rank == 0) {
                a.row_loss[row] = w * l;
                if (a.row_losses) a.row_losses[row] = (float)l;
            }
            const double c = w * a.inv_t, norm = a.rest ? mass + left : mass / mass;  // NaN from the teacher reaches the row
            of_p_s = c * norm / total;
            of_q_s = a.rest ? c : c / mass;
            top_s = top;
            factor_s = (float)(c * (norm * exp(dr) / total - (left > 0.0 ? left / sr : 0.0)));
            max_s = mr;
        }
    }
    if (!g) return;
    __syncthreads();
    float f = factor_s;
    const float mr = max_s, top = mr * a.scale;
    const bool plain = one_step(top);
    if (plain) f *= exp2_fast(-__fmaf_rn(mr, a.scale, -top));
    const auto grad_of = [&](float v) {
        return f == 0.0f ? 0.0f : f * exp2_fast(plain ? __fmaf_rn(v, a.scale, -top) : (v - mr) * a.scale);
    };
    const f32x2 f2 = pair2(f, f), scale2 = pair2(a.scale, a.scale), top2 = pair2(-top, -top);
    const bool aligned = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
    T* gbody = g + sh.head + (size_t)first * kN;
#pragma unroll 2
    for (int k = t; k < cnt; k += kDistillThreads) {
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
    if (edge >= 0) put(g, edge, grad_of(xe));
    __syncthreads();  // the listed ones over what the stream left in their places
    const bool outside = rank == 0 && (tok < sh.head || tok >= sh.head + sh.vecs * kN);
    if (entry && (held || outside))
        put(g, tok, (float)(of_p_s * exp(xk == -INFINITY ? -(double)INFINITY : ((double)xk - top_s) * a.inv_t) - of_q_s * q));
}

// How a row is spread: as the policy loss's rows (qs_losses.cu), CTAs per row
// doubled while a share is above 40 KB, and while the rows alone would leave some
// of the 148 SMs idle and a share keeps 4 KB.
template <typename T>
static int distill_launch(DistillArgs<T>& a, cudaStream_t st) {
    const int vecs = a.V / Pack<T>::kN;
    int log_c = 0;
    const auto share = [&] { return (vecs + (1 << log_c) - 1) >> log_c; };
    while (log_c < 3 && (share() > 2560 || ((long long)a.rows << log_c) < 148 && share() > 256)) log_c++;
    a.log_c = log_c;
    a.buckets = 2;
    while (a.buckets < 2 * a.k) a.buckets *= 2;
    const size_t smem = (size_t)share() * 16 + (a.k + a.buckets) * sizeof(int);
    static DeviceOnce once;
    const int rc = once.raise((const void*)distill_kernel<T>, 200 * 1024);
    if (rc) return rc;
    return launch("distill_kernel", distill_kernel<T>, (long long)a.rows << log_c, kDistillThreads, 1 << log_c, smem, false, st, a,
                  share());
}

}  // namespace qs

using namespace qs;

extern "C" {

size_t qs_distill_loss_workspace(int rows) { return round256((rows > 0 ? (size_t)rows : 1) * sizeof(double)); }

int qs_distill_loss(const void* d_logits, int dtype, int rows, int vocab, long long row_stride,
                    const int* d_teacher_tokens, const float* d_teacher_logprobs, int k, const float* d_weights,
                    const qs_distill_params* params, float* d_loss, float* d_row_losses, void* d_grad,
                    long long grad_row_stride, void* d_workspace, size_t workspace_bytes, void* stream) {
    set_error(QS_OK, "");
    if (!params) return fail(QS_ERR_INVALID, "params is NULL");
    const qs_distill_params p = *params;
    const Rows r{d_logits, dtype, rows, vocab, row_stride, d_teacher_tokens, 1.0 / p.temperature, d_grad, grad_row_stride};
    const int rc = check_rows(r, p.temperature);
    if (rc) return rc;
    if (k < 1 || k > QS_MAX_LISTED) return fail(QS_ERR_UNSUPPORTED, "k %d outside [1, %d]", k, QS_MAX_LISTED);
    if (!d_loss) return fail(QS_ERR_INVALID, "NULL output buffer");
    const cudaStream_t st = (cudaStream_t)stream;
    double* row_loss = (double*)d_workspace;
    if (rows > 0) {
        if (!d_teacher_logprobs) return fail(QS_ERR_INVALID, "NULL device pointer");
        const int bad = check_workspace(d_workspace, workspace_bytes, qs_distill_loss_workspace(rows));
        if (bad) return bad;
        const auto go = [&](auto a) {
            a.rows = rows;
            a.V = vocab;
            a.ld = row_stride;
            a.tokens = d_teacher_tokens;
            a.lps = d_teacher_logprobs;
            a.k = k;
            a.weights = d_weights;
            a.scale = (float)(r.inv_t * 1.4426950408889634);
            a.inv_t = r.inv_t;
            a.rest = p.rest != 0;
            a.row_loss = row_loss;
            a.row_losses = d_row_losses;
            a.logits = (decltype(a.logits))d_logits;
            a.grad = (decltype(a.grad))d_grad;
            a.gld = grad_row_stride;
            return distill_launch(a, st);
        };
        const int e = dtype == QS_F32 ? go(DistillArgs<float>{}) : go(DistillArgs<__nv_bfloat16>{});
        if (e) return e;
    }
    return launch("sum_rows_kernel", sum_rows_kernel, 1, rows > 512 ? 1024 : 128, 1, 0, rows > 0, st, row_loss, rows, d_loss);
}

}  // extern "C"
