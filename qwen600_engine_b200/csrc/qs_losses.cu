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
#include <type_traits>

#include "qs_rows.cuh"
#include "qs_stream.cuh"

namespace qs {

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

constexpr int kScoreThreads = 256;  // at most, in a CTA

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

// Joins a row's units as the stream leaves them (qs_stream.cuh), one warp a row.
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
    const int rc = stream_rows<T, false>(a, st);
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
