// Divergence from a teacher known by the best tokens of each row, and the
// gradient of the logits (include/qwen600_sampler.h gives the formula).
//
// With m_l the maximum of the listed logits,
//   S_l = sum over listed e of exp((x[e] - m_l) / T)       64 bits
//   S_r = sum over unlisted j of exp((x[j] - m_l) / T)     fp32, joined in 64 bits
// and S their sum.  The unlisted sum is taken by itself: as what is left of 1 it
// would be nothing but rounding wherever the list holds nearly all, and p_r stands
// in a logarithm and a denominator.  The gradient is
//   listed    w / T (Q p[e] - q[e])                        64 bits
//   unlisted  f exp((x[j] - m_l) / T),  f = w / T (Q / S - r / S_r)
// so that one coefficient, formed without a logarithm, serves every token but the
// listed.  m_l is known before the row has arrived, which saves the pass that looks
// for a maximum; where S_r shows that the list lies far from the unlisted tokens, they
// are summed again against their own maximum.
#include "qs_rows.cuh"

namespace qs {

// Where the unlisted terms against the list's maximum come out below or above these,
// they are summed again against their own.  A term's exponent is rounded to a 2^-24th of
// itself; with sums from 2^-28 on it lies on the average below log2 V + 28.
constexpr double kLeastRest = 0x1p-28, kMostRest = 0x1p20;

// A row's list as the list kernel leaves it.  Its entries follow: tokens (int), then
// exp((x - m_l) / T) and q of each (double).
struct __align__(16) RowList {
    double mass;  // sum q
    double cost;  // sum q (log q - (x - m_l) / T); where the logits mask all of it, of q (log q - x / T)
    double sl;    // S_l
    float ml;
    int some;     // the row adds something
    double sr;    // S_r, against ref
    float ref;    // m_l, or where the list lies far from them the unlisted tokens' maximum
    int unused;
};

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
    int share;    // vectors of a CTA
    RowList* lists;
    double* list_p;   // [rows][k] exp((x - m_l) / T)
    double* list_q;   // [rows][k]
    int* list_token;  // [rows][k] -1: no entry
    T* grad;
    long long gld;
};

__device__ __forceinline__ double warp_sum_double(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The lists, a warp for a row: each token where it stands first, its logit, and what
// the loss takes of both.  Once for a row, where the row's CTAs would all have to
// (2048 rows 279 us then, 247 with it).  Latency: 2.4 us for 8 rows with lists of 20, 8
// for 300 with lists of 129, whose entries are each compared with all earlier ones; the
// rows' copies begin beside it.
constexpr int kListWarps = 4;

// kListMine: entries of a lane.
template <typename T, int kListMine>
__global__ void __launch_bounds__(kListWarps * 32)
distill_list_kernel(const __grid_constant__ DistillArgs<T> a) {
    __shared__ __align__(16) int tokens[kListWarps][kListMine * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x * kListWarps + warp;
    dependents_may_start();
    if (row >= a.rows) return;
    const float w = a.weights ? a.weights[row] : 1.0f;
    const T* x = a.logits + (size_t)row * a.ld;
    const size_t at = (size_t)row * a.k;
    int tok[kListMine];
    float lp[kListMine], v[kListMine];
#pragma unroll
    for (int i = 0; i < kListMine; i++) {
        const int e = i * 32 + lane;
        tok[i] = e < a.k ? a.tokens[at + e] : -1;
        lp[i] = e < a.k ? a.lps[at + e] : -INFINITY;
        if (tok[i] < 0 || tok[i] >= a.V) tok[i] = -1;
    }
    if (w == 0.0f) return;
#pragma unroll
    for (int i = 0; i < kListMine; i++) {
        v[i] = tok[i] >= 0 ? elem(x, tok[i]) : -INFINITY;
        tokens[warp][i * 32 + lane] = tok[i];
    }
    __syncwarp();
    // without a rest the teacher's numbers count up to a common factor
    float ml = -INFINITY, shift = -INFINITY;
    bool some = false;
#pragma unroll
    for (int i = 0; i < kListMine; i++) {
        const int e = i * 32 + lane;
        if (i * 32 >= a.k) break;
        const int4* all = reinterpret_cast<const int4*>(tokens[warp]);
        bool again = false;
        for (int j = 0; j < i * 8 + 8; j++) {
            const int4 o = all[j];
            again |= (o.x == tok[i] && j * 4 < e) | (o.y == tok[i] && j * 4 + 1 < e) | (o.z == tok[i] && j * 4 + 2 < e) |
                     (o.w == tok[i] && j * 4 + 3 < e);
        }
        if (again) tok[i] = -1;
        if (tok[i] < 0) continue;
        ml = fmaxf(ml, v[i]);
        shift = fmaxf(shift, lp[i]);
        some |= a.rest || !(lp[i] == -INFINITY);
    }
    ml = warp_max(ml);
    shift = a.rest ? 0.0f : warp_max(shift);
    some = __any_sync(0xffffffffu, some);
    const double from = ml == -INFINITY ? 0.0 : (double)ml;
    double mass = 0.0, cost = 0.0, sl = 0.0;
#pragma unroll
    for (int i = 0; i < kListMine; i++) {
        const int e = i * 32 + lane;
        if (i * 32 >= a.k) break;
        double q = 0.0, p = 0.0;
        if (tok[i] >= 0) {
            const double l = (double)lp[i] - (double)shift, d = ((double)v[i] - from) * a.inv_t;
            q = exp(l);
            p = exp(d);
            if (q != 0.0) cost += q * (l - d);
        }
        mass += q;
        sl += p;
        if (e < a.k) {
            a.list_token[at + e] = tok[i];
            a.list_p[at + e] = p;
            a.list_q[at + e] = q;
        }
    }
    mass = warp_sum_double(mass);
    cost = warp_sum_double(cost);
    sl = warp_sum_double(sl);
    if (lane == 0) a.lists[row] = RowList{mass, cost, sl, ml, some, 0.0, 0.0f, 0};
}

// Writes v to *slot of the cluster's CTA `rank`.
__device__ __forceinline__ void push_double(double* slot, int rank, double v) {
    uint32_t addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(addr)
                 : "r"((uint32_t)__cvta_generic_to_shared(slot)), "r"(rank));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

// One row per cluster of 1 to 8 CTAs.  Each CTA holds a contiguous share of the row's
// 16-byte vectors in shared memory, each of its warps a piece of that: a warp brings
// its piece with one bulk copy, sums it, and once the cluster has exchanged its sums
// forms the gradient from the same copy, so that the row is read from memory once and
// a CTA's warps meet once.  The listed entries' places in the pieces are overwritten
// with -inf, which takes them out of the sum and of the gradient's stream.
//
// Bound: memory, and the waits between a row's phases, two CTAs an SM: 208 us for 2048 bf16
// rows of 151,936 a quarter of which is left out (1089 MB, 5.2 TB/s), 26 for 300 fp32 rows
// of 37,999.  Its exponentials alone, two a token, would take 104.  Without a gradient the
// same way is taken: 111 us a call for the former (467 MB, 4.2 TB/s), 18.6 for the latter.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 512 / kThreads)
distill_kernel(const __grid_constant__ DistillArgs<T> a) {
    constexpr int kN = Pack<T>::kN;
    constexpr int kW = kThreads / 32;
    extern __shared__ __align__(16) uint4 vecs[];  // [warp][piece]
    __shared__ double parts[3][8], pass_sum[kW];
    __shared__ float red_max[kW];
    __shared__ unsigned long long full[kW];
    __shared__ int gave_up;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, C = 1 << a.log_c;
    const int row = blockIdx.x >> a.log_c, rank = blockIdx.x & (C - 1);
    const T* x = a.logits + (size_t)row * a.ld;
    const float w_row = a.weights ? a.weights[row] : 1.0f;
    dependents_may_start();
    const auto nothing = [&] {  // what a row is that adds nothing
        if (!a.grad) return;
        T* g = a.grad + (size_t)row * a.gld;
        const RowShape<T> gs(g, a.V);
        for (int i = rank * kThreads + t; i < gs.vecs; i += C * kThreads)
            store16(g + gs.head + (size_t)i * kN, make_uint4(0u, 0u, 0u, 0u));
        const int e = rank == 0 ? gs.edge(t, a.V) : -1;
        if (e >= 0) put(g, e, 0.0f);
    };
    if (w_row == 0.0f) {  // alike for the whole cluster
        nothing();
        // Where every row is left out, one CTA sees to it that this grid does not end before the list kernel has:
        // what follows on the stream waits for this grid and the loss's, and may write what the lists are read from.
        if (blockIdx.x == 0) wait_for_previous();
        return;
    }
    const int piece = (a.share + kW - 1) / kW;
    uint4* mine = vecs + warp * piece;
    const RowShape<T> sh(x, a.V);
    const int begin = rank * a.share + warp * piece;
    const int cnt = max(0, min(min(piece, a.share - warp * piece), sh.vecs - begin)), from = sh.head + begin * kN;
    if (lane == 0) {
        mbar_init(&full[warp], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_expect_tx(&full[warp], (uint32_t)cnt * 16u);
        if (cnt > 0)
            asm volatile(
                "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(mine)),
                "l"(x + from), "r"((uint32_t)cnt * 16u), "r"(smem_u32(&full[warp]))
                : "memory");
    }
    if (C > 1) cluster_arrive_relaxed();  // waited for before the first store into another CTA
    if (t == 0) gave_up = 0;
    const int edge = rank == 0 && warp == 0 ? sh.edge(lane, a.V) : -1;
    float xe = edge >= 0 ? elem(x, edge) : -INFINITY;
    wait_for_previous();
    const RowList list = a.lists[row];
    const int* list_token = a.list_token + (size_t)row * a.k;
    const float ml = list.ml;
    // this lane's entries that lie in the warp's piece, or outside the vectors; requested again at the end
    uint32_t own = 0;
    const bool outside = rank == 0 && warp == 0;
    for (int i = 0; i * 32 < a.k; i++) {
        const int e = i * 32 + lane, token = e < a.k ? list_token[e] : -1, at = token - from;
        if (token < 0) continue;
        if ((at >= 0 && at < cnt * kN) || (outside && (token < sh.head || token >= sh.head + sh.vecs * kN))) {
            own |= 1u << i;
            asm volatile("prefetch.global.L1 [%0];" ::"l"(a.list_p + (size_t)row * a.k + e));
            asm volatile("prefetch.global.L1 [%0];" ::"l"(a.list_q + (size_t)row * a.k + e));
        }
    }
    __syncthreads();  // gave_up, and each warp's barrier for all of its lanes
    if (!mbar_wait(&full[warp], 0, &gave_up, kLoadWaitNs))
        mbar_wait(&full[warp], 0, &gave_up, kLoadWaitNs, false);  // the copy lands before the CTA leaves
    if (!list.some) {
        __syncthreads();  // every warp's
        if (C > 1) cluster_wait();
        nothing();
        return;
    }

    // the listed entries of this warp's piece, and of what lies outside the vectors
    for (uint32_t m = own; m; m &= m - 1) {
        const int at = list_token[(__ffs(m) - 1) * 32 + lane] - from;
        if (at >= 0 && at < cnt * kN) put(reinterpret_cast<T*>(mine), at, -INFINITY);
    }
    if (edge >= 0)
        for (int e = 0; e < a.k; e++)
            if (list_token[e] == edge) xe = -INFINITY;
    __syncwarp();

    // v of this CTA's threads 0 to C - 1 to every CTA's slots, then all may read them
    const auto exchange = [&](double* slots, double v) {
        if (C == 1) {
            if (t == 0) slots[0] = v;
            __syncthreads();
            return;
        }
        if (t < C) push_double(&slots[rank], t, v);
        if (t < 32) cluster_arrive_release();  // only this warp has stores to release
        else cluster_arrive_relaxed();
        cluster_wait();
    };
    const auto sum_of = [&](const double* v, int n) {
        double s = 0.0;
        for (int i = 0; i < n; i++) s += v[i];
        return s;
    };

    // the sum against the list's maximum: subtract and scale in one instruction where one_step allows it
    const f32x2 scale2 = pair2(a.scale, a.scale);
    float ref = ml, bias = ref * a.scale, s = INFINITY;
    if (one_step(bias)) {
        const f32x2 bias2 = pair2(-bias, -bias);
        f32x2 s2 = pair2(exp2_fast(__fmaf_rn(xe, a.scale, -bias)), 0.0f);
#pragma unroll 2
        for (int k = lane; k < cnt; k += 32) {
            float o[kN];
            Pack<T>::widen(mine[k], o);
#pragma unroll
            for (int j = 0; j < kN; j += 2) s2 = add2(s2, exp2_pair(fma2(pair2(o[j], o[j + 1]), scale2, bias2)));
        }
        const float2 u = unpair2(s2);
        s = (u.x + u.y) * exp2_fast(-__fmaf_rn(ref, a.scale, -bias));
    }
    s = warp_sum(s);
    if (lane == 0) pass_sum[warp] = *(volatile int*)&gave_up ? (double)NAN : (double)s;
    __syncthreads();
    if (C > 1) cluster_wait();  // every CTA of the cluster runs
    exchange(parts[0], t < C ? sum_of(pass_sum, kW) : 0.0);
    double sr = sum_of(parts[0], C);
    double top = ref, dl = 0.0, dr = 0.0;  // the row's maximum, and the list's and the others' distances from it
    const double least = a.rest ? kLeastRest : 0.0;
    const bool far = !(sr >= least && sr <= kMostRest);
    if (far) {
        // the unlisted tokens against their own maximum
        float m = xe;
        for (int k = lane; k < cnt; k += 32) {
            float o[kN];
            Pack<T>::widen(mine[k], o);
#pragma unroll
            for (int j = 0; j < kN; j++) m = fmaxf(m, o[j]);
        }
        m = warp_max(m);
        if (lane == 0) red_max[warp] = m;
        __syncthreads();
        for (int w = 0; w < kW; w++) m = fmaxf(m, red_max[w]);
        exchange(parts[1], (double)m);
        ref = -INFINITY;
        for (int c = 0; c < C; c++) ref = fmaxf(ref, (float)parts[1][c]);
        const float zero = ref == -INFINITY ? 0.0f : ref;
        s = exp2_fast((xe - zero) * a.scale);
        for (int k = lane; k < cnt; k += 32) {
            float o[kN];
            Pack<T>::widen(mine[k], o);
#pragma unroll
            for (int j = 0; j < kN; j++) s += exp2_fast((o[j] - zero) * a.scale);
        }
        s = warp_sum(s);
        if (lane == 0) pass_sum[warp] = *(volatile int*)&gave_up ? (double)NAN : (double)s;
        __syncthreads();
        exchange(parts[2], t < C ? sum_of(pass_sum, kW) : 0.0);
        sr = sum_of(parts[2], C);
        top = fmax((double)ref, (double)ml);
        dr = ref == -INFINITY ? -(double)INFINITY : ((double)ref - top) * a.inv_t;
        dl = ml == -INFINITY ? -(double)INFINITY : ((double)ml - top) * a.inv_t;
    }
    const double w = a.weights ? (double)w_row : 1.0 / a.rows, c = w * a.inv_t;
    // an infinite maximum has no distribution; a NaN among the unlisted logits is in sr, one among the listed in sl
    const double total = isinf(top) ? (double)NAN : far ? list.sl * exp(dl) + sr * exp(dr) : list.sl + sr;
    const double left = a.rest && list.mass < 1.0 && !(ref == -INFINITY && sr == 0.0) ? 1.0 - list.mass : 0.0;
    const double norm = a.rest ? list.mass + left : list.mass / list.mass;  // NaN from the teacher reaches the row
    if (rank == 0 && t == 0) {  // for the loss
        a.lists[row].sr = sr;
        a.lists[row].ref = ref;
    }
    if (!a.grad) return;

    // of every unlisted token; its two parts in fp32, which the sums' precision bears
    float f = (float)(c * norm) / (float)total;
    if (far) f *= (float)exp(dr);
    if (left > 0.0) f -= (float)(c * left) / (float)sr;
    bias = ref * a.scale;
    const bool plain = one_step(bias);
    if (plain) f *= exp2_fast(-__fmaf_rn(ref, a.scale, -bias));
    const auto grad_of = [&](float v) {
        return f == 0.0f ? 0.0f : f * exp2_fast(plain ? __fmaf_rn(v, a.scale, -bias) : (v - ref) * a.scale);
    };
    T* g = a.grad + (size_t)row * a.gld;
    const f32x2 f2 = pair2(f, f), bias2 = pair2(-bias, -bias);
    const bool aligned = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
#pragma unroll 2
    for (int k = lane; k < cnt; k += 32) {
        float o[kN];
        Pack<T>::widen(mine[k], o);
        if (plain && f != 0.0f) {
#pragma unroll
            for (int j = 0; j < kN; j += 2) {
                const float2 r = unpair2(mul2(f2, exp2_pair(fma2(pair2(o[j], o[j + 1]), scale2, bias2))));
                o[j] = r.x;
                o[j + 1] = r.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < kN; j++) o[j] = grad_of(o[j]);
        }
        if (aligned) {
            store16(g + from + (size_t)k * kN, Pack<T>::narrow(o));
        } else {  // 2048 bf16 rows whose logits lie one element off a vector's border: 689 us, 219 without
#pragma unroll
            for (int j = 0; j < kN; j++) put(g + from, (long long)k * kN + j, o[j]);
        }
    }
    if (edge >= 0) put(g, edge, grad_of(xe));
    __syncwarp();  // then the listed ones, over what the stream left in their places
    for (uint32_t m = own; m; m &= m - 1) {
        const int e = (__ffs(m) - 1) * 32 + lane, token = list_token[e];
        const double p = a.list_p[(size_t)row * a.k + e], q = a.list_q[(size_t)row * a.k + e];
        put(g, token, (float)(c * (norm / total * (far ? p * exp(dl) : p) - (a.rest ? q : q / list.mass))));
    }
}

// The rows' losses from their sums, and their sum in a fixed order.
__global__ void __launch_bounds__(1024)
distill_loss_kernel(const RowList* lists, int rows, const float* __restrict__ weights, double inv_t, int rest, float* row_losses,
                    float* __restrict__ loss) {
    __shared__ double red[32];
    wait_for_previous();
    double sum = 0.0;
    for (int i = threadIdx.x; i < rows; i += blockDim.x) {
        const double w = weights ? (double)weights[i] : 1.0 / rows;
        double l = 0.0;
        if (w != 0.0 && lists[i].some) {
            const RowList r = lists[i];
            // distances of the list's and the others' maximum from the row's
            const double top = fmax((double)r.ref, (double)r.ml);
            const double dr = r.ref == -INFINITY ? -(double)INFINITY : ((double)r.ref - top) * inv_t;
            const double dl = r.ml == -INFINITY ? -(double)INFINITY : ((double)r.ml - top) * inv_t;
            const double total = isinf(top) ? (double)NAN : r.sl * (dl == 0.0 ? 1.0 : exp(dl)) + r.sr * (dr == 0.0 ? 1.0 : exp(dr));
            const double log_total = log(total);
            // cost counts from the list's maximum (from 0 where all of it is masked), log p from the row's
            const double away = log_total - (r.ml == -INFINITY ? -top * inv_t : dl);
            if (rest) {
                const double left = r.mass < 1.0 && !(r.ref == -INFINITY && r.sr == 0.0) ? 1.0 - r.mass : 0.0;
                l = r.cost + (r.mass == 0.0 ? 0.0 : r.mass * away);
                if (left > 0.0) l += left * (log(left) - (dr + log(r.sr) - log_total));
            } else {
                l = r.cost / r.mass - log(r.mass) + away;
            }
            if (isnan(total)) l = total;  // no distribution, also where nothing is summed: the gradient is NaN then
            sum += w * l;
        }
        if (row_losses) row_losses[i] = (float)l;
    }
    sum = block_sum(sum, red);
    if (threadIdx.x == 0) *loss = (float)sum;
}

// How rows are spread: CTAs per row (a power of two up to 8), doubled while a share is
// above 80 KB, two of which fit on an SM, and while the rows alone would leave some of
// the 148 SMs idle and a share is above 4 KB (halves of it are 2 KB and more).  2048 bf16
// rows of 151,936, a quarter of them left out: 218 us with 4 CTAs a row (76 KB shares), 241
// with 8 (38 KB, five an SM), 312 with 2; 300 fp32 rows of 37,999 29 us with 2, 31 with 4.
// CTAs of 224 threads 232 us, of 384 259.  CTAs that have an SM for themselves take 512
// threads (8 rows 6.2 us, 7.0 with 256).
template <typename T>
static int distill_launch(DistillArgs<T>& a, cudaStream_t st) {
    const int vecs = a.V / Pack<T>::kN;
    int log_c = 0;
    const auto share = [&] { return (vecs + (1 << log_c) - 1) >> log_c; };
    while (log_c < 3 && (share() > 5120 || ((long long)a.rows << log_c) < 148 && share() > 256)) log_c++;
    a.log_c = log_c;
    a.share = share();
    const auto lists = [&](auto kernel) {
        return launch("distill_list_kernel", kernel, (a.rows + kListWarps - 1) / kListWarps, kListWarps * 32, 1, 0, false, st, a);
    };
    int rc = a.k <= 32    ? lists(distill_list_kernel<T, 1>)
             : a.k <= 64  ? lists(distill_list_kernel<T, 2>)
             : a.k <= 128 ? lists(distill_list_kernel<T, 4>)
                          : lists(distill_list_kernel<T, 8>);
    if (rc) return rc;
    const auto rows = [&](auto kernel, int threads, DeviceOnce& once) {
        const int warps = threads / 32, e = once.raise((const void*)kernel, 200 * 1024);
        if (e) return e;
        const size_t smem = (size_t)((a.share + warps - 1) / warps * warps) * 16;
        return launch("distill_kernel", kernel, (long long)a.rows << log_c, threads, 1 << log_c, smem, true, st, a);
    };
    static DeviceOnce few, many;
    return (long long)a.rows << log_c <= 148 ? rows(distill_kernel<T, 512>, 512, few) : rows(distill_kernel<T, 256>, 256, many);
}

// Workspace: the rows' lists, and their entries.
static size_t distill_bytes(int rows, int k) {
    const size_t n = rows > 0 ? (size_t)rows : 1, e = n * k;
    return round256(n * sizeof(RowList)) + 2 * round256(e * sizeof(double)) + round256(e * sizeof(int));
}

}  // namespace qs

using namespace qs;

extern "C" {

size_t qs_distill_loss_workspace(int rows, int k) { return k < 1 || k > QS_MAX_LISTED ? 0 : distill_bytes(rows, k); }

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
    if (rows > 0) {
        if (!d_teacher_logprobs) return fail(QS_ERR_INVALID, "NULL device pointer");
        const int bad = check_workspace(d_workspace, workspace_bytes, distill_bytes(rows, k));
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
            const size_t e = round256((size_t)rows * k * sizeof(double));
            a.lists = (RowList*)d_workspace;
            a.list_p = (double*)((char*)a.lists + round256((size_t)rows * sizeof(RowList)));
            a.list_q = (double*)((char*)a.list_p + e);
            a.list_token = (int*)((char*)a.list_q + e);
            a.logits = (decltype(a.logits))d_logits;
            a.grad = (decltype(a.grad))d_grad;
            a.gld = grad_row_stride;
            return distill_launch(a, st);
        };
        const int e = dtype == QS_F32 ? go(DistillArgs<float>{}) : go(DistillArgs<__nv_bfloat16>{});
        if (e) return e;
    }
    return launch("distill_loss_kernel", distill_loss_kernel, 1, rows > 128 ? 1024 : 128, 1, 0, rows > 0, st, (const RowList*)d_workspace, rows,
                  d_weights, r.inv_t, p.rest != 0, d_row_losses, d_loss);
}

}  // extern "C"
