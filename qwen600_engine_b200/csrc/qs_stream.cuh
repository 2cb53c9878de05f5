// A stream over rows of logits that leaves each unit's maximum and sum of
// exponentials, and where it is asked for the maximum of each lane's part.
#pragma once
#include "qs_rows.cuh"

namespace qs {

// What a scored row leaves for the losses and the gradient.
struct RowScore {
    double logprob;  // 0 for a row that scores nothing
    float max;
    float excess;
};

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
// were 16 us slower.  The lanes' maxima for the best tokens cost it 1 us.
constexpr int kUnitVecs = 256;
constexpr int kStreamWarps = 24;
constexpr int kStreamStages = 2;

template <typename T>
struct StreamArgs {
    const T* logits;
    int rows, V;
    long long ld;
    const int* tokens;              // logprobs: a row whose token is outside the vocabulary is left out
    const float* scores;            // best tokens: a row whose score is not finite is left out (NULL: none is)
    const unsigned char* finished;  // and one that is marked here (NULL: none is)
    float scale;
    double inv_t;
    int units;     // per row
    T* lanes;      // best tokens: [rows][units][32], the maximum of each lane's part of a unit: 8 vectors behind one
                   // another (and of a row's first unit what lies outside the vectors)
    float4* parts; // [rows][units]: maximum, sum of exponentials against it, how many 1s were left out of it
    RowScore* out;
    float* coefs;  // with out: set to 0
    float* logprobs;
    float* stats;
};

// The vector of a unit that a lane takes i-th: for logprobs the lanes' vectors lie
// between one another's, for the best tokens a lane has 128 bytes of its own, taken
// from another one on in each lane, which keeps the banks apart.
template <bool kBest>
__device__ __forceinline__ int vec_of(int i, int lane) {
    return kBest ? lane * (kUnitVecs / 32) + ((i + lane) & (kUnitVecs / 32 - 1)) : i * 32 + lane;
}

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

template <typename T, bool kBest>
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
    // what says whether a row takes part, as it is loaded: looked at when it is needed, one unit later
    struct Look {
        int mark;
        float score;
    };
    const auto look = [&](int row) {
        Look l{-1, 0.0f};
        if (row >= a.rows) return l;
        if (kBest) {
            l.mark = a.finished ? -(int)a.finished[row] : 0;
            if (a.scores) l.score = a.scores[row];
        } else {
            l.mark = a.tokens[row];
        }
        return l;
    };
    const auto scored = [&](const Look& l) { return l.mark >= 0 && (kBest ? isfinite(l.score) : l.mark < a.V); };
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
        if (scored(look(ahead.row))) {
            request(ahead, i);
            live |= 1u << i;
        }
        ahead.step(dr, du, a.units);
    }
    Look next = look(ahead.row);
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
                const int k = vec_of<kBest>(i, lane);
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
            if (kBest) put(a.lanes, ((long long)now.row * a.units + now.unit) * 32 + lane, own);
            const float m = warp_max(own);
            const uint32_t holders = __ballot_sync(0xffffffffu, own == m);
            const bool one = (holders & (holders - 1)) == 0;
            const int holder = __ffs(holders) - 1;
            float again = 0.0f;  // this lane's share of the holder's elements
            int at_max = 0;
            if (one) {
                const int k = vec_of<kBest>(lane >> 2, holder);
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
            if (scored(next) && !dead) {
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
            if (scored(next) && !dead) {
                request(ahead, stage);
                live |= 1u << stage;
            }
        }
        now.step(dr, du, a.units);
        ahead.step(dr, du, a.units);
        next = look(ahead.row);
    }
}

[[maybe_unused]] static int row_units(int dtype, int vocab) {
    const int vecs = vocab / (dtype == QS_F32 ? 4 : 8);
    return vecs > kUnitVecs ? (vecs + kUnitVecs - 1) / kUnitVecs : 1;
}

// The stream over all of a call's rows.
template <typename T, bool kBest>
static int stream_rows(const StreamArgs<T>& a, cudaStream_t st) {
    const size_t smem = (size_t)kStreamWarps * kStreamStages * kUnitVecs * 16;
    static DeviceOnce once;
    int rc = once.raise((const void*)stream_kernel<T, kBest>, (int)smem);
    if (rc) return rc;
    int dev = 0, sms = 148;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail(QS_ERR_CUDA, "device: %s", cudaGetErrorString(e));
    return launch("stream_kernel", stream_kernel<T, kBest>, sms, kStreamWarps * 32, 1, smem, false, st, a);
}

}  // namespace qs
