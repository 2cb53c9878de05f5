// The best tokens of a row of logits with their log-probabilities, and a step of
// beam search over them (include/qwen600_sampler.h gives the formulas).
//
// Two kernels.  The stream (qs_stream.cuh) reads every row once and leaves, for
// each unit of 256 vectors, its maximum and sum of exponentials, and the maximum
// of each lane's part: 8 vectors, 64 bf16 or 32 fp32 elements.  The pick takes a
// group (a row, or the rows of an entry's beams), joins the sums, and narrows
// down: if n parts have a maximum of at least v, then n elements do, so whatever
// is below v is none of the n best.  With v the n-th largest maximum that leaves
// about n parts to be read again, 128 bytes each, and few more than n elements to
// be ranked.
#include "qs_rows.cuh"
#include "qs_stream.cuh"

namespace qs {

constexpr int kPickThreads = 256;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kTokenBits = 18;
static_assert(kMaxVocab <= 1 << kTokenBits && QS_MAX_BEAMS <= 1 << (32 - kTokenBits), "beam and token in one word");
constexpr int kMaxCands = 2 * QS_MAX_LISTED;  // elements that are ranked, beside ended beams
// Parts that a bound may hold beyond those it counts: a part counts from the last
// place it may hold on, and is looked at from its first; among equal scores that
// is one unit, its neighbour and a row's first unit (which also holds what lies
// behind the row's last vector), or their 32 lanes, and as many again that count
// from the same place.
constexpr int kUnitExtra = 6;
constexpr int kPartExtra = 160;
constexpr double kLowest = -1.7976931348623157e308;  // the lowest finite number

template <typename T>
struct PickArgs {
    const T* logits;
    int V;
    long long ld;
    int units;  // per row
    const float4* parts;
    const T* lanes;
    float scale;
    double inv_t;
    int beams, n;
    int unit_cap;  // units whose lanes are looked at: all of the group, or the best
    int part_cap;  // lanes whose elements are looked at
    const float* scores;            // of beams (NULL: 0)
    const unsigned char* finished;  // beams that go on with `pad` alone (NULL: none)
    int pad, eos, keep;
    float* out_scores;
    int* parents;  // NULL: rows' lists
    int* tokens;
    unsigned char* out_finished;
};

// What is left of a group's elements, by score and, among equal ones, by place:
// those above v, and those at v with a place up to `last`.
struct Bound {
    double v;
    uint32_t last;
    template <typename Place>
    __device__ __forceinline__ bool has(double s, Place place) const { return s > v || (s == v && place() <= last); }
};

// Doubles as whole numbers of the same order, and back.
__device__ __forceinline__ unsigned long long dkey(double d) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(d + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double dkey_inv(unsigned long long k) {
    return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

// Sum over the CTA, in every thread; `turn` alternates, so that one barrier is enough.
__device__ __forceinline__ int total_of(int v, int (*red)[kPickWarps], int& turn) {
    v = __reduce_add_sync(0xffffffffu, v);
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kPickWarps; w++) v += red[turn][w];
    return v;
}

// A bound that n items at least are within, and n + slack at most if their places
// allow it; `within` where that already has no more.  each(f) calls f(score,
// place) for this thread's items, place() being the item's; best: the largest score.
template <typename Each>
__device__ Bound narrow(Bound within, int n, int slack, double best, int (*red)[kPickWarps], int& turn, Each each) {
    const auto count = [&](const Bound& b) {
        int c = 0;
        each([&](double s, auto place) { c += within.has(s, place) && b.has(s, place); });
        return total_of(c, red, turn);
    };
    if (count(within) <= n + slack) return within;
    // scores a few units below the best, then halves of what is left
    unsigned long long low = dkey(within.v), high = dkey(best) + 1;  // n or more from low on, fewer from high on
    double below = 1.0;
    while (high - low > 1) {
        unsigned long long mid = low + (high - low) / 2;
        if (below <= 64.0) {
            const unsigned long long k = dkey(best - below);
            below *= 2.0;
            if (k > low && k < high) mid = k;
            else below = 128.0;
        }
        const Bound b{dkey_inv(mid), 0xFFFFFFFFu};
        const int c = count(b);
        if (c < n) {
            high = mid;
            continue;
        }
        if (c <= n + slack) return b;
        low = mid;
        below = 128.0;
    }
    // more than n + slack, because many are equal: the first ones
    Bound b{dkey_inv(low), within.last};
    if (b.v != within.v) b.last = 0xFFFFFFFFu;
    long long none = -1;
    while ((long long)b.last - none > 1) {
        const long long mid = none + ((long long)b.last - none) / 2;
        const int c = count(Bound{b.v, (uint32_t)mid});
        if (c < n) {
            none = mid;
            continue;
        }
        b.last = (uint32_t)mid;
        if (c <= n + slack) break;
    }
    return b;
}

// One CTA per group.
template <typename T>
__global__ void __launch_bounds__(kPickThreads, 4)
pick_kernel(const __grid_constant__ PickArgs<T> a) {
    constexpr int kN = Pack<T>::kN;
    constexpr int kPartVecs = kUnitVecs / 32;
    extern __shared__ __align__(16) double pool[];  // lanes' scores, units' scores, lists of units and of parts
    __shared__ double add_s[QS_MAX_BEAMS];
    __shared__ float max_s[QS_MAX_BEAMS];
    __shared__ unsigned char state_s[QS_MAX_BEAMS];  // 0: offers its tokens, 1: ended, 2: nothing, 3: NaN
    __shared__ double cand[kMaxCands + QS_MAX_BEAMS];
    __shared__ uint32_t cand_place[kMaxCands + QS_MAX_BEAMS];
    __shared__ int red[2][kPickWarps];
    __shared__ int chosen_units, chosen_parts, cands;
    __shared__ unsigned char slot_of[QS_MAX_BEAMS], parent_of[QS_MAX_BEAMS];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, group = blockIdx.x;
    const int all_units = a.beams * a.units;
    double* lane_score = pool;                      // [unit_cap][32]
    double* unit_score = lane_score + a.unit_cap * 32;
    int* unit_list = reinterpret_cast<int*>(unit_score + (a.unit_cap < all_units ? all_units : 0));  // [unit_cap]
    int* part_list = unit_list + a.unit_cap;        // [part_cap]
    int turn = 0;
    if (t == 0) chosen_units = chosen_parts = cands = 0;
    dependents_may_start();
    wait_for_previous();

    // each row's maximum and sum
    for (int i = warp; i < a.beams; i += kPickWarps) {
        const size_t row = (size_t)group * a.beams + i;
        const double base = a.scores ? (double)a.scores[row] : 0.0;
        int state = base < INFINITY ? (base > -INFINITY ? (a.finished && a.finished[row] ? 1 : 0) : 2) : 3;
        double add = base;
        float M = -INFINITY;
        if (state == 0) {
            const float4* p = a.parts + row * a.units;
            for (int u = lane; u < a.units; u += 32) M = fmaxf(M, p[u].x);
            M = warp_max(M);
            double sum = 0.0;
            for (int u = lane; u < a.units; u += 32) {
                const float4 v = p[u];
                sum += v.x == M ? (double)v.y + (double)v.z : (double)(exp2_fast((v.x - M) * a.scale) * (v.y + v.z));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (M == -INFINITY) state = sum == 0.0 ? 2 : 3;
            else if (!(M < INFINITY) || sum != sum) state = 3;
            else add = base - log(sum);
        }
        if (lane == 0) {
            add_s[i] = add;
            max_s[i] = M;
            state_s[i] = (unsigned char)state;
        }
    }
    __syncthreads();
    double best = -INFINITY;
    bool bad = false;
    for (int i = 0; i < a.beams; i++) {
        bad |= state_s[i] == 3;
        if (state_s[i] == 0) best = fmax(best, add_s[i]);
    }
    const size_t out = (size_t)group * a.n;
    if (bad) {
        for (int i = t; i < a.n; i += kPickThreads) {
            a.out_scores[out + i] = NAN;
            a.tokens[out + i] = -1;
            if (a.parents) a.parents[out + i] = -1;
            if (a.out_finished) a.out_finished[out + i] = 1;
        }
        return;
    }
    const auto score_of = [&](float x, int beam) { return ((double)x - (double)max_s[beam]) * a.inv_t + add_s[beam]; };
    Bound bound{kLowest, 0xFFFFFFFFu};

    // the units: all of them, or those that may hold one of the best
    if (a.unit_cap < all_units) {
        for (int u = t; u < all_units; u += kPickThreads) {
            const int beam = u / a.units;
            unit_score[u] = state_s[beam] == 0 ? score_of(a.parts[((size_t)group * a.beams) * a.units + u].x, beam) : -INFINITY;
        }
        __syncthreads();
        const auto first_place = [&](int u) {
            const int beam = u / a.units, unit = u - beam * a.units;
            return (uint32_t)beam << kTokenBits | (unit == 0 ? 0u : (uint32_t)(unit * kUnitVecs * kN));
        };
        const auto last_place = [&](int u) {  // unit 0 also holds the elements behind the row's last vector
            const int beam = u / a.units, unit = u - beam * a.units;
            return (uint32_t)beam << kTokenBits | (uint32_t)(unit == 0 ? a.V - 1 : min(a.V - 1, (unit + 1) * kUnitVecs * kN + kN - 1));
        };
        bound = narrow(bound, a.n, a.unit_cap - kUnitExtra - a.n, best, red, turn, [&](auto f) {
            for (int u = t; u < all_units; u += kPickThreads) f(unit_score[u], [&] { return last_place(u); });
        });
        for (int u = t; u < all_units; u += kPickThreads)
            if (bound.has(unit_score[u], [&] { return first_place(u); })) {
                const int at = atomicAdd(&chosen_units, 1);
                if (at < a.unit_cap) unit_list[at] = u;
            }
    } else {
        for (int u = t; u < all_units; u += kPickThreads)
            if (state_s[u / a.units] == 0) unit_list[atomicAdd(&chosen_units, 1)] = u;
    }
    __syncthreads();
    const int units = min(chosen_units, a.unit_cap);

    // their lanes' parts
    for (int i = t; i < units * 32; i += kPickThreads) {
        const int u = unit_list[i >> 5];
        lane_score[i] = score_of(elem(a.lanes, ((long long)group * all_units + u) * 32 + lane), u / a.units);
    }
    __syncthreads();
    const auto part_first = [&](int u) {
        const int beam = u / a.units, unit = u - beam * a.units;
        return (uint32_t)beam << kTokenBits | (unit == 0 ? 0u : (uint32_t)((unit * kUnitVecs + lane) * kN));
    };
    const auto part_last = [&](int u) {
        const int beam = u / a.units, unit = u - beam * a.units;
        return (uint32_t)beam << kTokenBits |
               (uint32_t)(unit == 0 ? a.V - 1 : min(a.V - 1, (unit * kUnitVecs + kUnitVecs - 32 + lane + 1) * kN + kN - 1));
    };
    bound = narrow(bound, a.n, a.part_cap - kPartExtra - a.n, best, red, turn, [&](auto f) {
        for (int i = t; i < units * 32; i += kPickThreads) f(lane_score[i], [&] { return part_last(unit_list[i >> 5]); });
    });
    for (int i = t; i < units * 32; i += kPickThreads) {
        const int u = unit_list[i >> 5];
        if (bound.has(lane_score[i], [&] { return part_first(u); })) {
            const int at = atomicAdd(&chosen_parts, 1);
            if (at < a.part_cap) part_list[at] = u << 5 | lane;
        }
    }
    __syncthreads();
    const int parts = min(chosen_parts, a.part_cap);

    // their elements: kPartVecs vectors each, and in a row's first unit what lies outside the vectors
    const auto elements = [&](auto f) {
        for (int i = t; i < parts * (kPartVecs + 1); i += kPickThreads) {
            const int part = part_list[i / (kPartVecs + 1)], k = i % (kPartVecs + 1);
            const int u = part >> 5, l = part & 31, beam = u / a.units, unit = u - beam * a.units;
            const T* x = a.logits + ((size_t)group * a.beams + beam) * a.ld;
            const RowShape<T> sh(x, a.V);
            if (k == kPartVecs) {
                const int e = unit == 0 ? sh.edge(l, a.V) : -1;
                if (e >= 0) f(score_of(elem(x, e), beam), [&] { return (uint32_t)beam << kTokenBits | (uint32_t)e; });
                continue;
            }
            const int v = unit * kUnitVecs + k * 32 + l;
            if (v >= sh.vecs) continue;
            const int token = sh.head + v * kN;
            float o[kN];
            Pack<T>::widen(load16(x + token), o);
#pragma unroll
            for (int j = 0; j < kN; j++) f(score_of(o[j], beam), [&] { return (uint32_t)beam << kTokenBits | (uint32_t)(token + j); });
        }
    };
    const auto gather = [&] {
        elements([&](double s, auto place) {
            if (!bound.has(s, place)) return;
            const int at = atomicAdd(&cands, 1);
            if (at < kMaxCands) {
                cand[at] = s;
                cand_place[at] = place();
            }
        });
        __syncthreads();
    };
    gather();
    if (cands > kMaxCands) {  // few parts hold them, or few parts there are
        __syncthreads();
        bound = narrow(bound, a.n, kMaxCands - a.n, best, red, turn, elements);
        if (t == 0) cands = 0;
        __syncthreads();
        gather();
    }
    if (t == 0 && cands > kMaxCands) cands = kMaxCands;
    __syncthreads();
    for (int i = t; i < a.beams; i += kPickThreads)
        if (state_s[i] == 1) {
            const int at = atomicAdd(&cands, 1);
            cand[at] = add_s[i];
            cand_place[at] = (uint32_t)i << kTokenBits;
        }
    __syncthreads();

    // in order: a candidate's place is how many are better
    const int found = cands, listed = min(found, a.n);
    const auto rank_of = [&](int i) {
        const double s = cand[i];
        const uint32_t place = cand_place[i];
        int rank = 0;
        for (int j = 0; j < found; j++) rank += cand[j] > s || (cand[j] == s && cand_place[j] < place);
        return rank;
    };
    const auto write = [&](int slot, double s, int parent, int token, bool ended) {
        a.out_scores[out + slot] = (float)s;
        a.tokens[out + slot] = token;
        if (a.parents) a.parents[out + slot] = parent;
        if (a.out_finished) a.out_finished[out + slot] = ended;
    };
    if (a.keep) {  // n = beams: where each goes
        for (int i = t; i < found; i += kPickThreads) {
            const int rank = rank_of(i);
            if (rank < a.n) parent_of[rank] = (unsigned char)(cand_place[i] >> kTokenBits);
        }
        __syncthreads();
        if (t == 0) {
            unsigned long long stay = 0, used = 0;
            for (int r = 0; r < listed; r++) stay |= 1ull << parent_of[r];
            for (int r = 0; r < a.n; r++) {
                const bool first = r < listed && !(used >> parent_of[r] & 1);
                const int slot = first ? parent_of[r] : __ffsll((long long)~(used | stay)) - 1;
                used |= 1ull << slot;
                slot_of[r] = (unsigned char)slot;
            }
        }
        __syncthreads();
    }
    for (int i = t; i < found; i += kPickThreads) {
        const int rank = rank_of(i);
        if (rank >= a.n) continue;
        const int beam = (int)(cand_place[i] >> kTokenBits);
        const bool was = state_s[beam] == 1;
        const int token = was ? a.pad : (int)(cand_place[i] & ((1u << kTokenBits) - 1));
        write(a.keep ? slot_of[rank] : rank, cand[i], beam, token, was || (a.eos >= 0 && token == a.eos));
    }
    for (int r = listed + t; r < a.n; r += kPickThreads) write(a.keep ? slot_of[r] : r, -(double)INFINITY, -1, -1, true);
}

// Workspace: the units' records, then the lanes' maxima.
static size_t parts_bytes(int dtype, long long rows, int vocab) {
    return round256((size_t)rows * row_units(dtype, vocab) * sizeof(float4));
}
static size_t best_workspace(int dtype, int rows, int vocab, int n) {
    if ((dtype != QS_F32 && dtype != QS_BF16) || rows < 1 || vocab < 1 || vocab > kMaxVocab || n < 1 || n > QS_MAX_LISTED) return 0;
    return parts_bytes(dtype, rows, vocab) + round256((size_t)rows * row_units(dtype, vocab) * 32 * (dtype == QS_F32 ? 4 : 2));
}

template <typename T>
static int best(const Rows& r, PickArgs<T> p, void* workspace, cudaStream_t st) {
    StreamArgs<T> s = {};
    s.logits = (const T*)r.logits;
    s.rows = r.rows;
    s.V = r.vocab;
    s.ld = r.ld;
    s.scores = p.scores;
    s.finished = p.finished;
    s.scale = (float)(r.inv_t * 1.4426950408889634);
    s.inv_t = r.inv_t;
    s.units = row_units(r.dtype, r.vocab);
    s.parts = (float4*)workspace;
    s.lanes = (T*)((char*)workspace + parts_bytes(r.dtype, r.rows, r.vocab));
    const int rc = stream_rows<T, true>(s, st);
    if (rc) return rc;
    p.logits = s.logits;
    p.V = s.V;
    p.ld = s.ld;
    p.units = s.units;
    p.parts = s.parts;
    p.lanes = s.lanes;
    p.scale = s.scale;
    p.inv_t = s.inv_t;
    const int units = p.beams * p.units, most = p.n + p.n / 4 + 8 + kUnitExtra;
    p.unit_cap = units < most ? units : most;
    p.part_cap = p.n + p.n / 4 + 16 + kPartExtra;
    const size_t smem = ((size_t)p.unit_cap * 32 + (p.unit_cap < units ? units : 0)) * sizeof(double) +
                        ((size_t)p.unit_cap + p.part_cap) * sizeof(int);
    static DeviceOnce once;
    const int e = once.raise((const void*)pick_kernel<T>, 216 * 1024);
    if (e) return e;
    return launch("pick_kernel", pick_kernel<T>, r.rows / p.beams, kPickThreads, 1, smem, true, st, p);
}

}  // namespace qs

using namespace qs;

extern "C" {

size_t qs_top_logprobs_workspace(int dtype, int rows, int vocab, int k) { return best_workspace(dtype, rows, vocab, k); }

int qs_top_logprobs(const void* d_logits, int dtype, int rows, int vocab, long long row_stride, int k,
                    double temperature, float* d_logprobs, int* d_tokens, void* d_workspace,
                    size_t workspace_bytes, void* stream) {
    set_error(QS_OK, "");
    const Rows r{d_logits, dtype, rows, vocab, row_stride, nullptr, 1.0 / temperature, nullptr, 0};
    int rc = check_rows(r, temperature, false);
    if (rc) return rc;
    if (k < 1 || k > QS_MAX_LISTED) return fail(QS_ERR_UNSUPPORTED, "k %d outside [1, %d]", k, QS_MAX_LISTED);
    if (rows == 0) return QS_OK;
    if (!d_logprobs || !d_tokens) return fail(QS_ERR_INVALID, "NULL output buffer");
    rc = check_workspace(d_workspace, workspace_bytes, best_workspace(dtype, rows, vocab, k));
    if (rc) return rc;
    const auto go = [&](auto p) {
        p.beams = 1;
        p.n = k;
        p.out_scores = d_logprobs;
        p.tokens = d_tokens;
        p.eos = -1;
        return best(r, p, d_workspace, (cudaStream_t)stream);
    };
    return dtype == QS_F32 ? go(PickArgs<float>{}) : go(PickArgs<__nv_bfloat16>{});
}

size_t qs_beam_select_workspace(int dtype, int batch, int beams, int vocab, int n) {
    if (batch < 1 || beams < 1 || beams > QS_MAX_BEAMS || batch > (1 << 27) / beams) return 0;
    return best_workspace(dtype, batch * beams, vocab, n);
}

int qs_beam_select(const void* d_logits, int dtype, int batch, int beams, int vocab, long long row_stride,
                   const float* d_scores, const unsigned char* d_finished, int n, const qs_beam_params* params,
                   float* d_out_scores, int* d_parents, int* d_tokens, unsigned char* d_out_finished,
                   void* d_workspace, size_t workspace_bytes, void* stream) {
    set_error(QS_OK, "");
    if (!params) return fail(QS_ERR_INVALID, "params is NULL");
    const qs_beam_params b = *params;
    if (batch < 0) return fail(QS_ERR_INVALID, "batch %d < 0", batch);
    if (beams < 1 || beams > QS_MAX_BEAMS) return fail(QS_ERR_UNSUPPORTED, "beams %d outside [1, %d]", beams, QS_MAX_BEAMS);
    if (batch > (1 << 27) / beams) return fail(QS_ERR_UNSUPPORTED, "%d x %d rows above 2^27", batch, beams);
    const Rows r{d_logits, dtype, batch * beams, vocab, row_stride, nullptr, 1.0 / b.temperature, nullptr, 0};
    int rc = check_rows(r, b.temperature, false);
    if (rc) return rc;
    if (n < 1 || n > QS_MAX_LISTED) return fail(QS_ERR_UNSUPPORTED, "n %d outside [1, %d]", n, QS_MAX_LISTED);
    if (b.keep_slots && n != beams) return fail(QS_ERR_INVALID, "keep_slots wants n %d = beams %d", n, beams);
    if (b.eos_token < -1 || b.eos_token >= vocab) return fail(QS_ERR_INVALID, "eos_token %d outside [-1, %d)", b.eos_token, vocab);
    if (batch == 0) return QS_OK;
    if (!d_scores) return fail(QS_ERR_INVALID, "NULL device pointer");
    if (!d_out_scores || !d_parents || !d_tokens) return fail(QS_ERR_INVALID, "NULL output buffer");
    rc = check_workspace(d_workspace, workspace_bytes, best_workspace(dtype, batch * beams, vocab, n));
    if (rc) return rc;
    const auto go = [&](auto p) {
        p.beams = beams;
        p.n = n;
        p.scores = d_scores;
        p.finished = d_finished;
        p.pad = b.pad_token;
        p.eos = b.eos_token;
        p.keep = b.keep_slots != 0;
        p.out_scores = d_out_scores;
        p.parents = d_parents;
        p.tokens = d_tokens;
        p.out_finished = d_out_finished;
        return best(r, p, d_workspace, (cudaStream_t)stream);
    };
    return dtype == QS_F32 ? go(PickArgs<float>{}) : go(PickArgs<__nv_bfloat16>{});
}

}  // extern "C"
