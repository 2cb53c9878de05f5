// The best tokens of a row of logits with their log-probabilities, and a step of
// beam search over them (include/qwen600_sampler.h gives the formulas).
//
// Two kernels.  The stream (qs_stream.cuh) reads every row once and leaves, for
// each unit of 256 vectors, its maximum and sum of exponentials, and the maximum
// of each lane's part: 128 bytes, 64 bf16 or 32 fp32 elements.  The pick takes a
// group (a row, or the rows of an entry's beams), joins the sums, and narrows
// down: if n parts of a row have a maximum of at least v, then n elements do, so
// whatever is below v is none of the n best.  With v near the n-th largest maximum
// that leaves few more than n parts of 128 bytes to be read again, and few more
// than n elements to be ranked.
#include <type_traits>

#include "qs_rows.cuh"
#include "qs_stream.cuh"

namespace qs {

constexpr int kTokenBits = 18;
static_assert(kMaxVocab <= 1 << kTokenBits && QS_MAX_BEAMS <= 1 << (32 - kTokenBits), "beam and token in one word");
constexpr int kMaxCands = 2 * QS_MAX_LISTED;  // elements that are ranked, beside ended beams
// Parts that a bound may let through beyond those it counts: a part counts from
// the last place that it may hold on, and is looked at from its first.  Among equal
// scores that is a neighbour and the lanes of a row's first unit (some of which
// also hold what lies behind the row's last vector), and as many that count from
// the row's last place.
constexpr int kExtra = 96;
// Parts that are listed at most.  Their elements are counted in 16 bits: 64 bf16 a part,
// and up to 14 of each beam's row outside its vectors.
constexpr int kMaxParts = 3 * QS_MAX_LISTED + 2 * kExtra;
static_assert(kMaxParts * 64 + QS_MAX_BEAMS * 14 < 1 << 16, "counts of elements");
template <typename S> constexpr S kLowest = 0;  // the lowest finite number
template <> constexpr float kLowest<float> = -3.402823466e38f;
template <> constexpr double kLowest<double> = -1.7976931348623157e308;
constexpr int kMaxUnits = kMaxVocab / 4 / kUnitVecs;  // of a row

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
    int log_lanes;  // lanes of an item of the first narrowing: 32 (a unit), a vector of maxima, or 1
    int item_cap, part_cap;
    int staged;  // the lanes' maxima are brought to shared memory
    int coarse;  // few parts for what is wanted: their elements are narrowed down before any is listed
    const float* scores;            // of beams (NULL: 0)
    const unsigned char* finished;  // beams that go on with `pad` alone (NULL: none)
    int pad, eos, keep;
    float* out_scores;
    int* parents;  // NULL: rows' lists
    int* tokens;
    unsigned char* out_finished;
};

// What is left of a group's elements, by score and, among equal ones, by place:
// those above v, and those at v with a place up to `last`.  Scores are logits as
// they are (float), or sums over beams (double).
template <typename S>
struct Bound {
    S v;
    uint32_t last;
    template <typename Place>
    __device__ __forceinline__ bool has(S s, Place place) const { return s > v || (s == v && place() <= last); }
};

// Scores as whole numbers of the same order, and back.
__device__ __forceinline__ uint32_t key_of(float f) { return fkey(f + 0.0f); }
__device__ __forceinline__ float score_at(uint32_t k) { return fkey_inv(k); }
__device__ __forceinline__ unsigned long long key_of(double d) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(d + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double score_at(unsigned long long k) {
    return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

// An element that is ranked: larger numbers first.
template <typename S> struct Cand;
template <> struct Cand<float> {
    unsigned long long rank;  // the score's key, then the place from the end
    __device__ __forceinline__ Cand() {}
    __device__ __forceinline__ Cand(float s, uint32_t place) : rank((unsigned long long)key_of(s) << 32 | ~place) {}
    __device__ __forceinline__ static Cand last() { Cand c; c.rank = 0; return c; }
    __device__ __forceinline__ bool before(const Cand& o) const { return rank > o.rank; }
    __device__ __forceinline__ float score() const { return fkey_inv((uint32_t)(rank >> 32)); }
    __device__ __forceinline__ uint32_t place() const { return ~(uint32_t)rank; }
};
template <> struct __align__(16) Cand<double> {
    unsigned long long key;
    uint32_t at, unused;
    __device__ __forceinline__ Cand() {}
    __device__ __forceinline__ Cand(double s, uint32_t place) : key(key_of(s)), at(place), unused(0) {}
    __device__ __forceinline__ static Cand last() { Cand c; c.key = 0; c.at = c.unused = 0; return c; }
    __device__ __forceinline__ bool before(const Cand& o) const { return (key > o.key) | ((key == o.key) & (at < o.at)); }
    __device__ __forceinline__ double score() const { return score_at(key); }
    __device__ __forceinline__ uint32_t place() const { return at; }
};

template <int kThreads>
struct Counter {
    uint2 (*red)[kThreads / 32];  // [2]: used in turn, so that one barrier a sum is enough
    int turn;
    // Sums over the CTA, in every thread, each below 2^16.
    __device__ __forceinline__ int4 total(int4 c) {
        const uint2 own = make_uint2(__reduce_add_sync(0xffffffffu, (unsigned)(c.x | c.y << 16)),
                                     __reduce_add_sync(0xffffffffu, (unsigned)(c.z | c.w << 16)));
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = own;
        __syncthreads();
        uint2 s = red[turn][0];
#pragma unroll
        for (int w = 1; w < kThreads / 32; w++) {
            const uint2 o = red[turn][w];
            s.x += o.x;
            s.y += o.y;
        }
        return make_int4(s.x & 0xFFFF, s.x >> 16, s.y & 0xFFFF, s.y >> 16);
    }
};

// A bound that n items at least are within, and n + slack at most if their places
// allow it; `within` where that already has no more.  each(f) calls f(score,
// place) for this thread's items, place() being the item's; best: the largest
// score.  Three bounds are tried at a time: 1 to 1024 below the best ones first, then
// quarters of what is left of the scores (as whole numbers of their order, so
// that any scores come to an end), then of the places of equal ones.
template <typename S, int kThreads, typename Each>
__device__ __forceinline__ Bound<S> narrow(Bound<S> within, int n, int slack, S best, Counter<kThreads>& counter, Each each) {
    using K = decltype(key_of(best));
    K low = key_of(within.v), high = key_of(best) + 1;  // fewer than n from high on
    S below = 1;
    while (below == 1 || high - low > 1) {
        const bool first = below == 1, near = below <= 64;
        K k[3];
        S p[3];
#pragma unroll
        for (int i = 0; i < 3; i++) {
            const K range = high - low, part = (range >> 2) * (3 - i);
            k[i] = near ? key_of(best - below * (S)(1 << 2 * i)) : low + (part ? part : 1);
            p[i] = score_at(k[i]);
        }
        int4 c = make_int4(0, 0, 0, 0);
        if (first)
            each([&](S s, auto place) {
                c.x += s >= p[0];
                c.y += s >= p[1];
                c.z += s >= p[2];
                c.w += within.has(s, place);
            });
        else
            each([&](S s, auto) {
                c.x += s >= p[0];
                c.y += s >= p[1];
                c.z += s >= p[2];
            });
        c = counter.total(c);
        if (first && c.w <= n + slack) return within;
        below *= 64;
        // the largest of them that n items reach, if one is between low and high
        const int at = c.x >= n ? 0 : c.y >= n ? 1 : c.z >= n ? 2 : 3;
        const K fewer = at == 0 ? high : at == 1 ? k[0] : at == 2 ? k[1] : k[2];
        if (fewer < high && fewer > low) high = fewer;
        if (at == 3) continue;
        const int enough = at == 0 ? c.x : at == 1 ? c.y : c.z;
        const K there = at == 0 ? k[0] : at == 1 ? k[1] : k[2];
        if (there <= low) continue;
        if (enough <= n + slack) return Bound<S>{score_at(there), 0xFFFFFFFFu};
        low = there;
        below = 4096;  // between two of them
    }
    // more than n + slack, because many are equal: the first ones
    const S v = score_at(low);
    long long none = -1, enough = v == within.v ? within.last : 0xFFFFFFFFll;
    while (enough - none > 1) {
        long long p[3];
#pragma unroll
        for (int i = 0; i < 3; i++) p[i] = none + max((enough - none) * (i + 1) >> 2, 1ll);
        int4 c = make_int4(0, 0, 0, 0);
        each([&](S s, auto place) {
            if (!(s >= v)) return;
            const long long at = s > v ? -1 : (long long)place();
            c.x += at <= p[0];
            c.y += at <= p[1];
            c.z += at <= p[2];
        });
        c = counter.total(c);
        const int counts[3] = {c.x, c.y, c.z};
#pragma unroll
        for (int i = 2; i >= 0; i--) {
            if (counts[i] < n) none = max(none, p[i]);
            else enough = min(enough, p[i]);
        }
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (counts[i] >= n && counts[i] <= n + slack) return Bound<S>{v, (uint32_t)p[i]};
    }
    return Bound<S>{v, (uint32_t)enough};
}

// The usual way to a first bound: the items counted by their distance below the best,
// in 256 steps of a quarter.  The steps are made smaller within one that holds too many,
// and larger behind the last where fewer than n items came; where that does not end
// soon (many equal scores, or masks of finite numbers near which n lies) narrow() does.
// The CTA's threads find the same: an item is within if it is less than `from` below the
// best, or its step behind that is at most `step`.
constexpr int kSteps = 256;
struct Within {
    float best, from, per;  // steps a unit
    int step;               // -1: all; -2: not found
    // Below all of them, whatever was rounded.
    template <typename S>
    __device__ __forceinline__ S below() const {
        const S d = (S)(from + (float)(step + 1) / per);
        return step < 0 ? kLowest<S> : (S)best - d - (S)1e-6f * ((S)fabsf(best) + d);
    }
    __device__ __forceinline__ bool has(float s) const {
        const float d = best - s;
        return s > -INFINITY && (step == -1 || d < from || (int)fminf((d - from) * per, 1e6f) <= step);
    }
};

// each(f) calls f(score) for this thread's scores; `steps` is clear on entry.
template <int kThreads, typename Each>
__device__ __forceinline__ Within find_within(int n, int slack, float best, int* steps, int2* found, Each each) {
    const int t = threadIdx.x;
    Within w{best, 0.0f, 4.0f, -2};
    int before = 0;
    for (int pass = 0; pass < 4; pass++) {  // as long as every step's border is a number of 24 bits, so that none counts twice
        if (pass > 0) {
            for (int i = t; i <= kSteps; i += kThreads) steps[i] = 0;
            __syncthreads();
        }
        each([&](float s) {
            const float d = best - s;
            if (s > -INFINITY && d >= w.from) atomicAdd(&steps[(int)fminf((d - w.from) * w.per, (float)kSteps)], 1);
        });
        __syncthreads();
        if (t < 32) {  // eight steps a lane: where the count reaches n
            int own[kSteps / 32], sum = 0;
#pragma unroll
            for (int i = 0; i < kSteps / 32; i++) {
                own[i] = steps[t * (kSteps / 32) + i];
                sum += own[i];
            }
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (t >= o) upto += v;
            }
            const int total = __shfl_sync(0xffffffffu, upto, 31), all = before + total + steps[kSteps];
            if (t == 0) *found = make_int2(all <= n + slack ? -1 : -2, before + total);
            __syncwarp();
            int c = before + upto - sum;
            if (all > n + slack && c < n && c + sum >= n) {
#pragma unroll
                for (int i = 0; i < kSteps / 32; i++) {
                    if (c < n && c + own[i] >= n) *found = make_int2(t * (kSteps / 32) + i, c + own[i] <= n + slack ? -1 : c);
                    c += own[i];
                }
            }
        }
        __syncthreads();
        const int2 f = *found;
        if (f.x == -1 || (f.x >= 0 && f.y < 0)) {
            w.step = f.x;
            return w;
        }
        before = f.y;
        if (f.x >= 0) {
            w.from += (float)f.x / w.per;
            w.per *= (float)kSteps;
        } else {
            w.from += (float)kSteps / w.per;
            w.per /= (float)kSteps;
        }
    }
    return w;
}

// A group as the pick sees it.
template <typename T, bool kRows>
struct Group {
    using S = std::conditional_t<kRows, float, double>;
    static constexpr int kN = Pack<T>::kN;
    static constexpr int kPartVecs = kUnitVecs / 32;
    const T* logits;  // its first row
    const T* lanes;
    const float4* unit_parts;
    const unsigned char* state;  // of beams, 0: offers its tokens
    const float* max;            // of beams
    const double* add;           // and what their logits' distances from it are added to
    int* item_list;
    int* part_list;
    long long ld;
    double inv_t;
    float per_unit;  // 1 / units
    int V, units, lg;  // 2^lg lanes an item

    // An item's largest logit; of a beam that offers nothing -inf.
    __device__ __forceinline__ float item(int i) const {
        if (!kRows && state[beam_of(i >> (5 - lg))] != 0) return -INFINITY;
        if (lg == 5) return unit_parts[i].x;
        if (lg == 0) return elem(lanes, i);
        float o[kN];
        Pack<T>::widen(*reinterpret_cast<const uint4*>(lanes + (size_t)i * kN), o);
#pragma unroll
        for (int j = 1; j < kN; j++) o[0] = fmaxf(o[0], o[j]);
        return o[0];
    }
    __device__ __forceinline__ double logprob(float x, int beam) const { return ((double)x - (double)max[beam]) * inv_t + add[beam]; }
    __device__ __forceinline__ S score(float x, int beam) const {
        if constexpr (kRows) return x;
        else return logprob(x, beam);
    }
    // Exact: units are below 2^14, and the quotient's distance from a whole number is at least half a unit's share.
    __device__ __forceinline__ int beam_of(int unit) const { return kRows ? 0 : (int)(((float)unit + 0.5f) * per_unit); }
    // The first and the last place that `count` lanes from `id` on may hold (a lane's id: its unit's and its own number).
    __device__ __forceinline__ uint32_t first_place(int id) const {
        const int u = id >> 5, beam = beam_of(u), unit = u - beam * units;
        return (uint32_t)beam << kTokenBits | (unit == 0 ? 0u : (uint32_t)((unit * 32 + (id & 31)) * kPartVecs * kN));
    }
    __device__ __forceinline__ uint32_t last_place(int id, int count) const {
        const int u = id >> 5, beam = beam_of(u), unit = u - beam * units;
        const int behind = (unit * 32 + (id & 31) + count) * kPartVecs * kN;
        return (uint32_t)beam << kTokenBits | (uint32_t)(unit == 0 ? V - 1 : min(V - 1, behind + kN - 1));
    }
    // Vector i of the listed parts: its row, its first token, and the element outside the vectors that goes with it or -1.
    struct At {
        const T* row;
        int beam, token, edge;
        bool whole;  // a vector of the row
    };
    __device__ __forceinline__ At at(int i) const {
        const int id = part_list[i / kPartVecs], u = id >> 5, beam = beam_of(u), unit = u - beam * units;
        const T* row = logits + (long long)beam * ld;
        const RowShape<T> sh(row, V);
        const int vec = (unit * 32 + (id & 31)) * kPartVecs + i % kPartVecs;
        return At{row, beam, sh.head + vec * kN, unit == 0 && i % kPartVecs == 0 ? sh.edge(id & 31, V) : -1, vec < sh.vecs};
    }
};

// Narrows by the items, by the listed items' lanes, or by the listed parts' elements: out
// of line so that the usual way's values stay in registers.  Of full vocabularies few calls
// reach it.  Short rows with short lists do by their size alone: where all items fit into the
// first list the bound stays at the lowest number, and lanes or elements are narrowed down
// instead.  One bf16 row's best token: 36 us of 10,000 columns, 20 of 4,000 (by elements), 7.5
// of 40,000; a step of 4 beams of 2,000 54, of 151,936 10.2.
enum { kByItems, kByLanes, kByElements };

template <typename T, bool kRows, int kThreads>
__device__ __noinline__ Bound<typename Group<T, kRows>::S> narrow_by(Group<T, kRows> g, int by, int count,
                                                                     Bound<typename Group<T, kRows>::S> within, int n, int slack,
                                                                     typename Group<T, kRows>::S best, uint2 (*red)[kThreads / 32]) {
    using S = typename Group<T, kRows>::S;
    __syncthreads();
    Counter<kThreads> counter{red, 0};
    const Bound<S> b = narrow(within, n, slack, best, counter, [&](auto f) {
        if (by == kByItems) {
            for (int i = threadIdx.x; i < count; i += kThreads)
                f(g.score(g.item(i), g.beam_of(i >> (5 - g.lg))), [&] { return g.last_place(i << g.lg, 1 << g.lg); });
            return;
        }
        if (by == kByLanes) {
            for (int i = threadIdx.x; i < count << g.lg; i += kThreads) {
                const int id = (g.item_list[i >> g.lg] << g.lg) + (i & ((1 << g.lg) - 1));
                f(g.score(elem(g.lanes, id), g.beam_of(id >> 5)), [&] { return g.last_place(id, 1); });
            }
            return;
        }
        for (int i = threadIdx.x; i < count * g.kPartVecs; i += kThreads) {
            const auto at = g.at(i);
            const uint32_t beam = (uint32_t)at.beam << kTokenBits;
            if (at.whole)
                for (int j = 0; j < g.kN; j++)
                    f(g.score(elem(at.row, at.token + j), at.beam), [&] { return beam | (uint32_t)(at.token + j); });
            if (at.edge >= 0) f(g.score(elem(at.row, at.edge), at.beam), [&] { return beam | (uint32_t)at.edge; });
        }
    });
    __syncthreads();
    return b;
}

// A score rounded to fp32 as the steps take it.
__device__ __forceinline__ float rounded(float s) { return s; }
__device__ __forceinline__ float rounded(double s) { return s > -(double)INFINITY ? fmaxf((float)s, kLowest<float>) : -INFINITY; }

// By the listed parts' elements, counted in steps: where few parts there are (small
// vocabularies and long lists) they hold thousands.  `steps` need not be clear.
template <typename T, bool kRows, int kThreads>
__device__ __noinline__ Bound<typename Group<T, kRows>::S> step_by_elements(Group<T, kRows> g, int count,
                                                                            Bound<typename Group<T, kRows>::S> within, int n, int slack,
                                                                            typename Group<T, kRows>::S best, uint2 (*red)[kThreads / 32],
                                                                            int* steps, int2* found) {
    using S = typename Group<T, kRows>::S;
    __syncthreads();
    for (int i = threadIdx.x; i <= kSteps; i += kThreads) steps[i] = 0;
    __syncthreads();
    const Within w = find_within<kThreads>(n, slack, rounded(best), steps, found, [&](auto f) {
        for (int i = threadIdx.x; i < count * g.kPartVecs; i += kThreads) {
            const auto at = g.at(i);
            if (at.whole) {
                float o[Group<T, kRows>::kN];
                Pack<T>::widen(load16(at.row + at.token), o);
#pragma unroll
                for (int j = 0; j < g.kN; j++) f(rounded(g.score(o[j], at.beam)));
            }
            if (at.edge >= 0) f(rounded(g.score(elem(at.row, at.edge), at.beam)));
        }
    });
    if (w.step == -1) return within;  // no more than that
    if (w.step < 0 || !(w.template below<S>() > within.v))
        return narrow_by<T, kRows, kThreads>(g, kByElements, count, within, n, slack, best, red);
    __syncthreads();
    return Bound<S>{w.template below<S>(), 0xFFFFFFFFu};
}

// By the items, and lists them.
template <typename T, bool kRows, int kThreads>
__device__ __noinline__ Bound<typename Group<T, kRows>::S> list_items(Group<T, kRows> g, int items, int n, int cap,
                                                                      typename Group<T, kRows>::S best, uint2 (*red)[kThreads / 32],
                                                                      int* listed) {
    using S = typename Group<T, kRows>::S;
    const Bound<S> b = narrow_by<T, kRows, kThreads>(g, kByItems, items, Bound<S>{kLowest<S>, 0xFFFFFFFFu}, n, cap - kExtra - n, best, red);
    for (int i = threadIdx.x; i < items; i += kThreads)
        if (b.has(g.score(g.item(i), g.beam_of(i >> (5 - g.lg))), [&] { return g.first_place(i << g.lg); })) {
            const int at = atomicAdd(listed, 1);
            if (at < cap) g.item_list[at] = i;
        }
    return b;
}

// Element j of a vector.
template <typename T>
__device__ __forceinline__ float element(const uint4& w, int j) {
    constexpr int kLog = Pack<T>::kN == 8 ? 1 : 0;  // of a word's elements
    const int i = j >> kLog;
    const uint32_t word = i < 2 ? (i == 0 ? w.x : w.y) : (i == 2 ? w.z : w.w);
    float o[1 << kLog];
    Pack<T>::widen_word(word, o);
    return j & kLog ? o[kLog] : o[0];
}

// Bound: latency.  A group's chain of dependent steps (sums, items, bound, parts,
// elements, ranks) takes 10 to 20 thousand cycles, most of them round trips to memory and
// barriers; 1024 rows' lists of 64 take 13 us behind a stream of 57, one row's of 20 8.1
// with its stream, an entry of 4 beams 10.6.  More threads for long lists: 250 of 61 rows
// 18 us with 512, 35 with 256; for several beams' sums a warp each.  64 registers for rows
// (128 for beams) keep 1024 (512) threads on an SM; 68 to 84 bytes a thread of rows spill
// then, 20 to 76 of beams.  Ranks compare all candidates with one another: up to 512 of them.
//
// One CTA per group.  kRows: a group is a row, and its logits are the scores that
// are compared; else they are the beams' sums.
template <typename T, bool kRows, int kThreads>
__global__ void __launch_bounds__(kThreads, (kRows ? 1024 : 512) / kThreads)
pick_kernel(const __grid_constant__ PickArgs<T> a) {
    using G = Group<T, kRows>;
    using S = typename G::S;
    constexpr int kN = Pack<T>::kN;
    constexpr int kPartVecs = G::kPartVecs;
    constexpr int kWarps = kThreads / 32;
    constexpr int kRoom = kMaxCands + (kRows ? 0 : QS_MAX_BEAMS);
    extern __shared__ __align__(16) unsigned char pool[];
    float* item_score = reinterpret_cast<float*>(pool);  // of sums, rounded
    __shared__ double add_s[kRows ? 1 : QS_MAX_BEAMS];
    __shared__ float max_s[kRows ? 1 : QS_MAX_BEAMS], floor_s[kRows ? 1 : QS_MAX_BEAMS];
    __shared__ unsigned char state_s[kRows ? 1 : QS_MAX_BEAMS];  // 0: offers its tokens, 1: ended, 2: nothing, 3: NaN
    __shared__ __align__(16) unsigned char cand_raw[kRoom * sizeof(Cand<S>)];
    __shared__ short rank_s[kRoom];
    __shared__ uint2 red[2][kWarps];
    __shared__ double sum_s[kWarps];
    __shared__ float top_s[kWarps];
    __shared__ int items_s, parts_s, cands_s, steps[kSteps + 1];
    __shared__ int2 found_s;
    __shared__ unsigned char slot_of[QS_MAX_BEAMS], parent_of[QS_MAX_BEAMS];
    __shared__ unsigned owns_s[2], stays_s[2];
    Cand<S>* cand = reinterpret_cast<Cand<S>*>(cand_raw);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, group = blockIdx.x;
    const int beams = kRows ? 1 : a.beams;
    const int lg = a.log_lanes, all_items = beams * a.units << (5 - lg);
    int* item_list = reinterpret_cast<int*>(item_score + all_items);  // [item_cap]
    int* part_list = item_list + a.item_cap;                          // [part_cap]
    if (t == 0) {
        items_s = parts_s = cands_s = 0;
    }
    for (int i = t; i <= kSteps; i += kThreads) steps[i] = 0;
    dependents_may_start();
    wait_for_previous();
    const float4* unit_parts = a.parts + (size_t)group * beams * a.units;
    const T* all_lanes = a.lanes + (size_t)group * beams * a.units * 32;
    T* stage = reinterpret_cast<T*>((reinterpret_cast<uintptr_t>(part_list + a.part_cap) + 15) & ~(uintptr_t)15);
    const G g{a.logits + (size_t)group * beams * a.ld, a.staged ? stage : all_lanes, unit_parts, state_s, max_s, add_s, item_list,
              part_list, a.ld, a.inv_t, 1.0f / (float)a.units, a.V, a.units, lg};
    const auto no_part = [] { return make_float4(-INFINITY, 0.0f, 0.0f, 0.0f); };
    // a unit's sum against the row's maximum
    const auto sum_of = [&](const float4& v, float M) {
        return v.x == M ? (double)v.y + (double)v.z : (double)(exp2_fast((v.x - M) * a.scale) * (v.y + v.z));
    };
    // 0: a distribution, 2: everything masked, 3: none
    const auto state_of = [](float M, double sum) { return M == -INFINITY ? (sum == 0.0 ? 2 : 3) : M < INFINITY && sum == sum ? 0 : 3; };

    // each beam's maximum and sum, a warp each
    if (!kRows) {
        for (int i = warp; i < beams; i += kWarps) {
            const size_t row = (size_t)group * beams + i;
            const double base = a.scores ? (double)a.scores[row] : 0.0;
            int state = base < INFINITY ? (base > -INFINITY ? (a.finished && a.finished[row] ? 1 : 0) : 2) : 3;
            double add = base;
            float M = -INFINITY;
            if (state == 0) {
                const float4* p = unit_parts + (size_t)i * a.units;
                double sum = 0.0;
                if (a.units <= 128) {
                    float4 v[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) v[k] = lane + 32 * k < a.units ? p[lane + 32 * k] : no_part();
                    M = warp_max(fmaxf(fmaxf(v[0].x, v[1].x), fmaxf(v[2].x, v[3].x)));
#pragma unroll
                    for (int k = 0; k < 4; k++) sum += sum_of(v[k], M);
                } else {
                    for (int u = lane; u < a.units; u += 32) M = fmaxf(M, p[u].x);
                    M = warp_max(M);
                    for (int u = lane; u < a.units; u += 32) sum += sum_of(p[u], M);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                state = state_of(M, sum);
                if (state == 0) add = base - log(sum);
            }
            if (lane == 0) {
                add_s[i] = add;
                max_s[i] = M;
                state_s[i] = (unsigned char)state;
            }
        }
        __syncthreads();
    }
    // of a row: one or two units a thread, requested before anything waits
    constexpr int kMine = (kMaxUnits + kThreads - 1) / kThreads;
    float4 mine[kMine];
    if (kRows)
#pragma unroll
        for (int k = 0; k < kMine; k++) mine[k] = t + k * kThreads < a.units ? unit_parts[t + k * kThreads] : no_part();

    // the lanes' maxima, and the items' scores; four loads under way
    constexpr int kLog = kN == 8 ? 3 : 2;
    float top = -INFINITY;
    const auto put_item = [&](int i, float x, int beam) {
        const bool offered = kRows || state_s[beam] == 0;
        if (offered) top = fmaxf(top, x);
        item_score[i] = offered && x > -INFINITY ? fmaxf((float)g.score(x, beam), kLowest<float>) : -INFINITY;
    };
    if (a.staged || lg == kLog) {
        const int vecs = beams * a.units * (32 / kN);
        for (int i0 = t; i0 < vecs; i0 += 4 * kThreads) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i0 + j * kThreads < vecs) v[j] = load16(all_lanes + (size_t)(i0 + j * kThreads) * kN);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = i0 + j * kThreads;
                if (i >= vecs) break;
                if (a.staged) reinterpret_cast<uint4*>(stage)[i] = v[j];
                if (lg != kLog) continue;
                float o[kN];
                Pack<T>::widen(v[j], o);
#pragma unroll
                for (int k = 1; k < kN; k++) o[0] = fmaxf(o[0], o[k]);
                put_item(i, o[0], g.beam_of(i >> (5 - kLog)));
            }
        }
    }
    if (kRows && lg == 5) {
#pragma unroll
        for (int k = 0; k < kMine; k++)
            if (t + k * kThreads < a.units) put_item(t + k * kThreads, mine[k].x, 0);
    } else if (lg != kLog) {
        if (lg == 0) __syncthreads();
        for (int i0 = t; i0 < all_items; i0 += 4 * kThreads) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = i0 + j * kThreads;
                if (i < all_items) x[j] = lg == 5 ? unit_parts[i].x : elem(g.lanes, i);
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i0 + j * kThreads < all_items) put_item(i0 + j * kThreads, x[j], g.beam_of((i0 + j * kThreads) >> (5 - lg)));
        }
    }
    S best = -(S)INFINITY;
    bool bad = false;
    if constexpr (kRows) {
        top = warp_max(top);
        if (lane == 0) top_s[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; w++) best = fmaxf(best, top_s[w]);
        double sum = 0.0;
#pragma unroll
        for (int k = 0; k < kMine; k++) sum += sum_of(mine[k], best);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) sum_s[warp] = sum;
    } else {
        for (int i = 0; i < beams; i++) {
            bad |= state_s[i] == 3;
            if (state_s[i] == 0) best = fmax(best, add_s[i]);
        }
        __syncthreads();
    }
    const size_t out = (size_t)group * a.n;
    if (!bad) {
        const Within within =
            find_within<kThreads>(a.n, a.item_cap - kExtra - a.n, fmaxf((float)best, kLowest<float>), steps, &found_s, [&](auto f) {
                for (int i = t; i < all_items; i += kThreads) f(item_score[i]);
            });
        Bound<S> bound{kLowest<S>, 0xFFFFFFFFu};
        if (within.step > -2) {
            for (int i = t; i < all_items; i += kThreads)
                if (within.has(item_score[i])) {
                    const int at = atomicAdd(&items_s, 1);
                    if (at < a.item_cap) item_list[at] = i;
                }
            bound.v = within.below<S>();
        } else {
            bound = list_items<T, kRows, kThreads>(g, all_items, a.n, a.item_cap, best, red, &items_s);
        }
        __syncthreads();
        if (kRows && t == kThreads - 1) {  // needed when the list is written
            double sum = 0.0;
            for (int w = 0; w < kWarps; w++) sum += sum_s[w];
            max_s[0] = (float)best;
            add_s[0] = -log(sum);
            state_s[0] = (unsigned char)state_of((float)best, sum);
        }
        const int items = min(items_s, a.item_cap);

        // Their lanes' parts.  A logit is held against the least that its score's bound wants of it first (of a beam: or a
        // little less); few pass, and of those the score itself decides.
        while (true) {
            if constexpr (!kRows) {
                for (int i = t; i < beams; i += kThreads) {
                    // the sum's rounding, 2^-53 of its parts, hides what is smaller
                    const double x = (double)max_s[i] + (bound.v - add_s[i] - 1e-15 * (fabs(bound.v) + fabs(add_s[i]))) / a.inv_t;
                    floor_s[i] = __double2float_rd(x - 1e-6 * (fabs(x) + fabs((double)max_s[i])));
                }
                __syncthreads();
            }
            if (lg == 0) {
                for (int i = t; i < items; i += kThreads) part_list[i] = item_list[i];
                if (t == 0) parts_s = items;
            } else {
                const int more = lg - kLog, vecs = items << more;  // a vector of lanes at a time
                for (int i = t; i < vecs; i += kThreads) {
                    const int id = (item_list[i >> more] << lg) + ((i & ((1 << more) - 1)) << kLog), beam = g.beam_of(id >> 5);
                    const uint4 w = *reinterpret_cast<const uint4*>(g.lanes + id);
                    float least, o[kN];
                    if constexpr (kRows) least = bound.v;
                    else least = floor_s[beam];
                    Pack<T>::widen(w, o);
                    uint32_t hits = 0;
#pragma unroll
                    for (int k = 0; k < kN; k++) hits |= o[k] >= least ? 1u << k : 0u;
                    for (; hits; hits &= hits - 1) {
                        const int k = __ffs(hits) - 1;
                        if (!bound.has(g.score(element<T>(w, k), beam), [&] { return g.first_place(id + k); })) continue;
                        const int at = atomicAdd(&parts_s, 1);
                        if (at < a.part_cap) part_list[at] = id + k;
                    }
                }
            }
            __syncthreads();
            if (parts_s <= a.part_cap) break;
            bound = narrow_by<T, kRows, kThreads>(g, kByLanes, items, bound, a.n, a.part_cap - kExtra - a.n, best, red);
            if (t == 0) parts_s = 0;
            __syncthreads();
        }
        const int parts = min(parts_s, a.part_cap);

        // Their elements, in the same way: kPartVecs vectors a part, and in a row's first unit what lies outside the vectors.
        if (a.coarse) {
            bound = step_by_elements<T, kRows, kThreads>(g, parts, bound, a.n, kMaxCands - 64 - a.n, best, red, steps, &found_s);
            if constexpr (!kRows) {
                for (int i = t; i < beams; i += kThreads) floor_s[i] = -INFINITY;  // the score decides
                __syncthreads();
            }
        }
        for (int again = a.coarse;; again++) {
            const int vecs = parts * kPartVecs;
            for (int i0 = t; i0 < vecs; i0 += 4 * kThreads) {
                uint4 w[4];
                float least[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    w[j] = Pack<T>::lowest();
                    least[j] = INFINITY;
                    if (i0 + j * kThreads < vecs) {
                        const auto at = g.at(i0 + j * kThreads);
                        if (at.whole) w[j] = load16(at.row + at.token);
                        if constexpr (kRows) least[j] = bound.v;
                        else least[j] = floor_s[at.beam];
                    }
                }
                uint32_t hits = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float o[kN];
                    Pack<T>::widen(w[j], o);
#pragma unroll
                    for (int k = 0; k < kN; k++) hits |= o[k] >= least[j] ? 1u << (j * kN + k) : 0u;
                }
                for (; hits; hits &= hits - 1) {
                    const int bit = __ffs(hits) - 1;
                    const auto at = g.at(i0 + bit / kN * kThreads);
                    const int token = at.token + bit % kN;
                    if (!at.whole) continue;
                    const int j = bit / kN;
                    const uint4 v = j < 2 ? (j == 0 ? w[0] : w[1]) : (j == 2 ? w[2] : w[3]);
                    const S s = g.score(element<T>(v, bit % kN), at.beam);
                    const uint32_t place = (uint32_t)at.beam << kTokenBits | (uint32_t)token;
                    if (!bound.has(s, [&] { return place; })) continue;
                    const int slot = atomicAdd(&cands_s, 1);
                    if (slot < kMaxCands) cand[slot] = Cand<S>(s, place);
                }
            }
            for (int i = t; i < parts; i += kThreads) {
                const auto at = g.at(i * kPartVecs);
                if (at.edge < 0) continue;
                const S s = g.score(elem(at.row, at.edge), at.beam);
                const uint32_t place = (uint32_t)at.beam << kTokenBits | (uint32_t)at.edge;
                if (!bound.has(s, [&] { return place; })) continue;
                const int slot = atomicAdd(&cands_s, 1);
                if (slot < kMaxCands) cand[slot] = Cand<S>(s, place);
            }
            __syncthreads();
            if (cands_s <= kMaxCands) break;  // else few parts hold them, or few parts there are
            // by steps first, with room for what rounding lets through, then exactly
            if (again == 0) bound = step_by_elements<T, kRows, kThreads>(g, parts, bound, a.n, kMaxCands - 64 - a.n, best, red, steps, &found_s);
            else bound = narrow_by<T, kRows, kThreads>(g, kByElements, parts, bound, a.n, kMaxCands - a.n, best, red);
            if (t == 0) cands_s = 0;
            if constexpr (!kRows) {
                for (int i = t; i < beams; i += kThreads) floor_s[i] = -INFINITY;  // the score decides
            }
            __syncthreads();
        }
        if constexpr (!kRows) {
            __syncthreads();  // all have seen that there is room
            for (int i = t; i < beams; i += kThreads)
                if (state_s[i] == 1) cand[atomicAdd(&cands_s, 1)] = Cand<S>(add_s[i], (uint32_t)i << kTokenBits);
            __syncthreads();
        }
    }

    // in order: a candidate's place is how many are better
    const int found = cands_s, padded = (found + 7) & ~7;
    if (t < padded - found) cand[found + t] = Cand<S>::last();
    __syncthreads();
    for (int i = t; i < found; i += kThreads) {
        const Cand<S> c = cand[i];
        int rank = 0;
        for (int j = 0; j < padded; j += 8)
#pragma unroll
            for (int k = 0; k < 8; k++) rank += cand[j + k].before(c);
        rank_s[i] = (short)rank;
    }
    __syncthreads();
    const bool nan = bad || (kRows && state_s[0] == 3);
    const int listed = nan ? 0 : min(found, a.n);
    const auto write = [&](int slot, double s, int parent, int token, bool ended) {
        a.out_scores[out + slot] = (float)s;
        a.tokens[out + slot] = token;
        if (kRows) return;
        a.parents[out + slot] = parent;
        if (a.out_finished) a.out_finished[out + slot] = ended;
    };
    const bool keep = !kRows && a.keep;
    if (keep) {  // n = beams: where each goes
        for (int i = t; i < found; i += kThreads)
            if (rank_s[i] < a.n) parent_of[rank_s[i]] = (unsigned char)(cand[i].place() >> kTokenBits);
        __syncthreads();
        // rank r's beam stays in its place if no better rank has the same; the others take the places left, in order
        if (t < QS_MAX_BEAMS) {
            bool own = t < listed, kept = false;
            for (int r = 0; r < listed; r++) {
                own &= !(r < t && parent_of[r] == parent_of[t]);
                kept |= parent_of[r] == t;
            }
            const unsigned owns = __ballot_sync(0xffffffffu, own), stays = __ballot_sync(0xffffffffu, kept);
            if (lane == 0) {
                owns_s[warp] = owns;
                stays_s[warp] = stays;
            }
        }
        __syncthreads();
        if (t < a.n) {
            const unsigned long long owns = owns_s[0] | (unsigned long long)owns_s[1] << 32;
            unsigned long long left = ~(stays_s[0] | (unsigned long long)stays_s[1] << 32);
            int slot = parent_of[t];
            if (!(owns >> t & 1)) {
                for (int k = __popcll(~owns & ((1ull << t) - 1)); k > 0; k--) left &= left - 1;
                slot = __ffsll((long long)left) - 1;
            }
            slot_of[t] = (unsigned char)slot;
        }
        __syncthreads();
    }
    for (int i = t; i < found; i += kThreads) {
        const int rank = rank_s[i];
        if (rank >= listed) continue;
        const Cand<S> c = cand[i];
        const uint32_t place = c.place();
        const int beam = kRows ? 0 : (int)(place >> kTokenBits);
        const bool was = !kRows && state_s[beam] == 1;
        const int token = was ? a.pad : (int)(place & ((1u << kTokenBits) - 1));
        write(keep ? slot_of[rank] : rank, kRows ? g.logprob((float)c.score(), 0) : (double)c.score(), beam, token,
              was || (a.eos >= 0 && token == a.eos));
    }
    for (int r = listed + t; r < a.n; r += kThreads) write(keep ? slot_of[r] : r, nan ? (double)NAN : -(double)INFINITY, -1, -1, true);
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
    // the first narrowing's items: three times as many as are wanted, so that a bound near the n-th lets few others through
    const int units = p.beams * p.units, log_n = r.dtype == QS_F32 ? 2 : 3;
    p.log_lanes = units >= 3 * p.n ? 5 : units << (5 - log_n) >= 3 * p.n ? log_n : 0;
    p.item_cap = p.n + p.n / 4 + 16 + kExtra;
    p.part_cap = 3 * p.n + 2 * kExtra;
    p.coarse = (long long)units * 32 < 2 * p.n;  // 700 bf16 rows of 15,000, 256 listed: 85 us without, 50 with it
    // The lanes' maxima go to shared memory where all of them are looked at (40 KB leave room for several groups an SM);
    // where units are narrowed down first, few are, and are read when their units are known.
    const size_t lanes = (size_t)units * 32 * sizeof(T), items = (size_t)units << (5 - p.log_lanes);
    p.staged = p.log_lanes != 5 && lanes <= 40 * 1024;
    const auto go = [&](auto kernel, int threads, DeviceOnce& once) {
        const int e = once.raise((const void*)kernel, 160 * 1024);
        if (e) return e;
        const size_t smem = items * sizeof(float) + ((size_t)p.item_cap + p.part_cap) * sizeof(int) + (p.staged ? lanes + 16 : 0);
        return launch("pick_kernel", kernel, r.rows / p.beams, threads, 1, smem, true, st, p);
    };
    static DeviceOnce once[4];
    if (!p.parents) return p.n > 64 ? go(pick_kernel<T, true, 512>, 512, once[0]) : go(pick_kernel<T, true, 128>, 128, once[1]);
    return p.n > 64 || p.beams > 4 ? go(pick_kernel<T, false, 256>, 256, once[2]) : go(pick_kernel<T, false, 128>, 128, once[3]);
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
    const size_t in = (size_t)batch * beams, out = (size_t)batch * n;
    const struct { const void* p; size_t bytes; } reads[] = {{d_scores, in * sizeof(float)}, {d_finished, in}},
        writes[] = {{d_out_scores, out * sizeof(float)}, {d_parents, out * sizeof(int)}, {d_tokens, out * sizeof(int)}, {d_out_finished, out}};
    for (const auto& r : reads)
        for (const auto& w : writes)
            if (r.p && w.p && (uintptr_t)r.p < (uintptr_t)w.p + w.bytes && (uintptr_t)w.p < (uintptr_t)r.p + r.bytes)
                return fail(QS_ERR_INVALID, "an output overlaps the scores or marks");
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
