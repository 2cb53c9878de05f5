// Per-row states moved to the beams that go on, in place
// (include/qwen600_sampler.h gives the meaning).
//
// Within an entry, place i takes what place parents[i] held: a parallel move.
// A byte of the state depends only on the same byte of the entry's other rows, so
// a thread that carries out the whole move for its own bytes needs no second
// copy of the state and waits for nobody.  It follows a list of single moves, the
// same for every byte of the entry: places that nobody takes from any more are
// written first, which frees the places they took from; what is left are cycles,
// each broken with the thread's registers.
#include "qs_rows.cuh"

namespace qs {

constexpr int kMoveThreads = 256;
constexpr int kMoveVecs = 4;      // of a thread at a time
constexpr int kMaxChunks = 8;     // of a CTA
constexpr int kMaxMoveBeams = 1024;
constexpr int kMoveStates = 40;   // of a launch: they travel in its parameters

struct MoveState {
    char* base;
    long long row_stride, outer_stride[2], position_stride;
    uint32_t run_vecs;  // vectors of a run; of one position where positions lie behind one another
    uint32_t outer1;
    uint32_t outers;    // outer[0] * outer[1]
    int positions;
    int joined;         // positions behind one another: a run holds all that are moved
    int ctas;           // per entry
};

struct MoveArgs {
    MoveState s[kMoveStates];
    int first_cta[kMoveStates + 1];
    int count;
    const int* parents;
    int beams;
    const int* lengths;
};

template <int kBytes> struct MoveWord;
template <> struct MoveWord<1> { using T = unsigned char; };
template <> struct MoveWord<2> { using T = unsigned short; };
template <> struct MoveWord<4> { using T = unsigned; };
template <> struct MoveWord<8> { using T = uint2; };
template <> struct MoveWord<16> { using T = uint4; };

// The list of moves for `parents`, by one thread: list[i] = {place written, place
// read}; place written -1: into the registers' copy, place read -1: from it.  Returns
// its length, and 2^16 more where it has cycles.
__device__ int list_moves(const int* parents, int beams, short* readers, short* ready, short2* list) {
    int n = 0, todo = 0, front = 0, back = 0;
    for (int i = 0; i < beams; i++) readers[i] = 0;
    for (int i = 0; i < beams; i++) {
        const int p = parents[i];
        if (p >= 0) readers[p]++;
    }
    for (int i = 0; i < beams; i++)
        if (parents[i] >= 0) {
            todo++;
            if (readers[i] == 0) ready[back++] = (short)i;
        }
    while (front < back) {
        const int d = ready[front++], p = parents[d];
        list[n++] = make_short2((short)d, (short)p);
        readers[d] = -1;  // written
        todo--;
        if (--readers[p] == 0 && parents[p] >= 0) ready[back++] = (short)p;
    }
    const int cycles = todo > 0;
    for (int i = 0; todo > 0 && i < beams; i++) {
        if (parents[i] < 0 || readers[i] < 0) continue;
        // every place left is read by exactly one other: a cycle through i
        list[n++] = make_short2(-1, (short)i);
        int d = i;
        while (parents[d] != i) {
            list[n++] = make_short2((short)d, (short)parents[d]);
            readers[d] = -1;
            todo--;
            d = parents[d];
        }
        list[n++] = make_short2((short)d, -1);
        readers[d] = -1;
        todo--;
    }
    return n | cycles << 16;
}

// Loads that do not stay in L1: most places are read once.
template <typename W> __device__ __forceinline__ W take(const char* p) { return *reinterpret_cast<const W*>(p); }
template <> __device__ __forceinline__ uint4 take<uint4>(const char* p) { return load16(p); }

// The list for this thread's bytes of an entry's rows, kMoveVecs vectors at a time.
// kCycles: some moves go through the registers' copy.
template <int kBytes, bool kCycles>
__device__ __forceinline__ void move_bytes(const MoveState& s, int entry, int beams, int length, int cta, const short2* list, int n) {
    using W = typename MoveWord<kBytes>::T;
    const uint32_t run = s.joined ? s.run_vecs * (uint32_t)length : s.run_vecs;
    const uint32_t per_outer = s.joined ? run : run * (uint32_t)length;
    const uint32_t total = per_outer * s.outers;
    char* rows = s.base + (size_t)entry * beams * s.row_stride;
    for (uint32_t i0 = (uint32_t)cta * kMoveThreads * kMoveVecs + threadIdx.x; i0 < total;
         i0 += (uint32_t)s.ctas * kMoveThreads * kMoveVecs) {
        char* at[kMoveVecs];
#pragma unroll
        for (int j = 0; j < kMoveVecs; j++) {
            const uint32_t i = i0 + j * kMoveThreads;
            const uint32_t o = s.outers == 1 ? 0 : i / per_outer, in = i - o * per_outer;
            const uint32_t position = s.joined ? 0 : in / run, v = in - position * run;
            const uint32_t o0 = s.outer1 == 1 ? o : o / s.outer1, o1 = o - o0 * s.outer1;
            at[j] = i < total ? rows + (long long)o0 * s.outer_stride[0] + (long long)o1 * s.outer_stride[1] +
                                    (long long)position * s.position_stride + (size_t)v * kBytes
                              : nullptr;
        }
        W kept[kMoveVecs] = {};
        for (int k = 0; k < n; k++) {
            const short2 m = list[k];
            W v[kMoveVecs];
#pragma unroll
            for (int j = 0; j < kMoveVecs; j++) {
                if (kCycles && m.y < 0) v[j] = kept[j];
                else if (at[j]) v[j] = take<W>(at[j] + m.y * s.row_stride);
                if (kCycles && m.x < 0) kept[j] = v[j];
            }
            if (kCycles && m.x < 0) continue;
#pragma unroll
            for (int j = 0; j < kMoveVecs; j++)
                if (at[j]) *reinterpret_cast<W*>(at[j] + m.x * s.row_stride) = v[j];
        }
    }
}

// Bound: memory; 64 KB of loads under way on an SM.  56 caches of 8 entries x 4 beams of
// up to 1000 positions of 2 KB, half of the places written: 443 us for 2.87 GB, 6.5 TB/s (a
// copy's rate).  Several moves' loads at once 618 us, 8 vectors a thread 636, two or five
// CTAs an SM 553 and 506; lists without cycles have code without the registers' copy (465).
template <int kBytes>
__global__ void __launch_bounds__(kMoveThreads, 4)
reorder_kernel(const __grid_constant__ MoveArgs a) {
    extern __shared__ int smem[];
    int* parents = smem;                                            // [beams] -1: keeps its own
    short2* list = reinterpret_cast<short2*>(parents + a.beams);    // [2 beams]
    short* readers = reinterpret_cast<short*>(list + 2 * a.beams);  // [beams]
    short* ready = readers + a.beams;                               // [beams]
    __shared__ int moves_s;
    int i = 0;
    while (i + 1 < a.count && (int)blockIdx.x >= a.first_cta[i + 1]) i++;
    const MoveState& s = a.s[i];
    const int at = blockIdx.x - a.first_cta[i], entry = at / s.ctas, cta = at - entry * s.ctas;
    int length = s.positions;
    if (a.lengths) length = max(0, min(length, a.lengths[entry]));
    if (threadIdx.x == 0) moves_s = 0;
    bool some = false;
    for (int j = threadIdx.x; j < a.beams; j += kMoveThreads) {
        int p = a.parents[(size_t)entry * a.beams + j];
        if (p < 0 || p >= a.beams || p == j) p = -1;
        parents[j] = p;
        some |= p >= 0;
    }
    if (!__syncthreads_or(some) || length == 0) return;
    // where no place that is read is written (each beam's best child stayed in its place), any order will do
    bool meets = false;
    for (int j = threadIdx.x; j < a.beams; j += kMoveThreads) meets |= parents[j] >= 0 && parents[parents[j]] >= 0;
    if (__syncthreads_or(meets)) {
        if (threadIdx.x == 0) moves_s = list_moves(parents, a.beams, readers, ready, list);
    } else {
        for (int j = threadIdx.x; j < a.beams; j += kMoveThreads)
            if (parents[j] >= 0) list[atomicAdd(&moves_s, 1)] = make_short2((short)j, (short)parents[j]);
    }
    __syncthreads();
    const int n = moves_s & 0xFFFF;
    const bool cycles = moves_s >> 16;
    if (cycles) move_bytes<kBytes, true>(s, entry, a.beams, length, cta, list, n);
    else move_bytes<kBytes, false>(s, entry, a.beams, length, cta, list, n);
}

// --------------------------------------------------------------- host side
struct Level {
    long long stride, count;
};

// A state's levels in the order of their strides, without those of one piece;
// rows: how many lie row_stride apart.  Returns how many there are.
static int levels_of(const qs_states& s, int rows, Level* out) {
    const Level all[4] = {{s.position_stride, s.positions}, {s.outer_stride[0], s.outer[0]}, {s.outer_stride[1], s.outer[1]},
                          {s.row_stride, rows}};
    int n = 0;
    for (const Level& l : all) {
        if (l.count == 1) continue;
        int at = n++;
        for (; at > 0 && out[at - 1].stride > l.stride; at--) out[at] = out[at - 1];
        out[at] = l;
    }
    return n;
}

constexpr long long kMaxStride = 1ll << 44, kMaxSpan = 1ll << 46;  // bytes

// Bytes from the first to behind the last of the levels whose stride is below
// `under`; -1 where a level's pieces do not lie behind one another, or the last
// lies farther than any memory reaches (a product of 75 bits at most: divided, not
// multiplied).  `unit` is above 0.
static long long span_of(long long unit, const Level* l, int n, long long under) {
    long long span = unit;
    for (int i = 0; i < n && l[i].stride < under; i++) {
        if (l[i].stride < span || l[i].stride > kMaxStride || l[i].count - 1 > kMaxSpan / l[i].stride) return -1;
        span += (l[i].count - 1) * l[i].stride;
        if (span > kMaxSpan) return -1;
    }
    return span;
}
constexpr long long kAllLevels = 1ll << 62;

// Two states whose bytes lie between one another's do not meet if both repeat
// with the same stride, larger ones being its multiples, and are apart within it.
static bool apart_within(const qs_states& a, const Level* la, int na, const qs_states& b, const Level* lb, int nb) {
    const uintptr_t pa = (uintptr_t)a.d_base, pb = (uintptr_t)b.d_base;
    for (int i = 0; i < na; i++) {
        const long long stride = la[i].stride, sa = span_of(a.unit, la, na, stride), sb = span_of(b.unit, lb, nb, stride);
        bool fits = sa <= stride && sb <= stride;
        for (int k = 0; k < na; k++) fits &= la[k].stride < stride || la[k].stride % stride == 0;
        for (int k = 0; k < nb; k++) fits &= lb[k].stride < stride || lb[k].stride % stride == 0;
        if (!fits) continue;
        const long long d = (long long)((pa > pb ? pa - pb : pb - pa) % (uintptr_t)stride);
        if (d >= (pa > pb ? sb : sa) && d + (pa > pb ? sa : sb) <= stride) return true;
    }
    return false;
}

// The largest vectors that a state's addresses allow: 2^width bytes.
static int width_of(const qs_states& s, int rows) {
    unsigned long long bits = (unsigned long long)(uintptr_t)s.d_base | (unsigned long long)s.unit;
    Level l[4];
    const int n = levels_of(s, rows, l);
    for (int i = 0; i < n; i++) bits |= (unsigned long long)l[i].stride;
    int width = 0;
    while (width < 4 && !(bits >> width & 1)) width++;
    return width;
}
static long long vecs_of(const qs_states& s, int width) { return (s.unit >> width) * s.positions * s.outer[0] * s.outer[1]; }

// Each state for itself, and every pair of them: 29 us of host time for 56 states, where
// one takes 1.5.
static int check_states(const qs_states* all, int count, int rows) {
    for (int i = 0; i < count; i++) {
        const qs_states& s = all[i];
        if (!s.d_base) return fail(QS_ERR_INVALID, "state %d: NULL", i);
        if (s.unit < 1 || s.positions < 1 || s.outer[0] < 1 || s.outer[1] < 1)
            return fail(QS_ERR_INVALID, "state %d: a size below 1", i);
        Level l[4];
        const int n = levels_of(s, rows, l);
        if (s.unit > kMaxStride || span_of(s.unit, l, n, kAllLevels) < 0)
            return fail(QS_ERR_INVALID, "state %d: its pieces overlap, or its strides are not those of nested blocks", i);
        if ((double)s.unit * s.positions * s.outer[0] * s.outer[1] > 2147483647.0 * (1 << width_of(s, rows)))
            return fail(QS_ERR_UNSUPPORTED, "state %d: above 2^31 - 1 vectors of %d bytes in a row", i, 1 << width_of(s, rows));
        for (int j = 0; j < i; j++) {
            Level k[4];
            const int m = levels_of(all[j], rows, k);
            const uintptr_t a = (uintptr_t)s.d_base, b = (uintptr_t)all[j].d_base;
            if (a + span_of(s.unit, l, n, kAllLevels) <= b || b + span_of(all[j].unit, k, m, kAllLevels) <= a) continue;
            if (!apart_within(s, l, n, all[j], k, m)) return fail(QS_ERR_INVALID, "states %d and %d overlap", j, i);
        }
    }
    return QS_OK;
}

// Moves a call's states, as many at a time as a launch's parameters hold.  A CTA
// takes up to kMaxChunks chunks of 1024 vectors of a row (one more parents' list for each
// CTA otherwise), fewer where that would leave the call with less than two CTAs per SM.
int reorder_states(const qs_states* all, int count, const int* d_parents, int batch, int beams, const int* d_lengths,
                   cudaStream_t st) {
    if (batch < 0) return fail(QS_ERR_INVALID, "batch %d < 0", batch);
    if (beams < 1 || beams > kMaxMoveBeams) return fail(QS_ERR_UNSUPPORTED, "beams %d outside [1, %d]", beams, kMaxMoveBeams);
    if (batch > (1 << 27) / beams) return fail(QS_ERR_UNSUPPORTED, "%d x %d rows above 2^27", batch, beams);
    if (count < 0) return fail(QS_ERR_INVALID, "count %d < 0", count);
    if (batch == 0 || count == 0) return QS_OK;
    if (!all || !d_parents) return fail(QS_ERR_INVALID, "NULL pointer");
    const int rows = batch * beams;
    const int bad = check_states(all, count, rows);
    if (bad) return bad;
    for (int i = 0; i < count; i++) {
        Level l[4];
        const int levels = levels_of(all[i], rows, l);
        const uintptr_t from = (uintptr_t)all[i].d_base, to = from + span_of(all[i].unit, l, levels, kAllLevels);
        const uintptr_t p = (uintptr_t)d_parents, n = (uintptr_t)d_lengths;
        if ((p < to && from < p + rows * sizeof(int)) || (n && n < to && from < n + batch * sizeof(int)))
            return fail(QS_ERR_INVALID, "state %d overlaps the parents or lengths", i);
    }
    // states whose vectors have the same width go together
    for (int width = 0; width <= 4; width++) {
        int begin = 0;
        while (begin < count) {
            MoveArgs a = {};
            a.parents = d_parents;
            a.beams = beams;
            a.lengths = d_lengths;
            long long chunks = 0;
            for (; begin < count && a.count < kMoveStates; begin++) {
                const qs_states& s = all[begin];
                if (width_of(s, rows) != width) continue;
                MoveState& m = a.s[a.count++];
                m.base = (char*)s.d_base;
                m.row_stride = s.row_stride;
                m.outer_stride[0] = s.outer_stride[0];
                m.outer_stride[1] = s.outer_stride[1];
                m.position_stride = s.position_stride;
                m.positions = s.positions;
                m.outer1 = s.outer[1];
                m.joined = s.positions == 1 || s.position_stride == s.unit;
                m.run_vecs = (uint32_t)(s.unit >> width);
                m.outers = (uint32_t)s.outer[0] * s.outer[1];
                m.ctas = (int)((vecs_of(s, width) + kMoveThreads * kMoveVecs - 1) / (kMoveThreads * kMoveVecs));
                chunks += (long long)m.ctas * batch;
            }
            if (a.count == 0) break;
            const long long each = chunks / (148 * 2) < 1 ? 1 : chunks / (148 * 2) > kMaxChunks ? kMaxChunks : chunks / (148 * 2);
            long long grid = 0;
            for (int i = 0; i < a.count; i++) {
                a.s[i].ctas = (int)((a.s[i].ctas + each - 1) / each);
                a.first_cta[i] = (int)grid;
                grid += (long long)a.s[i].ctas * batch;
                if (grid > 0x7FFFFFFFll) return fail(QS_ERR_UNSUPPORTED, "reorder_kernel: %lld CTAs", grid);
            }
            a.first_cta[a.count] = (int)grid;
            const auto go = [&](auto kernel) {
                return launch("reorder_kernel", kernel, grid, kMoveThreads, 1, (size_t)beams * 16, false, st, a);
            };
            const int rc = width == 4   ? go(reorder_kernel<16>)
                           : width == 3 ? go(reorder_kernel<8>)
                           : width == 2 ? go(reorder_kernel<4>)
                           : width == 1 ? go(reorder_kernel<2>)
                                        : go(reorder_kernel<1>);
            if (rc) return rc;
        }
    }
    return QS_OK;
}

}  // namespace qs

using namespace qs;

extern "C" {

int qs_beam_reorder(const qs_states* states, int count, const int* d_parents, int batch, int beams, const int* d_lengths,
                    void* stream) {
    set_error(QS_OK, "");
    return reorder_states(states, count, d_parents, batch, beams, d_lengths, (cudaStream_t)stream);
}

}  // extern "C"
