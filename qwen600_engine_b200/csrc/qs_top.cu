// The best tokens of a row of logits with their log-probabilities, and a step of
// beam search over them (include/qwen600_sampler.h gives the formulas).
#include "qs_rows.cuh"

namespace qs {

struct BestArgs {
    const void* logits;
    int rows, V;
    long long ld;
    int n;
    float scale;
    double inv_t;
    const float* scores;            // of beams (NULL: 0)
    const unsigned char* finished;  // beams that go on with `pad` alone (NULL: none)
    int pad;
    double* value;                  // [rows][n] the row's best, in order
    int* token;
};

constexpr int kBestThreads = 256;

__device__ __forceinline__ unsigned long long best_key(float v, int token) {
    return (unsigned long long)fkey(v + 0.0f) << 32 | (0xFFFFFFFFu - (uint32_t)token);
}

// One CTA per row: maximum, sum, then one pass for each listed token.
template <typename T>
__global__ void __launch_bounds__(kBestThreads)
best_rows_kernel(const BestArgs a) {
    __shared__ float redf[kBestThreads / 32];
    __shared__ double redd[kBestThreads / 32];
    __shared__ unsigned long long redk[kBestThreads / 32];
    __shared__ double total_s;
    __shared__ unsigned long long best_s;
    const int row = blockIdx.x, t = threadIdx.x;
    const T* x = (const T*)a.logits + (size_t)row * a.ld;
    double* value = a.value + (size_t)row * a.n;
    int* token = a.token + (size_t)row * a.n;
    const double base = a.scores ? (double)a.scores[row] : 0.0;
    const bool done = a.finished && a.finished[row];
    if (done || !(fabs(base) < INFINITY)) {
        const bool nan = !(base < INFINITY);
        for (int i = t; i < a.n; i += kBestThreads) {
            value[i] = nan ? (double)NAN : done && i == 0 ? base : -(double)INFINITY;
            token[i] = !nan && done && i == 0 && base > -INFINITY ? a.pad : -1;
        }
        return;
    }
    float m = -INFINITY;
    for (int j = t; j < a.V; j += kBestThreads) m = fmaxf(m, elem(x, j));
    m = warp_max(m);
    if ((t & 31) == 0) redf[t >> 5] = m;
    __syncthreads();
    for (int w = 0; w < kBestThreads / 32; w++) m = fmaxf(m, redf[w]);
    const float ref = m == -INFINITY ? 0.0f : m;
    double sum = 0.0;
    for (int j = t; j < a.V; j += kBestThreads) sum += (double)exp2_fast((elem(x, j) - ref) * a.scale);
    sum = block_sum(sum, redd);
    if (t == 0) total_s = sum;
    __syncthreads();
    sum = total_s;
    const double log_sum = log(sum);
    const bool nan = sum != sum;
    unsigned long long last = ~0ull;
    for (int i = 0; i < a.n; i++) {
        unsigned long long best = 0;
        for (int j = t; j < a.V && !nan; j += kBestThreads) {
            const float v = elem(x, j);
            const unsigned long long k = best_key(v, j);
            if (v > -INFINITY && k < last && k > best) best = k;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        __syncthreads();
        if ((t & 31) == 0) redk[t >> 5] = best;
        __syncthreads();
        for (int w = 0; w < kBestThreads / 32; w++) best = max(best, redk[w]);
        if (t == 0) {
            const float v = fkey_inv((uint32_t)(best >> 32));
            value[i] = nan ? (double)NAN : best ? base + ((double)v - (double)m) * a.inv_t - log_sum : -(double)INFINITY;
            token[i] = best ? (int)(0xFFFFFFFFu - (uint32_t)best) : -1;
        }
        last = best;
        if (best == 0) {
            for (int r = i + 1 + t; r < a.n; r += kBestThreads) {
                value[r] = nan ? (double)NAN : -(double)INFINITY;
                token[r] = -1;
            }
            break;
        }
    }
}

// The rows' lists as they are.
__global__ void __launch_bounds__(256)
list_kernel(const double* value, const int* token, long long n, float* logprobs, int* tokens) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    logprobs[i] = (float)value[i];
    tokens[i] = token[i];
}

struct BeamArgs {
    const double* value;
    const int* token;
    int batch, beams, n, eos, keep;
    const unsigned char* finished;
    float* scores;
    int* parents;
    int* tokens;
    unsigned char* out_finished;
};

// One thread per entry: the beams' lists merged, then placed.
__global__ void __launch_bounds__(32)
beam_kernel(const BeamArgs a) {
    const int b = blockIdx.x * 32 + threadIdx.x;
    if (b >= a.batch) return;
    int head[QS_MAX_BEAMS];
    bool nan = false;
    for (int i = 0; i < a.beams; i++) {
        head[i] = 0;
        const double v = a.value[((size_t)b * a.beams + i) * a.n];
        nan |= v != v;
    }
    const size_t out = (size_t)b * a.n;
    unsigned long long stay = 0, used = 0;  // keep: places whose beam goes on
    for (int round = a.keep ? 0 : 1; round < 2; round++) {
        // keep's first round only finds the beams that go on
        for (int i = 0; i < a.beams; i++) head[i] = 0;
        for (int r = 0; r < a.n; r++) {
            int parent = -1, tok = -1;
            double best = nan ? (double)NAN : -(double)INFINITY;
            for (int i = 0; i < a.beams && !nan; i++) {
                if (head[i] == a.n) continue;
                const size_t at = ((size_t)b * a.beams + i) * a.n + head[i];
                if (a.value[at] > best) {
                    best = a.value[at];
                    parent = i;
                    tok = a.token[at];
                }
            }
            if (parent >= 0) head[parent]++;
            if (round == 0) {
                if (parent >= 0) stay |= 1ull << parent;
                continue;
            }
            int slot = r;
            if (a.keep) {
                slot = parent >= 0 && !(used >> parent & 1) ? parent : __ffsll(~(used | stay)) - 1;
                used |= 1ull << slot;
            }
            a.scores[out + slot] = (float)best;
            a.parents[out + slot] = parent;
            a.tokens[out + slot] = tok;
            if (a.out_finished)
                a.out_finished[out + slot] =
                    parent < 0 || (a.eos >= 0 && tok == a.eos) || (a.finished && a.finished[(size_t)b * a.beams + parent]);
        }
    }
}

static size_t lists_bytes(long long rows, int n) {
    return round256((size_t)rows * n * sizeof(double)) + round256((size_t)rows * n * sizeof(int));
}

template <typename T>
static int best_rows(const BestArgs& a, cudaStream_t st) {
    return launch("best_rows_kernel", best_rows_kernel<T>, a.rows, kBestThreads, 1, 0, false, st, a);
}

static BestArgs best_args(const Rows& r, int n, void* ws) {
    BestArgs a = {};
    a.logits = r.logits;
    a.rows = r.rows;
    a.V = r.vocab;
    a.ld = r.ld;
    a.n = n;
    a.scale = (float)(r.inv_t * 1.4426950408889634);
    a.inv_t = r.inv_t;
    a.value = (double*)ws;
    a.token = (int*)((char*)ws + round256((size_t)r.rows * n * sizeof(double)));
    return a;
}

}  // namespace qs

using namespace qs;

extern "C" {

size_t qs_top_logprobs_workspace(int dtype, int rows, int vocab, int k) {
    if ((dtype != QS_F32 && dtype != QS_BF16) || rows < 1 || vocab < 1 || vocab > kMaxVocab || k < 1 || k > QS_MAX_LISTED) return 0;
    return lists_bytes(rows, k);
}

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
    rc = check_workspace(d_workspace, workspace_bytes, qs_top_logprobs_workspace(dtype, rows, vocab, k));
    if (rc) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    const BestArgs a = best_args(r, k, d_workspace);
    rc = dtype == QS_F32 ? best_rows<float>(a, st) : best_rows<__nv_bfloat16>(a, st);
    if (rc) return rc;
    const long long n = (long long)rows * k;
    return launch("list_kernel", list_kernel, (n + 255) / 256, 256, 1, 0, false, st, a.value, a.token, n, d_logprobs, d_tokens);
}

size_t qs_beam_select_workspace(int dtype, int batch, int beams, int vocab, int n) {
    if (batch < 1 || beams < 1 || beams > QS_MAX_BEAMS || batch > (1 << 27) / beams) return 0;
    return qs_top_logprobs_workspace(dtype, batch * beams, vocab, n);
}

int qs_beam_select(const void* d_logits, int dtype, int batch, int beams, int vocab, long long row_stride,
                   const float* d_scores, const unsigned char* d_finished, int n, const qs_beam_params* params,
                   float* d_out_scores, int* d_parents, int* d_tokens, unsigned char* d_out_finished,
                   void* d_workspace, size_t workspace_bytes, void* stream) {
    set_error(QS_OK, "");
    if (!params) return fail(QS_ERR_INVALID, "params is NULL");
    const qs_beam_params p = *params;
    if (batch < 0) return fail(QS_ERR_INVALID, "batch %d < 0", batch);
    if (beams < 1 || beams > QS_MAX_BEAMS) return fail(QS_ERR_UNSUPPORTED, "beams %d outside [1, %d]", beams, QS_MAX_BEAMS);
    if (batch > (1 << 27) / beams) return fail(QS_ERR_UNSUPPORTED, "%d x %d rows above 2^27", batch, beams);
    const Rows r{d_logits, dtype, batch * beams, vocab, row_stride, nullptr, 1.0 / p.temperature, nullptr, 0};
    int rc = check_rows(r, p.temperature, false);
    if (rc) return rc;
    if (n < 1 || n > QS_MAX_LISTED) return fail(QS_ERR_UNSUPPORTED, "n %d outside [1, %d]", n, QS_MAX_LISTED);
    if (p.keep_slots && n != beams) return fail(QS_ERR_INVALID, "keep_slots wants n %d = beams %d", n, beams);
    if (p.eos_token < -1 || p.eos_token >= vocab) return fail(QS_ERR_INVALID, "eos_token %d outside [-1, %d)", p.eos_token, vocab);
    if (batch == 0) return QS_OK;
    if (!d_scores) return fail(QS_ERR_INVALID, "NULL device pointer");
    if (!d_out_scores || !d_parents || !d_tokens) return fail(QS_ERR_INVALID, "NULL output buffer");
    rc = check_workspace(d_workspace, workspace_bytes, qs_beam_select_workspace(dtype, batch, beams, vocab, n));
    if (rc) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    BestArgs a = best_args(r, n, d_workspace);
    a.scores = d_scores;
    a.finished = d_finished;
    a.pad = p.pad_token;
    rc = dtype == QS_F32 ? best_rows<float>(a, st) : best_rows<__nv_bfloat16>(a, st);
    if (rc) return rc;
    const BeamArgs b{a.value, a.token, batch, beams, n, p.eos_token, p.keep_slots, d_finished, d_out_scores, d_parents, d_tokens,
                     d_out_finished};
    return launch("beam_kernel", beam_kernel, (batch + 31) / 32, 32, 1, 0, false, st, b);
}

}  // extern "C"
