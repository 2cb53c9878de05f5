// What the kernels over rows of logits share: a row as 16-byte vectors at any
// alignment, exponentials, the exchange between the CTAs of a cluster; and on
// the host the checks of a call's rows and the launch.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <atomic>

#include "qs_common.cuh"
#include "qs_f32x2.cuh"
#include "qs_pipe.cuh"
#include "qwen600_sampler.h"

namespace qs {

int set_error(int code, const char* msg);  // qs_api.cu

constexpr unsigned long long kLoadWaitNs = 2000000000ull;  // a copy that has not landed by then: NaN in the results

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

[[maybe_unused]] static int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return set_error(code, buf);
}

[[maybe_unused]] static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

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

[[maybe_unused]] static int check_workspace(const void* p, size_t bytes, size_t need) {
    if (need == 0 || (p && bytes >= need && ((uintptr_t)p & 15) == 0)) return QS_OK;
    return fail(QS_ERR_INVALID, "workspace is NULL, unaligned or below %zu bytes", need);
}

[[maybe_unused]] static int check_rows(const Rows& r, double temperature, bool tokens = true) {
    if (r.dtype != QS_F32 && r.dtype != QS_BF16) return fail(QS_ERR_INVALID, "unknown dtype %d", r.dtype);
    if (r.rows < 0) return fail(QS_ERR_INVALID, "rows %d < 0", r.rows);
    if (r.rows > 1 << 27) return fail(QS_ERR_UNSUPPORTED, "rows %d above 2^27", r.rows);
    if (r.vocab < 1 || r.vocab > kMaxVocab)
        return fail(QS_ERR_UNSUPPORTED, "vocab %d outside [1, %d]", r.vocab, kMaxVocab);
    if (!(temperature >= 1e-6 && temperature <= 1e6))
        return fail(QS_ERR_INVALID, "temperature %g outside [1e-6, 1e6]", temperature);
    if (r.rows == 0) return QS_OK;
    if (!r.logits || (tokens && !r.tokens)) return fail(QS_ERR_INVALID, "NULL device pointer");
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

}  // namespace qs
