// The lm_head with 4-bit weights for few tokens: quantisation, the packed
// layout and the projection (include/qwen600_sampler.h gives the formulas).
//
// Bound: the stream of the codes.  For 151,936 x 1024 that is 78 MB, 12.3 us at
// the measured 6549 GB/s, so all else has to fit beside 23 bytes a clock and
// SM.  What counts is the instructions a code costs.  Codes go from memory to
// registers and meet the tokens on mma.sync m16n8k16, 16 vocabulary rows x 8
// tokens, tokens on the narrow side.  A word of 8 codes becomes four registers
// of fp16 pairs q - z with 9 instructions: one shift, four and / ors into
// 1024 + q or 1024 + 16 q, four fp16 subtractions or multiply-adds, all exact.
// (As fp16 denormals, q 2^-24, codes need only the shift and four ands, but the
// tensor cores align products by nominal exponents and lose 6 bits of a sum; as
// bf16 pairs they take 11.)  Turning codes into fp16 by the bits of 1024 is a
// published method; layout, zero points and the sharing of units are this
// file's.  The tokens are scaled by a power of two to fp16,
// exactly for values of at least 2^-31 of a row's largest (smaller ones lose
// what lies 2^-39 below it).  (tcgen05 takes its wider operand from shared or
// tensor memory; 4-bit weights would have to be written there as 16-bit numbers,
// four times the bytes of their stream.)
//
// Measured, 151,936 x 1,024: one token 18.8 us with groups of 128 (16.2 without
// the arithmetic), 16 tokens 23.9, 32 tokens 34.4; with groups of 32 and zero
// points 22.8, 28.6 and 39.8.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "qs_common.cuh"
#include "qs_f32x2.cuh"
#include "qs_w4.h"
#include "qs_rmsnorm.cuh"

namespace qs {

// One thread per group of a row: the range that holds the group and zero, a
// bf16 scale of a fifteenth of it, codes rounded to nearest.  A NaN makes the
// scale NaN, an infinity infinite: either way the group's products are NaN.
__global__ void w4_quantize_kernel(const __nv_bfloat16* __restrict__ w, int V, int K, int group,
                                   unsigned char* __restrict__ codes, __nv_bfloat16* __restrict__ scales,
                                   unsigned char* __restrict__ zeros) {
    const size_t g = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int per = K / group;
    if (g >= (size_t)V * per) return;
    const __nv_bfloat16* x = w + g * group;
    float lo = 0.0f, hi = 0.0f;
    bool number = true;
    for (int i = 0; i < group; i++) {
        const float v = __bfloat162float(x[i]);
        number &= v == v;
        lo = fminf(lo, v);  // passes over a NaN
        hi = fmaxf(hi, v);
    }
    const __nv_bfloat16 sb = __float2bfloat16_rn(number ? (hi - lo) / 15.0f : NAN);
    const float s = __bfloat162float(sb);
    const float d = s > 0.0f ? s : 1.0f;  // a group of zeros: scale 0, codes 0
    const float z = fminf(fmaxf(rintf(-lo / d), 0.0f), 15.0f);
    for (int i = 0; i < group; i += 2) {
        const float a = fminf(fmaxf(rintf(__bfloat162float(x[i]) / d) + z, 0.0f), 15.0f);
        const float b = fminf(fmaxf(rintf(__bfloat162float(x[i + 1]) / d) + z, 0.0f), 15.0f);
        codes[(g * group + i) / 2] = (unsigned char)((int)a | ((int)b << 4));
    }
    scales[g] = sb;
    zeros[g] = (unsigned char)z;
}

cudaError_t launch_w4_quantize(const __nv_bfloat16* w, int V, int K, int group, unsigned char* codes,
                               __nv_bfloat16* scales, unsigned char* zeros, cudaStream_t st) {
    const size_t n = (size_t)V * (K / group);
    w4_quantize_kernel<<<(unsigned)((n + 127) / 128), 128, 0, st>>>(w, V, K, group, codes, scales, zeros);
    return cudaGetLastError();
}

// ---------------------------------------------------------------- layout
// Vocabulary rows in tiles of 32, columns in chunks of 128 (the last padded
// with zeros).  A unit is one tile's chunk: 2 KB of codes, and units lie one
// after another, tile by tile.  In a unit lane l = 4 g + q of a warp finds
// 16 bytes for each of rows g, g + 8, g + 16 and g + 24 (512 bytes apart): four
// words, word w for columns 32 w + 8 q + 0..7 of the chunk.  Nibble i < 4 of a
// word is column 2 i, nibble i + 4 column 2 i + 1, so masks take pairs of
// neighbouring columns, one in each half.  A group of 32 columns is then one
// word of every lane, and any group is whole mma instructions.
// Scales (16-bit) and zero points (bytes) of a unit: [g][group of the chunk]
// [rows g, g + 8, g + 16, g + 24].
constexpr int kUnitCodes = 2048;

static int w4_chunks(int K) { return (K + 127) / 128; }
static int w4_tiles(int V) { return (V + 31) / 32; }

size_t w4_codes_bytes(int V, int K) { return (size_t)w4_tiles(V) * w4_chunks(K) * kUnitCodes; }
size_t w4_scales_bytes(int V, int K, int group) { return (size_t)w4_tiles(V) * w4_chunks(K) * (128 / group) * 64; }
size_t w4_zeros_bytes(int V, int K, int group) { return w4_scales_bytes(V, K, group) / 2; }

__global__ void w4_pack_codes_kernel(const unsigned char* __restrict__ codes, int V, int K, int chunks, size_t n,
                                     uint32_t* __restrict__ out) {
    const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;  // one word
    if (i >= n) return;
    const int w = i & 3, lane = (i >> 2) & 31, block = (i >> 7) & 3;
    const size_t unit = i >> 9;
    const int row = (int)(unit / chunks) * 32 + block * 8 + (lane >> 2);
    const int k = (int)(unit % chunks) * 128 + 32 * w + 8 * (lane & 3);
    uint32_t word = 0;
    if (row < V && k < K) {
        const unsigned char* p = codes + ((size_t)row * K + k) / 2;
        for (int b = 0; b < 4; b++) word |= (uint32_t)(p[b] & 15) << (4 * b) | (uint32_t)(p[b] >> 4) << (16 + 4 * b);
    }
    out[i] = word;
}

__global__ void w4_pack_scales_kernel(const uint16_t* __restrict__ scales, const unsigned char* __restrict__ zeros,
                                      int V, int per_row, int chunks, int per_chunk, size_t n,
                                      uint16_t* __restrict__ out_s, unsigned char* __restrict__ out_z) {
    const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int block = i & 3, j = (int)(i >> 2) % per_chunk, g = (int)((i >> 2) / per_chunk) & 7;
    const size_t unit = i / (32 * per_chunk);
    const int row = (int)(unit / chunks) * 32 + block * 8 + g, grp = (int)(unit % chunks) * per_chunk + j;
    const bool in = row < V && grp < per_row;
    out_s[i] = in ? scales[(size_t)row * per_row + grp] : 0;
    if (zeros) out_z[i] = in ? zeros[(size_t)row * per_row + grp] & 15 : 0;
}

cudaError_t launch_w4_pack(const unsigned char* codes, const void* scales, const unsigned char* zeros, int V, int K,
                           int group, unsigned char* pc, void* ps, unsigned char* pz, cudaStream_t st) {
    const int chunks = w4_chunks(K);
    size_t n = w4_codes_bytes(V, K) / 4;
    w4_pack_codes_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(codes, V, K, chunks, n, (uint32_t*)pc);
    n = w4_scales_bytes(V, K, group) / 2;
    w4_pack_scales_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>((const uint16_t*)scales, zeros, V, K / group,
                                                                      chunks, 128 / group, n, (uint16_t*)ps, pz);
    return cudaGetLastError();
}

// -------------------------------------------------------------------- rows
// RMSNorm of one token's row per CTA, and the row as the products take it, in
// the workspace: fp16 columns (zeros behind the last) scaled by 2^s so that the
// largest finite value lies in [2^14, 2^15), then 2^-s.
__host__ __device__ static inline size_t w4_row_bytes(int chunks) { return (size_t)chunks * 256 + 16; }

// kPairs: column pairs of a thread, the row's whole share, requested with its
// norm weights before anything waits.
template <int kPairs>
__global__ void __launch_bounds__(kNormThreads)
w4_rows_kernel(const __nv_bfloat16* __restrict__ X, const __nv_bfloat16* __restrict__ w, __nv_bfloat16* __restrict__ Y,
               int K, int chunks, unsigned char* __restrict__ ws, float inv_d, float eps) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the projection may request its first codes
    __shared__ float red_max[kNormThreads / 32];
    const int t = threadIdx.x, warp = t >> 5, half = K / 2;
    const __nv_bfloat162* in = reinterpret_cast<const __nv_bfloat162*>(X + (size_t)blockIdx.x * K);
    const __nv_bfloat162* wt = reinterpret_cast<const __nv_bfloat162*>(w);
    __nv_bfloat162* out = reinterpret_cast<__nv_bfloat162*>(Y + (size_t)blockIdx.x * K);
    ws += blockIdx.x * w4_row_bytes(chunks);
    uint32_t* xs = reinterpret_cast<uint32_t*>(ws);
    __nv_bfloat162 xv[kPairs], wv[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; j++) {
        const int i = j * kNormThreads + t;
        if (i < half) xv[j] = in[i];
        if (wt && i < half) wv[j] = wt[i];
    }
    float lsum = 0.0f;
#pragma unroll
    for (int j = 0; j < kPairs; j++)
        if (j * kNormThreads + t < half) lsum = rms_add(lsum, xv[j]);
    const float mul = rms_factor(lsum, inv_d, eps);
    float2 y[kPairs];
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < kPairs; j++) {
        const int i = j * kNormThreads + t;
        y[j] = make_float2(0.0f, 0.0f);
        if (i < half) {
            const __nv_bfloat162 b = rms_scaled(xv[j], mul, wt ? __bfloat1622float2(wv[j]) : make_float2(1.0f, 1.0f));
            out[i] = b;
            y[j] = __bfloat1622float2(b);
            const float a0 = fabsf(y[j].x), a1 = fabsf(y[j].y);
            if (a0 < INFINITY) m = fmaxf(m, a0);
            if (a1 < INFINITY) m = fmaxf(m, a1);
        }
    }
    m = warp_max(m);
    if ((t & 31) == 0) red_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kNormThreads / 32; k++) m = fmaxf(m, red_max[k]);
    const int e = (int)(__float_as_uint(m) >> 23) - 127;
    const int s = m == 0.0f ? 0 : min(14 - e, 120);
    const float up = __uint_as_float((uint32_t)(s + 127) << 23);
    if (t == 0) *reinterpret_cast<float*>(ws + (size_t)chunks * 256) = __uint_as_float((uint32_t)(127 - s) << 23);
#pragma unroll
    for (int j = 0; j < kPairs; j++) {
        const int i = j * kNormThreads + t;
        if (i < chunks * 64) {  // 64 pairs a chunk
            const __half2 h = __floats2half2_rn(y[j].x * up, y[j].y * up);
            xs[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
}

// -------------------------------------------------------------- projection
constexpr int kW4Depth = 2;  // units a warp has in flight

// d = a * b + d, or a * b alone, on 16 x 8 x 16.
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// (v & mask) | 1024 in each half.
__device__ __forceinline__ __half2 code_bits(uint32_t v, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(0x64006400u));
    return *reinterpret_cast<const __half2*>(&r);
}
__device__ __forceinline__ uint32_t bits_of(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 half2_of(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// The eight codes of a word minus their zero point: columns 0 and 1, 2 and 3, 4
// and 5, 6 and 7.  z1024: 1024 + z twice; z64: -(64 + z) twice.
__device__ __forceinline__ void code_pairs(uint32_t v, __half2 z1024, __half2 z64, uint32_t* r) {
    const uint32_t v8 = v >> 8;
    const __half2 sixteenth = half2_of(0x2C002C00u);
    r[0] = bits_of(__hsub2(code_bits(v, 0x000F000Fu), z1024));
    r[1] = bits_of(__hfma2(code_bits(v, 0x00F000F0u), sixteenth, z64));
    r[2] = bits_of(__hsub2(code_bits(v8, 0x000F000Fu), z1024));
    r[3] = bits_of(__hfma2(code_bits(v8, 0x00F000F0u), sixteenth, z64));
}

// The scales of rows g (low half) and g + 8.
template <bool kF16>
__device__ __forceinline__ float2 scales_of(uint32_t bits) {
    if (kF16) return __half22float2(*reinterpret_cast<const __half2*>(&bits));
    return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xFFFF0000u));
}

__device__ __forceinline__ uint4 load_codes(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// One unit as a lane holds it.
template <int kGroups>
struct W4Unit {
    uint4 codes[4];                // rows g, g + 8, g + 16, g + 24
    uint32_t scales[2 * kGroups];  // of a group: rows g and g + 8, rows g + 16 and g + 24
    uint32_t zeros[kGroups];
};

// Where a lane's part of its warp's next unit lies.
struct W4At {
    const unsigned char* codes;
    const unsigned char* scales;
    const unsigned char* zeros;
};

template <int kWords>
__device__ __forceinline__ void load_words(uint32_t* out, const void* p) {
    if (kWords == 1) {
        out[0] = __ldg(static_cast<const uint32_t*>(p));
    } else if (kWords == 2) {
        const uint2 v = __ldg(static_cast<const uint2*>(p));
        out[0] = v.x; out[1 % kWords] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < kWords / 4; i++) {
            const uint4 v = __ldg(static_cast<const uint4*>(p) + i);
            out[4 * i] = v.x; out[(4 * i + 1) % kWords] = v.y; out[(4 * i + 2) % kWords] = v.z; out[(4 * i + 3) % kWords] = v.w;
        }
    }
}

// Loads the unit `ahead` units behind the next one.
template <int kGroups, bool kZeros>
__device__ __forceinline__ void w4_load(W4Unit<kGroups>& u, const W4At& at, int ahead) {
    const uint4* c = reinterpret_cast<const uint4*>(at.codes + ahead * kUnitCodes);
#pragma unroll
    for (int i = 0; i < 4; i++) u.codes[i] = load_codes(c + 32 * i);
    load_words<2 * kGroups>(u.scales, at.scales + ahead * (64 * kGroups));
    if (kZeros) load_words<kGroups>(u.zeros, at.zeros + ahead * (32 * kGroups));
}

struct W4Out {
    __nv_bfloat16* logits;
    int tokens;  // rows of this launch
    uint32_t* segk;
    int segk_stride;
};

constexpr int kStageRow = 40;  // a token's 32 values in a warp's staging rows, 80 bytes apart: the lanes' stores meet no bank twice

// Stores a finished tile: 32 vocabulary rows of up to 8 kNt tokens, through the
// warp's staging rows so that a lane stores 16 bytes of one token.
template <int kNt>
__device__ __forceinline__ void w4_store(const float (&acc)[2][kNt][4], const float* unscale, __nv_bfloat16* stage,
                                         const W4Out& o, int V, int tile, int lane) {
    const int g = lane >> 2, q = lane & 3;
    __syncwarp();
#pragma unroll
    for (int n = 0; n < kNt; n++) {
#pragma unroll
        for (int j = 0; j < 2; j++) {  // token 2 q or 2 q + 1
            const int token = n * 8 + 2 * q + j;
            const float f = unscale[token];
#pragma unroll
            for (int b = 0; b < 4; b++)  // row g + 8 b
                stage[token * kStageRow + g + b * 8] = __float2bfloat16_rn(acc[b >> 1][n][(b & 1) * 2 + j] * f);
        }
    }
    __syncwarp();
    const bool whole = (V & 7) == 0;  // every row of logits starts on 16 bytes
    if (whole || o.segk) {
#pragma unroll
        for (int i = 0; i < kNt; i++) {
            const int p = i * 32 + lane, token = p >> 2, col = tile * 32 + (p & 3) * 8;
            const uint4 v = *reinterpret_cast<const uint4*>(stage + token * kStageRow + (p & 3) * 8);
            if (token >= o.tokens || col >= V) continue;
            if (whole) *reinterpret_cast<uint4*>(o.logits + (size_t)token * V + col) = v;
            // whole blocks of 16 columns, as the bf16 epilogue folds them: they never straddle a 256-column segment,
            // and the sampler takes the maxima of whole segments
            if (o.segk && (col & ~15) + 16 <= V)
                atomicMax(o.segk + (size_t)token * o.segk_stride + (col >> 8), fkey(vec_max<__nv_bfloat16>(v)));
        }
    }
    if (!whole && tile * 32 + lane < V) {  // a column a lane
        for (int token = 0; token < o.tokens; token++)
            o.logits[(size_t)token * V + tile * 32 + lane] = stage[token * kStageRow + lane];
    }
}

// A CTA takes a contiguous range of tiles and its warps equal shares of their
// units, so warps end together whatever the number of tiles; a tile that
// several warps share is added from their partial sums at the end, in order.
// kNt blocks of 8 tokens, kGroups groups in a chunk.  A tile is two mma rows of
// 16, so that a token's columns, read from shared memory, serve both (with one,
// these reads took half of the L1 pipe at 16 tokens: 29.5 us, with two 27.6).
// Up to 16 tokens 16 warps of 128 registers, above 8 of 255.
template <int kNt, int kGroups, bool kZeros, bool kF16>
__global__ void __launch_bounds__(kNt <= 2 ? 512 : 256, 1)
lm_head_w4_kernel(const unsigned char* rows, const __grid_constant__ W4View w, const __grid_constant__ W4Out o, int chunks,
                  int tiles) {
    constexpr int kWarps = kNt <= 2 ? 16 : 8;
    extern __shared__ __align__(16) unsigned char smem[];
    const int pitch = chunks * 256 + 64;  // bytes of a token's row: neighbours 64 bytes apart in the banks
    unsigned char* xs = smem;                                           // fp16 rows
    float4* slots = reinterpret_cast<float4*>(smem + kNt * 8 * pitch);  // [warp][continued, begun][2][kNt][lane]
    __nv_bfloat16* stage = reinterpret_cast<__nv_bfloat16*>(slots + kWarps * 2 * 2 * kNt * 32);
    float* unscale = reinterpret_cast<float*>(stage + kWarps * kNt * 8 * kStageRow);  // [token]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    stage += warp * kNt * 8 * kStageRow;
    const int t0 = (int)((long long)blockIdx.x * tiles / gridDim.x), t1 = (int)((long long)(blockIdx.x + 1) * tiles / gridDim.x);
    const int u0 = t0 * chunks, un = (t1 - t0) * chunks;
    const auto share = [&](int wi) { return u0 + (int)((long long)un * wi / kWarps); };
    const int a = share(warp), b = share(warp + 1);

    W4At at;
    at.codes = w.codes + (size_t)a * kUnitCodes + lane * 16;
    at.scales = reinterpret_cast<const unsigned char*>(w.scales) + ((size_t)a * 8 + g) * (8 * kGroups);
    at.zeros = w.zeros + (kZeros ? ((size_t)a * 8 + g) * (4 * kGroups) : 0);
    W4Unit<kGroups> buf[kW4Depth];
#pragma unroll
    for (int d = 0; d < kW4Depth; d++)
        if (a + d < b) w4_load<kGroups, kZeros>(buf[d], at, d);
    // two more units on their way to L2 while the RMSNorm runs (one token 18.2 to 17.7 us, 5 tokens of 32,003 x 4,096
    // 19.3 to 18.3; 4 or 8 units gain less)
    for (int i = lane; i < min(2, b - a - kW4Depth) * (kUnitCodes / 128); i += 32)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(w.codes + (size_t)(a + kW4Depth) * kUnitCodes + i * 128));
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the RMSNorm's rows
    const size_t row_bytes = w4_row_bytes(chunks);
    for (int i = threadIdx.x; i < kNt * 8 * chunks * 16; i += kWarps * 32) {
        const int row = i / (chunks * 16), c = i - row * (chunks * 16);
        *reinterpret_cast<uint4*>(xs + row * pitch + c * 16) =
            row < o.tokens ? *reinterpret_cast<const uint4*>(rows + row * row_bytes + c * 16) : make_uint4(0u, 0u, 0u, 0u);
    }
    if (threadIdx.x < kNt * 8)
        unscale[threadIdx.x] = threadIdx.x < o.tokens
                                   ? *reinterpret_cast<const float*>(rows + threadIdx.x * row_bytes + chunks * 256)
                                   : 0.0f;
    __syncthreads();

    float acc[2][kNt][4];
    const auto clear = [&] {
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int n = 0; n < kNt; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[m][n][j] = 0.0f;
    };
    clear();
    int tile = a / chunks, c = a - tile * chunks;
    bool begun = c == 0;
    const unsigned char* xl = xs + g * pitch + q * 16;
    const unsigned char* xc = xl + c * 256;
    for (int left = b - a; left > 0; left -= kW4Depth) {
        at.codes += kW4Depth * kUnitCodes;
        at.scales += kW4Depth * 64 * kGroups;
        if (kZeros) at.zeros += kW4Depth * 32 * kGroups;
#pragma unroll
        for (int d = 0; d < kW4Depth; d++) {
            if (d >= left) break;
#pragma unroll
            for (int j = 0; j < kGroups; j++) {
                __half2 z1024[4], z64[4];
#pragma unroll
                for (int b4 = 0; b4 < 4; b4++) {
                    if (kZeros) {  // bytes z, 0x64, z, 0x64
                        z1024[b4] = half2_of(__byte_perm(buf[d].zeros[j], 0x64646464u, 0x4040u + 0x0101u * b4));
                        z64[b4] = __hsub2(half2_of(0x63806380u), z1024[b4]);  // 960 - (1024 + z)
                    } else {
                        z1024[b4] = half2_of(0x64086408u);
                        z64[b4] = half2_of(0xD480D480u);
                    }
                }
                float part[2][kNt][4];
#pragma unroll
                for (int k = 0; k < 4 / kGroups; k++) {
                    const int word = j * (4 / kGroups) + k;
                    uint32_t r[4][4];  // rows g + 8 b
#pragma unroll
                    for (int b4 = 0; b4 < 4; b4++)
                        code_pairs(reinterpret_cast<const uint32_t*>(&buf[d].codes[b4])[word], z1024[b4], z64[b4], r[b4]);
#pragma unroll
                    for (int n = 0; n < kNt; n++) {
                        const uint4 xv = *reinterpret_cast<const uint4*>(xc + n * 8 * pitch + word * 64);
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            const uint32_t *lo = r[2 * m], *hi = r[2 * m + 1];
                            if (k == 0) mma_first(part[m][n], lo[0], hi[0], lo[1], hi[1], xv.x, xv.y);
                            else mma(part[m][n], lo[0], hi[0], lo[1], hi[1], xv.x, xv.y);
                            mma(part[m][n], lo[2], hi[2], lo[3], hi[3], xv.z, xv.w);
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    const float2 sg = scales_of<kF16>(buf[d].scales[2 * j + m]);
#pragma unroll
                    for (int n = 0; n < kNt; n++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {  // row g, row g + 8; both tokens at once
                            const float f = h ? sg.y : sg.x;
                            const float2 v = unpair2(fma2(pair2(f, f), pair2(part[m][n][2 * h], part[m][n][2 * h + 1]),
                                                          pair2(acc[m][n][2 * h], acc[m][n][2 * h + 1])));
                            acc[m][n][2 * h] = v.x;
                            acc[m][n][2 * h + 1] = v.y;
                        }
                }
            }
            if (d + kW4Depth < left) w4_load<kGroups, kZeros>(buf[d], at, d);
            const bool ends = ++c == chunks;
            xc += 256;
            if (ends || d + 1 == left) {
                if (ends && begun) {
                    w4_store<kNt>(acc, unscale, stage, o, w.vocab, tile, lane);
                } else {
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int n = 0; n < kNt; n++)
                            slots[(((warp * 2 + begun) * 2 + m) * kNt + n) * 32 + lane] =
                                make_float4(acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]);
                }
                clear();
                if (ends) {
                    c = 0;
                    xc = xl;
                    tile++;
                    begun = true;
                }
            }
        }
    }
    __syncthreads();
    // the warp that began a tile which later warps continued adds their sums
    if (a < b && b % chunks != 0 && (b - 1) / chunks * chunks >= a) {
        const int last = (b - 1) / chunks, stop = (last + 1) * chunks;
        int slot = warp * 2 + 1;  // its own part, then the following warps' continued ones
        for (int wi = warp; wi < kWarps && share(wi) < stop; wi++) {
            if (share(wi) < share(wi + 1)) {
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int n = 0; n < kNt; n++) {
                        const float4 p = slots[((slot * 2 + m) * kNt + n) * 32 + lane];
                        acc[m][n][0] += p.x; acc[m][n][1] += p.y; acc[m][n][2] += p.z; acc[m][n][3] += p.w;
                    }
            }
            slot = (wi + 1) * 2;
        }
        w4_store<kNt>(acc, unscale, stage, o, w.vocab, last, lane);
    }
}

static size_t w4_smem(int nt, int K) {
    return (size_t)nt * 8 * (w4_chunks(K) * 256 + 64) + (size_t)(nt <= 2 ? 16 : 8) * nt * (2 * 2 * 512 + 16 * kStageRow) +
           (size_t)nt * 8 * sizeof(float);
}

template <int kNt, int kGroups, bool kZeros, bool kF16>
static cudaError_t w4_go(const unsigned char* rows, const W4View& w, const W4Out& o, int grid, cudaStream_t st) {
    const size_t smem = w4_smem(kNt, w.hidden);
    static std::atomic<unsigned long long> raised{0};  // devices on which the kernel may use all shared memory
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !(raised.load() >> dev & 1))) {
        e = cudaFuncSetAttribute(lm_head_w4_kernel<kNt, kGroups, kZeros, kF16>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e == cudaSuccess && dev < 64) raised.fetch_or(1ull << dev);
    }
    if (e != cudaSuccess) return e;
    // programmatic dependent launch: the first units are requested while the
    // RMSNorm runs
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kNt <= 2 ? 512 : 256);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, lm_head_w4_kernel<kNt, kGroups, kZeros, kF16>, rows, w, o, w4_chunks(w.hidden), w4_tiles(w.vocab));
}

template <int kNt, int kGroups>
static cudaError_t w4_types(const unsigned char* rows, const W4View& w, const W4Out& o, int grid, cudaStream_t st) {
    const bool f16 = w.scale_dtype == QS_F16;
    if (w.zeros)
        return f16 ? w4_go<kNt, kGroups, true, true>(rows, w, o, grid, st) : w4_go<kNt, kGroups, true, false>(rows, w, o, grid, st);
    return f16 ? w4_go<kNt, kGroups, false, true>(rows, w, o, grid, st) : w4_go<kNt, kGroups, false, false>(rows, w, o, grid, st);
}

template <int kNt>
static cudaError_t w4_group(const unsigned char* rows, const W4View& w, const W4Out& o, int grid, cudaStream_t st) {
    return w.group == 128 ? w4_types<kNt, 1>(rows, w, o, grid, st)
         : w.group == 64  ? w4_types<kNt, 2>(rows, w, o, grid, st)
                          : w4_types<kNt, 4>(rows, w, o, grid, st);
}

size_t w4_workspace(int batch, int K) { return (size_t)batch * w4_row_bytes(w4_chunks(K)); }

cudaError_t launch_lm_head_w4(const __nv_bfloat16* hidden, const __nv_bfloat16* norm_weight, const W4View& w, int batch,
                              __nv_bfloat16* normed, __nv_bfloat16* logits, unsigned char* ws, int num_sms,
                              uint32_t* segk, int segk_stride, cudaStream_t st) {
    const int chunks = w4_chunks(w.hidden);
    const auto rows_kernel = w.hidden <= 1024 ? w4_rows_kernel<2> : w.hidden <= 4096 ? w4_rows_kernel<8> : w4_rows_kernel<16>;
    rows_kernel<<<batch, kNormThreads, 0, st>>>(hidden, norm_weight, normed, w.hidden, chunks, ws,
                                               1.0f / (float)w.hidden, kNormEps);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int tiles = w4_tiles(w.vocab), grid = tiles < num_sms ? tiles : num_sms;
    int most = 4;  // blocks of 8 tokens whose rows fit in shared memory
    while (w4_smem(most, w.hidden) > 227 * 1024) most--;
    for (int b = 0; b < batch;) {
        const int left = (batch - b + 7) / 8, nt = left < most ? left : most;
        const int n = batch - b < nt * 8 ? batch - b : nt * 8;
        const W4Out o{logits + (size_t)b * w.vocab, n, segk ? segk + (size_t)b * segk_stride : nullptr, segk_stride};
        const unsigned char* rows = ws + b * w4_row_bytes(chunks);
        e = nt == 1 ? w4_group<1>(rows, w, o, grid, st)
          : nt == 2 ? w4_group<2>(rows, w, o, grid, st)
          : nt == 3 ? w4_group<3>(rows, w, o, grid, st)
                    : w4_group<4>(rows, w, o, grid, st);
        if (e != cudaSuccess) return e;
        b += n;
    }
    return cudaSuccess;
}

}  // namespace qs
