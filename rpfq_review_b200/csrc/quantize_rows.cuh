// Rows to 8-bit codes with one scale per row (the tokens of an activation
// matrix, or the output channels of a weight matrix):
//
//   t = max(amax |x|, 1e-30);  s = fl(fl(1 / t) 127);  q = rint(fl(x s))  (half to even)
//   scale = fl(t / 127),  x ~ q scale
//
// the same reciprocal-multiply arithmetic as the other quantizers here. |x| <= t
// bounds fl(x s) by 127 (1 + 2^-20) (1 / t may be subnormal), so |q| <= 127
// without a clamp. The 1e-30
// floor keeps s finite: a row of zeros (or of values far below it) gets codes of
// zero. A row that holds a NaN or an infinity has no scale: its scale is NaN and
// its codes are zero, so that every output of the product reads NaN.
//
// Bound by memory: each value is read once from DRAM and leaves as one byte. The
// row stays in registers between its maximum and its codes (KEEP 16-byte vectors
// per thread). 8, 16 or 32 lanes take a row, the fewest that keep it in 8 vectors
// each (16 for the longest that a warp takes): what a row costs besides its values
// (the reduction, a reciprocal, a division) is then shared out over more rows of a
// warp. 50432 rows of 1024 fp16 values, 155 MB: 31.5 us with a warp per row, 27.8 us
// so. When the rows are too few to fill the GPU, or too long, a block of 256 threads
// takes one and reads what it cannot keep again, from L1 / L2.
// Rows off the 16-byte grid are read in the vectors of the grid all the same; their
// codes are shifted into place with the next lane's. The maximum of fp16 rows is taken on half pairs; fl(x s) is rounded by adding
// 1.5 * 2^23 (half to even, as rint), which leaves the code in the low byte of the
// sum.
#pragma once

#include "actquant.cuh"
#include "ptx.cuh"

namespace rpfq {

constexpr float kQuantRowTiny = 1e-30f;

struct QuantizeRowsParams {
    const void* x;   // fp16 or fp32 [m, k], row stride ldx
    int64_t ldx;
    int8_t* q;       // int8 [m, k], row stride ldq
    int64_t ldq;
    float* scale;    // fp32 [m]
    int64_t m;
    int32_t k;
};

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN when either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 16 bytes of a row: 8 fp16 or 4 fp32 values.
template <typename T>
struct QuantVec;
template <>
struct QuantVec<__half> {
    static constexpr int N = 8;
    uint4 raw;
    __device__ __forceinline__ float amax() const {
        const __half2* h = reinterpret_cast<const __half2*>(&raw);
        const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])),
                                      __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
        return max_nan(__low2float(m), __high2float(m));
    }
    __device__ __forceinline__ void values(float (&f)[8]) const {
        const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 v = __half22float2(h[e]);
            f[2 * e] = v.x, f[2 * e + 1] = v.y;
        }
    }
};
template <>
struct QuantVec<float> {
    static constexpr int N = 4;
    uint4 raw;
    __device__ __forceinline__ float amax() const {
        return max_nan(max_nan(fabsf(__uint_as_float(raw.x)), fabsf(__uint_as_float(raw.y))),
                       max_nan(fabsf(__uint_as_float(raw.z)), fabsf(__uint_as_float(raw.w))));
    }
    __device__ __forceinline__ void values(float (&f)[4]) const {
        f[0] = __uint_as_float(raw.x), f[1] = __uint_as_float(raw.y);
        f[2] = __uint_as_float(raw.z), f[3] = __uint_as_float(raw.w);
    }
};

struct QuantScale {
    float s;      // value -> code
    float scale;  // code -> value
    bool bad;     // a NaN or an infinity in the row
};
__device__ __forceinline__ QuantScale quant_scale(float amax) {
    QuantScale q;
    const float t = fmaxf(amax, kQuantRowTiny);
    q.bad = !(amax <= 3.402823466e38f);
    q.s = __fmul_rn(__frcp_rn(t), 127.0f);
    q.scale = q.bad ? __int_as_float(0x7fffffff) : __fdiv_rn(t, 127.0f);
    return q;
}

// The codes of N values, one per byte.
template <int N>
__device__ __forceinline__ void quant_codes(const float (&f)[N], float s, uint32_t (&out)[N / 4]) {
    constexpr float kMagic = 12582912.0f;
    // __fmul_rn / __fadd_rn are never contracted: an fma would skip the rounding of x s
    auto code = [s](float v) { return __float_as_uint(__fadd_rn(__fmul_rn(v, s), kMagic)); };
#pragma unroll
    for (int g = 0; g < N / 4; ++g) {
        const uint32_t lo = __byte_perm(code(f[4 * g]), code(f[4 * g + 1]), 0x0040);
        const uint32_t hi = __byte_perm(code(f[4 * g + 2]), code(f[4 * g + 3]), 0x0040);
        out[g] = __byte_perm(lo, hi, 0x5410);
    }
}

// How rows are read: vector by vector with nothing over; with a last vector put
// together value by value; in the vectors of the 16-byte grid, the codes shifted
// (parts of a warp only); value by value.
enum : int { kQuantWhole = 0, kQuantTail = 1, kQuantShift = 2, kQuantSingle = 3 };

// THREADS per row: 8, 16, 32 or 256, each with KEEP vectors in registers.
template <typename T, int MODE, int THREADS, int KEEP>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantizeRowsParams p) {
    using V = QuantVec<T>;
    constexpr int N = V::N;
    static_assert(MODE != kQuantShift || THREADS <= 32, "shifted codes come from the next lane");
    const int tid = threadIdx.x & (THREADS - 1);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / THREADS) + threadIdx.x / THREADS;
    pdl_wait();
    pdl_launch_dependents();
    const bool live = row < p.m;  // lanes of other rows share the warp's shuffles
    const T* __restrict__ x = static_cast<const T*>(p.x) + (live ? row : 0) * p.ldx;
    int8_t* __restrict__ q = p.q + (live ? row : 0) * p.ldq;
    // vector i holds the values from i N - off on
    const int off = MODE == kQuantShift ? static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) : 0;
    const int vecs = live ? (p.k + off + N - 1) / N : 0;
    auto whole = [&](int i) {
        if (MODE == kQuantWhole) return true;
        if (MODE == kQuantSingle) return false;
        return i * N >= off && (i + 1) * N - off <= p.k;
    };
    auto load = [&](int i) {
        V v;
        if (whole(i)) {
            v.raw = *reinterpret_cast<const uint4*>(x + i * N - off);
        } else {
            alignas(16) T e[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int at = i * N - off + j;
                e[j] = at >= 0 && at < p.k ? x[at] : T(0.0f);
            }
            v.raw = *reinterpret_cast<const uint4*>(e);
        }
        return v;
    };
    V kept[KEEP];
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
        if (tid + c * THREADS < vecs) kept[c] = load(tid + c * THREADS);
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
        if (tid + c * THREADS < vecs) amax = max_nan(amax, kept[c].amax());
    if constexpr (THREADS == 256)
        for (int i = tid + KEEP * THREADS; i < vecs; i += THREADS) amax = max_nan(amax, load(i).amax());
#pragma unroll
    for (int o = (THREADS < 32 ? THREADS : 32) / 2; o > 0; o >>= 1)
        amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if constexpr (THREADS == 256) {
        __shared__ float part[8];
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
        __syncthreads();
        amax = part[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) amax = max_nan(amax, part[w]);
    }
    if (MODE != kQuantShift && !live) return;
    const QuantScale qs = quant_scale(amax);
    constexpr int W = N / 4;  // 32-bit words of codes per vector
    auto codes = [&](const V& v, uint32_t (&code)[W]) {
        float f[N];
        v.values(f);
        quant_codes<N>(f, qs.s, code);
#pragma unroll
        for (int g = 0; g < W; ++g)
            if (qs.bad) code[g] = 0;
    };
    auto put = [&](int i, const uint32_t (&code)[W]) {  // the codes of values i N ..
        if (MODE == kQuantWhole || (MODE != kQuantSingle && (i + 1) * N <= p.k)) {
            if constexpr (W == 2)
                *reinterpret_cast<uint2*>(q + i * N) = make_uint2(code[0], code[1]);
            else
                *reinterpret_cast<uint32_t*>(q + i * N) = code[0];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (i * N + j < p.k) q[i * N + j] = static_cast<int8_t>(code[j / 4] >> (8 * (j % 4)));
        }
    };
    if constexpr (MODE == kQuantShift) {
        uint32_t code[KEEP + 1][W] = {};
#pragma unroll
        for (int c = 0; c < KEEP; ++c)
            if (tid + c * THREADS < vecs) codes(kept[c], code[c]);
        const int next = (threadIdx.x & 31 & ~(THREADS - 1)) | ((tid + 1) & (THREADS - 1));
#pragma unroll
        for (int c = 0; c < KEEP; ++c) {
            // the vector after this one: the next lane's, the first lane's next after the last
            uint32_t both[2 * W + 1];
#pragma unroll
            for (int g = 0; g < W; ++g) {
                both[g] = code[c][g];
                both[W + g] = __shfl_sync(0xffffffffu, tid == 0 ? code[c + 1][g] : code[c][g], next);
            }
            both[2 * W] = 0;
            const int words = off / 4, bits = 8 * (off % 4);
            uint32_t out[W];
#pragma unroll
            for (int g = 0; g < W; ++g)
                out[g] = words == 0 ? __funnelshift_r(both[g], both[g + 1], bits)
                                    : __funnelshift_r(both[g + 1], both[g + 2], bits);
            const int i = tid + c * THREADS;
            if (i < vecs && i * N < p.k) put(i, out);
        }
    } else {
#pragma unroll
        for (int c = 0; c < KEEP; ++c) {
            if (tid + c * THREADS < vecs) {
                uint32_t code[W];
                codes(kept[c], code);
                put(tid + c * THREADS, code);
            }
        }
        if constexpr (THREADS == 256) {
            for (int i = tid + KEEP * THREADS; i < vecs; i += THREADS) {
                uint32_t code[W];
                codes(load(i), code);
                put(i, code);
            }
        }
    }
    if (live && tid == 0) p.scale[row] = qs.scale;
}

}  // namespace rpfq
