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
// per thread; longer rows are read again, from L1 / L2). A warp takes a row; when
// the rows are too few to fill the GPU or too long for a warp's registers, a block
// of 256 threads does. The maximum of fp16 rows is taken on half pairs; fl(x s)
// is rounded by adding 1.5 * 2^23 (half to even, as rint), which leaves the code
// in the low byte of the sum.
#pragma once

#include "actquant.cuh"
#include "ptx.cuh"

namespace rpfq {

constexpr float kQuantRowTiny = 1e-30f;
constexpr int kQuantRowKeep = 8;  // 16-byte vectors of a row that a thread keeps

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

// VECTOR: rows of x on 16 bytes and rows of q on QuantVec::N bytes; otherwise
// vectors are put together value by value. THREADS per row: 32 or 256.
template <typename T, bool VECTOR, int THREADS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantizeRowsParams p) {
    using V = QuantVec<T>;
    constexpr int N = V::N;
    const int tid = threadIdx.x & (THREADS - 1);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / THREADS) + threadIdx.x / THREADS;
    pdl_wait();
    pdl_launch_dependents();
    if (row >= p.m) return;  // a whole warp or block
    const T* __restrict__ x = static_cast<const T*>(p.x) + row * p.ldx;
    int8_t* __restrict__ q = p.q + row * p.ldq;
    const int vecs = (p.k + N - 1) / N;
    auto load = [&](int i) {
        V v;
        if (VECTOR && (i + 1) * N <= p.k) {
            v.raw = *reinterpret_cast<const uint4*>(x + i * N);
        } else {
            alignas(16) T e[N];
#pragma unroll
            for (int j = 0; j < N; ++j) e[j] = i * N + j < p.k ? x[i * N + j] : T(0.0f);
            v.raw = *reinterpret_cast<const uint4*>(e);
        }
        return v;
    };
    V kept[kQuantRowKeep];
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < kQuantRowKeep; ++c)
        if (tid + c * THREADS < vecs) kept[c] = load(tid + c * THREADS);
#pragma unroll
    for (int c = 0; c < kQuantRowKeep; ++c)
        if (tid + c * THREADS < vecs) amax = max_nan(amax, kept[c].amax());
    for (int i = tid + kQuantRowKeep * THREADS; i < vecs; i += THREADS) amax = max_nan(amax, load(i).amax());
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if constexpr (THREADS == 256) {
        __shared__ float part[8];
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
        __syncthreads();
        amax = part[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) amax = max_nan(amax, part[w]);
    }
    const QuantScale qs = quant_scale(amax);
    auto store = [&](int i, const V& v) {
        uint32_t code[N / 4];
        float f[N];
        v.values(f);
        quant_codes<N>(f, qs.s, code);
#pragma unroll
        for (int g = 0; g < N / 4; ++g)
            if (qs.bad) code[g] = 0;
        if (VECTOR && (i + 1) * N <= p.k) {
            if constexpr (N == 8)
                *reinterpret_cast<uint2*>(q + i * N) = make_uint2(code[0], code[1]);
            else
                *reinterpret_cast<uint32_t*>(q + i * N) = code[0];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (i * N + j < p.k) q[i * N + j] = static_cast<int8_t>(code[j / 4] >> (8 * (j % 4)));
        }
    };
#pragma unroll
    for (int c = 0; c < kQuantRowKeep; ++c)
        if (tid + c * THREADS < vecs) store(tid + c * THREADS, kept[c]);
    for (int i = tid + kQuantRowKeep * THREADS; i < vecs; i += THREADS) store(i, load(i));
    if (tid == 0) p.scale[row] = qs.scale;
}

}  // namespace rpfq
