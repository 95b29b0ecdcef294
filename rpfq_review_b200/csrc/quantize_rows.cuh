// Rows to 8-bit codes with one scale per row (the tokens of an activation
// matrix, or the output channels of a weight matrix):
//
//   t = max(amax |x|, 1e-30);  s = fl(fl(1 / t) 127);  q = rint(fl(x s))  (half to even)
//   scale = fl(t / 127),  x ~ q scale
//
// the same reciprocal-multiply arithmetic as the other quantizers here. |x| <= t
// bounds fl(x s) by 127 (1 + 2^-22), so |q| <= 127 without a clamp. The 1e-30
// floor keeps s finite: a row of zeros (or of values far below it) gets codes of
// zero. A row that holds a NaN or an infinity has no scale: its scale is NaN and
// its codes are zero, so that every output of the product reads NaN.
//
// Bound by memory: each value is read once from DRAM and leaves as one byte.
// One warp per row; the second pass over the row hits L1 / L2.
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

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// fmaxf drops a NaN, so non-finite values are tracked on the side.
struct RowMax {
    float amax = 0.0f;
    bool bad = false;
    __device__ __forceinline__ void add(float v) {
        const float a = fabsf(v);
        bad |= !(a <= 3.402823466e38f);
        amax = fmaxf(amax, a);
    }
};

template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantizeRowsParams p) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents();
    if (row >= p.m) return;
    const T* __restrict__ x = static_cast<const T*>(p.x) + row * p.ldx;
    int8_t* __restrict__ q = p.q + row * p.ldq;
    RowMax r;
    for (int i = lane; i < p.k; i += 32) r.add(to_f32(x[i]));
    const float amax = warp_max(r.amax);
    const bool bad = __any_sync(0xffffffffu, r.bad);
    const float t = fmaxf(amax, kQuantRowTiny);
    const float s = bad ? 0.0f : __fmul_rn(__frcp_rn(t), 127.0f);
    for (int i = lane; i < p.k; i += 32)
        q[i] = bad ? int8_t(0) : static_cast<int8_t>(__float2int_rn(__fmul_rn(to_f32(x[i]), s)));
    if (lane == 0) p.scale[row] = bad ? __int_as_float(0x7fffffff) : __fdiv_rn(t, 127.0f);
}

}  // namespace rpfq
