// The int8 product for at most 8 rows (single tokens): bound by reading w once.
//
// A block stages the codes of all rows in shared memory (quantizing fp16 / fp32
// rows itself, each block for itself: the rows are a few KB, so nothing has to be
// written, awaited or read back), then each warp takes COLS output channels: its
// lanes walk k in 16-byte chunks of w, multiply four codes at a time (dp4a) and
// add up over the lanes once at the end. The sums are exact int32, so the result
// is that of the tensor-core kernels bit for bit. More channels per warp reuse a
// chunk of x more often; fewer leave more loads in flight when there is one row.
#pragma once

#include "gemm_i8.cuh"
#include "quantize_rows.cuh"

namespace rpfq {

constexpr int kFewRows = 8;
constexpr int kFewThreads = 256;
constexpr int kFewSmem = 98304;  // codes of the rows: two blocks per SM

enum : int { kXCodes = 0, kXHalf = 1, kXFloat = 2 };

struct GemmI8FewParams {
    GemmI8Params g;
    const void* x;      // codes, fp16 or fp32 [m, k]
    int64_t ldx;        // in elements
    const int8_t* w;
    int64_t ldw;
    int32_t x_vector;   // rows of x on 16 bytes
};

template <typename T>
__device__ __forceinline__ void few_quantize_row(const T* __restrict__ x, int k, int kp, bool vector, int8_t* codes,
                                                 float* scale, float* part) {
    using V = QuantVec<T>;
    constexpr int N = V::N;
    const int vecs = (k + N - 1) / N;
    auto load = [&](int i) {
        V v;
        if (vector && (i + 1) * N <= k) {
            v.raw = *reinterpret_cast<const uint4*>(x + i * N);
        } else {
            alignas(16) T e[N];
#pragma unroll
            for (int j = 0; j < N; ++j) e[j] = i * N + j < k ? x[i * N + j] : T(0.0f);
            v.raw = *reinterpret_cast<const uint4*>(e);
        }
        return v;
    };
    float amax = 0.0f;
    for (int i = threadIdx.x; i < vecs; i += kFewThreads) amax = max_nan(amax, load(i).amax());
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
    __syncthreads();
    amax = part[0];
#pragma unroll
    for (int w = 1; w < kFewThreads / 32; ++w) amax = max_nan(amax, part[w]);
    const QuantScale qs = quant_scale(amax);
    for (int i = threadIdx.x; i < vecs; i += kFewThreads) {
        uint32_t code[N / 4];
        float f[N];
        load(i).values(f);
        quant_codes<N>(f, qs.s, code);
#pragma unroll
        for (int g = 0; g < N / 4; ++g) reinterpret_cast<uint32_t*>(codes + i * N)[g] = qs.bad ? 0u : code[g];
    }
    for (int i = vecs * N + threadIdx.x; i < kp; i += kFewThreads) codes[i] = 0;
    if (threadIdx.x == 0) *scale = qs.scale;
}

template <int ROWS, int COLS, int XT, bool OUT_F32>
__global__ void __launch_bounds__(kFewThreads) gemm_i8_few_kernel(const GemmI8FewParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ float s_scale[kFewRows];
    __shared__ float s_part[kFewRows][8];
    int8_t* codes = reinterpret_cast<int8_t*>(smem_raw);
    const int k = p.g.k, kp = (k + 15) / 16 * 16, chunks = kp / 16;
    const int rows = static_cast<int>(p.g.m);  // <= ROWS
    const int lane = threadIdx.x & 31;
    const int col0 = (static_cast<int>(blockIdx.x) * (kFewThreads / 32) + (threadIdx.x >> 5)) * COLS;
    pdl_wait();
    pdl_launch_dependents();
    // the first chunks of w are on their way while the rows are staged
    auto load_w = [&](int c, int chunk) {
        const int col = col0 + c < p.g.n ? col0 + c : p.g.n - 1;
        const int8_t* w = p.w + col * p.ldw + chunk * 16;
        if (chunk * 16 + 16 <= k) return __ldg(reinterpret_cast<const uint4*>(w));
        alignas(16) int8_t e[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) e[j] = chunk * 16 + j < k ? w[j] : int8_t(0);
        return *reinterpret_cast<const uint4*>(e);
    };
    uint4 first[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) first[c] = lane < chunks ? load_w(c, lane) : make_uint4(0, 0, 0, 0);
    if constexpr (XT == kXCodes) {
        for (int i = threadIdx.x; i < rows * chunks; i += kFewThreads) {
            const int r = i / chunks, c = i - r * chunks;
            const int8_t* x = static_cast<const int8_t*>(p.x) + r * p.ldx + c * 16;
            if (c * 16 + 16 <= k) {
                *reinterpret_cast<uint4*>(codes + r * kp + c * 16) = *reinterpret_cast<const uint4*>(x);
            } else {
                for (int j = 0; j < 16; ++j) codes[r * kp + c * 16 + j] = c * 16 + j < k ? x[j] : int8_t(0);
            }
        }
        if (threadIdx.x < rows) s_scale[threadIdx.x] = p.g.x_scale[threadIdx.x];
    } else {
        using T = typename std::conditional<XT == kXHalf, __half, float>::type;
        for (int r = 0; r < rows; ++r)
            few_quantize_row<T>(static_cast<const T*>(p.x) + r * p.ldx, k, kp, p.x_vector != 0, codes + r * kp,
                                &s_scale[r], s_part[r]);
    }
    __syncthreads();
    int acc[ROWS][COLS] = {};
    for (int chunk = lane; chunk < chunks; chunk += 32) {
        uint4 w[COLS];
#pragma unroll
        for (int c = 0; c < COLS; ++c) w[c] = chunk == lane ? first[c] : load_w(c, chunk);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (r < rows) {
                const uint4 x = *reinterpret_cast<const uint4*>(codes + r * kp + chunk * 16);
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    int a = acc[r][c];
                    a = __dp4a(static_cast<int>(x.x), static_cast<int>(w[c].x), a);
                    a = __dp4a(static_cast<int>(x.y), static_cast<int>(w[c].y), a);
                    a = __dp4a(static_cast<int>(x.z), static_cast<int>(w[c].z), a);
                    a = __dp4a(static_cast<int>(x.w), static_cast<int>(w[c].w), a);
                    acc[r][c] = a;
                }
            }
        }
    }
    // lane r * COLS + c keeps output (r, c)
    int mine = 0;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            const int sum = __reduce_add_sync(0xffffffffu, acc[r][c]);
            if (lane == r * COLS + c) mine = sum;
        }
    const int r = lane / COLS, col = col0 + lane % COLS;
    if (r >= rows || col >= p.g.n) return;
    float b = 0.0f;
    if (p.g.bias != nullptr)
        b = p.g.bias_f32 ? static_cast<const float*>(p.g.bias)[col] : __half2float(static_cast<const __half*>(p.g.bias)[col]);
    float v[4] = {fmaf(__int2float_rn(mine) * p.g.w_scale[col], s_scale[r], b), 0.0f, 0.0f, 0.0f};
    store_i8_outputs<OUT_F32>(p.g, r, col, 1, v);
}

}  // namespace rpfq
