// The int8 product for a few rows (single tokens): bound by reading w once. One row
// of k = 4096 against n = 1024 / 4096: 2.3 / 3.4 us of device time in a graph, 2.1
// us of it what k = 768 takes too.
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

// All rows at once: 256 / ROWS threads per row (ROWS a power of two).
template <int ROWS, typename T>
__device__ __forceinline__ void few_quantize(const T* __restrict__ x0, int64_t ldx, int rows, int k, int kp, bool vector,
                                             int8_t* codes, float* scale, float (*part)[8]) {
    using V = QuantVec<T>;
    constexpr int N = V::N;
    constexpr int TPR = kFewThreads / ROWS;
    constexpr int WARPS = TPR / 32;  // per row
    const int r = threadIdx.x / TPR, t = threadIdx.x % TPR;
    const int vecs = r < rows ? (k + N - 1) / N : 0;
    const T* x = x0 + r * ldx;
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
    constexpr int KEEP = 4;  // vectors of a thread that stay in registers
    V kept[KEEP];
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
        if (t + c * TPR < vecs) kept[c] = load(t + c * TPR);
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
        if (t + c * TPR < vecs) amax = max_nan(amax, kept[c].amax());
#pragma unroll 4
    for (int i = t + KEEP * TPR; i < vecs; i += TPR) amax = max_nan(amax, load(i).amax());
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if constexpr (WARPS > 1) {
        const int w = t >> 5;
        if ((t & 31) == 0) part[r][w] = amax;
        __syncthreads();
        amax = part[r][0];
#pragma unroll
        for (int i = 1; i < WARPS; ++i) amax = max_nan(amax, part[r][i]);
    }
    if (r >= rows) return;
    const QuantScale qs = quant_scale(amax);
    int8_t* q = codes + r * kp;
    auto store = [&](int i, const V& v) {
        uint32_t code[N / 4];
        float f[N];
        v.values(f);
        quant_codes<N>(f, qs.s, code);
#pragma unroll
        for (int g = 0; g < N / 4; ++g) reinterpret_cast<uint32_t*>(q + i * N)[g] = qs.bad ? 0u : code[g];
    };
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
        if (t + c * TPR < vecs) store(t + c * TPR, kept[c]);
#pragma unroll 4
    for (int i = t + KEEP * TPR; i < vecs; i += TPR) store(i, load(i));
    for (int i = vecs * N + t; i < kp; i += TPR) q[i] = 0;
    if (t == 0) scale[r] = qs.scale;
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
        const int8_t* src = p.w + col * p.ldw + chunk * 16;
        if (chunk * 16 + 16 <= k) return __ldg(reinterpret_cast<const uint4*>(src));
        alignas(16) int8_t e[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) e[j] = chunk * 16 + j < k ? src[j] : int8_t(0);
        return *reinterpret_cast<const uint4*>(e);
    };
    constexpr int U = 8 / COLS;  // chunks of a lane in flight
    uint4 w[U][COLS];
    auto load_chunks = [&](int c0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < COLS; ++c) w[u][c] = c0 + 32 * u < chunks ? load_w(c, c0 + 32 * u) : make_uint4(0, 0, 0, 0);
    };
    load_chunks(lane);
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
        few_quantize<ROWS, T>(static_cast<const T*>(p.x), p.ldx, rows, k, kp, p.x_vector != 0, codes, s_scale, s_part);
    }
    __syncthreads();
    int acc[ROWS][COLS] = {};
    for (int c0 = lane; c0 < chunks; c0 += 32 * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int chunk = c0 + 32 * u < chunks ? c0 + 32 * u : chunks - 1;  // past the row: w is zero
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const uint4 x = *reinterpret_cast<const uint4*>(codes + (r < rows ? r : 0) * kp + chunk * 16);
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    int a = acc[r][c];
                    a = __dp4a(static_cast<int>(x.x), static_cast<int>(w[u][c].x), a);
                    a = __dp4a(static_cast<int>(x.y), static_cast<int>(w[u][c].y), a);
                    a = __dp4a(static_cast<int>(x.z), static_cast<int>(w[u][c].z), a);
                    a = __dp4a(static_cast<int>(x.w), static_cast<int>(w[u][c].w), a);
                    acc[r][c] = a;
                }
            }
        }
        if (c0 + 32 * U < chunks) load_chunks(c0 + 32 * U);
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
    float v = fmaf(__int2float_rn(mine) * p.g.w_scale[col], s_scale[r], b), unused = 0.0f;
    if (p.g.activation == kActGelu) gelu_log_pair(v, unused);
    using Out = typename std::conditional<OUT_F32, float, __half>::type;
    if (p.g.residual != nullptr) v += static_cast<float>(static_cast<const Out*>(p.g.residual)[r * p.g.ldr + col]);
    static_cast<Out*>(p.g.y)[r * p.g.ldy + col] = static_cast<Out>(v);
}

}  // namespace rpfq
