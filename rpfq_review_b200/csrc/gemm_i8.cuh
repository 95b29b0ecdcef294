// Matrix product of 8-bit codes with a scale per token and per output channel:
//
//   y[m, n] = act( x_scale[m] w_scale[n] sum_k xq[m, k] wq[n, k] + bias[n] ) (+ residual[m, n])
//
// xq: int8 [M, K], wq: int8 [N, K] (both K-major), sums in int32 on the tensor
// cores (tcgen05 kind::i8, K = 32 per instruction), which is exact: K < 2^17
// keeps |sum| < 2^31. The sum is rounded to fp32 once and scaled there; y and
// residual are fp16 or fp32 (same dtype), rounded once at the end.
//
// Tile kernel: one CTA per 128 x BN tile. Warp 0 loads k-blocks of 128 bytes of
// x and w by TMA (128-byte swizzle) into a ring, warp 1 issues the MMAs into
// BN TMEM columns; then all six warps move the accumulator through shared memory
// and write whole rows, lane = column, so any n, stride and alignment is
// written in order.
#pragma once

#include "gemm.cuh"
#include "ptx.cuh"

namespace rpfq {

struct GemmI8Params {
    const float* x_scale;    // [M]
    const float* w_scale;    // [N]
    const void* bias;        // [N] fp16 (fp32 with bias_f32) or nullptr
    const void* residual;    // [M, N], same dtype as y, or nullptr
    int64_t ldr;
    void* y;
    int64_t ldy;
    int64_t m;
    int32_t n, k;
    int32_t activation;
    int32_t bias_f32;
    int32_t vec_out;         // y rows (tile kernel: and the residual's) take vectors of four values; pairs: TMA stores
    int32_t vec_res;         // pairs: residual rows take TMA loads
    int32_t x_rows;          // rows of the x box: 128, or fewer when m is small
    int32_t tail_tiles;      // pair kernel: last-wave tiles cut into `pieces` column pieces
    int32_t pieces;          // 0: none; else 2 or 4
    int* err;
};

template <int BN>
struct GemmI8TileCfg {
    static constexpr int BM = 128;
    static constexpr int BK = 128;  // int8: one swizzle row
    static constexpr int STAGES = BN == 128 ? 4 : 6;
    static constexpr int A_BYTES = BM * BK;
    static constexpr int B_BYTES = BN * BK;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int THREADS = 192;
    static constexpr int ROW = BN + 4;  // int32 words of a staged row: lanes of a warp store to all banks
    static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + 256;
    static_assert(BM * ROW * 4 <= STAGES * STAGE_BYTES, "the staged tile reuses the ring");
};

// GELU(v) = v Phi(v) = max(v, 0) - a Phi(-a) with a = |v|, and Phi(-a) = 2^Q(a) for a
// polynomial Q of degree 8 fitted to log2 Phi(-a) on [0, 5.5] (weighted by
// Phi(-a)^0.8, iteratively reweighted least squares); Q falls on beyond that. Off by
// at most 1.3 x 2^-24 |v| with an exact 2^x in fp32 Horner steps. One
// special-function result per value, where erf by exponential and reciprocal takes
// two: with those the epilogue of m = 50432, k = 1024, n = 4096 took 205 us.
// max.NaN keeps a NaN; the clamp at 64 keeps Q finite (GELU(inf) = inf).
__device__ __forceinline__ void gelu_log_pair(float& v0, float& v1) {
    const uint64_t na = f2_pack(fmaxf(-fabsf(v0), -64.0f), fmaxf(-fabsf(v1), -64.0f));
    auto c2 = [](float c) { return f2_pack(c, c); };
    uint64_t q = f2_fma(na, c2(-2.02745741e-06f), c2(-3.01461678e-05f));
    q = f2_fma(na, q, c2(-0.00014467015f));
    q = f2_fma(na, q, c2(0.000230890437f));
    q = f2_fma(na, q, c2(0.00717717316f));
    q = f2_fma(na, q, c2(0.0525683947f));
    q = f2_fma(na, q, c2(-0.459186375f));
    q = f2_fma(na, q, c2(1.15110767f));
    q = f2_fma(na, q, c2(-0.99999994f));
    float q0, q1;
    f2_unpack(q, q0, q1);
    asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(v0));
    asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(v1));
    f2_unpack(f2_fma(na, f2_pack(ex2_approx(q0), ex2_approx(q1)), f2_pack(v0, v1)), v0, v1);
}

// The four outputs at (row, col..col + 3), `live` of them inside n.
template <bool OUT_F32>
__device__ __forceinline__ void store_i8_outputs(const GemmI8Params& p, int64_t row, int col, int live, float (&v)[4]) {
    if (p.activation == kActGelu) {
        gelu_log_pair(v[0], v[1]);
        gelu_log_pair(v[2], v[3]);
    }
    if constexpr (OUT_F32) {
        float* y = static_cast<float*>(p.y) + row * p.ldy + col;
        const float* r = p.residual ? static_cast<const float*>(p.residual) + row * p.ldr + col : nullptr;
        if (p.vec_out && live == 4) {
            if (r) {
                const float4 a = *reinterpret_cast<const float4*>(r);
                v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
            }
            *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < live) y[e] = v[e] + (r ? r[e] : 0.0f);
        }
    } else {
        __half* y = static_cast<__half*>(p.y) + row * p.ldy + col;
        const __half* r = p.residual ? static_cast<const __half*>(p.residual) + row * p.ldr + col : nullptr;
        if (p.vec_out && live == 4) {
            if (r) {
                const uint2 a = *reinterpret_cast<const uint2*>(r);
                const float2 a0 = __half22float2(*reinterpret_cast<const __half2*>(&a.x));
                const float2 a1 = __half22float2(*reinterpret_cast<const __half2*>(&a.y));
                v[0] += a0.x, v[1] += a0.y, v[2] += a1.x, v[3] += a1.y;
            }
            const __half2 h0 = __floats2half2_rn(v[0], v[1]), h1 = __floats2half2_rn(v[2], v[3]);
            uint2 o;
            o.x = *reinterpret_cast<const uint32_t*>(&h0);
            o.y = *reinterpret_cast<const uint32_t*>(&h1);
            *reinterpret_cast<uint2*>(y) = o;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < live) y[e] = __float2half_rn(v[e] + (r ? __half2float(r[e]) : 0.0f));
        }
    }
}

template <int BN, bool OUT_F32>
__global__ void __launch_bounds__(192)
    gemm_i8_tile_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                        const GemmI8Params p) {
    using C = GemmI8TileCfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES);
    uint64_t* full_bar = bars;
    uint64_t* empty_bar = bars + C::STAGES;
    uint64_t* done_bar = bars + 2 * C::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::STAGES + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int num_n = (p.n + BN - 1) / BN;
    const int64_t m0 = static_cast<int64_t>(blockIdx.x / num_n) * C::BM;
    const int n0 = static_cast<int>(blockIdx.x % num_n) * BN;
    const int num_k = (p.k + C::BK - 1) / C::BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&tm_x);
        prefetch_tmap(&tm_w);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, BN);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    bool ok = true;
    if (warp == 0 && lane == 0) {
        // ------------------------------------------------------------ producer
        const uint32_t bytes = static_cast<uint32_t>(p.x_rows * C::BK + C::B_BYTES);
        int kb = 0;
        for (; kb < num_k; ++kb) {
            const int s = kb % C::STAGES;
            if (!wait_bar(&empty_bar[s], ((kb / C::STAGES) & 1) ^ 1, abort_flag, p.err, 111)) break;
            uint8_t* sa = smem + s * C::STAGE_BYTES;
            mbar_arrive_expect_tx(&full_bar[s], bytes);
            tma_load_2d(sa, &tm_x, &full_bar[s], kb * C::BK, static_cast<int32_t>(m0));
            tma_load_2d(sa + C::A_BYTES, &tm_w, &full_bar[s], kb * C::BK, n0);
        }
        // every load has landed before the ring is used again or the CTA exits
        for (int i = kb > C::STAGES ? kb - C::STAGES : 0; i < kb; ++i) {
            volatile int no_abort = 0;
            wait_bar(&full_bar[i % C::STAGES], (i / C::STAGES) & 1, &no_abort, p.err, 112);
        }
    } else if (warp == 1 && lane == 0) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t idesc = umma_idesc_i8(C::BM, BN);
        for (int kb = 0; kb < num_k; ++kb) {
            const int s = kb % C::STAGES;
            if (!wait_bar(&full_bar[s], (kb / C::STAGES) & 1, abort_flag, p.err, 211)) break;
            tc_fence_after();
            const uint32_t a_addr = smem_u32(smem + s * C::STAGE_BYTES);
            const uint64_t a_desc = umma_desc_sw128_kmajor(a_addr);
            const uint64_t b_desc = umma_desc_sw128_kmajor(a_addr + C::A_BYTES);
#pragma unroll
            for (int kk = 0; kk < C::BK / 32; ++kk)
                umma_i8(tmem_base, a_desc + 2 * kk, b_desc + 2 * kk, idesc, kb + kk != 0);
            umma_commit(&empty_bar[s]);
        }
        umma_commit(done_bar);
    }
    __syncwarp();
    {
        // the MMAs have read the ring and written TMEM
        volatile int no_abort = 0;
        ok = wait_bar(done_bar, 0, &no_abort, p.err, 311);
        ok = ok && *abort_flag == 0;
    }
    tc_fence_after();
    __syncthreads();
    // ---------------------------------------------------------------- accumulator to shared memory
    int32_t* staged = reinterpret_cast<int32_t*>(smem);
    const int rows = static_cast<int>(p.m - m0 < C::BM ? p.m - m0 : C::BM);
    if (warp >= 2) {
        const int q = warp & 3;  // TMEM lane quarter of this warp
        const int r = 32 * q + lane;
        if (32 * q < rows) {
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(32 * q) << 16) + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int g = 0; g < 8; ++g)
                    *reinterpret_cast<uint4*>(staged + r * C::ROW + c + 4 * g) =
                        make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem_base, BN);
    if (!ok) return;
    // ---------------------------------------------------------------- scales, bias, activation, residual
    constexpr int LANES = BN / 4;           // threads of a row, four columns each
    constexpr int STEP = C::THREADS / LANES;  // rows at once
    const int col = n0 + 4 * (threadIdx.x % LANES);
    const int live = p.n - col < 4 ? p.n - col : 4;
    if (live <= 0) return;
    float ws[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        ws[e] = e < live ? __ldg(p.w_scale + col + e) : 0.0f;
        b[e] = 0.0f;
        if (p.bias != nullptr && e < live)
            b[e] = p.bias_f32 ? static_cast<const float*>(p.bias)[col + e]
                              : __half2float(static_cast<const __half*>(p.bias)[col + e]);
    }
    for (int r = threadIdx.x / LANES; r < rows; r += STEP) {
        const float xs = __ldg(p.x_scale + m0 + r);
        const int4 a = *reinterpret_cast<const int4*>(staged + r * C::ROW + 4 * (threadIdx.x % LANES));
        float v[4] = {fmaf(__int2float_rn(a.x) * ws[0], xs, b[0]), fmaf(__int2float_rn(a.y) * ws[1], xs, b[1]),
                      fmaf(__int2float_rn(a.z) * ws[2], xs, b[2]), fmaf(__int2float_rn(a.w) * ws[3], xs, b[3])};
        store_i8_outputs<OUT_F32>(p, m0 + r, col, live, v);
    }
}

}  // namespace rpfq
