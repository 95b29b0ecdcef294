// Matrix product of 8-bit codes with a scale per token and per output channel:
//
//   y[m, n] = act( x_scale[m] w_scale[n] sum_k xq[m, k] wq[n, k] + bias[n] ) (+ residual[m, n])
//
// xq: int8 [M, K], wq: int8 [N, K] (both K-major), sums in int32 on the tensor
// cores (tcgen05 kind::i8, K = 32 per instruction), which is exact: K < 2^17
// keeps |sum| < 2^31. The sum is rounded to fp32 once and scaled there; y and
// residual are fp16 or fp32 (same dtype), rounded once at the end.
//
// Tile kernel (fewer rows than fill the GPU with CTA pairs): a cluster of S CTAs
// per 128 x BN tile, each with every S-th part of the k-blocks. Warp 0 loads
// k-blocks of 128 bytes of x and w by TMA (128-byte swizzle) into a ring, warp 1
// issues the MMAs into BN TMEM columns; then all eight warps move the int32 sums to
// shared memory. With S > 1 CTA r of the cluster adds up the S parts of its share of
// the rows over distributed shared memory: no workspace, and integers add to the
// same sum in any order. Rows are written whole, lane = column, so any n, stride and
// alignment is written in order.
#pragma once

#include <type_traits>

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
    int32_t x_rows;          // tile kernel: rows of the x box: 128, or fewer when m is small
    int32_t splits;          // tile kernel: CTAs of a tile (the cluster), each with a part of k
    int32_t tail_tiles;      // pair kernel: last-wave tiles cut into `pieces` column pieces
    int32_t pieces;          // 0: none; else 2 or 4
    int* err;
};

template <int BN>
struct GemmI8TileCfg {
    static constexpr int BM = 128;
    static constexpr int BK = 128;  // int8: one swizzle row
    static constexpr int STAGES = BN == 128 ? 6 : 8;
    static constexpr int A_BYTES = BM * BK;
    static constexpr int B_BYTES = BN * BK;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int THREADS = 256;
    static constexpr int ROW = BN + 4;  // int32 words of a staged row: lanes of a warp store to all banks
    static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + 128 * 4 + 256;
    static_assert(BM * ROW * 4 <= STAGES * STAGE_BYTES, "the staged tile reuses the ring");
    static_assert((2 * STAGES + 2) * 8 <= 256, "barriers");
};

// GELU(v) = v Phi(v) = max(v, 0) - a Phi(-a) with a = |v|, and Phi(-a) = 2^Q(a) for a
// polynomial Q of degree 8 fitted to log2 Phi(-a) on [0, 5.5] (weighted by
// Phi(-a)^0.8, iteratively reweighted least squares); Q falls on beyond that. Off by
// at most 0.75 x 2^-24 |v| in fp32 Horner steps with an exact 2^x; the hardware's 2^x
// and the last rounding make it 1.9 (measured over 10^7 arguments; 0.5 v (1 + erf) in
// fp32: 1.95). One special-function result per value, where erf by exponential and
// reciprocal takes two (m = 50432, k = 1024, n = 4096: 177 against 191 us).
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

// Four outputs of a row lie at columns col + e * step (those inside n). Their
// residual, to be read for several rows before the first is written: y may be the
// residual.
template <bool OUT_F32, bool VEC>
__device__ __forceinline__ void load_i8_residual(const GemmI8Params& p, int64_t row, int col, int step, float (&r)[4]) {
    using Out = typename std::conditional<OUT_F32, float, __half>::type;
    const Out* src = static_cast<const Out*>(p.residual) + row * p.ldr + col;
    if (VEC && col + 4 <= p.n) {
        if constexpr (OUT_F32) {
            const float4 a = *reinterpret_cast<const float4*>(src);
            r[0] = a.x, r[1] = a.y, r[2] = a.z, r[3] = a.w;
        } else {
            const uint2 a = *reinterpret_cast<const uint2*>(src);
            const float2 a0 = __half22float2(*reinterpret_cast<const __half2*>(&a.x));
            const float2 a1 = __half22float2(*reinterpret_cast<const __half2*>(&a.y));
            r[0] = a0.x, r[1] = a0.y, r[2] = a1.x, r[3] = a1.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = col + e * step < p.n ? static_cast<float>(src[e * step]) : 0.0f;
    }
}

// The value, activated, plus the residual, rounded once.
template <bool OUT_F32, bool RES, bool VEC>
__device__ __forceinline__ void store_i8_outputs(const GemmI8Params& p, int64_t row, int col, int step, float (&v)[4],
                                                 const float (&r)[4]) {
    using Out = typename std::conditional<OUT_F32, float, __half>::type;
    if (p.activation == kActGelu) {
        gelu_log_pair(v[0], v[1]);
        gelu_log_pair(v[2], v[3]);
    }
    if constexpr (RES) v[0] += r[0], v[1] += r[1], v[2] += r[2], v[3] += r[3];
    Out* y = static_cast<Out*>(p.y) + row * p.ldy + col;
    if (VEC && col + 4 <= p.n) {
        if constexpr (OUT_F32) {
            *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            const __half2 h0 = __floats2half2_rn(v[0], v[1]), h1 = __floats2half2_rn(v[2], v[3]);
            *reinterpret_cast<uint2*>(y) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e * step < p.n) y[e * step] = static_cast<Out>(v[e]);
}

// RES: with a residual; VEC: rows of y (and of the residual) take vectors of four.
// Both at compile time: a launch this short pays for every instruction it fetches.
template <int BN, bool OUT_F32, bool RES, bool VEC>
__global__ void __launch_bounds__(256)
    gemm_i8_tile_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                        const GemmI8Params p) {
    using C = GemmI8TileCfg<BN>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* s_xs = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE_BYTES);  // the tile's x scales
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_xs + 128);
    uint64_t* full_bar = bars;
    uint64_t* empty_bar = bars + C::STAGES;
    uint64_t* done_bar = bars + 2 * C::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::STAGES + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

    const int S = p.splits;
    const int split = static_cast<int>(blockIdx.x) % S;  // the rank in the cluster
    const int tile = static_cast<int>(blockIdx.x) / S;
    const int num_n = (p.n + BN - 1) / BN;
    const int64_t m0 = static_cast<int64_t>(tile / num_n) * C::BM;
    const int n0 = tile % num_n * BN;
    const int num_k = (p.k + C::BK - 1) / C::BK;
    const int kb_lo = static_cast<int>(static_cast<int64_t>(split) * num_k / S);
    const int nkb = static_cast<int>(static_cast<int64_t>(split + 1) * num_k / S) - kb_lo;  // >= 1: S <= num_k
    const int rows = static_cast<int>(p.m - m0 < C::BM ? p.m - m0 : C::BM);

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

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        const uint32_t elected = elect_one();
        const uint32_t bytes = static_cast<uint32_t>(p.x_rows * C::BK + C::B_BYTES);
        const uint32_t ring = smem_u32(smem), full0 = smem_u32(full_bar);
        int stage = 0;
        uint32_t phase = 0;
        int i = 0;
        for (; i < nkb; ++i) {
            if (!__all_sync(0xffffffffu, wait_bar(&empty_bar[stage], phase ^ 1, abort_flag, p.err, 111))) break;
            const uint32_t sa = ring + stage * C::STAGE_BYTES;
            mbar_arrive_expect_tx_elected(elected, full0 + 8 * stage, bytes);
            tma_load_2d_elected(elected, sa, &tm_x, full0 + 8 * stage, (kb_lo + i) * C::BK, static_cast<int32_t>(m0));
            tma_load_2d_elected(elected, sa + C::A_BYTES, &tm_w, full0 + 8 * stage, (kb_lo + i) * C::BK, n0);
            if (++stage == C::STAGES) {
                stage = 0;
                phase ^= 1;
            }
        }
        // every load has landed before the ring is used again or the CTA exits
        for (int b = i > C::STAGES ? i - C::STAGES : 0; b < i; ++b) {
            volatile int no_abort = 0;
            wait_bar(&full_bar[b % C::STAGES], (b / C::STAGES) & 1, &no_abort, p.err, 112);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t elected = elect_one();
        constexpr uint32_t idesc = umma_idesc_i8(C::BM, BN);
        const uint64_t a_desc0 = umma_desc_sw128_kmajor(smem_u32(smem));
        const uint64_t b_desc0 = umma_desc_sw128_kmajor(smem_u32(smem) + C::A_BYTES);
        const uint32_t empty0 = smem_u32(empty_bar);
        int stage = 0;
        uint32_t phase = 0;
        for (int i = 0; i < nkb; ++i) {
            if (!__all_sync(0xffffffffu, wait_bar(&full_bar[stage], phase, abort_flag, p.err, 211))) break;
            tc_fence_after();
            const uint64_t at = static_cast<uint64_t>(stage * (C::STAGE_BYTES >> 4));
#pragma unroll
            for (int kk = 0; kk < C::BK / 32; ++kk)
                umma_i8_elected(elected, tmem_base, a_desc0 + at + 2 * kk, b_desc0 + at + 2 * kk, idesc, i + kk != 0);
            umma_commit_elected(elected, empty0 + 8 * stage);
            if (++stage == C::STAGES) {
                stage = 0;
                phase ^= 1;
            }
        }
        umma_commit_elected(elected, smem_u32(done_bar));
    }
    // what the outputs need besides the sums is on its way meanwhile
    constexpr int LANES = BN / 4;             // threads of a row, four columns each
    constexpr int STEP = C::THREADS / LANES;  // rows at once
    // the four columns of a thread: neighbours where rows take vectors of four, else
    // LANES apart, so that single values of a row are still written side by side
    const int my = threadIdx.x % LANES;
    constexpr int cstep = VEC ? 1 : LANES;
    const int my_col = VEC ? 4 * my : my;
    const int col = n0 + my_col;
    float ws[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int c = col + e * cstep;
        ws[e] = c < p.n ? __ldg(p.w_scale + c) : 0.0f;
        b[e] = 0.0f;
        if (p.bias != nullptr && c < p.n)
            b[e] = p.bias_f32 ? static_cast<const float*>(p.bias)[c] : __half2float(static_cast<const __half*>(p.bias)[c]);
    }
    // rows of a thread at once; with a residual eight (with 64 columns all it has), whose
    // values come early: y may be the residual, so none of them may wait behind a store
    constexpr int BATCH = RES ? 8 : 4;
    const int r_lo = split * rows / S, r_hi = (split + 1) * rows / S;  // this CTA's share of the rows
    const int r_first = r_lo + threadIdx.x / LANES;
    float res[BATCH][4];
    auto load_residuals = [&](int r0) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (r0 + i * STEP < r_hi && col < p.n)
                load_i8_residual<OUT_F32, VEC>(p, m0 + r0 + i * STEP, col, cstep, res[i]);
    };
    if constexpr (RES) load_residuals(r_first);
    if (threadIdx.x < 128) s_xs[threadIdx.x] = static_cast<int>(threadIdx.x) < rows ? __ldg(p.x_scale + m0 + threadIdx.x) : 0.0f;
    __syncwarp();
    volatile int no_abort = 0;
    bool ok = wait_bar(done_bar, 0, &no_abort, p.err, 311);  // the MMAs have read the ring and written TMEM
    ok = ok && *abort_flag == 0;
    tc_fence_after();
    __syncthreads();
    // ---------------------------------------------------------------- sums to shared memory
    int32_t* staged = reinterpret_cast<int32_t*>(smem);
    {
        const int q = warp & 3;  // TMEM lane quarter of this warp
        const int r = 32 * q + lane;
        constexpr int HALF = BN / 2;
        if (32 * q < rows) {
#pragma unroll
            for (int c = (warp >> 2) * HALF; c < (warp >> 2) * HALF + HALF; c += 32) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(32 * q) << 16) + c, v);
                tmem_ld_wait(v);
#pragma unroll
                for (int g = 0; g < 8; ++g)
                    *reinterpret_cast<uint4*>(staged + r * C::ROW + c + 4 * g) =
                        make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
            }
        }
        tc_fence_before();
    }
    if (S > 1)
        cluster_sync();
    else
        __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem_base, BN);
    // ---------------------------------------------------------------- scales, bias, activation, residual
    if (ok && col < p.n) {
        for (int r0 = r_first; r0 < r_hi; r0 += BATCH * STEP) {
            if (RES && r0 != r_first) load_residuals(r0);
            int a[BATCH][4];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int32_t* at = staged + (r0 + i * STEP) * C::ROW + my_col;
                if (r0 + i * STEP >= r_hi) continue;
                if constexpr (VEC) {
                    const int4 t = *reinterpret_cast<const int4*>(at);
                    a[i][0] = t.x, a[i][1] = t.y, a[i][2] = t.z, a[i][3] = t.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[i][e] = at[e * LANES];
                }
            }
            for (int o = 1; o < S; ++o) {
                const uint32_t from = static_cast<uint32_t>(split + o < S ? split + o : split + o - S);
                const uint32_t base = mapa_shared(smem_u32(staged + my_col), from);
                int t[BATCH][4];
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const uint32_t at = base + (r0 + i * STEP) * C::ROW * 4;
                    if (r0 + i * STEP >= r_hi) continue;
                    if constexpr (VEC) {
                        const int4 u = ld_shared_cluster_v4(at);
                        t[i][0] = u.x, t[i][1] = u.y, t[i][2] = u.z, t[i][3] = u.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) t[i][e] = ld_shared_cluster(at + 4 * e * LANES);
                    }
                }
#pragma unroll
                for (int i = 0; i < BATCH; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (r0 + i * STEP < r_hi) a[i][e] += t[i][e];
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int r = r0 + i * STEP;
                if (r >= r_hi) break;
                const float xs = s_xs[r];
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = fmaf(__int2float_rn(a[i][e]) * ws[e], xs, b[e]);
                store_i8_outputs<OUT_F32, RES, VEC>(p, m0 + r, col, cstep, v, res[i]);
            }
        }
    }
    __syncwarp();
    if (S > 1) cluster_sync();  // no CTA leaves while another reads its sums
}

}  // namespace rpfq
