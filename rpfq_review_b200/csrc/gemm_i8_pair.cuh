// The int8 product for many rows: persistent CTA pairs, 256 x 256 tiles.
//
// A cluster of two CTAs computes a tile with tcgen05.mma.cta_group::2.kind::i8
// (M = 256 over the two SMs' TMEM, N = 256, K = 32); each CTA loads its 128 rows
// of x and half of the 256 rows of w per k-block of 128 bytes, so that an SM
// streams 32 KB per 512 cycles of its tensor core at full rate. Two TMEM
// accumulators (2 x 256 columns): the epilogue of one tile runs under the main
// loop of the next.
//
// CTA = 12 warps: warp 0 TMA producer, warp 1 TMEM owner and (leader CTA) MMA
// issuer, warps 4..11 epilogue, each with the 32 rows of its TMEM lane quarter
// and one column half of the tile, in steps of 128 bytes of output per row. The
// scales and the bias of a tile's columns are staged in shared memory once per
// tile (a thread holds one row, so every lane reads the same column); the sum is
// converted to fp32, scaled and biased in packed fp32 pairs.
//
// Output and residual steps go through the warp's 128-B-swizzled staging slots by
// TMA when their addresses and row strides are multiples of 16 bytes, and by
// row-wise loads and stores of the warp otherwise (n odd). With a residual there
// are two slots: the next step's residual lands while this one is used.
//
// The last wave of tiles, where at most half full, is cut into column pieces
// (Schedule, gemm.cuh).
#pragma once

#include "gemm.cuh"
#include "gemm_i8.cuh"
#include "ptx.cuh"

namespace rpfq {

template <bool RES>
struct GemmI8PairCfg {
    static constexpr int BM = 128;
    static constexpr int BN = 256;
    static constexpr int BK = 128;  // bytes = int8 values: one swizzle row
    static constexpr int STAGES = RES ? 5 : 6;
    static constexpr int A_BYTES = BM * BK;
    static constexpr int B_BYTES = BN / 2 * BK;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int EPI_WARPS = 8;
    static constexpr int SLOTS = RES ? 2 : 1;
    static constexpr int SLOT_BYTES = 32 * 128;
    static constexpr int COL_BYTES = BN * 2 * 4;  // w_scale and bias of the tile's columns
    static constexpr int BAR_BYTES = 384;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_WARPS * SLOTS * SLOT_BYTES + COL_BYTES + BAR_BYTES;
    static constexpr int THREADS = 384;
    // bars: full, empty [STAGES], tfull, tempty [2], drain, residual [2 per warp], then two words
    static_assert((2 * STAGES + 5 + 2 * EPI_WARPS + 1) * 8 <= BAR_BYTES, "barriers");
    static_assert(SMEM_BYTES <= 232448, "shared memory budget");
    // 128 x 40 + 256 x 232 registers <= 384 x 168 at launch
    static_assert(128 * 40 + 256 * 232 <= THREADS * 168, "register split exceeds the launch allocation");
};

template <bool OUT_F32, bool RES>
__global__ void __launch_bounds__(384, 1)
    gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                        const __grid_constant__ CUtensorMap tm_wp, const __grid_constant__ CUtensorMap tm_y,
                        const __grid_constant__ CUtensorMap tm_r, const GemmI8Params p) {
    using C = GemmI8PairCfg<RES>;
    constexpr int BN = C::BN;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw;
    if (smem_u32(smem) & 1023) {  // the swizzled tiles need it; uniform over the cluster
        if (threadIdx.x == 0) atomicCAS(p.err, 0, 121);
        return;
    }
    uint8_t* slot_base = smem + C::STAGES * C::STAGE_BYTES;
    float* col_base = reinterpret_cast<float*>(slot_base + C::EPI_WARPS * C::SLOTS * C::SLOT_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(col_base) + C::COL_BYTES);
    uint64_t* full_bar = bars;
    uint64_t* empty_bar = bars + C::STAGES;
    uint64_t* tfull_bar = bars + 2 * C::STAGES;
    uint64_t* tempty_bar = tfull_bar + 2;
    uint64_t* drain_bar = tfull_bar + 4;
    uint64_t* res_bar = tfull_bar + 5;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_bar + 2 * C::EPI_WARPS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int num_n = (p.n + BN - 1) / BN;
    const int num_k = (p.k + C::BK - 1) / C::BK;
    const int num_tiles = static_cast<int>((p.m + 255) / 256) * num_n;
    auto schedule = [&]() {
        return Schedule<BN>(static_cast<int>(blockIdx.x >> 1), static_cast<int>(gridDim.x >> 1), num_tiles, num_k, 0, 0,
                            num_k, p.tail_tiles, p.pieces);
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull_bar[b], 1);
            mbar_init(&tempty_bar[b], 2 * C::EPI_WARPS);
        }
        mbar_init(drain_bar, 1);
        for (int b = 0; b < 2 * C::EPI_WARPS; ++b) mbar_init(&res_bar[b], 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&tm_x);
        prefetch_tmap(&tm_w);
        if (p.pieces) prefetch_tmap(&tm_wp);
        if (p.tma_out) prefetch_tmap(&tm_y);
        if (RES && p.tma_res) prefetch_tmap(&tm_r);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 2 * BN);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers exist before any cross-CTA signal
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    if (warp < 4) {
        setmaxnreg_dec40();
        if (warp == 0 && lane == 0) {
            // -------------------------------------------------------- producer
            int stage = 0;
            uint32_t phase = 0;
            int issued = 0;
            bool ok = true;
            auto sched = schedule();
            WorkItem w;
            while (ok && sched.next(w)) {
                const int b_rows = w.width / 2;  // rows of w per CTA: half of the item's columns
                const uint32_t bytes = static_cast<uint32_t>(C::A_BYTES + b_rows * C::BK);
                const int m0 = (w.tile / num_n) * 256 + static_cast<int>(rank) * C::BM;
                const int n0 = (w.tile % num_n) * BN + w.n_off + static_cast<int>(rank) * b_rows;
                const CUtensorMap* tw = w.width == BN ? &tm_w : &tm_wp;
                for (int kb = 0; kb < num_k; ++kb) {
                    if (!wait_bar(&empty_bar[stage], phase ^ 1, abort_flag, p.err, 131)) {
                        ok = false;
                        break;
                    }
                    uint8_t* sa = smem + stage * C::STAGE_BYTES;
                    // both CTAs' bytes complete on the leader's barrier
                    if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * bytes);
                    const uint32_t leader_full = mapa_shared(smem_u32(&full_bar[stage]), 0);
                    tma_load_2d_pair(sa, &tm_x, leader_full, kb * C::BK, m0);
                    tma_load_2d_pair(sa + C::A_BYTES, tw, leader_full, kb * C::BK, n0);
                    ++issued;
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // every load has landed before the CTA may exit; the leader drains for both
            const int pending = rank != 0 ? 0 : (issued < C::STAGES ? issued : C::STAGES);
            for (int i = 1; i <= pending; ++i) {
                int s = stage - i;
                uint32_t ph = phase;
                if (s < 0) {
                    s += C::STAGES;
                    ph ^= 1;
                }
                volatile int no_abort = 0;
                wait_bar(&full_bar[s], ph, &no_abort, p.err, 132);
            }
        } else if (warp == 1 && lane == 0 && rank == 0) {
            // -------------------------------------------------------- MMA issuer
            auto commit_both = [&](uint64_t* bar) {
                const uint32_t a = smem_u32(bar);
                umma_commit_pair(a);
                umma_commit_pair(mapa_shared(a, 1));
            };
            int stage = 0;
            uint32_t phase = 0;
            int acc = 0;
            uint32_t acc_phase = 0;
            bool ok = true;
            auto sched = schedule();
            WorkItem w;
            while (ok && sched.next(w)) {
                if (!wait_bar<true>(&tempty_bar[acc], acc_phase ^ 1, abort_flag, p.err, 231)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
                const uint32_t idesc = umma_idesc_i8(256, w.width);
                for (int kb = 0; kb < num_k; ++kb) {
                    if (!wait_bar(&full_bar[stage], phase, abort_flag, p.err, 232)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(smem + stage * C::STAGE_BYTES);
                    const uint64_t a_desc = umma_desc_sw128_kmajor(a_addr);
                    const uint64_t b_desc = umma_desc_sw128_kmajor(a_addr + C::A_BYTES);
#pragma unroll
                    for (int kk = 0; kk < C::BK / 32; ++kk)
                        umma_i8_pair(d_tmem, a_desc + 2 * kk, b_desc + 2 * kk, idesc, kb + kk != 0);
                    commit_both(&empty_bar[stage]);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                commit_both(&tfull_bar[acc]);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
            // no MMA still writes TMEM when it is freed
            umma_commit_pair(smem_u32(drain_bar));
            volatile int no_abort = 0;
            wait_bar(drain_bar, 0, &no_abort, p.err, 233);
        }
    } else {
        setmaxnreg_inc232();
        // ------------------------------------------------------------ epilogue
        constexpr int CW = OUT_F32 ? 32 : 64;  // output columns of a step: 128 bytes per row
        constexpr int ESZ = OUT_F32 ? 4 : 2;
        constexpr int HALF = BN / 2;
        const int q = warp & 3;
        const int ew = warp - 4;
        const int col_half = ew >> 2;
        uint8_t* slots = slot_base + ew * C::SLOTS * C::SLOT_BYTES;
        float* s_ws = col_base + col_half * 2 * HALF;  // [HALF] scales, then [HALF] biases
        float* s_b = s_ws + HALF;
        const int my_col = threadIdx.x & (HALF - 1);  // the column this thread stages (128 threads per half)
        int acc = 0;
        uint32_t acc_phase = 0;
        uint32_t j = 0;      // running step counter of this warp (slot = j & 1 with a residual)
        uint32_t loads = 0;  // residual steps requested (lane 0)
        bool ok = true;      // after a wait that gave up: only the warps' named barriers are kept up
        auto load_residual = [&](int s, int col0, int64_t row0) {
            mbar_arrive_expect_tx(&res_bar[2 * ew + s], C::SLOT_BYTES);
            tma_load_2d(slots + s * C::SLOT_BYTES, &tm_r, &res_bar[2 * ew + s], col0, static_cast<int32_t>(row0));
            ++loads;
        };
        const uint32_t tempty_leader0 = mapa_shared(smem_u32(&tempty_bar[0]), 0);
        const uint32_t tempty_leader1 = mapa_shared(smem_u32(&tempty_bar[1]), 0);
        auto sched = schedule();
        WorkItem w;
        while (sched.next(w)) {
            const int64_t row0 = static_cast<int64_t>(w.tile / num_n) * 256 + static_cast<int64_t>(rank) * C::BM + 32 * q;
            // a piece (width <= HALF) is drained by the first column half's warps
            const bool piece = w.width != BN;
            const int c_begin = (w.tile % num_n) * BN + w.n_off + (piece ? 0 : col_half * HALF);
            const int valid = piece ? (col_half == 0 ? min(w.width, p.n - c_begin) : 0) : min(HALF, p.n - c_begin);
            const int nsteps = (valid > 0 && row0 < p.m) ? (valid + CW - 1) / CW : 0;
            const float xs = row0 + lane < p.m ? __ldg(p.x_scale + row0 + lane) : 0.0f;
            float ws = 0.0f, bias = 0.0f;
            if (my_col < valid) {
                ws = __ldg(p.w_scale + c_begin + my_col);
                if (p.bias != nullptr)
                    bias = p.bias_f32 ? __ldg(static_cast<const float*>(p.bias) + c_begin + my_col)
                                      : __half2float(static_cast<const __half*>(p.bias)[c_begin + my_col]);
            }
            if constexpr (RES) {
                // the first residual step lands while the main loop runs
                if (ok && p.tma_res && lane == 0 && nsteps > 0) {
                    bulk_wait_group_read<0>();
                    load_residual(j & 1, c_begin, row0);
                }
            }
            named_bar_sync(1 + col_half, 128);  // the four warps are done with the previous tile's columns
            s_ws[my_col] = ws;
            s_b[my_col] = bias;
            named_bar_sync(1 + col_half, 128);
            const uint32_t t_row = tmem_base + (static_cast<uint32_t>(32 * q) << 16) +
                                   static_cast<uint32_t>(acc * BN + (piece ? 0 : col_half * HALF));
            if (ok) ok = __all_sync(0xffffffffu, wait_bar(&tfull_bar[acc], acc_phase, abort_flag, p.err, 331));
            if (!ok) continue;
            tc_fence_after();
            const uint64_t xs2 = f2_pack(xs, xs);
            const int rows_live = p.m - row0 < 32 ? static_cast<int>(p.m - row0) : 32;
#pragma unroll 1
            for (int c = 0; c < nsteps; ++c, ++j) {
                const int col0 = c_begin + c * CW;
                const uint32_t slot = RES ? (j & 1) : 0;
                uint8_t* buf = slots + slot * C::SLOT_BYTES;
                if constexpr (RES) {
                    if (p.tma_res) {
                        // the next step's residual, once that slot's last store has been read out
                        if (lane == 0 && c + 1 < nsteps) {
                            bulk_wait_group_read<0>();
                            load_residual((j + 1) & 1, col0 + CW, row0);
                        }
                    } else {
                        if (p.tma_out && lane == 0) bulk_wait_group_read<0>();
                        __syncwarp();
                        const int cols = min(CW, p.n - col0);
                        for (int r = 0; r < rows_live; ++r)
                            for (int cc = lane; cc < cols; cc += 32) {
                                uint8_t* d = buf + r * 128 + (((cc * ESZ >> 4) ^ (r & 7)) << 4) + (cc * ESZ & 15);
                                const int64_t at = (row0 + r) * p.ldr + col0 + cc;
                                if constexpr (OUT_F32)
                                    *reinterpret_cast<float*>(d) = static_cast<const float*>(p.residual)[at];
                                else
                                    *reinterpret_cast<__half*>(d) = static_cast<const __half*>(p.residual)[at];
                            }
                        __syncwarp();
                    }
                }
                uint32_t r[CW];
#pragma unroll
                for (int h = 0; h < CW / 32; ++h)
                    tmem_ld_32x32b_x32(t_row + c * CW + 32 * h, *reinterpret_cast<uint32_t(*)[32]>(&r[32 * h]));
                tmem_ld_wait();
                float v[CW];
#pragma unroll
                for (int g = 0; g < CW / 4; ++g) {
                    const float4 sw = *reinterpret_cast<const float4*>(s_ws + c * CW + 4 * g);
                    const float4 sb = *reinterpret_cast<const float4*>(s_b + c * CW + 4 * g);
                    const uint64_t a0 = f2_pack(__int2float_rn(static_cast<int>(r[4 * g])),
                                                __int2float_rn(static_cast<int>(r[4 * g + 1])));
                    const uint64_t a1 = f2_pack(__int2float_rn(static_cast<int>(r[4 * g + 2])),
                                                __int2float_rn(static_cast<int>(r[4 * g + 3])));
                    f2_unpack(f2_fma(f2_mul(a0, f2_pack(sw.x, sw.y)), xs2, f2_pack(sb.x, sb.y)), v[4 * g], v[4 * g + 1]);
                    f2_unpack(f2_fma(f2_mul(a1, f2_pack(sw.z, sw.w)), xs2, f2_pack(sb.z, sb.w)), v[4 * g + 2],
                              v[4 * g + 3]);
                }
                if (p.activation == kActGelu) {
#pragma unroll
                    for (int jj = 0; jj < CW; jj += 2) gelu_erf_pair(v[jj], v[jj + 1]);
                }
                if constexpr (RES) {
                    if (p.tma_res)
                        ok = __all_sync(0xffffffffu,
                                        wait_bar(&res_bar[2 * ew + slot], (j >> 1) & 1, abort_flag, p.err, 332));
                    if (!ok) break;
                    // this thread's row of the residual step (128-B swizzle)
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        const uint4 rv = *reinterpret_cast<const uint4*>(buf + lane * 128 + ((g ^ (lane & 7)) << 4));
                        if constexpr (OUT_F32) {
                            v[4 * g + 0] += __uint_as_float(rv.x);
                            v[4 * g + 1] += __uint_as_float(rv.y);
                            v[4 * g + 2] += __uint_as_float(rv.z);
                            v[4 * g + 3] += __uint_as_float(rv.w);
                        } else {
                            const __half2* rh = reinterpret_cast<const __half2*>(&rv);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 f = __half22float2(rh[e]);
                                v[8 * g + 2 * e] += f.x;
                                v[8 * g + 2 * e + 1] += f.y;
                            }
                        }
                    }
                    __syncwarp();  // every lane has read its row before any lane overwrites the slot
                } else {
                    // single slot: the previous step has left it
                    if (p.tma_out && lane == 0) bulk_wait_group_read<0>();
                    __syncwarp();
                }
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    uint4 pk;
                    if constexpr (OUT_F32) {
                        pk = make_uint4(__float_as_uint(v[4 * g]), __float_as_uint(v[4 * g + 1]),
                                        __float_as_uint(v[4 * g + 2]), __float_as_uint(v[4 * g + 3]));
                    } else {
                        const __half2 h0 = __floats2half2_rn(v[8 * g + 0], v[8 * g + 1]);
                        const __half2 h1 = __floats2half2_rn(v[8 * g + 2], v[8 * g + 3]);
                        const __half2 h2 = __floats2half2_rn(v[8 * g + 4], v[8 * g + 5]);
                        const __half2 h3 = __floats2half2_rn(v[8 * g + 6], v[8 * g + 7]);
                        pk = make_uint4(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1),
                                        *reinterpret_cast<const uint32_t*>(&h2), *reinterpret_cast<const uint32_t*>(&h3));
                    }
                    *reinterpret_cast<uint4*>(buf + lane * 128 + ((g ^ (lane & 7)) << 4)) = pk;
                }
                if (p.tma_out) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tm_y, buf, col0, static_cast<int32_t>(row0));
                        bulk_commit_group();
                    }
                } else {
                    __syncwarp();
                    const int cols = min(CW, p.n - col0);
                    for (int r2 = 0; r2 < rows_live; ++r2)
                        for (int cc = lane; cc < cols; cc += 32) {
                            const uint8_t* d = buf + r2 * 128 + (((cc * ESZ >> 4) ^ (r2 & 7)) << 4) + (cc * ESZ & 15);
                            const int64_t at = (row0 + r2) * p.ldy + col0 + cc;
                            if constexpr (OUT_F32)
                                static_cast<float*>(p.y)[at] = *reinterpret_cast<const float*>(d);
                            else
                                static_cast<__half*>(p.y)[at] = *reinterpret_cast<const __half*>(d);
                        }
                    __syncwarp();
                    // the next residual may reach this slot by TMA: order these reads before it
                    if (RES && p.tma_res) fence_proxy_async_smem();
                }
            }
            if (!ok) continue;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc ? tempty_leader1 : tempty_leader0);
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1;
            }
        }
        if (lane == 0) {
            bulk_wait_group<0>();
            // residual steps still in flight (only after a wait that gave up)
            for (; j < loads; ++j) {
                volatile int no_abort = 0;
                wait_bar(&res_bar[2 * ew + (j & 1)], (j >> 1) & 1, &no_abort, p.err, 333);
            }
        }
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer is done with TMEM and with our barriers
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem_base, 2 * BN);
}

}  // namespace rpfq
