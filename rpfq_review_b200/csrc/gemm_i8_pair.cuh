// The int8 product for many rows: persistent CTA pairs, 256 x 256 tiles.
//
// A cluster of two CTAs computes a tile with tcgen05.mma.cta_group::2.kind::i8
// (M = 256 over the two SMs' TMEM, N = 256, K = 32); each CTA loads its 128 rows
// of x and half of the 256 rows of w per k-block of 128 bytes, so that an SM
// streams 32 KB per 512 cycles of its tensor core at full rate. Two TMEM
// accumulators (2 x 256 columns): the epilogue of one tile runs under the main
// loop of the next.
//
// Warp 0 TMA producer, warp 1 TMEM owner and (leader CTA) MMA issuer, from warp 4
// on the epilogue, each warp with the 32 rows of its TMEM lane quarter and one
// column group of the tile, in steps of 128 bytes of output per row. A thread holds
// one row, so the scales and biases of a tile's columns are staged in shared memory
// (loaded one tile ahead, one copy for the four warps of a column group: a copy per
// warp would cost a stage of the ring); the sum is converted to fp32, scaled and
// biased in packed fp32 pairs.
// The accumulator is released as soon as the warp's last part of it is in
// registers, by an arrival without release semantics: a release waits for the
// warp's other memory traffic, which the MMA warp does not read (m = 50432, k =
// 1024, n = 4096: 150 us without GELU against 174..191 with a release). TMEM is
// not ordered by releases and acquires but by PTX's rule for tcgen05 operations of
// different threads: every lane's loads have completed at its tcgen05.wait::ld, its
// tcgen05.fence::before_thread_sync puts them before what follows in execution
// (__syncwarp, then lane 0's arrival), and the MMA warp issues behind a
// tcgen05.fence::after_thread_sync that follows the wait which saw the arrivals.
//
// The loops of warps 0 and 1 run on all lanes with only the issuing instruction
// predicated. On one lane the MMA warp took over 800 cycles for the instructions of
// a k-block while the epilogue competed for its scheduler; a k-block takes 512.
//
// Output and residual steps go through the warp's 128-B-swizzled staging slots by
// TMA when their addresses and row strides are multiples of 16 bytes, and by
// row-wise loads and stores of the warp otherwise (n odd). With a residual there
// are two slots: the next step's residual lands while this one is used.
//
// EW: eight epilogue warps, or sixteen (without a residual) at the price of one stage
// of the ring; rpfq_b200.cu says when, with both sides measured.
//
// Bound by the power-capped tensor cores for long k (m = 50432, k = 4096, n = 1024,
// fp16 out: 135 us, 3.1 POPS, the tensor pipe busy in 98 % of the cycles), by
// the GELU's instructions for k = 1024, by the residual stream beside them for
// fp32 in and out (160 us).
//
// The last wave of tiles, where at most half full, is cut into column pieces
// (Schedule, gemm.cuh).
#pragma once

#include "gemm.cuh"
#include "gemm_i8.cuh"
#include "ptx.cuh"

namespace rpfq {

template <bool RES, int EW>
struct GemmI8PairCfg {
    static_assert(EW == 8 || (EW == 16 && !RES), "epilogue warps");
    static constexpr int BM = 128;
    static constexpr int BN = 256;
    static constexpr int BK = 128;  // bytes = int8 values: one swizzle row
    static constexpr int A_BYTES = BM * BK;
    static constexpr int B_BYTES = BN / 2 * BK;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int GROUP_COLS = BN / (EW / 4);  // columns of a warp
    static constexpr int SLOTS = RES ? 2 : 1;
    static constexpr int SLOT_BYTES = 32 * 128;
    static constexpr int COL_BYTES = BN * 2 * 4;  // w_scale and bias of the tile's columns
    static constexpr int BAR_BYTES = 512;
    static constexpr int OTHER_BYTES = EW * SLOTS * SLOT_BYTES + COL_BYTES + BAR_BYTES;
    static constexpr int STAGES = (232448 - OTHER_BYTES) / STAGE_BYTES;  // 6; 5 with 16 warps or a residual
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + OTHER_BYTES;
    static constexpr int THREADS = 128 + 32 * EW;
    // barriers: full, empty [STAGES], tfull, tempty [2], drain, residual [2 per warp]; two words
    static_assert((2 * STAGES + 5 + 2 * EW + 1) * 8 <= BAR_BYTES, "barriers");
    // registers per thread: at launch, of warps 0..3 and of the epilogue warps
    static constexpr int LAUNCH_REGS = EW == 8 ? 168 : 96;
    static constexpr int REGS_LOW = EW == 8 ? 40 : 24;
    static constexpr int REGS_HIGH = EW == 8 ? 232 : 112;
    static_assert(128 * REGS_LOW + 32 * EW * REGS_HIGH <= THREADS * LAUNCH_REGS,
                  "register split exceeds the launch allocation");
};

template <int REGS>
__device__ __forceinline__ void setmaxnreg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REGS) : "memory");
}
template <int REGS>
__device__ __forceinline__ void setmaxnreg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(REGS) : "memory");
}

template <bool OUT_F32, bool RES, int EW>
__global__ void __launch_bounds__(GemmI8PairCfg<RES, EW>::THREADS, 1)
    gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                        const __grid_constant__ CUtensorMap tm_wp, const __grid_constant__ CUtensorMap tm_y,
                        const __grid_constant__ CUtensorMap tm_r, const GemmI8Params p) {
    using C = GemmI8PairCfg<RES, EW>;
    constexpr int BN = C::BN;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw;
    if (smem_u32(smem) & 1023) {  // the swizzled tiles need it; uniform over the cluster
        if (threadIdx.x == 0) atomicCAS(p.err, 0, 121);
        return;
    }
    uint8_t* slot_base = smem + C::STAGES * C::STAGE_BYTES;
    float* col_base = reinterpret_cast<float*>(slot_base + EW * C::SLOTS * C::SLOT_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(col_base) + C::COL_BYTES);
    uint64_t* full_bar = bars;
    uint64_t* empty_bar = bars + C::STAGES;
    uint64_t* tfull_bar = bars + 2 * C::STAGES;
    uint64_t* tempty_bar = tfull_bar + 2;
    uint64_t* drain_bar = tfull_bar + 4;
    uint64_t* res_bar = tfull_bar + 5;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_bar + 2 * EW);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // uniform
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
            mbar_init(&tempty_bar[b], 2 * EW);
        }
        mbar_init(drain_bar, 1);
        for (int b = 0; b < 2 * EW; ++b) mbar_init(&res_bar[b], 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&tm_x);
        prefetch_tmap(&tm_w);
        if (p.pieces) prefetch_tmap(&tm_wp);
        if (p.vec_out) prefetch_tmap(&tm_y);
        if (RES && p.vec_res) prefetch_tmap(&tm_r);
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
        setmaxnreg_dec<C::REGS_LOW>();
        if (warp == 0) {
            // -------------------------------------------------------- producer
            const uint32_t elected = elect_one();
            const uint32_t ring = smem_u32(smem), full0 = smem_u32(full_bar);
            const uint32_t leader_full0 = mapa_shared(full0, 0);
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
                    ok = __all_sync(0xffffffffu, wait_bar(&empty_bar[stage], phase ^ 1, abort_flag, p.err, 131));
                    if (!ok) break;
                    const uint32_t sa = ring + stage * C::STAGE_BYTES;
                    // both CTAs' bytes complete on the leader's barrier
                    if (rank == 0) mbar_arrive_expect_tx_elected(elected, full0 + 8 * stage, 2 * bytes);
                    tma_load_2d_pair_elected(elected, sa, &tm_x, leader_full0 + 8 * stage, kb * C::BK, m0);
                    tma_load_2d_pair_elected(elected, sa + C::A_BYTES, tw, leader_full0 + 8 * stage, kb * C::BK, n0);
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
        } else if (warp == 1 && rank == 0) {
            // -------------------------------------------------------- MMA issuer
            const uint32_t elected = elect_one();
            const uint64_t a_desc0 = umma_desc_sw128_kmajor(smem_u32(smem));
            const uint64_t b_desc0 = umma_desc_sw128_kmajor(smem_u32(smem) + C::A_BYTES);
            const uint32_t empty0 = smem_u32(empty_bar), tfull0 = smem_u32(tfull_bar);
            int stage = 0;
            uint32_t phase = 0;
            int acc = 0;
            uint32_t acc_phase = 0;
            bool ok = true;
            auto sched = schedule();
            WorkItem w;
            while (ok && sched.next(w)) {
                ok = __all_sync(0xffffffffu, wait_bar<true>(&tempty_bar[acc], acc_phase ^ 1, abort_flag, p.err, 231));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
                const uint32_t idesc = umma_idesc_i8(256, w.width);
                for (int kb = 0; kb < num_k; ++kb) {
                    ok = __all_sync(0xffffffffu, wait_bar(&full_bar[stage], phase, abort_flag, p.err, 232));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t at = static_cast<uint64_t>(stage * (C::STAGE_BYTES >> 4));
#pragma unroll
                    for (int kk = 0; kk < C::BK / 32; ++kk)
                        umma_i8_pair_elected(elected, d_tmem, a_desc0 + at + 2 * kk, b_desc0 + at + 2 * kk, idesc,
                                             kb + kk != 0);
                    umma_commit_both_elected(elected, empty0 + 8 * stage);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                umma_commit_both_elected(elected, tfull0 + 8 * acc);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
            // no MMA still writes TMEM when it is freed
            if (elected) umma_commit_pair(smem_u32(drain_bar));
            __syncwarp();
            volatile int no_abort = 0;
            wait_bar(drain_bar, 0, &no_abort, p.err, 233);
        }
    } else {
        setmaxnreg_inc<C::REGS_HIGH>();
        // ------------------------------------------------------------ epilogue
        constexpr int ESZ = OUT_F32 ? 4 : 2;
        constexpr int CW = 128 / ESZ;  // output columns of a step
        constexpr int PER = 16 / ESZ;  // values of a 16-byte granule
        constexpr int GC = C::GROUP_COLS;
        using Out = typename std::conditional<OUT_F32, float, __half>::type;
        const int q = warp & 3;
        const int ew = warp - 4;
        const int group = ew >> 2;
        uint8_t* slots = slot_base + ew * C::SLOTS * C::SLOT_BYTES;
        float* s_ws = col_base + group * 2 * GC;  // [GC] scales, then [GC] biases
        float* s_b = s_ws + GC;
        const int my_col = threadIdx.x & 127;  // the column that this thread stages, if below GC
        float ws, bias, xs;                    // of the next tile
        auto load_columns = [&](const WorkItem& w) {
            const int c = (w.tile % num_n) * BN + w.n_off + group * GC + my_col;
            const int64_t row = static_cast<int64_t>(w.tile / num_n) * 256 + static_cast<int64_t>(rank) * C::BM + 32 * q + lane;
            const bool live = my_col < GC && c < p.n;
            ws = live ? __ldg(p.w_scale + c) : 0.0f;
            bias = 0.0f;
            if (p.bias != nullptr && live)
                bias = p.bias_f32 ? __ldg(static_cast<const float*>(p.bias) + c)
                                  : __half2float(static_cast<const __half*>(p.bias)[c]);
            xs = row < p.m ? __ldg(p.x_scale + row) : 0.0f;
        };
        int acc = 0;
        uint32_t acc_phase = 0;
        uint32_t j = 0;      // running step counter of this warp (slot = j & 1 with a residual)
        uint32_t loads = 0;  // residual steps requested (lane 0)
        bool ok = true;  // after a wait that gave up: only the warps' named barriers are kept up
        auto load_residual = [&](int s, int col0, int64_t row0) {
            mbar_arrive_expect_tx(&res_bar[2 * ew + s], C::SLOT_BYTES);
            tma_load_2d(slots + s * C::SLOT_BYTES, &tm_r, &res_bar[2 * ew + s], col0, static_cast<int32_t>(row0));
            ++loads;
        };
        const uint32_t tempty_leader0 = mapa_shared(smem_u32(&tempty_bar[0]), 0);
        const uint32_t tempty_leader1 = mapa_shared(smem_u32(&tempty_bar[1]), 0);
        auto sched = schedule();
        WorkItem w, next;
        bool more = sched.next(w);
        if (more) load_columns(w);
        while (more) {
            const int64_t row0 = static_cast<int64_t>(w.tile / num_n) * 256 + static_cast<int64_t>(rank) * C::BM + 32 * q;
            const int c_begin = (w.tile % num_n) * BN + w.n_off + group * GC;
            const int valid = min(min(GC, w.width - group * GC), p.n - c_begin);  // <= 0: past a piece or past n
            const int nsteps = (valid > 0 && row0 < p.m) ? (valid + CW - 1) / CW : 0;
            const int rows_live = static_cast<int>(p.m - row0 < 32 ? p.m - row0 : 32);
            if constexpr (RES) {
                // the first residual step lands while the main loop runs
                if (ok && p.vec_res && lane == 0 && nsteps > 0) {
                    bulk_wait_group_read<0>();
                    load_residual(j & 1, c_begin, row0);
                }
            }
            named_bar_sync(1 + group, 128);  // the four warps are done with the previous tile's columns
            if (my_col < GC) {
                s_ws[my_col] = ws;
                s_b[my_col] = bias;
            }
            const uint64_t xs2 = f2_pack(xs, xs);
            named_bar_sync(1 + group, 128);
            more = sched.next(next);
            if (more) load_columns(next);
            const uint32_t t_row = tmem_base + (static_cast<uint32_t>(32 * q) << 16) +
                                   static_cast<uint32_t>(acc * BN + group * GC);
            // residual rows that TMA cannot load: a step ahead in registers, 32 rows in flight
            Out rv[RES ? 32 : 1][CW / 32];
            auto fetch_residual = [&](int c) {
                const Out* src = static_cast<const Out*>(p.residual) + row0 * p.ldr + c_begin + c * CW + lane;
#pragma unroll
                for (int r = 0; r < (RES ? 32 : 1); ++r)
#pragma unroll
                    for (int cc = 0; cc < CW / 32; ++cc)
                        if (r < rows_live && c_begin + c * CW + 32 * cc + lane < p.n) rv[r][cc] = src[r * p.ldr + 32 * cc];
            };
            if constexpr (RES) {
                if (!p.vec_res && nsteps > 0) fetch_residual(0);
            }
            if (ok) ok = __all_sync(0xffffffffu, wait_bar(&tfull_bar[acc], acc_phase, abort_flag, p.err, 331));
            if (!ok) {
                w = next;
                continue;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < nsteps; ++c, ++j) {
                const int col0 = c_begin + c * CW;
                const int cols = min(CW, p.n - col0);
                const uint32_t slot = RES ? (j & 1) : 0;
                uint8_t* buf = slots + slot * C::SLOT_BYTES;
                // granule g of row r lives at g ^ (r & 7): the TMA maps' 128-byte swizzle
                auto granule = [&](int r, int g) { return reinterpret_cast<uint4*>(buf + r * 128 + ((g ^ (r & 7)) << 4)); };
                auto value = [&](int r, int c) { return reinterpret_cast<Out*>(granule(r, c / PER)) + c % PER; };
                if constexpr (RES) {
                    if (p.vec_res) {
                        // the next step's residual, once that slot's last store has been read out
                        if (lane == 0 && c + 1 < nsteps) {
                            bulk_wait_group_read<0>();
                            load_residual((j + 1) & 1, col0 + CW, row0);
                        }
                    } else {
                        if (lane == 0) bulk_wait_group_read<0>();
                        __syncwarp();
#pragma unroll
                        for (int r = 0; r < 32; ++r)
#pragma unroll
                            for (int cc = 0; cc < CW / 32; ++cc) *value(r, 32 * cc + lane) = rv[r][cc];
                        if (c + 1 < nsteps) fetch_residual(c + 1);
                        __syncwarp();
                    }
                } else {
                    // single slot: the previous step has left it
                    if (lane == 0) bulk_wait_group_read<0>();
                    __syncwarp();
                }
                // a few columns at a time (with sixteen warps 16: 32 left the GELU's constants no
                // registers); a thread reads and writes its own row of the slot only
                constexpr int CB = EW == 16 ? 16 : 32;
#pragma unroll
                for (int h = 0; h < CW / CB; ++h) {
                    uint32_t r[CB];
                    if constexpr (CB == 32)
                        tmem_ld_32x32b_x32(t_row + c * CW + CB * h, r);
                    else
                        tmem_ld_32x32b_x16(t_row + c * CW + CB * h, r);
                    tmem_ld_wait(r);
                    if (c + 1 == nsteps && h + 1 == CW / CB) {
                        // this warp has read its part of the accumulator into registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster_relaxed(acc ? tempty_leader1 : tempty_leader0);
                    }
                    float v[CB];
#pragma unroll
                    for (int g = 0; g < CB / 4; ++g) {
                        const float4 sw = *reinterpret_cast<const float4*>(s_ws + c * CW + CB * h + 4 * g);
                        const float4 sb = *reinterpret_cast<const float4*>(s_b + c * CW + CB * h + 4 * g);
                        const uint64_t a0 = f2_pack(__int2float_rn(static_cast<int>(r[4 * g])),
                                                    __int2float_rn(static_cast<int>(r[4 * g + 1])));
                        const uint64_t a1 = f2_pack(__int2float_rn(static_cast<int>(r[4 * g + 2])),
                                                    __int2float_rn(static_cast<int>(r[4 * g + 3])));
                        f2_unpack(f2_fma(f2_mul(a0, f2_pack(sw.x, sw.y)), xs2, f2_pack(sb.x, sb.y)), v[4 * g],
                                  v[4 * g + 1]);
                        f2_unpack(f2_fma(f2_mul(a1, f2_pack(sw.z, sw.w)), xs2, f2_pack(sb.z, sb.w)), v[4 * g + 2],
                                  v[4 * g + 3]);
                    }
                    if (p.activation == kActGelu) {
#pragma unroll
                        for (int e = 0; e < CB; e += 2) gelu_log_pair(v[e], v[e + 1]);
                    }
                    if constexpr (RES) {
                        if (h == 0 && p.vec_res) {
                            ok = __all_sync(0xffffffffu,
                                            wait_bar(&res_bar[2 * ew + slot], (j >> 1) & 1, abort_flag, p.err, 332));
                            if (!ok) break;
                        }
                    }
#pragma unroll
                    for (int g = 0; g < CB / PER; ++g) {
                        uint4* at = granule(lane, h * (CB / PER) + g);
                        float* e = v + PER * g;
                        if constexpr (RES) {
                            const uint4 a = *at;
                            if constexpr (OUT_F32) {
                                e[0] += __uint_as_float(a.x);
                                e[1] += __uint_as_float(a.y);
                                e[2] += __uint_as_float(a.z);
                                e[3] += __uint_as_float(a.w);
                            } else {
                                const __half2* rh = reinterpret_cast<const __half2*>(&a);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float2 f = __half22float2(rh[i]);
                                    e[2 * i] += f.x;
                                    e[2 * i + 1] += f.y;
                                }
                            }
                        }
                        if constexpr (OUT_F32) {
                            *at = make_uint4(__float_as_uint(e[0]), __float_as_uint(e[1]), __float_as_uint(e[2]),
                                             __float_as_uint(e[3]));
                        } else {
                            const __half2 h0 = __floats2half2_rn(e[0], e[1]), h1 = __floats2half2_rn(e[2], e[3]);
                            const __half2 h2 = __floats2half2_rn(e[4], e[5]), h3 = __floats2half2_rn(e[6], e[7]);
                            *at = make_uint4(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1),
                                             *reinterpret_cast<const uint32_t*>(&h2), *reinterpret_cast<const uint32_t*>(&h3));
                        }
                    }
                }
                if (!ok) break;
                if (p.vec_out) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tm_y, buf, col0, static_cast<int32_t>(row0));
                        bulk_commit_group();
                    }
                } else {
                    __syncwarp();
                    Out* dst = static_cast<Out*>(p.y) + row0 * p.ldy + col0;
                    for (int r = 0; r < rows_live; r += 8) {
                        Out t[8][CW / 32];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int cc = 0; cc < CW / 32; ++cc) t[i][cc] = *value(r + i, 32 * cc + lane);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int cc = 0; cc < CW / 32; ++cc)
                                if (r + i < rows_live && 32 * cc + lane < cols)
                                    dst[(r + i) * p.ldy + 32 * cc + lane] = t[i][cc];
                    }
                    __syncwarp();
                    // the next residual may reach this slot by TMA: order these reads before it
                    if (RES && p.vec_res) fence_proxy_async_smem();
                }
            }
            if (ok && nsteps == 0) {  // nothing to read: release the accumulator all the same
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(acc ? tempty_leader1 : tempty_leader0);
            }
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1;
            }
            w = next;
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
