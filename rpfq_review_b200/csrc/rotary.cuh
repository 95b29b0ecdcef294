// Rotary positions. Pair j of a head's first 2 P values is turned by the angle
// pos * inv_freq[j]:
//
//   y_a = c (a cos - b sin),   y_b = c (b cos + a sin)      c: magnitude
//
// with the pair at (j, j + P) (half layout) or (2 j, 2 j + 1) (interleaved); the
// transposed map, which is the gradient, turns by the negative angle. With two
// axes the first P / 2 pairs use a token's first position and the rest its
// second. The values past 2 P are copied (left alone in place).
//
// Angles are products in fp64 (a position past 2^24 / (2 pi) has no usable angle
// in fp32), reduced by 2 pi in two fp64 steps; the remainder r goes to fp32 as
// hi + lo, and sin / cos are taken of hi and corrected to first order in lo, so
// they are good to fp32 rounding (past angles of 2^28 to the product's 2^-53 of them).
//
// Bound by memory: every value is read and written once. A block takes a tile of
// tokens: its cos / sin pairs go to shared memory once and serve all of its heads.
// A thread then owns one pair of 16-byte vectors of a token's heads (both ends of
// its pairs in the half layout), keeps their cos / sin in registers and walks the
// heads: no index arithmetic per value, and neighbouring lanes hold neighbouring
// pieces, then neighbouring heads. The loads run several
// heads ahead as asynchronous copies into a ring in shared memory, of which each
// thread reads only what it has copied itself; the first of them run while the cos /
// sin pairs are made. (Held in registers instead, enough of them to cover the
// latency of DRAM left too few threads: 256 x 197 tokens of 32 fp16 heads of 64 took
// 74 us, and take 65 us here, 413 MB at the rate of a plain copy; 66 us in place on
// qkv rows.) In vectors of 8 bytes (24 heads of 96, 36 pairs) the same tokens take 82 us
// in the half and 91 us in the interleaved layout for 72 us of copying. Value by value (an
// odd number of pairs in the half layout, odd strides or addresses) nothing runs ahead:
// 260 to 270 us for the 64 us of 32 heads of 64.
#pragma once

#include "ptx.cuh"

namespace rpfq {

enum : int { kPosI32 = 0, kPosI64 = 1, kPosF32 = 2, kPosF64 = 3 };

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTable = 2048;  // (cos, sin) entries of a block: 16 KB
constexpr int kRotaryTokens = 64;   // tokens of a block at most
constexpr int kRotaryDepth = 4;     // heads of a thread on their way: 32 KB a block, four blocks an SM

struct RotaryParams {
    const void* x;
    void* y;
    int64_t xb, xl, xh;       // strides of x in elements: sequence, token, head
    int64_t yb, yl, yh;
    const void* positions;    // [length, axes], or [batch, length, axes] with pos_b != 0
    int64_t pos_b;            // positions between sequences (0: shared)
    const double* inv_freq;   // [pairs]
    int64_t tokens;           // batch * length
    int32_t length;
    int32_t heads, dim, pairs, axes;
    int32_t pos_type;
    int32_t copy_rest;        // out of place: the values past 2 * pairs are copied
    int32_t token_tile;       // tokens of a block
    int32_t head_step;        // threads of a token that share a piece: heads h, h + head_step, ...
    float magnitude;          // scales cos and sin
    float sign;               // -1: the transposed map
};

__device__ __forceinline__ double load_position(const void* p, int type, int64_t i) {
    switch (type) {
        case kPosI32: return static_cast<double>(static_cast<const int32_t*>(p)[i]);
        case kPosI64: return static_cast<double>(static_cast<const int64_t*>(p)[i]);
        case kPosF32: return static_cast<double>(static_cast<const float*>(p)[i]);
        default: return static_cast<const double*>(p)[i];
    }
}

// cos and sin of an fp64 angle to fp32 accuracy.
__device__ __forceinline__ float2 cos_sin(double angle) {
    const double n = rint(angle * 0.15915494309189533577);  // 1 / (2 pi)
    double r = fma(-n, 6.283185307179586232, angle);        // 2 pi, head
    r = fma(-n, 2.449293598294706414e-16, r);               // 2 pi, tail
    const float hi = static_cast<float>(r);
    const float lo = static_cast<float>(r - static_cast<double>(hi));
    float s, c;
    sincosf(hi, &s, &c);
    return make_float2(fmaf(-s, lo, c), fmaf(c, lo, s));
}

template <typename T, int VEC, int ALIGN>
struct alignas(ALIGN) RotaryVec {
    T v[VEC];
};

__device__ __forceinline__ float rot_f32(float v) { return v; }
__device__ __forceinline__ float rot_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void rot_store(float& d, float v) { d = v; }
__device__ __forceinline__ void rot_store(__half& d, float v) { d = __float2half_rn(v); }

// How a head is cut. BYTES > 0: vectors of BYTES; the host picks 16 or 8 where that
// divides every run of values (P in the half layout, 2 P interleaved, the rest),
// every stride and both addresses. BYTES = 0: value by value. A piece is two
// vectors: c and c + P / VEC in the half layout, c and c + half of the vectors
// interleaved (neighbours value by value: a pair) and past the turned part, so that
// neighbouring lanes always copy neighbouring vectors. The last may be alone.
template <typename T, int BYTES, bool INTERLEAVED>
struct RotaryPieces {
    static constexpr int VEC = BYTES ? BYTES / static_cast<int>(sizeof(T)) : 1;
    __host__ __device__ static int turned(int pairs) {
        return INTERLEAVED ? (2 * pairs / VEC + 1) / 2 : pairs / VEC;
    }
    __host__ __device__ static int all(int dim, int pairs, bool copy_rest) {
        return turned(pairs) + (copy_rest ? ((dim - 2 * pairs) / VEC + 1) / 2 : 0);
    }
};

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t smem, const void* src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem), "l"(src) : "memory");
}

template <typename T, int BYTES, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads, 4) rotary_kernel(const RotaryParams p) {
    using S = RotaryPieces<T, BYTES, INTERLEAVED>;
    constexpr int VEC = S::VEC;
    using V = RotaryVec<T, VEC, BYTES ? BYTES : static_cast<int>(sizeof(T))>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    V* ring = reinterpret_cast<V*>(smem_raw);  // [kRotaryDepth][2][threads] (BYTES > 0)
    float2* table = reinterpret_cast<float2*>(smem_raw + kRotaryDepth * 2 * kRotaryThreads * BYTES);  // [tokens][pairs]
    const int tok0 = static_cast<int>(static_cast<int64_t>(blockIdx.x) * p.token_tile);  // tokens < 2^31
    const int ntok = static_cast<int>(p.tokens - tok0 < p.token_tile ? p.tokens - tok0 : p.token_tile);
    const int P = p.pairs;
    const int turned = S::turned(P);
    const int pieces = S::all(p.dim, P, p.copy_rest != 0);
    const int span = pieces < kRotaryThreads ? pieces : kRotaryThreads;  // pieces of a head at once
    const int team = span * p.head_step;                                 // threads of a token
    const int slot = threadIdx.x / team, in_team = threadIdx.x - slot * team;
    const int first_head = in_team / span, first_piece = in_team - first_head * span;
    const int slots = kRotaryThreads / team;
    const int heads = (p.heads - first_head + p.head_step - 1) / p.head_step;  // of this thread
    const int64_t x_step = p.head_step * p.xh, y_step = p.head_step * p.yh;
    pdl_wait();
    pdl_launch_dependents();

    // the two vectors of piece c: their places in the head, and whether there is a second
    int c = first_piece, at0, at1;
    bool two, turn;
    auto place = [&]() {
        turn = c < turned;
        if (turn && !INTERLEAVED) {
            at0 = c * VEC;
            at1 = P + c * VEC;
            two = true;
        } else if (turn && VEC == 1) {
            at0 = 2 * c;
            at1 = 2 * c + 1;
            two = true;
        } else {
            const int i = turn ? c : c - turned;
            const int from = turn ? 0 : 2 * P, to = turn ? 2 * P : p.dim;
            at0 = from + i * VEC;
            at1 = at0 + (turn ? turned : pieces - turned) * VEC;
            two = at1 < to;
        }
    };
    // the loads: head next_h of token next_t into ring entry next_d
    int next_t = slots, next_h = 0, next_d = 0;
    const T* next_x = nullptr;
    auto start = [&](int t) {
        next_t = t;
        next_h = 0;
        if (t >= ntok) return;
        const int tok = tok0 + t, b = tok / p.length, l = tok - b * p.length;
        next_x = static_cast<const T*>(p.x) + b * p.xb + l * p.xl + first_head * p.xh;
    };
    auto request = [&]() {
        if constexpr (BYTES > 0) {
            if (next_t < ntok) {
                copy_async<BYTES>(smem_u32(ring + 2 * next_d * kRotaryThreads + threadIdx.x), next_x + at0);
                if (two) copy_async<BYTES>(smem_u32(ring + (2 * next_d + 1) * kRotaryThreads + threadIdx.x), next_x + at1);
                next_x += x_step;
                if (++next_h == heads) start(next_t + slots);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (++next_d == kRotaryDepth) next_d = 0;
        }
    };
    const bool mine = slot < slots && slot < ntok;
    if (mine) {
        place();
        start(slot);
#pragma unroll
        for (int d = 0; d < kRotaryDepth; ++d) request();
    }
    const int per_axis = P / p.axes;
    for (int i = threadIdx.x; i < ntok * P; i += kRotaryThreads) {
        const int t = i / P, j = i - t * P;
        const int tok = tok0 + t, b = tok / p.length, l = tok - b * p.length;
        const double pos = load_position(p.positions, p.pos_type, b * p.pos_b + static_cast<int64_t>(l) * p.axes + j / per_axis);
        const float2 cs = cos_sin(pos * p.inv_freq[j]);
        table[i] = make_float2(cs.x * p.magnitude, cs.y * p.magnitude * p.sign);
    }
    __syncthreads();
    if (!mine) return;
    int d = 0;
    for (;;) {
        for (int t = slot; t < ntok; t += slots) {
            // half layout: cos and sin of VEC pairs; interleaved: of VEC / 2 of either vector
            float cs[VEC], sn[VEC];
            if (turn) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    int j = c * VEC + e;
                    if (INTERLEAVED && VEC > 1) j = (e < VEC / 2 ? at0 : at1 - VEC) / 2 + e;
                    const float2 v = table[t * P + (j < P ? j : P - 1)];
                    cs[e] = v.x;
                    sn[e] = v.y;
                }
            }
            const int tok = tok0 + t, b = tok / p.length, l = tok - b * p.length;
            T* y = static_cast<T*>(p.y) + b * p.yb + l * p.yl + first_head * p.yh;
            for (int h = 0; h < heads; ++h, y += y_step) {
                V lo, hi;
                if constexpr (BYTES > 0) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kRotaryDepth - 1) : "memory");
                    lo = ring[2 * d * kRotaryThreads + threadIdx.x];
                    if (two) hi = ring[(2 * d + 1) * kRotaryThreads + threadIdx.x];
                    if (++d == kRotaryDepth) d = 0;
                } else {
                    const T* x = static_cast<const T*>(p.x) + b * p.xb + l * p.xl + first_head * p.xh + h * x_step;
                    lo = *reinterpret_cast<const V*>(x + at0);
                    if (two) hi = *reinterpret_cast<const V*>(x + at1);
                }
                if (turn) {
                    if constexpr (!INTERLEAVED || VEC == 1) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float v0 = rot_f32(lo.v[e]), v1 = rot_f32(hi.v[e]);
                            rot_store(lo.v[e], v0 * cs[e] - v1 * sn[e]);
                            rot_store(hi.v[e], v1 * cs[e] + v0 * sn[e]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < VEC / 2; ++e) {
                            float v0 = rot_f32(lo.v[2 * e]), v1 = rot_f32(lo.v[2 * e + 1]);
                            rot_store(lo.v[2 * e], v0 * cs[e] - v1 * sn[e]);
                            rot_store(lo.v[2 * e + 1], v1 * cs[e] + v0 * sn[e]);
                            v0 = rot_f32(hi.v[2 * e]), v1 = rot_f32(hi.v[2 * e + 1]);
                            rot_store(hi.v[2 * e], v0 * cs[VEC / 2 + e] - v1 * sn[VEC / 2 + e]);
                            rot_store(hi.v[2 * e + 1], v1 * cs[VEC / 2 + e] + v0 * sn[VEC / 2 + e]);
                        }
                    }
                }
                *reinterpret_cast<V*>(y + at0) = lo;
                if (two) *reinterpret_cast<V*>(y + at1) = hi;
                request();  // into the entry just read: its values have been used
            }
        }
        // heads of more pieces than threads
        c += span;
        if (c >= pieces) break;
        place();
        start(slot);
        if constexpr (BYTES > 0) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            d = next_d = 0;
        }
#pragma unroll
        for (int i = 0; i < kRotaryDepth; ++i) request();
    }
}

}  // namespace rpfq
