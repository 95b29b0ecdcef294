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
// they are good to fp32 rounding.
//
// Bound by memory: every value is read and written once. A block takes a tile of
// tokens: its cos / sin pairs go to shared memory once and serve all of its heads.
#pragma once

#include "ptx.cuh"

namespace rpfq {

enum : int { kPosI32 = 0, kPosI64 = 1, kPosF32 = 2, kPosF64 = 3 };

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTable = 2048;  // (cos, sin) entries of a block: 16 KB

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
    int32_t token_tile, head_tile;
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

// BYTES > 0: loads and stores of BYTES; the host picks 16 or 8 where that divides
// every run of values (P in the half layout, 2 P interleaved, the rest), every
// stride and both addresses. BYTES = 0: value by value.
template <typename T, int BYTES, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p) {
    __shared__ float2 table[kRotaryTable];
    const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * p.token_tile;
    const int ntok = static_cast<int>(p.tokens - tok0 < p.token_tile ? p.tokens - tok0 : p.token_tile);
    const int head0 = static_cast<int>(blockIdx.y) * p.head_tile;
    const int nheads = p.heads - head0 < p.head_tile ? p.heads - head0 : p.head_tile;
    const int P = p.pairs;
    pdl_wait();
    pdl_launch_dependents();
    const int per_axis = P / p.axes;
    for (int i = threadIdx.x; i < ntok * P; i += kRotaryThreads) {
        const int t = i / P, j = i - t * P;
        const int64_t tok = tok0 + t;
        const int64_t b = tok / p.length, l = tok - b * p.length;
        const double pos = load_position(p.positions, p.pos_type, b * p.pos_b + l * p.axes + j / per_axis);
        const float2 cs = cos_sin(pos * p.inv_freq[j]);
        table[i] = make_float2(cs.x * p.magnitude, cs.y * p.magnitude * p.sign);
    }
    __syncthreads();
    constexpr int VEC = BYTES ? BYTES / static_cast<int>(sizeof(T)) : (INTERLEAVED ? 2 : 1);
    constexpr int REST = BYTES ? VEC : 1;
    using V = RotaryVec<T, VEC, BYTES ? BYTES : static_cast<int>(sizeof(T))>;
    using R = RotaryVec<T, REST, BYTES ? BYTES : static_cast<int>(sizeof(T))>;
    const int turned = INTERLEAVED ? 2 * P / VEC : P / VEC;  // items of a head that rotate
    const int per_head = turned + (p.copy_rest ? (p.dim - 2 * P) / REST : 0);
    const int per_token = per_head * nheads;
    for (int i = threadIdx.x; i < ntok * per_token; i += kRotaryThreads) {
        const int t = i / per_token, u = i - t * per_token;
        const int h = u / per_head, c = u - h * per_head;
        const int64_t tok = tok0 + t;
        const int64_t b = tok / p.length, l = tok - b * p.length;
        const T* x = static_cast<const T*>(p.x) + b * p.xb + l * p.xl + (head0 + h) * p.xh;
        T* y = static_cast<T*>(p.y) + b * p.yb + l * p.yl + (head0 + h) * p.yh;
        if (c >= turned) {  // past the rotated part
            const int at = 2 * P + (c - turned) * REST;
            *reinterpret_cast<R*>(y + at) = *reinterpret_cast<const R*>(x + at);
            continue;
        }
        if constexpr (INTERLEAVED) {
            const V in = *reinterpret_cast<const V*>(x + c * VEC);
            const float2* cs = table + t * P + c * (VEC / 2);
            V out;
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) {
                const float a0 = rot_f32(in.v[2 * e]), a1 = rot_f32(in.v[2 * e + 1]);
                rot_store(out.v[2 * e], a0 * cs[e].x - a1 * cs[e].y);
                rot_store(out.v[2 * e + 1], a1 * cs[e].x + a0 * cs[e].y);
            }
            *reinterpret_cast<V*>(y + c * VEC) = out;
        } else {
            const V lo = *reinterpret_cast<const V*>(x + c * VEC);
            const V hi = *reinterpret_cast<const V*>(x + P + c * VEC);
            const float2* cs = table + t * P + c * VEC;
            V out_lo, out_hi;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float a0 = rot_f32(lo.v[e]), a1 = rot_f32(hi.v[e]);
                rot_store(out_lo.v[e], a0 * cs[e].x - a1 * cs[e].y);
                rot_store(out_hi.v[e], a1 * cs[e].x + a0 * cs[e].y);
            }
            *reinterpret_cast<V*>(y + c * VEC) = out_lo;
            *reinterpret_cast<V*>(y + P + c * VEC) = out_hi;
        }
    }
}

}  // namespace rpfq
