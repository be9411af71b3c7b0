// Rows to e4m3 with one fp32 scale per 128 columns: s = max(amax / 448, 2^-80), q = e4m3(x / s), where s and the quotient
// are rounded to 32 bits (as a division does) and the quotient to the nearest e4m3 value, halves to even.
//
// 448 is e4m3's largest value, so nothing saturates (the quotient of the largest element is 448 or its neighbour, which
// rounds to 448). The floor keeps every step of the division exact in 32 bits; a block below 448 * 2^-80 loses precision
// down to 0. An infinite or NaN element makes its block's scale infinite or NaN, and with it the row of a product.
#pragma once
#include "exl3_common.cuh"

namespace exl3 {

constexpr float kE4m3Max = 448.0f;
constexpr float kFp8MinScale = 0x1p-80f;

// |x| as an integer: ordered as the magnitudes are, NaN above infinity, so that the largest is the block's amax
__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

__device__ __forceinline__ float fp8_scale(uint32_t amax_bits) {
    const float s = __builtin_bit_cast(float, amax_bits) / kE4m3Max;
    return s < kFp8MinScale ? kFp8MinScale : s;
}

// x / s for the elements of one block, correctly rounded: with inv the rounded 1 / s, q0 = x inv is within one unit of the
// quotient, x - q0 s is exact in a multiply-add, and adding its share to q0 rounds once. (|x| >= 2^-10 s: below that both
// give values that round to 0.) An infinite or NaN scale leaves q0: 0 for finite x, NaN else.
struct Fp8Div {
    float s, inv;
    __device__ __forceinline__ explicit Fp8Div(float scale) {
        inv = 1.0f / scale;
        s = abs_bits(scale) < 0x7F800000u ? scale : 0.0f;
    }
    __device__ __forceinline__ float operator()(float x) const {
        const float q = x * inv;
        return __builtin_fmaf(__builtin_fmaf(-q, s, x), inv, q);
    }
};

// four values as e4m3, the first in the low byte
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// silu(g) * u = g u / (1 + exp(-g)). exp(-g) = 2^t (1 + e ln 2) with t = -g log2(e) rounded and e what that lost, to the
// product's rounding and to log2(e)'s own (1.3e-8 of t: 9 units of 2^-24 at g = -40), on the hardware's exp2 and
// reciprocal: within 8 units of 2^-24. g = +-inf has no e.
constexpr float kLn2 = 0.693147180559945309f;
struct ExpMinus {
    float t, e;
    __device__ __forceinline__ explicit ExpMinus(float g) {
        constexpr float kLog2e = 1.44269504088896341f, kLog2eRest = 1.92596299e-8f;
        t = -g * kLog2e;
        e = abs_bits(t) < 0x7F800000u ? __builtin_fmaf(-g, kLog2eRest, __builtin_fmaf(-g, kLog2e, -t)) : 0.0f;
    }
};
__device__ __forceinline__ float silu_times(float g, float u) {
    const ExpMinus x(g);
    const float p = __builtin_amdgcn_exp2f(x.t);
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_fmaf(p, x.e * kLn2, p)) * u;
}

// The same of gates below kSiluFar, for which exp(-g) may be beyond fp32 (from -88.8 down): the 1 beside it is less than 2^-57 of
// it, so the value is g u exp(g), with exp(g) in two halves, 2^(-t / 2) (1 - e ln 2) 2^(-t / 2), so that it is lost only where the
// product is too. g = -inf gives NaN, as 0 times it is.
constexpr float kSiluFar = -40.0f;
__device__ __forceinline__ float silu_times_far(float g, float u) {
    const ExpMinus x(g);
    const float h = __builtin_amdgcn_exp2f(-0.5f * x.t);
    return g * h * u * __builtin_fmaf(h, -x.e * kLn2, h);
}

// 8 consecutive elements of a row as fp32. WIDE: 16-byte aligned and all inside the row; else one by one, from the `n`-th on
// (n > 0) the last one again
template <int DT, bool WIDE>
__device__ __forceinline__ void load8(const void* x, size_t at, int n, float (&v)[8]) {
    if constexpr (WIDE) {
        if constexpr (DT == 2) {
            const float4* p = (const float4*)((const float*)x + at);
            const float4 a = p[0], b = p[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 r = *(const uint4*)((const uint16_t*)x + at);
            const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DT == 0) {
                    const half2_t h = __builtin_bit_cast(half2_t, u[j]);
                    v[2 * j] = (float)h[0];
                    v[2 * j + 1] = (float)h[1];
                } else {
                    v[2 * j] = __builtin_bit_cast(float, u[j] << 16);
                    v[2 * j + 1] = __builtin_bit_cast(float, u[j] & 0xFFFF0000u);
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const size_t i = at + min(j, n - 1);
            if constexpr (DT == 0) v[j] = (float)((const _Float16*)x)[i];
            else if constexpr (DT == 1) v[j] = __builtin_bit_cast(float, (uint32_t)((const uint16_t*)x)[i] << 16);
            else v[j] = ((const float*)x)[i];
        }
    }
}

// the largest over the 16 lanes of a DPP row, in every one of them (row_ror 8, 4, 2, 1)
template <int CTRL>
__device__ __forceinline__ uint32_t ror_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    return ror_max<0x121>(ror_max<0x122>(ror_max<0x124>(ror_max<0x128>(v))));
}

// 8 of a block's 128 values before they are quantised: those of x at `at`, or silu(x[at]) x[at + k]; `n` of them (any
// number, also negative) lie inside the row, the others are 0. In two steps, for callers that load several blocks before they need
// the first: what is in memory (u: only for silu), and the values out of it, in v
template <int DT, bool SILU, bool WIDE>
__device__ __forceinline__ void block_load(const void* x, size_t at, int k, int n, float (&v)[8], float (&u)[8]) {
    // (no branches: the rows' first elements are loaded for none)
    at = n > 0 ? at : 0;
    const int some = max(n, 1);
    load8<DT, WIDE>(x, at, some, v);
    if constexpr (SILU) load8<DT, WIDE>(x, at + k, some, u);
}
template <bool SILU, bool WIDE>
__device__ __forceinline__ void block_values(int n, float (&v)[8], const float (&u)[8]) {
    if constexpr (SILU) {
        float g[8], least = v[0];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[j] = v[j];
            least = __builtin_fminf(least, g[j]);
            v[j] = silu_times(g[j], u[j]);
        }
        if (least < kSiluFar)                        // (rare, so a branch)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = g[j] < kSiluFar ? silu_times_far(g[j], u[j]) : v[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (WIDE ? 0 : j) < n ? v[j] : 0.0f;
}

// the 8 values' e4m3 and the scale of the block that the 16 lanes of a DPP row hold
__device__ __forceinline__ uint2 quant_block(const float (&v)[8], float& s) {
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, abs_bits(v[j]));
    s = fp8_scale(row16_max(amax));
    const Fp8Div d(s);
    return {pack_e4m3(d(v[0]), d(v[1]), d(v[2]), d(v[3])), pack_e4m3(d(v[4]), d(v[5]), d(v[6]), d(v[7]))};
}

}  // namespace exl3
