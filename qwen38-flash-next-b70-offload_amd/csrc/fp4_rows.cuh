// Rows of microscaled 4-bit floats: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte with the first
// in the low half, and one power of two per 32 columns, held as exponent + 127 in 8 bits.
//
// The scale is 2^(floor(log2(amax)) - 2), so that the block's largest magnitude lies in [4, 8) of e2m1's 6, and 2^-126 at the
// least (a block of zeros has it). Dividing by it is exact; a quotient is rounded to the nearest code, halves to even, and
// one above 6 is 6: at most a quarter of a magnitude in (7, 8) is lost, which the next larger scale would lose in the small values.
// An infinite or NaN element makes its block's scale 255, a NaN, and with it the row of a product.
//
// Layout: codes [M, kp / 2] with kp = k rounded up to 128 and zeros behind k; scales by stages of 256 columns, 8 bytes to a
// row, [ceil(k / 256)][M][8], and 0 behind k: the rows that a product's tile needs for one stage are next to each other.
#pragma once
#include "fp8_rows.cuh"

namespace exl3 {

__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax_bits) {
    return amax_bits >= 0x7F800000u ? 255u : max(amax_bits >> 23, 3u) - 2u;
}

// the largest over 4 neighbouring lanes, in each of them (quad_perm [1,0,3,2], then [2,3,0,1])
__device__ __forceinline__ uint32_t quad_max(uint32_t v) { return ror_max<0x4E>(ror_max<0xB1>(v)); }

// 8 values as codes, the first in the low half of the low byte, divided by the scale of byte b (a NaN block's as they come)
__device__ __forceinline__ uint32_t pack_e2m1(const float (&v)[8], uint32_t b) {
    const float s = __builtin_bit_cast(float, b == 255u ? 127u << 23 : b << 23);
    uint32_t u = 0;
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[0], v[1], s, 0);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[2], v[3], s, 1);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[4], v[5], s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[6], v[7], s, 3);
}

// 16 lanes of a DPP row hold 128 columns, 8 to a lane: the lane's codes, and in `scales` the four blocks' scale bytes (in every
// lane), those of blocks that start behind the row (`n`: its columns from the lane's first on) 0
__device__ __forceinline__ uint32_t quant4_block(const float (&v)[8], int n, uint32_t& scales) {
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, abs_bits(v[j]));
    const uint32_t b = fp4_scale_byte(quad_max(amax));
    const int lane = lane_id() & 15;
    uint32_t all = n + (lane & 3) * 8 > 0 ? b << 8 * (lane >> 2) : 0;
    all |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)all, 0x124, 0xF, 0xF, false);       // row_ror 4, then 8
    scales = all | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)all, 0x128, 0xF, 0xF, false);
    return pack_e2m1(v, b);
}

}  // namespace exl3
