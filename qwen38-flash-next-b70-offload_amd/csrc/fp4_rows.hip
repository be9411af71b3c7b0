// Rows to 4-bit floats (fp4_rows.cuh), of x or of silu(gate) * up of fused gate|up rows, and back.
//
// 32 lanes hold a stage of 256 columns of a row, 8 elements each: a block of 32 is four lanes, its amax two DPP steps, and each
// element is read once. A workgroup's 8 rows are neighbours, so that their scales are one 64-byte piece. Bound by memory. us per
// call out of a graph: 8,192 x 2,048 bf16 10.4 (42 MB, 4.1 TB/s; a large copy 5.2; two or four groups of rows to a workgroup 10.4
// and 9.8, but 2,000 rows 4.1 and 4.5 for 3.9; 16-bit pairs never unpacked 10.3), back to bf16 8.4 (11.4 with codes decoded by
// shifts), 301 x 1,000 fp16 2.2, any launch's. silu(gate) * up of gate|up rows: 8,192 x 512 bf16 5.9 (19 MB), 8,192 x 2,048 18.9
// (76 MB, 4.0 TB/s), 8,192 x 2,047 23.4, 64 x 512 2.2.
#include "exl3_kernels.h"
#include "fp4_rows.cuh"

namespace exl3 {
namespace {

constexpr int kRowsThreads = 256;                    // 8 rows, 32 lanes each

template <int DT, bool SILU, bool WIDE>
__global__ void __launch_bounds__(kRowsThreads) fp4_rows_kernel(Fp4RowsArgs A, int kb) {
    const int i = threadIdx.x & 31, b = blockIdx.x % kb;
    const int64_t row = (int64_t)(blockIdx.x / kb) * 8 + (threadIdx.x >> 5);
    if (row >= A.M) return;                          // (whole rows of 32 lanes)
    const int c = b * kFp4Stage + i * 8, kp = fp4_cols(A.k);
    float v[8], u[8];
    block_load<DT, SILU, WIDE>(A.x, (size_t)row * A.x_stride + c, A.k, A.k - c, v, u);
    block_values<SILU, WIDE>(A.k - c, v, u);
    uint32_t scales;
    const uint32_t codes = quant4_block(v, A.k - c, scales);
    if (c < kp) *(uint32_t*)(A.q + (size_t)row * (kp / 2) + c / 2) = codes;
    if (i % 16 == 0) *(uint32_t*)(A.s + (size_t)b * A.s_stage + (size_t)row * 8 + i / 4) = scales;
}

template <bool SILU, bool WIDE>
void launch_rows(const Fp4RowsArgs& a, int x_dt, hipStream_t st) {
    const int kb = fp4_stages(a.k);
    const dim3 grid((unsigned)(((int64_t)a.M + 7) / 8 * kb));
    if (x_dt == 0) hipLaunchKernelGGL((fp4_rows_kernel<0, SILU, WIDE>), grid, kRowsThreads, 0, st, a, kb);
    else if (x_dt == 1) hipLaunchKernelGGL((fp4_rows_kernel<1, SILU, WIDE>), grid, kRowsThreads, 0, st, a, kb);
    else hipLaunchKernelGGL((fp4_rows_kernel<2, SILU, WIDE>), grid, kRowsThreads, 0, st, a, kb);
}

// 8 codes to their values; a quotient times its scale is rounded to the output's type once
template <int DT, bool WIDE>
__global__ void __launch_bounds__(kRowsThreads) fp4_dequant_kernel(Fp4DequantArgs A, int kb) {
    const int i = threadIdx.x & 31, b = blockIdx.x % kb;
    const int64_t row = (int64_t)(blockIdx.x / kb) * 8 + (threadIdx.x >> 5);
    const int c = b * kFp4Stage + i * 8, n = A.k - c;
    if (row >= A.M || n <= 0) return;
    const uint32_t u = *(const uint32_t*)(A.q + (size_t)row * (fp4_cols(A.k) / 2) + c / 2);
    const uint32_t byte = A.s[(size_t)b * A.s_stage + (size_t)row * 8 + i / 4];
    // (2^-127, byte 0, is below fp32's normal values)
    const float s = __builtin_bit_cast(float, byte == 255u ? 0x7FC00000u : byte ? byte << 23 : 1u << 22);
    const auto v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 1);
    const auto v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 3);
    const float v[8] = {v0[0] * s, v0[1] * s, v1[0] * s, v1[1] * s, v2[0] * s, v2[1] * s, v3[0] * s, v3[1] * s};
    store8<DT, WIDE>(A.out, (size_t)row * A.k + c, n, v);
}

template <bool WIDE>
void launch_dequant(const Fp4DequantArgs& a, int dt, hipStream_t st) {
    const int kb = fp4_stages(a.k);
    const dim3 grid((unsigned)(((int64_t)a.M + 7) / 8 * kb));
    if (dt == 0) hipLaunchKernelGGL((fp4_dequant_kernel<0, WIDE>), grid, kRowsThreads, 0, st, a, kb);
    else if (dt == 1) hipLaunchKernelGGL((fp4_dequant_kernel<1, WIDE>), grid, kRowsThreads, 0, st, a, kb);
    else hipLaunchKernelGGL((fp4_dequant_kernel<2, WIDE>), grid, kRowsThreads, 0, st, a, kb);
}

}  // namespace

hipError_t launch_fp4_rows(const Fp4RowsArgs& a, int x_dt, bool silu, hipStream_t st) {
    const bool wide = fp8_rows_wide(a.x, a.x_stride, a.k, x_dt);
    if (silu) wide ? launch_rows<true, true>(a, x_dt, st) : launch_rows<true, false>(a, x_dt, st);
    else wide ? launch_rows<false, true>(a, x_dt, st) : launch_rows<false, false>(a, x_dt, st);
    return hipGetLastError();
}

hipError_t launch_fp4_dequant(const Fp4DequantArgs& a, int dt, hipStream_t st) {
    fp8_rows_wide(a.out, a.k, a.k, dt) ? launch_dequant<true>(a, dt, st) : launch_dequant<false>(a, dt, st);
    return hipGetLastError();
}

}  // namespace exl3
