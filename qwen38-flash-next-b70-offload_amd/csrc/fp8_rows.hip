// Quantised rows of the 8-bit float linear (fp8_rows.cuh), of x or of silu(gate) * up of fused gate|up rows.
//
// 16 lanes hold a block of 128 columns, 8 elements each (16 bytes of bf16 in, 8 bytes out), so the block's amax is four DPP
// steps and each element is read once. One pass over the data: bound by memory.
#include "exl3_kernels.h"
#include "fp8_rows.cuh"

namespace exl3 {
namespace {

constexpr int kRowsThreads = 256;                    // 16 blocks of 128 columns

// the largest over the 16 lanes of a DPP row, in every one of them (row_ror 8, 4, 2, 1)
template <int CTRL>
__device__ __forceinline__ uint32_t ror_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    return ror_max<0x121>(ror_max<0x122>(ror_max<0x124>(ror_max<0x128>(v))));
}

// A workgroup covers 16 >> shift rows of 1 << shift blocks each, the column chunks of a row next to each other
template <int DT, bool SILU, bool WIDE>
__global__ void __launch_bounds__(kRowsThreads) fp8_rows_kernel(Fp8RowsArgs A, int kb, int shift, int chunks) {
    const int t = threadIdx.x >> 4, i = threadIdx.x & 15;
    const int64_t row = (int64_t)(blockIdx.x / chunks) * (16 >> shift) + (t >> shift);
    const int b = (blockIdx.x % chunks << shift) + (t & ((1 << shift) - 1));
    if (row >= A.M || b >= kb) return;               // (whole rows of 16 lanes)
    const int c = b * kFp8Block + i * 8, n = min(8, A.k - c);
    const size_t at = (size_t)row * A.x_stride + c;
    float v[8];
    if (n <= 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    } else {
        load8<DT, WIDE>(A.x, at, n, v);
        if constexpr (SILU) {
            float u[8];
            load8<DT, WIDE>(A.x, at + A.k, n, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = silu_times(v[j], u[j]);
        }
    }
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, abs_bits(v[j]));
    const float s = fp8_scale(row16_max(amax));
    const Fp8Div d(s);
    const uint2 o = {pack_e4m3(d(v[0]), d(v[1]), d(v[2]), d(v[3])), pack_e4m3(d(v[4]), d(v[5]), d(v[6]), d(v[7]))};
    *(uint2*)(A.q + ((size_t)row * kb + b) * kFp8Block + i * 8) = o;
    if (i == 0) A.s[(size_t)row * kb + b] = s;
}

template <bool SILU, bool WIDE>
void launch_rows(const Fp8RowsArgs& a, int x_dt, hipStream_t st) {
    const int kb = fp8_blocks(a.k);
    int shift = 0;
    while (shift < 4 && (1 << shift) < kb) ++shift;
    const int chunks = (kb + (1 << shift) - 1) >> shift, rows = 16 >> shift;
    const dim3 grid((unsigned)((int64_t)((a.M - 1) / rows + 1) * chunks));
    if (x_dt == 0) hipLaunchKernelGGL((fp8_rows_kernel<0, SILU, WIDE>), grid, kRowsThreads, 0, st, a, kb, shift, chunks);
    else if (x_dt == 1) hipLaunchKernelGGL((fp8_rows_kernel<1, SILU, WIDE>), grid, kRowsThreads, 0, st, a, kb, shift, chunks);
    else hipLaunchKernelGGL((fp8_rows_kernel<2, SILU, WIDE>), grid, kRowsThreads, 0, st, a, kb, shift, chunks);
}

}  // namespace

hipError_t launch_fp8_rows(const Fp8RowsArgs& a, int x_dt, bool silu, hipStream_t st) {
    // 16-byte loads where every row starts on 16 bytes and no group of 8 elements crosses the row's end
    const int esz = x_dt == 2 ? 4 : 2;
    const bool wide = (uintptr_t)a.x % 16 == 0 && a.x_stride * esz % 16 == 0 && a.k % 8 == 0;
    if (silu) wide ? launch_rows<true, true>(a, x_dt, st) : launch_rows<true, false>(a, x_dt, st);
    else wide ? launch_rows<false, true>(a, x_dt, st) : launch_rows<false, false>(a, x_dt, st);
    return hipGetLastError();
}

}  // namespace exl3
