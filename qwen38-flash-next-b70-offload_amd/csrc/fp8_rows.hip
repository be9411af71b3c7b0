// Quantised rows of the 8-bit float linear (fp8_rows.cuh), of x or of silu(gate) * up of fused gate|up rows.
//
// 16 lanes hold a block of 128 columns, 8 elements each (16 bytes of bf16 in, 8 bytes out), so the block's amax is four DPP
// steps and each element is read once. One pass over the data: bound by memory. us per call out of a graph: 8,192 x 2,048 bf16
// 10.9 (4.7 TB/s; a large copy 5.2), gate|up 8,192 x 2 x 512 6.2 (3.4 TB/s); 301 x 1,000 fp16 2.4, any launch's.
#include "exl3_kernels.h"
#include "fp8_rows.cuh"

namespace exl3 {
namespace {

constexpr int kRowsThreads = 256;                    // 16 blocks of 128 columns

// (Fp8RowsGrid; the column chunks of a row are next to each other)
template <int DT, bool SILU, bool WIDE>
__global__ void __launch_bounds__(kRowsThreads) fp8_rows_kernel(Fp8RowsArgs A, int kb, int shift, int chunks) {
    const int t = threadIdx.x >> 4, i = threadIdx.x & 15;
    const int64_t row = (int64_t)(blockIdx.x / chunks) * (16 >> shift) + (t >> shift);
    const int b = (blockIdx.x % chunks << shift) + (t & ((1 << shift) - 1));
    if (row >= A.M || b >= kb) return;               // (whole rows of 16 lanes)
    const int c = b * kFp8Block + i * 8;
    float v[8], u[8], s;
    block_load<DT, SILU, WIDE>(A.x, (size_t)row * A.x_stride + c, A.k, A.k - c, v, u);
    block_values<SILU, WIDE>(A.k - c, v, u);
    *(uint2*)(A.q + ((size_t)row * kb + b) * kFp8Block + i * 8) = quant_block(v, s);
    if (i == 0) A.s[(size_t)row * kb + b] = s;
}

template <bool SILU, bool WIDE>
void launch_rows(const Fp8RowsArgs& a, int x_dt, hipStream_t st) {
    const int kb = fp8_blocks(a.k);
    const auto [shift, chunks, workgroups] = fp8_rows_grid(a.M, a.k);
    const dim3 grid((unsigned)workgroups);
    if (x_dt == 0) hipLaunchKernelGGL((fp8_rows_kernel<0, SILU, WIDE>), grid, kRowsThreads, 0, st, a, kb, shift, chunks);
    else if (x_dt == 1) hipLaunchKernelGGL((fp8_rows_kernel<1, SILU, WIDE>), grid, kRowsThreads, 0, st, a, kb, shift, chunks);
    else hipLaunchKernelGGL((fp8_rows_kernel<2, SILU, WIDE>), grid, kRowsThreads, 0, st, a, kb, shift, chunks);
}

}  // namespace

hipError_t launch_fp8_rows(const Fp8RowsArgs& a, int x_dt, bool silu, hipStream_t st) {
    const bool wide = fp8_rows_wide(a.x, a.x_stride, a.k, x_dt);
    if (silu) wide ? launch_rows<true, true>(a, x_dt, st) : launch_rows<true, false>(a, x_dt, st);
    else wide ? launch_rows<false, true>(a, x_dt, st) : launch_rows<false, false>(a, x_dt, st);
    return hipGetLastError();
}

}  // namespace exl3
