// The residual's addition and the root-mean-square norm: held = x + residual in the residual's type (fp32 sum, one rounding),
// y = h / sqrt(mean(h^2) + eps) * w of what is held (x itself without a residual), in fp32. y leaves as rows of x's type, as
// e4m3 rows with fp32 scales (fp8_rows.cuh) or as 4-bit rows (fp4_rows.cuh), the last two from its fp32 values.
//
// A row is held in registers between its sum and its outputs: T lanes, up to C times 8 elements each, so every input is
// read once and every output written once. 16 lanes hold 128 neighbouring columns, which is a block of e4m3 and four of the
// 4-bit ones. Rows of more than 32,768 columns are read again for their outputs (they were just read: from the caches).
#include "exl3_kernels.h"
#include "fp4_rows.cuh"

namespace exl3 {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float row16_sum(float v) {
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) v += lane_xor(v, m);
    return v;
}

// the sum over the T threads of a row, in each of them
template <int T>
__device__ __forceinline__ float row_sum(float v) {
    if constexpr (T == 16) return row16_sum(v);
    v = wave_sum(v);
    if constexpr (T > 64) {
        __shared__ float part[T / 64];
        if (lane_id() == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = row16_sum((lane_id() & 15) < T / 64 ? part[lane_id() & 15] : 0.0f);
    }
    return v;
}

template <int DT, int RDT, bool WIDE>
struct Row {
    const RmsNormArgs& A;
    int64_t m;
    size_t x0, r0;
    __device__ __forceinline__ Row(const RmsNormArgs& a, int64_t row) : A(a), m(row) {
        x0 = A.inner == 1 ? (size_t)m * A.x_outer : (size_t)(m / A.inner) * A.x_outer + (size_t)(m % A.inner) * A.x_stride;
        r0 = (size_t)m * A.res_stride;
    }
    // 8 elements from column c on, zeros behind the row; the held sum is written
    __device__ __forceinline__ void load(int c, float (&v)[8]) const {
        const int n = A.k - c, some = max(n, 1);
        const size_t at = n > 0 ? c : 0;
        load8<DT, WIDE>(A.x, x0 + at, some, v);
        if constexpr (RDT >= 0) {
            float r[8];
            load8<RDT, WIDE>(A.res, r0 + at, some, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] += r[j];
                if constexpr (RDT == 0) v[j] = (float)(_Float16)v[j];
                if constexpr (RDT == 1) v[j] = (float)(__bf16)v[j];
            }
            if (n > 0) store8<RDT, WIDE>(A.held, (size_t)m * A.k + c, n, v);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (WIDE ? 0 : j) < n ? v[j] : 0.0f;
    }
    // the same again, of what is held
    __device__ __forceinline__ void again(int c, float (&v)[8]) const {
        const int n = A.k - c, some = max(n, 1);
        const size_t at = n > 0 ? c : 0;
        if constexpr (RDT >= 0) load8<RDT, WIDE>(A.held, (size_t)m * A.k + at, some, v);
        else load8<DT, WIDE>(A.x, x0 + at, some, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (WIDE ? 0 : j) < n ? v[j] : 0.0f;
    }
    __device__ __forceinline__ void out(int c, float (&v)[8], float by) const {
        const int n = A.k - c;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= by;
        if (A.w) {
            float w[8];
            load8<2, WIDE>(A.w, n > 0 ? c : 0, max(n, 1), w);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= w[j];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (WIDE ? 0 : j) < n ? v[j] : 0.0f;       // (an infinite weight's 0 times it)
        }
        if (A.y && n > 0) store8<DT, WIDE>(A.y, (size_t)m * A.k + c, n, v);
        if (A.form == kFormFp8) {
            const int kb = fp8_blocks(A.k), b = c / kFp8Block;
            float s;
            const uint2 q = quant_block(v, s);
            if (b >= kb) return;
            *(uint2*)(A.q + ((size_t)m * kb) * kFp8Block + c) = q;
            if (lane_id() % 16 == 0) ((float*)A.s)[(size_t)m * kb + b] = s;
        } else if (A.form == kFormFp4) {
            const int kp = fp4_cols(A.k);
            uint32_t s;
            const uint32_t q = quant4_block(v, n, s);
            if (c < kp) *(uint32_t*)(A.q + (size_t)m * (kp / 2) + c / 2) = q;
            if (lane_id() % 16 == 0 && c < fp4_stages(A.k) * kFp4Stage)
                *(uint32_t*)((uint8_t*)A.s + (size_t)(c / kFp4Stage) * A.s_stage + (size_t)m * 8 + (c / 128 & 1) * 4) = s;
        }
    }
};

template <int DT, int RDT, bool WIDE, int T, int C>
__global__ void __launch_bounds__(T < kThreads ? kThreads : T) rms_norm_kernel(RmsNormArgs A) {
    constexpr int kRows = T < kThreads ? kThreads / T : 1;
    const int64_t m = (int64_t)blockIdx.x * kRows + threadIdx.x / T;
    if (m >= A.M) return;                            // (whole rows of T threads)
    const int i = threadIdx.x % T, ks = (A.k + kFp4Stage - 1) / kFp4Stage * kFp4Stage;
    const Row<DT, RDT, WIDE> row(A, m);
    float sum = 0;
    if constexpr (C > 0) {
        float v[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[c][j] = 0;
            if (c == 0 || c * T * 8 < ks) row.load((c * T + i) * 8, v[c]);
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(v[c][j], v[c][j], sum);
        const float by = 1.0f / __builtin_sqrtf(row_sum<T>(sum) / (float)A.k + A.eps);
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (c == 0 || c * T * 8 < ks) row.out((c * T + i) * 8, v[c], by);
    } else {
        float v[8];
        for (int c = 0; c < ks; c += T * 8) {
            row.load(c + i * 8, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(v[j], v[j], sum);
        }
        const float by = 1.0f / __builtin_sqrtf(row_sum<T>(sum) / (float)A.k + A.eps);
        for (int c = 0; c < ks; c += T * 8) {
            row.again(c + i * 8, v);
            row.out(c + i * 8, v, by);
        }
    }
}

template <int DT, int RDT, bool WIDE, int T, int C>
void launch_rows(const RmsNormArgs& a, hipStream_t st) {
    constexpr int kRows = T < kThreads ? kThreads / T : 1;
    hipLaunchKernelGGL((rms_norm_kernel<DT, RDT, WIDE, T, C>), dim3((unsigned)((a.M - 1) / kRows + 1)),
                       dim3(T < kThreads ? kThreads : T), 0, st, a);
}

template <int DT, int RDT, bool WIDE>
void launch_norm(const RmsNormArgs& a, hipStream_t st) {
    const int t = rms_norm_threads(a.k);
    if (t == 16) launch_rows<DT, RDT, WIDE, 16, 2>(a, st);
    else if (t == 64) launch_rows<DT, RDT, WIDE, 64, 4>(a, st);
    else if (t == 256) launch_rows<DT, RDT, WIDE, 256, 4>(a, st);
    else if (a.k <= 32768) launch_rows<DT, RDT, WIDE, 1024, 4>(a, st);
    else launch_rows<DT, RDT, WIDE, 1024, 0>(a, st);
}

template <int DT, int RDT>
void launch_norm(const RmsNormArgs& a, hipStream_t st) {
    auto on16 = [](const void* p) { return (uintptr_t)p % 16 == 0; };
    const int size = DT == 2 ? 4 : 2, rsize = RDT == 2 ? 4 : 2;
    const bool wide = a.k % 8 == 0 && on16(a.x) && a.x_stride * size % 16 == 0 && a.x_outer * size % 16 == 0 && on16(a.w) &&
                      on16(a.y) && (RDT < 0 || (on16(a.res) && on16(a.held) && a.res_stride * rsize % 16 == 0));
    wide ? launch_norm<DT, RDT, true>(a, st) : launch_norm<DT, RDT, false>(a, st);
}

}  // namespace

hipError_t launch_rms_norm(const RmsNormArgs& a, int x_dt, int res_dt, hipStream_t st) {
    if (!a.res) x_dt == 0 ? launch_norm<0, -1>(a, st) : x_dt == 1 ? launch_norm<1, -1>(a, st) : launch_norm<2, -1>(a, st);
    else if (x_dt == 2) launch_norm<2, 2>(a, st);
    else if (x_dt == 0) res_dt == 0 ? launch_norm<0, 0>(a, st) : launch_norm<0, 2>(a, st);
    else res_dt == 1 ? launch_norm<1, 1>(a, st) : launch_norm<1, 2>(a, st);
    return hipGetLastError();
}

}  // namespace exl3
