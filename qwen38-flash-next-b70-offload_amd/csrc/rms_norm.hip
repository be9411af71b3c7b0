// The residual's addition and the root-mean-square norm: held = x + residual in the residual's type (fp32 sum, one rounding),
// y = h / sqrt(mean(h^2) + eps) * w of what is held (x itself without a residual). y leaves as rows of x's type, as e4m3 rows with
// fp32 scales (fp8_rows.cuh's form) or as 4-bit rows (fp4_rows.cuh).
//
// The sum and everything behind it are computed in 64 bits and rounded to 32 once, rows of 16 bits from there (for e4m3 only its
// scale and its quotient are): an error of 2^-24 takes one of 10^6 values over a border between two of e4m3's. It costs 2 us of
// 27 at 8,192 x 2,048 to e4m3.
//
// A row is held in registers between its sum and its outputs: T lanes, up to C times 8 elements each, so every input is read once
// and every output written once. 16 lanes hold 128 neighbouring columns, which is a block of e4m3 and four of the 4-bit ones.
// Rows of more than 32,768 columns are read again for their outputs (they were just read: from the caches). Those of 8,193 to
// 32,768 fill the 128 registers that 1,024 threads have and spill 1 to 8 more (8 to 36 bytes a lane), and a CU has one workgroup,
// with nothing under way beside its sum's barrier: 2,000 x 20,000 at 62 % of a large copy's rate.
//
// Bound by memory, few rows by a launch and one chain of loads. us per call out of a graph, bf16 with a bf16 residual: 1 x 2,048 to
// e4m3 2.6, 8,192 x 2,048 to bf16 24.0 (134 MB, 5.6 TB/s), to e4m3 27.2 (117 MB, 4.3 TB/s), to e2m1 23.3; 8,192 x 4,096 to bf16
// 44.5; 1,500 x 16 heads of 128 4.9. Rows of any size, with nothing but their elements aligned: 3,962 x 2,883 fp16 with an fp32
// residual to e4m3 35.4 (126 MB; 75 with elements one by one and their places held in registers), 2,000 x 8,192 28.5 (115 MB), x
// 8,191 34.4, x 20,000 89, x 20,001 96 (239 and 461 where the registers did not hold the weights and places too).
#include "exl3_kernels.h"
#include "fp4_rows.cuh"

#include <type_traits>

namespace exl3 {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ double lane_xor64(double v, int m) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __float_as_uint(lane_xor(__uint_as_float((uint32_t)u), m));
    const uint32_t hi = __float_as_uint(lane_xor(__uint_as_float((uint32_t)(u >> 32)), m));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// the sum over the T threads of a row, in each of them
template <int T>
__device__ __forceinline__ double row_sum(double v) {
#pragma unroll
    for (int m = 1; m < (T < 64 ? T : 64); m <<= 1) v += lane_xor64(v, m);
    if constexpr (T > 64) {
        __shared__ double part[T / 64];
        if (lane_id() == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int i = 1; i < T / 64; ++i) v += part[i];
    }
    return v;
}

// 1 / sqrt(a) for a > 0, to 2^-44: the hardware's 2^-23 and a step of Newton's; 0 for infinity
__device__ __forceinline__ double root_inverse(double a) {
    const double y = __builtin_amdgcn_rsq(a), e = __builtin_fma(-a * y, y, 1.0);
    return a > 1.7e308 ? 0.0 : __builtin_fma(0.5 * y, e, y);
}

// a block of 128 values, 8 to each of 16 lanes, as quant_block has it, without a rounding before the scale's and the quotient's
__device__ __forceinline__ uint2 quant_block64(const double (&t)[8], float& s) {
    double top = 0;
    uint32_t bits = 0;                               // (a maximum passes over NaN)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        top = __builtin_fmax(top, __builtin_fabs(t[j]));
        bits = max(bits, abs_bits((float)t[j]));
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) top = __builtin_fmax(top, lane_xor64(top, m));
    bits = row16_max(bits);
    s = (float)(top * (1.0 / kE4m3Max));
    s = s < kFp8MinScale ? kFp8MinScale : s;
    const double inv0 = (double)__builtin_amdgcn_rcpf(s), inv = __builtin_fma(__builtin_fma(-(double)s, inv0, 1.0), inv0, inv0);
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = (float)(t[j] * inv);
    if (bits >= 0x7F800000u) {                       // (rare, so a branch)
        s = fp8_scale(bits);
        const Fp8Div d(s);
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = d((float)t[j]);
    }
    return {pack_e4m3(q[0], q[1], q[2], q[3]), pack_e4m3(q[4], q[5], q[6], q[7])};
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
    // (weights that are held in 32 bits get their 1 here: 1 + w has more bits than they)
    __device__ __forceinline__ double gain(double w) const { return w; }
    __device__ __forceinline__ double gain(float w) const { return (double)w + A.unit_offset; }
    // w: the weights of these columns
    template <class W>
    __device__ __forceinline__ void out(int c, float (&v)[8], double by, const W (&w)[8]) const {
        const int n = A.k - c;
        double t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = (WIDE ? 0 : j) < n ? (double)v[j] * by * gain(w[j]) : 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
        if (A.y && n > 0) store8<DT, WIDE>(A.y, (size_t)m * A.k + c, n, v);
        if (A.form == kFormFp8) {
            const int kb = fp8_blocks(A.k), b = c / kFp8Block;
            float s;
            const uint2 q = quant_block64(t, s);
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

template <bool WIDE, class W>
__device__ __forceinline__ void weights(const RmsNormArgs& A, int c, W (&w)[8]) {
    const int n = A.k - c;
    float f[8] = {1, 1, 1, 1, 1, 1, 1, 1};
    if (A.w) load8<2, WIDE>(A.w, n > 0 ? c : 0, max(n, 1), f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        w[j] = f[j];
        if constexpr (sizeof(W) == 8) w[j] += A.unit_offset;
    }
}

template <int DT, int RDT, bool WIDE, int T, int C>
__global__ void __launch_bounds__(T < kThreads ? kThreads : T) rms_norm_kernel(RmsNormArgs A) {
    constexpr int kRows = T < kThreads ? kThreads / T : 1;
    // (4-bit rows have whole stages of scales)
    const int i = threadIdx.x % T, ks = A.form == kFormFp4 ? fp4_stages(A.k) * kFp4Stage : fp4_cols(A.k);
    if constexpr (C > 0) {
        // (weights of one or two chunks stay in the 64 bits that they are used in; those of four would not fit beside the row)
        constexpr bool kKept = C <= 2;
        std::conditional_t<kKept, double, float> w[kKept ? C : 1][8];
        if constexpr (kKept)
#pragma unroll
            for (int c = 0; c < C; ++c) weights<WIDE>(A, (c * T + i) * 8, w[c]);
        // (whole rows of T threads; the same number of turns for all threads of a row)
        for (int64_t m = (int64_t)blockIdx.x * kRows + threadIdx.x / T; m < A.M; m += (int64_t)gridDim.x * kRows) {
            const Row<DT, RDT, WIDE> row(A, m);
            // (kept from being taken out of the loop over the rows: the elements' places, which would fill the registers)
            int at = i * 8;
            if constexpr (!WIDE || !kKept) asm volatile("" : "+v"(at));
            double sum = 0;
            float v[C][8];
#pragma unroll
            for (int c = 0; c < C; ++c) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = 0;
                if (c == 0 || c * T * 8 < ks) row.load(c * T * 8 + at, v[c]);
            }
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum = __builtin_fma((double)v[c][j], (double)v[c][j], sum);
            const double by = root_inverse(row_sum<T>(sum) * A.inv_k + (double)A.eps);
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (c == 0 || c * T * 8 < ks) {
                    if constexpr (!kKept) {
                        __builtin_amdgcn_sched_barrier(0);           // (a chunk at a time)
                        weights<WIDE>(A, c * T * 8 + at, w[0]);
                    }
                    row.out(c * T * 8 + at, v[c], by, w[kKept ? c : 0]);
                }
            if constexpr (T > 64) __syncthreads();   // (the sum's LDS is used again)
        }
    } else {
        const int64_t m = blockIdx.x;
        const Row<DT, RDT, WIDE> row(A, m);
        double sum = 0;
        float v[8], w[8];
        for (int c = 0; c < ks; c += T * 8) {
            row.load(c + i * 8, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = __builtin_fma((double)v[j], (double)v[j], sum);
        }
        const double by = root_inverse(row_sum<T>(sum) * A.inv_k + (double)A.eps);
        for (int c = 0; c < ks; c += T * 8) {
            row.again(c + i * 8, v);
            weights<WIDE>(A, c + i * 8, w);
            row.out(c + i * 8, v, by, w);
        }
    }
}

template <int DT, int RDT, bool WIDE, int T, int C>
void launch_rows(const RmsNormArgs& a, hipStream_t st) {
    constexpr int kRows = T < kThreads ? kThreads / T : 1;
    // (8 workgroups per CU, each with every 2,048th row: as many as are there at a time, and the weights are loaded once; 8,192 x
    // 2,048 bf16 to bf16 23.9 us, a workgroup for every row 26.1)
    const int64_t all = (int64_t)(a.M - 1) / kRows + 1, most = C > 0 ? kCus * 8 : all;
    hipLaunchKernelGGL((rms_norm_kernel<DT, RDT, WIDE, T, C>), dim3((unsigned)(all < most ? all : most)),
                       dim3(T < kThreads ? kThreads : T), 0, st, a);
}

template <int DT, int RDT, bool WIDE>
void launch_norm(const RmsNormArgs& a, hipStream_t st) {
    const int t = rms_norm_threads(a.M, a.k);
    if (t == 16 && a.k <= 128 && a.form != kFormFp4) launch_rows<DT, RDT, WIDE, 16, 1>(a, st);
    else if (t == 16) launch_rows<DT, RDT, WIDE, 16, 2>(a, st);
    else if (t == 64) launch_rows<DT, RDT, WIDE, 64, 2>(a, st);
    else if (t == 256 && a.k <= 2048) launch_rows<DT, RDT, WIDE, 256, 1>(a, st);
    else if (t == 256 && a.k <= 4096) launch_rows<DT, RDT, WIDE, 256, 2>(a, st);
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
