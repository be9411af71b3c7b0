// The 4-bit float product of few rows (fp4_tiles.cuh has the definition): 16 to 48 columns to a workgroup, whose waves share the
// stages of 256 columns of k among them, so that no two waves need the same operands: they go from memory straight to registers,
// and a wave's loads are all under way at once. The waves' sums join in LDS, in the waves' order.
//
// A lane's 16 bytes of an MFMA (16 x 16 x 128) are one block of 32 of one row, and its scale is one byte. Rows that are not
// quantised yet (x, or the gates and ups of a gated MLP) are quantised by each wave for its own stages, in LDS: about 0.3 us a
// row for each round of workgroups, against 2.2 for a launch of its own.
//
// What bounds it: the weights' way from HBM and one chain of loads, MFMAs and the join. us per call out of a graph, weights from
// HBM: 1 quantised row 2048 -> 12,288 5.5 (13.4 MB, 4.2 TB/s without the 2.3 of any launch), 4096 -> 2048 4.2, 512 -> 2048 2.3;
// 1 row quantised inside 6.5, 4.7, 2.6 (with a launch before it 7.6, 6.4, 4.4); 40 rows 4096 -> 2048 5.5.
#include "fp4_tiles.cuh"

namespace exl3 {
namespace {

enum { kRowsQuantised, kRowsX, kRowsSilu };

// The scales of a lane's two blocks of a stage (columns 128 j + 32 g) out of its row's eight, byte j for step j. Only one of them
// where the stage is half a one: the other's, 2^-127 for both operands, takes whatever was loaded to 0
__device__ __forceinline__ int two_scales(uint2 row, int g, bool half) {
    return (int)__builtin_amdgcn_perm(row.y, row.x, (uint32_t)(g | (g + 4) << 8)) & (half ? 0xFF : 0xFFFF);
}

template <int J>
__device__ __forceinline__ v4f fp4_mfma16(v4i w, v4i q, v4f acc, int sw, int sq) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(w), fp4_operand(q), acc, 4, 4, J, sw, J, sq);
}

// 4 elements of a row from column c on, zeros behind its k columns (no branches: the row's first or last one is loaded for those)
template <int DT, bool WIDE>
__device__ __forceinline__ v4f load4(const void* x, size_t row, int c, int k) {
    v4f v;
    if constexpr (WIDE) {
        const size_t at = row + (c < k ? c : 0);
        if constexpr (DT == 2) v = *(const v4f*)((const float*)x + at);
        else {
            const uint2 u = *(const uint2*)((const uint16_t*)x + at);
            const uint32_t p[4] = {u.x << 16, u.x & 0xFFFF0000u, u.y << 16, u.y & 0xFFFF0000u};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = DT == 0 ? (float)__builtin_bit_cast(_Float16, (uint16_t)(p[j] >> 16)) : __builtin_bit_cast(float, p[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const size_t at = row + min(c + j, k - 1);
            if constexpr (DT == 2) v[j] = ((const float*)x)[at];
            else if constexpr (DT == 1) v[j] = __builtin_bit_cast(float, (uint32_t)((const uint16_t*)x)[at] << 16);
            else v[j] = (float)((const _Float16*)x)[at];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c + (WIDE ? 0 : j) < k ? v[j] : 0.0f;
    return v;
}

// 4 rows of a wave's stage: lane i has columns 4 i, 8 lanes a block. Codes q[m * 128], scales s[m * 8]
__device__ __forceinline__ void quant_four(const v4f (&v)[4], int m0, int M, uint8_t* q, uint8_t* s) {
    const int l = lane_id();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if (m0 + u >= M) break;
        uint32_t amax = max(max(abs_bits(v[u][0]), abs_bits(v[u][1])), max(abs_bits(v[u][2]), abs_bits(v[u][3])));
        amax = ror_max<0x141>(quad_max(amax));       // (row_half_mirror: the other four of eight)
        const uint32_t b = fp4_scale_byte(amax);
        const float by = __builtin_bit_cast(float, b == 255u ? 127u << 23 : b << 23);
        uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[u][0], v[u][1], by, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[u][2], v[u][3], by, 1);
        *(uint16_t*)(q + (m0 + u) * 128 + l * 2) = (uint16_t)c;
        if (l % 8 == 0) s[(m0 + u) * 8 + l / 8] = (uint8_t)b;
    }
}

// f with the rows' type and whether they can be loaded by fours as constants
template <int SRC, class F>
__device__ __forceinline__ void by_type(const Fp4ProductArgs& A, F f) {
    using std::integral_constant;
    if constexpr (SRC == kRowsSilu) f(integral_constant<int, 2>(), std::true_type());
    else if (A.x_wide) {
        if (A.x_dt == 0) f(integral_constant<int, 0>(), std::true_type());
        else if (A.x_dt == 1) f(integral_constant<int, 1>(), std::true_type());
        else f(integral_constant<int, 2>(), std::true_type());
    } else {
        if (A.x_dt == 0) f(integral_constant<int, 0>(), std::false_type());
        else if (A.x_dt == 1) f(integral_constant<int, 1>(), std::false_type());
        else f(integral_constant<int, 2>(), std::false_type());
    }
}

// TM x TN fragments of 16 rows x 16 columns by NW waves, S stages of a wave under way; R rows to a group of workgroups
template <int SRC, int TM, int TN, int NW, int S>
__global__ void __launch_bounds__(64 * NW) fp4_few_kernel(Fp4ProductArgs A, int per, int ct, int R, int out_dt) {
    constexpr bool OWN = SRC != kRowsQuantised;
    static_assert(!OWN || TM == 1, "one fragment of rows");
    __shared__ v4f sums[NW][TM * TN][64];
    __shared__ struct {
        alignas(16) uint8_t q[OWN ? 16 * 128 : 16], s[OWN ? 16 * 8 : 16];
    } own[OWN ? NW : 1];
    const int l = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = l >> 4, r = l & 15;
    // neighbouring workgroups go to different XCDs: each XCD takes a run of columns, the groups of rows by turns
    const int rt = (A.M - 1) / R + 1, t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (t >= ct * rt) return;
    const int n0 = t / rt * TN * 16, mb = t % rt * R, M = min(R, A.M - mb);
    const int pitch = A.kp / 2;
    // (this thread's outputs' biases: on their way before anything else)
    constexpr int kOuts = (TM * TN + NW - 1) / NW;
    v4f bias[kOuts];
    const Rsrc biases = buffer_of(A.bias, A.bias ? (uint32_t)A.n * 4 : 0);
#pragma unroll
    for (int o = 0; o < kOuts; ++o) bias[o] = floats_of(biases, n0 + (wave + o * NW) % TN * 16 + g * 4);
    v4f acc[TM][TN] = {};
    for (int b0 = wave; b0 < A.kb; b0 += NW * S) {
        v4i wf[S][TN][2], qf[S][TM][2];
        uint2 ws[S][TN], qs[S][TM];
        auto stage = [&](int u) { return S == 1 ? b0 : min(b0 + u * NW, A.kb - 1); };    // (one too many is not used)
        auto weights = [&] {
#pragma unroll
            for (int u = 0; u < S; ++u)
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    const int b = stage(u), col = min(n0 + i * 16 + r, A.n - 1);
                    const uint8_t* w = A.w + (size_t)col * pitch + g * 16 + (size_t)b * 128;
                    wf[u][i][0] = *(const v4i*)w;
                    wf[u][i][1] = *(const v4i*)(w + ((b + 1) * kFp4Stage > A.kp ? 0 : 64));
                    ws[u][i] = *(const uint2*)(A.sw + ((size_t)b * A.n + col) * 8);
                }
        };
        if constexpr (!OWN) {
#pragma unroll
            for (int u = 0; u < S; ++u)
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    const int b = stage(u), m = mb + min(j * 16 + r, M - 1);
                    const uint8_t* q = A.q + (size_t)m * pitch + g * 16 + (size_t)b * 128;
                    qf[u][j][0] = *(const v4i*)q;
                    qf[u][j][1] = *(const v4i*)(q + ((b + 1) * kFp4Stage > A.kp ? 0 : 64));
                    qs[u][j] = *(const uint2*)(A.s + (size_t)b * A.s_stage + (size_t)m * 8);
                }
            weights();
        } else {
            // (the rows before the weights: they come from caches, and are quantised while the weights are under way)
            auto& o = own[wave];
            by_type<SRC>(A, [&](auto dt, auto wide) {
                constexpr int DT = decltype(dt)::value;
                v4f v[S][4];
                auto rows = [&](int m0) {
#pragma unroll
                    for (int u = 0; u < S; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (m0 + i >= M) break;
                            const size_t row = (size_t)(mb + m0 + i) * A.x_stride;
                            const int c = stage(u) * kFp4Stage + l * 4;
                            if constexpr (SRC == kRowsSilu) {
                                // 32 gates and their 32 ups by turns
                                const float* p = (const float*)A.x + row + (c < A.kp ? c / 32 * 64 + c % 32 : 0);
                                const v4f gate = *(const v4f*)p, up = *(const v4f*)(p + 32);
#pragma unroll
                                for (int j = 0; j < 4; ++j) v[u][i][j] = c < A.kp ? gated(gate[j], up[j]) : 0.0f;
                            } else {
                                v[u][i] = load4<DT, decltype(wide)::value>(A.x, row, c, A.k);
                            }
                        }
                };
                rows(0);
                weights();
                for (int m0 = 0;;) {
                    static_assert(S == 1 || !OWN, "a stage at a time");
                    quant_four(v[0], m0, M, o.q, o.s);
                    m0 += 4;
                    if (m0 >= M) break;
                    rows(m0);
                }
            });
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int m = min(r, M - 1);
            qf[0][0][0] = *(const v4i*)(o.q + m * 128 + g * 16);
            qf[0][0][1] = *(const v4i*)(o.q + m * 128 + 64 + g * 16);
            qs[0][0] = *(const uint2*)(o.s + m * 8);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int u = 0; u < S; ++u) {
            const int b = b0 + u * NW;
            if (b >= A.kb) break;
            const bool half = (b + 1) * kFp4Stage > A.kp;
            int sw[TN];
#pragma unroll
            for (int i = 0; i < TN; ++i) sw[i] = two_scales(ws[u][i], g, half);
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                const int sq = two_scales(qs[u][j], g, half);
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    acc[j][i] = fp4_mfma16<0>(wf[u][i][0], qf[u][j][0], acc[j][i], sw[i], sq);
                    acc[j][i] = fp4_mfma16<1>(wf[u][i][1], qf[u][j][1], acc[j][i], sw[i], sq);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int i = 0; i < TN; ++i) sums[wave][j * TN + i][l] = acc[j][i];
    __syncthreads();
    // a thread's four columns n0 + 16 i + 4 g of row 16 j + r
#pragma unroll
    for (int o = 0; o < kOuts; ++o) {
        const int f = wave + o * NW;
        if (f >= TM * TN) break;
        const int m = f / TN * 16 + r, n = n0 + f % TN * 16 + g * 4;
        if (m >= M || n >= A.n) continue;
        v4f v = {};
#pragma unroll
        for (int i = 0; i < NW; ++i) v += sums[i][f][l];
        v += bias[o];
        const bool whole = n + 4 <= A.n;             // (at any element: one store takes them)
        const size_t at = (size_t)(mb + m) * A.out_stride + n;
        if (out_dt == 2) {
            float* p = (float*)A.out + at;
            if (whole) *(Bytes16At4*)p = __builtin_bit_cast(Bytes16, v);
            else
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n + c < A.n) p[c] = v[c];
        } else {
            const v4u u = out_dt == 0 ? narrow4<0>(v) : narrow4<1>(v);
            uint16_t* p = (uint16_t*)A.out + at;
            if (whole) *(Bytes8At2*)p = __builtin_bit_cast(Bytes8, u);
            else
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n + c < A.n) p[c] = u[c];
        }
    }
}

template <int SRC, int TM, int TN, int NW, int S>
void launch_few(const Fp4ProductArgs& a, int R, int out_dt, hipStream_t st) {
    const int ct = (a.n - 1) / (16 * TN) + 1, rt = (a.M - 1) / R + 1, per = (ct * rt + 7) / 8;
    hipLaunchKernelGGL((fp4_few_kernel<SRC, TM, TN, NW, S>), dim3((unsigned)per * 8), dim3(64 * NW), 0, st, a, per, ct, R, out_dt);
}

// as many waves as there are stages, 4, 8 or 16 of them; of more stages than that, two to a wave at a time
template <int SRC, int TM, int TN>
void launch_few(const Fp4ProductArgs& a, int R, int out_dt, hipStream_t st) {
    if (a.kb <= 4) launch_few<SRC, TM, TN, 4, 1>(a, R, out_dt, st);
    else if (a.kb <= 8) launch_few<SRC, TM, TN, 8, 1>(a, R, out_dt, st);
    else if constexpr (SRC != kRowsQuantised) launch_few<SRC, TM, TN, 16, 1>(a, R, out_dt, st);
    else if constexpr (TM * TN > 8) launch_few<SRC, TM, TN, 8, 2>(a, R, out_dt, st);
    else if (a.kb <= 16) launch_few<SRC, TM, TN, 16, 1>(a, R, out_dt, st);
    else launch_few<SRC, TM, TN, 16, 2>(a, R, out_dt, st);
}
template <int SRC, int TM>
void launch_few(const Fp4ProductArgs& a, int tn, int R, int out_dt, hipStream_t st) {
    if (tn == 1) launch_few<SRC, TM, 1>(a, R, out_dt, st);
    else if (tn == 2) launch_few<SRC, TM, 2>(a, R, out_dt, st);
    else launch_few<SRC, TM, 3>(a, R, out_dt, st);
}

}  // namespace

// tn fragments of 16 columns and R rows (up to 48; 16 where they are quantised here) to a workgroup
void launch_fp4_few(const Fp4ProductArgs& a, int tn, int R, int out_dt, hipStream_t st) {
    if (a.x && a.silu) launch_few<kRowsSilu, 1>(a, tn, R, out_dt, st);
    else if (a.x) launch_few<kRowsX, 1>(a, tn, R, out_dt, st);
    else if (R <= 16) launch_few<kRowsQuantised, 1>(a, tn, R, out_dt, st);
    else if (R <= 32) launch_few<kRowsQuantised, 2>(a, tn, R, out_dt, st);
    else launch_few<kRowsQuantised, 3>(a, tn, R, out_dt, st);
}

}  // namespace exl3
