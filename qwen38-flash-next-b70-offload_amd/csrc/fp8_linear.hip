// The 8-bit float product: out[m][n] = sum_b s[m][b] sw[n / 128][b] sum_(k in b) q[m][k] w[n][k] + bias[n], with the sum
// over a block's 128 values in one MFMA (16 x 16 x 128, e4m3 operands, fp32 sums) and its two scales applied in fp32.
//
// The weights are the MFMA's A operand and the rows its B operand, so a lane's accumulators are four neighbouring columns
// of one row: one row scale per lane, and the outputs are stored four at a time.
#include "exl3_common.cuh"
#include "exl3_kernels.h"
#include "fp8_rows.cuh"

#include <algorithm>

namespace exl3 {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint16_t v4u __attribute__((ext_vector_type(4)));
typedef uint16_t v8u __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_any;

// A lane's 32 of the 128 values of a block, of one row of either operand. EXACT: as bf16, for which e4m3's values fit
template <bool EXACT> struct Frag { v8i v; };
template <> struct Frag<true> { v8b v[4]; };

__device__ __forceinline__ v8b widen(int lo, int hi) {
    const v2b a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const v2b b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const v2b c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const v2b d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return v8b{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <bool EXACT>
__device__ __forceinline__ Frag<EXACT> frag_of(v4i a, v4i b) {
    if constexpr (EXACT) return {widen(a[0], a[1]), widen(a[2], a[3]), widen(b[0], b[1]), widen(b[2], b[3])};
    else return {v8i{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
}

// The sum over one block. The e4m3 MFMA adds products in groups of 8 k, aligned to the group's largest and cut 13 bits
// below its leading one (1.5e-5 of the sum's own size for normal values, up to 1.7e-4 of the magnitudes for wild ones):
// far below the rounding of bf16 or fp16 outputs, and not what fp32 outputs promise. Those take the bf16 MFMA on the same
// values (products exact, fp32 sums: 3e-8), at half the rate and with the conversions.
__device__ __forceinline__ v4f block_sum(const Frag<false>& a, const Frag<false>& b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ v4f block_sum(const Frag<true>& a, const Frag<true>& b) {
    v4f p = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], p, 0, 0, 0);
    return p;
}

template <int DT>
__device__ __forceinline__ v4u narrow4(v4f v) {
    v4u u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (DT == 0) u[j] = __builtin_bit_cast(uint16_t, (_Float16)v[j]);
        else u[j] = __builtin_bit_cast(uint16_t, (__bf16)v[j]);
    }
    return u;
}

// ---- tiles -----------------------------------------------------------------------------------------------------------
// A workgroup of WM x WN waves computes BM rows x BN columns. Per block of k its weights and rows come into LDS by
// direct loads (one stage ahead), 128 bytes a row, the row's 16-byte pieces in an order that differs from row to row so
// that the fragment reads of 16 rows meet every bank once.

template <int BM, int BN>
struct Stage {
    uint8_t w[BN * 128];
    uint8_t q[BM * 128];
    float s[BM];
    float sw[64];                                    // [0], and [1] for 256 columns
};

// place of 16-byte piece c of a row (the same for every 16 rows)
__device__ __forceinline__ int piece_at(int row, int c) { return c ^ ((row >> 1) & 7); }

using Rsrc = __amdgpu_buffer_rsrc_t;
// a buffer of `bytes`, zeros behind it
__device__ __forceinline__ Rsrc buffer_of(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
// 16 bytes a lane (or 4) from the buffer to LDS, the lanes' pieces one after the other
template <int BYTES>
__device__ __forceinline__ void to_lds(void* lds, Rsrc from, uint32_t lane_off, uint32_t off) {
    if constexpr (BYTES == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_any*)lds, 16, lane_off, off, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_any*)lds, 4, lane_off, off, 0, 0);
}

template <int DT, int BM, int BN, int WM, int WN, int ST>
__global__ void __launch_bounds__(64 * WM * WN) fp8_tile_kernel(Fp8ProductArgs A, int mt, int nt, int per) {
    constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
    constexpr bool EXACT = DT == 2;
    union Lds {
        Stage<BM, BN> stage[ST];
        uint16_t out[NW][TM * 16 * TN * 16];
    };
    __shared__ Lds lds;
    const int l = lane_id(), wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = l >> 4, r = l & 15;
    // neighbouring workgroups go to different XCDs: each XCD takes a run of tiles, 4 tiles of rows by turns
    const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (t >= mt * nt) return;
    const int band = t / (4 * nt), in = t - band * 4 * nt, bm = min(4, mt - band * 4);
    const int m0 = (band * 4 + in % bm) * BM, n0 = in / bm * BN;
    const int kp = A.kb * kFp8Block, rows = min(BM, A.M - m0), cols = min(BN, A.n - n0);

    // A wave's share of a stage: kLoads instructions, the last one for the scales. One of the others brings 8 rows; rows past
    // the end are zeros
    constexpr int kW = BN / 8 / NW, kLoads = kW + BM / 8 / NW + 1;
    const Rsrc wb = buffer_of(A.w + (size_t)n0 * kp, (uint32_t)cols * kp), qb = buffer_of(A.q + (size_t)m0 * kp, (uint32_t)rows * kp);
    uint32_t off[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads - 1; ++i) {
        const int row = ((i < kW ? i : i - kW) * NW + wv) * 8 + (l >> 3);
        off[i] = (uint32_t)row * kp + piece_at(row, l & 7) * 16;
    }
    // the first BM / 64 waves bring 64 row scales each, the others the weights' (one or two)
    const bool rows_scales = wv < BM / 64;
    const Rsrc sb = rows_scales ? buffer_of(A.s + (size_t)m0 * A.kb, (uint32_t)rows * A.kb * 4)
                                : buffer_of(A.sw + (size_t)(n0 / kFp8Block) * A.kb, (uint32_t)fp8_blocks(cols) * A.kb * 4);
    off[kLoads - 1] = (uint32_t)(rows_scales ? wv * 64 + l : BN > kFp8Block ? l & 1 : 0) * A.kb * 4;
    auto load = [&](int b, int i) {
        Stage<BM, BN>& st = lds.stage[b & (ST - 1)];
        b = min(b, A.kb - 1);                        // (stages after the last are not used)
        if (i < kW) to_lds<16>(st.w + (i * NW + wv) * 1024, wb, off[i], b * kFp8Block);
        else if (i < kLoads - 1) to_lds<16>(st.q + ((i - kW) * NW + wv) * 1024, qb, off[i], b * kFp8Block);
        else to_lds<4>(rows_scales ? st.s + wv * 64 : st.sw, sb, off[i], b * 4);
    };
    const int wm = wv / WN * (BM / WM), wn = wv % WN * (BN / WN);
    const int at0 = r * 128 + piece_at(r, g) * 16, at1 = r * 128 + piece_at(r, g + 4) * 16;
    v4f acc[TM][TN] = {};
    v4f x[2][TN] = {};                               // a fragment's block sums, and the scale that awaits them
    float sc[2] = {};
    auto add = [&](int j) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[j][i][c] = __builtin_fmaf(x[j & 1][i][c], sc[j & 1], acc[j][i][c]);
    };
#pragma unroll
    for (int b = 0; b < ST - 1; ++b)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(b, i);
    for (int b = 0; b < A.kb; ++b) {
        // stage b has arrived for every wave (later ones may be under way), and every wave has read stage b - 1
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * kLoads) : "memory");
        const Stage<BM, BN>& st = lds.stage[b & (ST - 1)];
        const float sw = st.sw[wn / kFp8Block];
        auto frag = [&](const uint8_t* p) { return frag_of<EXACT>(*(const v4i*)(p + at0), *(const v4i*)(p + at1)); };
        constexpr int kEach = TM == 1 ? kLoads : (kLoads + TM - 2) / (TM - 1);   // loads of a later stage per fragment
        Frag<EXACT> qf[2], wf[TN];
        qf[0] = frag(st.q + wm * 128);
#pragma unroll
        for (int i = 0; i < TN; ++i) wf[i] = frag(st.w + (wn + i * 16) * 128);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            // under this fragment's MFMAs the next one is read and the last one's sums are scaled (at j = 0 those of the
            // block before)
#pragma unroll
            for (int i = j * kEach; i < min((j + 1) * kEach, kLoads); ++i) load(b + ST - 1, i);
            if (j + 1 < TM) qf[(j + 1) & 1] = frag(st.q + (wm + (j + 1) * 16) * 128);
#pragma unroll
            for (int i = 0; i < TN; ++i) x[j & 1][i] = block_sum(wf[i], qf[j & 1]);
            add(j ? j - 1 : TM - 1);
            sc[j & 1] = st.s[wm + j * 16 + r] * sw;
            __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 5, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    add(TM - 1);
    // no load to LDS may outlive the workgroup, and the outputs go through LDS
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    v4f bias[TN] = {};
    if (A.bias)
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int n = n0 + wn + i * 16 + g * 4 + c;
                bias[i][c] = n < A.n ? A.bias[n] : 0.0f;
            }
    if constexpr (DT == 2) {
        // a lane's four columns at once where they are there and every row's fours start on 16 bytes
        const bool wide = A.n % 4 == 0 && A.out_stride % 4 == 0 && (uintptr_t)A.out % 16 == 0;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                const int n = n0 + wn + i * 16 + g * 4, m = m0 + wm + j * 16 + r;
                if (n >= A.n || m >= A.M) continue;
                float* p = (float*)A.out + (size_t)m * A.out_stride + n;
                const v4f v = acc[j][i] + bias[i];
                if (wide) *(v4f*)p = v;
                else
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (n + c < A.n) p[c] = v[c];
            }
    } else {
        // the wave's outputs [rows][16 TN] through its own part of LDS, so that a lane stores 16 bytes and a row's pieces
        // are next to each other; the pieces of a row in an order that differs from row to row (banks)
        constexpr int kPieces = TN * 2;              // 16-byte pieces of a row
        uint16_t* o = lds.out[wv];
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const int m = j * 16 + r, piece = (i * 2 + (g >> 1)) ^ (m & (kPieces - 1));
                *(v4u*)(o + (m * kPieces + piece) * 8 + (g & 1) * 4) = narrow4<DT>(acc[j][i] + bias[i]);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const bool wide = A.out_stride % 8 == 0 && (uintptr_t)A.out % 16 == 0;
#pragma unroll
        for (int k = 0; k < TM * 16 * kPieces / 64; ++k) {
            const int at = k * 64 + l, row = at / kPieces, piece = at % kPieces;
            const int m = m0 + wm + row, n = n0 + wn + piece * 8;
            if (m >= A.M || n >= A.n) continue;
            const v8u v = *(const v8u*)(o + (row * kPieces + (piece ^ (row & (kPieces - 1)))) * 8);
            uint16_t* p = (uint16_t*)A.out + (size_t)m * A.out_stride + n;
            if (wide && n + 8 <= A.n) *(v8u*)p = v;
            else
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (n + c < A.n) p[c] = v[c];
        }
    }
}

// ---- few rows --------------------------------------------------------------------------------------------------------
// A workgroup of 8 waves computes up to 16 MT rows x 16 NT columns; its waves share the blocks of k, each with its weights
// straight from memory to registers (requested before anything else), and their sums are joined over LDS in the waves'
// order. QUANT: the workgroup quantises the rows itself, into LDS, while its weights are on their way; else the rows'
// fragments come from memory too.
constexpr int kFewWaves = 8;

// quantised row m in LDS: blocks of 128 bytes, an odd number of them per row, pieces in an order of their own per row (banks)
__device__ __forceinline__ int few_row_bytes(int kb) { return (kb | 1) * kFp8Block; }

template <int DT, bool SILU>
__device__ __forceinline__ void few_quant(const Fp8ProductArgs& A, uint8_t* q, float* s) {
    const int i = threadIdx.x & 15, tasks = A.M * A.kb, rb = few_row_bytes(A.kb);
    constexpr int kTogether = 4, kGroups = kFewWaves * 4;
    for (int t0 = threadIdx.x >> 4; t0 < tasks; t0 += kTogether * kGroups) {
        float v[kTogether][8];
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {        // (the loads of four blocks before the first is needed)
            const int t = t0 + u * kGroups, m = t / A.kb, c = (t - m * A.kb) * kFp8Block + i * 8;
            const size_t at = (size_t)m * A.x_stride + c;
            if (A.x_wide) block_values<DT, SILU, true>(A.x, at, A.k, t < tasks ? A.k - c : 0, v[u]);
            else block_values<DT, SILU, false>(A.x, at, A.k, t < tasks ? A.k - c : 0, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
            const int t = t0 + u * kGroups, m = t / A.kb, b = t - m * A.kb;
            float sc;
            const uint2 o = quant_block(v[u], sc);
            if (t >= tasks) continue;
            *(uint2*)(q + m * rb + b * kFp8Block + piece_at(m, i >> 1) * 16 + (i & 1) * 8) = o;
            if (i == 0) s[t] = sc;
        }
    }
}

template <bool EXACT, bool QUANT, int MT, int NT>
__global__ void __launch_bounds__(64 * kFewWaves) fp8_few_kernel(Fp8ProductArgs A, int out_dt, int s_at) {
    extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
    const int l = lane_id(), wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = l >> 4, r = l & 15;
    const int n0 = blockIdx.x * 16 * NT, kp = A.kb * kFp8Block, cols = min(16 * NT, A.n - n0);
    const Rsrc wb = buffer_of(A.w + (size_t)n0 * kp, (uint32_t)cols * kp);
    constexpr int kDepth = NT == 1 ? 4 : NT == 2 ? 3 : 2;        // blocks of weights under way per wave
    v4i w[kDepth][NT][2];
    float sw[kDepth][NT];
    auto load_w = [&](int d, int b) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint32_t off = (uint32_t)(i * 16 + r) * kp + g * 16;
            w[d][i][0] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(wb, off, b * kFp8Block, 0));
            w[d][i][1] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(wb, off + 64, b * kFp8Block, 0));
            sw[d][i] = A.sw[(size_t)(min(n0 + i * 16, A.n - 1) / kFp8Block) * A.kb + b];
        }
    };
    const int nb = (A.kb - wv + kFewWaves - 1) / kFewWaves;      // this wave's blocks: wv, wv + 8, ...
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
        if (d < nb) load_w(d, wv + d * kFewWaves);
    float* ls = (float*)(few_lds + s_at);
    if constexpr (QUANT) {
        if (A.silu) {
            if (A.x_dt == 0) few_quant<0, true>(A, few_lds, ls);
            else if (A.x_dt == 1) few_quant<1, true>(A, few_lds, ls);
            else few_quant<2, true>(A, few_lds, ls);
        } else {
            if (A.x_dt == 0) few_quant<0, false>(A, few_lds, ls);
            else if (A.x_dt == 1) few_quant<1, false>(A, few_lds, ls);
            else few_quant<2, false>(A, few_lds, ls);
        }
        __syncthreads();
    }
    v4f acc[MT][NT] = {};
    for (int i0 = 0; i0 < nb; i0 += kDepth) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            if (i0 + d >= nb) break;
            const int b = wv + (i0 + d) * kFewWaves;
            Frag<EXACT> wf[NT];
            float swd[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) wf[i] = frag_of<EXACT>(w[d][i][0], w[d][i][1]), swd[i] = sw[d][i];
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const int m = min(j * 16 + r, A.M - 1);
                v4i a0, a1;
                float sm;
                if constexpr (QUANT) {
                    const uint8_t* p = few_lds + m * few_row_bytes(A.kb) + b * kFp8Block;
                    a0 = *(const v4i*)(p + piece_at(m, g) * 16), a1 = *(const v4i*)(p + piece_at(m, g + 4) * 16);
                    sm = ls[m * A.kb + b];
                } else {
                    const uint8_t* p = A.q + ((size_t)m * A.kb + b) * kFp8Block + g * 16;
                    a0 = *(const v4i*)p, a1 = *(const v4i*)(p + 64);
                    sm = A.s[(size_t)m * A.kb + b];
                }
                const Frag<EXACT> qf = frag_of<EXACT>(a0, a1);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const v4f x = block_sum(wf[i], qf);
                    const float sc = sm * swd[i];
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[j][i][c] = __builtin_fmaf(x[c], sc, acc[j][i][c]);
                }
            }
            if (i0 + d + kDepth < nb) load_w(d, b + kDepth * kFewWaves);
        }
    }
    if constexpr (QUANT) __syncthreads();            // (the rows in LDS are read)
    v4f* red = (v4f*)few_lds;                        // [wave][tile][lane]
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < NT; ++i) red[(wv * MT * NT + j * NT + i) * 64 + l] = acc[j][i];
    __syncthreads();
    if (wv >= MT * NT) return;                       // one tile per wave
    v4f y = red[wv * 64 + l];
#pragma unroll
    for (int k = 1; k < kFewWaves; ++k) y += red[(k * MT * NT + wv) * 64 + l];
    const int m = wv / NT * 16 + r, n = n0 + wv % NT * 16 + g * 4;
    if (m >= A.M) return;
    const size_t at = (size_t)m * A.out_stride + n;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (n + c < A.n && A.bias) y[c] += A.bias[n + c];
    const bool wide = n + 4 <= A.n && A.out_stride % 4 == 0 && (uintptr_t)A.out % (EXACT ? 16 : 8) == 0;
    if constexpr (EXACT) {
        float* p = (float*)A.out + at;
        if (wide) *(v4f*)p = y;
        else
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (n + c < A.n) p[c] = y[c];
    } else {
        const v4u u = out_dt == 0 ? narrow4<0>(y) : narrow4<1>(y);
        uint16_t* p = (uint16_t*)A.out + at;
        if (wide) *(v4u*)p = u;
        else
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (n + c < A.n) p[c] = u[c];
    }
}

template <bool EXACT, bool QUANT, int MT, int NT>
void launch_few(const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    const int s_at = QUANT ? a.M * (a.kb | 1) * kFp8Block : 0;
    const int lds = std::max(QUANT ? s_at + a.M * a.kb * 4 : 0, kFewWaves * MT * NT * 1024);
    hipLaunchKernelGGL((fp8_few_kernel<EXACT, QUANT, MT, NT>), dim3((unsigned)((a.n - 1) / (16 * NT) + 1)), dim3(64 * kFewWaves),
                       lds, st, a, out_dt, s_at);
}

template <bool EXACT, bool QUANT, int MT>
void launch_few_n(const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    // columns per workgroup: enough workgroups for every CU first
    const int tiles = (a.n - 1) / 16 + 1;
    if constexpr (MT <= 2) {
        if (tiles > 512 && MT * 3 <= 8) return launch_few<EXACT, QUANT, MT, 3>(a, out_dt, st);
    }
    if (tiles > 256) return launch_few<EXACT, QUANT, MT, 2>(a, out_dt, st);
    launch_few<EXACT, QUANT, MT, 1>(a, out_dt, st);
}

template <bool EXACT>
void launch_few_m(const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    if (!a.q) launch_few_n<EXACT, true, 1>(a, out_dt, st);
    else if (a.M <= 16) launch_few_n<EXACT, false, 1>(a, out_dt, st);
    else if (a.M <= 32) launch_few_n<EXACT, false, 2>(a, out_dt, st);
    else launch_few_n<EXACT, false, 4>(a, out_dt, st);
}

template <int DT, int BM, int BN, int WM, int WN, int ST>
void launch_tiles(const Fp8ProductArgs& a, hipStream_t st) {
    const int mt = (a.M - 1) / BM + 1, nt = (a.n - 1) / BN + 1, per = (mt * nt + 7) / 8;
    hipLaunchKernelGGL((fp8_tile_kernel<DT, BM, BN, WM, WN, ST>), dim3((unsigned)per * 8), dim3(64 * WM * WN), 0, st, a,
                       mt, nt, per);
}

template <int DT>
void launch_dt(const Fp8ProductArgs& a, hipStream_t st) {
    auto tiles = [&](int bm, int bn) { return (int64_t)((a.M - 1) / bm + 1) * ((a.n - 1) / bn + 1); };
    if constexpr (DT != 2) {
        if (tiles(256, 256) >= 192) return launch_tiles<DT, 256, 256, 2, 4, 2>(a, st);
        if (tiles(128, 128) >= 192) return launch_tiles<DT, 128, 128, 2, 2, 2>(a, st);
    }
    launch_tiles<DT, 64, 64, 2, 2, 4>(a, st);
}

}  // namespace

// rows up to which the product quantises them itself, and the bytes of LDS that they may take
constexpr int kQuantRows = 16, kQuantBytes = 48 * 1024;
constexpr int kFewRows = 64;

bool fp8_product_quantises(int M, int k, int n) {
    const int kb = fp8_blocks(k);
    return M <= kQuantRows && (int64_t)M * ((kb | 1) * (int64_t)kFp8Block + kb * 4) <= kQuantBytes;
}

hipError_t launch_fp8_product(const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    if (!a.q || a.M <= kFewRows) {
        if (out_dt == 2) launch_few_m<true>(a, out_dt, st);
        else launch_few_m<false>(a, out_dt, st);
    } else if (out_dt == 0) launch_dt<0>(a, st);
    else if (out_dt == 1) launch_dt<1>(a, st);
    else launch_dt<2>(a, st);
    return hipGetLastError();
}

}  // namespace exl3
