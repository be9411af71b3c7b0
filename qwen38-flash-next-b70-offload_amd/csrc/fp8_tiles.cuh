// The product of the 8-bit float linear (fp8_linear.hip has the rule that picks a tile): out[m][n] = sum_b s[m][b]
// sw[n / 128][b] sum_(k in b) q[m][k] w[n][k] + bias[n], with the sum over a block's 128 values in one MFMA (16 x 16 x 128,
// e4m3 operands, fp32 sums) and its two scales applied in fp32.
//
// What bounds it, by size: few rows, the weights' way from HBM and the steps of one workgroup, which are few and each waits for
// its loads (medians of a kernel trace: 1 row, 2048 -> 12,288: 7.2 us, 3.5 TB/s; 40 rows, 4096 -> 2048: 5.8 us); more, what a CU
// takes in (fp8_linear.hip); the largest, MFMAs and the power they draw (fp8_tiles_e4m3.hip).
//
// The weights are the MFMA's A operand and the rows its B operand, so a lane's accumulators are four neighbouring columns
// of one row: one row scale per lane.
#pragma once
#include "exl3_common.cuh"
#include "exl3_kernels.h"
#include "fp8_rows.cuh"

#include <type_traits>

namespace exl3 {
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
// below its leading one: fewer bits than fp32 sums keep. It loses 1.5e-5 of the outputs' root mean square for normal values, up to
// 1.7e-4 of the magnitudes for wild ones, 8.5e-4 at the most. bf16 and fp16 outputs take it all the same, for twice the rate:
// bf16's own rounding is 1.7e-3 of the outputs, fp16's 2.1e-4, so the error against 64 bits grows by 1e-4 and by 5e-3 of itself
// (40 and 300 rows, 4096 -> 2048: 1.66202e-3 for 1.66190e-3, 2.082e-4 for 2.072e-4). But an output that cancels to less than
// about a hundredth of its row's others, or an fp16 one of wild values, may be off by more than its rounding. fp32 outputs
// promise more, and so do sums that are quantised again (there 1.5e-5 takes 3e-4 of the values over a border between two of
// e4m3's, 1.5e-3 in what they are multiplied to): those take the bf16 MFMA on the same values (products exact, fp32 sums: 3e-8),
// at half the rate and with the conversions: 777 rows, 2000 -> 1000: 10.9 us for 8.0, 8,192 rows, 2048 -> 12,288: 425 for 217
// (medians of a kernel trace). (A bf16 MFMA takes 18 cycles of a SIMD, with 3 vector instructions of any kind beside it 23-25;
// an e4m3 one 34 either way.)
__device__ __forceinline__ v4f block_sum(const Frag<false>& a, const Frag<false>& b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ v4f block_sum(const Frag<true>& a, const Frag<true>& b) {
    v4f p = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], p, 0, 0, 0);
    return p;
}

// four outputs as fp16 (DT 0) or bf16 (DT 1)
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

// place of 16-byte piece c of a row in LDS: rows are 128 bytes apart (or an odd multiple), and with this the fragment reads
// of 16 rows meet every bank once
__device__ __forceinline__ int piece_at(int row, int c) { return c ^ ((row >> 1) & 7); }

// One block of k of a tile's operands. QB rows of q (none where the workgroup quantises its rows itself). On 16 bytes, as the loads
// to LDS and the fragments' reads are
template <int QB, int BN>
struct alignas(16) Stage {
    uint8_t w[BN * 128];
    uint8_t q[QB ? QB * 128 : 16];
    float s[QB < 64 ? 64 : QB];
    float sw[64];                                    // [0], and [1] for 256 columns
};

// ---- rows quantised by the workgroup itself -----------------------------------------------------------------------------
// into LDS: row m at m * row_bytes, an odd number of blocks apart; its scales s[m * kb + b]
__device__ __forceinline__ int own_row_bytes(int kb) { return (kb | 1) * kFp8Block; }

template <int THREADS, int DT, bool SILU, bool WIDE, class F>
__device__ __forceinline__ void quant_rows(const Fp8ProductArgs& A, uint8_t* q, float* s, F between) {
    constexpr int kTogether = 4, kGroups = THREADS / 16;
    const int i = threadIdx.x & 15, tasks = A.M * A.kb, rb = own_row_bytes(A.kb);
    const uint32_t magic = (65536 + A.kb - 1) / A.kb;        // t / kb for t < 65536 / kb (t is below 128, and so is kb, or 128)
    auto row_of = [&](int t) { return (int)((uint32_t)t * magic >> 16); };
    int t0 = threadIdx.x >> 4;
    float v[kTogether][8], up[kTogether][8];
    auto load = [&] {                                // (four blocks before the first is needed)
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
            const int t = t0 + u * kGroups, m = row_of(t), c = (t - m * A.kb) * kFp8Block + i * 8;
            block_load<DT, SILU, WIDE>(A.x, (size_t)m * A.x_stride + c, A.k, t < tasks ? A.k - c : 0, v[u], up[u]);
        }
    };
    load();
    between();
    while (true) {
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
            const int t = t0 + u * kGroups, m = row_of(t), b = t - m * A.kb;
            float sc;
            block_values<SILU, WIDE>(t < tasks ? A.k - b * kFp8Block - i * 8 : 0, v[u], up[u]);
            const uint2 o = quant_block(v[u], sc);
            if (t >= tasks) continue;
            *(uint2*)(q + m * rb + b * kFp8Block + piece_at(m, i >> 1) * 16 + (i & 1) * 8) = o;
            if (i == 0) s[t] = sc;
        }
        t0 += kTogether * kGroups;
        if (t0 >= tasks) break;
        load();
    }
}

// `between` runs once, after the first rows are requested and before they are needed
template <int THREADS, class F>
__device__ __forceinline__ void quant_rows(const Fp8ProductArgs& A, uint8_t* q, float* s, F between) {
    auto of = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (A.silu && A.x_wide) quant_rows<THREADS, DT, true, true>(A, q, s, between);
        else if (A.silu) quant_rows<THREADS, DT, true, false>(A, q, s, between);
        else if (A.x_wide) quant_rows<THREADS, DT, false, true>(A, q, s, between);
        else quant_rows<THREADS, DT, false, false>(A, q, s, between);
    };
    if (A.x_dt == 0) of(std::integral_constant<int, 0>());
    else if (A.x_dt == 1) of(std::integral_constant<int, 1>());
    else of(std::integral_constant<int, 2>());
}

// ---- the tile ----------------------------------------------------------------------------------------------------------
// A workgroup computes BM rows x BN columns: KG groups of WM x WN waves, of which group i takes the blocks of k i, KG + i, ...
// and brings them to LDS by direct loads, ST stages of its own. The groups' sums join at the end, in the groups' order. OWN:
// the workgroup quantises its (up to 16) rows itself while its first weights are on their way, and `own` is their LDS.
// EXACT: sums without the e4m3 MFMA's losses, outputs in fp16, bf16 or fp32 (out_dt 0, 1, 2); else fp16 or bf16 outputs.
// Two waves per SIMD at least: with more registers than that leaves, MFMAs write accumulation registers, which the multiply-adds
// cannot read (8,192 rows, 2048 -> 12,288, fp32 outputs, side by side: 412 us with the copies, 390 without).
template <bool EXACT, bool OWN, int BM, int BN, int WM, int WN, int KG, int ST>
__global__ void __launch_bounds__(64 * WM * WN * KG, WM * WN * KG <= 4 ? 2 : 1)
    fp8_tile_kernel(Fp8ProductArgs A, int mt, int nt, int per, int out_dt) {
    constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, QB = OWN ? 0 : BM;
    static_assert(!OWN || BM == 16, "one fragment of rows");
    union Lds {
        Stage<QB, BN> stage[KG][ST];
        struct {
            v4f sums[KG > 1 ? KG - 1 : 1][KG > 1 ? NW : 1][TM * TN][KG > 1 ? 64 : 1];
            alignas(16) uint16_t out[NW][TM * 16 * TN * 16];
        } last;
    };
    static_assert(alignof(Lds) >= 16);
    __shared__ Lds lds;
    extern __shared__ __attribute__((aligned(16))) uint8_t own[];
    const int l = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = l >> 4, r = l & 15;
    const int kg = wave / NW, wv = wave % NW;        // (the group of waves, and the wave's place in it)
    // neighbouring workgroups go to different XCDs: each XCD takes a run of tiles, 4 tiles of rows by turns
    const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (t >= mt * nt) return;
    const int band = t / (4 * nt), in = t - band * 4 * nt, bm = min(4, mt - band * 4);
    const int m0 = (band * 4 + in % bm) * BM, n0 = in / bm * BN;
    const int kp = A.kb * kFp8Block, rows = min(BM, A.M - m0), cols = min(BN, A.n - n0);

    // A wave's share of a stage: kLoads instructions, the last one for the scales. One of the others brings 8 rows; rows past
    // the end are zeros
    constexpr int kW = BN / 8 / NW, kLoads = kW + QB / 8 / NW + 1;
    const Rsrc wb = buffer_of(A.w + (size_t)n0 * kp, (uint32_t)cols * kp);
    const Rsrc qb = buffer_of(A.q + (size_t)m0 * kp, OWN ? 0 : (uint32_t)rows * kp);
    uint32_t off[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads - 1; ++i) {
        const int row = ((i < kW ? i : i - kW) * NW + wv) * 8 + (l >> 3);
        off[i] = (uint32_t)row * kp + piece_at(row, l & 7) * 16;
    }
    // the first waves bring 64 row scales each, the others the weights' (one or two; a single wave brings both)
    constexpr bool kBoth = !OWN && NW == 1;
    const bool rows_scales = !OWN && wv < (QB + 63) / 64;
    const Rsrc swb = buffer_of(A.sw + (size_t)(n0 / kFp8Block) * A.kb, (uint32_t)fp8_blocks(cols) * A.kb * 4);
    const Rsrc sb = rows_scales ? buffer_of(A.s + (size_t)m0 * A.kb, (uint32_t)rows * A.kb * 4) : swb;
    const uint32_t sw_off = (uint32_t)(BN > kFp8Block ? l & 1 : 0) * A.kb * 4;
    off[kLoads - 1] = rows_scales ? (uint32_t)(wv * 64 + l) * A.kb * 4 : sw_off;
    auto load = [&](int b, int i) {
        Stage<QB, BN>& st = lds.stage[kg][b & (ST - 1)];
        b = min(b * KG + kg, A.kb - 1);              // (stages after the last are not used)
        if (i < kW) to_lds<16>(st.w + (i * NW + wv) * 1024, wb, off[i], b * kFp8Block);
        else if (i < kLoads - 1) to_lds<16>(st.q + ((i - kW) * NW + wv) * 1024, qb, off[i], b * kFp8Block);
        else {
            to_lds<4>(rows_scales ? st.s + wv * 64 : st.sw, sb, off[i], b * 4);
            if constexpr (kBoth) to_lds<4>(st.sw, swb, sw_off, b * 4);
        }
    };

    const int wm = wv / WN * (BM / WM), wn = wv % WN * (BN / WN);
    const int at0 = r * 128 + piece_at(r, g) * 16, at1 = r * 128 + piece_at(r, g + 4) * 16;
    auto frag = [&](const uint8_t* p) { return frag_of<EXACT>(*(const v4i*)(p + at0), *(const v4i*)(p + at1)); };
    v4f acc[TM][TN] = {};
    v4f x[2][TN] = {};                               // a fragment's block sums, and the scale that awaits them
    float sc[2] = {};
    auto add = [&](int j) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[j][i][c] = __builtin_fmaf(x[j & 1][i][c], sc[j & 1], acc[j][i][c]);
    };
    auto load_first = [&] {
#pragma unroll
        for (int b = 0; b < ST - 1; ++b)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) load(b, i);
    };
    float* own_s = (float*)(own + (OWN ? A.M * own_row_bytes(A.kb) : 0));
    const int om = OWN ? min(r, A.M - 1) : 0;        // (this lane's row)
    if constexpr (OWN) quant_rows<64 * NW * KG>(A, own, own_s, load_first);
    else load_first();
    const int steps = (A.kb + KG - 1) / KG;
    for (int b = 0; b < steps; ++b) {
        // stage b has arrived for every wave (later ones may be under way), and every wave has read stage b - 1
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * (kLoads + kBoth)) : "memory");
        if (KG > 1 && b * KG + kg >= A.kb) break;    // (the last step; nothing is waited for before the join)
        const Stage<QB, BN>& st = lds.stage[kg][b & (ST - 1)];
        const float sw = st.sw[wn / kFp8Block];
        auto q_frag = [&](int j) {
            if constexpr (OWN) {
                const uint8_t* p = own + om * own_row_bytes(A.kb) + (b * KG + kg) * kFp8Block;
                return frag_of<EXACT>(*(const v4i*)(p + piece_at(om, g) * 16), *(const v4i*)(p + piece_at(om, g + 4) * 16));
            } else {
                return frag(st.q + (wm + j * 16) * 128);
            }
        };
        constexpr int kEach = TM == 1 ? kLoads : (kLoads + TM - 2) / (TM - 1);   // loads of a later stage per fragment
        Frag<EXACT> qf[2], wf[TN];
        qf[0] = q_frag(0);
#pragma unroll
        for (int i = 0; i < TN; ++i) wf[i] = frag(st.w + (wn + i * 16) * 128);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            // under this fragment's MFMAs the next one is read and the last one's sums are scaled (at j = 0 those of the
            // block before)
#pragma unroll
            for (int i = j * kEach; i < min((j + 1) * kEach, kLoads); ++i) load(b + ST - 1, i);
            if (j + 1 < TM) qf[(j + 1) & 1] = q_frag(j + 1);
            if constexpr (TM == 1) {
                sc[0] = (OWN ? own_s[om * A.kb + b * KG + kg] : st.s[wm + r]) * sw;
#pragma unroll
                for (int i = 0; i < TN; ++i) x[0][i] = block_sum(wf[i], qf[0]);
                add(0);
            } else {
#pragma unroll
                for (int i = 0; i < TN; ++i) x[j & 1][i] = block_sum(wf[i], qf[j & 1]);
                add(j ? j - 1 : TM - 1);
                sc[j & 1] = st.s[wm + j * 16 + r] * sw;
                // (the exact sums' conversions between their MFMAs too where there are 8 of those: 777 rows, 2000 -> 1000, side by
                // side, 10.4 -> 9.9 us; with 4 of them, 256 rows, 5.8 against 5.7)
                constexpr bool kThrees = EXACT && TN > 1;
                __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
                for (int i = 0; i < (kThrees ? 4 : 1) * TN; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x2, kThrees ? 3 : 5, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if constexpr (TM > 1) add(TM - 1);
    // no load to LDS may outlive the workgroup, and sums and outputs go through LDS
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (KG > 1) {
        // the groups' sums join in the groups' order, in the first one
        if (kg)
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int i = 0; i < TN; ++i) lds.last.sums[kg - 1][wv][j * TN + i][l] = acc[j][i];
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int k = 0; k < KG - 1; ++k) acc[j][i] += lds.last.sums[k][wv][j * TN + i][l];
    }
    v4f bias[TN] = {};
    if (A.bias)
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int n = n0 + wn + i * 16 + g * 4 + c;
                bias[i][c] = n < A.n ? A.bias[n] : 0.0f;
            }
    if (EXACT && out_dt == 2) {
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
        uint16_t* o = lds.last.out[wv];
        auto to_out = [&](auto dt) {
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    const int m = j * 16 + r, piece = (i * 2 + (g >> 1)) ^ (m & (kPieces - 1));
                    *(v4u*)(o + (m * kPieces + piece) * 8 + (g & 1) * 4) = narrow4<decltype(dt)::value>(acc[j][i] + bias[i]);
                }
        };
        if (out_dt == 0) to_out(std::integral_constant<int, 0>());
        else to_out(std::integral_constant<int, 1>());
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const bool wide = A.out_stride % 8 == 0 && (uintptr_t)A.out % 16 == 0;
#pragma unroll
        for (int k = 0; k < (TM * 16 * kPieces + 63) / 64; ++k) {
            const int at = k * 64 + l, row = at / kPieces, piece = at % kPieces;
            if (TM * 16 * kPieces < 64 && row >= 16) continue;
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

template <bool EXACT, bool OWN, int BM, int BN, int WM, int WN, int KG, int ST>
void launch_fp8_tiles(const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    const int mt = (a.M - 1) / BM + 1, nt = (a.n - 1) / BN + 1, per = (int)(((int64_t)mt * nt + 7) / 8);
    const int own = OWN ? a.M * ((a.kb | 1) * kFp8Block + a.kb * 4) : 0;
    hipLaunchKernelGGL((fp8_tile_kernel<EXACT, OWN, BM, BN, WM, WN, KG, ST>), dim3((unsigned)per * 8), dim3(64 * WM * WN * KG),
                       own, st, a, mt, nt, per, out_dt);
}

// `few`: at most one workgroup per CU, so that it may have the CU's LDS. More stages pay where more than two steps follow each
// other (weights from HBM, us per call out of a graph, side by side: 4096 -> 2048, 16 rows 7.2 -> 6.6, 64 rows 9.5 -> 7.2, exact
// 9.8 -> 7.3, 128 rows 10.6 -> 8.6, exact 11.2 -> 9.2; with one step, k 512, 17 rows 3.2 -> 3.7), and e4m3's 128 x 128 as one group
// of 8 waves, whose registers allow it (1,500 rows 28.0 -> 25.0; exact, whose waves would convert more, 36.0 -> 40.2).
// Rows quantised inside: as many blocks of 128 as 256 threads have in hand at once, else 512 threads (4096 -> 2048, 1 row 6.0
// us, with 512 7.0; 2048 -> 1024, 8 rows 6.0 and 5.2). As few rows that were quantised before take the same groups of waves, so
// that the product is the same to the last bit.
template <bool EXACT>
void launch_fp8_tile(int tile, bool few, const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    const bool little = a.M <= 16 && (int64_t)a.M * a.kb <= 64;
    if (!a.q) {                                      // (no other tile may have these: their rows come from q)
        if (tile == kTile16 && little) launch_fp8_tiles<EXACT, true, 16, 16, 1, 1, 4, 4>(a, out_dt, st);
        else if (tile == kTile16) launch_fp8_tiles<EXACT, true, 16, 16, 1, 1, 8, 2>(a, out_dt, st);
        else launch_fp8_tiles<EXACT, true, 16, 32, 1, 2, 2, 4>(a, out_dt, st);
        return;
    }
    if constexpr (EXACT) {
        if (few && tile == kTile128) return launch_fp8_tiles<EXACT, false, 128, 128, 2, 2, 2, 2>(a, out_dt, st);
    } else {
        if (few && tile == kTile128) return launch_fp8_tiles<EXACT, false, 128, 128, 2, 4, 1, 4>(a, out_dt, st);
        if (tile == kTile128x64) return launch_fp8_tiles<EXACT, false, 128, 64, 4, 2, 1, 4>(a, out_dt, st);
    }
    if (tile == kTile16 && little) launch_fp8_tiles<EXACT, false, 16, 16, 1, 1, 4, 4>(a, out_dt, st);
    else if (tile == kTile16x32 && little) launch_fp8_tiles<EXACT, false, 16, 32, 1, 2, 2, 4>(a, out_dt, st);
    else if (tile == kTile16 && few && a.kb > 16) launch_fp8_tiles<EXACT, false, 16, 16, 1, 1, 8, 4>(a, out_dt, st);
    else if (tile == kTile16) launch_fp8_tiles<EXACT, false, 16, 16, 1, 1, 8, 2>(a, out_dt, st);
    else if (tile == kTile16x32 && few && a.kb > 8) launch_fp8_tiles<EXACT, false, 16, 32, 1, 2, 4, 4>(a, out_dt, st);
    else if (tile == kTile16x32) launch_fp8_tiles<EXACT, false, 16, 32, 1, 2, 4, 2>(a, out_dt, st);
    else if (tile == kTile32 && few && a.kb > 8) launch_fp8_tiles<EXACT, false, 32, 32, 1, 2, 4, 4>(a, out_dt, st);
    else if (tile == kTile32) launch_fp8_tiles<EXACT, false, 32, 32, 1, 2, 4, 2>(a, out_dt, st);
    else if (tile == kTile64 && few) launch_fp8_tiles<EXACT, false, 64, 64, 2, 2, 2, 4>(a, out_dt, st);
    else if (tile == kTile64) launch_fp8_tiles<EXACT, false, 64, 64, 2, 2, 2, 2>(a, out_dt, st);
    else launch_fp8_tiles<EXACT, false, 128, 128, 2, 2, 1, 2>(a, out_dt, st);
}

}  // namespace exl3
