// The product of the 4-bit float linear (fp4_linear.hip has the rule that picks a tile): out[m][n] = sum_k q[m][k] w[n][k], each
// times its block's scale, + bias[n].
//
// One MFMA (32 x 32 x 64, both operands e2m1 with a scale byte per lane) takes two blocks of 32 with their scales. Its products
// are exact and its sums keep the bits that fp32 additions in a row would: against 64 bits, random scales 2^-7 to 2^7 and 4,096
// columns, 1.312e-7 of the outputs' norm, a chain of fp32 additions of exact block sums 1.311e-7; scales 2^-3 to 2^3, 0. So
// outputs of every type come from it. From registers, 4 x 4 accumulators to a wave, it runs at 6.4 to 6.6 PFLOP/s on random codes
// (8.8 to 9.6 on zeros); 16 x 16 x 128 at 7.5 (9.2), but takes twice the fragments' reads per product.
//
// The weights are the MFMA's A operand and the rows its B operand, so a lane's accumulators are fours of neighbouring
// columns of one row.
#pragma once
#include "exl3_kernels.h"
#include "fp4_rows.cuh"
#include "tile_common.cuh"

#include <type_traits>

namespace exl3 {
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v2i __attribute__((ext_vector_type(2)));

// 32 codes of a lane as an operand
__device__ __forceinline__ v8i fp4_operand(v4i v) { return v8i{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

// The scales of a lane's four blocks of a stage (columns 64 j + 32 h) out of its row's eight, byte j for step j
__device__ __forceinline__ int lane_scales(v2i row, int h) {
    return (int)__builtin_amdgcn_perm(row.y, row.x, h ? 0x07050301u : 0x06040200u);
}

template <int J>
__device__ __forceinline__ v16f fp4_mfma(v8i w, v8i q, v16f acc, int sw, int sq) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, q, acc, 4, 4, J, sw, J, sq);
}

// f(0), ..., f(3) with constants
template <class F>
__device__ __forceinline__ void four_steps(F f) {
    f(std::integral_constant<int, 0>());
    f(std::integral_constant<int, 1>());
    f(std::integral_constant<int, 2>());
    f(std::integral_constant<int, 3>());
}

// One stage of 256 columns of a tile's operands: 128 bytes and 8 scales to a row
template <int BM, int BN>
struct alignas(16) Fp4Stage {
    uint8_t w[BN * 128];
    uint8_t q[BM * 128];
    uint8_t sw[BN * 8];
    uint8_t sq[BM * 8];
};

__device__ __forceinline__ float gated(float g, float u) { return g < kSiluFar ? silu_times_far(g, u) : silu_times(g, u); }

// One block of 32 of a row's values, of which a lane has those at 8 b + 4 h + c in v[4 b + c] and the lane 32 further the others:
// its codes and scale are written
__device__ __forceinline__ void silu_block(const Fp4ProductArgs& A, const float (&v)[16], int m, int block, int h) {
    uint32_t amax = 0;
#pragma unroll
    for (int c = 0; c < 16; ++c) amax = max(amax, abs_bits(v[c]));
    amax = max(amax, __float_as_uint(lane_xor(__uint_as_float(amax), 32)));
    const uint32_t scale = fp4_scale_byte(amax);
    const float lo[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
    const float hi[8] = {v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]};
    const uint32_t own[2] = {pack_e2m1(lo, scale), pack_e2m1(hi, scale)};       // 16 bits of each b
    // the lower lane takes the first 8 bytes of the block, the upper one the last
    const uint32_t other = __float_as_uint(lane_xor(__uint_as_float(h ? own[0] : own[1]), 32));
    const uint32_t a = h ? other : own[0], b = h ? own[1] : other;
    if (m >= A.M) return;
    *(uint2*)(A.hq + (size_t)m * (A.n / 4) + block * 16 + h * 8) = {(a & 0xFFFFu) | b << 16, a >> 16 | (b & 0xFFFF0000u)};
    if (h == 0) A.hs[(size_t)(block / 8) * A.M * 8 + (size_t)m * 8 + block % 8] = (uint8_t)scale;
}

// A workgroup computes BM rows x BN columns: KG groups of WM x WN waves, of which group i takes the stages i, KG + i, ... and
// brings them to LDS by direct loads, ST stages of its own. The groups' sums join at the end, in the groups' order.
// SILU: the weights' rows are 32 gates and their 32 ups by turns, and instead of the products silu(gate) * up leaves as 4-bit rows,
// out of the accumulators: a pair of fragments holds one block of 32 of them, 16 of a row's in each half of the wave.
template <bool SILU, int BM, int BN, int WM, int WN, int KG, int ST>
__global__ void __launch_bounds__(64 * WM * WN * KG) fp4_tile_kernel(Fp4ProductArgs A, int mt, int nt, int per, int out_dt) {
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    static_assert(!SILU || TN % 2 == 0, "a gate's ups are in the same wave");
    union Lds {
        Fp4Stage<BM, BN> stage[KG][ST];
        struct {
            v16f sums[KG > 1 ? KG - 1 : 1][KG > 1 ? NW : 1][TM * TN][KG > 1 ? 64 : 1];
            alignas(16) uint16_t out[NW][TM * 32 * TN * 32];
        } last;
    };
    __shared__ Lds lds;
    const int l = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5, r = l & 31;
    const int kg = wave / NW, wv = wave % NW;        // (the group of waves, and the wave's place in it)
    // neighbouring workgroups go to different XCDs: each XCD takes a run of tiles, 4 tiles of rows by turns
    const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (t >= mt * nt) return;
    const int band = t / (4 * nt), in = t - band * 4 * nt, bm = min(4, mt - band * 4);
    const int m0 = (band * 4 + in % bm) * BM, n0 = in / bm * BN;
    const int pitch = A.kp / 2, rows = min(BM, A.M - m0), cols = min(BN, A.n - n0);

    // A wave's share of a stage: kLoads instructions, of which a code one brings 8 rows and a scale one 32; rows past the end are
    // zeros. (Where the scales' are fewer than the waves, some waves bring the same.)
    constexpr int kW = BN / 8 / NW, kQ = BM / 8 / NW, kScales = (BM + BN) / 32, kS = (kScales + NW - 1) / NW, kLoads = kW + kQ + kS;
    static_assert(kW > 0 && kQ > 0, "every wave brings rows of both operands");
    const Rsrc wb = buffer_of(A.w + (size_t)n0 * pitch, (uint32_t)cols * pitch);
    const Rsrc qb = buffer_of(A.q + (size_t)m0 * pitch, (uint32_t)rows * pitch);
    uint32_t off[kW + kQ];
#pragma unroll
    for (int i = 0; i < kW + kQ; ++i) {
        const int row = ((i < kW ? i : i - kW) * NW + wv) * 8 + (l >> 3);
        off[i] = (uint32_t)row * pitch + piece_at(row, l & 7) * 16;
    }
    auto load = [&](int b, int i) {
        Fp4Stage<BM, BN>& st = lds.stage[kg][b % ST];
        b = min(b * KG + kg, A.kb - 1);              // (stages after the last are not used)
        if (i < kW) to_lds<16>(st.w + (i * NW + wv) * 1024, wb, off[i], b * 128);
        else if (i < kW + kQ) to_lds<16>(st.q + ((i - kW) * NW + wv) * 1024, qb, off[i], b * 128);
        else {
            const int si = ((i - kW - kQ) * NW + wv) % kScales, sr = si - BN / 32;
            const uint8_t* sw = A.sw + ((size_t)b * A.n + n0) * 8;
            const uint8_t* sq = A.s + (size_t)b * A.s_stage + (size_t)m0 * 8;
            if (si < BN / 32) to_lds<4>(st.sw + si * 256, buffer_of(sw, (uint32_t)cols * 8), si * 256 + l * 4, 0);
            else to_lds<4>(st.sq + sr * 256, buffer_of(sq, (uint32_t)rows * 8), sr * 256 + l * 4, 0);
        }
    };

    const int wm = wv / WN * (BM / WM), wn = wv % WN * (BN / WN);
    v16f acc[TM][TN] = {};
#pragma unroll
    for (int b = 0; b < ST - 1; ++b)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(b, i);
    const int steps = (A.kb + KG - 1) / KG;
    for (int b = 0; b < steps; ++b) {
        // stage b has arrived for every wave (later ones may be under way), and every wave has read stage b - 1
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * kLoads) : "memory");
        auto more = [&](int i0, int i1) {
#pragma unroll
            for (int i = i0; i < i1; ++i) load(b + ST - 1, i);
        };
        if (KG > 1 && b * KG + kg >= A.kb) {         // (the last step)
            more(0, kLoads);
            continue;
        }
        const Fp4Stage<BM, BN>& st = lds.stage[kg][b % ST];
        // (columns behind kp, in the last stage, count for nothing whatever was loaded)
        const int keep = (b * KG + kg + 1) * kFp4Stage > A.kp ? 0xFFFF : -1;
        v4i wf[2][TN], qf[2][TM];
        auto read = [&](int j, int to) {
            const int at = r * 128 + piece_at(r, j * 2 + h) * 16;
#pragma unroll
            for (int i = 0; i < TN; ++i) wf[to][i] = *(const v4i*)(st.w + (wn + i * 32) * 128 + at);
#pragma unroll
            for (int i = 0; i < TM; ++i) qf[to][i] = *(const v4i*)(st.q + (wm + i * 32) * 128 + at);
        };
        int sw[TN], sq[TM];
#pragma unroll
        for (int i = 0; i < TN; ++i) sw[i] = lane_scales(*(const v2i*)(st.sw + (wn + i * 32 + r) * 8), h) & keep;
#pragma unroll
        for (int j = 0; j < TM; ++j) sq[j] = lane_scales(*(const v2i*)(st.sq + (wm + j * 32 + r) * 8), h) & keep;
        read(0, 0);
        four_steps([&](auto step) {
            // under a step's MFMAs the next one's fragments are read, and a part of a later stage's loads issued (behind the
            // reads: the compiler keeps their order)
            constexpr int J = decltype(step)::value, X = J & 1, kEach = (kLoads + 2) / 3;
            if constexpr (J < 3) {
                read(J + 1, X ^ 1);
                more(J * kEach, min((J + 1) * kEach, kLoads));
            }
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int i = 0; i < TN; ++i)
                    acc[j][i] = fp4_mfma<J>(fp4_operand(wf[X][i]), fp4_operand(qf[X][j]), acc[j][i], sw[i], sq[j]);
            // (the MFMAs of a step stay in it: nothing else holds them to their place; in the registers that the compiler chooses)
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    if constexpr (TM * TN > 2) asm volatile("" : "+a"(acc[j][i]));
                    else asm volatile("" : "+v"(acc[j][i]));
                }
        });
    }
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
    // a lane's columns of fragment i: fours at n0 + wn + 32 i + 8 b + 4 h, of row m0 + wm + 32 j + r
    v4f bias[TN][4] = {};
    const Rsrc biases = buffer_of(A.bias, (uint32_t)A.n * 4);
    if (A.bias)
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) bias[i][b] = floats_of(biases, n0 + wn + i * 32 + b * 8 + h * 4);
    auto four = [&](int j, int i, int b) {
        return v4f{acc[j][i][b * 4], acc[j][i][b * 4 + 1], acc[j][i][b * 4 + 2], acc[j][i][b * 4 + 3]} + bias[i][b];
    };
    if constexpr (SILU) {
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int i = 0; i < TN; i += 2) {
                float v[16];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const v4f g = four(j, i, b), u = four(j, i + 1, b);
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[b * 4 + c] = gated(g[c], u[c]);
                }
                silu_block(A, v, m0 + wm + j * 32 + r, (n0 + wn) / 64 + i / 2, h);
            }
        return;
    }
    if (out_dt == 2) {
        // a lane's four columns at once where they are there
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int n = n0 + wn + i * 32 + b * 8 + h * 4, m = m0 + wm + j * 32 + r;
                    const v4f v = four(j, i, b);
                    if (n >= A.n || m >= A.M) continue;
                    float* p = (float*)A.out + (size_t)m * A.out_stride + n;
                    if (n + 4 <= A.n) *(Bytes16At4*)p = __builtin_bit_cast(Bytes16, v);
                    else
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (n + c < A.n) p[c] = v[c];
                }
        return;
    }
    // the wave's outputs [rows][32 TN] through its own part of LDS, so that a lane stores 16 bytes and a row's pieces
    // are next to each other; the pieces of a row in an order that differs from row to row (banks)
    constexpr int kPieces = TN * 4;                  // 16-byte pieces of a row
    uint16_t* o = lds.last.out[wv];
    auto to_out = [&](auto dt) {
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int m = j * 32 + r, piece = (i * 4 + b) ^ (m & (kPieces - 1));
                    *(v4u*)(o + (m * kPieces + piece) * 8 + h * 4) = narrow4<decltype(dt)::value>(four(j, i, b));
                }
    };
    if (out_dt == 0) to_out(std::integral_constant<int, 0>());
    else to_out(std::integral_constant<int, 1>());
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < TM * 32 * kPieces / 64; ++k) {
        const int at = k * 64 + l, row = at / kPieces, piece = at % kPieces;
        const int m = m0 + wm + row, n = n0 + wn + piece * 8;
        if (m >= A.M || n >= A.n) continue;
        const v8u v = *(const v8u*)(o + (row * kPieces + (piece ^ (row & (kPieces - 1)))) * 8);
        uint16_t* p = (uint16_t*)A.out + (size_t)m * A.out_stride + n;
        if (n + 8 <= A.n) *(Bytes16At2*)p = __builtin_bit_cast(Bytes16, v);
        else
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (n + c < A.n) p[c] = v[c];
    }
}

template <bool SILU, int BM, int BN, int WM, int WN, int KG, int ST>
void launch_fp4_tiles(const Fp4ProductArgs& a, int out_dt, hipStream_t st) {
    const int mt = (a.M - 1) / BM + 1, nt = (a.n - 1) / BN + 1, per = (int)(((int64_t)mt * nt + 7) / 8);
    hipLaunchKernelGGL((fp4_tile_kernel<SILU, BM, BN, WM, WN, KG, ST>), dim3((unsigned)per * 8), dim3(64 * WM * WN * KG), 0,
                       st, a, mt, nt, per, out_dt);
}

}  // namespace exl3
