// The 8-bit float product on e4m3 MFMAs, with fp16 and bf16 outputs: the tiles of fp8_tiles.cuh and the largest one.
#include "fp8_tiles.cuh"

namespace exl3 {

// ---- 256 x 256 tiles, one after the other ---------------------------------------------------------------------------------
// For the large products: as many workgroups as CUs, each with every 32nd tile of its XCD's run (its 32 CUs have neighbouring
// ones at a time). A block's loads are issued while the block before is multiplied, the next tile's first among them, so that
// they are on their way while this tile's outputs are stored. 8,192 rows, 2048 -> 12,288, kernel trace: 217 us at the median, 181
// to 234 (1.9 PFLOP/s, 1.8-2.3), as the power allows. MFMAs alone reach 4.6 (4.3 with the scales' multiply-adds); they are at work
// 69 % of a wave's time, at the 1.95 GHz that the power leaves.
__global__ void __launch_bounds__(512) fp8_tile256_kernel(Fp8ProductArgs A, int mt, int nt, int per, int out_dt) {
    constexpr int B = 256, WM = 2, WN = 4, NW = WM * WN, TM = B / WM / 16, TN = B / WN / 16, kPieces = TN * 2;
    // (one variable: where there are two the compiler tells their accesses apart, and waits for all loads to LDS before it
    // reads any)
    struct Lds {
        Stage<B, B> stage[2];
        alignas(16) uint16_t outs[NW][16 * TN * 16]; // 16 rows of a wave's outputs
    };
    static_assert(alignof(Lds) >= 16);
    __shared__ Lds lds;
    const int l = lane_id(), wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = l >> 4, r = l & 15;
    const int first = (blockIdx.x & 7) * per, step = gridDim.x >> 3, end = min(first + per, mt * nt);
    int t = first + (blockIdx.x >> 3);
    if (t >= end) return;
    const int kp = A.kb * kFp8Block;

    constexpr int kW = B / 8 / NW, kLoads = 2 * kW + 1;
    uint32_t off[kW];                                // (the same for the weights and the rows)
#pragma unroll
    for (int i = 0; i < kW; ++i) {
        const int row = (i * NW + wv) * 8 + (l >> 3);
        off[i] = (uint32_t)row * kp + piece_at(row, l & 7) * 16;
    }
    const bool rows_scales = wv < B / 64;            // waves that bring 64 row scales each; the others bring the weights' two
    const uint32_t s_off = (uint32_t)(rows_scales ? wv * 64 + l : l & 1) * A.kb * 4;
    struct Tile {
        int m0, n0;
        Rsrc wb, qb, sb;
    };
    auto tile_at = [&](int i) {                      // (4 tiles of rows by turns)
        const int band = i / (4 * nt), in = i - band * 4 * nt, bm = min(4, mt - band * 4);
        const int m0 = (band * 4 + in % bm) * B, n0 = in / bm * B, rows = min(B, A.M - m0), cols = min(B, A.n - n0);
        return Tile{m0, n0, buffer_of(A.w + (size_t)n0 * kp, (uint32_t)cols * kp),
                    buffer_of(A.q + (size_t)m0 * kp, (uint32_t)rows * kp),
                    rows_scales ? buffer_of(A.s + (size_t)m0 * A.kb, (uint32_t)rows * A.kb * 4)
                                : buffer_of(A.sw + (size_t)(n0 / kFp8Block) * A.kb, (uint32_t)fp8_blocks(cols) * A.kb * 4)};
    };
    auto load = [&](Stage<B, B>& st, const Tile& of, int b, int i) {
        if (i < kW) to_lds<16>(st.w + (i * NW + wv) * 1024, of.wb, off[i], b * kFp8Block);
        else if (i < kLoads - 1) to_lds<16>(st.q + ((i - kW) * NW + wv) * 1024, of.qb, off[i - kW], b * kFp8Block);
        else to_lds<4>(rows_scales ? st.s + wv * 64 : st.sw, of.sb, s_off, b * 4);
    };

    const int wm = wv / WN * (B / WM), wn = wv % WN * (B / WN);
    const int at0 = r * 128 + piece_at(r, g) * 16, at1 = r * 128 + piece_at(r, g + 4) * 16;
    auto frag = [&](const uint8_t* p) { return frag_of<false>(*(const v4i*)(p + at0), *(const v4i*)(p + at1)); };
    Tile tile = tile_at(t);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(lds.stage[0], tile, 0, i);
    int at = 0;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    while (true) {
        const bool more = t + step < end;
        const Tile next = more ? tile_at(t + step) : tile;
        v4f acc[TM][TN] = {};
        v4f x[2][TN] = {};                           // a fragment's block sums, and the scale that awaits them
        float sc[2] = {};
        auto add = [&](int j) {
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[j][i][c] = __builtin_fmaf(x[j & 1][i][c], sc[j & 1], acc[j][i][c]);
        };
        for (int b = 0; b < A.kb; ++b) {
            // the block has arrived for every wave (each waited for its loads), and every wave has read the one before
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            const Stage<B, B>& st = lds.stage[at];
            at ^= 1;
            const bool last = b + 1 == A.kb;
            const Tile& from = last ? next : tile;
            const int nb = !last ? b + 1 : more ? 0 : b;     // (the block after the last one is not used)
            const float sw = st.sw[wn / kFp8Block];
            constexpr int kEach = (kLoads + TM - 2) / (TM - 1);
            Frag<false> qf[2], wf[TN];
            qf[0] = frag(st.q + wm * 128);
#pragma unroll
            for (int i = 0; i < TN; ++i) wf[i] = frag(st.w + (wn + i * 16) * 128);
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                // under this fragment's MFMAs the next one is read and the last one's sums are scaled (at j = 0 those of
                // the block before)
#pragma unroll
                for (int i = j * kEach; i < min((j + 1) * kEach, kLoads); ++i) load(lds.stage[at], from, nb, i);
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
            if (!last) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        add(TM - 1);
        int e = l;                                   // (kept from being computed with before the loop: registers)
        asm volatile("" : "+v"(e));
        const int r = e & 15, g = e >> 4;
        v4f bias[TN] = {};
        if (A.bias)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int n = tile.n0 + wn + i * 16 + g * 4 + c;
                    bias[i][c] = n < A.n ? A.bias[n] : 0.0f;
                }
        // 16 rows at a time through the wave's part of LDS (its reads and writes there are in order)
        uint16_t* o = lds.outs[wv];
        const bool whole = tile.m0 + B <= A.M && tile.n0 + B <= A.n, wide = A.out_stride % 8 == 0 && (uintptr_t)A.out % 16 == 0;
        const bool plain = whole && wide;
        auto store = [&](auto dt, auto full) {
#pragma unroll
            for (int j = 0; j < TM; ++j) {
#pragma unroll
                for (int i = 0; i < TN; ++i)
                    *(v4u*)(o + (r * kPieces + ((i * 2 + (g >> 1)) ^ (r & (kPieces - 1)))) * 8 + (g & 1) * 4) =
                        narrow4<decltype(dt)::value>(acc[j][i] + bias[i]);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int row = k * 8 + (e >> 3), piece = e & 7;
                    const int m = tile.m0 + wm + j * 16 + row, n = tile.n0 + wn + piece * 8;
                    const v8u v = *(const v8u*)(o + (row * kPieces + (piece ^ (row & (kPieces - 1)))) * 8);
                    uint16_t* p = (uint16_t*)A.out + (size_t)m * A.out_stride + n;
                    if constexpr (decltype(full)::value) {
                        // (past the caches: 178 us against 185 in one run, 8,192 rows, 2048 -> 12,288)
                        __builtin_nontemporal_store(v, (v8u*)p);
                    } else if (m < A.M && n < A.n) {
                        if (wide && n + 8 <= A.n) *(v8u*)p = v;
                        else
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                if (n + c < A.n) p[c] = v[c];
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        };
        if (out_dt == 0 && plain) store(std::integral_constant<int, 0>(), std::true_type());
        else if (out_dt == 0) store(std::integral_constant<int, 0>(), std::false_type());
        else if (plain) store(std::integral_constant<int, 1>(), std::true_type());
        else store(std::integral_constant<int, 1>(), std::false_type());
        if (!more) break;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // (the next tile's first block)
        t += step;
        tile = next;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // (no load to LDS may outlive the workgroup)
}

void launch_fp8_tiles256(const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    const int mt = (a.M - 1) / 256 + 1, nt = (a.n - 1) / 256 + 1, per = (int)(((int64_t)mt * nt + 7) / 8);
    hipLaunchKernelGGL(fp8_tile256_kernel, dim3((unsigned)(per < kCus / 8 ? per : kCus / 8) * 8), dim3(512), 0, st, a, mt, nt,
                       per, out_dt);
}

void launch_fp8_tile_e4m3(int tile, bool few, const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    if (tile == kTile256) launch_fp8_tiles256(a, out_dt, st);
    else launch_fp8_tile<false>(tile, few, a, out_dt, st);
}

}  // namespace exl3
