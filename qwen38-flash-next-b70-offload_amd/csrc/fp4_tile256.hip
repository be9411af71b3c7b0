// The 4-bit float product in tiles of 256 x 256 (fp4_tiles.cuh has the definition), for the large ones: as many workgroups as
// CUs, each with every 32nd tile of its XCD's run (its 32 CUs have neighbouring ones at a time).
//
// Four waves of 128 x 128, one to a SIMD: the fragments that they read from LDS per MFMA are the fewest (32 KB a step of 64
// columns, 256 of its 512 cycles; as 8 waves of 128 x 64 48 KB, and with the loads' writes LDS would be the bound). A wave has no
// other to hide behind, so everything is a step ahead of its use: a step's fragments are read under the MFMAs of the step before,
// the first ones of a stage under the last step of the stage before, and a stage's loads to LDS are issued as soon as the stage
// two before it has been read. The next tile's first stages are on their way while this tile's outputs are stored.
//
// 8,192 rows, 2048 -> 12,288: 118 to 123 us (3.4-3.5 PFLOP/s; with rows and weights of zeros 97, so 20 % of it is the power that
// random codes draw: MFMAs alone reach 6.4 to 6.6 PFLOP/s with them, 8.8 to 9.6 with zeros). About 42 us of it are the 201 MB of
// outputs, which all CUs store at the same time; a stage of 256 columns takes 1.6 us, 0.85 of them MFMAs at the full clock. 8,192
// columns: 357 us, 4.6 PFLOP/s. Measured and not kept: half of a tile's outputs held in registers and stored under the next
// tile's products (129 us for 123: the wait for a stage's loads waits for the stores before them too; with waits that leave the
// stores out 143, as the registers that they wait in cost others), starts at different times (130 for 134). Rows of outputs that
// start at any element (12,287 columns) 142 us, 260 with their elements stored one by one.
#include "fp4_tiles.cuh"

namespace exl3 {

template <bool SILU, bool BIAS>
__global__ void __launch_bounds__(256, 1) fp4_tile256_kernel(Fp4ProductArgs A, int mt, int nt, int per, int out_dt) {
    constexpr int B = 256, NW = 4, T = 4, kCode = B / 8 / NW, kScale = 2 * B / 32 / NW, kLoads = 2 * kCode + kScale;
    // (one variable: where there are two the compiler tells their accesses apart, and waits for all loads to LDS before it
    // reads any)
    struct Lds {
        Fp4Stage<B, B> stage[2];
        alignas(16) uint8_t outs[NW][4096];          // 32 rows of 128 bytes of a wave's outputs
    };
    __shared__ Lds lds;
    const int l = lane_id(), wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5, r = l & 31;
    const int first = (blockIdx.x & 7) * per, step = gridDim.x >> 3, end = min(first + per, mt * nt);
    int t = first + (blockIdx.x >> 3);
    if (t >= end) return;
    const int pitch = A.kp / 2;

    // a stage's loads: those of the step after it is free, of the next stage's first step and of its second one
    constexpr int kPart[4] = {0, 7, 14, kLoads};
    uint32_t off[kCode];                             // (the same for the weights and the rows)
#pragma unroll
    for (int i = 0; i < kCode; ++i) {
        const int row = (i * NW + wv) * 8 + (l >> 3);
        off[i] = (uint32_t)row * pitch + piece_at(row, l & 7) * 16;
    }
    struct Tile {
        int m0, n0, rows, cols;
        Rsrc wb, qb;
    };
    auto tile_at = [&](int i) {                      // (4 tiles of rows by turns)
        const int band = i / (4 * nt), in = i - band * 4 * nt, bm = min(4, mt - band * 4);
        const int m0 = (band * 4 + in % bm) * B, n0 = in / bm * B, rows = min(B, A.M - m0), cols = min(B, A.n - n0);
        return Tile{m0, n0, rows, cols, buffer_of(A.w + (size_t)n0 * pitch, (uint32_t)cols * pitch),
                    buffer_of(A.q + (size_t)m0 * pitch, (uint32_t)rows * pitch)};
    };
    auto load = [&](Fp4Stage<B, B>& st, const Tile& of, int b, int i) {
        if (i < kCode) to_lds<16>(st.w + (i * NW + wv) * 1024, of.wb, off[i], b * 128);
        else if (i < 2 * kCode) to_lds<16>(st.q + ((i - kCode) * NW + wv) * 1024, of.qb, off[i - kCode], b * 128);
        else {
            // (the first two of a wave's four are the weights')
            const int j = i - 2 * kCode, si = (j & 1) * NW + wv;
            const uint8_t* sw = A.sw + ((size_t)b * A.n + of.n0) * 8;
            const uint8_t* sq = A.s + (size_t)b * A.s_stage + (size_t)of.m0 * 8;
            if (j < 2) to_lds<4>(st.sw + si * 256, buffer_of(sw, (uint32_t)of.cols * 8), si * 256 + l * 4, 0);
            else to_lds<4>(st.sq + si * 256, buffer_of(sq, (uint32_t)of.rows * 8), si * 256 + l * 4, 0);
        }
    };

    const int wm = wv / 2 * 128, wn = wv % 2 * 128;
    int at[4];                                       // of a row's piece of step j, from the fragment's first row on
#pragma unroll
    for (int j = 0; j < 4; ++j) at[j] = r * 128 + piece_at(r, j * 2 + h) * 16;
    v4i wf[2][T], qf[2][T];
    int sw[2][T], sq[2][T];
    auto read_w = [&](const Fp4Stage<B, B>& st, int j, int i, int to) {
        wf[to][i] = *(const v4i*)(st.w + (wn + i * 32) * 128 + at[j]);
    };
    auto read_q = [&](const Fp4Stage<B, B>& st, int j, int i, int to) {
        qf[to][i] = *(const v4i*)(st.q + (wm + i * 32) * 128 + at[j]);
    };
    auto read_scales = [&](const Fp4Stage<B, B>& st, int keep, int to) {
#pragma unroll
        for (int i = 0; i < T; ++i) {
            sw[to][i] = lane_scales(*(const v2i*)(st.sw + (wn + i * 32 + r) * 8), h) & keep;
            sq[to][i] = lane_scales(*(const v2i*)(st.sq + (wm + i * 32 + r) * 8), h) & keep;
        }
    };
    // columns behind kp, in the last stage, count for nothing whatever was loaded
    auto kept = [&](int b) { return (b + 1) * kFp4Stage > A.kp ? 0xFFFF : -1; };

    // the stages of this workgroup's tiles, one after the other: `tile`, b the one that is multiplied, `far`, fb two further on
    Tile tile = tile_at(t), far = tile;
    int ft = t, fb = 0;
    auto advance = [&] {                             // (after the last stage it stays there: loaded again, and not used)
        if (fb + 1 < A.kb) ++fb;
        else if (ft + step < end) {
            ft += step;
            far = tile_at(ft);
            fb = 0;
        }
    };
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(lds.stage[0], far, fb, i);
    advance();
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < kPart[1]; ++i) load(lds.stage[1], far, fb, i);
#pragma unroll
    for (int i = 0; i < T; ++i) {
        read_w(lds.stage[0], 0, i, 0);
        read_q(lds.stage[0], 0, i, 0);
    }
    read_scales(lds.stage[0], kept(0), 0);
    int cur = 0;
    while (true) {
        v16f acc[T][T] = {};
        for (int b = 0; b < A.kb; ++b) {
            Fp4Stage<B, B>& st = lds.stage[cur];
            Fp4Stage<B, B>& next = lds.stage[cur ^ 1];
            const int keep = kept(b + 1 < A.kb ? b + 1 : 0);
            four_steps([&](auto j) {
                constexpr int J = decltype(j)::value, X = J & 1;
                // the next stage has arrived for every wave, and every wave has read this one
                if constexpr (J == 3) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
                for (int i = 0; i < T; ++i) {
                    read_w(J == 3 ? next : st, (J + 1) & 3, i, X ^ 1);
                    read_q(J == 3 ? next : st, (J + 1) & 3, i, X ^ 1);
                }
                if constexpr (J == 3) read_scales(next, keep, 1);
                // (the loads behind the reads: the compiler keeps their order)
                if constexpr (J == 2) advance();
                else
#pragma unroll
                    for (int i = kPart[(J + 1) & 3]; i < kPart[((J + 1) & 3) + 1]; ++i) load(J == 3 ? st : next, far, fb, i);
#pragma unroll
                for (int jm = 0; jm < T; ++jm)
#pragma unroll
                    for (int i = 0; i < T; ++i)
                        acc[jm][i] = fp4_mfma<J>(fp4_operand(wf[X][i]), fp4_operand(qf[X][jm]), acc[jm][i], sw[0][i], sq[0][jm]);
#pragma unroll
                for (int i = 0; i < T * T / 2; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, J == 3 ? 2 : 1, 0);
                }
#pragma unroll
                for (int i = 0; i < T * T / 2; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    if constexpr (J != 2) __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
                }
                // (the MFMAs of a step stay in it: nothing else holds them to their place)
#pragma unroll
                for (int jm = 0; jm < T; ++jm)
#pragma unroll
                    for (int i = 0; i < T; ++i) asm volatile("" : "+a"(acc[jm][i]));
            });
#pragma unroll
            for (int i = 0; i < T; ++i) sw[0][i] = sw[1][i], sq[0][i] = sq[1][i];
            cur ^= 1;
        }
        int e = l;                                   // (kept from being computed with before the loop: registers)
        asm volatile("" : "+v"(e));
        const int eh = e >> 5, er = e & 31;
        v4f bias[T][4];
        if constexpr (BIAS) {
            const Rsrc biases = buffer_of(A.bias, (uint32_t)A.n * 4);
#pragma unroll
            for (int i = 0; i < T; ++i)
#pragma unroll
                for (int b = 0; b < 4; ++b) bias[i][b] = floats_of(biases, tile.n0 + wn + i * 32 + b * 8 + eh * 4);
        }
        auto four = [&](int j, int i, int b) {
            const v4f v = {acc[j][i][b * 4], acc[j][i][b * 4 + 1], acc[j][i][b * 4 + 2], acc[j][i][b * 4 + 3]};
            if constexpr (BIAS) return v + bias[i][b];
            else return v;
        };
        // (a fragment stays in accumulation registers until its turn: moved out at once, they would not fit the others)
        auto hold = [&](int j, int i) { asm volatile("" : "+a"(acc[j][i])); };
        if constexpr (SILU) {
#pragma unroll
            for (int j = 0; j < T; ++j)
#pragma unroll
                for (int i = 0; i < T; i += 2) {
                    hold(j, i);
                    hold(j, i + 1);
                    float v[16];
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const v4f g = four(j, i, b), u = four(j, i + 1, b);
#pragma unroll
                        for (int c = 0; c < 4; ++c) v[b * 4 + c] = gated(g[c], u[c]);
                    }
                    silu_block(A, v, tile.m0 + wm + j * 32 + er, (tile.n0 + wn) / 64 + i / 2, eh);
                }
        } else {
            // 32 rows of 128 bytes at a time through the wave's part of LDS (its reads and writes there are in order), the 8 pieces
            // of a row in an order that differs from row to row (banks)
            uint8_t* o = lds.outs[wv];
            const int size = out_dt == 2 ? 4 : 2, each = 16 / size;
            const bool plain = A.out_stride % each == 0 && (uintptr_t)A.out % 16 == 0 && tile.rows == B && tile.cols == B;
            auto store = [&](int j, int n, auto full) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int row = k * 8 + (e >> 3), piece = e & 7, m = tile.m0 + wm + j * 32 + row;
                    const v4i v = *(const v4i*)(o + row * 128 + (piece ^ (row & 7)) * 16);
                    const int c = n + piece * each;
                    uint8_t* p = (uint8_t*)A.out + ((size_t)m * A.out_stride + c) * size;
                    if constexpr (decltype(full)::value) __builtin_nontemporal_store(v, (v4i*)p);
                    else if (m < A.M && c < A.n) {
                        if (c + each <= A.n) *(Bytes16At2*)p = __builtin_bit_cast(Bytes16, v);
                        else if (size == 4) {
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                if (c + x < A.n) ((int*)p)[x] = v[x];
                        } else {
                            const v8u u = __builtin_bit_cast(v8u, v);
#pragma unroll
                            for (int x = 0; x < 8; ++x)
                                if (c + x < A.n) ((uint16_t*)p)[x] = u[x];
                        }
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            };
            auto outs = [&](auto dt, auto full) {
                constexpr int DT = decltype(dt)::value;
#pragma unroll
                for (int j = 0; j < T; ++j)
                    if constexpr (DT == 2) {
#pragma unroll
                        for (int i = 0; i < T; ++i) {
                            hold(j, i);
#pragma unroll
                            for (int b = 0; b < 4; ++b) *(v4f*)(o + er * 128 + ((b * 2 + eh) ^ (er & 7)) * 16) = four(j, i, b);
                            store(j, tile.n0 + wn + i * 32, full);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < T; i += 2) {
                            hold(j, i);
                            hold(j, i + 1);
#pragma unroll
                            for (int b = 0; b < 8; ++b)
                                *(v4u*)(o + er * 128 + (b ^ (er & 7)) * 16 + eh * 8) = narrow4<DT>(four(j, i + b / 4, b & 3));
                            store(j, tile.n0 + wn + i * 32, full);
                        }
                    }
            };
            auto by_dt = [&](auto full) {
                if (out_dt == 0) outs(std::integral_constant<int, 0>(), full);
                else if (out_dt == 1) outs(std::integral_constant<int, 1>(), full);
                else outs(std::integral_constant<int, 2>(), full);
            };
            if (plain) by_dt(std::true_type());
            else by_dt(std::false_type());
        }
        t += step;
        if (t >= end) break;
        tile = tile_at(t);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // (no load to LDS may outlive the workgroup)
}

void launch_fp4_tiles256(const Fp4ProductArgs& a, bool silu, int out_dt, hipStream_t st) {
    const int mt = (a.M - 1) / 256 + 1, nt = (a.n - 1) / 256 + 1, per = (int)(((int64_t)mt * nt + 7) / 8);
    const dim3 grid((unsigned)(per < kCus / 8 ? per : kCus / 8) * 8);
    // (biases are a kernel of their own: the additions alone take 1.5 us a tile)
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a, mt, nt, per, out_dt); };
    if (silu) a.bias ? launch(fp4_tile256_kernel<true, true>) : launch(fp4_tile256_kernel<true, false>);
    else a.bias ? launch(fp4_tile256_kernel<false, true>) : launch(fp4_tile256_kernel<false, false>);
}

}  // namespace exl3
