// Which kernel computes a 4-bit float product: fp4_few.hip's, a tile of fp4_tiles.cuh or fp4_tile256.hip's.
//
// What takes the time is what a CU has to bring in (fp8_linear.hip has the rates): BM + BN rows of k for each tile. The tile is
// the one for which that is least, max(1, tiles / 256 CUs) (BM + BN), the larger one where two are equal, but for these: 128 x 64
// only where each CU has one at most; 128 x 128 with more than one counts by the tile, since two share a CU; 256 x 256, whose
// rounds are whole, costs a fifth more, and for a gate|up product is for four stages of k at least: silu and the rows' conversion,
// with no products beside them, are as much work as fewer stages' products. MLPs of 8,192 rows out of a graph, both forms on one
// card, us with gate|up in tiles of 128 x 128 and of 256 x 256: 512 -> 2 x 1024 26.0 and 29.1, 768 -> 2 x 2048 50.0 and 54.5.
// Plain products take them with fewer stages too:
//   rows, k -> n   4,096, 128 -> 4096   8,192, 256 -> 2048   8,192, 512 -> 2048   2,048, 512 -> 12,288   8,192, 768 -> 12,288
//   128 x 128                    12.9                 11.9                 13.6                   19.7                   88.7
//   256 x 256                    10.9                 11.1                 12.8                   19.3                   64.3
//
// Quantised rows, bf16 outputs, weights from HBM, us per call out of a graph; * is what the rule takes.
//   4096 -> 2048, rows  100   200   400   777  1,024  1,500  2,048  4,096  8,192
//   32 x 32             6.3*  7.0  11.9  20.8   22.6   32.1   42.6   83.2  163.7
//   64 x 64             7.0   7.0*  7.4* 11.1   11.7   18.5   21.0   39.2   76.1
//   128 x 64            8.8   8.9   9.2   9.5*   9.9*  17.0   18.7   33.4   65.6
//   128 x 128          11.2  11.3  11.6  11.9   12.1   12.7*  14.1*  23.5*  43.1
//   256 x 256          26.2  26.6  26.6  25.4   25.5   29.2   25.9   28.1   38.1*
//   2048 -> 12,288
//   32 x 32            15.1  25.4  40.7  71.2   98.4  130.9  181.3  346.6  677.1
//   64 x 64             9.4  14.5  21.6  32.7   42.6   55.1   82.3  146.4  273.3
//   128 x 64            7.8* 12.8  18.0  32.8   35.3   46.4   70.0  143.3  249.2
//   128 x 128           9.4  10.1* 15.7* 26.6   27.6   35.2*  46.3   89.8  159.3
//   256 x 256          21.1  21.8  21.8  20.8*  22.1*  40.2   40.8*  65.8* 120.7*
//
// Few rows (fp4_few.hip) cost by what a workgroup brings in too, 14 for each 16 columns and 1 for each row (5 where it quantises
// them), and 10 for each further fragment of columns, which leaves fewer waves to load. They take that kernel up to a cost of
// 50, and up to 48 rows where that is three quarters of the tile's at most (4096 -> 2048: 64 rows, cost 46, 5.9 us, in tiles 6.3;
// 100 rows, cost 63, 6.7 and 6.3; 2048 -> 12,288: 32 rows, cost 94 and 128, 6.8 and 7.3). 12 rows and fewer are quantised inside
// (2048 -> 12,288: 12 rows 8.1 us, by a launch before it 8.6; 16 rows 9.9 and 9.1).
//
// A gate|up product of more rows than those 12 takes a tile by the same rule, with 32 x 64 ones where it says 32 x 32 (a wave has a
// gate and its up). They are counted as 32 x 32, which takes 64 x 64 for some calls of one round of 32 x 64: MLP of 300 rows 2048
// -> 2 x 512 -> 2048 14.4 us, with gate|up in 32 x 64 13.3; of 300 rows 512 -> 2 x 512 -> 512 11.3 and 11.8.
#include "fp4_tiles.cuh"

namespace exl3 {

void launch_fp4_few(const Fp4ProductArgs& a, int tn, int R, int out_dt, hipStream_t st);
void launch_fp4_tiles256(const Fp4ProductArgs& a, bool silu, int out_dt, hipStream_t st);

namespace {

enum { kFp4Tile32, kFp4Tile64, kFp4Tile128x64, kFp4Tile128, kFp4Tile256 };

struct Pick {
    int tile;
    bool few;                                        // at most one workgroup per CU
    int64_t cost;
};
Pick pick_tile(int M, int n, int kb, bool silu) {
    constexpr int kSizes[][2] = {{32, 32}, {64, 64}, {128, 64}, {128, 128}, {256, 256}};
    Pick best{kFp4Tile256, false, 0};
    for (int i = kFp4Tile32; i <= kFp4Tile256; ++i) {
        const int64_t tiles = (int64_t)((M - 1) / kSizes[i][0] + 1) * ((n - 1) / kSizes[i][1] + 1);
        const int64_t rounds = (tiles + kCus - 1) / kCus;
        const int rows = kSizes[i][0] + kSizes[i][1];
        int64_t cost = rounds * rows;
        if (i == kFp4Tile128x64 && rounds > 1) continue;
        if (i == kFp4Tile128 && rounds > 1) cost = tiles * rows / kCus;
        if (i == kFp4Tile256 && silu && kb < 4 && best.cost) continue;
        if (i == kFp4Tile256) cost = rounds * (rows + rows / 5);
        else if ((tiles + 7) * 512 >= kMaxThreads) continue;
        if (!best.cost || cost <= best.cost) best = {i, rounds == 1, cost};
    }
    return best;
}

// The few-rows kernel's tile: tn fragments of 16 columns and R rows to a workgroup (tn 0: it cannot take the call)
struct FewTile {
    int tn, R;
    int64_t cost;
};
FewTile pick_few(int M, int n, bool own) {
    FewTile best{};
    for (int tn = 1; tn <= 3; ++tn)
        for (int groups = 1; groups <= 4 && groups <= M; groups *= 2) {
            const int R = (M + groups - 1) / groups;
            const int64_t workgroups = (int64_t)((n - 1) / (16 * tn) + 1) * ((M - 1) / R + 1);
            const int64_t rounds = (workgroups + kCus - 1) / kCus;
            if (R > (own ? 16 : 48) || (workgroups + 7) * 1024 >= kMaxThreads) continue;
            const int64_t cost = rounds * (14 * tn + (own ? 5 * R : R)) + (own ? 0 : 10 * (tn - 1));
            if (!best.tn || cost < best.cost) best = {tn, R, cost};
        }
    return best;
}

constexpr int kOwnRows = 12;

template <bool SILU>
void launch_tile(const Pick& p, const Fp4ProductArgs& a, int out_dt, hipStream_t st) {
    if (p.tile == kFp4Tile256) return launch_fp4_tiles256(a, SILU, out_dt, st);
    if constexpr (SILU) {                            // (a wave has 64 columns)
        if (p.tile == kFp4Tile32) launch_fp4_tiles<true, 32, 64, 1, 1, 4, 2>(a, out_dt, st);
        else if (p.tile == kFp4Tile64) launch_fp4_tiles<true, 64, 64, 2, 1, 2, 2>(a, out_dt, st);
        else if (p.tile == kFp4Tile128x64) launch_fp4_tiles<true, 128, 64, 4, 1, 1, 4>(a, out_dt, st);
        else if (p.few) launch_fp4_tiles<true, 128, 128, 2, 2, 1, 4>(a, out_dt, st);
        else launch_fp4_tiles<true, 128, 128, 2, 2, 1, 2>(a, out_dt, st);
    } else {
        if (p.tile == kFp4Tile32) launch_fp4_tiles<false, 32, 32, 1, 1, 4, 2>(a, out_dt, st);
        else if (p.tile == kFp4Tile64 && p.few && a.kb > 4) launch_fp4_tiles<false, 64, 64, 2, 2, 2, 4>(a, out_dt, st);
        else if (p.tile == kFp4Tile64) launch_fp4_tiles<false, 64, 64, 2, 2, 2, 2>(a, out_dt, st);
        else if (p.tile == kFp4Tile128x64) launch_fp4_tiles<false, 128, 64, 4, 2, 1, 4>(a, out_dt, st);
        else if (p.few) launch_fp4_tiles<false, 128, 128, 2, 4, 1, 4>(a, out_dt, st);
        else launch_fp4_tiles<false, 128, 128, 2, 2, 1, 2>(a, out_dt, st);
    }
}

}  // namespace

bool fp4_product_quantises(int M) { return M <= kOwnRows; }

hipError_t launch_fp4_product(const Fp4ProductArgs& a, int out_dt, hipStream_t st) {
    const FewTile f = pick_few(a.M, a.n, !a.q);
    const Pick p = pick_tile(a.M, a.n, a.kb, false);
    const bool few = f.tn && (f.cost <= 50 || (a.M <= 48 && f.cost * 4 <= p.cost * 3));
    if (!a.q || a.M <= kOwnRows || few) launch_fp4_few(a, f.tn, f.R, out_dt, st);
    else launch_tile<false>(p, a, out_dt, st);
    return hipGetLastError();
}

bool fp4_gate_up_in_tiles(int M) { return M > kOwnRows; }

hipError_t launch_fp4_gate_up(const Fp4ProductArgs& a, hipStream_t st) {
    launch_tile<true>(pick_tile(a.M, a.n, a.kb, true), a, 2, st);
    return hipGetLastError();
}

}  // namespace exl3
