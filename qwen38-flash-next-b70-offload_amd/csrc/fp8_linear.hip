// Which tile computes an 8-bit float product (fp8_tiles.cuh has the kernel).
//
// A tile of BM rows x BN columns brings (BM + BN) 128 bytes to its CU per block of k, and a CU takes them in at 60-70 GB/s
// whatever the tile (512 KB of a 64 x 64 tile at k 4096: 8.8 us; 256 KB of a 32 x 32 one: 4.0 us): what a CU has to bring in
// is what takes the time, and the tile is the one for which that is least,
//
//     max(1, tiles / 256 CUs) (BM + BN)
//
// the smaller one where two are equal, but for these, since a CU with one tile has its LDS for more stages (us, weights from HBM):
// 16 x 16 and, of more than 16 rows, 16 x 32 only where each CU has one at most (4096 -> 2048, 40 rows 7.7, 16 x 32 6.9; 80 rows
// 10.0, 32 x 32 7.9), 64 x 64 only so where 128 x 64 is (700 rows 20.4, 128 x 64 17.1), and that only so and without exact sums
// (1,100 rows 27.8, 128 x 128 20.8; 1,024 rows, exact 26.0, 64 x 64 25.4).
//
// 4096 -> 2048, weights from HBM, us: 16 rows 6.6 and 32 rows 6.5 (16 x 16), 64 rows 7.2 (16 x 32), 128 rows 8.6 and 256 rows 12.1
// (32 x 32), 700 rows 17.1 (128 x 64), 1,500 rows 25.0 (128 x 128). Every tile at every size, in an earlier form with fewer stages,
// weights in the caches, us for 16 / 64 / 128 / 512 / 2,048 rows: 16 x 16 4.0 / 5.5 / 10.2 / - / -, 16 x 32 5.1 / 5.4 / 8.2 / - / -,
// 32 x 32 6.0 / 6.4 / 6.6 / 17.3 / -, 64 x 64 9.3 / 9.6 / 9.6 / 11.3 / 34, 128 x 128 17 / 18 / 18 / 22 / 27, 256 x 256 40 / 40 / 41 /
// 43 / 45.
#include "exl3_kernels.h"

namespace exl3 {

void launch_fp8_tile_e4m3(int tile, bool few, const Fp8ProductArgs& a, int out_dt, hipStream_t st);
void launch_fp8_tile_exact(int tile, bool few, const Fp8ProductArgs& a, int out_dt, hipStream_t st);

namespace {

struct Pick {
    int tile;
    bool few;                                        // at most one workgroup per CU
};
Pick pick_tile(int M, int n, int largest, bool exact) {
    constexpr int kSizes[][2] = {{16, 16}, {16, 32}, {32, 32}, {64, 64}, {128, 64}, {128, 128}, {256, 256}};
    auto tiles_of = [&](int i) { return (int64_t)((M - 1) / kSizes[i][0] + 1) * ((n - 1) / kSizes[i][1] + 1); };
    const bool one_128x64 = !exact && tiles_of(kTile128x64) <= kCus;
    Pick best{};
    int64_t least = 0;
    for (int i = 0; i <= largest; ++i) {
        const int64_t tiles = tiles_of(i), bytes = (tiles > kCus ? tiles : kCus) * (kSizes[i][0] + kSizes[i][1]);
        if (tiles > kCus && (i == kTile16 || (i == kTile16x32 && M > 16) || (i == kTile64 && one_128x64))) continue;
        if (i == kTile128x64 && !one_128x64) continue;
        // (of up to 512 threads, in eighths; the callers' limit is that of the largest)
        if (i < largest && (tiles + 7) * 512 >= kMaxThreads) continue;
        if (least == 0 || bytes < least) least = bytes, best = {i, tiles <= kCus};
    }
    return best;
}

}  // namespace

// As many blocks of 128 as the workgroup has in hand at once (4 for each 16 lanes of up to 512 threads at 16 columns, of 256 at
// 32). More rows are quantised by a launch of their own: 2048 -> 1024, 8 rows 5.1 us, by two launches 6.1; 4096 -> 2048, 8 rows
// 8.0 us, by two launches 7.4.
bool fp8_product_quantises(int M, int k, int n) {
    return M <= 16 && (int64_t)M * fp8_blocks(k) <= (pick_tile(M, n, kTile16x32, false).tile == kTile16 ? 128 : 64);
}

hipError_t launch_fp8_product(const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    const bool exact = a.exact || out_dt == 2;
    const Pick p = pick_tile(a.M, a.n, !a.q ? kTile16x32 : exact ? kTile128 : kTile256, exact);
    if (exact) launch_fp8_tile_exact(p.tile, p.few, a, out_dt, st);
    else launch_fp8_tile_e4m3(p.tile, p.few, a, out_dt, st);
    return hipGetLastError();
}

}  // namespace exl3
