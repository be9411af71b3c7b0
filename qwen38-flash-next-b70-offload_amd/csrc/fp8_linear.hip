// Which tile computes an 8-bit float product (fp8_tiles.cuh has the kernel).
//
// A tile of BM rows x BN columns brings (BM + BN) 128 bytes to its CU per block of k, and a CU takes them in at 42-46 GB/s
// whatever the tile (4096 -> 2048, one tile per CU, weights from HBM: 256 KB of 32 x 32 in 8.8 us, 512 KB of 64 x 64 in 13.8, 1 MB
// of 128 x 128 in 27.1, of each 2.4 any launch's): what a CU has to bring in is what takes the time, and the tile is the one for
// which that is least,
//
//     max(1, tiles / 256 CUs) (BM + BN)
//
// the smaller one where two are equal, but for these, since a CU with one tile has its LDS for more stages: 16 x 16 and, of more
// than 16 rows, 16 x 32 only where each CU has one at most (100 rows below), 64 x 64 only so where 128 x 64 is (700 rows), and that
// only so (1,500 rows) and without exact sums (1,024 rows of those, in an earlier form: 26.0, 64 x 64 25.4).
//
// Every tile, quantised rows, bf16 outputs, weights from HBM, us per call out of a graph; * is what the rule takes. With fp32
// outputs, and at 2000 -> 1000, the rule's tile is the fastest as well, or within 7 % of it (the runs' own differences).
//   4096 -> 2048, rows   16    64   100   128   256   512   700  1,000  1,500  2,048  4,096
//   16 x 16            6.7*   8.2  13.0  13.5  24.4  45.7  53.8
//   16 x 32            7.5    7.3* 10.0  10.3  19.7  29.8  33.5   48.3
//   32 x 32            8.0    8.9   7.7*  8.8* 12.5* 22.2  27.1   38.8   50.4   71.9  131.4
//   64 x 64           11.3   15.8  12.7  15.4  14.6  13.8* 20.3   22.0   34.9   43.9   75.4
//   128 x 64                 16.7  21.2  24.1  22.8  21.3  17.1*  20.0*  33.4   39.5   77.5
//   128 x 128                      26.5  29.3  27.5  26.4  22.6   25.1   25.4*  27.1*  45.9*
//   256 x 256                                  57.7  53.9  54.9   56.2   52.5   53.1   53.4
//   2048 -> 12,288
//   16 x 16           10.8   25.2  40.4  45.3
//   16 x 32            9.1*  16.0  23.8  26.4
//   32 x 32            9.4   14.9  19.2  21.0  37.5  70.6
//   64 x 64            8.6   10.4* 13.1  14.8  24.2  34.9  49.1   65.5   84.9  129.8  225.3
//   128 x 64          10.1   10.7  12.2* 13.5* 22.4  32.5  45.5   58.8   79.1  119.4  233.5
//   128 x 128         12.7   13.6  15.3  16.5  16.3* 26.6* 36.9   43.6   56.4   73.0  140.7
//   256 x 256                28.4  30.0  30.2  31.4  30.2  29.9*  31.0*  54.6*  59.2*  96.4*
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
// 32). More rows are quantised by a launch of their own (measured side by side: 2048 -> 1024, 8 rows 5.1 us, by two launches 6.1;
// 4096 -> 2048, 8 rows 8.0 us, by two launches 7.4).
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
