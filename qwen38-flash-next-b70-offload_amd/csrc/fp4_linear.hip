// Which kernel computes a 4-bit float product: fp4_few.hip's, a tile of fp4_tiles.cuh or fp4_tile256.hip's.
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
Pick pick_tile(int M, int n, int kb) {
    constexpr int kSizes[][2] = {{32, 32}, {64, 64}, {128, 64}, {128, 128}, {256, 256}};
    Pick best{kFp4Tile256, false, 0};
    for (int i = kFp4Tile32; i <= kFp4Tile256; ++i) {
        const int64_t tiles = (int64_t)((M - 1) / kSizes[i][0] + 1) * ((n - 1) / kSizes[i][1] + 1), rounds = (tiles + kCus - 1) / kCus;
        const int rows = kSizes[i][0] + kSizes[i][1];
        int64_t cost = rounds * rows;
        if (i == kFp4Tile128x64 && rounds > 1) continue;
        if (i == kFp4Tile128 && rounds > 1) cost = tiles * rows / kCus;
        if (i == kFp4Tile256 && kb < 4 && best.cost) continue;
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
            const int64_t workgroups = (int64_t)((n - 1) / (16 * tn) + 1) * ((M - 1) / R + 1), rounds = (workgroups + kCus - 1) / kCus;
            if (R > (own ? 16 : 64) || (workgroups + 7) * 1024 >= kMaxThreads) continue;
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

bool fp4_product_quantises(int M, int, int) { return M <= kOwnRows; }

hipError_t launch_fp4_product(const Fp4ProductArgs& a, int out_dt, hipStream_t st) {
    const FewTile f = pick_few(a.M, a.n, !a.q);
    const Pick p = pick_tile(a.M, a.n, a.kb);
    if (!a.q || a.M <= kOwnRows || (f.tn && f.cost * 4 <= p.cost * 3)) launch_fp4_few(a, f.tn, f.R, out_dt, st);
    else launch_tile<false>(p, a, out_dt, st);
    return hipGetLastError();
}

bool fp4_gate_up_in_tiles(int M) { return M > kOwnRows; }

hipError_t launch_fp4_gate_up(const Fp4ProductArgs& a, hipStream_t st) {
    launch_tile<true>(pick_tile(a.M, a.n, a.kb), a, 2, st);
    return hipGetLastError();
}

}  // namespace exl3
