// The 8-bit float product on bf16 MFMAs, with outputs of every type (fp8_tiles.cuh).
#include "fp8_tiles.cuh"

namespace exl3 {
void launch_fp8_tile_exact(int tile, bool few, const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    launch_fp8_tile<true>(tile, few, a, out_dt, st);
}
}  // namespace exl3
