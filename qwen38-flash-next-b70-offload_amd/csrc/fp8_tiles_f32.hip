// The 8-bit float product with fp32 outputs (fp8_tiles.cuh).
#include "fp8_tiles.cuh"

namespace exl3 {
void launch_fp8_tile_32(int tile, bool few, const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    launch_fp8_tile<true>(tile, few, a, out_dt, st);
}
}  // namespace exl3
