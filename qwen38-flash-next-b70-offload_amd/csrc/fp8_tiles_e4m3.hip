// The 8-bit float product on e4m3 MFMAs, with fp16 and bf16 outputs (fp8_tiles.cuh).
#include "fp8_tiles.cuh"

namespace exl3 {
void launch_fp8_tile_e4m3(int tile, bool few, const Fp8ProductArgs& a, int out_dt, hipStream_t st) {
    launch_fp8_tile<false>(tile, few, a, out_dt, st);
}
}  // namespace exl3
