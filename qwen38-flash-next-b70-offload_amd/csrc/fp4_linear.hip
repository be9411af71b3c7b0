// Which tile computes a 4-bit float product (fp4_tiles.cuh has the kernel).
#include "fp4_tiles.cuh"

namespace exl3 {

hipError_t launch_fp4_product(const Fp4ProductArgs& a, int out_dt, hipStream_t st) {
    if (a.M <= 32 && a.n <= 1 << 26) launch_fp4_tiles<false, 32, 32, 1, 1, 4, 2>(a, out_dt, st);
    else if (a.M <= 256 && a.n <= 1 << 24) launch_fp4_tiles<false, 64, 64, 2, 2, 2, 2>(a, out_dt, st);
    else launch_fp4_tiles<false, 128, 128, 2, 2, 1, 2>(a, out_dt, st);
    return hipGetLastError();
}

hipError_t launch_fp4_gate_up(const Fp4ProductArgs& a, hipStream_t st) {
    if (a.M <= 32 && a.n <= 1 << 25) launch_fp4_tiles<true, 32, 64, 1, 1, 4, 2>(a, 2, st);
    else launch_fp4_tiles<true, 128, 128, 2, 2, 1, 2>(a, 2, st);
    return hipGetLastError();
}

}  // namespace exl3
