// What the tile kernels of the 8-bit and the 4-bit float linear share: vector types, loads from buffers to LDS, the order of a
// row's pieces there, outputs in 16 bits.
#pragma once
#include "exl3_common.cuh"

namespace exl3 {
typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint16_t v4u __attribute__((ext_vector_type(4)));
typedef uint16_t v8u __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_any;

// four outputs as fp16 (DT 0) or bf16 (DT 1)
template <int DT>
__device__ __forceinline__ v4u narrow4(v4f v) {
    v4u u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (DT == 0) u[j] = __builtin_bit_cast(uint16_t, (_Float16)v[j]);
        else u[j] = __builtin_bit_cast(uint16_t, (__bf16)v[j]);
    }
    return u;
}

using Rsrc = __amdgpu_buffer_rsrc_t;
// a buffer of `bytes`, zeros behind it
__device__ __forceinline__ Rsrc buffer_of(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
// 16 bytes a lane (or 4) from the buffer to LDS, the lanes' pieces one after the other
template <int BYTES>
__device__ __forceinline__ void to_lds(void* lds, Rsrc from, uint32_t lane_off, uint32_t off) {
    if constexpr (BYTES == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_any*)lds, 16, lane_off, off, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_any*)lds, 4, lane_off, off, 0, 0);
}

// four floats from element n on, 0 behind the buffer's end
__device__ __forceinline__ v4f floats_of(Rsrc from, int n) {
    return __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(from, n * 4, 0, 0));
}

// place of 16-byte piece c of a row in LDS: rows are 128 bytes apart (or an odd multiple), and with this the fragment reads
// of 16 rows meet every bank once
__device__ __forceinline__ int piece_at(int row, int c) { return c ^ ((row >> 1) & 7); }

}  // namespace exl3
