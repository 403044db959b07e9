// The microscaled 4-bit format (MXFP4) shared by the quantiser, the expert product and the few-token layer.
//
// Elements are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign), two to a byte, the even column in the low half. A block of
// 32 consecutive columns of a row shares one e8m0 scale byte s = 2^(s - 127); 255 stands for NaN. Scales are kept in the
// order in which the tensor cores take them: tiles of 128 rows x 4 blocks, 512 bytes each,
//   byte (row, block) of a matrix = tile (row / 128, block / 4), [row % 32][row / 32 % 4][block % 4],
// tiles of a matrix row-tile-major. Rows and blocks that only fill up a tile have scale 0 (2^-127).
#pragma once
#include <cuda_fp4.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace aristos {

constexpr int FP4_BLOCK = 32;             // elements per scale
constexpr int FP4_TILE_ROWS = 128;
constexpr int FP4_TILE_COLS = 128;        // 4 blocks
constexpr int FP4_TILE_BYTES = 512;

__host__ __device__ __forceinline__ int fp4_row_tiles(int rows) { return (rows + FP4_TILE_ROWS - 1) / FP4_TILE_ROWS; }
__host__ __device__ __forceinline__ int fp4_col_tiles(int cols) { return (cols + FP4_TILE_COLS - 1) / FP4_TILE_COLS; }
__host__ __device__ __forceinline__ size_t fp4_matrix_scale_bytes(int rows, int cols) {
    return (size_t)fp4_row_tiles(rows) * fp4_col_tiles(cols) * FP4_TILE_BYTES;
}
// Place of row `row`'s 4-byte word (blocks 4 t .. 4 t + 3) inside its tile.
__host__ __device__ __forceinline__ int fp4_tile_word(int row) { return (row & 31) * 16 + ((row >> 5) & 3) * 4; }

#ifdef __CUDACC__
// 2^(s - 127) as fp32 (255: NaN; 0: the subnormal 2^-127).
__device__ __forceinline__ float fp4_scale_value(uint32_t s) {
    return s == 255u ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(s == 0u ? 0x00400000u : s << 23);
}

// Scale byte of a block whose largest magnitude is amax: floor(log2 amax) - 2 is the exponent (the largest element
// power of two is 4 = 2^2), at least -127. A block that holds an infinity or a NaN gets the NaN scale, so that it comes
// back as NaN instead of as something finite. The exponent field of amax is floor(log2) + 127 for normal numbers; a
// subnormal amax is below 2^-126 and its scale is clamped either way.
__device__ __forceinline__ uint32_t fp4_scale_of(float amax) {
    const uint32_t field = __float_as_uint(amax) >> 23;
    if (field == 255u) return 255u;
    return field > 2u ? field - 2u : 0u;
}
// What the elements of a block are multiplied with before they are rounded: 2^(127 - s). s <= 252 for finite amax, so
// the factor is a normal number and the products are exact (or so small that they round to zero either way).
__device__ __forceinline__ float fp4_inverse_scale(uint32_t s) { return __uint_as_float((254u - min(s, 253u)) << 23); }

// Two values, already divided by their scale, to one byte (a in the low half); round to nearest even, saturate at 6.
__device__ __forceinline__ uint32_t fp4_pack2(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(a, b), __NV_E2M1, cudaRoundNearest);
}
// The two elements of a byte as fp16 (exact).
__device__ __forceinline__ __half2 fp4_unpack2(uint32_t byte) {
    const __half2_raw r = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)byte, __NV_E2M1);
    return *reinterpret_cast<const __half2*>(&r);
}
#endif

}  // namespace aristos
