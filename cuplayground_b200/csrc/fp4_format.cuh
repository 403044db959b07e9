// The microscaled 4-bit format (MXFP4) shared by the quantiser, the expert product and the few-token layer.
//
// Elements are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign), two to a byte, the even column in the low half. A block of
// 32 consecutive columns of a row shares one e8m0 scale byte s = 2^(s - 127); 255 stands for NaN. Scales are kept in the
// order in which the tensor cores take them: tiles of 128 rows x 4 blocks, 512 bytes each,
//   byte (row, block) of a matrix = tile (row / 128, block / 4), [row % 32][row / 32 % 4][block % 4],
// tiles of a matrix row-tile-major. Rows and blocks that only fill up a tile have scale 0 (2^-127).
#pragma once
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

// Eight values, already divided by their scale, to a word of codes (v[0] in the lowest four bits); round to nearest even,
// saturate at 6.
__device__ __forceinline__ uint32_t fp4_pack8(float v0, float v1, float v2, float v3, float v4, float v5, float v6, float v7) {
    uint32_t w;
    asm("{\n\t"
        ".reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t"
        "}"
        : "=r"(w)
        : "f"(v0), "f"(v1), "f"(v2), "f"(v3), "f"(v4), "f"(v5), "f"(v6), "f"(v7));
    return w;
}
// The eight elements of a word as fp16 pairs (exact), adjacent ones together. All magnitudes have an empty low byte in
// fp16, so the high bytes of four codes come out of one byte permutation (the codes select from the table), their signs out
// of another (which spreads the top bits of bytes), and two more put zero bytes between them.
__device__ __forceinline__ void fp4_unpack8(uint32_t w, uint32_t (&v)[4]) {
    const uint32_t mag = w & 0x77777777u, up = w << 4;
    // high bytes of 0, 0.5, 1, 1.5 | 2, 3, 4, 6
    const uint32_t lo = __byte_perm(0x3E3C3800u, 0x46444240u, mag), hi = __byte_perm(0x3E3C3800u, 0x46444240u, mag >> 16);
    uint32_t sl, sh;                                    // byte i: the sign of code i (of code 4 + i) in every bit
    asm("prmt.b32 %0, %1, %2, 0x9D8C;" : "=r"(sl) : "r"(w), "r"(up));
    asm("prmt.b32 %0, %1, %2, 0xBFAE;" : "=r"(sh) : "r"(w), "r"(up));
    const uint32_t a = lo | (sl & 0x80808080u), b = hi | (sh & 0x80808080u);
    v[0] = __byte_perm(a, 0, 0x1404);
    v[1] = __byte_perm(a, 0, 0x3424);
    v[2] = __byte_perm(b, 0, 0x1404);
    v[3] = __byte_perm(b, 0, 0x3424);
}
#endif

}  // namespace aristos
