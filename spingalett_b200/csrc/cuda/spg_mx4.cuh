// spg_mx4.cuh -- one block of microscaled 4-bit numbers: its scale, its elements, and where they lie.
#pragma once

#include "spg_common.cuh"

namespace spgmx4 {

// blocks of 32 in a row, and tiles of four of them
__host__ __device__ inline uint32_t blocks(uint32_t cols) { return cols / 32u + (cols % 32u != 0); }
__host__ __device__ inline uint32_t tiles4(uint32_t cols) { return cols / 128u + (cols % 128u != 0); }
// byte of the scale of block 0 of a tile's row inside the tile of 128 rows x 4 blocks (the order in which tcgen05.cp takes it to tensor memory)
__host__ __device__ inline uint32_t scale_in_tile(uint32_t row) { return (row % 32u) * 16u + (row % 128u) / 32u * 4u; }

// Scale byte of a block whose largest magnitude has these bits (as fp32, sign cleared): 2^(byte - 127) with byte - 127 = floor(log2 a) - 2, the exponent
// field less two; below 2^-125 (subnormals among them) it stays at 0.  0xFF, NaN, where the block holds an infinity or a NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits)
{
    const uint32_t e = amax_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// what its elements are multiplied with: 2^(127 - byte), exact, a normal number for every byte that scale_byte gives; 0 for NaN blocks
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23); }
// 2^(byte - 127); 2^-127 is a subnormal
__device__ __forceinline__ float scale_value(uint32_t byte)
{
    return byte == 255u ? __uint_as_float(0x7fffffffu) : (byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23));
}

// eight values below 8 in magnitude -> eight E2M1 codes, the first in the lowest nibble (nearest, ties to even, 6 at most)
__device__ __forceinline__ uint32_t encode8(const float (&v)[8])
{
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// eight codes -> four pairs of fp16
__device__ __forceinline__ void decode8(uint32_t codes, uint32_t (&h)[4])
{
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
}

}  // namespace spgmx4

// SPGK_OK, or SPGK_E_ARG with a message naming `who`
int spg_mx4_check(const char *who, const spgk_mx4 *m);
