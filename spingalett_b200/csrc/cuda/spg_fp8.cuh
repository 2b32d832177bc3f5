// spg_fp8.cuh -- one block of 8-bit floating-point numbers with a scale: the scale, the elements, and where they lie.
#pragma once

#include "spg_common.cuh"

namespace spgfp8 {

constexpr uint32_t BLOCK = 128, GROUP = 4 * BLOCK;              // GROUP: the columns of one word of scales

// blocks in a row, and words of four of them
__host__ __device__ inline uint32_t blocks(uint32_t cols) { return cols / BLOCK + (cols % BLOCK != 0); }
__host__ __device__ inline uint32_t groups(uint32_t cols) { return cols / GROUP + (cols % GROUP != 0); }

// Scale byte of a block whose largest magnitude has these bits (as fp32, sign cleared): the least power of two by which it comes to 448 = 1.75 * 2^8 or
// less, its exponent less eight, one more where its mantissa is above 1.75; 0 (2^-127) at least.  0xFF, NaN, where the block holds an infinity or a NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits)
{
    const uint32_t e = (amax_bits + 0x1fffffu) >> 23;           // (a mantissa above 1.75 carries into the exponent)
    return amax_bits >= 0x7f800000u ? 255u : (e > 8u ? e - 8u : 0u);
}
// what its elements are multiplied with: 2^(127 - byte), exact, a normal number for every byte that scale_byte gives; 0 for NaN blocks
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23); }
// 2^(byte - 127); 2^-127 is a subnormal
__device__ __forceinline__ float scale_value(uint32_t byte)
{
    return byte == 255u ? __uint_as_float(0x7fffffffu) : (byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23));
}

// four values of at most 448 in magnitude -> four E4M3 codes, the first in the lowest byte (nearest, ties to even)
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d)
{
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
// four codes -> what they stand for without the scale
__device__ __forceinline__ void decode4(uint32_t codes, float (&v)[4])
{
    uint32_t lo, hi;
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(codes));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo)), b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}

// rows of any of the three types
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

}  // namespace spgfp8

// SPGK_OK, or SPGK_E_ARG with a message naming `who`
int spg_fp8_check(const char *who, const spgk_fp8 *m);
