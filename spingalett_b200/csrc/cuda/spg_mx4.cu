// spg_mx4.cu -- rows of values to microscaled 4-bit numbers (E2M1 elements, an E8M0 scale for 32 of them), and back.
//
//   E = clamp(floor(log2 max|x|) - 2, -127, 127),  code = nearest E2M1 of x / 2^E   (per block of 32)
//
// All of it is exact but the last rounding: the exponent of the largest magnitude is a bit field, division by 2^E a multiplication.
// Both directions are bound by bytes.  Four lanes share a block (eight values a lane: 16-byte loads of 16-bit values, two of fp32; four
// bytes of codes), sixteen lanes the four blocks whose scales are neighbours, so a scale word is one 4-byte store.
#include "spg_mx4.cuh"

namespace {

using namespace spgmx4;

constexpr uint32_t THREADS = 256;
constexpr uint32_t GROUPS = THREADS / 16;      // of sixteen lanes, 128 values each

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC: rows of x lie on 16 bytes
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) spg_mx4_quantize_kernel(const T *__restrict__ x, uint32_t ldx, uint8_t *__restrict__ codes, uint32_t pitch,
                                                                  uint8_t *__restrict__ scales, uint32_t rows, uint32_t cols, uint32_t row_tiles)
{
    spg_grid_wait();
    const uint32_t kt = tiles4(cols), lane16 = threadIdx.x % 16u;
    const uint64_t at = (uint64_t)blockIdx.x * GROUPS + threadIdx.x / 16u;
    if (at >= (uint64_t)row_tiles * 128u * kt) return;           // (a whole group of sixteen leaves)
    const uint32_t row = (uint32_t)(at / kt), tile = (uint32_t)(at % kt);
    const uint32_t c0 = tile * 128u + lane16 * 8u;
    const uint32_t lanes = 0xffffu << (threadIdx.x & 16u);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = 0.0f;
    if (row < rows) {
        const T *src = x + (uint64_t)row * ldx + c0;
        if (VEC && c0 + 8u <= cols) {
            alignas(16) T t[8];
#pragma unroll
            for (int i = 0; i < (int)sizeof(t) / 16; i++) reinterpret_cast<uint4 *>(t)[i] = __ldg(reinterpret_cast<const uint4 *>(src) + i);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = to_f32(t[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) if (c0 + i < cols) v[i] = to_f32(src[i]);
        }
    }
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) a = max(a, __float_as_uint(v[i]) & 0x7fffffffu);     // (as bits: a NaN is above all)
    a = max(a, __shfl_xor_sync(lanes, a, 1));
    a = max(a, __shfl_xor_sync(lanes, a, 2));
    const uint32_t byte = scale_byte(a);
    const float inv = inverse_scale(byte);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = byte == 255u ? 0.0f : v[i] * inv;
    if (row < rows && c0 < (cols + 31u) / 32u * 32u)
        *reinterpret_cast<uint32_t *>(codes + (uint64_t)row * pitch + c0 / 2u) = encode8(v);
    uint32_t word = byte << (lane16 / 4u * 8u);
    word |= __shfl_xor_sync(lanes, word, 4);
    word |= __shfl_xor_sync(lanes, word, 8);
    if (lane16 == 0)
        *reinterpret_cast<uint32_t *>(scales + ((uint64_t)(row / 128u) * kt + tile) * 512u + scale_in_tile(row)) = word;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) spg_mx4_dequantize_kernel(const uint8_t *__restrict__ codes, uint32_t pitch, const uint8_t *__restrict__ scales,
                                                                    T *__restrict__ y, uint32_t ldy, uint32_t rows, uint32_t cols)
{
    spg_grid_wait();
    const uint32_t kt = tiles4(cols), lane16 = threadIdx.x % 16u;
    const uint64_t at = (uint64_t)blockIdx.x * GROUPS + threadIdx.x / 16u;
    if (at >= (uint64_t)rows * kt) return;
    const uint32_t row = (uint32_t)(at / kt), tile = (uint32_t)(at % kt);
    const uint32_t c0 = tile * 128u + lane16 * 8u;
    if (c0 >= cols) return;
    const uint32_t code = __ldg(reinterpret_cast<const uint32_t *>(codes + (uint64_t)row * pitch + c0 / 2u));
    const float s = scale_value(__ldg(scales + ((uint64_t)(row / 128u) * kt + tile) * 512u + scale_in_tile(row) + lane16 / 4u));
    uint32_t h[4];
    decode8(code, h);
    alignas(16) T t[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
        t[2 * i] = from_f32<T>(f.x * s);
        t[2 * i + 1] = from_f32<T>(f.y * s);
    }
    T *dst = y + (uint64_t)row * ldy + c0;
    if (VEC && c0 + 8u <= cols) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(t) / 16; i++) reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<const uint4 *>(t)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) if (c0 + i < cols) dst[i] = t[i];
    }
}

template <typename T> int quantize(const void *x, uint32_t ldx, const spgk_mx4 *m, cudaStream_t stream)
{
    const uint32_t row_tiles = m->rows / 128u + (m->rows % 128u != 0);
    const uint64_t groups = (uint64_t)row_tiles * 128u * tiles4(m->cols);
    const dim3 grid((uint32_t)((groups + GROUPS - 1) / GROUPS));
    const bool vec = ((uintptr_t)x % 16u == 0) && (uint64_t)ldx * sizeof(T) % 16u == 0;
    SPGK_CUDA(spg_launch_chained(vec ? spg_mx4_quantize_kernel<T, true> : spg_mx4_quantize_kernel<T, false>, grid, dim3(THREADS), 0, stream,
                                 (const T *)x, ldx, (uint8_t *)m->codes, m->pitch, (uint8_t *)m->scales, m->rows, m->cols, row_tiles));
    return spgk_check_launch("spg_mx4_quantize_kernel");
}

template <typename T> int dequantize(const spgk_mx4 *m, void *y, uint32_t ldy, cudaStream_t stream)
{
    const uint64_t groups = (uint64_t)m->rows * tiles4(m->cols);
    const dim3 grid((uint32_t)((groups + GROUPS - 1) / GROUPS));
    const bool vec = ((uintptr_t)y % 16u == 0) && (uint64_t)ldy * sizeof(T) % 16u == 0;
    SPGK_CUDA(spg_launch_chained(vec ? spg_mx4_dequantize_kernel<T, true> : spg_mx4_dequantize_kernel<T, false>, grid, dim3(THREADS), 0, stream,
                                 (const uint8_t *)m->codes, m->pitch, (const uint8_t *)m->scales, (T *)y, ldy, m->rows, m->cols));
    return spgk_check_launch("spg_mx4_dequantize_kernel");
}

}  // namespace

int spg_mx4_check(const char *who, const spgk_mx4 *m)
{
    const char *why = nullptr;
    if (!m) why = "no matrix";
    else if (m->cols == 0 || m->cols > 0x7fffff00u || m->rows > 0x7fffff00u) why = "columns or rows out of range";
    else if (((uint64_t)m->rows + 127u) / 128u * spgmx4::tiles4(m->cols) > 0x0fffffffu) why = "more than 2^28 tiles of scales";
    else if (m->rows && (!m->codes || !m->scales)) why = "no memory for codes or scales";
    else if (((uintptr_t)m->codes | (uintptr_t)m->scales) % 16u) why = "codes and scales lie on 16 bytes";
    else if (m->pitch % 16u || m->pitch < spgk_mx4_pitch(m->cols)) why = "the pitch is a multiple of 16 and holds a row's blocks";
    if (!why) return SPGK_OK;
    spgk_set_error(who, why);
    return SPGK_E_ARG;
}

extern "C" {

uint32_t spgk_mx4_pitch(uint32_t cols) { return spgmx4::blocks(cols) * 16u; }

size_t spgk_mx4_scales_bytes(uint32_t rows, uint32_t cols)
{
    return ((size_t)rows / 128u + (rows % 128u != 0)) * spgmx4::tiles4(cols) * 512u;
}

size_t spgk_mx4_scale_index(uint32_t cols, uint32_t row, uint32_t block)
{
    return ((size_t)(row / 128u) * spgmx4::tiles4(cols) + block / 4u) * 512u + spgmx4::scale_in_tile(row) + block % 4u;
}

int spgk_mx4_quantize(const void *x, int type, uint32_t ldx, const spgk_mx4 *dst, void *stream)
{
    const int rc = spg_mx4_check("spgk_mx4_quantize", dst);
    if (rc) return rc;
    if (type != SPGK_T_F16 && type != SPGK_T_BF16 && type != SPGK_T_F32) { spgk_set_error("spgk_mx4_quantize", "unknown type"); return SPGK_E_ARG; }
    if (dst->rows == 0) return SPGK_OK;
    if (!x || (uintptr_t)x % (type == SPGK_T_F32 ? 4u : 2u)) { spgk_set_error("spgk_mx4_quantize", "no rows, or not aligned to their type"); return SPGK_E_ARG; }
    if (dst->rows > 1 && ldx < dst->cols) { spgk_set_error("spgk_mx4_quantize", "rows overlap"); return SPGK_E_ARG; }
    if (type == SPGK_T_F32) return quantize<float>(x, ldx, dst, (cudaStream_t)stream);
    if (type == SPGK_T_F16) return quantize<__half>(x, ldx, dst, (cudaStream_t)stream);
    return quantize<__nv_bfloat16>(x, ldx, dst, (cudaStream_t)stream);
}

int spgk_mx4_dequantize(const spgk_mx4 *src, void *y, int type, uint32_t ldy, void *stream)
{
    const int rc = spg_mx4_check("spgk_mx4_dequantize", src);
    if (rc) return rc;
    if (type != SPGK_T_F16 && type != SPGK_T_BF16 && type != SPGK_T_F32) { spgk_set_error("spgk_mx4_dequantize", "unknown type"); return SPGK_E_ARG; }
    if (src->rows == 0) return SPGK_OK;
    if (!y || (uintptr_t)y % (type == SPGK_T_F32 ? 4u : 2u)) { spgk_set_error("spgk_mx4_dequantize", "no rows, or not aligned to their type"); return SPGK_E_ARG; }
    if (src->rows > 1 && ldy < src->cols) { spgk_set_error("spgk_mx4_dequantize", "rows overlap"); return SPGK_E_ARG; }
    if (type == SPGK_T_F32) return dequantize<float>(src, y, ldy, (cudaStream_t)stream);
    if (type == SPGK_T_F16) return dequantize<__half>(src, y, ldy, (cudaStream_t)stream);
    return dequantize<__nv_bfloat16>(src, y, ldy, (cudaStream_t)stream);
}

}  // extern "C"
