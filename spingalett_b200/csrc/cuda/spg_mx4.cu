// spg_mx4.cu -- rows of values to microscaled 4-bit numbers (E2M1 elements, an E8M0 scale for 32 of them), and back.
//
//   E = clamp(floor(log2 max|x|) - 2, -127, 127),  code = nearest E2M1 of x / 2^E   (per block of 32)
//
// All of it is exact but the last rounding: the exponent of the largest magnitude is a bit field, division by 2^E a multiplication.
// Both directions are bound by bytes.  A block of threads has one tile of 128 rows x 128 columns, whose 512 bytes of scales leave or come at once; sixteen
// lanes have a row of it, eight values a lane (16-byte loads of 16-bit values, two of fp32; four bytes of codes), four rows on their way at a time.
// 16384 x 8192: to 4 bits 93 us of fp32 (6.5 TB/s), 65 of bf16 (5.2 TB/s; 64 % of the issue slots: eight values are some fifty instructions), back 115 us to
// fp32 (5.3 TB/s, nearly all of it writes), 55 to bf16 (6.1).
#include "spg_mx4.cuh"

namespace {

using namespace spgmx4;

constexpr uint32_t THREADS = 256;
constexpr uint32_t GROUPS = THREADS / 16;      // of sixteen lanes

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// what a block of threads has of a tile: `share` rows of it, from row `begin` on to `end` where the matrix has so many
struct Part {
    uint32_t row0, tile, begin, end;
    __device__ __forceinline__ Part(uint32_t rows, uint32_t kt, uint32_t share)
    {
        const uint32_t parts = 128u / share, at = blockIdx.x / parts;
        row0 = at / kt * 128u; tile = at % kt; begin = blockIdx.x % parts * share; end = min(begin + share, rows - row0);
    }
};

// The largest magnitude's bits (as fp32) of eight values.  Of 16-bit values their own bits are compared, two at a time.
__device__ __forceinline__ uint32_t largest(const float (&t)[8])
{
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) a = max(a, __float_as_uint(t[i]) & 0x7fffffffu);         // (as bits: a NaN is above all)
    return a;
}
template <typename T> __device__ __forceinline__ uint32_t largest(const T (&t)[8])
{
    const uint32_t *w = reinterpret_cast<const uint32_t *>(t);
    const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    const uint16_t a = (uint16_t)max(m >> 16, m & 0xffffu);
    return __float_as_uint(to_f32(*reinterpret_cast<const T *>(&a)));
}

// (Plain loads, here and below: those through the read-only path may be moved in front of the wait for the launch that writes what they read.)
// VEC: rows of x lie on 16 bytes.  AT_ONCE: rows of a group on their way at a time
template <typename T, bool VEC, uint32_t AT_ONCE>
__global__ void __launch_bounds__(THREADS) spg_mx4_quantize_kernel(const T *x, uint32_t ldx, uint8_t *codes, uint32_t pitch,
                                                                  uint8_t *scales, uint32_t rows, uint32_t cols, uint32_t share)
{
    spg_grid_trigger();
    spg_grid_wait();
    const Part p(rows, tiles4(cols), share);
    const uint32_t lane16 = threadIdx.x % 16u, group = threadIdx.x / 16u, row0 = p.row0, c0 = p.tile * 128u + lane16 * 8u, lanes = 0xffffu << (threadIdx.x & 16u);
    uint32_t *words = reinterpret_cast<uint32_t *>(scales) + (uint64_t)(blockIdx.x / (128u / share)) * 128u;      // the tile's scales, four bytes a row
    for (uint32_t r = max(p.begin, p.end) + threadIdx.x; r < p.begin + share; r += THREADS) words[scale_in_tile(r) / 4u] = 0;
    for (uint32_t r0 = p.begin + group; r0 < p.end; r0 += GROUPS * AT_ONCE) {
        alignas(16) T t[AT_ONCE][8];
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; k++) {
            const uint32_t r = r0 + k * GROUPS;
            const T *src = x + (uint64_t)(row0 + r) * ldx + c0;
            if (VEC && r < p.end && c0 + 8u <= cols) {
#pragma unroll
                for (uint32_t i = 0; i < sizeof(T) / 2; i++) reinterpret_cast<uint4 *>(t[k])[i] = reinterpret_cast<const uint4 *>(src)[i];
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) t[k][i] = r < p.end && c0 + i < cols ? src[i] : from_f32<T>(0.0f);
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; k++) {
            const uint32_t r = r0 + k * GROUPS;
            if (r >= p.end) break;                               // (the same in a group)
            uint32_t a = largest(t[k]);
            a = max(a, __shfl_xor_sync(lanes, a, 1));
            a = max(a, __shfl_xor_sync(lanes, a, 2));
            const uint32_t byte = scale_byte(a);
            const float inv = inverse_scale(byte);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = to_f32(t[k][i]) * inv;
            const uint32_t code = encode8(v);
            if (c0 < (cols + 31u) / 32u * 32u) *reinterpret_cast<uint32_t *>(codes + (uint64_t)(row0 + r) * pitch + c0 / 2u) = byte == 255u ? 0u : code;
            uint32_t word = byte << (lane16 / 4u * 8u);
            word |= __shfl_xor_sync(lanes, word, 4);
            word |= __shfl_xor_sync(lanes, word, 8);
            if (lane16 == 0) words[scale_in_tile(r) / 4u] = word;
        }
    }
}

template <typename T, bool VEC, uint32_t AT_ONCE>
__global__ void __launch_bounds__(THREADS) spg_mx4_dequantize_kernel(const uint8_t *codes, uint32_t pitch, const uint8_t *scales,
                                                                    T *y, uint32_t ldy, uint32_t rows, uint32_t cols, uint32_t share)
{
    __shared__ float side[VEC ? 1 : THREADS / 32][2][128];       // values whose rows do not lie on 16 bytes leave side by side, one a lane
    spg_grid_trigger();
    spg_grid_wait();
    const Part p(rows, tiles4(cols), share);
    constexpr bool HALVES = sizeof(T) == 4 && VEC;               // a lane has elements 4 l .. and 64 + 4 l ..
    const uint32_t lane16 = threadIdx.x % 16u, group = threadIdx.x / 16u, row0 = p.row0, tile0 = p.tile * 128u;
    const uint32_t c0 = tile0 + lane16 * (HALVES ? 4u : 8u), c1 = HALVES ? c0 + 64u : c0 + 4u;
    const uint32_t *words = reinterpret_cast<const uint32_t *>(scales) + (uint64_t)(blockIdx.x / (128u / share)) * 128u;
    for (uint32_t r0 = p.begin + group; r0 - group < p.end; r0 += GROUPS * AT_ONCE) {                              // (whole warps)
        uint32_t code[AT_ONCE], word[AT_ONCE];
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; k++) {
            const uint32_t r = r0 + k * GROUPS;
            code[k] = word[k] = 0;
            if (r >= p.end) continue;
            const uint8_t *src = codes + (uint64_t)(row0 + r) * pitch;
            word[k] = words[scale_in_tile(r) / 4u];
            if (HALVES) {
                if (c0 < cols) code[k] = *reinterpret_cast<const uint16_t *>(src + c0 / 2u);
                if (c1 < cols) code[k] |= (uint32_t)*reinterpret_cast<const uint16_t *>(src + c1 / 2u) << 16;
            } else if (c0 < cols) code[k] = *reinterpret_cast<const uint32_t *>(src + c0 / 2u);
        }
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; k++) {
            const uint32_t r = r0 + k * GROUPS;
            uint32_t h[4];
            decode8(code[k], h);
            const float s0 = scale_value(word[k] >> (c0 % 128u / 32u * 8u) & 255u), s1 = HALVES ? scale_value(word[k] >> (c1 % 128u / 32u * 8u) & 255u) : s0;
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
                v[2 * i] = f.x * (i < 2 ? s0 : s1); v[2 * i + 1] = f.y * (i < 2 ? s0 : s1);
            }
            if (VEC) {
                if (r >= p.end) break;
                alignas(16) T t[8];
#pragma unroll
                for (int i = 0; i < 8; i++) t[i] = from_f32<T>(v[i]);
                T *dst = y + (uint64_t)(row0 + r) * ldy;
                if (c1 + 4u <= cols) {
                    *reinterpret_cast<uint4 *>(dst + c0) = reinterpret_cast<const uint4 *>(t)[0];
                    if (HALVES) *reinterpret_cast<uint4 *>(dst + c1) = reinterpret_cast<const uint4 *>(t)[sizeof(T) == 4];
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) { const uint32_t c = i < 4 ? c0 + i : c1 + i - 4u; if (c < cols) dst[c] = t[i]; }
                }
            } else {
                const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, first = r - (group & 1u);      // (the warp has rows first and first + 1)
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4 *>(&side[warp][group & 1u][lane16 * 8u + i]) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                __syncwarp();
#pragma unroll
                for (uint32_t q = 0; q < 2; q++) {
                    if (first + q >= p.end) continue;
                    T *dst = y + (uint64_t)(row0 + first + q) * ldy + tile0;
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) if (tile0 + i * 32u + lane < cols) dst[i * 32u + lane] = from_f32<T>(side[warp][q][i * 32u + lane]);
                }
            }
        }
    }
}

// Rows of a tile that a block of threads has, four a group of lanes on their way, where there are enough tiles for the device; a row a group where there are few.
// us with 16 and 128: 3001 x 777 of fp16 3.6 and 7.1, 4096 x 4096 of bf16 15.7 and 10.4 (64: 10.8; back to fp32 16.3, 19.6, 17.3), 16384 x 8192 of bf16
// 115 and 65.  Up to 16 rows there is nothing to share (1 x 8192: 1.9 and 1.5).
uint32_t share_of(uint32_t rows, uint32_t tiles) { return rows <= GROUPS || tiles >= 148u * 16u ? 128u : (tiles >= 148u * 4u ? 64u : GROUPS); }

template <typename T> int quantize(const void *x, uint32_t ldx, const spgk_mx4 *m, cudaStream_t stream)
{
    const uint32_t tiles = (m->rows / 128u + (m->rows % 128u != 0)) * tiles4(m->cols), share = share_of(m->rows, tiles);
    const dim3 grid(tiles * (128u / share));
    const bool vec = ((uintptr_t)x % 16u == 0) && (uint64_t)ldx * sizeof(T) % 16u == 0;
    SPGK_CUDA(spg_launch_chained(share > GROUPS ? (vec ? spg_mx4_quantize_kernel<T, true, 4> : spg_mx4_quantize_kernel<T, false, 4>) : (vec ? spg_mx4_quantize_kernel<T, true, 1> : spg_mx4_quantize_kernel<T, false, 1>), grid, dim3(THREADS), 0, stream,
                                 (const T *)x, ldx, (uint8_t *)m->codes, m->pitch, (uint8_t *)m->scales, m->rows, m->cols, share));
    return spgk_check_launch("spg_mx4_quantize_kernel");
}

template <typename T> int dequantize(const spgk_mx4 *m, void *y, uint32_t ldy, cudaStream_t stream)
{
    const uint32_t tiles = (m->rows / 128u + (m->rows % 128u != 0)) * tiles4(m->cols), share = share_of(m->rows, tiles);
    const dim3 grid(tiles * (128u / share));
    const bool vec = ((uintptr_t)y % 16u == 0) && (uint64_t)ldy * sizeof(T) % 16u == 0;
    SPGK_CUDA(spg_launch_chained(share > GROUPS ? (vec ? spg_mx4_dequantize_kernel<T, true, 4> : spg_mx4_dequantize_kernel<T, false, 4>) : (vec ? spg_mx4_dequantize_kernel<T, true, 1> : spg_mx4_dequantize_kernel<T, false, 1>), grid, dim3(THREADS), 0, stream,
                                 (const uint8_t *)m->codes, m->pitch, (const uint8_t *)m->scales, (T *)y, ldy, m->rows, m->cols, share));
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
