// spg_fp8.cu -- rows of values to 8-bit floating point (E4M3 elements, an E8M0 scale for 128 of them), and back.
//
//   E = the least integer from -127 on with max|x| <= 448 * 2^E,  code = nearest E4M3 of x / 2^E   (per block of 128)
//
// All of it is exact but the last rounding: E is the exponent of the largest magnitude, and division by 2^E a multiplication.
// Both directions are bound by bytes.  A warp has 512 columns of a row, the four blocks of one word of scales: its lanes have four neighbouring elements of each block,
// so loads, stores of codes and the four maxima are of whole warps.  A gather of rows (an expert's, from the router's order) is an index per warp.
// us: 16384 x 8192 of fp32 102 (6.6 TB/s), of bf16 73 (5.5 TB/s; 93 with a row a warp, 84 with loads that stay in the caches, which fp32 is quicker with: 109 without), back to fp32
// 111 (6.0 TB/s, most of it writes) and bf16 69 (5.8).
#include "spg_fp8.cuh"

namespace {

using namespace spgfp8;

constexpr uint32_t THREADS = 256, WARPS = THREADS / 32;

// four elements from column c on, zero beyond cols; VEC: rows lie on the size of four
template <typename T, bool VEC> __device__ __forceinline__ void load4(const T *row, uint32_t c, uint32_t cols, T (&v)[4])
{
    if (VEC && c + 4u <= cols) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(row + c);
        else *reinterpret_cast<uint2 *>(v) = __ldcs(reinterpret_cast<const uint2 *>(row + c));
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) v[i] = c + i < cols ? row[c + i] : from_f32<T>(0.0f);
    }
}
// Rows of a warp where there are enough for the device; the next one is on its way while one is worked on.
constexpr uint32_t MANY = 8;

// (Plain loads, here and below: those through the read-only path may be moved in front of the wait for the launch that writes what they read.)
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) spg_fp8_quantize_kernel(const T *x, uint32_t ldx, uint32_t x_rows, const int32_t *index, uint8_t *codes, uint32_t pitch,
                                                                  uint32_t *words, uint32_t rows, uint32_t cols, uint32_t row_blocks, uint32_t each)
{
    spg_grid_trigger();
    spg_grid_wait();
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
    const uint32_t group = blockIdx.x / row_blocks, lo = blockIdx.x % row_blocks * WARPS * each + warp, hi = min(rows, (blockIdx.x % row_blocks + 1) * WARPS * each);
    const uint32_t c0 = group * GROUP + lane * 4u, end = (cols + 15u) / 16u * 16u;
    alignas(16) T next[4][4];
    const auto load = [&](uint32_t r) {
        const uint32_t from = index ? (uint32_t)index[r] : r;     // (a negative one is none of x's rows either)
        const uint32_t here = from < x_rows ? cols : 0u;          // its columns that there are
        const T *row = x + (uint64_t)(here ? from : 0u) * ldx;
#pragma unroll
        for (uint32_t b = 0; b < 4; b++) load4<T, VEC>(row, c0 + b * BLOCK, here, next[b]);
    };
    if (lo < hi) load(lo);
    for (uint32_t r = lo; r < hi; r += WARPS) {
        float v[4][4];
#pragma unroll
        for (uint32_t b = 0; b < 4; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) v[b][i] = to_f32(next[b][i]);
        if (r + WARPS < hi) load(r + WARPS);
        uint32_t word = 0;
#pragma unroll
        for (uint32_t b = 0; b < 4; b++) {
            uint32_t a = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) a = max(a, __float_as_uint(v[b][i]) & 0x7fffffffu);    // (as bits: a NaN is above all)
            const uint32_t byte = scale_byte(__reduce_max_sync(0xffffffffu, a));
            const float inv = inverse_scale(byte);
            const uint32_t code = encode4(v[b][0] * inv, v[b][1] * inv, v[b][2] * inv, v[b][3] * inv), c = c0 + b * BLOCK;
            if (c < end) *reinterpret_cast<uint32_t *>(codes + (uint64_t)r * pitch + c) = byte == 255u ? 0u : code;
            word |= byte << 8 * b;
        }
        if (lane == 0) words[(uint64_t)group * rows + r] = word;
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) spg_fp8_dequantize_kernel(const uint8_t *codes, uint32_t pitch, const uint32_t *words, T *y, uint32_t ldy,
                                                                    uint32_t rows, uint32_t cols, uint32_t row_blocks, uint32_t each)
{
    // Values whose rows do not lie on the size of four leave side by side, one a lane (us of 16384 x 4097: fp32 67, 130 by four neighbours a lane, bf16 50 and 97; codes made of such
    // rows were slower that way, 63 and 49)
    __shared__ alignas(16) float side[VEC ? 1 : WARPS][BLOCK];
    spg_grid_trigger();
    spg_grid_wait();
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
    const uint32_t group = blockIdx.x / row_blocks, lo = blockIdx.x % row_blocks * WARPS * each + warp, hi = min(rows, (blockIdx.x % row_blocks + 1) * WARPS * each);
    const uint32_t c0 = group * GROUP + lane * 4u;
    uint32_t next[4], next_word = 0;
    const auto load = [&](uint32_t r) {
        next_word = words[(uint64_t)group * rows + r];
#pragma unroll
        for (uint32_t b = 0; b < 4; b++) {
            const uint32_t c = c0 + b * BLOCK;
            next[b] = c < cols ? *reinterpret_cast<const uint32_t *>(codes + (uint64_t)r * pitch + c) : 0u;
        }
    };
    if (lo < hi) load(lo);
    for (uint32_t r = lo; r < hi; r += WARPS) {
        uint32_t code[4];
        const uint32_t word = next_word;
#pragma unroll
        for (uint32_t b = 0; b < 4; b++) code[b] = next[b];
        if (r + WARPS < hi) load(r + WARPS);
        T *row = y + (uint64_t)r * ldy;
#pragma unroll
        for (uint32_t b = 0; b < 4; b++) {
            const uint32_t c = c0 + b * BLOCK;
            const float s = scale_value(word >> 8 * b & 255u);
            float v[4];
            decode4(code[b], v);
            if constexpr (VEC) {
                alignas(16) T t[4];
#pragma unroll
                for (int i = 0; i < 4; i++) t[i] = from_f32<T>(v[i] * s);
                if (c + 4u <= cols) {
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(row + c) = *reinterpret_cast<const uint4 *>(t);
                    else *reinterpret_cast<uint2 *>(row + c) = *reinterpret_cast<const uint2 *>(t);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) if (c + i < cols) row[c + i] = t[i];
                }
            } else {
                __syncwarp();
                *reinterpret_cast<float4 *>(&side[warp][lane * 4u]) = make_float4(v[0] * s, v[1] * s, v[2] * s, v[3] * s);
                __syncwarp();
                const uint32_t first = group * GROUP + b * BLOCK + lane;
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) if (first + i * 32u < cols) row[first + i * 32u] = from_f32<T>(side[warp][i * 32u + lane]);
            }
        }
    }
}

// blocks of threads: rows by WARPS times `each`, times groups of columns (with at most 2^31 - 1 in all)
struct Grid { uint32_t row_blocks, all, each; };
bool grid_of(const spgk_fp8 *m, Grid &g)
{
    uint64_t n = 0;
    for (g.each = MANY;; g.each /= 2) {
        g.row_blocks = m->rows / (WARPS * g.each) + (m->rows % (WARPS * g.each) != 0);
        n = (uint64_t)g.row_blocks * groups(m->cols);
        if (g.each == 1 || n >= 148u * 8u) break;
    }
    g.all = (uint32_t)n;
    return n <= 0x7fffffffu;
}

template <typename T> int quantize(const void *x, uint32_t ldx, uint32_t x_rows, const int32_t *index, const spgk_fp8 *m, const Grid &g, cudaStream_t stream)
{
    const bool vec = (uintptr_t)x % (4 * sizeof(T)) == 0 && ldx % 4u == 0;
    SPGK_CUDA(spg_launch_chained(vec ? spg_fp8_quantize_kernel<T, true> : spg_fp8_quantize_kernel<T, false>, dim3(g.all), dim3(THREADS), 0, stream,
                                 (const T *)x, ldx, x_rows, index, (uint8_t *)m->codes, m->pitch, (uint32_t *)m->scales, m->rows, m->cols, g.row_blocks, g.each));
    return spgk_check_launch("spg_fp8_quantize_kernel");
}

template <typename T> int dequantize(const spgk_fp8 *m, void *y, uint32_t ldy, const Grid &g, cudaStream_t stream)
{
    const bool vec = (uintptr_t)y % (4 * sizeof(T)) == 0 && ldy % 4u == 0;
    SPGK_CUDA(spg_launch_chained(vec ? spg_fp8_dequantize_kernel<T, true> : spg_fp8_dequantize_kernel<T, false>, dim3(g.all), dim3(THREADS), 0, stream,
                                 (const uint8_t *)m->codes, m->pitch, (const uint32_t *)m->scales, (T *)y, ldy, m->rows, m->cols, g.row_blocks, g.each));
    return spgk_check_launch("spg_fp8_dequantize_kernel");
}

int refuse(const char *who, const char *why) { spgk_set_error(who, why); return SPGK_E_ARG; }

}  // namespace

int spg_fp8_check(const char *who, const spgk_fp8 *m)
{
    const char *why = nullptr;
    if (!m) why = "no matrix";
    else if (m->cols == 0 || m->cols > 0x7fffff00u || m->rows > 0x7fffff00u) why = "columns or rows out of range";
    else if (m->rows && (!m->codes || !m->scales)) why = "no memory for codes or scales";
    else if (((uintptr_t)m->codes | (uintptr_t)m->scales) % 16u) why = "codes and scales lie on 16 bytes";
    else if (m->pitch % 16u || m->pitch < spgk_fp8_pitch(m->cols)) why = "the pitch is a multiple of 16 and holds a row";
    return why ? refuse(who, why) : SPGK_OK;
}

extern "C" {

uint32_t spgk_fp8_pitch(uint32_t cols) { return cols / 16u * 16u + (cols % 16u ? 16u : 0u); }

size_t spgk_fp8_scales_bytes(uint32_t rows, uint32_t cols) { return (size_t)spgfp8::groups(cols) * rows * 4u; }

size_t spgk_fp8_scale_index(uint32_t rows, uint32_t row, uint32_t block) { return ((size_t)(block / 4u) * rows + row) * 4u + block % 4u; }

int spgk_fp8_quantize(const void *x, int type, uint32_t ldx, uint32_t x_rows, const int32_t *rows_idx, const spgk_fp8 *dst, void *stream)
{
    const char *who = "spgk_fp8_quantize";
    const int rc = spg_fp8_check(who, dst);
    if (rc) return rc;
    if (type != SPGK_T_F16 && type != SPGK_T_BF16 && type != SPGK_T_F32) return refuse(who, "unknown type");
    if (dst->rows == 0) return SPGK_OK;
    if ((!x && x_rows) || (uintptr_t)x % (type == SPGK_T_F32 ? 4u : 2u)) return refuse(who, "no rows, or not aligned to their type");
    if ((uintptr_t)rows_idx % 4u) return refuse(who, "indexes not aligned");
    if (!rows_idx && x_rows < dst->rows) return refuse(who, "fewer rows than the matrix has");
    if (x_rows > 0x80000000u) return refuse(who, "more rows than an index can name");
    if (x_rows > 1 && ldx < dst->cols) return refuse(who, "rows overlap");
    Grid g;
    if (!grid_of(dst, g)) return refuse(who, "too many rows and columns for one call");
    if (type == SPGK_T_F32) return quantize<float>(x, ldx, x_rows, rows_idx, dst, g, (cudaStream_t)stream);
    if (type == SPGK_T_F16) return quantize<__half>(x, ldx, x_rows, rows_idx, dst, g, (cudaStream_t)stream);
    return quantize<__nv_bfloat16>(x, ldx, x_rows, rows_idx, dst, g, (cudaStream_t)stream);
}

int spgk_fp8_dequantize(const spgk_fp8 *src, void *y, int type, uint32_t ldy, void *stream)
{
    const char *who = "spgk_fp8_dequantize";
    const int rc = spg_fp8_check(who, src);
    if (rc) return rc;
    if (type != SPGK_T_F16 && type != SPGK_T_BF16 && type != SPGK_T_F32) return refuse(who, "unknown type");
    if (src->rows == 0) return SPGK_OK;
    if (!y || (uintptr_t)y % (type == SPGK_T_F32 ? 4u : 2u)) return refuse(who, "no rows, or not aligned to their type");
    if (src->rows > 1 && ldy < src->cols) return refuse(who, "rows overlap");
    Grid g;
    if (!grid_of(src, g)) return refuse(who, "too many rows and columns for one call");
    if (type == SPGK_T_F32) return dequantize<float>(src, y, ldy, g, (cudaStream_t)stream);
    if (type == SPGK_T_F16) return dequantize<__half>(src, y, ldy, g, (cudaStream_t)stream);
    return dequantize<__nv_bfloat16>(src, y, ldy, g, (cudaStream_t)stream);
}

}  // extern "C"
