// spg_fp8_layer.cu -- dense layers on 8-bit operands with a scale for each block of 128, one layer or one for each group of rows.
//
//   y[n][j] = act(bias[j] + sum_b 2^(Ew[j,b] + Ex[n,b]) * sum_{k in block b} w[j][k] x[n][k])
//
// A block of threads has 32 rows and 128 units, a thread four by four of them; elements go through shared memory as fp32, and a block's sum is scaled as a whole, by
// 2^(Ew + Ex) in two factors (neither operand's values need fit fp32).
#include "spg_fp8.cuh"

namespace {

using namespace spgfp8;

constexpr uint32_t TM = 128, TN = 32, TK = 32, THREADS = 256;

struct LayerParams {
    uint32_t N, out, cols, experts, w_rows;
    const uint8_t *w, *x; uint32_t w_pitch, x_pitch;
    const uint8_t *w_scales, *x_scales;
    const int32_t *starts;
    const float *bias;
    int act;
    void *y; int type; uint32_t ldy;
    uint8_t *next_codes, *next_scales; uint32_t next_pitch;
};

__global__ void __launch_bounds__(THREADS) spg_fp8_layer_kernel(const LayerParams p)
{
    __shared__ float ws[TK][TM + 4], xs[TK][TN + 4];
    __shared__ uint32_t bytes[TM + TN];
    __shared__ uint32_t place[3];
    spg_grid_trigger();
    spg_grid_wait();
    if (threadIdx.x == 0) {
        // the tile of rows that this block has, of all groups' one behind the other
        uint32_t t = blockIdx.y, at = 0;
        place[0] = place[1] = place[2] = 0;
        for (uint32_t e = 0; e < p.experts; e++) {
            uint32_t lo = at, hi = p.N;
            if (p.starts) {
                lo = max(at, min((uint32_t)max(p.starts[e], 0), p.N));
                hi = max(lo, min((uint32_t)max(p.starts[e + 1], 0), p.N));
            }
            at = hi;
            const uint32_t tiles = (hi - lo + TN - 1) / TN;
            if (t < tiles) { place[0] = e; place[1] = lo + t * TN; place[2] = hi; break; }
            t -= tiles;
        }
    }
    __syncthreads();
    const uint32_t e = place[0], n0 = place[1], end = place[2], j0 = blockIdx.x * TM;
    if (n0 >= end) return;
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
    float acc[4][4] = {}, sub[4][4] = {};
    for (uint32_t k0 = 0; k0 < p.cols; k0 += TK) {
        const uint32_t b = k0 / BLOCK;
        for (uint32_t i = threadIdx.x; i < (TM + TN) * (TK / 4); i += THREADS) {
            const uint32_t r = i / (TK / 4), c = i % (TK / 4) * 4, k = k0 + c;
            const bool w = r < TM;
            const uint64_t row = w ? (uint64_t)e * p.out + j0 + r : (uint64_t)n0 + (r - TM);
            const bool there = (w ? j0 + r < p.out : n0 + (r - TM) < end) && k < p.cols;
            float v[4] = {};
            if (there) {
                decode4(*reinterpret_cast<const uint32_t *>((w ? p.w + row * p.w_pitch : p.x + row * p.x_pitch) + k), v);
                for (uint32_t q = 0; q < 4; q++) if (k + q >= p.cols) v[q] = 0.0f;
                if (c == 0) bytes[r] = (w ? p.w_scales : p.x_scales)[((uint64_t)(b / 4) * (w ? p.w_rows : p.N) + row) * 4 + b % 4];
            }
            for (uint32_t q = 0; q < 4; q++) if (w) ws[c + q][r] = v[q]; else xs[c + q][r - TM] = v[q];
        }
        __syncthreads();
        for (uint32_t k = 0; k < TK; k++) {
            const float4 a = *reinterpret_cast<const float4 *>(&xs[k][warp * 4]), b4 = *reinterpret_cast<const float4 *>(&ws[k][lane * 4]);
            const float x[4] = { a.x, a.y, a.z, a.w }, w[4] = { b4.x, b4.y, b4.z, b4.w };
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) sub[i][j] = fmaf(x[i], w[j], sub[i][j]);
        }
        if (k0 % BLOCK == BLOCK - TK || k0 + TK >= p.cols) {
            for (uint32_t i = 0; i < 4; i++)
                for (uint32_t j = 0; j < 4; j++) {
                    const uint32_t a = bytes[lane * 4 + j], c = bytes[TM + warp * 4 + i], half = (a + c) / 2;
                    acc[i][j] += a == 255u || c == 255u ? __uint_as_float(0x7fffffffu) : sub[i][j] * scale_value(half) * scale_value(a + c - half);
                    sub[i][j] = 0.0f;
                }
        }
        __syncthreads();
    }
    for (uint32_t i = 0; i < 4; i++) {
        const uint32_t n = n0 + warp * 4 + i;
        if (n >= end) break;
        float v[4];
        uint32_t most = 0;
        for (uint32_t q = 0; q < 4; q++) {
            const uint32_t j = j0 + lane * 4 + q;
            v[q] = j < p.out ? spg_activate(acc[i][q] + (p.bias ? p.bias[(uint64_t)e * p.out + j] : 0.0f), p.act) : 0.0f;
            most = max(most, __float_as_uint(v[q]) & 0x7fffffffu);
            if (!p.y || j >= p.out) continue;
            const uint64_t at = (uint64_t)n * p.ldy + j;
            if (p.type == SPGK_T_F32) ((float *)p.y)[at] = v[q];
            else if (p.type == SPGK_T_F16) ((__half *)p.y)[at] = from_f32<__half>(v[q]);
            else ((__nv_bfloat16 *)p.y)[at] = from_f32<__nv_bfloat16>(v[q]);
        }
        if (p.next_codes) {
            const uint32_t byte = scale_byte(__reduce_max_sync(0xffffffffu, most)), b = j0 / BLOCK;
            const float inv = inverse_scale(byte);
            const uint32_t code = byte == 255u ? 0u : encode4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
            if (j0 + lane * 4 < (p.out + 15) / 16 * 16) *reinterpret_cast<uint32_t *>(p.next_codes + (uint64_t)n * p.next_pitch + j0 + lane * 4) = code;
            if (lane == 0) p.next_scales[((uint64_t)(b / 4) * p.N + n) * 4 + b % 4] = (uint8_t)byte;
        }
    }
}

int refuse(const char *who, const char *why) { spgk_set_error(who, why); return SPGK_E_ARG; }

int layers(const char *who, const spgk_fp8 *W, uint32_t experts, const float *bias, int act, const spgk_fp8 *X, const int32_t *starts,
           void *y, int type, uint32_t ldy, const spgk_fp8 *next, int32_t *status, void *stream)
{
    int rc;
    if ((rc = spg_fp8_check(who, W)) || (rc = spg_fp8_check(who, X))) return rc;
    if (next && (rc = spg_fp8_check(who, next))) return rc;
    if (W->rows == 0 || W->rows % experts || W->cols != X->cols) return refuse(who, "weights and inputs do not belong together");
    const uint32_t out = W->rows / experts;
    if (W->cols > (1u << 27)) return refuse(who, "more than 2^27 inputs");      // (a tile's products end well before the waits for them give up)
    if (act < SPG_ACT_SIGMOID || act > SPG_ACT_NONE) return refuse(who, "unknown activation");
    if (!y && !next) return refuse(who, "no output");
    if (y && type != SPGK_T_F16 && type != SPGK_T_BF16 && type != SPGK_T_F32) return refuse(who, "unknown type");
    if (y && (uintptr_t)y % (type == SPGK_T_F32 ? 4u : 2u)) return refuse(who, "output not aligned to its type");
    if (y && X->rows > 1 && ldy < out) return refuse(who, "rows of the output overlap");
    if (next && (next->rows != X->rows || next->cols != out)) return refuse(who, "the next operand has other rows or columns");
    if (next && act == SPG_ACT_SOFTMAX) return refuse(who, "a softmax is left to spgk_softmax_rows");
    if (!status || (uintptr_t)status % 4u) return refuse(who, "no status word");
    if ((uintptr_t)bias % 4u) return refuse(who, "bias not aligned");
    if (X->rows == 0) return SPGK_OK;
    LayerParams p{};
    p.N = X->rows; p.out = out; p.cols = W->cols; p.experts = experts; p.w_rows = W->rows;
    p.w = (const uint8_t *)W->codes; p.x = (const uint8_t *)X->codes; p.w_pitch = W->pitch; p.x_pitch = X->pitch;
    p.w_scales = (const uint8_t *)W->scales; p.x_scales = (const uint8_t *)X->scales;
    p.starts = starts; p.bias = bias; p.act = act; p.y = y; p.type = type; p.ldy = ldy;
    if (next) { p.next_codes = (uint8_t *)next->codes; p.next_scales = (uint8_t *)next->scales; p.next_pitch = next->pitch; }
    const uint64_t tiles = (uint64_t)p.N / TN + (experts < p.N ? experts : p.N) + 1;
    if (tiles > 65535u) return refuse(who, "too many tiles of rows");
    SPGK_CUDA(spg_launch_chained(spg_fp8_layer_kernel, dim3((out + TM - 1) / TM, (uint32_t)tiles), dim3(THREADS), 0, (cudaStream_t)stream, p));
    return spgk_check_launch("spg_fp8_layer_kernel");
}

}  // namespace

extern "C" {

int spgk_layer_fp8(const spgk_fp8 *W, const float *bias, int act, const spgk_fp8 *X, void *y, int type, uint32_t ldy, const spgk_fp8 *next, int32_t *status, void *stream)
{
    return layers("spgk_layer_fp8", W, 1, bias, act, X, nullptr, y, type, ldy, next, status, stream);
}

int spgk_experts_fp8(const spgk_fp8 *W, uint32_t experts, const float *bias, int act, const spgk_fp8 *X, const int32_t *starts,
                     void *y, int type, uint32_t ldy, const spgk_fp8 *next, int32_t *status, void *stream)
{
    if (experts == 0 || experts > SPGK_MAX_EXPERTS) return refuse("spgk_experts_fp8", "no experts, or too many");
    if (!starts || (uintptr_t)starts % 4u) return refuse("spgk_experts_fp8", "no starts, or not aligned");
    return layers("spgk_experts_fp8", W, experts, bias, act, X, starts, y, type, ldy, next, status, stream);
}

}  // extern "C"
