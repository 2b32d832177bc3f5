// spg_route.cu -- rows to experts and back: a router's choice, the order of the rows by expert, and the weighted sum of what the experts made of them.
//
//   choice : the first top_k of a row by (logit, falling; index, rising); gate = exp(l - m) / sum
//   order  : place(n, j) = starts[e] + how many pairs in front of (n, j), in the order of the rows, have the same expert e = chosen[n][j]
//   sum    : out[n] = sum_j gate[n][j] * y[place[n][j]]
//
// A warp has a row of logits, up to 32 a lane, and takes its largest out one after the other.  The order is a counting sort by one cluster of up to eight
// blocks: warps count their part of the pairs, what is in front of a warp is summed up in shared memory, what is in front of a block over the cluster, and
// each warp walks its part once more.  Neither hangs on the order in which anything runs.
#include "spg_fp8.cuh"

namespace {

using namespace spgfp8;

constexpr uint32_t CHOOSE_THREADS = 256;
constexpr uint32_t SORT_WARPS = 32, SORT_THREADS = 32 * SORT_WARPS, SORT_CLUSTER = 8;

// order of floats as that of unsigned numbers; -infinity comes lowest, above 0, which no logit has
__device__ __forceinline__ uint32_t key_of(float v)
{
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
constexpr uint32_t KEY_CLOSED = 0x007fffffu;                    // of -infinity

// one row by one warp; V: logits a lane
template <typename T, uint32_t V>
__device__ __forceinline__ void choose(const T *row, uint32_t experts, uint32_t top_k, bool normalise, int32_t *chosen, float *gates, uint32_t lane)
{
    uint32_t key[V];
    uint32_t most = 0;
#pragma unroll
    for (uint32_t i = 0; i < V; i++) {
        const uint32_t e = i * 32u + lane;
        float l = e < experts ? to_f32(row[e]) : __int_as_float(0xff800000);
        l = l == l ? l + 0.0f : __int_as_float(0xff800000);     // (-0 is 0)
        key[i] = e < experts ? key_of(l) : 0u;
        most = max(most, key[i]);
    }
    const uint32_t first = __reduce_max_sync(0xffffffffu, most);
    const float m = value_of(first);
    const auto weight = [&](uint32_t k) { return k == first ? 1.0f : k <= KEY_CLOSED ? 0.0f : expf(value_of(k) - m); };
    float total = 0.0f;
    if (!normalise) {
#pragma unroll
        for (uint32_t i = 0; i < V; i++) total += weight(key[i]);
        total = spg_warp_sum(total);
    }
    int32_t mine = -1;
    float w = 0.0f;
    for (uint32_t j = 0; j < top_k; j++) {
        uint32_t best = 0, at = 0;
#pragma unroll
        for (uint32_t i = 0; i < V; i++) if (key[i] > best) { best = key[i]; at = i; }
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        if (top <= KEY_CLOSED) break;
        const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? at * 32u + lane : 0xffffffffu);
#pragma unroll
        for (uint32_t i = 0; i < V; i++) if (i * 32u + lane == e) key[i] = 0;
        const float v = weight(top);
        if (normalise) total += v;
        if (lane == j) { mine = (int32_t)e; w = v; }
    }
    if (lane < top_k) { chosen[lane] = mine; gates[lane] = mine >= 0 ? w / total : 0.0f; }
}

template <typename T, uint32_t V>
__global__ void __launch_bounds__(CHOOSE_THREADS) spg_route_choose_kernel(const T *logits, uint32_t ld, uint32_t N, uint32_t experts, uint32_t top_k, int normalise, int32_t *chosen, float *gates)
{
    spg_grid_trigger();
    spg_grid_wait();
    const uint32_t n = blockIdx.x * (CHOOSE_THREADS / 32u) + threadIdx.x / 32u;
    if (n < N) choose<T, V>(logits + (uint64_t)n * ld, experts, top_k, normalise, chosen + (uint64_t)n * top_k, gates + (uint64_t)n * top_k, threadIdx.x % 32u);
}

__device__ __forceinline__ uint32_t ld_cluster(const uint32_t *here, uint32_t rank)
{
    uint32_t addr = (uint32_t)__cvta_generic_to_shared(here), v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// shared memory: [SORT_WARPS][experts] pairs in front of a warp, [experts] pairs of the block, [experts] first places, [SORT_WARPS] sums of warps
__global__ void __launch_bounds__(SORT_THREADS) spg_route_order_kernel(const int32_t *chosen, uint32_t pairs, uint32_t experts, uint32_t top_k, int32_t *starts, int32_t *order, int32_t *places)
{
    extern __shared__ uint32_t sh[];
    uint32_t *counts = sh, *all = counts + SORT_WARPS * experts, *base = all + experts, *sums = base + experts;
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, rank = blockIdx.x, blocks = gridDim.x;
    spg_grid_trigger();
    for (uint32_t i = threadIdx.x; i < SORT_WARPS * experts; i += SORT_THREADS) counts[i] = 0;
    __syncthreads();
    spg_grid_wait();
    // this warp's pairs: whole turns of 32
    const uint32_t turns = (pairs + 31u) / 32u, per = (turns + blocks * SORT_WARPS - 1) / (blocks * SORT_WARPS);
    const uint32_t lo = min(turns, (rank * SORT_WARPS + warp) * per) * 32u, hi = min(pairs, lo + per * 32u);
    uint32_t *mine = counts + warp * experts;
    for (uint32_t i = lo + lane; i < hi; i += 32u) {
        const int32_t e = chosen[i];
        if (e >= 0) atomicAdd(mine + e, 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += SORT_THREADS) {
        uint32_t sum = 0;
        for (uint32_t w = 0; w < SORT_WARPS; w++) { const uint32_t c = counts[w * experts + e]; counts[w * experts + e] = sum; sum += c; }
        all[e] = sum;
    }
    cluster_sync();
    // first places: the experts in front (a scan; thread e has expert e), then the blocks in front
    uint32_t before = 0, whole = 0;
    if (threadIdx.x < experts)
        for (uint32_t r = 0; r < blocks; r++) {
            const uint32_t c = ld_cluster(all + threadIdx.x, r);
            whole += c;
            if (r < rank) before += c;
        }
    uint32_t upto = whole;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= (uint32_t)o) upto += v; }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    uint32_t front = 0, total = 0;
    for (uint32_t w = 0; w < SORT_WARPS; w++) { const uint32_t s = sums[w]; if (w < warp) front += s; total += s; }
    if (threadIdx.x < experts) {
        base[threadIdx.x] = front + upto - whole + before;
        if (rank == 0) starts[threadIdx.x] = (int32_t)(front + upto - whole);
    }
    if (rank == 0 && threadIdx.x == 0) starts[experts] = (int32_t)total;
    __syncthreads();
    for (uint32_t i0 = lo; i0 < hi; i0 += 32u) {
        const uint32_t i = i0 + lane;
        const int32_t e = i < hi ? chosen[i] : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        uint32_t at = 0;
        if (e >= 0) at = base[e] + mine[e] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (e >= 0 && (same >> lane) == 1u) mine[e] += __popc(same);              // (the last of its kind)
        __syncwarp();
        if (i < hi) places[i] = e >= 0 ? (int32_t)at : -1;
        if (e >= 0) order[at] = (int32_t)(i / top_k);
    }
    for (uint32_t i = total + rank * SORT_THREADS + threadIdx.x; i < pairs; i += blocks * SORT_THREADS) order[i] = -1;
    cluster_sync();                                              // (the others may still read this block's sums)
}

// A thread has 16 bytes of a row's output, or one element where rows do not lie on 16 bytes.
template <typename T, typename O, uint32_t W>
__global__ void __launch_bounds__(256) spg_combine_kernel(const T *y, uint32_t ldy, uint32_t y_rows, const int32_t *places, const float *gates, uint32_t N, uint32_t top_k, uint32_t width,
                                                          O *out, uint32_t ldo, uint32_t pieces)
{
    spg_grid_trigger();
    spg_grid_wait();
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint32_t n = (uint32_t)(i / pieces), c = (uint32_t)(i % pieces) * W;
    if (n >= N) return;
    float v[W];
#pragma unroll
    for (uint32_t q = 0; q < W; q++) v[q] = 0.0f;
    for (uint32_t j = 0; j < top_k; j++) {
        const uint32_t p = (uint32_t)places[(uint64_t)n * top_k + j];
        if (p >= y_rows) continue;
        const float g = gates[(uint64_t)n * top_k + j];
        const T *row = y + (uint64_t)p * ldy + c;
        alignas(16) T t[W];
        if constexpr (W * sizeof(T) % 16 == 0) {
#pragma unroll
            for (uint32_t q = 0; q < W * sizeof(T) / 16; q++) reinterpret_cast<uint4 *>(t)[q] = reinterpret_cast<const uint4 *>(row)[q];
        } else {
#pragma unroll
            for (uint32_t q = 0; q < W; q++) t[q] = row[q];
        }
#pragma unroll
        for (uint32_t q = 0; q < W; q++) v[q] = fmaf(g, to_f32(t[q]), v[q]);
    }
    O *dst = out + (uint64_t)n * ldo + c;
    alignas(16) O o[W];
#pragma unroll
    for (uint32_t q = 0; q < W; q++) o[q] = from_f32<O>(v[q]);
    if constexpr (W * sizeof(O) % 16 == 0) {
#pragma unroll
        for (uint32_t q = 0; q < W * sizeof(O) / 16; q++) reinterpret_cast<uint4 *>(dst)[q] = reinterpret_cast<const uint4 *>(o)[q];
    } else {
#pragma unroll
        for (uint32_t q = 0; q < W; q++) dst[q] = o[q];
    }
}

int refuse(const char *who, const char *why) { spgk_set_error(who, why); return SPGK_E_ARG; }
bool known(int type) { return type == SPGK_T_F16 || type == SPGK_T_BF16 || type == SPGK_T_F32; }
uint32_t size_of(int type) { return type == SPGK_T_F32 ? 4u : 2u; }

template <typename T, uint32_t V>
int choose_all(const void *logits, uint32_t ld, uint32_t N, uint32_t experts, uint32_t top_k, int normalise, int32_t *chosen, float *gates, cudaStream_t stream)
{
    constexpr uint32_t rows = CHOOSE_THREADS / 32u;
    SPGK_CUDA(spg_launch_chained(spg_route_choose_kernel<T, V>, dim3((N + rows - 1) / rows), dim3(CHOOSE_THREADS), 0, stream, (const T *)logits, ld, N, experts, top_k, normalise, chosen, gates));
    return spgk_check_launch("spg_route_choose_kernel");
}
template <typename T>
int choose_all(const void *logits, uint32_t ld, uint32_t N, uint32_t experts, uint32_t top_k, int normalise, int32_t *chosen, float *gates, cudaStream_t stream)
{
    if (experts <= 64) return choose_all<T, 2>(logits, ld, N, experts, top_k, normalise, chosen, gates, stream);
    if (experts <= 256) return choose_all<T, 8>(logits, ld, N, experts, top_k, normalise, chosen, gates, stream);
    return choose_all<T, 32>(logits, ld, N, experts, top_k, normalise, chosen, gates, stream);
}

template <typename T, typename O>
int combine(const void *y, uint32_t ldy, uint32_t y_rows, const int32_t *places, const float *gates, uint32_t N, uint32_t top_k, uint32_t width, void *out, uint32_t ldo, cudaStream_t stream)
{
    constexpr uint32_t W = 16 / (sizeof(T) < sizeof(O) ? sizeof(T) : sizeof(O));
    const bool wide = width % W == 0 && (uint64_t)ldy * sizeof(T) % 16 == 0 && (uint64_t)ldo * sizeof(O) % 16 == 0 && ((uintptr_t)y | (uintptr_t)out) % 16 == 0;
    const uint32_t pieces = wide ? width / W : width;
    const uint64_t blocks = ((uint64_t)N * pieces + 255) / 256;
    if (blocks > 0x7fffffffu) return refuse("spgk_combine_rows", "too many rows and columns for one call");
    SPGK_CUDA(spg_launch_chained(wide ? spg_combine_kernel<T, O, W> : spg_combine_kernel<T, O, 1>, dim3((uint32_t)blocks), dim3(256), 0, stream,
                                 (const T *)y, ldy, y_rows, places, gates, N, top_k, width, (O *)out, ldo, pieces));
    return spgk_check_launch("spg_combine_kernel");
}
template <typename T>
int combine(const void *y, uint32_t ldy, uint32_t y_rows, const int32_t *places, const float *gates, uint32_t N, uint32_t top_k, uint32_t width, void *out, int type, uint32_t ldo, cudaStream_t stream)
{
    if (type == SPGK_T_F32) return combine<T, float>(y, ldy, y_rows, places, gates, N, top_k, width, out, ldo, stream);
    if (type == SPGK_T_F16) return combine<T, __half>(y, ldy, y_rows, places, gates, N, top_k, width, out, ldo, stream);
    return combine<T, __nv_bfloat16>(y, ldy, y_rows, places, gates, N, top_k, width, out, ldo, stream);
}

}  // namespace

extern "C" {

int spgk_route_rows(const void *logits, int type, uint32_t ld, uint32_t N, uint32_t experts, uint32_t top_k, int normalise,
                    int32_t *chosen, float *gates, int32_t *starts, int32_t *order, int32_t *places, void *stream)
{
    const char *who = "spgk_route_rows";
    if (!known(type)) return refuse(who, "unknown type");
    if (experts == 0 || experts > SPGK_MAX_EXPERTS) return refuse(who, "no experts, or too many");
    if (top_k == 0 || top_k > SPGK_ROUTE_MAX_TOP || top_k > experts) return refuse(who, "no choice, or of too many");
    if ((uint64_t)N * top_k >= (1u << 30)) return refuse(who, "too many rows");
    if (!starts || (N && (!logits || !chosen || !gates || !order || !places))) return refuse(who, "no logits, or no place for a result");
    if ((uintptr_t)logits % size_of(type) || ((uintptr_t)chosen | (uintptr_t)gates | (uintptr_t)starts | (uintptr_t)order | (uintptr_t)places) % 4u) return refuse(who, "not aligned");
    if (N > 1 && ld < experts) return refuse(who, "rows overlap");
    cudaStream_t st = (cudaStream_t)stream;
    int rc = SPGK_OK;
    if (N) {
        if (type == SPGK_T_F32) rc = choose_all<float>(logits, ld, N, experts, top_k, normalise, chosen, gates, st);
        else if (type == SPGK_T_F16) rc = choose_all<__half>(logits, ld, N, experts, top_k, normalise, chosen, gates, st);
        else rc = choose_all<__nv_bfloat16>(logits, ld, N, experts, top_k, normalise, chosen, gates, st);
        if (rc) return rc;
    }
    const uint32_t pairs = N * top_k, cluster = pairs > 4096u ? SORT_CLUSTER : 1u;
    const size_t bytes = ((size_t)(SORT_WARPS + 2) * experts + SORT_WARPS) * 4u;
    int dev = 0;
    SPGK_CUDA(cudaGetDevice(&dev));
    static SpgOncePerDevice once;
    rc = once.run(dev, [&]() -> int {
        SPGK_CUDA(cudaFuncSetAttribute(spg_route_order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(((SORT_WARPS + 2) * SPGK_MAX_EXPERTS + SORT_WARPS) * 4u)));
        return SPGK_OK;
    });
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster); cfg.blockDim = dim3(SORT_THREADS); cfg.dynamicSmemBytes = bytes; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    SPGK_CUDA(cudaLaunchKernelEx(&cfg, spg_route_order_kernel, (const int32_t *)chosen, pairs, experts, top_k, starts, order, places));
    return spgk_check_launch("spg_route_order_kernel");
}

int spgk_combine_rows(const void *y, int type, uint32_t ldy, uint32_t y_rows, const int32_t *places, const float *gates, uint32_t N, uint32_t top_k,
                      uint32_t width, void *out, int out_type, uint32_t ldo, void *stream)
{
    const char *who = "spgk_combine_rows";
    if (!known(type) || !known(out_type)) return refuse(who, "unknown type");
    if (top_k == 0 || width == 0) return refuse(who, "nothing to add up");
    if (N == 0) return SPGK_OK;
    if ((!y && y_rows) || !places || !gates || !out) return refuse(who, "no rows, places, gates or output");
    if ((uintptr_t)y % size_of(type) || (uintptr_t)out % size_of(out_type) || ((uintptr_t)places | (uintptr_t)gates) % 4u) return refuse(who, "not aligned");
    if (y_rows > 0x80000000u) return refuse(who, "more rows than a place can name");
    if ((y_rows > 1 && ldy < width) || (N > 1 && ldo < width)) return refuse(who, "rows overlap");
    if (type == SPGK_T_F32) return combine<float>(y, ldy, y_rows, places, gates, N, top_k, width, out, out_type, ldo, (cudaStream_t)stream);
    if (type == SPGK_T_F16) return combine<__half>(y, ldy, y_rows, places, gates, N, top_k, width, out, out_type, ldo, (cudaStream_t)stream);
    return combine<__nv_bfloat16>(y, ldy, y_rows, places, gates, N, top_k, width, out, out_type, ldo, (cudaStream_t)stream);
}

}  // extern "C"
