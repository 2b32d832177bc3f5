// spg_sample.cu -- a token drawn from every row of logits: temperature, top-k, top-p, min-p.
//
//   w_i = exp((l_i - m) / T), m the largest logit.  Ordered by (l falling, i rising) a row is cut after the first k logits, after the
//   shortest beginning with p of their weight, after the last w_i >= min_p; the token is the first index at which the running sum of the
//   weights that are left exceeds u times their total.
//
// All three cuts leave a beginning of the same order, so what is left is told by one key and a number: the logits above the key, and the first r of
// those equal to it.  Nothing is sorted.  A row belongs to a cluster of up to eight CTAs and is read once, into shared memory, as integers
// in the order of the logits; a cut is found by a histogram over the range in question (counts for top-k, weights for top-p), a closer look at the bin
// in which the border falls, and so on until few enough are left to be counted bit by bit.
// Weights are whole multiples of 2^-44 (of the largest, which is 1): their sums do not hang on an order, and they err by less than the sums of
// 131072 weights in 32 bits by a factor of 10^4, which would put a number drawn close to a border on its wrong side in some rows of a hundred.
#include "spg_common.cuh"
#include "spg_tc.cuh"
#include <algorithm>

namespace {

using spgtc::smem_u32; using spgtc::mapa; using spgtc::cluster_rank;

constexpr uint32_t THREADS = 512, WARPS = THREADS / 32;
constexpr uint32_t BINS = 512;
constexpr uint32_t LIST = 2048;               // logits of a range that are counted bit by bit
constexpr uint32_t MAX_SPLIT = 8;
constexpr uint32_t SLICE = SPGK_SAMPLE_MAX_WIDTH / MAX_SPLIT;
constexpr uint32_t BELOW = 0x007fffffu;       // key of -infinity: no logit at or below it takes part
constexpr int ONE_BITS = 44;
static_assert(BINS == THREADS && LIST % THREADS == 0, "a thread a bin");

struct SampleParams {
    const void *logits; int type; uint32_t ld, N, width, split, slice;
    const float *temperature; const int32_t *top_k; const float *top_p, *min_p, *u;
    int32_t *tokens; float *probs; int32_t *kept;
};

// order-preserving integer of a logit; a NaN like -infinity; -0 like 0
__device__ __forceinline__ uint32_t key_of(float l)
{
    if (!(l >= -INFINITY)) return BELOW;
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

struct Weights {
    double m, inv_t;
    uint32_t top;
    __device__ __forceinline__ uint64_t operator()(uint32_t key) const
    {
        if (key == top) return 1ull << ONE_BITS;
        if (isinf(m)) return 0;
        return __double2ull_rn(exp(((double)logit_of(key) - m) * inv_t) * (double)(1ull << ONE_BITS));
    }
};

struct Shared {
    uint64_t mass[BINS];
    uint32_t count[BINS];
    uint32_t list[LIST];
    uint64_t out[2][4];                        // what this CTA tells the others, by turns
    uint64_t warp_a[WARPS], warp_b[WARPS];
    uint32_t listed;
    uint32_t found_bin; uint64_t found_above; uint32_t found_count;
};

__device__ __forceinline__ uint64_t ld_cluster_u64(uint32_t addr)
{
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr)
{
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

struct Row {
    Shared &s;
    const uint32_t *keys;
    uint32_t n, split, rank, turn;             // keys of this CTA; CTAs of the row

    __device__ __forceinline__ void sync() { if (split > 1) spgtc::cluster_sync(); else __syncthreads(); }
    __device__ __forceinline__ uint64_t sum_warp(uint64_t v)
    {
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    // sum over the CTA, to all threads
    __device__ __forceinline__ uint64_t sum_cta(uint64_t v)
    {
        v = sum_warp(v);
        __syncthreads();
        if (threadIdx.x % 32 == 0) s.warp_a[threadIdx.x / 32] = v;
        __syncthreads();
        uint64_t r = 0;
        for (uint32_t i = 0; i < WARPS; i++) r += s.warp_a[i];
        return r;
    }
    __device__ __forceinline__ uint32_t max_cta(uint32_t v)
    {
        v = __reduce_max_sync(0xffffffffu, v);
        __syncthreads();
        if (threadIdx.x % 32 == 0) s.warp_a[threadIdx.x / 32] = v;
        __syncthreads();
        uint32_t r = 0;
        for (uint32_t i = 0; i < WARPS; i++) r = max(r, (uint32_t)s.warp_a[i]);
        return r;
    }
    // three values of every CTA (the same in all its threads) to every CTA
    __device__ __forceinline__ void tell(uint64_t a, uint64_t b, uint64_t c)
    {
        turn ^= 1;
        if (threadIdx.x == 0) { s.out[turn][0] = a; s.out[turn][1] = b; s.out[turn][2] = c; }
        sync();
    }
    __device__ __forceinline__ uint64_t heard(uint32_t from, int which) { return ld_cluster_u64(mapa(smem_u32(&s.out[turn][which]), from)); }

    // The largest key v above `floor` with (amount of keys above v) < goal <= (amount of keys from v on), amounts being counts or weights;
    // goal >= 1 and no more than the amount of all keys above floor.  [lo, hi]: the smallest and the largest key above floor.  above: the amount above v.
    template <bool MASS> __device__ uint32_t select(const Weights &w, uint32_t lo, uint32_t hi, uint64_t goal, uint64_t &above)
    {
        above = 0;
        for (bool first = true; lo < hi; first = false) {
            const float top = logit_of(hi), per = first ? (float)BINS / (top - logit_of(lo)) : 0.0f;
            const bool even = first && per > 0.0f && per < INFINITY;             // bins of equal width in the logits, else in the keys
            const uint64_t step = (((uint64_t)BINS << 32) - 1) / ((uint64_t)(hi - lo) + 1);
            const auto bin = [&](uint32_t key) -> uint32_t {
                if (even) return min(BINS - 1, (uint32_t)((top - logit_of(key)) * per));
                return (uint32_t)((hi - key) * step >> 32);
            };
            for (uint32_t i = threadIdx.x; i < BINS; i += THREADS) { s.count[i] = 0; s.mass[i] = 0; }
            if (threadIdx.x == 0) s.listed = 0;
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const uint32_t k = keys[i];
                if (k < lo || k > hi) continue;
                const uint32_t b = bin(k);
                atomicAdd(&s.count[b], 1u);
                if (MASS) atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)w(k));
            }
            sync();
            // the bin in which the goal is reached: a thread a bin
            uint64_t amount = 0; uint32_t count = 0;
            for (uint32_t r = 0; r < split; r++) {
                const uint32_t c = ld_cluster_u32(mapa(smem_u32(&s.count[threadIdx.x]), r));
                count += c;
                amount += MASS ? ld_cluster_u64(mapa(smem_u32(&s.mass[threadIdx.x]), r)) : c;
            }
            uint64_t upto = amount;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t v = __shfl_up_sync(0xffffffffu, upto, o);
                if (threadIdx.x % 32 >= (uint32_t)o) upto += v;
            }
            if (threadIdx.x % 32 == 31) s.warp_b[threadIdx.x / 32] = upto;
            __syncthreads();
            for (uint32_t i = 0; i < threadIdx.x / 32; i++) upto += s.warp_b[i];
            if (above + upto - amount < goal && above + upto >= goal && amount) { s.found_bin = threadIdx.x; s.found_above = above + upto - amount; s.found_count = count; }
            sync();                                                              // (the others have read this CTA's bins)
            const uint32_t b = s.found_bin, many = s.found_count;
            above = s.found_above;
            uint32_t least = 0xffffffffu, most = 0;
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const uint32_t k = keys[i];
                if (k < lo || k > hi || bin(k) != b) continue;
                least = min(least, k); most = max(most, k);
                if (many <= LIST) s.list[atomicAdd(&s.listed, 1u)] = k;
            }
            least = ~max_cta(~least); most = max_cta(most);
            tell(least, most, s.listed);
            lo = 0xffffffffu; hi = 0;
            for (uint32_t r = 0; r < split; r++) { lo = min(lo, (uint32_t)heard(r, 0)); hi = max(hi, (uint32_t)heard(r, 1)); }
            if (lo < hi && many <= LIST) {
                // every thread takes its part of all CTAs' lists, and the border is found bit by bit
                uint32_t mine[LIST / THREADS];
                uint64_t weigh[LIST / THREADS];
                uint32_t at = 0;
#pragma unroll
                for (uint32_t i = 0; i < LIST / THREADS; i++) { mine[i] = 0; weigh[i] = 0; }
                for (uint32_t r = 0; r < split; r++) {
                    const uint32_t c = (uint32_t)heard(r, 2);
#pragma unroll
                    for (uint32_t i = 0; i < LIST / THREADS; i++) {
                        const uint32_t want = i * THREADS + threadIdx.x;
                        if (want >= at && want < at + c) mine[i] = ld_cluster_u32(mapa(smem_u32(&s.list[want - at]), r));
                    }
                    at += c;
                }
#pragma unroll
                for (uint32_t i = 0; i < LIST / THREADS; i++) if (i * THREADS + threadIdx.x < at) weigh[i] = MASS ? w(mine[i]) : 1;
                // v = the largest key with amount(>= v) reaching the goal
                uint32_t bit = 1u << (31 - __clz((int)(hi ^ lo))), v = lo & ~(2u * bit - 1u);
                for (; bit; bit >>= 1) {
                    const uint32_t trial = v | bit;
                    if (trial > hi) continue;
                    uint64_t a = 0;
#pragma unroll
                    for (uint32_t i = 0; i < LIST / THREADS; i++) if (mine[i] >= trial) a += weigh[i];
                    if (above + sum_cta(a) >= goal) v = trial;
                }
                uint64_t a = 0;
#pragma unroll
                for (uint32_t i = 0; i < LIST / THREADS; i++) if (mine[i] > v) a += weigh[i];
                above += sum_cta(a);
                lo = hi = v;
            }
            sync();                                                              // (lists and bins are free again)
        }
        return lo;
    }
};

template <typename T> __device__ __forceinline__ float logit(const T *x, uint64_t at);
template <> __device__ __forceinline__ float logit<float>(const float *x, uint64_t at) { return __ldg(x + at); }
template <> __device__ __forceinline__ float logit<__half>(const __half *x, uint64_t at) { return __half2float(x[at]); }
template <> __device__ __forceinline__ float logit<__nv_bfloat16>(const __nv_bfloat16 *x, uint64_t at) { return __bfloat162float(x[at]); }

template <typename T>
__global__ void __launch_bounds__(THREADS) spg_sample_kernel(const SampleParams p)
{
    extern __shared__ __align__(16) uint8_t raw[];
    Shared &s = *reinterpret_cast<Shared *>(raw);
    uint32_t *keys = reinterpret_cast<uint32_t *>(raw + sizeof(Shared));
    const uint32_t row = blockIdx.x / p.split, rank = blockIdx.x % p.split, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t from = min(p.width, rank * p.slice), n = min(p.width - from, p.slice);
    spg_grid_wait();
    Row R{ s, keys, n, p.split, rank, 0 };

    // the row, its largest and smallest logits and how many there are
    const T *x = reinterpret_cast<const T *>(p.logits) + (uint64_t)row * p.ld + from;
    uint32_t most = 0, least = 0xffffffffu, have = 0;
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
        const uint32_t k = key_of(logit<T>(x, i));
        keys[i] = k;
        if (k > BELOW) { most = max(most, k); least = min(least, k); have++; }
    }
    most = R.max_cta(most); least = ~R.max_cta(~least);
    have = (uint32_t)R.sum_cta(have);
    R.tell(most, least, have);
    uint32_t top = 0, low = 0xffffffffu, all = 0;
    for (uint32_t r = 0; r < p.split; r++) { top = max(top, (uint32_t)R.heard(r, 0)); low = min(low, (uint32_t)R.heard(r, 1)); all += (uint32_t)R.heard(r, 2); }

    const float t = p.temperature ? p.temperature[row] : 1.0f;
    const bool greedy = !(t > 0.0f);
    Weights w{ (double)logit_of(top), 1.0 / (double)t, top };
    // what is left: keys above `cut`, and the first `ties` keys equal to it
    uint32_t cut = BELOW, ties = 0;
    if (all && greedy) { cut = top; ties = 1; }
    if (all && !greedy) {
        const int32_t k = p.top_k ? p.top_k[row] : 0;
        if (k >= 1 && (uint32_t)k < all) {
            uint64_t above;
            cut = R.select<false>(w, low, top, (uint64_t)k, above);
            ties = (uint32_t)(k - above);
        }
        const float pp = p.top_p ? p.top_p[row] : 1.0f;
        if (pp < 1.0f) {
            uint64_t sum = 0;
            uint32_t nearest = 0xffffffffu;
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) if (keys[i] > cut) { sum += w(keys[i]); nearest = min(nearest, keys[i]); }
            sum = R.sum_cta(sum); nearest = ~R.max_cta(~nearest);
            R.tell(sum, nearest, 0);
            sum = 0; nearest = 0xffffffffu;
            for (uint32_t r = 0; r < p.split; r++) { sum += R.heard(r, 0); nearest = min(nearest, (uint32_t)R.heard(r, 1)); }
            const uint64_t each = ties ? w(cut) : 0;
            const double want = ceil((double)pp * (double)(sum + ties * each));
            const uint64_t goal = want >= 1.0 ? (uint64_t)want : 1;
            if (sum < goal) ties = (uint32_t)min((uint64_t)ties, (goal - sum + each - 1) / max(each, (uint64_t)1));
            else {
                uint64_t above;
                cut = R.select<true>(w, nearest, top, goal, above);
                const uint64_t one = w(cut);
                ties = (uint32_t)((goal - above + one - 1) / one);
            }
        }
        const float mp = p.min_p ? p.min_p[row] : 0.0f;
        if (mp > 0.0f) {
            // the smallest key whose weight is at least mp, by halving
            if (mp > 1.0f) { cut = top; ties = 1; }
            else {
                const double least_d = log((double)mp);
                uint32_t a = BELOW, b = top;                                     // a: too light, b: heavy enough
                while (b - a > 1) {
                    const uint32_t mid = a + (b - a) / 2;
                    const bool heavy = !isinf(w.m) && ((double)logit_of(mid) - w.m) * w.inv_t >= least_d;
                    if (heavy) b = mid; else a = mid;
                }
                if (b - 1 >= cut) { cut = b - 1; ties = 0; }
            }
        }
    }

    // Sums of what is left, for every warp's part of the slice (parts lie in the order of the vocabulary)
    const uint32_t part = (n + WARPS - 1) / WARPS, begin = min(n, warp * part), end = min(n, begin + part);
    uint32_t equal = 0;
    if (ties) for (uint32_t i = begin + lane; i < end; i += 32) equal += keys[i] == cut;
    equal = __reduce_add_sync(0xffffffffu, equal);
    __syncthreads();
    if (lane == 0) s.warp_b[warp] = equal;
    __syncthreads();
    uint32_t equal_before = 0, equal_cta = 0;
    for (uint32_t i = 0; i < WARPS; i++) { if (i < warp) equal_before += (uint32_t)s.warp_b[i]; equal_cta += (uint32_t)s.warp_b[i]; }
    R.tell(equal_cta, 0, 0);
    for (uint32_t r = 0; r < rank; r++) equal_before += (uint32_t)R.heard(r, 0);
    const uint64_t each = ties ? w(cut) : 0;
    uint32_t ties_here = ties > equal_before ? min(equal, ties - equal_before) : 0;
    uint64_t sum = 0;
    uint32_t left = 0;
    for (uint32_t i = begin + lane; i < end; i += 32) if (keys[i] > cut) { sum += w(keys[i]); left++; }
    sum = R.sum_warp(sum) + ties_here * each;
    left = __reduce_add_sync(0xffffffffu, left) + ties_here;
    __syncthreads();
    if (lane == 0) { s.warp_a[warp] = sum; s.warp_b[warp] = left; }
    __syncthreads();
    uint64_t before = 0, cta = 0, left_cta = 0;
    for (uint32_t i = 0; i < WARPS; i++) { if (i < warp) before += s.warp_a[i]; cta += s.warp_a[i]; left_cta += s.warp_b[i]; }
    R.tell(cta, left_cta, 0);
    uint64_t total = 0, left_all = 0;
    for (uint32_t r = 0; r < p.split; r++) { if (r < rank) before += R.heard(r, 0); total += R.heard(r, 0); left_all += R.heard(r, 1); }

    if (total == 0) {
        if (rank == 0 && threadIdx.x == 0) { p.tokens[row] = -1; if (p.probs) p.probs[row] = 0.0f; if (p.kept) p.kept[row] = 0; }
    } else {
        const float u = p.u[row];
        const double goal_d = (u > 0.0f ? (double)u : 0.0) * (double)total;
        const uint64_t goal = goal_d >= (double)(total - 1) ? total - 1 : (uint64_t)goal_d;
        if (before <= goal && goal < before + sum) {                             // in this warp's part
            uint64_t run = before;
            uint32_t seen = equal_before;
            for (uint32_t i0 = begin; i0 < end; i0 += 32) {
                const uint32_t i = i0 + lane, k = i < end ? keys[i] : 0;
                const uint32_t same = __ballot_sync(0xffffffffu, k == cut);
                const bool tie = k == cut && seen + __popc(same & ((1u << lane) - 1)) < ties;
                const uint64_t one = k > cut ? w(k) : (tie ? each : 0);
                uint64_t upto = one;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint64_t v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= (uint32_t)o) upto += v;
                }
                const uint32_t over = __ballot_sync(0xffffffffu, run + upto > goal);
                if (over) {
                    if (lane == (uint32_t)__ffs((int)over) - 1) {
                        p.tokens[row] = (int32_t)(from + i);
                        if (p.probs) p.probs[row] = (float)((double)one / (double)total);
                        if (p.kept) p.kept[row] = (int32_t)left_all;
                    }
                    break;
                }
                run += __shfl_sync(0xffffffffu, upto, 31);
                seen += __popc(same);
            }
        }
    }
    R.sync();                                                                    // (nobody leaves while its shared memory is read)
}

template <typename T> int launch(SampleParams p, const SpgDeviceProps &dp, int dev, cudaStream_t stream)
{
    static SpgOncePerDevice once;
    const int rc = once.run(dev, [&]() -> int {
        SPGK_CUDA(cudaFuncSetAttribute(spg_sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dp.smem_optin));
        return SPGK_OK;
    });
    if (rc) return rc;
    p.split = 1;
    while (p.split < MAX_SPLIT && (p.width > p.split * SLICE || (p.width > p.split * 2048u && (uint64_t)p.N * p.split * 2 <= (uint32_t)dp.sm_count * 2u))) p.split *= 2;
    p.slice = (p.width + p.split - 1) / p.split;
    if ((uint64_t)p.N * p.split > 0x7fffffffu) { spgk_set_error("spgk_sample_rows", "too many rows"); return SPGK_E_ARG; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.N * p.split); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = sizeof(Shared) + (size_t)p.slice * 4; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    SPGK_CUDA(cudaLaunchKernelEx(&cfg, spg_sample_kernel<T>, p));
    return spgk_check_launch("spg_sample_kernel");
}

}  // namespace

extern "C" int spgk_sample_rows(const void *logits, int type, uint32_t ld, uint32_t N, uint32_t width, const float *temperature,
                                const int32_t *top_k, const float *top_p, const float *min_p, const float *u,
                                int32_t *tokens, float *probs, int32_t *kept, void *stream)
{
    const char *why = nullptr;
    if (type != SPGK_T_F16 && type != SPGK_T_BF16 && type != SPGK_T_F32) why = "unknown type";
    else if (width == 0 || width > SPGK_SAMPLE_MAX_WIDTH) why = "width is 1 to SPGK_SAMPLE_MAX_WIDTH";
    else if (N && (!logits || !u || !tokens)) why = "no logits, no random numbers or nowhere to write";
    else if ((uintptr_t)logits % (type == SPGK_T_F32 ? 4u : 2u)) why = "logits not aligned to their type";
    else if (((uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)u | (uintptr_t)tokens | (uintptr_t)probs | (uintptr_t)kept) % 4u) why = "arrays not aligned";
    else if (N > 1 && ld < width) why = "rows overlap";
    if (why) { spgk_set_error("spgk_sample_rows", why); return SPGK_E_ARG; }
    if (N == 0) return SPGK_OK;
    SpgDeviceProps dp;
    int dev = 0;
    const int rc = spg_device_props(&dp);
    if (rc) return rc;
    SPGK_CUDA(cudaGetDevice(&dev));
    SampleParams p{ logits, type, ld, N, width, 1, width, temperature, top_k, top_p, min_p, u, tokens, probs, kept };
    if (type == SPGK_T_F32) return launch<float>(p, dp, dev, (cudaStream_t)stream);
    if (type == SPGK_T_F16) return launch<__half>(p, dp, dev, (cudaStream_t)stream);
    return launch<__nv_bfloat16>(p, dp, dev, (cudaStream_t)stream);
}
