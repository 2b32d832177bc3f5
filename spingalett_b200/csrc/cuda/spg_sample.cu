// spg_sample.cu -- a token drawn from every row of logits: temperature, top-k, top-p, min-p.
//
//   w_i = exp((l_i - m) / T), m the largest logit.  Ordered by (l falling, i rising) a row is cut after the first k logits, after the
//   shortest beginning with p of their weight, after the last w_i >= min_p; the token is the first index at which the running sum of the
//   weights that are left exceeds u times their total.
//
// All three cuts leave a beginning of the same order, so what is left is told by one logit and a number: the logits above it, and the first r of
// those equal to it.  Nothing is sorted.  A row belongs to a cluster of up to eight CTAs and is read once, into shared memory.
//   - A small top_k: each thread has the largest of its logits, and the (k / CTAs)-th largest of those in a CTA bounds the k-th logit of the row from
//     below; the few logits above the least of these bounds meet in one CTA, where every thread counts what stands before its own.
//   - Otherwise a cut is found by a histogram over the range in question (counts for top-k, weights for top-p), a closer look at the bins
//     in which the border may fall, and so on until few enough are left to be searched bit by bit.
// Sums of 131072 weights in 32 bits would put a number drawn close to a border on its wrong side in some rows of a hundred.  Here a weight is a
// whole multiple of 2^-44 (the largest is 1) that is good to 2^-30 of itself: errors that are independent of one another, so a sum of n of them is good to
// 2^-30 / sqrt(n), and sums in 64 bits that do not hang on an order.
#include "spg_common.cuh"
#include "spg_tc.cuh"
#include <algorithm>

namespace {

using spgtc::smem_u32; using spgtc::mapa; using spgtc::cluster_rank;

constexpr uint32_t THREADS = 512, WARPS = THREADS / 32;
constexpr uint32_t BINS = 512;
constexpr uint32_t LIST = 2048;               // logits of a range that are searched bit by bit
constexpr uint32_t FEW = 512;                 // logits among which every thread counts what stands before its own
constexpr uint32_t MAX_SPLIT = 8;
constexpr uint32_t SLICE = SPGK_SAMPLE_MAX_WIDTH / MAX_SPLIT;
constexpr int ONE_BITS = 44;
constexpr uint32_t STEPS = 1024;              // of the table of 2^(i / STEPS)
static_assert(BINS == THREADS && LIST % THREADS == 0 && FEW <= THREADS && STEPS % THREADS == 0, "a thread a bin, a logit, two steps");

struct SampleParams {
    const void *logits; int type; uint32_t ld, N, width, split, slice;
    const float *temperature; const int32_t *top_k; const float *top_p, *min_p, *u;
    int32_t *tokens; float *probs; int32_t *kept;
};

// a NaN like -infinity, -0 like 0
__device__ __forceinline__ float logit_of(float l) { return l >= -INFINITY ? l + 0.0f : -INFINITY; }
// integers in the order of the logits
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// exp((l - m) / T) as a multiple of 2^-44.  With c = log2(e) / T, l * c = K / 1024 + y for the nearest whole K: fma(l, c, -K / 1024) leaves a small number with
// all its bits, so y less that of m is good to 2^-34, and 2^(y) = 1 + p needs two terms: 2^(K / 1024) from a table in 31 bits, p in 24.
struct Weights {
    double m, inv_t;
    float top, c, c_lo, c_steps, floor, y_top;
    int k_top;
    bool fast;                                 // |m * c| is small enough for whole K / 1024 in 24 bits
    const uint32_t *table;

    static constexpr float MAGIC = 12582912.0f;            // 1.5 * 2^23: the sum's low bits are a whole number
    __device__ __forceinline__ float rest(float l, float kf) const { return fmaf(l, c_lo, fmaf(l, c, (kf - MAGIC) * (-1.0f / STEPS))); }
    __device__ __forceinline__ void set(float largest, float t, const uint32_t *tab)
    {
        top = largest; m = largest; inv_t = 1.0 / (double)t; table = tab;
        const double cd = 1.4426950408889634 * inv_t;
        fast = fabs(m) * cd <= 4000.0 && cd >= 1e-6 && cd <= 1e30;
        c = (float)cd; c_lo = (float)(cd - (double)c); c_steps = c * (float)STEPS;
        floor = (float)(m - 60.0 / cd);                      // weighs less than 2^-45
        const float kf = fmaf(top, c_steps, MAGIC);
        k_top = __float_as_int(kf);
        y_top = rest(top, kf);
    }
    // without the table; few calls
    __device__ __forceinline__ uint64_t exact(float l) const
    {
        if (l == top) return 1ull << ONE_BITS;
        if (isinf(top) || l == -INFINITY) return 0;
        return __double2ull_rn(exp(((double)l - m) * inv_t) * (double)(1ull << ONE_BITS));
    }
    __device__ __forceinline__ uint64_t operator()(float l) const
    {
        if (!fast) return exact(l);
        l = fmaxf(l, floor);
        const float kf = fmaf(l, c_steps, MAGIC);
        const float y = rest(l, kf) - y_top;
        const int k = __float_as_int(kf) - k_top;            // <= 0
        const uint32_t t = table[k & (int)(STEPS - 1)];
        const float p = y * fmaf(y, 0.24022650695910072f, 0.69314718055994531f);
        const uint32_t w = t + (uint32_t)__float2int_rn(__uint2float_rn(t) * p);      // [2^30, 2^31)
        const int up = (k >> 10) + (ONE_BITS - 30);
        return (uint64_t)(w >> min(max(-up, 0), 31)) * (uint64_t)(1u << max(up, 0));
    }
};

struct Item { float l; uint32_t index; uint64_t w; };

struct alignas(16) Shared {
    uint64_t mass[BINS];
    uint32_t count[BINS];
    union { uint32_t list[LIST]; Item few[FEW]; };
    uint32_t table[STEPS];
    uint64_t out[2][4];                        // what this CTA tells the others, by turns
    uint64_t warp_a[WARPS], warp_b[WARPS];
    uint32_t listed;
    uint32_t found_bin, found_last; uint64_t found_above; uint32_t found_count;
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
    const float *logits;
    uint32_t n, split, rank, turn;             // logits of this CTA; CTAs of the row

    __device__ __forceinline__ void sync() { if (split > 1) spgtc::cluster_sync(); else __syncthreads(); }
    __device__ __forceinline__ uint64_t sum_warp(uint64_t v)
    {
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    // over the CTA, to all threads
    __device__ __forceinline__ uint64_t sum_cta(uint64_t v)
    {
        v = sum_warp(v);
        __syncthreads();
        if (threadIdx.x % 32 == 0) s.warp_a[threadIdx.x / 32] = v;
        __syncthreads();
        uint64_t r = 0;
#pragma unroll
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
#pragma unroll
        for (uint32_t i = 0; i < WARPS; i++) r = max(r, (uint32_t)s.warp_a[i]);
        return r;
    }
    __device__ __forceinline__ uint64_t scan_cta(uint64_t v)                     // sum over the threads up to this one
    {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
            if (threadIdx.x % 32 >= (uint32_t)o) v += u;
        }
        __syncthreads();
        if (threadIdx.x % 32 == 31) s.warp_b[threadIdx.x / 32] = v;
        __syncthreads();
        for (uint32_t i = 0; i < threadIdx.x / 32; i++) v += s.warp_b[i];
        return v;
    }
    // up to four values of every CTA (the same in all its threads) to every CTA
    __device__ __forceinline__ void tell(uint64_t a, uint64_t b = 0, uint64_t c = 0, uint64_t d = 0)
    {
        turn ^= 1;
        if (threadIdx.x == 0) { s.out[turn][0] = a; s.out[turn][1] = b; s.out[turn][2] = c; s.out[turn][3] = d; }
        sync();
    }
    __device__ __forceinline__ uint64_t heard(uint32_t from, int which) { return ld_cluster_u64(mapa(smem_u32(&s.out[turn][which]), from)); }

    // [lo, hi] to the smallest and largest key in question, of which every CTA has told its own beside how many it has listed; where all are listed,
    // the border is found bit by bit: every thread takes its part of all CTAs' lists
    template <bool MASS> __device__ void search(const Weights &w, uint32_t &lo, uint32_t &hi, uint32_t many, uint64_t goal, uint64_t &above)
    {
        lo = 0xffffffffu; hi = 0;
        for (uint32_t r = 0; r < split; r++) { lo = min(lo, (uint32_t)heard(r, 0)); hi = max(hi, (uint32_t)heard(r, 1)); }
        if (lo >= hi || many > LIST) return;
        uint32_t mine[LIST / THREADS], at = 0;
        uint64_t weigh[LIST / THREADS];
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
        for (uint32_t i = 0; i < LIST / THREADS; i++) if (i * THREADS + threadIdx.x < at) weigh[i] = MASS ? w(of_key(mine[i])) : 1;
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

    // The largest key v above `cut` with (amount of keys above v) < goal <= (amount of keys from v on), amounts being counts or weights;
    // goal >= 1 and no more than the amount of all keys above cut.  [lo, hi]: the smallest and the largest key in question.  above: the amount above v.
    // MASS: `total` the weight of `have` logits at most above cut, share = goal / total
    template <bool MASS> __device__ uint32_t select(const Weights &w, uint32_t lo, uint32_t hi, uint64_t goal, uint64_t total, uint32_t have, double share, uint64_t &above)
    {
        above = 0;
        bool first = true;
        if (MASS && w.fast && lo < hi) {
            // Weights in 32 bits, a unit being 2^-30 of the total; a bin's amount is off by a unit and `off` of itself a logit at most.  Logits whose weights
            // come to less than (1 - share) / 2 of the total, all of them together, are left aside.
            const double cd = (double)w.c, one = (double)(1ull << ONE_BITS), light = 0.5 * fmax(1.0 - share, 0.0) * (double)total / (double)have / one;
            const float least = light > 0.0 ? fmaxf(of_key(lo), (float)(w.m + log(light) / w.inv_t)) : of_key(lo), top = of_key(hi), per = (float)BINS / (top - least);
            if (share < 1.0 - 1e-7 && per > 0.0f && per < INFINITY) {
                first = false;
                const float bias = (float)(30.0 - w.m * cd - log2((double)total / one));
                const double off = (fabs(w.m) * cd + 130.0) * 0x1p-21 + 0x1p-20, goal_units = (double)goal / (double)total * 0x1p30;
                const auto bin = [&](float l) { return min(BINS - 1, (uint32_t)((top - l) * per)); };
                s.count[threadIdx.x] = 0;
                if (threadIdx.x == 0) s.listed = 0;
                __syncthreads();
                for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                    const float l = logits[i];
                    if (l >= least && l <= top) {
                        float e;
                        asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(fmaf(l, w.c, bias)));
                        atomicAdd(&s.count[bin(l)], (uint32_t)e);
                    }
                }
                sync();
                uint32_t amount = 0;
                for (uint32_t r = 0; r < split; r++) amount += ld_cluster_u32(mapa(smem_u32(&s.count[threadIdx.x]), r));
                const uint64_t upto = scan_cta(amount);
                if (threadIdx.x == 0) { s.found_bin = BINS - 1; s.found_last = BINS - 1; }
                __syncthreads();
                if (((double)upto + (double)have) >= goal_units * (1.0 - off)) atomicMin(&s.found_bin, threadIdx.x);
                if ((double)upto >= goal_units * (1.0 + off)) atomicMin(&s.found_last, threadIdx.x);
                sync();
                const uint32_t b0 = s.found_bin, b1 = s.found_last;
                uint64_t over = 0;
                uint32_t small = 0xffffffffu, large = 0, many = 0;
                for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                    const float l = logits[i];
                    if (!(l >= least && l <= top)) continue;
                    const uint32_t b = bin(l);
                    if (b > b1) continue;
                    if (b < b0) over += w(l);
                    else {
                        const uint32_t k = key_of(l), at = atomicAdd(&s.listed, 1u);
                        small = min(small, k); large = max(large, k);
                        if (at < LIST) s.list[at] = k;
                    }
                }
                over = sum_cta(over);
                small = ~max_cta(~small); large = max_cta(large);
                tell(small, large, s.listed, over);
                for (uint32_t r = 0; r < split; r++) { many += (uint32_t)heard(r, 2); above += heard(r, 3); }
                search<MASS>(w, lo, hi, many, goal, above);
                sync();
            }
        }
        for (; lo < hi; first = false) {
            const float top = of_key(hi), bottom = of_key(lo), per = first ? (float)BINS / (top - bottom) : 0.0f;
            const bool even = per > 0.0f && per < INFINITY;                      // bins of equal width in the logits, else in the keys
            const uint64_t step = (((uint64_t)BINS << 32) - 1) / ((uint64_t)(hi - lo) + 1);
            const auto bin = [&](float l) -> uint32_t {
                if (even) return min(BINS - 1, (uint32_t)((top - l) * per));
                return (uint32_t)((hi - key_of(l)) * step >> 32);
            };
            s.count[threadIdx.x] = 0; s.mass[threadIdx.x] = 0;
            if (threadIdx.x == 0) s.listed = 0;
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const float l = logits[i];
                if (!(l >= bottom && l <= top)) continue;
                const uint32_t b = bin(l);
                atomicAdd(&s.count[b], 1u);
                if (MASS) atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)w(l));
            }
            sync();
            // the bin in which the goal is reached: a thread a bin
            uint64_t amount = 0; uint32_t count = 0;
            for (uint32_t r = 0; r < split; r++) {
                const uint32_t c = ld_cluster_u32(mapa(smem_u32(&s.count[threadIdx.x]), r));
                count += c;
                amount += MASS ? ld_cluster_u64(mapa(smem_u32(&s.mass[threadIdx.x]), r)) : c;
            }
            const uint64_t upto = scan_cta(amount);
            if (above + upto - amount < goal && above + upto >= goal && amount) { s.found_bin = threadIdx.x; s.found_above = above + upto - amount; s.found_count = count; }
            sync();                                                              // (the others have read this CTA's bins)
            const uint32_t b = s.found_bin, many = s.found_count;
            above = s.found_above;
            uint32_t small = 0xffffffffu, large = 0;
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const float l = logits[i];
                if (!(l >= bottom && l <= top) || bin(l) != b) continue;
                const uint32_t k = key_of(l);
                small = min(small, k); large = max(large, k);
                if (many <= LIST) s.list[atomicAdd(&s.listed, 1u)] = k;
            }
            small = ~max_cta(~small); large = max_cta(large);
            tell(small, large, s.listed);
            search<MASS>(w, lo, hi, many, goal, above);
            sync();                                                              // (lists and bins are free again)
        }
        return lo;
    }
};

// whether l weighs min_p of the largest
__device__ __forceinline__ bool heavy(const Weights &w, float l, double log_min_p) { return l == w.top || (!isinf(w.top) && ((double)l - w.m) * w.inv_t >= log_min_p); }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__global__ void __launch_bounds__(THREADS) spg_sample_kernel(const SampleParams p)
{
    extern __shared__ __align__(16) uint8_t raw[];
    Shared &s = *reinterpret_cast<Shared *>(raw);
    float *logits = reinterpret_cast<float *>(raw + sizeof(Shared));
    const uint32_t row = blockIdx.x / p.split, rank = blockIdx.x % p.split, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t from = min(p.width, rank * p.slice), n = min(p.width - from, p.slice);
    for (uint32_t i = threadIdx.x; i < STEPS; i += THREADS) s.table[i] = __double2uint_rn(exp2((double)i / STEPS) * (double)(1u << 30));
    spg_grid_wait();

    // The row, its largest and smallest logits and how many there are: 16 bytes a load between the ends that do not lie on 16 bytes
    const T *x = reinterpret_cast<const T *>(p.logits) + (uint64_t)row * p.ld + from;
    constexpr uint32_t PER = 16 / sizeof(T);
    const uint32_t off = (uint32_t)((uintptr_t)x % 16u / sizeof(T)), first = min(n, (PER - off) % PER), packs = (n - first) / PER;
    logits += (4u - first % 4u) % 4u;                                            // packs lie on 16 bytes here too
    float mine = -INFINITY, least = INFINITY;
    uint32_t have = 0;
    const auto take = [&](float l) -> float {
        l = logit_of(l);
        if (l > -INFINITY) { mine = fmaxf(mine, l); least = fminf(least, l); have++; }
        return l;
    };
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < packs; i += THREADS) {
        alignas(16) T v[PER];
        *reinterpret_cast<uint4 *>(v) = __ldg(reinterpret_cast<const uint4 *>(x + first) + i);
#pragma unroll
        for (uint32_t j = 0; j < PER; j += 4)
            *reinterpret_cast<float4 *>(logits + first + i * PER + j) = make_float4(take(to_f32(v[j])), take(to_f32(v[j + 1])), take(to_f32(v[j + 2])), take(to_f32(v[j + 3])));
    }
    if (threadIdx.x < 2 * PER) {                                                 // the ends
        const uint32_t i = threadIdx.x < PER ? threadIdx.x : first + packs * PER + threadIdx.x - PER;
        if (i < (threadIdx.x < PER ? first : n)) logits[i] = take(to_f32(x[i]));
    }
    Row R{ s, logits, n, p.split, rank, 0 };
    uint32_t top = R.max_cta(key_of(mine)), low = ~R.max_cta(~key_of(least));
    have = (uint32_t)R.sum_cta(have);
    R.tell(top, low, have);
    uint32_t all = 0;
    for (uint32_t r = 0; r < p.split; r++) { top = max(top, (uint32_t)R.heard(r, 0)); low = min(low, (uint32_t)R.heard(r, 1)); all += (uint32_t)R.heard(r, 2); }
    const float largest = of_key(top);

    const float t = p.temperature ? p.temperature[row] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const int32_t k = p.top_k ? p.top_k[row] : 0;
    const float pp = p.top_p ? p.top_p[row] : 1.0f, mp = p.min_p ? p.min_p[row] : 0.0f;
    const double log_min_p = mp > 0.0f ? log((double)mp) : -INFINITY;
    const double u = p.u[row] > 0.0f ? (double)p.u[row] : 0.0;
    Weights w;
    w.set(largest, greedy ? 1.0f : t, s.table);

    if (all && !greedy && k >= 1 && (uint32_t)k < all && (uint32_t)k <= FEW / 2) {
        // the k / split largest threads' largest of every CTA: at least k logits of the row are no smaller than the least of them
        const uint32_t want = ((uint32_t)k + p.split - 1) / p.split, key = key_of(mine);
        uint32_t bound = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
            const uint32_t c = (uint32_t)__syncthreads_count(key >= (bound | bit));
            if (c >= want) bound |= bit;
            if (c == want) break;
        }
        if (threadIdx.x == 0) s.listed = 0;
        R.tell(bound);
        for (uint32_t r = 0; r < p.split; r++) bound = min(bound, (uint32_t)R.heard(r, 0));
        const float at_least = bound > key_of(-INFINITY) ? of_key(bound) : -FLT_MAX;
        for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
            const float l = logits[i];
            if (l >= at_least) {
                const uint32_t at = atomicAdd(&s.listed, 1u);
                if (at < FEW) { s.few[at].l = l; s.few[at].index = from + i; }
            }
        }
        __syncthreads();
        R.tell(s.listed);
        uint32_t many = 0;
        for (uint32_t r = 0; r < p.split; r++) many += (uint32_t)R.heard(r, 0);
        if (many <= FEW) {
            if (rank == 0) {
                Item me{ -INFINITY, 0xffffffffu, 0 };
                uint32_t at = 0;
                for (uint32_t r = 0; r < p.split; r++) {
                    const uint32_t c = (uint32_t)R.heard(r, 0);
                    if (threadIdx.x >= at && threadIdx.x < at + c) {
                        me.l = __uint_as_float(ld_cluster_u32(mapa(smem_u32(&s.few[threadIdx.x - at].l), r)));
                        me.index = ld_cluster_u32(mapa(smem_u32(&s.few[threadIdx.x - at].index), r));
                        me.w = w.exact(me.l);
                    }
                    at += c;
                }
                __syncthreads();
                if (threadIdx.x < many) s.few[threadIdx.x] = me;
                __syncthreads();
                uint32_t place = 0;
                uint64_t before = 0;
                if (warp * 32 < many)
                    for (uint32_t i = 0; i < many; i++) {
                        const Item o = s.few[i];
                        if (o.l > me.l || (o.l == me.l && o.index < me.index)) { place++; before += o.w; }
                    }
                bool keep = threadIdx.x < many && place < (uint32_t)k;
                if (pp < 1.0f) {
                    const double reach = ceil((double)pp * (double)R.sum_cta(keep ? me.w : 0));
                    keep = keep && before < (reach >= 1.0 ? (uint64_t)reach : 1);
                }
                if (mp > 0.0f) keep = keep && (place == 0 || (mp <= 1.0f && heavy(w, me.l, log_min_p)));
                if (!keep) me.w = 0;
                const uint64_t total = R.sum_cta(me.w);                          // (everybody has read the items)
                if (threadIdx.x < many) s.few[threadIdx.x].w = me.w;
                const int left = __syncthreads_count(keep);
                const double goal_d = u * (double)total;
                const uint64_t goal = goal_d >= (double)(total - 1) ? total - 1 : (uint64_t)goal_d;
                uint64_t upto = 0;
                if (warp * 32 < many)
                    for (uint32_t i = 0; i < many; i++) {
                        const Item o = s.few[i];
                        if (o.index <= me.index) upto += o.w;
                    }
                if (me.w && upto > goal && upto - me.w <= goal) {
                    p.tokens[row] = (int32_t)me.index;
                    if (p.probs) p.probs[row] = (float)((double)me.w / (double)total);
                    if (p.kept) p.kept[row] = left;
                }
            }
            R.sync();
            return;
        }
    }

    // what is left: logits above `cut`, and the first `ties` equal to it
    uint32_t cut = key_of(-INFINITY), ties = 0;
    if (all && greedy) { cut = top; ties = 1; }
    if (all && !greedy) {
        if (k >= 1 && (uint32_t)k < all) {
            uint64_t above;
            cut = R.select<false>(w, low, top, (uint64_t)k, 0, 0, 0.0, above);
            ties = (uint32_t)(k - above);
        }
        if (pp < 1.0f) {
            uint64_t sum = 0;
            uint32_t nearest = 0xffffffffu;
            const float over = of_key(cut);
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const float l = logits[i];
                if (l > over) { sum += w(l); nearest = min(nearest, key_of(l)); }
            }
            sum = R.sum_cta(sum); nearest = ~R.max_cta(~nearest);
            R.tell(sum, nearest);
            sum = 0; nearest = 0xffffffffu;
            for (uint32_t r = 0; r < p.split; r++) { sum += R.heard(r, 0); nearest = min(nearest, (uint32_t)R.heard(r, 1)); }
            const uint64_t each = ties ? w(over) : 0;
            const double want = ceil((double)pp * (double)(sum + ties * each));
            const uint64_t goal = want >= 1.0 ? (uint64_t)want : 1;
            if (sum < goal) ties = (uint32_t)min((uint64_t)ties, (goal - sum + each - 1) / max(each, (uint64_t)1));
            else {
                uint64_t above;
                cut = R.select<true>(w, nearest, top, goal, sum, all, (double)goal / (double)sum, above);
                const uint64_t one = w(of_key(cut));
                ties = (uint32_t)((goal - above + one - 1) / one);
            }
        }
        if (mp > 0.0f) {
            if (mp > 1.0f) { cut = top; ties = 1; }
            else {
                // the smallest key whose weight is at least mp, by halving: from a guess on both sides where that brackets it
                uint32_t a = key_of(-INFINITY), b = top;                         // a: too light, b: heavy enough
                const float guess = (float)(w.m + log_min_p / w.inv_t), wide = fabsf(guess) * 0x1p-20f + 1e-30f;
                if (guess > -FLT_MAX && guess < largest) {
                    if (!heavy(w, guess - wide, log_min_p)) a = max(a, key_of(guess - wide));
                    if (guess + wide < largest && heavy(w, guess + wide, log_min_p)) b = key_of(guess + wide);
                }
                while (b - a > 1) {
                    const uint32_t mid = a + (b - a) / 2;
                    if (heavy(w, of_key(mid), log_min_p)) b = mid; else a = mid;
                }
                if (b - 1 >= cut) { cut = b - 1; ties = 0; }
            }
        }
    }

    // Sums of what is left, for every warp's part of the slice (parts lie in the order of the vocabulary) and its quarters
    constexpr uint32_t PIECES = 4;
    const float over = of_key(cut);
    const uint32_t piece = ((n + WARPS - 1) / WARPS + PIECES * 32 - 1) / (PIECES * 32) * 32, begin = min(n, warp * piece * PIECES), end = min(n, begin + piece * PIECES);
    uint32_t equal = 0, left = 0;
    uint64_t sums[PIECES];
    uint32_t equals[PIECES];
#pragma unroll
    for (uint32_t q = 0; q < PIECES; q++) {
        const uint32_t a = min(end, begin + q * piece), b = min(end, a + piece);
        uint64_t sum = 0;
        uint32_t same = 0;
        for (uint32_t i = a + lane; i < b; i += 32) {
            const float l = logits[i];
            if (l > over) { sum += w(l); left++; }
            same += ties && l == over;
        }
        sums[q] = R.sum_warp(sum);
        equals[q] = __reduce_add_sync(0xffffffffu, same);
        equal += equals[q];
    }
    left = __reduce_add_sync(0xffffffffu, left);
    uint32_t equal_before = 0;
    if (ties) {                                                                  // (the same in all threads of the cluster)
        __syncthreads();
        if (lane == 0) s.warp_b[warp] = equal;
        __syncthreads();
        uint32_t equal_cta = 0;
        for (uint32_t i = 0; i < WARPS; i++) { if (i < warp) equal_before += (uint32_t)s.warp_b[i]; equal_cta += (uint32_t)s.warp_b[i]; }
        R.tell(equal_cta);
        for (uint32_t r = 0; r < rank; r++) equal_before += (uint32_t)R.heard(r, 0);
    }
    const uint64_t each = ties ? w(over) : 0;
    uint64_t sum = 0;
    uint32_t seen = equal_before;
#pragma unroll
    for (uint32_t q = 0; q < PIECES; q++) {
        const uint32_t here = ties > seen ? min(equals[q], ties - seen) : 0;
        seen += equals[q];
        left += here;
        sums[q] += here * each;
        sum += sums[q];
    }
    __syncthreads();
    if (lane == 0) { s.warp_a[warp] = sum; s.warp_b[warp] = left; }
    __syncthreads();
    uint64_t before = 0, cta = 0, left_cta = 0;
    for (uint32_t i = 0; i < WARPS; i++) { if (i < warp) before += s.warp_a[i]; cta += s.warp_a[i]; left_cta += s.warp_b[i]; }
    R.tell(cta, left_cta);
    uint64_t total = 0, left_all = 0;
    for (uint32_t r = 0; r < p.split; r++) { if (r < rank) before += R.heard(r, 0); total += R.heard(r, 0); left_all += R.heard(r, 1); }

    if (total == 0) {
        if (rank == 0 && threadIdx.x == 0) { p.tokens[row] = -1; if (p.probs) p.probs[row] = 0.0f; if (p.kept) p.kept[row] = 0; }
    } else {
        const double goal_d = u * (double)total;
        const uint64_t goal = goal_d >= (double)(total - 1) ? total - 1 : (uint64_t)goal_d;
        if (before <= goal && goal < before + sum) {                             // in this warp's part: in which quarter, and where
            uint64_t run = before;
            uint32_t a = begin;
            seen = equal_before;
#pragma unroll
            for (uint32_t q = 0; q + 1 < PIECES; q++)
                if (a == min(end, begin + q * piece) && run + sums[q] <= goal) { run += sums[q]; seen += equals[q]; a = min(end, begin + (q + 1) * piece); }
            for (uint32_t i0 = a; i0 < end; i0 += 32) {
                const uint32_t i = i0 + lane;
                const float l = i < end ? logits[i] : -INFINITY;
                const uint32_t same = __ballot_sync(0xffffffffu, ties && l == over);
                const bool tie = ties && l == over && seen + __popc(same & ((1u << lane) - 1)) < ties;
                const uint64_t one = l > over ? w(l) : (tie ? each : 0);
                uint64_t upto = one;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint64_t v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= (uint32_t)o) upto += v;
                }
                const uint32_t past = __ballot_sync(0xffffffffu, run + upto > goal);
                if (past) {
                    if (lane == (uint32_t)__ffs((int)past) - 1) {
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
    p.slice = ((p.width + p.split - 1) / p.split + 7u) / 8u * 8u;
    if ((uint64_t)p.N * p.split > 0x7fffffffu) { spgk_set_error("spgk_sample_rows", "too many rows"); return SPGK_E_ARG; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.N * p.split); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = sizeof(Shared) + (size_t)p.slice * 4 + 16; cfg.stream = stream;
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
