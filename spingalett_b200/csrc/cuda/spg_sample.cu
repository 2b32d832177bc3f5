// spg_sample.cu -- a token drawn from every row of logits: temperature, top-k, top-p, min-p.
//
//   w_i = exp((l_i - m) / T), m the largest logit.  Ordered by (l falling, i rising) a row is cut after the first k logits, after the
//   shortest beginning with p of their weight, after the last w_i >= min_p; the token is the first index at which the running sum of the
//   weights that are left exceeds u times their total.
//
// All three cuts leave a beginning of the same order, so what is left is told by one logit and a number: the logits above it, and the first r of
// those equal to it.  Nothing is sorted.  A row belongs to a cluster of up to eight CTAs and is read once, into shared memory; many long rows have a CTA each, which
// reads its row anew for every pass, from L2 as far as that holds what all of them read.
//   - A small top_k: each thread has the largest of its logits, and the (k / CTAs)-th largest of those in a CTA bounds the k-th logit of the row from
//     below; the few logits above the least of these bounds meet in one CTA, where every thread counts what stands before its own.  So do the logits
//     of a short row, or of one with nearly all of them masked.
//   - Otherwise a cut is found by a histogram over the range in question (counts for top-k, weights for top-p), a list of the bin in which the border
//     falls (or, where that is too long, another histogram over it), and a search in the list digit by digit.
// Sums of 131072 weights in 32 bits would put a number drawn close to a border on its wrong side in some rows of a hundred.  Here a weight is good to 2^-30 of itself
// and a whole multiple of 2^-44 (the largest is 1; what is below is cut off where the weight comes from the table, and rounded where it comes from exp()), so sums in 64 bits
// do not hang on an order, and one of n weights is good to 2^-30 of itself and n * 2^-44.  A number closer than that to a border may still fall on its other side.
// What bounds it: 256 x 131072 of fp32 142 us with top_p, 84 without a cut, 80 at temperature 0, 64 with top_k 50 (HBM would take 21), 64 x 50001 of bf16 with all cuts 14,
// 1 x 1000 6.7; 512 x 131072 of bf16 with top_k 500 and top_p 430.
// With top_p 83 instructions a logit, issued at 58 % of the rate with 26 warps an SM, bound it; and the bytes: the rows of one launch are more than L2 holds, so that of the 403 MB of its
// three passes 330 come from HBM, which would take 50 us for them.  Kept in shared memory, such rows fill it, so that sixteen warps have an SM (228 us).  Slower there: two
// CTAs with half the logits each on an SM (the same rows at work), 1024 threads (what every warp does for itself), 64-bit atomics, additions to bins left out for light logits, rows
// fetched to L2 ahead.
// Where |largest| * log2(e) / temperature is beyond 4000 every weight is an exp() in 64 bits: 256 x 131072 with top_p 440 us, without a cut 152.
#include "spg_common.cuh"
#include "spg_tc.cuh"
#include <type_traits>

namespace {

using spgtc::smem_u32; using spgtc::mapa; using spgtc::cluster_rank;

constexpr uint32_t THREADS = 512, WARPS = THREADS / 32;
constexpr uint32_t BINS = 512;
constexpr uint32_t ONCE = 65536 / 4;          // fours whose mantissas' halves, all in one bin, come to less than 2^32
constexpr uint32_t DENSE = 512;               // places that a warp puts side by side
constexpr uint32_t LIST = 2048;               // logits of a range that are searched digit by digit
constexpr uint32_t FEW = 512;                 // logits among which every thread counts what stands before its own
constexpr uint32_t TINY = 128;                // rows with no more logits are all of them few (512 x 100 with top_p: 15.5 us, as long rows 25.0; without a cut 14.9 and 12.4)
constexpr uint32_t MAX_SPLIT = 8;
constexpr uint32_t SLICE = SPGK_SAMPLE_MAX_WIDTH / MAX_SPLIT;
constexpr int ONE_BITS = 44;
constexpr uint32_t STEPS = 1024;              // of the table of 2^(i / STEPS)
static_assert(BINS == THREADS && LIST % THREADS == 0 && FEW <= THREADS && STEPS % THREADS == 0, "a thread a bin, a logit, two steps");

// 2^(i / STEPS) in units of 2^-30 (repeated multiplication errs by less than 2^-42)
struct Steps {
    uint32_t v[STEPS];
    constexpr Steps() : v()
    {
        double x = 1.0;
        for (uint32_t i = 0; i < STEPS; i++, x *= 1.000677130693066356678727) v[i] = (uint32_t)(x * (double)(1u << 30) + 0.5);
    }
};
__device__ const Steps g_steps;

struct SampleParams {
    const void *logits; uint32_t ld, N, width, split, slice;
    const float *temperature; const int32_t *top_k; const float *top_p, *min_p, *u;
    int32_t *tokens; float *probs; int32_t *kept;
};

// Integers in the order of the logits, -0 like 0.  (A NaN has none: it is in none of the ranges that are asked for before a key is.)
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t b = __float_as_uint(l + 0.0f);
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
    __device__ __forceinline__ float rest(float l, float kf) const { return fmaf(l, c_lo, fmaf(l, c, fmaf(kf, -1.0f / STEPS, MAGIC / STEPS))); }      // (-K / 1024 is exact)
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
    // m * 2^((k >> 10) - 30), with m in [2^30, 2^31)
    __device__ __forceinline__ uint32_t mantissa(float l, int &k) const
    {
        l = fmaxf(l, floor);
        const float kf = fmaf(l, c_steps, MAGIC);
        const float y = rest(l, kf) - y_top;
        k = __float_as_int(kf) - k_top;                      // <= 0
        const uint32_t t = table[k & (int)(STEPS - 1)];
        const float p = y * fmaf(y, 0.24022650695910072f * (1 << 30), 0.69314718055994531f * (1 << 30));
        // t * p in whole numbers, without a conversion: t's upper bits are the fraction of a number from 1 to 2, and MAGIC rounds the product
        return t + (uint32_t)(__float_as_int(fmaf(__uint_as_float((t >> 7) + 0x3f000000u), p, MAGIC)) - 0x4b400000);
    }
    __device__ __forceinline__ uint64_t quick(float l) const
    {
        int k;
        const uint32_t w = mantissa(l, k);
        const int up = (k >> 10) + (ONE_BITS - 30);
        return (uint64_t)(w >> min(max(-up, 0), 31)) * (uint64_t)(1u << max(up, 0));
    }
    // Bins of a sixteenth of an octave (-k = 0, 1 .. 64, 65 .. 128 and so on: sixteen of them share k >> 10), the last for all that is lighter; in a bin all
    // weights are mantissas times the same power of two (in the last one they are counted as they are)
    __device__ __forceinline__ uint32_t bin(float l) const
    {
        const int k = __float_as_int(fmaf(fmaxf(l, floor), c_steps, MAGIC)) - k_top;
        return min(BINS - 1, (uint32_t)(63 - k) >> 6);
    }
    __device__ __forceinline__ uint64_t operator()(float l) const { return fast ? quick(l) : exact(l); }
    // body(weight) with the one or the other: loops over many logits have no choice inside
    template <typename F> __device__ __forceinline__ void with(F body) const
    {
        if (fast) body([this](float l) { return quick(l); });
        else body([this](float l) { return exact(l); });
    }
};

struct Item { float l; uint32_t index; uint64_t w; };
constexpr uint32_t PIECES = 64;               // of a CTA's slice, in the order of the vocabulary: four a warp, two a lane
static_assert(PIECES == 64 && PIECES % WARPS == 0 && SLICE + 8 <= 65536, "two a lane; places in 16 bits");

// Place: what a warp puts side by side of a logit -- where it lies in shared memory, or itself
template <typename Place> struct alignas(16) Shared {
    uint64_t mass[BINS];
    uint32_t count[BINS + 32], count_low[BINS + 32];
    union { struct { uint32_t list[LIST]; uint16_t piece[LIST]; }; Item few[FEW]; };
    uint32_t table[STEPS];
    uint64_t piece_sum[PIECES]; uint32_t piece_equal[PIECES];
    Place dense[WARPS][DENSE];
    uint32_t left;
    uint64_t out[2][4];                        // what this CTA tells the others, by turns
    uint64_t warp[2][WARPS];
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

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// This CTA's logits by fours, -infinity in front of the first and behind the last: from its shared memory, or as they lie in the row
struct Kept {
    using Place = uint16_t;
    static constexpr uint32_t AT_ONCE = 1;     // fours of a thread on their way at a time
    const float4 *fours;
    __device__ __forceinline__ float4 operator()(uint32_t i) const { return fours[i]; }
    __device__ __forceinline__ float at(Place place) const { return reinterpret_cast<const float *>(fours)[place]; }
    __device__ __forceinline__ static Place place(uint32_t i, float) { return (Place)i; }
};
// (plain loads: one through the read-only path may be moved in front of the wait for the launch that writes the logits)
__device__ __forceinline__ float4 load4(const float *x) { return *reinterpret_cast<const float4 *>(x); }
template <typename T> __device__ __forceinline__ float4 load4(const T *x)
{
    const uint2 v = *reinterpret_cast<const uint2 *>(x);
    const T *t = reinterpret_cast<const T *>(&v);
    return make_float4(to_f32(t[0]), to_f32(t[1]), to_f32(t[2]), to_f32(t[3]));
}
template <typename T> struct Streamed {
    using Place = float;
    static constexpr uint32_t AT_ONCE = 4;
    const T *x;                                // four elements' alignment, `lead` of them in front of the row
    uint32_t lead, end;
    __device__ __forceinline__ float4 operator()(uint32_t i) const
    {
        const uint32_t e = 4 * i;
        if (e >= lead && e + 4 <= end) return load4(x + e);
        float v[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) v[j] = e + j >= lead && e + j < end ? to_f32(x[e + j]) : -INFINITY;
        return make_float4(v[0], v[1], v[2], v[3]);
    }
    __device__ __forceinline__ float at(Place place) const { return place; }
    __device__ __forceinline__ static Place place(uint32_t, float l) { return l; }
};

template <typename Source> struct Row {
    Shared<typename Source::Place> &s;
    Source fours;
    uint32_t count, per_piece;                 // fours, and fours of a piece (a multiple of 32)
    uint32_t split, rank, turn, place;         // CTAs of the row
    uint64_t told;

    static constexpr uint32_t AT_ONCE = Source::AT_ONCE;

    __device__ __forceinline__ static float4 nothing() { return make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }
    // fours a, a + step, ... below b
    template <typename F> __device__ __forceinline__ void each_four(uint32_t a, uint32_t b, uint32_t step, F f) const
    {
        for (uint32_t i = a; i < b; i += AT_ONCE * step) {
            float4 v[AT_ONCE];
#pragma unroll
            for (uint32_t u = 0; u < AT_ONCE; u++) v[u] = u == 0 || i + u * step < b ? fours(i + u * step) : nothing();
#pragma unroll
            for (uint32_t u = 0; u < AT_ONCE; u++) f(v[u]);
        }
    }
    // (four logits at a time, so that their chains of instructions overlap)
    template <typename F> __device__ __forceinline__ void each(F f) const
    {
        each_four(threadIdx.x, count, THREADS, [&](const float4 &v) { f(v.x); f(v.y); f(v.z); f(v.w); });
    }
    // the logits of piece q of this warp
    template <typename F> __device__ __forceinline__ void each_of_piece(uint32_t q, F f) const
    {
        const uint32_t a = (threadIdx.x / 32 * (PIECES / WARPS) + q) * per_piece, b = min(count, a + per_piece);
        each_four(a + threadIdx.x % 32, b, 32, [&](const float4 &v) { f(v.x); f(v.y); f(v.z); f(v.w); });
    }
    __device__ __forceinline__ void sync() { if (split > 1) spgtc::cluster_sync(); else __syncthreads(); }
    __device__ __forceinline__ uint64_t sum_warp(uint64_t v)
    {
        const uint32_t mask = (1u << 26) - 1;                                    // (three parts whose sums fit 32 bits)
        const uint64_t a = __reduce_add_sync(0xffffffffu, (uint32_t)v & mask), b = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 26) & mask);
        return a + (b << 26) + ((uint64_t)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> 52)) << 52);
    }
    // Over the CTA, to all threads.  The warps' results lie in one of two places by turns: who writes to one again has passed the barrier behind the other.
    __device__ __forceinline__ uint64_t *warps(uint64_t v, bool mine)
    {
        place ^= 1;
        if (mine) s.warp[place][threadIdx.x / 32] = v;
        __syncthreads();
        return s.warp[place];
    }
    __device__ __forceinline__ uint64_t sum_cta(uint64_t v)
    {
        const uint64_t *w = warps(sum_warp(v), threadIdx.x % 32 == 0);
        uint64_t r = 0;
#pragma unroll
        for (uint32_t i = 0; i < WARPS; i++) r += w[i];
        return r;
    }
    __device__ __forceinline__ uint32_t max_cta(uint32_t v)
    {
        const uint64_t *w = warps(__reduce_max_sync(0xffffffffu, v), threadIdx.x % 32 == 0);
        return __reduce_max_sync(0xffffffffu, (uint32_t)w[threadIdx.x % WARPS]);
    }
    // sum over the threads up to this one, and over all
    __device__ __forceinline__ uint64_t scan_cta(uint64_t v, uint64_t &total)
    {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
            if (threadIdx.x % 32 >= (uint32_t)o) v += u;
        }
        const uint64_t *w = warps(v, threadIdx.x % 32 == 31);
        total = 0;
#pragma unroll
        for (uint32_t i = 0; i < WARPS; i++) { const uint64_t x = w[i]; if (i < threadIdx.x / 32) v += x; total += x; }
        return v;
    }
    // Up to four values of every CTA (the same in all its threads) to every CTA: a lane fetches one of them, heard() asks it (whole warps)
    __device__ __forceinline__ void tell(uint64_t a, uint64_t b = 0, uint64_t c = 0, uint64_t d = 0)
    {
        turn ^= 1;
        if (threadIdx.x == 0) { s.out[turn][0] = a; s.out[turn][1] = b; s.out[turn][2] = c; s.out[turn][3] = d; }
        sync();
        const uint32_t from = threadIdx.x % 32 / 4;
        told = from < split ? ld_cluster_u64(mapa(smem_u32(&s.out[turn][threadIdx.x % 4]), from)) : 0;
    }
    __device__ __forceinline__ uint64_t heard(uint32_t from, int which) { return __shfl_sync(0xffffffffu, told, from * 4 + which); }

    // [lo, hi] to the smallest and largest key in question, of which every CTA has told its own beside how many it has listed; where all are listed,
    // the border is found digit by digit: every thread takes its part of all CTAs' lists
    template <typename F> __device__ void search(F weight, uint32_t &lo, uint32_t &hi, uint32_t many, uint64_t goal, uint64_t &above)
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
        for (uint32_t i = 0; i < LIST / THREADS; i++) if (i * THREADS + threadIdx.x < at) weigh[i] = weight(of_key(mine[i]));
        // digit by digit: a bin is 2^shift keys, counted from hi down
        uint32_t shift = 32 - __clz((int)(hi - lo));
        shift = shift > 9 ? shift - 9 : 0;
        for (;;) {
            __syncthreads();
            s.mass[threadIdx.x] = 0;
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < LIST / THREADS; i++)
                if (weigh[i] && mine[i] <= hi && mine[i] >= lo) atomicAdd((unsigned long long *)&s.mass[(hi - mine[i]) >> shift], (unsigned long long)weigh[i]);
            __syncthreads();
            uint64_t sum;
            const uint64_t amount = s.mass[threadIdx.x], upto = scan_cta(amount, sum);
            const uint64_t reach = min(goal, above + sum);
            if (above + upto - amount < reach && above + upto >= reach && amount) { s.found_bin = threadIdx.x; s.found_above = above + upto - amount; }
            __syncthreads();
            above = s.found_above;
            hi -= s.found_bin << shift;
            if (shift == 0) break;
            lo = max(lo, hi - ((1u << shift) - 1));
            shift = shift > 9 ? shift - 9 : 0;
        }
        lo = hi;
    }

    // The largest key v above `cut` with (amount of keys above v) < goal <= (amount of keys from v on), amounts being counts or weights;
    // goal >= 1 and no more than the amount of all keys above cut.  [lo, hi]: the smallest and the largest key in question.  above: the amount above v.
    template <bool MASS> __device__ uint32_t select(const Weights &w, uint32_t lo, uint32_t hi, uint64_t goal, uint64_t &above, bool first = true)
    {
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
            each([&](float l) {
                if (!(l >= bottom && l <= top)) return;
                const uint32_t b = bin(l);
                atomicAdd(&s.count[b], 1u);
                if (MASS) atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)w(l));
            });
            sync();
            // the bin in which the goal is reached: a thread a bin
            uint64_t amount = 0; uint32_t count = 0;
#pragma unroll
            for (uint32_t r = 0; r < MAX_SPLIT; r++) {
                if (r >= split) continue;
                const uint32_t c = ld_cluster_u32(mapa(smem_u32(&s.count[threadIdx.x]), r));
                count += c;
                amount += MASS ? ld_cluster_u64(mapa(smem_u32(&s.mass[threadIdx.x]), r)) : c;
            }
            uint64_t sum;
            const uint64_t upto = scan_cta(amount, sum);
            const uint64_t reach = min(goal, above + sum);
            if (above + upto - amount < reach && above + upto >= reach && amount) { s.found_bin = threadIdx.x; s.found_above = above + upto - amount; s.found_count = count; }
            sync();                                                              // (the others have read this CTA's bins)
            const uint32_t b = s.found_bin, many = s.found_count;
            above = s.found_above;
            uint32_t small = 0xffffffffu, large = 0;
            each([&](float l) {
                if (!(l >= bottom && l <= top) || bin(l) != b) return;
                const uint32_t k = key_of(l);
                small = min(small, k); large = max(large, k);
                if (many <= LIST) s.list[atomicAdd(&s.listed, 1u)] = k;
            });
            small = ~max_cta(~small); large = max_cta(large);
            tell(small, large, s.listed);
            search([&](float l) -> uint64_t { return MASS ? w(l) : 1; }, lo, hi, many, goal, above);
            sync();                                                              // (lists and bins are free again)
        }
        return lo;
    }

    // Cuts what is left -- the logits above `cut` and `ties` equal to it -- after the shortest beginning with `share` of its weight.  Two passes: the bins' weights
    // (sums of mantissas in two halves of 32 bits), then a list of the border's bin and, a piece at a time, the sums of what is above it.
    // Returns whether the pieces have the sums of what is above the new cut and the numbers of logits equal to it.
    __device__ bool mass_cut(const Weights &w, float share, uint32_t &cut, uint32_t &ties)
    {
        const float over = of_key(cut);
        const auto up_of = [](uint32_t bin) -> int { return bin == BINS - 1 ? 0 : ONE_BITS - 30 - (int)((bin + 15) >> 4); };
        s.count[threadIdx.x] = 0; s.count_low[threadIdx.x] = 0;
        if (threadIdx.x == 0) s.listed = 0;
        __syncthreads();
        uint64_t low = 0, high = 0;
        for (uint32_t from = 0; from < this->count; from += ONCE) {
            each_four(from + threadIdx.x, min(this->count, from + ONCE), THREADS, [&](const float4 &v) {
                const float l[4] = { v.x, v.y, v.z, v.w };
                uint32_t m[4], at[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    int k;
                    m[j] = w.mantissa(l[j], k);
                    const uint32_t bin = min(BINS - 1, (uint32_t)(63 - k) >> 6);
                    if (bin == BINS - 1) m[j] >>= min(-(k >> 10) - (ONE_BITS - 30), 31);
                    at[j] = l[j] > over ? bin : BINS + threadIdx.x % 32;             // (what is not left goes to a place of its lane: no branches)
                }
#pragma unroll
                for (int j = 0; j < 4; j++) { atomicAdd(&s.count_low[at[j]], m[j] & 0xffffu); atomicAdd(&s.count[at[j]], m[j] >> 16); }
            });
            if (from + ONCE < this->count) {                                     // (a whole long row: what is there is taken out of the 32 bits)
                __syncthreads();
                low += s.count_low[threadIdx.x]; high += s.count[threadIdx.x];
                s.count_low[threadIdx.x] = 0; s.count[threadIdx.x] = 0;
                __syncthreads();
            }
        }
        sync();
#pragma unroll
        for (uint32_t r = 0; r < MAX_SPLIT; r++) {
            if (r >= split) continue;
            low += ld_cluster_u32(mapa(smem_u32(&s.count_low[threadIdx.x]), r));
            high += ld_cluster_u32(mapa(smem_u32(&s.count[threadIdx.x]), r));
        }
        const int up = up_of(threadIdx.x);
        uint64_t amount = (high << 16) + low, total;
        amount = up >= 0 ? amount << up : amount >> -up;
        const uint64_t upto = scan_cta(amount, total), one_tie = ties ? w.quick(over) : 0;
        const double want = ceil((double)share * (double)(total + ties * one_tie));
        const uint64_t goal = want >= 1.0 ? (uint64_t)want : 1;
        if (upto - amount < goal && upto >= goal) { s.found_bin = threadIdx.x; s.found_above = upto - amount; }
        sync();                                                                  // (the others have read this CTA's bins)
        if (total < goal) {
            ties = (uint32_t)min((uint64_t)ties, (goal - total + one_tie - 1) / max(one_tie, (uint64_t)1));
            return false;
        }
        const uint32_t border = s.found_bin;
        const int border_up = up_of(border);
        // the goal in the units of the border's bin
        uint64_t rest = goal - s.found_above;
        rest = border_up >= 0 ? (rest + ((1ull << border_up) - 1)) >> border_up : rest << -border_up;
        // Few of a piece's logits are so large.  A warp first puts the places of those of all its pieces side by side, then weighs them, a lane each: the
        // way from a logit to its weight is long, and so it is gone a few times a warp.
        const float bottom = border == BINS - 1 ? -INFINITY : w.top - (float)(border * 64 + 2) / (w.c * (float)STEPS) - 1e-6f * fabsf(w.top);
        constexpr uint32_t MINE = PIECES / WARPS;
        typename Source::Place *const dense = s.dense[threadIdx.x / 32];
        const uint32_t lane = threadIdx.x % 32, first_piece = threadIdx.x / 32 * MINE;
        uint32_t small = 0xffffffffu, large = 0, many = 0, sure = 0, held = 0, ends[MINE];              // ends: of the pieces among the places
        uint64_t sums[MINE];
#pragma unroll
        for (uint32_t q = 0; q < MINE; q++) { sums[q] = 0; ends[q] = 0xffffffffu; }
        const auto weigh = [&]() {
            __syncwarp();
            for (uint32_t i = lane; i < held; i += 32) {
                const float x = fours.at(dense[i]);
                const uint32_t at_bin = w.bin(x);
                const uint64_t one = w.quick(x);
                uint32_t piece = 0;
#pragma unroll
                for (uint32_t q = 0; q + 1 < MINE; q++) piece += i >= ends[q];
                if (at_bin < border) {
                    sure++;
#pragma unroll
                    for (uint32_t q = 0; q < MINE; q++) sums[q] += piece == q ? one : 0;
                } else if (at_bin == border) {
                    const uint32_t k = key_of(x), at = atomicAdd(&s.listed, 1u);
                    small = min(small, k); large = max(large, k);
                    if (at < LIST) { s.list[at] = k; s.piece[at] = (uint16_t)(first_piece + piece); }
                }
            }
            __syncwarp();
            held = 0;
        };
#pragma unroll
        for (uint32_t q = 0; q < MINE; q++) {
            const uint32_t a = (first_piece + q) * per_piece, b = min(this->count, a + per_piece);
            for (uint32_t i0 = a; i0 < b; i0 += 64) {
                if (held > DENSE - 256) {
                    weigh();
#pragma unroll
                    for (uint32_t r = 0; r < q; r++) ends[r] = 0;
                }
                const float4 v = i0 + lane < b ? fours(i0 + lane) : nothing(), v2 = i0 + 32 + lane < b ? fours(i0 + 32 + lane) : nothing();
                const float l[8] = { v.x, v.y, v.z, v.w, v2.x, v2.y, v2.z, v2.w };
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) {
                    const bool in = l[j] > over && l[j] >= bottom;
                    const uint32_t set = __ballot_sync(0xffffffffu, in);
                    if (in) dense[held + __popc(set & ((1u << lane) - 1))] = Source::place(4 * (i0 + j / 4 * 32 + lane) + j % 4, l[j]);
                    held += __popc(set);
                }
            }
            ends[q] = held;
        }
        weigh();
#pragma unroll
        for (uint32_t q = 0; q < MINE; q++) {
            const uint64_t sum = sum_warp(sums[q]);
            if (lane == 0) { s.piece_sum[first_piece + q] = sum; s.piece_equal[first_piece + q] = 0; }
        }
        if (threadIdx.x == 0) s.left = 0;
        small = ~max_cta(~small); large = max_cta(large);
        sure = __reduce_add_sync(0xffffffffu, sure);
        if (lane == 0) atomicAdd(&s.left, sure);
        tell(small, large, s.listed);
        for (uint32_t r = 0; r < split; r++) many += (uint32_t)heard(r, 2);
        uint64_t above = 0;
        const auto weight = [&](float l) -> uint64_t { int k; return border == BINS - 1 ? w.quick(l) : w.mantissa(l, k); };
        uint32_t lo, hi;
        search(weight, lo, hi, many, rest, above);
        const bool listed = many <= LIST;
        if (lo < hi) {                                                           // too many for the list
            above = s.found_above;
            sync();
            lo = select<true>(w, lo, hi, goal, above, false);
            const uint64_t one = w(of_key(lo));
            cut = lo; ties = (uint32_t)((goal > above ? goal - above + one - 1 : one) / one);
            return false;
        }
        const uint64_t one = weight(of_key(lo));
        cut = lo; ties = (uint32_t)((rest - above + one - 1) / one);
        if (listed)
            for (uint32_t i = threadIdx.x; i < s.listed; i += THREADS) {
                const uint32_t k = s.list[i], piece = s.piece[i];
                if (k > lo) { atomicAdd((unsigned long long *)&s.piece_sum[piece], (unsigned long long)w.quick(of_key(k))); atomicAdd(&s.left, 1u); }
                else if (k == lo) atomicAdd(&s.piece_equal[piece], 1u);
            }
        sync();
        return listed;
    }
};

// whether l weighs min_p of the largest
__device__ __forceinline__ bool heavy(const Weights &w, float l, double log_min_p) { return l == w.top || (!isinf(w.top) && ((double)l - w.m) * w.inv_t >= log_min_p); }

template <typename T, bool STREAM>
__global__ void __launch_bounds__(THREADS, 2) spg_sample_kernel(const SampleParams p)
{
    extern __shared__ __align__(16) uint8_t raw[];
    using Source = std::conditional_t<STREAM, Streamed<T>, Kept>;
    Shared<typename Source::Place> &s = *reinterpret_cast<Shared<typename Source::Place> *>(raw);
    float *logits = reinterpret_cast<float *>(raw + sizeof(s));
    const uint32_t row = blockIdx.x / p.split, rank = blockIdx.x % p.split, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t from = min(p.width, rank * p.slice), n = min(p.width - from, p.slice);
    for (uint32_t i = threadIdx.x; i < STEPS; i += THREADS) s.table[i] = __ldg(&g_steps.v[i]);
    spg_grid_trigger();
    spg_grid_wait();

    const float t = p.temperature ? p.temperature[row] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const int32_t k = p.top_k ? p.top_k[row] : 0;
    const float pp = p.top_p ? p.top_p[row] : 1.0f, mp = p.min_p ? p.min_p[row] : 0.0f, number = p.u[row];

    // The row, its largest and smallest logits and how many there are: 16 bytes a load between the ends that do not lie on 16 bytes
    const T *x = reinterpret_cast<const T *>(p.logits) + (uint64_t)row * p.ld + from;
    float mine = -INFINITY, least = INFINITY;
    uint32_t have = 0;
    const auto take = [&](float l) -> float {
        const bool some = l > -INFINITY;
        mine = fmaxf(mine, l); least = fminf(least, some ? l : INFINITY); have += some;             // (of a NaN and a number both give the number)
        return l;
    };
    constexpr uint32_t PER = 16 / sizeof(T);
    const uint32_t off = (uint32_t)((uintptr_t)x % 16u / sizeof(T)), first = min(n, (PER - off) % PER), packs = (n - first) / PER;
    const uint32_t lead = STREAM ? off % 4u : (4u - first % 4u) % 4u, fours = (lead + n + 3u) / 4u;           // packs lie on 16 bytes here too
    Source source;
    if constexpr (STREAM) { source.x = x - lead; source.lead = lead; source.end = lead + n; }
    else source.fours = reinterpret_cast<const float4 *>(logits);
    Row<Source> R{ s, source, fours, ((fours + PIECES - 1) / PIECES + 31u) / 32u * 32u, p.split, rank, 0, 0, 0 };
    if constexpr (STREAM) R.each([&](float l) { take(l); });
    else {
        if (threadIdx.x < 8) {                                                       // what makes the first and the last four whole
            if (threadIdx.x < lead) logits[threadIdx.x] = -INFINITY;
            else if (threadIdx.x >= 4 && threadIdx.x - 4 < (4u - (lead + n) % 4u) % 4u) logits[lead + n + threadIdx.x - 4] = -INFINITY;
        }
        float *const row_logits = logits + lead;
        if (sizeof(T) == 4) {
            // straight to shared memory, the whole slice on its way at once (through registers 132 SMs drew 4 TB/s); a thread looks at what it has asked for, by quarters
            const uint32_t quarter = (packs + 4 * THREADS - 1) / (4 * THREADS) * THREADS;
#pragma unroll
            for (uint32_t q = 0; q < 4; q++) {
                for (uint32_t i = q * quarter + threadIdx.x; i < min(packs, (q + 1) * quarter); i += THREADS)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(row_logits + first) + 16 * i), "l"(reinterpret_cast<const uint4 *>(x + first) + i) : "memory");
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
            const auto look = [&](uint32_t q) {
                for (uint32_t i = q * quarter + threadIdx.x; i < min(packs, (q + 1) * quarter); i += THREADS) {
                    const float4 v = *reinterpret_cast<const float4 *>(row_logits + first + 4 * i);
                    take(v.x); take(v.y); take(v.z); take(v.w);
                }
            };
            asm volatile("cp.async.wait_group 3;" ::: "memory"); look(0);
            asm volatile("cp.async.wait_group 2;" ::: "memory"); look(1);
            asm volatile("cp.async.wait_group 1;" ::: "memory"); look(2);
            asm volatile("cp.async.wait_group 0;" ::: "memory"); look(3);
        } else {
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < packs; i += THREADS) {
                alignas(16) T v[PER];
                *reinterpret_cast<uint4 *>(v) = reinterpret_cast<const uint4 *>(x + first)[i];
#pragma unroll
                for (uint32_t j = 0; j < PER; j += 4)
                    *reinterpret_cast<float4 *>(row_logits + first + i * PER + j) = make_float4(take(to_f32(v[j])), take(to_f32(v[j + 1])), take(to_f32(v[j + 2])), take(to_f32(v[j + 3])));
            }
        }
        if (threadIdx.x < 2 * PER) {                                                 // the ends
            const uint32_t i = threadIdx.x < PER ? threadIdx.x : first + packs * PER + threadIdx.x - PER;
            if (i < (threadIdx.x < PER ? first : n)) row_logits[i] = take(to_f32(x[i]));
        }
    }
    uint32_t top = R.max_cta(key_of(mine)), low = ~R.max_cta(~key_of(least));
    have = (uint32_t)R.sum_cta(have);
    R.tell(top, low, have);
    uint32_t all = 0, rich = 0;                                                  // (rich: CTAs of whose logits no more than half are masked)
    for (uint32_t r = 0; r < p.split; r++) {
        const uint32_t c = (uint32_t)R.heard(r, 2);
        top = max(top, (uint32_t)R.heard(r, 0)); low = min(low, (uint32_t)R.heard(r, 1)); all += c; rich += c >= p.slice / 2;
    }
    const float largest = of_key(top);

    const double log_min_p = mp > 0.0f ? log((double)mp) : -INFINITY;
    const double u = number > 0.0f ? (double)number : 0.0;
    Weights w;
    w.set(largest, greedy ? 1.0f : t, s.table);

    const uint32_t first_k = k >= 1 && (uint32_t)k < all ? (uint32_t)k : all;    // logits that top_k leaves
    const bool cuts = first_k < all || pp < 1.0f || mp > 0.0f;
    if (all && !greedy && ((cuts && all <= TINY) || (rich && first_k < all && first_k <= FEW / 2))) {
        float at_least = -FLT_MAX;
        if (all > TINY) {
            // At least k logits of the row are no smaller than the least of the rich CTAs' (k / rich)-th largest of their threads' largest; a bin's lower end will do
            const uint32_t want = (first_k + rich - 1) / rich;
            s.count[threadIdx.x] = 0;
            if (threadIdx.x == 0) s.found_bin = BINS;
            const bool some = mine > -INFINITY;
            const float best = of_key(R.max_cta(key_of(mine))), worst = of_key(~R.max_cta(some ? ~key_of(mine) : 0)), width = (best - worst) * (1.0f / BINS);
            const bool even = width > 0.0f && width < INFINITY;                  // (else they are all equal: no bound)
            if (even && some) atomicAdd(&s.count[min(BINS - 1, (uint32_t)((best - mine) / width))], 1u);
            __syncthreads();
            uint64_t threads;
            const uint32_t c = s.count[threadIdx.x], upto = (uint32_t)R.scan_cta(c, threads);
            if (even && upto >= want && upto - c < want) s.found_bin = threadIdx.x;
            __syncthreads();
            const float end = best - ((float)s.found_bin + 1.001f) * width - 1e-6f * (fabsf(best) + fabsf(worst));
            R.tell(have < p.slice / 2 ? 0xffffffffu : key_of(s.found_bin < BINS && end > -FLT_MAX ? end : -FLT_MAX));
            uint32_t bound = 0xffffffffu;
            for (uint32_t r = 0; r < p.split; r++) bound = min(bound, (uint32_t)R.heard(r, 0));
            at_least = of_key(bound);
        }
        if (threadIdx.x == 0) s.listed = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < fours; i += THREADS) {
            const float4 v = R.fours(i);
            if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= at_least) {
                const float l[4] = { v.x, v.y, v.z, v.w };
#pragma unroll
                for (uint32_t j = 0; j < 4; j++)
                    if (l[j] >= at_least) {
                        const uint32_t at = atomicAdd(&s.listed, 1u);
                        if (at < FEW) { s.few[at].l = l[j]; s.few[at].index = from + 4 * i + j - lead; }
                    }
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
                if (threadIdx.x >= many && threadIdx.x < (many + 7) / 8 * 8) s.few[threadIdx.x] = me;       // (nothing, behind the last)
                __syncthreads();
                uint32_t place = 0;
                uint64_t before = 0;
                if (warp * 32 < many)
                    for (uint32_t i = 0; i < many; i += 8) {
                        Item o[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) o[j] = s.few[i + j];
#pragma unroll
                        for (int j = 0; j < 8; j++) if (o[j].l > me.l || (o[j].l == me.l && o[j].index < me.index)) { place++; before += o[j].w; }
                    }
                bool keep = threadIdx.x < many && place < first_k;
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
                    for (uint32_t i = 0; i < many; i += 8) {
                        uint32_t index[8];
                        uint64_t weigh[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) { index[j] = s.few[i + j].index; weigh[j] = s.few[i + j].w; }
#pragma unroll
                        for (int j = 0; j < 8; j++) if (index[j] <= me.index) upto += weigh[j];
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
    bool summed = false;
    if (all && greedy) { cut = top; ties = 1; }
    if (all && !greedy) {
        if (first_k < all) {
            uint64_t above = 0;
            cut = R.template select<false>(w, low, top, first_k, above);
            ties = (uint32_t)(first_k - above);
        }
        if (pp < 1.0f && w.fast) summed = R.mass_cut(w, pp, cut, ties);
        else if (pp < 1.0f) {
            uint64_t sum = 0;
            const float over = of_key(cut);
            float close = INFINITY;
            R.each([&](float l) { if (l > over) { sum += w.exact(l); close = fminf(close, l); } });
            sum = R.sum_cta(sum);
            uint32_t nearest = ~R.max_cta(~key_of(close));
            R.tell(sum, nearest);
            sum = 0; nearest = 0xffffffffu;
            for (uint32_t r = 0; r < p.split; r++) { sum += R.heard(r, 0); nearest = min(nearest, (uint32_t)R.heard(r, 1)); }
            const uint64_t each = ties ? w(over) : 0;
            const double want = ceil((double)pp * (double)(sum + ties * each));
            const uint64_t goal = want >= 1.0 ? (uint64_t)want : 1;
            if (sum < goal) ties = (uint32_t)min((uint64_t)ties, (goal - sum + each - 1) / max(each, (uint64_t)1));
            else {
                uint64_t above = 0;
                cut = R.template select<true>(w, nearest, top, goal, above);
                const uint64_t one = w(of_key(cut));
                ties = (uint32_t)((goal - above + one - 1) / one);
            }
        }
        if (mp > 0.0f) {
            if (mp > 1.0f) { cut = top; ties = 1; summed = false; }
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
                if (b - 1 >= cut) { cut = b - 1; ties = 0; summed = false; }
            }
        }
    }

    // Sums of what is left and numbers of logits equal to the cut, for every piece
    const float over = of_key(cut);
    if (!summed) {
        __syncthreads();
        if (threadIdx.x == 0) s.left = 0;
        __syncthreads();
        uint32_t left = 0;
        w.with([&](auto weight) {
            for (uint32_t q = 0; q < PIECES / WARPS; q++) {
                uint64_t sum = 0;
                uint32_t same = 0;
                R.each_of_piece(q, [&](float l) {
                    const uint64_t one = weight(l);
                    if (l > over) { sum += one; left++; }
                    same += l == over;
                });
                sum = R.sum_warp(sum);
                same = __reduce_add_sync(0xffffffffu, same);
                if (lane == 0) { s.piece_sum[warp * (PIECES / WARPS) + q] = sum; s.piece_equal[warp * (PIECES / WARPS) + q] = same; }
            }
        });
        left = __reduce_add_sync(0xffffffffu, left);
        if (lane == 0) atomicAdd(&s.left, left);
    }
    __syncthreads();
    // The ties that are left are the first in the order of the vocabulary.  (Every warp the same, two pieces a lane: no barrier in between.)
    const uint64_t each = ties ? w(over) : 0;
    const uint32_t e0 = ties ? s.piece_equal[2 * lane] : 0, e1 = ties ? s.piece_equal[2 * lane + 1] : 0;
    uint32_t before0 = 0, t0 = 0, t1 = 0;                                        // equal logits in front of this lane's pieces; ties of them
    if (ties) {                                                                  // (the same in all threads of the cluster)
        uint32_t upto = e0 + e1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= (uint32_t)o) upto += v; }
        R.tell(__shfl_sync(0xffffffffu, upto, 31));
        before0 = upto - e0 - e1;
        for (uint32_t r = 0; r < rank; r++) before0 += (uint32_t)R.heard(r, 0);
        t0 = ties > before0 ? min(e0, ties - before0) : 0;
        t1 = ties > before0 + e0 ? min(e1, ties - before0 - e0) : 0;
    }
    const uint64_t a0 = s.piece_sum[2 * lane] + t0 * each, a1 = s.piece_sum[2 * lane + 1] + t1 * each;
    uint64_t upto = a0 + a1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const uint64_t v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= (uint32_t)o) upto += v; }
    const uint64_t cta = __shfl_sync(0xffffffffu, upto, 31);
    R.tell(cta, s.left + __reduce_add_sync(0xffffffffu, t0 + t1));
    uint64_t before = 0, total = 0, left_all = 0;
    for (uint32_t r = 0; r < p.split; r++) { const uint64_t c = R.heard(r, 0); if (r < rank) before += c; total += c; left_all += R.heard(r, 1); }

    if (total == 0) {
        if (rank == 0 && threadIdx.x == 0) { p.tokens[row] = -1; if (p.probs) p.probs[row] = 0.0f; if (p.kept) p.kept[row] = 0; }
    } else {
        const double goal_d = u * (double)total;
        const uint64_t goal = goal_d >= (double)(total - 1) ? total - 1 : (uint64_t)goal_d;
        if (warp == 0 && before <= goal && goal < before + cta) {                // in this CTA: in which piece, and where
            const uint32_t in = (uint32_t)__ffs((int)__ballot_sync(0xffffffffu, before + upto > goal)) - 1;
            uint64_t run = before + __shfl_sync(0xffffffffu, upto - a0 - a1, in);
            uint32_t seen = __shfl_sync(0xffffffffu, before0, in), piece = 2 * in;
            const uint64_t first_sum = __shfl_sync(0xffffffffu, a0, in);
            const uint32_t first_equal = __shfl_sync(0xffffffffu, e0, in);
            if (run + first_sum <= goal) { run += first_sum; seen += first_equal; piece++; }
            const uint32_t a = piece * R.per_piece, b = min(fours, a + R.per_piece);
            for (uint32_t i0 = a; i0 < b; i0 += 32) {
                const uint32_t i = i0 + lane;
                const float4 four = i < b ? R.fours(i) : R.nothing();
                const float l[4] = { four.x, four.y, four.z, four.w };
                uint64_t one[4], mine4 = 0;
                uint32_t same = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) same += ties && l[j] == over;
                uint32_t tie = same;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const uint32_t v = __shfl_up_sync(0xffffffffu, tie, o); if (lane >= (uint32_t)o) tie += v; }
                const uint32_t ties_here = __shfl_sync(0xffffffffu, tie, 31);
                tie += seen - same;                                          // equal logits in front of this lane's
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    one[j] = l[j] > over ? w(l[j]) : (ties && l[j] == over && tie++ < ties ? each : 0);
                    mine4 += one[j];
                }
                uint64_t past = mine4;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const uint64_t v = __shfl_up_sync(0xffffffffu, past, o); if (lane >= (uint32_t)o) past += v; }
                const uint32_t over_goal = __ballot_sync(0xffffffffu, run + past > goal);
                if (over_goal) {
                    if (lane == (uint32_t)__ffs((int)over_goal) - 1) {
                        uint64_t sum = run + past - mine4;
                        int j = 0;
                        uint64_t w1 = one[0];
                        if (sum + w1 <= goal) { sum += w1; j = 1; w1 = one[1]; if (sum + w1 <= goal) { sum += w1; j = 2; w1 = one[2]; if (sum + w1 <= goal) { j = 3; w1 = one[3]; } } }
                        p.tokens[row] = (int32_t)(from + 4 * i + j - lead);
                        if (p.probs) p.probs[row] = (float)((double)w1 / (double)total);
                        if (p.kept) p.kept[row] = (int32_t)left_all;
                    }
                    break;
                }
                run += __shfl_sync(0xffffffffu, past, 31);
                seen += ties_here;
            }
        }
    }
    R.sync();                                                                    // (nobody leaves while its shared memory is read)
}

template <typename T, bool STREAM> int launch(const SampleParams &p, const SpgDeviceProps &dp, int dev, cudaStream_t stream)
{
    static SpgOncePerDevice once;
    const int rc = once.run(dev, [&]() -> int {
        SPGK_CUDA(cudaFuncSetAttribute(spg_sample_kernel<T, STREAM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dp.smem_optin));
        return SPGK_OK;
    });
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.N * p.split); cfg.blockDim = dim3(THREADS); cfg.stream = stream;
    cfg.dynamicSmemBytes = STREAM ? sizeof(Shared<float>) : sizeof(Shared<uint16_t>) + (size_t)p.slice * 4 + 32;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    SPGK_CUDA(cudaLaunchKernelEx(&cfg, spg_sample_kernel<T, STREAM>, p));
    return spgk_check_launch("spg_sample_kernel");
}

template <typename T> int launch_rows(SampleParams p, const SpgDeviceProps &dp, int dev, cudaStream_t stream)
{
    // Rows that would fill an SM's shared memory, and enough of them: a CTA each, two an SM, which reads its row again for every pass instead of keeping it.
    // us kept and streamed, with top_p: 256 x 131072 228 and 143, 148 x 131072 143 and 95, 148 x 60000 57 and 50, 512 x 32000 106 and 97; 96 x 131072 88 and 115,
    // 512 x 16000 with top_k 21 and 23, 64 x 50001 14 and 17.
    const bool streamed = p.width > SLICE / 2 && p.N >= (uint32_t)dp.sm_count * 7 / 8;
    p.split = 1;
    while (!streamed && p.split < MAX_SPLIT && (p.width > p.split * SLICE || (p.width > p.split * 2048u && (uint64_t)p.N * p.split * 2 <= (uint32_t)dp.sm_count * 2u))) p.split *= 2;
    p.slice = ((p.width + p.split - 1) / p.split + 7u) / 8u * 8u;
    if ((uint64_t)p.N * p.split > 0x7fffffffu) { spgk_set_error("spgk_sample_rows", "too many rows"); return SPGK_E_ARG; }
    return streamed ? launch<T, true>(p, dp, dev, stream) : launch<T, false>(p, dp, dev, stream);
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
    SampleParams p{ logits, ld, N, width, 1, width, temperature, top_k, top_p, min_p, u, tokens, probs, kept };
    if (type == SPGK_T_F32) return launch_rows<float>(p, dp, dev, (cudaStream_t)stream);
    if (type == SPGK_T_F16) return launch_rows<__half>(p, dp, dev, (cudaStream_t)stream);
    return launch_rows<__nv_bfloat16>(p, dp, dev, (cudaStream_t)stream);
}
