// spg_route.cu -- rows to experts and back: a router's choice, the order of the rows by expert, and the weighted sum of what the experts made of them.
//
//   choice : the first top_k of a row by (logit, falling; index, rising); gate = exp(l - m) / sum
//   order  : place(n, j) = starts[e] + how many pairs in front of (n, j), in the order of the rows, have the same expert e = chosen[n][j]
//   sum    : out[n] = sum_j gate[n][j] * y[place[n][j]]
//
// A warp has a row of logits, up to 32 a lane, and takes its largest out one after the other.  The order is a counting sort that hangs on nothing's timing.  Few rows go
// through one block of threads, choice and order (more than 256 experts do not: a row's logits need more registers than so many threads have); more rows' pairs, their choice made by all SMs,
// through a cluster.  Many pairs are cut into parts: as each part's choice is made its pairs are counted by expert, one cluster sums the counts up over the
// parts and experts, and then each part finds its pairs' places from where its experts begin.  The counts lie in the memory of the results on the way: in that of the order,
// which is written last, and where a part's experts begin in that of its places, which only this part reads and writes.
// What bounds it: latency, of three ways from memory to memory, and 520 instructions a row of 256 logits (us, bf16: 16384 rows to 8 of 256 experts 22.6, 12 of them the choice; 16384 to 2 of 64 13.1,
// the pairs in one cluster 14.5; 2000 to 8 of 256 14.3 in parts, 11.1 in one cluster; 32 to 2 of 8 4.6 in one block, 6.1 in two launches; one row 3.8).
#include "spg_fp8.cuh"
#include <type_traits>

namespace {

using namespace spgfp8;

constexpr uint32_t CHOOSE_THREADS = 512, CHOOSE_WARPS = CHOOSE_THREADS / 32u;
constexpr uint32_t THREADS = 256, WARPS = THREADS / 32u, LEAST = 64;       // of a part: its order's threads, and the pairs that it has at least
constexpr uint32_t ONE_THREADS = 1024, ONE_WARPS = ONE_THREADS / 32u, ONE_ROWS = 32, ONE_V = 8;      // where one block of threads has all rows
constexpr uint32_t SUM_THREADS = 1024, SUM_CLUSTER = 8, SUM_PAIRS = 16384;    // up to so many pairs, one cluster has all of them

// order of floats as that of unsigned numbers; -infinity comes lowest, above 0, which no logit has
__device__ __forceinline__ uint32_t key_of(float v)
{
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ float closed() { return __int_as_float(0xff800000); }

// V neighbouring logits from e0 on (-infinity beyond the last); vec: rows lie on what a lane reads
template <typename T, uint32_t V> struct Logits { alignas(16) T t[V]; };
template <typename T, uint32_t V> __device__ __forceinline__ void load_logits(const T *row, uint32_t e0, uint32_t experts, bool vec, Logits<T, V> &l)
{
    constexpr uint32_t bytes = V * sizeof(T), word = bytes >= 16 ? 16 : bytes;
    if (vec && e0 + V <= experts) {
#pragma unroll
        for (uint32_t i = 0; i < bytes / word; i++) {
            if constexpr (word == 16) reinterpret_cast<uint4 *>(l.t)[i] = reinterpret_cast<const uint4 *>(row + e0)[i];
            else if constexpr (word == 8) reinterpret_cast<uint2 *>(l.t)[i] = reinterpret_cast<const uint2 *>(row + e0)[i];
            else if constexpr (word == 4) reinterpret_cast<uint32_t *>(l.t)[i] = reinterpret_cast<const uint32_t *>(row + e0)[i];
            else l.t[i] = row[e0 + i];
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < V; i++) l.t[i] = e0 + i < experts ? row[e0 + i] : from_f32<T>(closed());
    }
}

// Falling order in a lane: exchanges whose places are known when this is compiled (Batcher's merges of odd and even places).  Equal keys change places only
// where LATER, the index behind the key, says so.
template <uint32_t V, bool LATER> __device__ __forceinline__ void sort_lane(uint32_t (&key)[V], uint32_t (&at)[V])
{
#pragma unroll
    for (uint32_t run = 1; run < V; run *= 2)
#pragma unroll
        for (uint32_t gap = run; gap >= 1; gap /= 2)
#pragma unroll
            for (uint32_t j = gap % run; j + gap < V; j += 2 * gap)
#pragma unroll
                for (uint32_t i = 0; i < gap; i++) {
                    const uint32_t a = i + j, b = i + j + gap;
                    if (b >= V || a / (2 * run) != b / (2 * run)) continue;
                    if constexpr (!LATER) {
                        const uint32_t hi = max(key[a], key[b]), lo = min(key[a], key[b]);
                        key[a] = hi; key[b] = lo;
                    } else {
                        const bool turn = key[b] > key[a] || (key[b] == key[a] && at[b] < at[a]);
                        const uint32_t k = key[a], n = at[a];
                        key[a] = turn ? key[b] : k; key[b] = turn ? k : key[b];
                        at[a] = turn ? at[b] : n; at[b] = turn ? n : at[b];
                    }
                }
}

// One row by one warp: lane j's expert and gate (-1, 0 where there are fewer).  V: logits a lane, whose order it makes first; then the largest of the lanes' first is the next,
// top_k times.  16-bit logits are searched as keys with the index behind them, so that the maximum over the warp names the expert too; of 32-bit ones that are equal the first
// lane's is the first.
template <typename T, uint32_t V>
__device__ __forceinline__ int32_t choose(const Logits<T, V> &logits, uint32_t top_k, bool normalise, uint32_t lane, float &gate)
{
    constexpr bool SHORT = sizeof(T) == 2;
    float l[V];
    uint32_t key[V], at[V];
    if constexpr (SHORT && V > 1) {
        // two at a time: the larger of a NaN and -infinity is -infinity, -0 and 0 are 0, and the order of numbers becomes that of their bits
#pragma unroll
        for (uint32_t i = 0; i < V; i += 2) {
            uint32_t w = *reinterpret_cast<const uint32_t *>(logits.t + i);
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 v = __hadd2(__hmax2(*reinterpret_cast<const __half2 *>(&w), __half2half2(__ushort_as_half(0xfc00))), __half2half2(__ushort_as_half(0)));
                const float2 f = __half22float2(v);
                l[i] = f.x; l[i + 1] = f.y;
                w = *reinterpret_cast<const uint32_t *>(&v);
            } else {
                const __nv_bfloat162 v = __hadd2(__hmax2(*reinterpret_cast<const __nv_bfloat162 *>(&w), __bfloat162bfloat162(__ushort_as_bfloat16(0xff80))), __bfloat162bfloat162(__ushort_as_bfloat16(0)));
                w = *reinterpret_cast<const uint32_t *>(&v);
                l[i] = __uint_as_float(w << 16); l[i + 1] = __uint_as_float(w & 0xffff0000u);
            }
            const uint32_t k = w ^ ((w >> 15 & 0x00010001u) * 0xffffu | 0x80008000u);
            key[i] = __byte_perm(0xffffu - (lane * V + i), k, 0x5410);
            key[i + 1] = __byte_perm(0xffffu - (lane * V + i + 1), k, 0x7610);
            at[i] = at[i + 1] = 0;
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < V; i++) {
            l[i] = fmaxf(to_f32(logits.t[i]), closed()) + 0.0f;                  // (as above)
            const uint32_t e = lane * V + i;
            at[i] = e;
            if constexpr (SHORT) {
                const T t = from_f32<T>(l[i]);
                const uint32_t b = *reinterpret_cast<const uint16_t *>(&t);
                key[i] = (b ^ (b & 0x8000u ? 0xffffu : 0x8000u)) << 16 | (0xffffu - e);
            } else key[i] = key_of(l[i]);
        }
    }
    const auto of = [](uint32_t k) {
        if constexpr (SHORT) {
            const uint16_t b = (uint16_t)(k & 0x80000000u ? k >> 16 & 0x7fffu : ~(k >> 16));
            return to_f32(*reinterpret_cast<const T *>(&b));
        } else return value_of(k);
    };
    // the largest logit, of which all weights are fractions
    uint32_t most = key[0];
#pragma unroll
    for (uint32_t i = 1; i < V; i++) most = max(most, key[i]);
    const float m = of(__reduce_max_sync(0xffffffffu, most));
    float total = 0.0f;
    if (!normalise) {
        if (m < __int_as_float(0x7f800000)) {
#pragma unroll
            for (uint32_t i = 0; i < V; i++) total += expf(l[i] - m);             // (0 for those closed; where all are, nobody asks)
        } else {
#pragma unroll
            for (uint32_t i = 0; i < V; i++) total += l[i] == m ? 1.0f : 0.0f;
        }
        total = spg_warp_sum(total);
    }
    sort_lane<V, !SHORT>(key, at);
    uint32_t mine = 0, place = 0;
    for (uint32_t j = 0; j < top_k; j++) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, key[0]);
        bool first = key[0] == top;
        uint32_t e = 0;
        if constexpr (!SHORT) {
            const uint32_t lanes = __ballot_sync(0xffffffffu, first), one = __ffs(lanes) - 1;
            e = __shfl_sync(0xffffffffu, at[0], one);
            first = lane == one;
        }
        if (lane == j) { mine = top; place = e; }
        if (first) {
#pragma unroll
            for (uint32_t i = 0; i + 1 < V; i++) { key[i] = key[i + 1]; at[i] = at[i + 1]; }
            key[V - 1] = 0;
        }
    }
    const float best = of(mine);
    const bool open = lane < top_k && best > closed();                            // (no key: a NaN)
    const float w = !open ? 0.0f : best == m ? 1.0f : expf(best - m);
    if (normalise) total = spg_warp_sum(w);
    gate = open ? w / total : 0.0f;
    return open ? (int32_t)(SHORT ? 0xffffu - (mine & 0xffffu) : place) : -1;
}

// Where the `count` pairs in `chosen` (shared memory), the first of them pair `first` of all, go: each behind those of its expert that come earlier; place[e] is that of the expert's
// first.  counts: `warps` times `experts` words; pairs: of all parts.  All threads of the block call it; `warps` of them have a run of pairs each.
// (What was written to the results' memory on the way is read back here: calls that wrongly share it read one another's, so nothing is indexed by it unchecked.)
__device__ __forceinline__ void order_pairs(const int32_t *chosen, uint32_t count, uint32_t first, uint32_t pairs, const uint32_t *place, uint32_t *counts, uint32_t warps, uint32_t experts, uint32_t top_k,
                                            int32_t *order, int32_t *places)
{
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, turns = (count + 31u) / 32u, per = (turns + warps - 1) / warps;
    const uint32_t lo = warp < warps ? min(turns, warp * per) * 32u : turns * 32u, hi = warp < warps ? min(count, lo + per * 32u) : 0u;
    uint32_t *mine = counts + warp * experts;
    for (uint32_t i = threadIdx.x; i < warps * experts; i += blockDim.x) counts[i] = 0;
    __syncthreads();
    for (uint32_t i = lo + lane; i < hi; i += 32u) {
        const uint32_t e = (uint32_t)chosen[i];
        if (e < experts) atomicAdd(mine + e, 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
        uint32_t at = place[e];
        for (uint32_t w = 0; w < warps; w++) { const uint32_t c = counts[w * experts + e]; counts[w * experts + e] = at; at += c; }
    }
    __syncthreads();
    for (uint32_t i0 = lo; i0 < hi; i0 += 32u) {
        const uint32_t i = i0 + lane;
        const uint32_t e = i < hi ? (uint32_t)chosen[i] : 0xffffffffu;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        const uint32_t at = e < experts ? mine[e] + __popc(same & ((1u << lane) - 1u)) : 0u;
        __syncwarp();
        if (e < experts && (same >> lane) == 1u) mine[e] = at + 1u;              // (the last of its kind)
        __syncwarp();
        if (i < hi) places[first + i] = e < experts ? (int32_t)at : -1;
        if (e < experts && at < pairs) order[at] = (int32_t)((first + i) / top_k);
    }
}

// Sum over the threads in front and over all, of one value a thread (sums: a word for each of the block's warps)
__device__ __forceinline__ uint32_t scan_block(uint32_t v, uint32_t *sums, uint32_t &all)
{
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
    uint32_t upto = v;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= (uint32_t)o) upto += u; }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    uint32_t front = 0;
    all = 0;
    for (uint32_t w = 0; w < blockDim.x / 32u; w++) { const uint32_t s = sums[w]; if (w < warp) front += s; all += s; }
    return front + upto - v;
}

// Few rows, choice and order.  Shared memory: chosen, counts of the warps, places of the experts
template <typename T, uint32_t V>
__global__ void __launch_bounds__(ONE_THREADS) spg_route_one_kernel(const T *logits, uint32_t ld, uint32_t N, uint32_t experts, uint32_t top_k, int normalise, bool vec, uint32_t warps,
                                                                    int32_t *chosen, float *gates, int32_t *starts, int32_t *order, int32_t *places)
{
    extern __shared__ uint32_t sh[];
    __shared__ uint32_t sums[ONE_WARPS];
    const uint32_t pairs = N * top_k, warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
    int32_t *mine = reinterpret_cast<int32_t *>(sh);
    uint32_t *counts = sh + (pairs + 31u) / 32u * 32u, *place = counts + warps * experts;
    spg_grid_trigger();
    for (uint32_t e = threadIdx.x; e < experts; e += ONE_THREADS) place[e] = 0;
    spg_grid_wait();
    __syncthreads();
    for (uint32_t n = warp; n < N; n += ONE_WARPS) {
        Logits<T, V> l;
        load_logits(logits + (uint64_t)n * ld, lane * V, experts, vec, l);
        float gate;
        const int32_t e = choose(l, top_k, normalise, lane, gate);
        if (lane < top_k) {
            const uint32_t i = n * top_k + lane;
            chosen[i] = mine[i] = e;
            gates[i] = gate;
            if (e >= 0) atomicAdd(place + e, 1u);
        }
    }
    __syncthreads();
    uint32_t all;
    const uint32_t begin = scan_block(threadIdx.x < experts ? place[threadIdx.x] : 0u, sums, all);
    if (threadIdx.x < experts) { place[threadIdx.x] = begin; starts[threadIdx.x] = (int32_t)begin; }
    if (threadIdx.x == 0) starts[experts] = (int32_t)all;
    __syncthreads();
    order_pairs(mine, pairs, 0, pairs, place, counts, warps, experts, top_k, order, places);
    for (uint32_t i = all + threadIdx.x; i < pairs; i += ONE_THREADS) order[i] = -1;
}

// A part's choice (rows `share` times blockIdx.x on; the last part has the rest), and how many of its pairs each expert has
template <typename T, uint32_t V>
__global__ void __launch_bounds__(CHOOSE_THREADS) spg_route_choose_kernel(const T *logits, uint32_t ld, uint32_t N, uint32_t experts, uint32_t top_k, int normalise, bool vec, uint32_t share, bool count,
                                                                   int32_t *chosen, float *gates, uint32_t *counts)
{
    extern __shared__ uint32_t sh[];
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, lo = blockIdx.x * share, hi = blockIdx.x + 1 == gridDim.x ? N : lo + share;
    spg_grid_trigger();
    if (count) for (uint32_t e = threadIdx.x; e < experts; e += CHOOSE_THREADS) sh[e] = 0;
    spg_grid_wait();
    __syncthreads();
    for (uint32_t n = lo + warp; n < hi; n += CHOOSE_WARPS) {
        Logits<T, V> l;
        load_logits(logits + (uint64_t)n * ld, lane * V, experts, vec, l);
        float gate;
        const int32_t e = choose(l, top_k, normalise, lane, gate);
        if (lane < top_k) {
            chosen[n * top_k + lane] = e;
            gates[n * top_k + lane] = gate;
            if (count && e >= 0) atomicAdd(sh + e, 1u);
        }
    }
    if (!count) return;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += CHOOSE_THREADS) counts[(uint64_t)blockIdx.x * experts + e] = sh[e];
}

__device__ __forceinline__ uint32_t ld_cluster(const uint32_t *here, uint32_t rank)
{
    uint32_t addr = (uint32_t)__cvta_generic_to_shared(here), v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ void cluster_sync()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Where one expert's pairs begin, over all blocks of a cluster and for this one, out of how many each block has (all: this thread's expert's; 0 from `experts` on).  blocks: SUM_CLUSTER at most
__device__ __forceinline__ uint32_t scan_cluster(const uint32_t *all, uint32_t experts, uint32_t blocks, uint32_t rank, uint32_t *sums, int32_t *starts, uint32_t &total)
{
    uint32_t before = 0, whole = 0;
    if (threadIdx.x < experts) {
        uint32_t v[SUM_CLUSTER];
#pragma unroll
        for (uint32_t r = 0; r < SUM_CLUSTER; r++) v[r] = r < blocks ? ld_cluster(all + threadIdx.x, r) : 0u;
#pragma unroll
        for (uint32_t r = 0; r < SUM_CLUSTER; r++) { whole += v[r]; if (r < rank) before += v[r]; }
    }
    const uint32_t at = scan_block(whole, sums, total);
    if (rank == 0 && threadIdx.x < experts) starts[threadIdx.x] = (int32_t)at;
    if (rank == 0 && threadIdx.x == 0) starts[experts] = (int32_t)total;
    return at + before;
}

// The order of pairs that are not many, their choice made: a cluster has them, its blocks a run each.  Shared memory: chosen, counts of the warps, places of the experts, and how many
// pairs of each the block has
__global__ void __launch_bounds__(ONE_THREADS) spg_route_pairs_kernel(const int32_t *chosen, uint32_t pairs, uint32_t experts, uint32_t top_k, uint32_t per, uint32_t warps,
                                                                      int32_t *starts, int32_t *order, int32_t *places)
{
    extern __shared__ uint32_t sh[];
    __shared__ uint32_t sums[ONE_WARPS];
    const uint32_t rank = blockIdx.x, blocks = gridDim.x, lo = min(pairs, rank * per), count = min(pairs, lo + per) - lo;
    int32_t *mine = reinterpret_cast<int32_t *>(sh);
    uint32_t *counts = sh + per, *place = counts + warps * experts, *all = place + experts;
    spg_grid_trigger();
    for (uint32_t e = threadIdx.x; e < experts; e += ONE_THREADS) all[e] = 0;
    spg_grid_wait();
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count; i += ONE_THREADS) {
        const uint32_t e = (uint32_t)chosen[lo + i];
        mine[i] = (int32_t)e;
        if (e < experts) atomicAdd(all + e, 1u);
    }
    __syncthreads();
    cluster_sync();
    uint32_t total;
    const uint32_t at = scan_cluster(all, experts, blocks, rank, sums, starts, total);
    if (threadIdx.x < experts) place[threadIdx.x] = at;
    __syncthreads();
    order_pairs(mine, count, lo, pairs, place, counts, warps, experts, top_k, order, places);
    for (uint64_t i = (uint64_t)total + rank * ONE_THREADS + threadIdx.x; i < pairs; i += blocks * ONE_THREADS) order[i] = -1;
    cluster_sync();                                              // (the others may still read this block's counts)
}

// Counts [parts][experts] to where each part's pairs of each expert begin (first[part * stride + expert]), and where each expert's do.  A cluster: its blocks have the parts in
// runs, a block's threads an expert each and, where there are few experts, a run of the block's parts.
__global__ void __launch_bounds__(SUM_THREADS) spg_route_sum_kernel(const uint32_t *counts, uint32_t parts, uint32_t experts, uint32_t wide, uint32_t stride, uint32_t *first, int32_t *starts)
{
    __shared__ uint32_t run[SUM_THREADS], all[SPGK_MAX_EXPERTS], begin[SPGK_MAX_EXPERTS], sums[SUM_THREADS / 32u];
    const uint32_t rank = blockIdx.x, e = threadIdx.x % wide, slice = threadIdx.x / wide, slices = SUM_THREADS / wide;      // wide: experts, up to a whole warp
    const uint32_t per = (parts + SUM_CLUSTER * slices - 1) / (SUM_CLUSTER * slices), lo = min(parts, (rank * slices + slice) * per), hi = e < experts && slice < slices ? min(parts, lo + per) : lo;
    constexpr uint32_t KEPT = 16;                                // of a run, on their way at a time and at hand the second time
    uint32_t c[KEPT];
    const auto load = [&](uint32_t b0) {
#pragma unroll
        for (uint32_t i = 0; i < KEPT; i++) c[i] = b0 + i < hi ? counts[(uint64_t)(b0 + i) * experts + e] : 0u;
    };
    spg_grid_trigger();
    spg_grid_wait();
    uint32_t sum = 0;
    for (uint32_t b = lo; b < hi; b += KEPT) {
        load(b);
#pragma unroll
        for (uint32_t i = 0; i < KEPT; i++) sum += c[i];
    }
    run[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < experts) {
        uint32_t upto = 0;
#pragma unroll 4
        for (uint32_t s = 0; s < slices; s++) { const uint32_t v = run[s * wide + threadIdx.x]; run[s * wide + threadIdx.x] = upto; upto += v; }
        all[threadIdx.x] = upto;
    }
    cluster_sync();
    uint32_t total;
    const uint32_t at = scan_cluster(all, experts, SUM_CLUSTER, rank, sums, starts, total);
    if (threadIdx.x < experts) begin[threadIdx.x] = at;
    __syncthreads();
    if (lo < hi) {
        uint32_t upto = begin[e] + run[slice * wide + e];
        for (uint32_t b = lo; b < hi; b += KEPT) {
            if (per > KEPT) load(b);
#pragma unroll
            for (uint32_t i = 0; i < KEPT; i++) if (b + i < hi) { first[(uint64_t)(b + i) * stride + e] = upto; upto += c[i]; }
        }
    }
    cluster_sync();                                              // (the others may still read this block's sums)
}

// A part's pairs to their places.  Shared memory: chosen, counts of the warps, places of the experts
__global__ void __launch_bounds__(THREADS) spg_route_order_kernel(const int32_t *chosen, uint32_t N, uint32_t experts, uint32_t top_k, uint32_t share, const int32_t *starts, int32_t *order, int32_t *places)
{
    extern __shared__ uint32_t sh[];
    const uint32_t lo = blockIdx.x * share * top_k, pairs = N * top_k, count = (blockIdx.x + 1 == gridDim.x ? pairs : lo + share * top_k) - lo;
    int32_t *mine = reinterpret_cast<int32_t *>(sh);
    uint32_t *counts = sh + (count + 31u) / 32u * 32u, *place = counts + WARPS * experts;
    spg_grid_trigger();
    spg_grid_wait();
    for (uint32_t i = threadIdx.x; i < count; i += THREADS) mine[i] = chosen[lo + i];
    for (uint32_t e = threadIdx.x; e < experts; e += THREADS) place[e] = (uint32_t)places[lo + e];     // (where the sums left them; this part's places go there)
    __syncthreads();
    order_pairs(mine, count, lo, pairs, place, counts, WARPS, experts, top_k, order, places);
    for (uint64_t i = (uint64_t)(uint32_t)starts[experts] + blockIdx.x * THREADS + threadIdx.x; i < pairs; i += gridDim.x * THREADS) order[i] = -1;
}

// A thread has U times W neighbouring columns of a row: W are 16 bytes of the narrower type, or one where rows do not lie on 16 bytes; U is 1, and the rows' pieces
// go to threads one behind the other, or 2 or 4 where a row has enough of them for a block of threads of its own.  ROWS of the rows that are added up are on their way at a time; where a block has
// one row, a warp's lanes have its places, and those that are none are passed over.
// What bounds it is how many bytes are on their way: a place, then the rows, then the sum is a way of three latencies.  us with U = 1, 2 and 4: 16384 x 2 rows of 8192 bf16 163, 126 and 120
// (6.7 TB/s; 145 through the caches as usual), 4096 x 2 of 4096 19.7, 14.2 and, half of the threads idle, 19.3.
template <typename T, typename O, uint32_t W, uint32_t U, uint32_t ROWS>
__global__ void __launch_bounds__(256) spg_combine_kernel(const T *y, uint32_t ldy, uint32_t y_rows, const int32_t *places, const float *gates, uint32_t N, uint32_t top_k,
                                                          O *out, uint32_t ldo, uint32_t pieces)
{
    spg_grid_trigger();
    spg_grid_wait();
    uint32_t n, first;                                           // the row, and the first of this thread's pieces, the next 256 from it
    if constexpr (U == 1) {
        const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
        if (i >> 32) { n = (uint32_t)(i / pieces); first = (uint32_t)(i % pieces); }
        else { n = (uint32_t)i / pieces; first = (uint32_t)i % pieces; }
        if (n >= N) return;
    } else {
        const uint32_t blocks = (pieces - 1) / (256u * U) + 1;
        n = blockIdx.x / blocks; first = blockIdx.x % blocks * 256u * U + threadIdx.x;
    }
    float v[U][W];
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
#pragma unroll
        for (uint32_t q = 0; q < W; q++) v[u][q] = 0.0f;
    // rows p[k] with gates g[k], those that there are
    const auto add = [&](const uint32_t (&p)[ROWS], const float (&g)[ROWS]) {
        alignas(16) T t[ROWS][U][W];
#pragma unroll
        for (uint32_t k = 0; k < ROWS; k++) {
            const T *row = y + (uint64_t)(p[k] < y_rows ? p[k] : 0u) * ldy;
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                const uint32_t c = (first + u * 256u) * W;
                if (p[k] >= y_rows || (U > 1 && first + u * 256u >= pieces)) continue;
                if constexpr (W * sizeof(T) % 16 == 0) {
#pragma unroll
                    for (uint32_t q = 0; q < W * sizeof(T) / 16; q++) reinterpret_cast<uint4 *>(t[k][u])[q] = __ldcs(reinterpret_cast<const uint4 *>(row + c) + q);
                } else {
#pragma unroll
                    for (uint32_t q = 0; q < W; q++) t[k][u][q] = row[c + q];
                }
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < ROWS; k++) {
            if (p[k] >= y_rows) continue;
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
#pragma unroll
                for (uint32_t q = 0; q < W; q++) v[u][q] = fmaf(g[k], to_f32(t[k][u][q]), v[u][q]);
        }
    };
    const uint64_t at = (uint64_t)n * top_k;
    if constexpr (U == 1) {
        for (uint32_t j = 0; j < top_k; j += ROWS) {
            uint32_t p[ROWS];
            float g[ROWS];
#pragma unroll
            for (uint32_t k = 0; k < ROWS; k++) {
                p[k] = j + k < top_k ? (uint32_t)places[at + j + k] : 0xffffffffu;
                g[k] = j + k < top_k ? gates[at + j + k] : 0.0f;
            }
            add(p, g);
        }
    } else {
        const uint32_t lane = threadIdx.x % 32u;
        for (uint32_t j = 0; j < top_k; j += 32u) {
            const uint32_t place = j + lane < top_k ? (uint32_t)places[at + j + lane] : 0xffffffffu;
            const float gate = j + lane < top_k ? gates[at + j + lane] : 0.0f;
            for (uint32_t left = __ballot_sync(0xffffffffu, place < y_rows); left;) {
                uint32_t p[ROWS];
                float g[ROWS];
#pragma unroll
                for (uint32_t k = 0; k < ROWS; k++) {
                    const uint32_t one = left ? __ffs(left) - 1 : 0u;
                    p[k] = __shfl_sync(0xffffffffu, place, one);
                    g[k] = __shfl_sync(0xffffffffu, gate, one);
                    if (!left) p[k] = 0xffffffffu;
                    left &= left - 1;
                }
                add(p, g);
            }
        }
    }
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
        const uint32_t c = (first + u * 256u) * W;
        if (U > 1 && first + u * 256u >= pieces) continue;
        O *dst = out + (uint64_t)n * ldo + c;
        alignas(16) O o[W];
#pragma unroll
        for (uint32_t q = 0; q < W; q++) o[q] = from_f32<O>(v[u][q]);
        if constexpr (W * sizeof(O) % 16 == 0) {
#pragma unroll
            for (uint32_t q = 0; q < W * sizeof(O) / 16; q++) __stcs(reinterpret_cast<uint4 *>(dst) + q, reinterpret_cast<const uint4 *>(o)[q]);
        } else {
#pragma unroll
            for (uint32_t q = 0; q < W; q++) dst[q] = o[q];
        }
    }
}

int refuse(const char *who, const char *why) { spgk_set_error(who, why); return SPGK_E_ARG; }
bool known(int type) { return type == SPGK_T_F16 || type == SPGK_T_BF16 || type == SPGK_T_F32; }
uint32_t size_of(int type) { return type == SPGK_T_F32 ? 4u : 2u; }

struct Route {
    uint32_t ld, N, experts, top_k; int normalise;
    int32_t *chosen; float *gates; int32_t *starts, *order, *places;
    int dev; cudaStream_t stream;
};
void launch_cluster(cudaLaunchConfig_t &cfg, cudaLaunchAttribute (&attr)[2], uint32_t blocks, uint32_t threads, size_t smem, cudaStream_t stream)
{
    cfg.gridDim = dim3(blocks); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
}

// One block of threads has all rows; or the rows are cut and one cluster has all pairs; or rows go in parts of as many pairs as there are experts at least (their counts lie in the memory
// of the pairs' results) and the pairs in the same parts.
template <typename T, uint32_t V> int route(const void *logits, const Route &r)
{
    const uint32_t pairs = r.N * r.top_k, share = ((r.experts > LEAST ? r.experts : LEAST) + r.top_k - 1) / r.top_k, parts = r.N / share;
    const bool vec = (uintptr_t)logits % 16 == 0 && (uint64_t)r.ld * sizeof(T) % 16 == 0, few = r.N <= ONE_ROWS && V <= ONE_V, some = pairs <= SUM_PAIRS;
    const T *x = (const T *)logits;
    int rc;
    if constexpr (V <= ONE_V) {
        if (few) {
            static SpgOncePerDevice once;
            rc = once.run(r.dev, [&]() -> int {
                SPGK_CUDA(cudaFuncSetAttribute(spg_route_one_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((ONE_ROWS * SPGK_ROUTE_MAX_TOP + (ONE_WARPS + 1) * ONE_V * 32u) * 4u)));
                return SPGK_OK;
            });
            if (rc) return rc;
            const uint32_t turns = (pairs + 31u) / 32u, warps = turns < 1 ? 1 : turns < ONE_WARPS ? turns : ONE_WARPS;
            SPGK_CUDA(spg_launch_chained(spg_route_one_kernel<T, V>, dim3(1), dim3(ONE_THREADS), ((size_t)turns * 32u + (size_t)(warps + 1) * r.experts) * 4u, r.stream,
                                         x, r.ld, r.N, r.experts, r.top_k, r.normalise, vec, warps, r.chosen, r.gates, r.starts, r.order, r.places));
            return spgk_check_launch("spg_route_one_kernel");
        }
    }
    if (r.N) SPGK_CUDA(spg_launch_chained(spg_route_choose_kernel<T, V>, dim3(some ? (r.N + CHOOSE_WARPS - 1) / CHOOSE_WARPS : parts), dim3(CHOOSE_THREADS), some ? 0 : r.experts * 4u, r.stream,
                                 x, r.ld, r.N, r.experts, r.top_k, r.normalise, vec, some ? CHOOSE_WARPS : share, !some, r.chosen, r.gates, (uint32_t *)r.order));
    if ((rc = spgk_check_launch("spg_route_choose_kernel"))) return rc;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    if (some) {
        static SpgOncePerDevice once;
        rc = once.run(r.dev, [&]() -> int {
            SPGK_CUDA(cudaFuncSetAttribute(spg_route_pairs_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((SUM_PAIRS / SUM_CLUSTER + 32u + (ONE_WARPS + 2) * SPGK_MAX_EXPERTS) * 4u)));
            return SPGK_OK;
        });
        if (rc) return rc;
        const uint32_t turns = pairs ? (pairs + 31u) / 32u : 1u;
        uint32_t blocks = 1;
        while (blocks < SUM_CLUSTER && turns > blocks * ONE_WARPS) blocks *= 2;
        const uint32_t each = (turns + blocks - 1) / blocks, warps = each < ONE_WARPS ? each : ONE_WARPS;
        launch_cluster(cfg, attr, blocks, ONE_THREADS, ((size_t)each * 32u + (size_t)(warps + 2) * r.experts) * 4u, r.stream);
        SPGK_CUDA(cudaLaunchKernelEx(&cfg, spg_route_pairs_kernel, (const int32_t *)r.chosen, pairs, r.experts, r.top_k, each * 32u, warps, r.starts, r.order, r.places));
        return spgk_check_launch("spg_route_pairs_kernel");
    }
    launch_cluster(cfg, attr, SUM_CLUSTER, SUM_THREADS, 0, r.stream);
    SPGK_CUDA(cudaLaunchKernelEx(&cfg, spg_route_sum_kernel, (const uint32_t *)r.order, parts, r.experts, (r.experts + 31u) / 32u * 32u, share * r.top_k, (uint32_t *)r.places, r.starts));
    if ((rc = spgk_check_launch("spg_route_sum_kernel"))) return rc;
    static SpgOncePerDevice once;
    const size_t most = (2 * (size_t)(SPGK_MAX_EXPERTS + SPGK_ROUTE_MAX_TOP) + 32u + (WARPS + 1) * SPGK_MAX_EXPERTS) * 4u;
    rc = once.run(r.dev, [&]() -> int {
        SPGK_CUDA(cudaFuncSetAttribute(spg_route_order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
        return SPGK_OK;
    });
    if (rc) return rc;
    const uint32_t last = (r.N - (parts - 1) * share) * r.top_k;                 // the most pairs of a part
    SPGK_CUDA(spg_launch_chained(spg_route_order_kernel, dim3(parts), dim3(THREADS), ((size_t)(last + 31u) / 32u * 32u + (size_t)(WARPS + 1) * r.experts) * 4u, r.stream,
                                 (const int32_t *)r.chosen, r.N, r.experts, r.top_k, share, (const int32_t *)r.starts, r.order, r.places));
    return spgk_check_launch("spg_route_order_kernel");
}
template <typename T> int route(const void *logits, const Route &r)
{
    if (r.experts <= 32) return route<T, 1>(logits, r);
    if (r.experts <= 64) return route<T, 2>(logits, r);
    if (r.experts <= 128) return route<T, 4>(logits, r);
    if (r.experts <= 256) return route<T, 8>(logits, r);
    if (r.experts <= 512) return route<T, 16>(logits, r);
    return route<T, 32>(logits, r);
}

template <typename T, typename O>
int combine(const void *y, uint32_t ldy, uint32_t y_rows, const int32_t *places, const float *gates, uint32_t N, uint32_t top_k, uint32_t width, void *out, uint32_t ldo, cudaStream_t stream)
{
    constexpr uint32_t W = 16 / (sizeof(T) < sizeof(O) ? sizeof(T) : sizeof(O));
    const bool wide = width % W == 0 && (uint64_t)ldy * sizeof(T) % 16 == 0 && (uint64_t)ldo * sizeof(O) % 16 == 0 && ((uintptr_t)y | (uintptr_t)out) % 16 == 0;
    const uint32_t pieces = wide ? width / W : width;
    // as many pieces a thread as leave few of them without one and blocks for all SMs (us with 2 and 4, single columns: 1942 x 1 rows of 2061 bf16 17 and 11.5)
    uint32_t u = wide ? 4u : 8u;
    for (; u > 2; u /= 2) {
        const uint64_t each = (pieces - 1) / (256u * u) + 1;
        if (pieces * 10ull >= each * 256u * u * 6u && each * N >= 148u * 4u) break;
    }
    if (u == 2 && pieces < 384u) u = 1;
    const uint64_t blocks = u > 1 ? (uint64_t)N * ((pieces - 1) / (256u * u) + 1) : ((uint64_t)N * pieces + 255) / 256;
    if (blocks > 0x7fffffffu) return refuse("spgk_combine_rows", "too many rows and columns for one call");
    const auto kernel = wide ? (u == 4 ? spg_combine_kernel<T, O, W, 4, 2> : u == 2 ? spg_combine_kernel<T, O, W, 2, 2> : spg_combine_kernel<T, O, W, 1, 4>)
                             : (u == 8 ? spg_combine_kernel<T, O, 1, 8, 2> : u == 4 ? spg_combine_kernel<T, O, 1, 4, 4> : u == 2 ? spg_combine_kernel<T, O, 1, 2, 4> : spg_combine_kernel<T, O, 1, 1, 4>);
    SPGK_CUDA(spg_launch_chained(kernel, dim3((uint32_t)blocks), dim3(256), 0, stream, (const T *)y, ldy, y_rows, places, gates, N, top_k, (O *)out, ldo, pieces));
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
    const void *const results[] = { chosen, gates, starts, order, places };      // (they hold counts on the way)
    for (uint32_t i = 0; N && i < 5; i++)
        for (uint32_t j = 0; j < i; j++) if (results[i] == results[j]) return refuse(who, "two results in one place");
    Route r = { ld, N, experts, top_k, normalise, chosen, gates, starts, order, places, 0, (cudaStream_t)stream };
    SPGK_CUDA(cudaGetDevice(&r.dev));
    if (type == SPGK_T_F32) return route<float>(logits, r);
    if (type == SPGK_T_F16) return route<__half>(logits, r);
    return route<__nv_bfloat16>(logits, r);
}

int spgk_combine_rows(const void *y, int type, uint32_t ldy, uint32_t y_rows, const int32_t *places, const float *gates, uint32_t N, uint32_t top_k,
                      uint32_t width, void *out, int out_type, uint32_t ldo, void *stream)
{
    const char *who = "spgk_combine_rows";
    if (!known(type) || !known(out_type)) return refuse(who, "unknown type");
    if (top_k == 0 || width == 0) return refuse(who, "nothing to add up");
    if (top_k > 0x7fffffffu) return refuse(who, "too many places a row");        // (they are counted through in 32 bits, up to 32 at a time)
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
