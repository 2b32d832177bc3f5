// spg_fp8_layer.cu -- dense layers on 8-bit operands with a scale for each block of 128, one layer for all rows or one for each group of them.
//
//   y[n][j] = act(bias[j] + sum_b 2^(Ew[j,b] + Ex[n,b]) * sum_{k in block b} w[j][k] x[n][k])
//
// tcgen05.mma kind::mxf8f6f4 multiplies E4M3 elements and their E8M0 scales as they lie in memory: nothing is unpacked.  It takes a scale for 32 elements; four products
// in a row are given the same one.  A word of scales has those of four k-blocks of 128, so it goes to tensor memory once for all four (tcgen05.cp, issued in
// front of the products by the same thread, runs in order with them) and the instruction's scale ids say which byte.
// The weights are the 128-row side of a tile, rows of the batch its columns (16 to 256): a batch of one costs no more products than one of sixteen, a lane of the epilogue has
// one output unit, and a tile's units are one block of the next layer's input.
// Groups of rows begin anywhere: a tile's codes come by boxes from any row on, and its scales by a warp that reads the words of its rows and lays them out as tcgen05.cp wants
// them.  What a box brings beyond a group's last row belongs to other columns and is not put out.
// The tensor core's additions, one for 32 products, cut off what does not fit: one after the other they lose bits always to the same side, 1.5 * 2^-24 of the sum each (measured; 256 of them, 8192 inputs
// of one sign, 1.9 * 10^-5 of the result; 32768, 2.6 * 10^-3).  So no more than CHAIN k-blocks follow one another: a chain's sums go to registers, where the chains are added up in fp32, rounded to
// nearest, while the next chain's products have another place in tensor memory.
// The grid has no more CTAs than the GPU has SMs; each walks the tiles of all groups, copies running ahead over a tile's end.  Where there are few tiles, up to eight CTAs of
// a cluster share one, each with its part of the k-blocks, and send one another their sums, which are added in rank order.
//
// What bounds it: one row x 8192 x 16384 24.3 us (5.6 TB/s; HBM at 6.6 TB/s between a launch's first and last block, and start and end of a launch), 64 rows in 32 groups x 4096 x 8192 140 us (6.6 TB/s),
// 1 x 8192 x 1024 6.2 us and 1 x 784 x 512 4.6 us (a launch, latency), 16384 x 8192 x 8192 785 us (2800 TFLOP/s, the tensor pipe and the sums that are taken out beside it; 920 us in a long run, under the power
// limit), 20011 rows in 12 groups x 4104 x 8001 650 us (2020 TFLOP/s, L2: rows 4112 bytes apart lie on two lines for every 128 bytes; 537 us for 4096 inputs).
//
// Every wait on an mbarrier is bounded.  A role whose wait gave up records a code in `status`, raises a flag that ends all other waits, and is not told of what follows; outputs are
// put out only of sums that are said to be complete.  Copies and products under way end, again waited for with a limit, before the memory that they write to is given back.
#include "spg_fp8.cuh"
#include "spg_gemm.cuh"
#include "spg_tc.cuh"
#include <cmath>
#include <cstdio>
#include <mutex>

namespace {

using namespace spgtc;
using namespace spgfp8;

constexpr uint32_t TM = 128;                  // output units of a tile
constexpr uint32_t KB = 128;                  // elements of a k-block: one block, four products
constexpr uint32_t W_BYTES = TM * KB;         // codes of a tile's weights
constexpr uint32_t SF_TILE = 512;             // words of scales of 128 rows
constexpr uint32_t SF_SLOTS = 4;              // words on their way, four k-blocks each
constexpr uint32_t ROLES = 3;                 // warp 0: copies, warp 1: products, warp 2: scales; the rest: outputs
constexpr uint32_t MAX_STAGES = 12;
constexpr uint32_t MAX_SPLIT = 8;
constexpr uint32_t AHEAD = 8;                 // k-blocks of weights asked for ahead (us with 0, 8 and 14: one row x 8192 x 16384 27.5, 26.1 and 26.4; one row through 2 of 16 experts with 4, 8, 16 and 32: 39.3, 39.2, 39.6 and 42.4)
constexpr uint32_t PART = 8 * TM * 4;         // a CTA's sums of eight rows
constexpr uint32_t MOST = 2 * 4 * 16;         // words of largest magnitudes that four warps leave to one another
constexpr uint32_t HEAD = 1024 + 4 * MOST * 4; // barriers and flags, and four times these
constexpr uint32_t DRAIN = 1u << 12;          // attempts of a last wait

struct LayerParams {
    uint32_t N, out, cols, experts;           // rows, units and inputs of a layer, layers
    uint32_t w_rows, kblocks, j_tiles, j_inverse, split, stages;
    const uint32_t *w_words, *x_words;        // scales
    const int32_t *starts;                    // of the groups, or NULL: one group
    const float *bias;
    int act;
    void *y; int type; uint32_t ldy;
    uint8_t *next_codes, *next_scales; uint32_t next_pitch;
    int32_t *status;
    int impatient;                            // (the check of the failure path: spgk_selftest_impatient)
};

__device__ __forceinline__ void st_cluster_if(uint32_t addr, float v, uint32_t yes)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.shared::cluster.f32 [%0], %1;\n\t}" ::"r"(addr), "f"(v), "r"(yes) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void cluster_arrive() { __syncwarp(); asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { __syncwarp(); asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// `id`: which of the CTA's barriers, for this many threads (whole warps, whose lanes come to it together)
__device__ __forceinline__ void some_meet(uint32_t id, uint32_t threads)
{
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool some_agree(uint32_t id, uint32_t threads, bool yes)
{
    uint32_t all;
    __syncwarp();
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbar.red.and.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"(id), "r"(threads), "r"((uint32_t)yes) : "memory");
    return all != 0;
}
// one look at a barrier's phase
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

// kind::mxf8f6f4, E4M3 on both sides, UE8M0 scales
__host__ __device__ constexpr uint32_t idesc_fp8(uint32_t m, uint32_t n) { return ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24); }

// (predicated: a k-block's products are one way without branches)
__device__ __forceinline__ void umma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate, uint32_t yes)
{
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(yes) : "memory");
}
__device__ __forceinline__ void umma_fp8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate, uint32_t yes)
{
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(yes) : "memory");
}
// 512 bytes (32 rows of 16) -> four columns of tensor memory, once for each quarter of the lanes; of a pair in both CTAs, each from its own shared memory to its own tensor memory
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) { asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory"); }
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc) { asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory"); }
// no swizzle, groups of eight rows of 16 bytes 128 bytes apart
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr)
{
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(128u >> 4) << 16 | (uint64_t)(128u >> 4) << 32 | (uint64_t)1u << 46;
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *v)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
          "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
          "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[8]) { tmem_ld8(taddr, v); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
          "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void prefetch_l2(const CUtensorMap *map, int c0, int c1)
{
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
}

// ---- groups of rows and their tiles -----------------------------------------------------------------------------------------------
// In shared memory: for each layer the first row of its group and how many tiles of rows the groups in front have; one entry more with the end of both.
struct Table { uint32_t *row, *first; };
__host__ __device__ constexpr uint32_t table_bytes(uint32_t experts) { return ((experts + 1) * 8 + 1023) / 1024 * 1024; }

__device__ __forceinline__ uint32_t start_of(const LayerParams &p, uint32_t e) { return min((uint32_t)max(__ldcg(p.starts + e), 0), p.N); }     // (past the SM's own cache: see below)
// by one warp
__device__ __forceinline__ void make_table(const LayerParams &p, const Table &tab, uint32_t tile_rows, uint32_t lane)
{
    if (!p.starts) {
        if (lane < 2) { tab.row[lane] = lane * p.N; tab.first[lane] = lane * ((p.N + tile_rows - 1) / tile_rows); }
        return;
    }
    uint32_t row = start_of(p, 0), tiles = 0;
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 256) {
        uint32_t end[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) { const uint32_t e = e0 + i * 32 + lane; end[i] = e < p.experts ? start_of(p, e + 1) : 0u; }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t e = e0 + i * 32 + lane;
            if (e0 + i * 32 >= p.experts) break;
            uint32_t hi = max(end[i], row);                                       // no group ends in front of an earlier one
#pragma unroll
            for (int o = 1; o < 32; o *= 2) { const uint32_t v = __shfl_up_sync(0xffffffffu, hi, o); if (lane >= (uint32_t)o) hi = max(hi, v); }
            uint32_t lo = __shfl_up_sync(0xffffffffu, hi, 1);
            if (lane == 0) lo = row;
            const uint32_t mine = (hi - lo + tile_rows - 1) / tile_rows;
            uint32_t upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) { const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= (uint32_t)o) upto += v; }
            if (e < p.experts) {
                tab.row[e] = lo; tab.first[e] = tiles + upto - mine;
                if (e + 1 == p.experts) { tab.row[e + 1] = hi; tab.first[e + 1] = tiles + upto; }
            }
            row = __shfl_sync(0xffffffffu, hi, 31);
            tiles += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
}
// Where there are starts the table is made in front of the wait for the launch in front, out of what then lies there, which is right where an earlier launch wrote them: it serves to
// fetch weights ahead.  Behind the wait they are looked at again, and the table is made anew if it shows that they are others: its ends of groups are then not
// the larger of the start and the end of the group before, one by one, which is how they come about.
__device__ __forceinline__ bool same_starts(const LayerParams &p, const Table &tab, uint32_t lane)
{
    uint32_t row = start_of(p, 0);
    bool same = tab.row[0] == row;
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 256) {
        uint32_t end[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) { const uint32_t e = e0 + i * 32 + lane; end[i] = e < p.experts ? start_of(p, e + 1) : 0u; }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t e = e0 + i * 32 + lane;
            if (e < p.experts) same = same && tab.row[e + 1] == max(end[i], tab.row[e]);
        }
    }
    return __all_sync(0xffffffffu, same);
}

// Tile t of all: its layer, its tile of units, its first row and how many rows of its group there are from there on (none: there is no such tile).  A group's tiles go in bands of so many
// tiles of units, the units fastest inside a band: what runs at a time shares weights and rows in L2.
// (A call, and few instructions for groups of one tile of rows: all roles look for their first tile when their own instructions are still on their way from L2.  Written out in each, a layer of one
// row's first copy left 0.9 us behind the wait for the launch in front, one of two groups' 1.7.)
struct Tile { uint32_t e, j, n0, rows; };
__device__ __noinline__ Tile find_tile(uint32_t t, const uint32_t *row, const uint32_t *first, uint32_t experts, uint32_t j_tiles, uint32_t j_inverse, uint32_t tile_rows, uint32_t band)
{
    uint32_t q = __umulhi(t, j_inverse), r = t - q * j_tiles;                    // t / j_tiles: j_inverse is 2^32 / j_tiles, rounded down, so q is at most one too small
    if (r >= j_tiles) { q++; r -= j_tiles; }
    if (q >= first[experts]) return { 0, 0, 0, 0 };
    uint32_t lo = 0, hi = experts;                                                // first[lo] <= q < first[hi]
    while (hi - lo > 1) { const uint32_t mid = (lo + hi) / 2; if (first[mid] <= q) lo = mid; else hi = mid; }
    const uint32_t at = first[lo], n_tiles = first[lo + 1] - at;
    uint32_t j = r, n = 0;
    if (n_tiles > 1) {
        r += (q - at) * j_tiles;
        const uint32_t one = band * n_tiles, g = r / one, left = r % one, here = min(band, j_tiles - g * band);
        j = g * band + left % here; n = left / here;
    }
    const uint32_t n0 = row[lo] + n * tile_rows;
    return { lo, j, n0, row[lo + 1] - n0 };
}

// ---- outputs ----------------------------------------------------------------------------------------------------------------------
// (predicated: a branch around each store costs more than the store)
__device__ __forceinline__ void put(float *y, float v, uint32_t yes)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.f32 [%0], %1;\n\t}" ::"l"(y), "f"(v), "r"(yes) : "memory");
}
__device__ __forceinline__ void put16(void *y, uint16_t v, uint32_t yes)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.u16 [%0], %1;\n\t}" ::"l"(y), "h"(v), "r"(yes) : "memory");
}
__device__ __forceinline__ void put(__half *y, float v, uint32_t yes) { put16(y, __half_as_ushort(__float2half_rn(v)), yes); }
__device__ __forceinline__ void put(__nv_bfloat16 *y, float v, uint32_t yes) { put16(y, __bfloat16_as_ushort(__float2bfloat16_rn(v)), yes); }

// what is chosen -- activation, type -- is chosen outside the loops over the rows: an epilogue's instructions come from L2 as it runs
template <int C, typename F> __device__ __forceinline__ void each(float (&v)[C], F f)
{
#pragma unroll
    for (int i = 0; i < C; i++) v[i] = f(v[i]);
}
template <int C> __device__ __forceinline__ void activate(float (&v)[C], int act)
{
    switch (act) {
        case SPG_ACT_RELU:    each(v, [](float x) { return spg_activate(x, SPG_ACT_RELU); }); break;
        case SPG_ACT_LEAKY:   each(v, [](float x) { return spg_activate(x, SPG_ACT_LEAKY); }); break;
        case SPG_ACT_SIGMOID: each(v, [](float x) { return spg_activate(x, SPG_ACT_SIGMOID); }); break;
        case SPG_ACT_TANH:    each(v, [](float x) { return spg_activate(x, SPG_ACT_TANH); }); break;
        case SPG_ACT_FOO52:   each(v, [](float x) { return spg_activate(x, SPG_ACT_FOO52); }); break;
        default: break;
    }
}
template <typename T, int C> __device__ __forceinline__ void put_rows(const LayerParams &p, const float (&v)[C], uint32_t n0, uint32_t rows, uint32_t j)
{
    T *y = reinterpret_cast<T *>(p.y) + (uint64_t)n0 * p.ldy + j;
#pragma unroll
    for (int i = 0; i < C; i++, y += p.ldy) put(y, v[i], (uint32_t)i < rows && j < p.out);
}

// The four warps that have the same rows of a tile, its 128 units between them: where they leave their largest magnitudes to one another, sixteen rows by turns in two places
struct Four {
    uint32_t *most;                           // [2][4][16]
    uint32_t id, quad, turn;                  // their barrier, this warp among them
};
// Eight or sixteen rows' values of this lane's unit, the four warps' 128 units being one block of the next layer's input: scales, codes, stores.
// Lane i makes row i's scale for all.  A lane's codes are bytes of words of four rows; two exchanges among four lanes turn each word into four units of one row.
template <int C> __device__ __forceinline__ void put_next(const LayerParams &p, const float *v, uint32_t n0, uint32_t rows, uint32_t j0, uint32_t lane, Four &four)
{
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < C; i++) {
        const uint32_t a = __reduce_max_sync(0xffffffffu, __float_as_uint(v[i]) & 0x7fffffffu);
        if (lane % C == (uint32_t)i) most = a;
    }
    uint32_t *place = four.most + four.turn * (MOST / 2);
    four.turn ^= 1u;
    if (lane < C) place[four.quad * 16u + lane] = most;
    some_meet(four.id, 128);
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) most = max(most, place[q * 16u + lane % C]);
    const uint32_t mine = scale_byte(most);                                      // row lane % C
    const float inv = inverse_scale(mine);
    const uint32_t j = j0 + lane / 4u * 4u, block = j0 / TM;
    const bool there = j < (p.out + 15u) / 16u * 16u;
#pragma unroll
    for (int h = 0; h < C; h += 4) {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = v[h + i] * __shfl_sync(0xffffffffu, inv, h + i);
        uint32_t w = encode4(q[0], q[1], q[2], q[3]);
        w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 2), lane & 2u ? 0x3276 : 0x5410);
        w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 1), lane & 1u ? 0x3715 : 0x6240);
        const uint32_t i = h + lane % 4u;                                        // this lane's row now
        if (__shfl_sync(0xffffffffu, mine, i) == 255u) w = 0;                    // a NaN block
        if (i < rows && there) *reinterpret_cast<uint32_t *>(p.next_codes + (uint64_t)(n0 + i) * p.next_pitch + j) = w;
    }
    if (four.quad == 0 && lane < C && lane < rows) p.next_scales[((uint64_t)(block / 4u) * p.N + n0 + lane) * 4u + block % 4u] = (uint8_t)mine;
}
// C rows' sums of this lane's unit to outputs (rows: how many of them there are; with none it only brings its instructions to the SM)
template <int C> __device__ __forceinline__ void finish(const LayerParams &p, float (&v)[C], uint32_t n0, uint32_t rows, uint32_t j0, uint32_t lane, float bias, Four &four)
{
    const uint32_t j = j0 + lane;
    each(v, [bias](float x) { return x + bias; });
    activate(v, p.act);
    if (p.y) {
        if (p.type == SPGK_T_F32) put_rows<float>(p, v, n0, rows, j);
        else if (p.type == SPGK_T_F16) put_rows<__half>(p, v, n0, rows, j);
        else put_rows<__nv_bfloat16>(p, v, n0, rows, j);
    }
    if (p.next_codes) {
        constexpr int AT_ONCE = C < 16 ? C : 16;
        each(v, [&](float x) { return j < p.out ? x : 0.0f; });
#pragma unroll
        for (int i = 0; i < C; i += AT_ONCE) put_next<AT_ONCE>(p, v + i, n0 + i, rows > (uint32_t)i ? rows - i : 0, j0, lane, four);
    }
}

// A chain's sums of a warp's rows from tensor memory, C at a time, `stride` columns from one C to the next, added to those of the chains before (rounded to nearest)
template <int COLS, int C> __device__ __forceinline__ void take(float (&v)[COLS], uint32_t from, uint32_t stride, uint32_t rows)
{
#pragma unroll
    for (int c = 0; c < COLS; c += C) {
        if (c / C * stride >= rows) break;
        float sums[C];
        tmem_ld(from + c / C * stride, sums);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < C; k++) v[c + k] += sums[k];
    }
}

// the last chain's sums of a warp's next rows and those of the chains before, which move up to leave
template <int C, int COLS> __device__ __forceinline__ void next_ones(float (&now)[C], float (&v)[COLS])
{
#pragma unroll
    for (int k = 0; k < C; k++) now[k] += v[k];
#pragma unroll
    for (int k = C; k < COLS; k++) v[k - C] = v[k];
}

// ---- scales -----------------------------------------------------------------------------------------------------------------------
// The words of a tile's rows for four k-blocks, R times 32 of them from row `first` on (zero from `rows` on): lane l has rows l, l + 32, ...
template <uint32_t R> __device__ __forceinline__ void load_words(uint32_t (&v)[R], const uint32_t *words, uint32_t group, uint32_t rows, uint32_t first, uint32_t lane)
{
    const uint32_t *at = words + (uint64_t)group * rows;
#pragma unroll
    for (uint32_t i = 0; i < R; i++) { const uint32_t r = first + i * 32u + lane; v[i] = r < rows ? at[r] : 0u; }
}
// to shared memory, 128 rows a tile of 512 bytes: row r's word is the r % 128 / 32'th of the 16 bytes r % 32
template <uint32_t R> __device__ __forceinline__ void store_words(uint32_t at, const uint32_t (&v)[R], uint32_t lane)
{
#pragma unroll
    for (uint32_t i = 0; i < R; i += 4)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at + i * (SF_TILE / 4) + lane * 16u), "r"(v[i]), "r"(i + 1 < R ? v[i + 1 < R ? i + 1 : i] : 0u),
                     "r"(i + 2 < R ? v[i + 2 < R ? i + 2 : i] : 0u), "r"(i + 3 < R ? v[i + 3 < R ? i + 3 : i] : 0u) : "memory");
}

// ---- single CTAs, and clusters that share a tile ------------------------------------------------------------------------------------
template <uint32_t NT> struct Shape {
    static constexpr uint32_t X_BYTES = NT * KB;
    static constexpr uint32_t STAGE = W_BYTES + X_BYTES;
    static constexpr uint32_t SFW = 2 * NT, SFX = 4, SF_COLS = 8;             // tensor memory: two sets of sums, two sets of scales
    static constexpr uint32_t USED = SFW + 2 * SF_COLS;
    static constexpr uint32_t COLS = USED <= 64 ? 64 : USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
    static constexpr uint32_t X_WORDS = (NT + 31) / 32;
    // k-blocks of a chain, whole words of scales.  Taking sums out costs the products beside it tensor memory's time, of few rows nothing that can be measured
    // (us with 4, 8 and one chain: 256 rows x 4096 x 4096 11.7, 11.4 and 11.1, 200 x 8192 x 8192 22.5, 22.2 and 21.8; 16 x 8192 x 8192 15.2 with any)
    static constexpr uint32_t CHAIN = NT >= 64 ? 8 : 4;
    static constexpr uint32_t EPI = NT >= 64 ? 16 : 8, THREADS = 32 * (ROLES + EPI), PARTS = EPI / 4;      // warps that put out, four of them all units of the same rows
    static constexpr uint32_t CHUNK = NT >= 128 ? 16 : 8;                     // columns that such a warp puts out at a time
    // Shared memory of a CTA; the rest of an SM's is its cache.  (us with 120, 180 and 212 KB: one row x 8192 x 16384 27.0, 26.0 and 26.1, 200 rows x 8192 x 8192 29.1, 22.9 and 21.9)
    static constexpr uint32_t ROOM = (NT >= 64 ? 212 : 180) * 1024;
};
constexpr uint32_t BAND = 16;

// Where CTAs share a tile, chunks of eight of its rows go to them by turns, and each sends its sums of a chunk to the CTA that has it
__host__ __device__ constexpr uint32_t chunks_of(uint32_t rows, uint32_t nt) { return ((rows < nt ? rows : nt) + 7) / 8; }
template <uint32_t NT> __host__ __device__ constexpr uint32_t parts_bytes(uint32_t rows, uint32_t split)
{
    return split > 1 ? (chunks_of(rows, NT) + split - 1) / split * split * PART : 0;
}

template <uint32_t NT>
__global__ void __launch_bounds__(Shape<NT>::THREADS, 1) spg_fp8_layer_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const LayerParams p)
{
    using L = Shape<NT>;
    constexpr uint32_t EPI = L::EPI, THREADS = L::THREADS;
    extern __shared__ uint8_t raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t head = smem_u32(base), table = head + HEAD, words = table + table_bytes(p.experts), parts = words + SF_SLOTS * 2 * SF_TILE, ring = parts + parts_bytes<NT>(p.N, p.split);
    const uint32_t full = head, empty = full + 8 * MAX_STAGES, sf_full = empty + 8 * MAX_STAGES, sf_empty = sf_full + 8 * SF_SLOTS, sums_full = sf_empty + 8 * SF_SLOTS, sums_free = sums_full + 16;
    const uint32_t ended = sums_free + 16, slot = ended + 8, aborted = slot + 4, late = aborted + 4, told = late + 4;
    // (aborted: a wait of this CTA gave up; late: one of the last waits did; told: one of the cluster's CTAs does not have its sums; behind them: the table was made anew; copies that were begun)
    volatile int *abort_flag = reinterpret_cast<volatile int *>(base + (aborted - head)), *told_flag = abort_flag + 2, *anew_flag = abort_flag + 3;
    volatile uint32_t *const begun_at = reinterpret_cast<volatile uint32_t *>(abort_flag + 4);
    uint32_t *const most = reinterpret_cast<uint32_t *>(base + 1024);
    const Table tab = { reinterpret_cast<uint32_t *>(base + HEAD), reinterpret_cast<uint32_t *>(base + HEAD) + p.experts + 1 };
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
    const uint32_t rank = blockIdx.x % p.split, team = blockIdx.x / p.split, teams = gridDim.x / p.split;
    const auto find = [&](uint32_t i) { return find_tile(i, tab.row, tab.first, p.experts, p.j_tiles, p.j_inverse, NT, BAND); };
    // this CTA's k-blocks
    const uint32_t lo = (uint32_t)((uint64_t)p.kblocks * rank / p.split), hi = (uint32_t)((uint64_t)p.kblocks * (rank + 1) / p.split);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.stages; s++) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (uint32_t s = 0; s < SF_SLOTS; s++) { mbar_init(sf_full + 8 * s, 1); mbar_init(sf_empty + 8 * s, 1); }
        for (uint32_t a = 0; a < 2; a++) { mbar_init(sums_full + 8 * a, 1); mbar_init(sums_free + 8 * a, EPI); }
        mbar_init(ended, 1);
        for (uint32_t i = 0; i < 4; i++) abort_flag[i] = 0;
        mbar_fence_init();
    }
    if (p.split > 1) cluster_arrive();                                           // (behind `told`, and in front of the wait for tensor memory: see below)
    if (warp == 1) tmem_alloc(slot, L::COLS);
    if (warp == 0 && elect_one()) { prefetch_map(&map_w); prefetch_map(&map_x); }
    if (warp == 2) make_table(p, tab, NT, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(base + (slot - head));
    spg_grid_trigger();
    // The first weights to L2 while the kernel in front still runs (whoever writes them: L2 is where writes meet)
    Tile tile = { 0, 0, 0, 0 };
    if (warp < ROLES) tile = find(team);
    if (warp == 0 && elect_one()) {
        if (tile.rows)
            for (uint32_t kb = lo; kb < hi && kb < lo + AHEAD; kb++) prefetch_l2(&map_w, (int)(kb * KB), (int)(tile.e * p.out + tile.j * TM));
    }
    __syncwarp();
    if (warp < ROLES) {
        spg_grid_wait();
        if (p.starts) {
            some_meet(5, 32 * ROLES);                                            // (all have found their first tile)
            if (warp == 2 && !same_starts(p, tab, lane)) {
                make_table(p, tab, NT, lane);
                *anew_flag = 1;
            }
            some_meet(1, THREADS);
            if (*anew_flag) tile = find(team);
        }
    }
    uint32_t t = team;
    if (warp == 0) {
        uint32_t begun = 0;
        if (elect_one()) {
            bool ok = true;
            for (uint32_t s = 0, phase = 1; ok && tile.rows; tile = find(t += teams)) {
                for (uint32_t kb = lo; kb < hi; kb++) {
                    if (!(ok = mbar_wait(empty + 8 * s, phase, abort_flag, p.status, 1))) break;
                    const uint32_t at = ring + s * L::STAGE;
                    mbar_expect_tx(full + 8 * s, L::STAGE);
                    tma_load_2d(at, &map_w, full + 8 * s, (int)(kb * KB), (int)(tile.e * p.out + tile.j * TM));
                    tma_load_2d(at + W_BYTES, &map_x, full + 8 * s, (int)(kb * KB), (int)tile.n0);
                    begun++;
                    if (++s == p.stages) { s = 0; phase ^= 1u; }
                }
            }
            *begun_at = begun;
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = idesc_fp8(TM, NT), last = tab.first[p.experts] * p.j_tiles;
            const uint64_t w0 = smem_desc_sw128(ring), x0 = smem_desc_sw128(ring + W_BYTES), words0 = scale_desc(words);
            uint32_t s = 0, phase = 0, q = 0, q_phase = 0, a = 0, a_phase = 1, odd = 0;
            bool ok = true;
            for (; ok && t < last; t += teams) {
                if (p.impatient == 1 && last - t <= teams && rank == 0) { atomicCAS(p.status, 0, 2); *abort_flag = 1; break; }
                // (Written out for the four blocks of a word: 260 cycles a k-block, 330 in a loop over them one by one; 27 of them are an instruction of products, 54 a wait, 6 a commit.)
                uint32_t first = lo;                                             // of the chain
                for (uint32_t kb = lo; ok && kb < hi;) {
                    if (kb == lo || kb % L::CHAIN == 0) {                        // a chain begins
                        ok = p.impatient != 2 ? mbar_wait(sums_free + 8 * a, a_phase, abort_flag, p.status, 6) : mbar_test(sums_free + 8 * a, a_phase);
                        if (!ok) { atomicCAS(p.status, 0, 6); *abort_flag = 1; break; }
                        first = kb;
                    }
                    if (!(ok = mbar_wait(sf_full + 8 * q, q_phase, abort_flag, p.status, 7))) break;
                    tc_fence_after();
                    odd ^= 1u;
                    const uint32_t sf = tmem + L::SFW + odd * L::SF_COLS, d = tmem + a * NT;
                    const uint64_t from = words0 + q * (2 * SF_TILE >> 4);
                    copy_scales(sf, from);
                    copy_scales(sf + L::SFX, from + (SF_TILE >> 4));
                    umma_commit(sf_empty + 8 * q);
                    if (++q == SF_SLOTS) { q = 0; q_phase ^= 1u; }
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) {
                        if (kb % 4u != i || kb >= hi) continue;
                        if (!(ok = mbar_wait(full + 8 * s, phase, abort_flag, p.status, 2))) break;
                        tc_fence_after();
                        const uint32_t left = p.cols - kb * KB, id = idesc | i << 4 | i << 29;
                        const uint64_t w = w0 + s * (L::STAGE >> 4), x = x0 + s * (L::STAGE >> 4);
                        umma_fp8(d, w, x, id, sf, sf + L::SFX, kb > first, 1);
                        umma_fp8(d, w + 2, x + 2, id, sf, sf + L::SFX, 1, left > 32);
                        umma_fp8(d, w + 4, x + 4, id, sf, sf + L::SFX, 1, left > 64);
                        umma_fp8(d, w + 6, x + 6, id, sf, sf + L::SFX, 1, left > 96);
                        umma_commit(empty + 8 * s);
                        if (++s == p.stages) { s = 0; phase ^= 1u; }
                        kb++;
                    }
                    if (!ok) break;
                    if (kb < hi && kb % L::CHAIN) continue;
                    umma_commit(sums_full + 8 * a);
                    if (++a == 2) { a = 0; a_phase ^= 1u; }
                }
            }
        }
        __syncwarp();
        if (p.split > 1) {
            // Given back before this CTA waits for the others: one that has none on its SM, and so cannot finish, may hold up a cluster that holds some elsewhere
            if (team < tab.first[p.experts] * p.j_tiles) some_meet(2, 32 * (EPI + 1));
            if (__any_sync(0xffffffffu, *abort_flag)) {
                if (elect_one()) umma_commit(ended);
                __syncwarp();
                mbar_wait_uniform(ended, 0, late, p.status, 5, DRAIN);
            }
            tc_fence_after();
            tmem_free(tmem, L::COLS);
        }
    } else if (warp == 2) {
        uint32_t q = 0, phase = 1, w[4], x[L::X_WORDS], g = lo / 4u;
        const uint32_t g_end = (hi + 3u) / 4u;
        bool more = tile.rows;
        const auto load = [&]() {
            load_words(w, p.w_words, g, p.w_rows, tile.e * p.out + tile.j * TM, lane);
            load_words(x, p.x_words, g, p.N, tile.n0, lane);
        };
        if (more) load();
        while (more) {
            uint32_t w0[4], x0[L::X_WORDS];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) w0[i] = w[i];
#pragma unroll
            for (uint32_t i = 0; i < L::X_WORDS; i++) x0[i] = x[i];
            if (++g == g_end) { g = lo / 4u; t += teams; tile = find(t); more = tile.rows; }
            if (more) load();                                                    // (on their way while these wait for their place)
            mbar_wait_uniform(sf_empty + 8 * q, phase, aborted, p.status, 8);
            if (__any_sync(0xffffffffu, *abort_flag)) break;
            store_words(words + q * 2 * SF_TILE, w0, lane);
            store_words(words + q * 2 * SF_TILE + SF_TILE, x0, lane);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(sf_full + 8 * q);
            if (++q == SF_SLOTS) { q = 0; phase ^= 1u; }
        }
    } else {
        const uint32_t quad = warp % 4u, part = (warp - ROLES) / 4u;
        Four four = { most + part * MOST, 6u + part, quad, 0u };
        constexpr uint32_t COLS = NT / L::PARTS;                               // of a tile's rows this warp's, so many at a time by turns
        const uint32_t chains = (hi - 1u) / L::CHAIN - lo / L::CHAIN + 1u;
        uint32_t a = 0, a_phase = 0;
        // Once without a row before the launch in front has ended: the outputs' instructions come from L2, and would follow the products
#pragma unroll 1
        for (uint32_t dry = 1;; dry = 0) {
            if (!dry) {
                if (!(tile = find(t)).rows) break;
            } else tile = { 0, 0, 0, 0 };
            const uint32_t j0 = tile.j * TM + quad * 32u, j = j0 + lane, rows = min(tile.rows, NT), mine = rows > part * L::CHUNK ? rows - part * L::CHUNK : 0u;
            float bias = 0.0f, v[COLS];
            bool ok = true;
            if (!dry && p.bias && j < p.out) bias = p.bias[(uint64_t)tile.e * p.out + j];
            each(v, [](float) { return 0.0f; });
            const auto lanes = [&]() { return tmem + a * NT + part * L::CHUNK + (quad * 32u << 16); };
            const auto taken = [&]() {                                           // of this warp's rows
                tc_fence_before();
                __syncwarp();
                if (!dry && lane == 0) mbar_arrive(sums_free + 8 * a);
                if (!dry && ++a == 2) { a = 0; a_phase ^= 1u; }
            };
#pragma unroll 1
            for (uint32_t i = 1; i < (dry ? 2u : chains); i++) {                 // (the last chain's are added as they are put out)
                if (!dry && !(ok = __all_sync(0xffffffffu, mbar_wait(sums_full + 8 * a, a_phase, abort_flag, p.status, 3)))) break;
                tc_fence_after();
                take<COLS, L::CHUNK>(v, lanes(), L::PARTS * L::CHUNK, mine);
                taken();
            }
            if (!dry) {
                // (all four warps of a row go one way)
                ok = some_agree(6u + part, 128, ok && mbar_wait(sums_full + 8 * a, a_phase, abort_flag, p.status, 3));
                tc_fence_after();
                if (p.split > 1) {
                    // This CTA's sums to those that put them out, [chunk][CTA][row][unit], sent before one barrier
                    cluster_wait();                                              // all have begun
                    const uint32_t left = ok ? mine : 0u;
#pragma unroll 1
                    for (uint32_t g = 0; g < COLS; g += 8) {
                        const uint32_t at = g / L::CHUNK * L::PARTS * L::CHUNK + g % L::CHUNK, c = (part * L::CHUNK + at) / 8u;
                        if (at >= left) break;
                        float now[8];
                        tmem_ld8(lanes() + at, now);
                        tmem_ld_wait();
                        next_ones(now, v);
                        const uint32_t to = mapa(parts + (c / p.split * p.split + rank) * PART + (quad * 32u + lane) * 4u, c % p.split);
#pragma unroll
                        for (uint32_t i = 0; i < 8; i++) st_cluster_if(to + i * TM * 4u, now[i], at + i < left);
                    }
                    if (!ok && lane < p.split) st_cluster_u32(mapa(told, lane), 1);
                    tc_fence_before();
                    __syncwarp();
                    some_meet(2, 32 * (EPI + 1));
                    cluster_arrive();
                    cluster_wait();
                    ok = !__any_sync(0xffffffffu, *told_flag);
                }
            }
            if (p.split == 1 || dry) {
#pragma unroll 1
                for (uint32_t c = 0; c < (dry ? 1u : ok ? mine : 0u); c += L::PARTS * L::CHUNK) {
                    float now[L::CHUNK];
                    each(now, [](float) { return 0.0f; });
                    if (!dry) { tmem_ld(lanes() + c, now); tmem_ld_wait(); }
                    next_ones(now, v);
                    finish(p, now, tile.n0 + part * L::CHUNK + c, dry ? 0u : mine - c, j0, lane, bias, four);
                }
            } else if (ok) {
#pragma unroll 1
                for (uint32_t c = (part * p.split + rank) * 8u; c < rows; c += p.split * L::PARTS * 8u) {
                    float all[8];
                    const float *sums = reinterpret_cast<const float *>(base + (parts - head)) + (c / 8 / p.split * p.split) * (PART / 4) + quad * 32u + lane;
                    each(all, [](float) { return 0.0f; });
#pragma unroll 1
                    for (uint32_t r = 0; r < p.split; r++, sums += PART / 4) {   // in rank order
#pragma unroll
                        for (int i = 0; i < 8; i++) all[i] += sums[i * TM];
                    }
                    finish(p, all, tile.n0 + c, rows - c, j0, lane, bias, four);
                }
            }
            if (dry) {
                spg_grid_wait();
                if (p.starts) some_meet(1, THREADS);
                continue;
            }
            if (!ok) break;
            taken();
            t += teams;
        }
    }
    if (p.split > 1) {
        // (a cluster without a tile has been through none of its barriers, one with a tile, whose outputs' warps have been through both, only by these)
        const bool none = team >= tab.first[p.experts] * p.j_tiles;
        if (warp < ROLES || none) { cluster_wait(); cluster_arrive(); cluster_wait(); }
    }
    __syncwarp();
    __syncthreads();
    if (*abort_flag) {
        // what is under way ends first: the products, which `ended` is told of, and the last copies, each of which has its barrier
        if (warp == 1 && p.split == 1) {
            if (elect_one()) umma_commit(ended);
            __syncwarp();
            mbar_wait_uniform(ended, 0, late, p.status, 5, DRAIN);
        }
        if (warp == 0) {
            const uint32_t begun = *begun_at;
            for (uint32_t i = begun > p.stages ? begun - p.stages : 0; i < begun; i++) mbar_wait_uniform(full + 8 * (i % p.stages), i / p.stages & 1u, late, p.status, 4, DRAIN);
        }
        __syncwarp();
        __syncthreads();
    }
    if (warp == 1 && p.split == 1) { tc_fence_after(); tmem_free(tmem, L::COLS); }
}

// ---- pairs of CTAs, many rows -------------------------------------------------------------------------------------------------
// (bands of tiles of units, us of 16384 x 8192 x 8192 in a long run: 4 954, 8 918, 12 903, 16 899, 24 934, 32 1018: wider ones share fewer of the rows' tiles, narrower ones fewer of the weights')
// 256 units x up to 256 rows of a group a tile on a cluster of two (cta_group::2): each CTA holds 128 units' weights and half of the rows, so a k-block costs it 32 KB
// for 512 cycles of products; a CTA alone would need 48. The last tile of a group multiplies no more rows than it has (in steps of 32).
// Chains of products have 16 k-blocks (us of 16384 x 8192 x 8192 with 8, 16 and one chain 877, 807 and 770, of 8192 rows in 8 groups x 4096 x 8192 246, 224 and 219), a tile's first one 24: the tile before is
// put out beside it (8192 rows as above to 8-bit outputs with a first chain of 16, 24 and 32: 250, 236 and 230, one chain 230).  Sixteen epilogue warps take 64 columns
// a thread to registers.  Tensor memory has no room for two chains of 256 columns beside the scales: they begin at its first column and at column 224 in turn, and have 32 columns in common, which one warp in four
// has.  It takes these first and says so; the next chain's products wait for no more (for all 64 columns of all warps: 12 % of the time; two halves of 128 columns a product, in places of their own, read the weights
// twice: 9 %; tiles of 224 rows, which have none in common, are 2 % quicker where there are many, and 30 % slower for 512 and 1024 rows).
constexpr uint32_t PN = 256;                                   // rows of the batch a tile
constexpr uint32_t P_EPI = 16, P_THREADS = 32 * (ROLES + P_EPI);
constexpr uint32_t P_COLS = PN / (P_EPI / 4);                   // columns of an epilogue warp
constexpr uint32_t P_FIRST = 24, P_CHAIN = 16;
constexpr uint32_t P_STAGE = W_BYTES + PN / 2 * KB;
constexpr uint32_t P_STAGES = 6;
constexpr uint32_t P_WORDS = 3 * SF_TILE;                       // of 128 units and 256 rows
constexpr uint32_t P_SHIFT = 224;                               // columns of tensor memory: chains begin at the first and at this one in turn
constexpr uint32_t P_SF = P_SHIFT + PN, P_SFX = 4, P_SF_COLS = 16;   // scales behind them, twice; those of the rows behind the weights'
constexpr uint32_t P_BAND = 12;
__device__ __forceinline__ bool begins_chain(uint32_t kb) { return kb >= P_FIRST && (kb - P_FIRST) % P_CHAIN == 0; }     // (besides a tile's first)
__host__ __device__ constexpr uint32_t pair_smem(uint32_t experts) { return 1024 + HEAD + table_bytes(experts) + SF_SLOTS * P_WORDS + P_STAGES * P_STAGE; }

// half of a warp's sums of a chain: the first chain's as they are, those behind added to them
__device__ __forceinline__ void take_half(float (&v)[32], uint32_t from, uint32_t rows, bool add)
{
    if (add) take<32, 16>(v, from, 16, rows);
    else { tmem_ld32(from, v); tmem_ld_wait(); }
}

__global__ void __launch_bounds__(P_THREADS, 1) spg_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const LayerParams p)
{
    extern __shared__ uint8_t raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t head = smem_u32(base), table = head + HEAD, words = table + table_bytes(p.experts), ring = words + SF_SLOTS * P_WORDS;
    const uint32_t full = head, empty = full + 8 * P_STAGES, sf_full = empty + 8 * P_STAGES, sf_empty = sf_full + 8 * SF_SLOTS, sums_full = sf_empty + 8 * SF_SLOTS, sums_free = sums_full + 16;
    const uint32_t ended = sums_free + 16, slot = ended + 8, aborted = slot + 4, late = aborted + 4, told = late + 4;
    // (told: of each of the two CTAs, how many k-blocks' copies it began, and then whether a wait gave up in it)
    volatile int *abort_flag = reinterpret_cast<volatile int *>(base + (aborted - head));
    volatile uint32_t *told_at = reinterpret_cast<volatile uint32_t *>(base + (told - head));
    uint32_t *const most = reinterpret_cast<uint32_t *>(base + 1024);
    const Table tab = { reinterpret_cast<uint32_t *>(base + HEAD), reinterpret_cast<uint32_t *>(base + HEAD) + p.experts + 1 };
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, rank = cluster_rank(), pairs = gridDim.x / 2u;
    const auto find = [&](uint32_t i) { return find_tile(i, tab.row, tab.first, p.experts, p.j_tiles, p.j_inverse, PN, P_BAND); };

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < P_STAGES; s++) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (uint32_t s = 0; s < SF_SLOTS; s++) { mbar_init(sf_full + 8 * s, 2); mbar_init(sf_empty + 8 * s, 1); }
        for (uint32_t a = 0; a < 2; a++) { mbar_init(sums_full + 8 * a, 1); mbar_init(sums_free + 8 * a, 2 * P_EPI); }
        mbar_init(ended, 1);
        for (uint32_t i = 0; i < 6; i++) abort_flag[i] = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc_pair(slot, 512);
    if (warp == 0 && elect_one()) { prefetch_map(&map_w); prefetch_map(&map_x); }
    if (warp == 2 && !p.starts) make_table(p, tab, PN, lane);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(base + (slot - head));
    spg_grid_trigger();
    if (warp < ROLES) {
        spg_grid_wait();
        if (p.starts) {
            if (warp == 2) make_table(p, tab, PN, lane);
            some_meet(1, P_THREADS);
        }
    }
    // columns of a tile with so many rows left in its group: each CTA has half of them, in whole eights
    const auto columns = [](uint32_t rows) { return rows >= PN ? PN : (rows + 31u) / 32u * 32u; };
    // a wait gave up: the other CTA's waits end as well
    const auto give_up = [&](int code) {
        atomicCAS(p.status, 0, code);
        for (uint32_t r = 0; r < 2; r++) st_cluster_u32(mapa(aborted, r), 1);
    };
    Tile tile;
    uint32_t t = blockIdx.x / 2u;
    if (warp == 0) {
        if (elect_one()) {
            const uint32_t leader = mapa(full, 0);
            uint32_t begun = 0;
            bool ok = true;
            for (uint32_t s = 0, phase = 1; ok && (tile = find(t)).rows; t += pairs) {
                const int row_w = (int)(tile.e * p.out + tile.j * 256u + rank * TM), row_x = (int)(tile.n0 + rank * columns(tile.rows) / 2u);
                for (uint32_t kb = 0; kb < p.kblocks; kb++) {
                    if (!(ok = mbar_wait(empty + 8 * s, phase, abort_flag, p.status, 1))) break;
                    const uint32_t at = ring + s * P_STAGE;
                    if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * P_STAGE);
                    tma_load_2d_pair(at, &map_w, leader + 8 * s, (int)(kb * KB), row_w);
                    tma_load_2d_pair(at + W_BYTES, &map_x, leader + 8 * s, (int)(kb * KB), row_x);
                    begun++;
                    if (++s == P_STAGES) { s = 0; phase ^= 1u; }
                }
            }
            for (uint32_t r = 0; r < 2; r++) st_cluster_u32(mapa(told + 8 * rank, r), begun);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            uint32_t s = 0, phase = 0, q = 0, q_phase = 0, a = 1, a_phase = 1, odd = 0, d = tmem + P_SHIFT;
            const uint32_t last = tab.first[p.experts] * p.j_tiles;
            bool ok = true;
            for (; ok && (tile = find(t)).rows; t += pairs) {
                if (p.impatient == 1 && last - t <= pairs) { give_up(2); break; }
                const uint32_t idesc = idesc_fp8(256, columns(tile.rows));
                for (uint32_t kb = 0; kb < p.kblocks; kb++) {
                    const bool begins = kb == 0 || begins_chain(kb);
                    if (begins) {
                        ok = p.impatient != 2 ? mbar_wait(sums_free + 8 * a, a_phase, abort_flag, p.status, 6) : mbar_test(sums_free + 8 * a, a_phase);
                        if (!ok) { give_up(6); break; }
                        tc_fence_after();
                        a_phase ^= a;
                        a ^= 1u;
                        d = tmem + P_SHIFT - (d - tmem);
                    }
                    if (kb % 4u == 0) {
                        if (!(ok = mbar_wait(sf_full + 8 * q, q_phase, abort_flag, p.status, 7))) break;
                        tc_fence_after();
                        const uint32_t to = tmem + P_SF + (odd ^= 1u) * P_SF_COLS;
                        const uint64_t from = scale_desc(words + q * P_WORDS);
                        copy_scales_pair(to, from);
                        copy_scales_pair(to + P_SFX, from + (SF_TILE >> 4));
                        copy_scales_pair(to + P_SFX + 4, from + (2 * SF_TILE >> 4));
                        umma_commit_pair(sf_empty + 8 * q);
                        if (++q == SF_SLOTS) { q = 0; q_phase ^= 1u; }
                    }
                    if (!(ok = mbar_wait(full + 8 * s, phase, abort_flag, p.status, 2))) break;
                    tc_fence_after();
                    const uint32_t at = ring + s * P_STAGE, sf = tmem + P_SF + odd * P_SF_COLS, left = p.cols - kb * KB, id = idesc | (kb % 4u) << 4 | (kb % 4u) << 29;
                    const uint64_t w = smem_desc_sw128(at), x = smem_desc_sw128(at + W_BYTES);
                    umma_fp8_pair(d, w, x, id, sf, sf + P_SFX, !begins, 1);
                    umma_fp8_pair(d, w + 2, x + 2, id, sf, sf + P_SFX, 1, left > 32);
                    umma_fp8_pair(d, w + 4, x + 4, id, sf, sf + P_SFX, 1, left > 64);
                    umma_fp8_pair(d, w + 6, x + 6, id, sf, sf + P_SFX, 1, left > 96);
                    umma_commit_pair(empty + 8 * s);
                    if (++s == P_STAGES) { s = 0; phase ^= 1u; }
                    if (kb + 1 == p.kblocks || begins_chain(kb + 1)) umma_commit_pair(sums_full + 8 * a);
                }
                if (!ok) { give_up(2); break; }
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        const uint32_t leader = mapa(sf_full, 0), groups = (p.kblocks + 3u) / 4u;
        uint32_t q = 0, phase = 1, w[4], x[8], g = 0;
        tile = find(t);
        bool more = tile.rows;
        const auto load = [&]() {
            load_words(w, p.w_words, g, p.w_rows, tile.e * p.out + tile.j * 256u + rank * TM, lane);
            load_words(x, p.x_words, g, p.N, tile.n0, lane);
        };
        if (more) load();
        while (more) {
            uint32_t w0[4], x0[8];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) w0[i] = w[i];
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) x0[i] = x[i];
            if (++g == groups) { g = 0; t += pairs; tile = find(t); more = tile.rows; }
            if (more) load();                                                    // (on their way while these wait for their place)
            mbar_wait_uniform_cluster(sf_empty + 8 * q, phase, aborted, p.status, 8);
            if (__any_sync(0xffffffffu, *abort_flag)) break;
            store_words(words + q * P_WORDS, w0, lane);
            store_words(words + q * P_WORDS + SF_TILE, x0, lane);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(leader + 8 * q);
            if (++q == SF_SLOTS) { q = 0; phase ^= 1u; }
        }
    } else {
        const uint32_t quad = warp % 4u, part = (warp - ROLES) / 4u, free_at = mapa(sums_free, 0);
        Four four = { most + part * MOST, 2u + part, quad, 0u };
        const uint32_t chains = p.kblocks <= P_FIRST ? 1u : 1u + (p.kblocks - P_FIRST + P_CHAIN - 1) / P_CHAIN, first = part * P_COLS;     // this warp's columns
        // Of each chain all warps say once that the next one may begin, which takes the place of the chain before and of the columns in common: where this warp has none of these, when the chain before is in its
        // registers, else when they are too, the first of its columns where the chain begins at P_SHIFT, the last where it begins at the first column.  (A word for one chain may come before all have given
        // theirs for the chain in front: a barrier for each of two in turn.  So for sums that are whole.)
        const auto in_common = [&](uint32_t shifted) { return part == (shifted ? 0u : P_EPI / 4 - 1); };
        uint32_t turn = 0, phase = 0;
        if (lane == 0 && !in_common(0)) mbar_arrive_cluster(free_at);
        spg_grid_wait();
        if (p.starts) some_meet(1, P_THREADS);
        for (; (tile = find(t)).rows; t += pairs) {
            const uint32_t j0 = tile.j * 256u + rank * TM + quad * 32u, j = j0 + lane, n0 = tile.n0 + first;
            const uint32_t rows = tile.rows > first ? min(tile.rows - first, P_COLS) : 0u;             // this warp's
            float bias = 0.0f, v[P_COLS], (&v_0)[32] = *reinterpret_cast<float (*)[32]>(v), (&v_1)[32] = *reinterpret_cast<float (*)[32]>(v + 32);
            if (p.bias && j < p.out) bias = p.bias[(uint64_t)tile.e * p.out + j];
            bool ok = true;
#pragma unroll 1
            for (uint32_t i = 0; i < chains; i++) {
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(sums_full + 8 * turn, phase, abort_flag, p.status, 3)))) break;
                tc_fence_after();
                const bool now = in_common(turn), next = in_common(turn ^ 1u), high = now && !turn;
                const uint32_t from = tmem + first + turn * P_SHIFT + (quad * 32u << 16);
#pragma unroll 1
                for (uint32_t h = 0; h < 2; h++) {
                    if (h == high) take_half(v_0, from, rows, i > 0); else take_half(v_1, from + 32, rows > 32u ? rows - 32u : 0u, i > 0);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0 && (h ? !next : now)) mbar_arrive_cluster(free_at + 8 * (h ^ turn));
                }
                phase ^= turn;
                turn ^= 1u;
            }
            // (all four warps of a row go one way)
            if (!some_agree(2u + part, 128, ok)) break;
            if (rows && j0 - quad * 32u < p.out) finish(p, v, n0, rows, j0, lane, bias, four);       // (the same in the four warps: some of this CTA's units there are)
        }
    }
    __syncwarp();
    __syncthreads();
    if (threadIdx.x == 0)
        for (uint32_t r = 0; r < 2; r++) st_cluster_u32(mapa(told + 8 * rank + 4, r), (uint32_t)*abort_flag);
    cluster_sync();
    if (told_at[1] | told_at[3]) {
        // Products and copies under way end first.  Each k-block's copies are counted for both CTAs at once, by the first one's barrier: where one of them began fewer, as many bytes
        // are fetched here once more, or expected of the other alone.
        if (rank == 0 && warp == 1) {
            if (elect_one()) umma_commit_pair(ended);
            __syncwarp();
            mbar_wait_uniform(ended, 0, late, p.status, 5, DRAIN);
        }
        if (rank == 0 && warp == 0) {
            const uint32_t mine = told_at[0], other = told_at[2], end = max(mine, other);
            for (uint32_t i = min(mine, other); i < end; i++) {
                const uint32_t s = i % P_STAGES, bar = full + 8 * s, at = ring + s * P_STAGE;
                if (elect_one()) {
                    if (i >= mine) mbar_expect_tx(bar, P_STAGE);                 // (the other's)
                    else {
                        tma_load_2d_pair(at, &map_w, mapa(bar, 0), 0, 0);
                        tma_load_2d_pair(at + W_BYTES, &map_x, mapa(bar, 0), 0, 0);
                    }
                }
                __syncwarp();
            }
            for (uint32_t i = end > P_STAGES ? end - P_STAGES : 0; i < end; i++) mbar_wait_uniform_cluster(full + 8 * (i % P_STAGES), i / P_STAGES & 1u, late, p.status, 4, DRAIN);
        }
        __syncwarp();
        __syncthreads();
        cluster_sync();
    }
    if (warp == 1) { tc_fence_after(); tmem_free_pair(tmem, 512); }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn()
{
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(f);
    });
    return fn;
}

// boxes of a k-block x box_rows rows of a matrix' codes; what lies behind its columns and rows is zero
int codes_map(CUtensorMap *map, const spgk_fp8 *m, uint32_t box_rows)
{
    EncodeTiledFn fn = encode_fn();
    if (!fn) { spgk_set_error("cuTensorMapEncodeTiled", "driver entry point not available"); return SPGK_E_CUDA; }
    const cuuint64_t dims[2] = { m->cols, m->rows }, strides[1] = { m->pitch };
    const cuuint32_t box[2] = { KB, box_rows }, steps[2] = { 1, 1 };
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, m->codes, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        char msg[64];
        snprintf(msg, sizeof msg, "CUresult %d", (int)r);
        spgk_set_error("cuTensorMapEncodeTiled (8-bit operand)", msg);
        return SPGK_E_CUDA;
    }
    return SPGK_OK;
}

// 2^32 / n, rounded down (of 1: the largest there is)
uint32_t inverse(uint32_t n) { return n == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / n); }

// the most tiles of `tile_rows` rows that p.N rows in any groups make: one for each layer that has some, and one more for every tile_rows of the rest
uint64_t most_tiles(const LayerParams &p, uint32_t tile_rows)
{
    const uint32_t some = p.experts < p.N ? p.experts : p.N;
    return (some + (uint64_t)(p.N - some) / tile_rows) * p.j_tiles;
}
// clusters of this many CTAs that find room at a time, one CTA an SM
uint32_t at_a_time(uint32_t split, uint32_t sms) { return (split == 8 ? 15u : split == 4 ? 33u : split == 2 ? 74u : 148u) * sms / 148u; }

// How a call is arranged: rows of a tile (256: pairs of CTAs), CTAs that share one.  What each takes is estimated in us on a B200 (with groups of equal sizes, for want of the real ones), fitted to 1285
// arrangements of 205 products: 1 to 5000 rows, in up to 200 groups, 128 to 16384 inputs, 128 to 8192 units, when sums were not yet taken out in chains.  Of 613 products of all such sizes, measured since in 4005
// arrangements, what it picks takes 2.5 % longer on average than the best, 14 % in one of twenty, and 47 % at most (2000 x 128 x 4096 by 64 rows 16.9 us, in pairs 11.5: the outputs of few inputs are what it
// knows least of).  Both ends of it, us: 64 rows x 8192 x 8192 by tiles of 64 rows, two CTAs each, 16.4, by tiles of 16 27.0, in pairs 23.4; 1 x 1024 x 8192 alone 4.9, two CTAs a tile 6.3;
// 1 x 8192 x 1024 13.9 and, eight a tile, 6.3; 512 x 8192 x 8192 in pairs 33.0, by 128 rows 38.1; 512 x 784 x 512 by 32 rows 5.5, in pairs 9.1.
// All that holds for groups of similar sizes.  Where they are not, tiles are made for the mean: of 512 rows x 64 x (4096 x 2048) all in one group take 28.0 us, where one layer for them takes 11.2 by its own
// arrangement, of 4096 rows 37.5 and 30.1 (in even groups, whose weights are all read, 82.8 and 98.1).
struct Plan { uint32_t rows, split; float us; };
float tiles_of(const LayerParams &p, uint32_t rows)
{
    const uint32_t groups = p.experts < p.N ? p.experts : p.N;
    if (groups == 1) return (float)(p.N / rows + (p.N % rows != 0));
    const float each = (float)p.N / (float)groups / (float)rows + 0.5f;          // (half of a last tile is empty)
    return (float)groups * (each > 1.0f ? each : 1.0f);
}
float whole(float v) { const float w = ceilf(v - 0.02f); return w > 1.0f ? w : 1.0f; }
Plan plan_of(const LayerParams &p, uint32_t sms)
{
    const float k = (float)p.kblocks, j_pairs = (float)((p.out + 255u) / 256u), j_tiles = (float)((p.out + TM - 1) / TM), each = (float)p.N / (float)(p.experts < p.N ? p.experts : p.N);
    Plan best = { PN, 1, 5.77f + whole(tiles_of(p, PN) * j_pairs / (float)(sms / 2)) * (k * 0.334f + 1.79f) };
    for (uint32_t rows = 16; rows <= 128; rows *= 2) {
        LayerParams q = p;
        q.j_tiles = (p.out + TM - 1) / TM;
        const uint64_t bound = most_tiles(q, rows);
        const float tiles = tiles_of(p, rows) * j_tiles, used = each < (float)rows ? each : (float)rows, outputs = 0.33f + used * 0.0092f;
        for (uint32_t s = 1; s <= MAX_SPLIT && s <= p.kblocks; s *= 2) {
            if (s > 1 && bound > at_a_time(s, sms)) break;
            const float at_work = tiles * (float)s < (float)sms ? tiles * (float)s : (float)sms, alone = 0.119f + (float)rows * 0.00068f, drawn = (float)(TM + rows) * at_work * 9.08e-6f;
            const float products = ceilf(k / (float)s) * (alone > drawn ? alone : drawn);
            float us = 3.22f + outputs;
            if (s == 1) us += whole(tiles / (float)sms) * (products > 0.9f * outputs ? products : 0.9f * outputs);
            else us += products + 0.40f + 0.116f * (float)s + 0.0108f * used + (tiles * (float)s > (float)sms / 2.0f ? 0.99f : 0.0f);
            if (us < best.us) best = { rows, s, us };
        }
    }
    return best;
}

int launch_as(const char *name, void (*kernel)(CUtensorMap, CUtensorMap, LayerParams), uint32_t grid, uint32_t threads, uint32_t smem, uint32_t cluster, const CUtensorMap &map_w, const CUtensorMap &map_x,
              const LayerParams &p, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    SPGK_CUDA(cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, p));
    return spgk_check_launch(name);
}

template <uint32_t NT> int launch(const spgk_fp8 *W, const spgk_fp8 *X, LayerParams p, uint32_t split, const SpgDeviceProps &dp, int dev, cudaStream_t stream)
{
    using L = Shape<NT>;
    static SpgOncePerDevice once;
    int rc = once.run(dev, [&]() -> int {
        SPGK_CUDA(cudaFuncSetAttribute(spg_fp8_layer_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dp.smem_optin));
        return SPGK_OK;
    });
    if (rc) return rc;
    CUtensorMap map_w, map_x;
    if ((rc = codes_map(&map_w, W, TM)) || (rc = codes_map(&map_x, X, NT))) return rc;
    const uint32_t sms = (uint32_t)dp.sm_count;
    const uint64_t tiles = most_tiles(p, NT);
    p.split = split;
    const uint32_t fixed = 1024 + HEAD + table_bytes(p.experts) + SF_SLOTS * 2 * SF_TILE + parts_bytes<NT>(p.N, p.split);
    const uint32_t most = (L::ROOM - fixed) / L::STAGE;
    p.stages = most < MAX_STAGES ? most : MAX_STAGES;
    const uint32_t grid = p.split > 1 ? (uint32_t)tiles * p.split : (tiles < sms ? (uint32_t)tiles : sms);
    return launch_as("spg_fp8_layer_kernel", spg_fp8_layer_kernel<NT>, grid, L::THREADS, fixed + p.stages * L::STAGE, p.split, map_w, map_x, p, stream);
}

int launch_pairs(const spgk_fp8 *W, const spgk_fp8 *X, LayerParams p, const SpgDeviceProps &dp, int dev, cudaStream_t stream)
{
    static SpgOncePerDevice once;
    int rc = once.run(dev, [&]() -> int {
        SPGK_CUDA(cudaFuncSetAttribute(spg_fp8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pair_smem(SPGK_MAX_EXPERTS)));
        return SPGK_OK;
    });
    if (rc) return rc;
    CUtensorMap map_w, map_x;
    if ((rc = codes_map(&map_w, W, TM)) || (rc = codes_map(&map_x, X, PN / 2))) return rc;
    const uint64_t tiles = most_tiles(p, PN);
    const uint32_t room = (uint32_t)dp.sm_count / 2, pairs = tiles < room ? (uint32_t)tiles : room;
    return launch_as("spg_fp8_pair_kernel", spg_fp8_pair_kernel, pairs * 2, P_THREADS, pair_smem(p.experts), 2, map_w, map_x, p, stream);
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
    SpgDeviceProps dp;
    int dev = 0;
    if ((rc = spg_device_props(&dp))) return rc;
    SPGK_CUDA(cudaGetDevice(&dev));
    LayerParams p{};
    p.N = X->rows; p.out = out; p.cols = W->cols; p.experts = experts; p.w_rows = W->rows;
    p.kblocks = (W->cols + KB - 1) / KB;
    p.w_words = (const uint32_t *)W->scales; p.x_words = (const uint32_t *)X->scales;
    p.starts = starts; p.bias = bias; p.act = act; p.y = y; p.type = type; p.ldy = ldy; p.status = status;
    if (next) { p.next_codes = (uint8_t *)next->codes; p.next_scales = (uint8_t *)next->scales; p.next_pitch = next->pitch; }
    p.impatient = spg_gemm_impatient();
    cudaStream_t st = (cudaStream_t)stream;
    const Plan plan = plan_of(p, (uint32_t)dp.sm_count);
    p.j_tiles = plan.rows == PN ? (out + 255) / 256 : (out + TM - 1) / TM;
    p.j_inverse = inverse(p.j_tiles);
    if (most_tiles(p, plan.rows) > 0x3fffffffu) return refuse(who, "too many tiles");
    switch (plan.rows) {
        case 16: return launch<16>(W, X, p, plan.split, dp, dev, st);
        case 32: return launch<32>(W, X, p, plan.split, dp, dev, st);
        case 64: return launch<64>(W, X, p, plan.split, dp, dev, st);
        case 128: return launch<128>(W, X, p, plan.split, dp, dev, st);
        default: break;
    }
    return launch_pairs(W, X, p, dp, dev, st);
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
