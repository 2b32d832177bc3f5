// spg_mx4_layer.cu -- a dense layer on two microscaled 4-bit operands.
//
//   y[n][j] = act(bias[j] + sum_b 2^(Ew[j,b] + Ex[n,b]) * sum_{k in block b} w[j][k] x[n][k])
//
// tcgen05.mma kind::mxf4 multiplies E2M1 elements and their E8M0 scales as they lie in memory: nothing is unpacked.  The weights are the
// 128-row side of a tile, rows of the batch its columns (16 to 256), so a batch of one costs no more products than one of sixteen, and a lane of
// the epilogue has one output unit: its bias is a register, and 32 lanes hold a whole block of the next layer's input.
// A k-block is 256 elements: rows of 128 bytes, 128-byte swizzle, four products of 64; its scales are two tiles of 512 bytes a side,
// which tcgen05.cp copies to tensor memory in front of the products (both are issued by one thread and run in order).
// Where there are few tiles, up to eight CTAs of a cluster share one, each with its part of the k-blocks, and send one another their sums, which are added in
// rank order.
//
// More than some hundred rows go to pairs of CTAs (below); which, and how many CTAs share a tile, an estimate in cycles says.
// What bounds it: one row x 8192 x 16384 12.8 us (5.6 TB/s; HBM, and start and end of a launch), 64 x 16384 x 16384 27.2 us (5.4 TB/s),
// 1 x 16384 x 1000 5.1 us (eight CTAs a tile), 1 x 784 x 512 3.1 us (a launch), 16384 x 8192 x 8192 366 us (6010 TFLOP/s, the tensor pipe; 430 us in a long run, under the
// power limit).
//
// Every wait on an mbarrier is bounded.  One that gave up records a code in `status`; the sums of its tile are then never said to be complete, and all CTAs that
// work on the tile leave its outputs alone.  Copies and products under way end, again waited for with a limit, before the memory that they write to is given back.
#include "spg_mx4.cuh"
#include "spg_gemm.cuh"
#include "spg_tc.cuh"
#include <cstdio>
#include <mutex>

namespace {

using namespace spgtc;

constexpr uint32_t TM = 128;                  // output units of a tile
constexpr uint32_t KB = 256;                  // elements of a k-block
constexpr uint32_t W_BYTES = TM * 128;        // codes of a tile's weights
constexpr uint32_t SF_TILE = 512;             // scales of 128 rows x 4 blocks
constexpr uint32_t SF_BYTES = 2 * SF_TILE;    // of 128 rows in a k-block
constexpr uint32_t EPI = 8, THREADS = 64 + 32 * EPI;   // warp 0: copies, warp 1: products, warps 2 to 9: outputs, two a quarter of the lanes
constexpr uint32_t MAX_STAGES = 8;
constexpr uint32_t MAX_SPLIT = 8;
constexpr uint32_t AHEAD = 2;
constexpr uint32_t PART = 8 * TM * 4;             // a CTA's sums of eight rows
constexpr uint32_t HEAD = 1024;
// Shared memory of a CTA: room for another one beside it where an SM has more than one to do (a wave's end under the next one's start), else a longer ring.
// (us with 112 and 180 KB: 64 x 16384 x 16384 on 128 CTAs 31.0 and 28.0, 64 x 8192 x 16384 16.9 and 14.9, 64 x 4096 x 65536 on 512 31.4 and 41; 227 KB
// leave the rest of an SM's memory too small a cache: one row x 8192 x 16384 14.2, 13.6 and, with 227, 14.4)
constexpr uint32_t ROOM_FOR_TWO = 112 * 1024, ROOM_ALONE = 180 * 1024;

struct LayerParams {
    uint32_t N, out, cols, kblocks, kt;       // rows, units, inputs; k-blocks; scale tiles of a row
    uint32_t split, stages;
    const uint8_t *w_scales, *x_scales;
    const float *bias;
    int act;
    void *y; int type; uint32_t ldy;
    uint8_t *next_codes, *next_scales; uint32_t next_pitch, next_kt;
    int32_t *status;
    // (the check of the failure path) the first tile whose products give up, in clusters their first CTA's; attempts of a pair's waits for a k-block and for tensor memory
    uint32_t patience, limit, limit_free;
};
constexpr uint32_t DRAIN = 1u << 12;          // attempts of a last wait

__device__ __forceinline__ uint32_t ld_shared(uint32_t addr) { uint32_t v; asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory"); return v; }
// The products' wait for a k-block, as mbar_wait_uniform.  Where it gives up, `to` and `end`, the barriers that are told of the products, become `nowhere`, others that nobody
// waits for: what follows makes products of whatever lies there, but no place of the ring is given back to copies, and no sums are said to be complete.  `steps` becomes 0:
// no products at all where sums that are not taken yet lie in their place.
// (Found out behind the wait instead, by its result and a branch, that cost 15 cycles a k-block.)
// (ASK: a first attempt that returns at once, so that with a limit of 0 nothing is waited for)
template <bool ASK = false>
__device__ __forceinline__ void wait_or_nowhere(uint32_t bar, uint32_t parity, uint32_t aborted, int32_t *status, int code, uint32_t &to, uint32_t &end, uint32_t &steps, uint32_t nowhere,
                                                uint32_t limit = 1u << 16)
{
#define SPG_MX4_WAIT(FIRST)                                                                                                                                             \
    asm volatile(                                                                                                                                                       \
        "{\n\t"                                                                                                                                                         \
        ".reg .pred p, q;\n\t"                                                                                                                                          \
        ".reg .u32 n, a;\n\t"                                                                                                                                           \
        "mbarrier." FIRST ".parity.shared::cta.b64 p, [%3], %4;\n\t"                                                                                                    \
        "@p bra SPG_MX4_DONE;\n\t"                                                                                                                                      \
        "mov.u32 n, 0;\n\t"                                                                                                                                             \
        "SPG_MX4_LOOP:\n\t"                                                                                                                                             \
        "ld.volatile.shared.u32 a, [%5];\n\t"                                                                                                                           \
        "setp.ne.u32 q, a, 0;\n\t"                                                                                                                                      \
        "@q bra SPG_MX4_NOWHERE;\n\t"                                                                                                                                   \
        "setp.ge.u32 q, n, %8;\n\t"                                                                                                                                     \
        "@q bra SPG_MX4_LATE;\n\t"                                                                                                                                      \
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%3], %4, %9;\n\t"                                                                                                 \
        "@p bra SPG_MX4_DONE;\n\t"                                                                                                                                      \
        "add.u32 n, n, 1;\n\t"                                                                                                                                          \
        "bra SPG_MX4_LOOP;\n\t"                                                                                                                                         \
        "SPG_MX4_LATE:\n\t"                                                                                                                                             \
        "st.volatile.shared.u32 [%5], 1;\n\t"                                                                                                                           \
        "atom.global.cas.b32 a, [%6], 0, %7;\n\t"                                                                                                                       \
        "SPG_MX4_NOWHERE:\n\t"                                                                                                                                          \
        "mov.u32 %0, %10;\n\t"                                                                                                                                          \
        "mov.u32 %1, %10;\n\t"                                                                                                                                          \
        "mov.u32 %2, 0;\n\t"                                                                                                                                            \
        "SPG_MX4_DONE:\n\t"                                                                                                                                             \
        "}"                                                                                                                                                             \
        : "+r"(to), "+r"(end), "+r"(steps)                                                                                                                              \
        : "r"(bar), "r"(parity), "r"(aborted), "l"(status), "r"(code), "r"(limit), "r"(SPG_WAIT_HINT_NS), "r"(nowhere) : "memory")
    if constexpr (ASK) SPG_MX4_WAIT("test_wait");
    else SPG_MX4_WAIT("try_wait");
#undef SPG_MX4_WAIT
}
// (the check of the failure path: as if it had)
__device__ __forceinline__ void give_up_if(uint32_t yes, uint32_t aborted, int32_t *status, int code, uint32_t &to, uint32_t &end, uint32_t nowhere)
{
    asm volatile(
        "{\n\t"
        ".reg .pred q;\n\t"
        ".reg .u32 a;\n\t"
        "setp.ne.u32 q, %2, 0;\n\t"
        "@q st.volatile.shared.u32 [%3], 1;\n\t"
        "@q atom.global.cas.b32 a, [%4], 0, %5;\n\t"
        "@q mov.u32 %0, %6;\n\t"
        "@q mov.u32 %1, %6;\n\t"
        "}"
        : "+r"(to), "+r"(end) : "r"(yes), "r"(aborted), "l"(status), "r"(code), "r"(nowhere) : "memory");
}
// After a wait for a k-block that gave up, by the warp of the products when they have ended: the copies under way end.  `begun`: where the k-blocks whose copies were begun
// are told, and one, when there will be no more.  (A call, so that its instructions are not in the way of CTAs that need none of them.)
__device__ __noinline__ void end_copies(uint32_t full, uint32_t stages, uint32_t begun, uint32_t late, int32_t *status)
{
    uint32_t count = 0;
    for (uint32_t i = 0; i < DRAIN && count == 0; i++) {
        __nanosleep(SPG_WAIT_HINT_NS);
        count = __reduce_max_sync(0xffffffffu, ld_shared(begun));
    }
    if (count == 0) return;
    count--;
    for (uint32_t i = count > stages ? count - stages : 0; i < count; i++) mbar_wait_uniform(full + 8 * (i % stages), i / stages & 1u, late, status, 4, DRAIN);
}

// kind::mxf4, E2M1 on both sides, UE8M0 scales, M = 128
__host__ __device__ constexpr uint32_t idesc_mx4(uint32_t n) { return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((128u >> 4) << 24); }

// (predicated: a k-block's products and copies are one way without branches)
__device__ __forceinline__ void umma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate, uint32_t yes)
{
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(yes) : "memory");
}
// 512 bytes (32 rows of 16) -> four columns of tensor memory, once for each quarter of the lanes
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc, uint32_t yes)
{
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(yes) : "memory");
}
// no swizzle, groups of eight rows of 16 bytes 128 bytes apart
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr)
{
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(128u >> 4) << 16 | (uint64_t)(128u >> 4) << 32 | (uint64_t)1u << 46;
}
__device__ __forceinline__ void st_cluster_if(uint32_t addr, float v, uint32_t yes)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.shared::cluster.f32 [%0], %1;\n\t}" ::"r"(addr), "f"(v), "r"(yes) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void cluster_arrive() { __syncwarp(); asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { __syncwarp(); asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// (predicated: branches around the stores cost 80 cycles each)
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

// Eight rows' values of this lane's unit, the warp's 32 units being one block of the next layer's input: scales, codes, stores.
// Lane i makes row i's scale for all.  A lane's eight codes are eight nibbles of a word, one a row; three exchanges among eight lanes turn that into
// eight nibbles of one row.  (Instructions bound it: with every lane making every scale a tile of 256 x 256 took longer to put out than 4096 inputs to multiply.)
__device__ __forceinline__ void put_next(const LayerParams &p, const float (&v)[8], uint32_t n0, uint32_t rows, uint32_t j0, uint32_t lane)
{
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t a = __reduce_max_sync(0xffffffffu, __float_as_uint(v[i]) & 0x7fffffffu);
        if (lane % 8u == (uint32_t)i) most = a;
    }
    const uint32_t mine = spgmx4::scale_byte(most);                              // row lane % 8
    const float inv = spgmx4::inverse_scale(mine);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = v[i] * __shfl_sync(0xffffffffu, inv, i);
    uint32_t w = spgmx4::encode8(q);
    w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 4), lane & 4u ? 0x3276 : 0x5410);
    w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 2), lane & 2u ? 0x3715 : 0x6240);
    const uint32_t other = __shfl_xor_sync(0xffffffffu, w, 1);
    w = lane & 1u ? ((w & 0xf0f0f0f0u) | ((other >> 4) & 0x0f0f0f0fu)) : ((w & 0x0f0f0f0fu) | ((other & 0x0f0f0f0fu) << 4));
    if (mine == 255u) w = 0;                                                     // a NaN block
    const uint32_t n = n0 + lane % 8u, j = j0 + lane / 8u * 8u;
    if (lane % 8u < rows && j0 < (p.out + 31u) / 32u * 32u) *reinterpret_cast<uint32_t *>(p.next_codes + (uint64_t)n * p.next_pitch + j / 2u) = w;
    if (lane < 8u && lane < rows)
        p.next_scales[((uint64_t)(n / 128u) * p.next_kt + j0 / 128u) * SF_TILE + spgmx4::scale_in_tile(n) + j0 % 128u / 32u] = (uint8_t)mine;
}

// C rows' sums of this lane's unit to outputs.  What is chosen -- activation, type -- is chosen outside the loops over them: an epilogue runs a few times a
// CTA and its instructions come from L2 as it runs (chosen inside, 128 columns took 36 000 cycles).
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
// (rows: how many of them there are; with none it only brings its instructions to the SM)
template <int C> __device__ __forceinline__ void finish(const LayerParams &p, float (&v)[C], uint32_t n0, uint32_t rows, uint32_t j0, uint32_t lane, float bias)
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
#pragma unroll
        for (int i = 0; i < C; i += 8) {
            float q[8];
#pragma unroll
            for (int k = 0; k < 8; k++) q[k] = j < p.out ? v[i + k] : 0.0f;
            put_next(p, q, n0 + i, rows > (uint32_t)i ? rows - i : 0, j0, lane);
        }
    }
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "r"(taddr) : "memory");
}

__device__ __forceinline__ void prefetch_l2(const CUtensorMap *map, int c0, int c1)
{
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
}

// the warps that read sums from tensor memory, and the one that gives it back
__device__ __forceinline__ void sums_taken() { asm volatile("bar.sync 1, %0;" ::"n"(32 * (EPI + 1)) : "memory"); }

template <uint32_t NT> struct Tile {
    static constexpr uint32_t X_BYTES = NT * 128;
    static constexpr uint32_t STAGE = (W_BYTES + X_BYTES + 2 * SF_BYTES + 1023) / 1024 * 1024;
    static constexpr uint32_t SFW = NT;                                        // tensor memory: sums, weights' scales, rows' scales
    static constexpr uint32_t SFX = 8;                                         // (behind the weights' scales)
    static constexpr uint32_t SF_COLS = 16;                                    // of a k-block, twice: copied while the products of the one before run
    static constexpr uint32_t USED = SFW + 2 * SF_COLS;
    static constexpr uint32_t COLS = USED <= 64 ? 64 : USED <= 128 ? 128 : 256;
};

// Where CTAs share a tile, chunks of eight of its rows go to them by turns, and each sends its sums of a chunk to the CTA that has it
__host__ __device__ constexpr uint32_t chunks_of(uint32_t n, uint32_t nt) { return ((n < nt ? n : nt) + 7) / 8; }
template <uint32_t NT> __host__ __device__ constexpr uint32_t parts_bytes(uint32_t n, uint32_t split)
{
    return split > 1 ? (chunks_of(n, NT) + split - 1) / split * split * PART : 0;
}

template <uint32_t NT>
__global__ void __launch_bounds__(THREADS) spg_mx4_layer_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const LayerParams p)
{
    using L = Tile<NT>;
    extern __shared__ uint8_t raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t head = smem_u32(base), parts = head + HEAD, ring = parts + parts_bytes<NT>(p.N, p.split);
    const uint32_t full = head, empty = head + 8 * MAX_STAGES, nowhere = empty + 8 * MAX_STAGES, done = nowhere + 8 * MAX_STAGES, ended = done + 8, slot = ended + 8, aborted = slot + 4, late = aborted + 4, begun = late + 4, told = begun + 4;
    // (aborted: a wait of this CTA gave up; late: one of the last waits did; begun: k-blocks whose copies were, and one; told: one of the cluster's CTAs does not have its sums)
    volatile int *abort_flag = reinterpret_cast<volatile int *>(base + (aborted - head)), *told_flag = reinterpret_cast<volatile int *>(base + (told - head));
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
    if (threadIdx.x == 0) *told_flag = 0;
    if (p.split > 1) cluster_arrive();                                           // (in front of the wait for tensor memory: see below)
    const uint32_t rank = blockIdx.x % p.split, j_tile = blockIdx.x / p.split, n0 = blockIdx.y * NT;
    // this CTA's k-blocks
    const uint32_t lo = (uint32_t)((uint64_t)p.kblocks * rank / p.split), hi = (uint32_t)((uint64_t)p.kblocks * (rank + 1) / p.split);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.stages; s++) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); mbar_init(nowhere + 8 * s, 1); }
        mbar_init(done, 1);
        mbar_init(ended, 1);
        for (uint32_t i = 0; i < 3; i++) abort_flag[i] = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(slot, L::COLS);
    if (warp == 0 && elect_one()) { prefetch_map(&map_w); prefetch_map(&map_x); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(base + (slot - head));
    spg_grid_trigger();
    // The first weights to L2 while the kernel in front still runs (whoever writes them: L2 is where writes meet).  Two k-blocks: none cost two layers
    // of 8 rows 0.1 us of 26.9, eight cost them 0.5 and a layer of one row 0.9 us of 15.1, as the copies behind the wait queue behind them.
    if (warp == 0 && elect_one())
        for (uint32_t kb = lo; kb < hi && kb < lo + AHEAD; kb++) prefetch_l2(&map_w, (int)(kb * 128u), (int)(j_tile * TM));
    __syncwarp();
    if (warp < 2) spg_grid_wait();
    if (warp == 0) {
        if (elect_one()) {
            uint32_t kb = lo;
            for (uint32_t s = 0, phase = 1; kb < hi; kb++) {
                if (!mbar_wait(empty + 8 * s, phase, abort_flag, p.status, 1)) break;
                const uint32_t at = ring + s * L::STAGE, sf = min(2u, p.kt - 2 * kb) * SF_TILE;
                mbar_expect_tx(full + 8 * s, W_BYTES + L::X_BYTES + sf * 2);
                tma_load_2d(at, &map_w, full + 8 * s, (int)(kb * 128u), (int)(j_tile * TM));
                tma_load_2d(at + W_BYTES, &map_x, full + 8 * s, (int)(kb * 128u), (int)n0);
                bulk_load(at + W_BYTES + L::X_BYTES, p.w_scales + ((uint64_t)j_tile * p.kt + 2 * kb) * SF_TILE, sf, full + 8 * s);
                bulk_load(at + W_BYTES + L::X_BYTES + SF_BYTES, p.x_scales + ((uint64_t)(n0 / 128u) * p.kt + 2 * kb) * SF_TILE, sf, full + 8 * s);
                if (++s == p.stages) { s = 0; phase ^= 1u; }
            }
            abort_flag[2] = (int)(kb - lo + 1);                                  // (begun)
        }
        __syncwarp();
    } else if (warp == 1) {
        // (One lane runs the loop, and the last k-block has one commit, not two: 340 cycles a k-block.  With the lane chosen anew for each, a way of its own for
        // a row's end and a second commit behind the loop it took 445, whatever the copies and products were, and a short layer 0.1 us more.)
        const uint32_t idesc = idesc_mx4(NT);
        uint32_t to = empty, end = done, steps = 0;
        if (elect_one()) {
            give_up_if(p.patience == 0 && rank == 0, aborted, p.status, 2, to, end, nowhere);
            for (uint32_t kb = lo, s = 0, phase = 0; kb < hi; kb++) {
                wait_or_nowhere(full + 8 * s, phase, aborted, p.status, 2, to, end, steps, nowhere);
                tc_fence_after();
                const uint32_t at = ring + s * L::STAGE, sf = tmem + L::SFW + ((kb - lo) & 1u) * L::SF_COLS, left = p.cols - kb * KB;
                const uint32_t sfw = at + W_BYTES + L::X_BYTES, sfx = sfw + SF_BYTES;
                const uint64_t dw = scale_desc(sfw), dx = scale_desc(sfx), a = smem_desc_sw128(at), b = smem_desc_sw128(at + W_BYTES);
                const auto scales = [&](uint32_t i, uint32_t yes) {
                    copy_scales(sf + 4 * i, dw + i * (SF_TILE >> 4), yes);
                    copy_scales(sf + L::SFX + 4 * i, dx + i * (SF_TILE >> 4), yes);
                };
                const auto product = [&](uint32_t i, uint32_t more, uint32_t yes) {
                    const uint32_t id = (i & 1u) * 2u;          // which two of a tile's four scales
                    umma_mx4(tmem, a + 2 * i, b + 2 * i, idesc | id << 4 | id << 29, sf + 4 * (i / 2), sf + L::SFX + 4 * (i / 2), more, yes);
                };
                scales(0, 1); scales(1, left > 128);
                product(0, kb > lo, 1); product(1, 1, left > 64); product(2, 1, left > 128); product(3, 1, left > 192);
                umma_commit(kb + 1 < hi ? to + 8 * s : end);
                if (++s == p.stages) { s = 0; phase ^= 1u; }
            }
        }
        __syncwarp();
        // The products end here, beside the outputs.  So have the copies then, each of which was waited for, but where a wait gave up
        if (elect_one()) umma_commit(ended);
        __syncwarp();
        mbar_wait_uniform(ended, 0, late, p.status, 5);
        if (__any_sync(0xffffffffu, end == nowhere)) end_copies(full, p.stages, begun, late, p.status);
        if (p.split > 1) {
            // Given back before this CTA waits for the others: one that has none on its SM, and so cannot finish, may hold up a cluster that holds some elsewhere
            sums_taken();
            tc_fence_after();
            tmem_free(tmem, L::COLS);
        }
    } else {
        const uint32_t quad = warp % 4u, half = (warp - 2u) / 4u, j0 = j_tile * TM + quad * 32u, j = j0 + lane;
        const uint32_t lanes = tmem + (quad * 32u << 16);
        // Once without a row before the launch in front has ended: the outputs' instructions come from L2, some 1500 cycles that would follow the products
        float bias = 0.0f;
        bool ok = true;
#pragma unroll 1
        for (uint32_t dry = 1;; dry = 0) {
            if (!dry) {
                spg_grid_wait();
                if (p.bias && j < p.out) bias = p.bias[j];
                ok = __all_sync(0xffffffffu, mbar_wait(done, 0, abort_flag, p.status, 3));           // (a warp goes one way)
                tc_fence_after();
                if (p.split > 1) {
                    // This CTA's sums to those that put them out, [chunk][CTA][row][unit].  (Sent before one barrier, not fetched behind it: reading the others' took 6800
                    // cycles from the last product to the end, 2700 of them the instructions of 64 loads.)
                    cluster_wait();                                              // all have begun
                    const uint32_t chunks = ok ? chunks_of(p.N, NT) : 0;
                    for (uint32_t c = half; c < chunks && n0 + 8 * c < p.N; c += 2) {
                        float v[8];
                        tmem_ld8(lanes + 8 * c, v);
                        tmem_ld_wait();
                        const uint32_t to = mapa(parts + (c / p.split * p.split + rank) * PART + (quad * 32u + lane) * 4u, c % p.split), left = p.N - (n0 + 8 * c);
#pragma unroll
                        for (int i = 0; i < 8; i++) st_cluster_if(to + i * TM * 4u, v[i], (uint32_t)i < left);
                    }
                    if (!ok && lane < p.split) st_cluster_u32(mapa(told, lane), 1);
                    tc_fence_before();
                    __syncwarp();
                    sums_taken();
                    cluster_arrive();
                    cluster_wait();
                    ok = !__any_sync(0xffffffffu, *told_flag);
                }
                if (!ok) break;
            }
            const uint32_t end = dry ? n0 + 1 : p.N;
#pragma unroll 1
            for (uint32_t c = dry ? 0 : (half * p.split + rank) * 8u; c < NT && n0 + c < end; c += p.split * 16u) {
                float v[8];
                if (p.split == 1 || dry) {
                    if (!dry) { tmem_ld8(lanes + c, v); tmem_ld_wait(); }
                    else each(v, [](float) { return 0.0f; });
                } else {
                    const float *part = reinterpret_cast<const float *>(base + HEAD) + (c / 8 / p.split * p.split) * (PART / 4) + quad * 32u + lane;
                    each(v, [](float) { return 0.0f; });
#pragma unroll 1
                    for (uint32_t r = 0; r < p.split; r++, part += PART / 4) {   // in rank order
#pragma unroll
                        for (int i = 0; i < 8; i++) v[i] += part[i * TM];
                    }
                }
                finish(p, v, n0 + c, dry ? 0u : p.N - (n0 + c), j0, lane, bias);
            }
            if (!dry) break;
        }
        tc_fence_before();
    }
    if (p.split > 1 && warp < 2) { cluster_wait(); cluster_arrive(); cluster_wait(); }
    __syncwarp();
    __syncthreads();
    if (warp == 1 && p.split == 1) { tc_fence_after(); tmem_free(tmem, L::COLS); }
}

// ---- pairs of CTAs, many rows -------------------------------------------------------------------------------------------------
// 256 units x 256 rows of the batch a tile on a cluster of two (cta_group::2): each CTA holds 128 units' weights and half of the rows, so a k-block costs it
// 35 KB for 512 cycles of products; a CTA alone would need 51. Persistent: the copies run ahead over the tile's end, and the sixteen
// epilogue warps take all 256 columns of sums to registers at once (64 a thread), so the next tile's products wait for that alone (there
// is no room in tensor memory for a second accumulator of 256 columns beside the scales).
constexpr uint32_t PN = 256;                                   // rows of the batch a tile
constexpr uint32_t P_EPI = 16, P_THREADS = 64 + 32 * P_EPI;
constexpr uint32_t P_COLS = PN / (P_EPI / 4);                   // columns of an epilogue warp
constexpr uint32_t P_CODES = W_BYTES + PN / 2 * 128;           // a CTA's codes of a k-block
constexpr uint32_t P_STAGE = P_CODES + SF_BYTES + 2 * SF_BYTES;
constexpr uint32_t P_STAGES = 6;
constexpr uint32_t P_SF = PN, P_SFX = 8, P_SF_COLS = 24;        // columns of tensor memory: scales behind the sums, twice; those of the rows behind the weights'
constexpr uint32_t P_SMEM = 1024 + HEAD + P_STAGES * P_STAGE;

__device__ __forceinline__ void umma_mx4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// in both CTAs, each from its own shared memory to its own tensor memory
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
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

// tile t of a walk over bands of eight tiles of units, the units fastest inside a band
__device__ __forceinline__ void pair_tile(uint32_t t, uint32_t j_tiles, uint32_t n_tiles, uint32_t &j, uint32_t &n)
{
    const uint32_t band = 8u * n_tiles, g = t / band, r = t % band, here = min(8u, j_tiles - g * 8u);
    j = g * 8u + r % here; n = r / here;
}

constexpr uint32_t P_ENDED = 24 * P_STAGES + 16, P_LATE = P_ENDED + 16, P_TOLD = P_LATE + 4;      // places in the head: the barrier of the last products, the flag of the last waits, k-blocks begun
// one k-block's copies of a CTA (one lane; leader: the first CTA's barrier, which counts those of both)
__device__ __forceinline__ void copy_pair(const CUtensorMap *w, const CUtensorMap *x, const CUtensorMap *sw, const CUtensorMap *sx, uint32_t at, uint32_t leader,
                                          uint32_t rank, uint32_t kb, uint32_t j, uint32_t n)
{
    tma_load_2d_pair(at, w, leader, (int)(kb * 128u), (int)(j * 256u + rank * 128u));
    tma_load_2d_pair(at + W_BYTES, x, leader, (int)(kb * 128u), (int)(n * PN + rank * (PN / 2)));
    tma_load_2d_pair(at + P_CODES, sw, leader, (int)(kb * 256u), (int)(j * 2u + rank));
    tma_load_2d_pair(at + P_CODES + SF_BYTES, sx, leader, (int)(kb * 256u), (int)(n * (PN / 128)));
}
// The same of a pair, by its first CTA, which first ends the waits of both.
// Each k-block's are counted for both CTAs at once: where one of them began fewer, as many bytes are fetched here once more, or expected of the other alone.
__device__ __noinline__ void end_pair(const CUtensorMap *w, const CUtensorMap *x, const CUtensorMap *sw, const CUtensorMap *sx, uint32_t head, uint32_t aborted, int32_t *status)
{
    atomicCAS(status, 0, 2);
    for (uint32_t r = 0; r < 2; r++) st_cluster_u32(mapa(aborted, r), 1);
    uint32_t mine = 0, other = 0;
    for (uint32_t i = 0; i < DRAIN && (mine == 0 || other == 0); i++) {
        __nanosleep(SPG_WAIT_HINT_NS);
        mine = __reduce_max_sync(0xffffffffu, ld_shared(head + P_TOLD));
        other = __reduce_max_sync(0xffffffffu, ld_shared(head + P_TOLD + 4));
    }
    if (mine == 0 || other == 0) return;
    const uint32_t most = max(--mine, --other);
    for (uint32_t i = min(mine, other); i < most; i++) {
        const uint32_t s = i % P_STAGES, bar = head + 8 * s;
        if (elect_one()) {
            if (i >= mine) mbar_expect_tx(bar, P_STAGE);                         // (the other's)
            else copy_pair(w, x, sw, sx, head + HEAD + s * P_STAGE, mapa(bar, 0), 0, 0, 0, 0);
        }
        __syncwarp();
    }
    for (uint32_t i = most > P_STAGES ? most - P_STAGES : 0; i < most; i++) mbar_wait_uniform_cluster(head + 8 * (i % P_STAGES), i / P_STAGES & 1u, head + P_LATE, status, 4, DRAIN);
}

__global__ void __launch_bounds__(P_THREADS, 1) spg_mx4_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                    const __grid_constant__ CUtensorMap map_sw, const __grid_constant__ CUtensorMap map_sx,
                                                                    const LayerParams p, uint32_t j_tiles, uint32_t n_tiles)
{
    extern __shared__ uint8_t raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t head = smem_u32(base), ring = head + HEAD;
    const uint32_t full = head, empty = full + 8 * P_STAGES, nowhere = empty + 8 * P_STAGES, sums_full = nowhere + 8 * P_STAGES, sums_free = sums_full + 8, ended = head + P_ENDED, slot = ended + 8, aborted = slot + 4, told = head + P_TOLD;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(base + (aborted - head));
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, rank = cluster_rank(), pairs = gridDim.x / 2u, pair = blockIdx.x / 2u, tiles = j_tiles * n_tiles;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < P_STAGES; s++) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); mbar_init(nowhere + 8 * s, 1); }
        mbar_init(sums_full, 1);
        mbar_init(sums_free, 2 * P_EPI);
        mbar_init(ended, 1);
        for (uint32_t i = 0; i < 4; i++) abort_flag[i] = 0;                      // (and the flag of the last waits, and what is told of k-blocks)
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc_pair(slot, 512);
    if (warp == 0 && elect_one()) { prefetch_map(&map_w); prefetch_map(&map_x); prefetch_map(&map_sw); prefetch_map(&map_sx); }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(base + (slot - head));
    spg_grid_trigger();
    if (warp < 2) spg_grid_wait();

    if (warp == 0) {
        const uint32_t leader = mapa(full, 0);
        uint32_t s = 0, phase = 1, begun = 0;
        for (uint32_t t = pair; t < tiles && !*abort_flag; t += pairs) {
            uint32_t j, n;
            pair_tile(t, j_tiles, n_tiles, j, n);
            for (uint32_t kb = 0; kb < p.kblocks; kb++) {
                mbar_wait_uniform_cluster(empty + 8 * s, phase, aborted, p.status, 1);
                if (*abort_flag) break;
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * P_STAGE);
                    copy_pair(&map_w, &map_x, &map_sw, &map_sx, ring + s * P_STAGE, leader + 8 * s, rank, kb, j, n);
                }
                __syncwarp();
                begun++;
                if (++s == P_STAGES) { s = 0; phase ^= 1u; }
            }
        }
        if (lane == 0) st_cluster_u32(mapa(told + 4 * rank, 0), begun + 1);       // (k-blocks whose copies were begun here, and one: see end_pair)
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = (idesc_mx4(PN) & ~(31u << 24)) | ((256u >> 4) << 24);
            uint32_t s = 0, phase = 0, turn = 1, back = empty, end = sums_full;
            for (uint32_t t = pair; t < tiles; t += pairs) {
                if (t >= p.patience) back = end = nowhere;
                uint32_t kblocks = p.kblocks;
                wait_or_nowhere<true>(sums_free, turn, aborted, p.status, 6, back, end, kblocks, nowhere, p.limit_free);
                turn ^= 1u;
                tc_fence_after();
                for (uint32_t kb = 0; kb < kblocks; kb++) {
                    wait_or_nowhere(full + 8 * s, phase, aborted, p.status, 2, back, end, kblocks, nowhere, p.limit);
                    tc_fence_after();
                    const uint32_t at = ring + s * P_STAGE, to = tmem + P_SF + (kb & 1u) * P_SF_COLS;
                    if (elect_one()) {
                        const uint64_t sf = scale_desc(at + P_CODES), a = smem_desc_sw128(at), b = smem_desc_sw128(at + W_BYTES);
                        const auto scales = [&](uint32_t i) {
                            copy_scales_pair(to + 4 * i, sf + i * (SF_TILE >> 4));
                            copy_scales_pair(to + P_SFX + 8 * i, sf + ((SF_BYTES + i * SF_TILE) >> 4));
                            copy_scales_pair(to + P_SFX + 8 * i + 4, sf + ((2 * SF_BYTES + i * SF_TILE) >> 4));
                        };
                        const auto product = [&](uint32_t i, uint32_t more) {
                            const uint32_t id = (i & 1u) * 2u;
                            umma_mx4_pair(tmem, a + 2 * i, b + 2 * i, idesc | id << 4 | id << 29, to + 4 * (i / 2), to + P_SFX + 8 * (i / 2), more);
                        };
                        if (kb * KB + KB - 64u < p.cols) {
                            scales(0); scales(1);
                            product(0, kb); product(1, 1); product(2, 1); product(3, 1);
                        } else {
                            const uint32_t steps = (p.cols - kb * KB + 63u) / 64u;
                            scales(0);
                            if (steps > 2) scales(1);
                            product(0, kb);
                            if (steps > 1) product(1, 1);
                            if (steps > 2) product(2, 1);
                        }
                        umma_commit_pair(back + 8 * s);
                    }
                    __syncwarp();
                    if (++s == P_STAGES) { s = 0; phase ^= 1u; }
                }
                if (elect_one()) umma_commit_pair(end);
                __syncwarp();
                if (__any_sync(0xffffffffu, end == nowhere)) break;
            }
            // The products end here, beside the last tile's outputs.  So have the copies then, each of which was waited for, but where a wait gave up
            if (elect_one()) umma_commit_pair(ended);
            __syncwarp();
            mbar_wait_uniform(ended, 0, head + P_LATE, p.status, 5);
            if (__any_sync(0xffffffffu, end == nowhere)) end_pair(&map_w, &map_x, &map_sw, &map_sx, head, aborted, p.status);
            __syncwarp();
        }
    } else {
        const uint32_t quad = warp % 4u, part = (warp - 2u) / 4u, free_at = mapa(sums_free, 0);
        uint32_t turn = 0, dry = 1;                                              // (dry: once without a row, as above)
#pragma unroll 1
        for (uint32_t t = pair; t < tiles;) {
            uint32_t jt, nt;
            pair_tile(t, j_tiles, n_tiles, jt, nt);
            const uint32_t j0 = jt * 256u + rank * 128u + quad * 32u, j = j0 + lane, n0 = nt * PN + part * P_COLS;
            const float bias = !dry && p.bias && j < p.out ? p.bias[j] : 0.0f;
            const uint32_t from = tmem + (quad * 32u << 16) + part * P_COLS;
            const bool some = j0 < (p.next_codes ? (p.out + 127u) / 128u * 128u : p.out);       // (the next operand's scale tiles are written whole)
            if (!dry) {
                if (!__all_sync(0xffffffffu, mbar_wait(sums_full, turn, abort_flag, p.status, 3))) break;           // (a warp goes one way)
                turn ^= 1u;
                tc_fence_after();
            }
            if (dry || t + pairs >= tiles) {
                // the last: nobody waits for tensor memory, and a short loop is quicker than 64 columns written out that come from L2
#pragma unroll 1
                for (uint32_t c = 0; c < (dry ? 1u : P_COLS) && (dry || (n0 + c < p.N && some)); c += 16) {
                    uint32_t r[16];
                    float v[16];
                    each(v, [](float) { return 0.0f; });
                    if (!dry) {
                        tmem_ld16(from + c, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
                    }
                    finish(p, v, n0 + c, dry ? 0u : p.N - (n0 + c), j0, lane, bias);
                }
                tc_fence_before();
                if (dry) { dry = 0; spg_grid_wait(); continue; }
            } else {
                float v[P_COLS];
#pragma unroll
                for (int i = 0; i < (int)P_COLS; i += 32) tmem_ld32(from + i, v + i);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(free_at);
                if (n0 < p.N && some) finish(p, v, n0, p.N - n0, j0, lane, bias);
            }
            t += pairs;
        }
    }
    __syncwarp();
    __syncthreads();
    cluster_sync();
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

int encode(CUtensorMap *map, CUtensorMapDataType type, void *at, uint64_t width, uint64_t rows, uint64_t pitch, uint32_t box_width, uint32_t box_rows, CUtensorMapSwizzle swizzle)
{
    EncodeTiledFn fn = encode_fn();
    if (!fn) { spgk_set_error("cuTensorMapEncodeTiled", "driver entry point not available"); return SPGK_E_CUDA; }
    const cuuint64_t dims[2] = { width, rows }, strides[1] = { pitch };
    const cuuint32_t box[2] = { box_width, box_rows }, steps[2] = { 1, 1 };
    const CUresult r = fn(map, type, 2, at, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        char msg[64];
        snprintf(msg, sizeof msg, "CUresult %d", (int)r);
        spgk_set_error("cuTensorMapEncodeTiled (4-bit operand)", msg);
        return SPGK_E_CUDA;
    }
    return SPGK_OK;
}
// boxes of 256 elements x box_rows rows of a matrix' codes
int codes_map(CUtensorMap *map, const spgk_mx4 *m, uint32_t box_rows)
{
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, m->codes, spgk_mx4_pitch(m->cols), m->rows, m->pitch, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}
// boxes of two scale tiles (of 256 elements a row) x box_tiles tiles of 128 rows
int scales_map(CUtensorMap *map, const spgk_mx4 *m, uint32_t box_tiles)
{
    const uint64_t kt = spgmx4::tiles4(m->cols);
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, m->scales, kt * 128, ((uint64_t)m->rows + 127) / 128, kt * SF_TILE, 256, box_tiles, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// How a product is arranged: CTAs that share a tile, and an estimate in cycles of a chain of launches on a B200 at 1.9 GHz.  Fitted to 1377 products (1 to 1000 rows,
// 256 to 16384 inputs, 128 to 16384 units): what it picks takes 0.7 % longer on average than the best of all arrangements, 17 % at most.  A k-block takes 310 cycles, and 580
// where all SMs draw on HBM; clusters on more than half of the SMs leave the next launch's no room beside them.
// clusters of this many CTAs that find room at a time, one CTA an SM
uint32_t at_a_time(uint32_t split, uint32_t sms) { return (split == 8 ? 15u : split == 4 ? 33u : split == 2 ? 74u : 148u) * sms / 148u; }
struct Plan { uint32_t split; uint64_t cycles; };
Plan plan_single(const LayerParams &p, uint32_t nt, uint32_t sms)
{
    const uint64_t tiles = (uint64_t)((p.out + TM - 1) / TM) * ((p.N + nt - 1) / nt);
    const uint32_t cols = p.N < nt ? p.N : nt;
    Plan best = { 1, ~0ull };
    for (uint32_t s = 1; s <= MAX_SPLIT && s <= p.kblocks; s *= 2) {
        if (s > 1 && tiles > at_a_time(s, sms)) break;
        const uint64_t ctas = tiles * s, waves = (ctas + sms - 1) / sms, block = 310 + (ctas < sms ? ctas : sms) * 9 / 5;
        const uint64_t outputs = s == 1 ? (cols + 31) / 32 * 1700 : 2010 + s * 190 + cols / s * 70 + cols * 20;
        const uint64_t cycles = 2660 + waves * ((uint64_t)((p.kblocks + s - 1) / s) * block + outputs) + (s > 1 && ctas * 2 > sms ? 1360 : 0);
        if (cycles < best.cycles) best = { s, cycles };
    }
    return best;
}
uint64_t pair_cycles(const LayerParams &p, uint32_t sms)
{
    const uint64_t tiles = (uint64_t)((p.out + 255) / 256) * ((p.N + PN - 1) / PN), waves = (tiles + sms / 2 - 1) / (sms / 2);
    return 4650 + waves * ((uint64_t)p.kblocks * 580 + 4660);
}

template <uint32_t NT> int launch(const spgk_mx4 *W, const spgk_mx4 *X, LayerParams p, const SpgDeviceProps &dp, int dev, cudaStream_t stream)
{
    using L = Tile<NT>;
    static SpgOncePerDevice once;
    int rc = once.run(dev, [&]() -> int {
        SPGK_CUDA(cudaFuncSetAttribute(spg_mx4_layer_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dp.smem_optin));
        return SPGK_OK;
    });
    if (rc) return rc;
    CUtensorMap map_w, map_x;
    if ((rc = codes_map(&map_w, W, TM)) || (rc = codes_map(&map_x, X, NT))) return rc;
    const uint32_t j_tiles = (p.out + TM - 1) / TM, n_tiles = (p.N + NT - 1) / NT;
    p.split = plan_single(p, NT, (uint32_t)dp.sm_count).split;
    const uint32_t room = NT > 64 ? (uint32_t)dp.smem_optin : (uint64_t)j_tiles * n_tiles > at_a_time(p.split, (uint32_t)dp.sm_count) ? ROOM_FOR_TWO : ROOM_ALONE;
    const uint32_t parts = parts_bytes<NT>(p.N, p.split), most = (room - HEAD - 1024 - parts) / L::STAGE, mine = (p.kblocks + p.split - 1) / p.split;
    p.stages = mine < most ? mine : most;
    if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
    const uint32_t bytes = parts + p.stages * L::STAGE;
    if (n_tiles > 65535u) { spgk_set_error("spgk_layer_mx4", "more than 65535 tiles of rows"); return SPGK_E_ARG; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(j_tiles * p.split, n_tiles); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = HEAD + 1024 + bytes; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    SPGK_CUDA(cudaLaunchKernelEx(&cfg, spg_mx4_layer_kernel<NT>, map_w, map_x, p));
    return spgk_check_launch("spg_mx4_layer_kernel");
}

int launch_pairs(const spgk_mx4 *W, const spgk_mx4 *X, LayerParams p, const SpgDeviceProps &dp, int dev, cudaStream_t stream)
{
    static SpgOncePerDevice once;
    int rc = once.run(dev, [&]() -> int {
        SPGK_CUDA(cudaFuncSetAttribute(spg_mx4_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P_SMEM));
        return SPGK_OK;
    });
    if (rc) return rc;
    CUtensorMap map_w, map_x, map_sw, map_sx;
    if ((rc = codes_map(&map_w, W, TM)) || (rc = codes_map(&map_x, X, PN / 2)) || (rc = scales_map(&map_sw, W, 1)) || (rc = scales_map(&map_sx, X, PN / 128))) return rc;
    const uint32_t j_tiles = (p.out + 255) / 256, n_tiles = (p.N + PN - 1) / PN;
    const uint64_t tiles = (uint64_t)j_tiles * n_tiles;
    if (tiles > 0x3fffffffu) { spgk_set_error("spgk_layer_mx4", "too many tiles"); return SPGK_E_ARG; }
    const uint32_t pairs = tiles < (uint32_t)dp.sm_count / 2 ? (uint32_t)tiles : (uint32_t)dp.sm_count / 2;
    if (p.patience == 0) p.patience = (uint32_t)tiles - pairs;             // (each pair's last tile)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(pairs * 2); cfg.blockDim = dim3(P_THREADS); cfg.dynamicSmemBytes = P_SMEM; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    SPGK_CUDA(cudaLaunchKernelEx(&cfg, spg_mx4_pair_kernel, map_w, map_x, map_sw, map_sx, p, j_tiles, n_tiles));
    return spgk_check_launch("spg_mx4_pair_kernel");
}

}  // namespace

extern "C" int spgk_layer_mx4(const spgk_mx4 *W, const float *bias, int act, const spgk_mx4 *X, void *y, int type, uint32_t ldy,
                              const spgk_mx4 *next, int32_t *status, void *stream)
{
    int rc;
    if ((rc = spg_mx4_check("spgk_layer_mx4 (weights)", W)) || (rc = spg_mx4_check("spgk_layer_mx4 (inputs)", X))) return rc;
    if (next && (rc = spg_mx4_check("spgk_layer_mx4 (next)", next))) return rc;
    const char *why = nullptr;
    if (W->rows == 0 || W->cols != X->cols) why = "weights and inputs do not belong together";
    else if (W->cols > (1u << 27)) why = "more than 2^27 inputs";             // (a tile's products end well before the waits for them give up)
    else if (act < SPG_ACT_SIGMOID || act > SPG_ACT_NONE) why = "unknown activation";
    else if (!y && !next) why = "no output";
    else if (y && type != SPGK_T_F16 && type != SPGK_T_BF16 && type != SPGK_T_F32) why = "unknown type";
    else if (y && (uintptr_t)y % (type == SPGK_T_F32 ? 4u : 2u)) why = "output not aligned to its type";
    else if (y && X->rows > 1 && ldy < W->rows) why = "rows of the output overlap";
    else if (next && (next->rows != X->rows || next->cols != W->rows)) why = "the next operand has other rows or columns";
    else if (next && act == SPG_ACT_SOFTMAX) why = "a softmax is left to spgk_softmax_rows";
    else if (!status) why = "no status word";
    else if ((uintptr_t)bias % 4u) why = "bias not aligned";
    if (why) { spgk_set_error("spgk_layer_mx4", why); return SPGK_E_ARG; }
    if (X->rows == 0) return SPGK_OK;
    SpgDeviceProps dp;
    int dev = 0;
    if ((rc = spg_device_props(&dp))) return rc;
    SPGK_CUDA(cudaGetDevice(&dev));
    LayerParams p{};
    p.N = X->rows; p.out = W->rows; p.cols = W->cols;
    p.kblocks = (W->cols + KB - 1) / KB; p.kt = spgmx4::tiles4(W->cols);
    p.w_scales = (const uint8_t *)W->scales; p.x_scales = (const uint8_t *)X->scales;
    p.bias = bias; p.act = act; p.y = y; p.type = type; p.ldy = ldy; p.status = status;
    const int impatient = spg_gemm_impatient();
    p.patience = impatient == 1 ? 0 : 0xffffffffu; p.limit = impatient == 1 ? 64 : 1u << 16; p.limit_free = impatient == 2 ? 0 : 1u << 16;
    if (next) { p.next_codes = (uint8_t *)next->codes; p.next_scales = (uint8_t *)next->scales; p.next_pitch = next->pitch; p.next_kt = spgmx4::tiles4(next->cols); }
    cudaStream_t st = (cudaStream_t)stream;
    if (p.N <= 16) return launch<16>(W, X, p, dp, dev, st);
    if (p.N <= 32) return launch<32>(W, X, p, dp, dev, st);
    if (p.N <= 64) return launch<64>(W, X, p, dp, dev, st);
    // (us with single CTAs and in pairs: 256 x 8192 x 8192 13.6 and 16.0, 512 rows 25.4 and 16.8, 300 x 1024 x 512 5.9 and 6.8, 130 x 8192 x 1000 9.7 and 14.0)
    if (plan_single(p, 128, (uint32_t)dp.sm_count).cycles <= pair_cycles(p, (uint32_t)dp.sm_count)) return launch<128>(W, X, p, dp, dev, st);
    return launch_pairs(W, X, p, dp, dev, st);
}
