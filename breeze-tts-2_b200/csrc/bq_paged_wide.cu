// Paged attention for tiles of many rows (prompts, a prefix shared by a batch)
// on the tcgen05 tensor cores: 256 rows per CTA in two halves of 128, keys and
// values in units of 128 positions.
//
// Bound: tensor cores and, as close, the exponentials: a half's unit is two
// products of 128 x 128 x D (512 cycles each at D = 128) and 128 x 128
// exponentials (1024 cycles on an SM's 16 lanes). So everything has to overlap.
// The halves take turns in one score buffer: as soon as a half's softmax warps
// have its scores in registers, the next scores (the other half's) are computed
// over them, and a half's second product runs while its next scores are being
// worked on. Both halves use the same k / v tiles, which halves what the tiles
// cost in L2 reads (32 bytes per cycle and SM).
//
// Roles (one CTA per SM, all 512 tensor-memory columns):
//   warps 0-3, 4-7  softmax of half 0 / 1, one row per thread: the row's 128
//                   scores from tensor memory, running maximum and sum, the
//                   probabilities back to tensor memory in 16 bits (the A
//                   operand of the second product). The output accumulator
//                   stays in tensor memory; a row's reference maximum may lag
//                   behind the true one by up to a factor 2^8 (probabilities up
//                   to 256 are exact enough in either type, and the factor
//                   cancels), so the accumulator is rescaled only when a maximum
//                   really moves.
//   warp 8          k and v by tiled TMA, one box per page (or 128 positions of
//                   one) and 64 dims, into a ring of 32 KB stages
//   warps 9, 10     issue the products, each its own: S = Q K^T (both operands in
//                   shared memory, K-major) and O += P V (A in tensor memory, V
//                   as stored, dims contiguous). Issuing blocks until the tensor
//                   cores take the product, so while one warp is between two
//                   products the other's keep them busy
//   warp 11         walks the tiles of the CTA's share, passes each on to the other
//                   roles through shared memory and fetches its queries (by TMA
//                   when the query heads of a kv head are a power of two: then
//                   128 rows are a box of whole tokens)
// Page slots behind the last position arrive with the last page, whatever they
// hold; before the product that would multiply them by zero probabilities the
// softmax warps of half 0 clear those rows of v. Scores there are never used.
// Infinite and NaN entries of v at positions that only some rows of a tile see
// are cleared likewise, and added in memory to the outputs of the rows that see
// them.
//
// Measured, join included (B200, calls in a row): 7000 new positions of 16 query and 8
// kv heads of 128, causal, 201 GFLOP in 209 us on the same inputs again, which are then
// in L2 (0.96 PFLOP/s; library products of 8192^3 run at 1.65), 233 us on others each
// call; 1474 ragged ones of 32 heads over 18 thousand in 111 and 120 us. The tensor cores
// and the exponential units are each busy half of the time; without the softmax's
// arithmetic the same pipeline takes 163 us, and a change of tile 7700 cycles.
// Dropped: units of 64 positions with a score buffer per half (271 against then 238
// us), two threads per row (291), outputs staged through shared memory (245 against
// 237), a peeled unit loop (266), every fourth, third or eighth pair of exponentials
// as a polynomial (211, 218 and 207 against 210): what the softmax warps wait for is
// mostly not the exponential units but their own chains of instructions. A score
// buffer per half, the probabilities through shared memory instead: 266.
#include <algorithm>
#include <climits>
#include <cstring>

#include "bq_host.h"
#include "bq_paged.cuh"
#include "bq_paged_host.h"
#include "bq_tmem.cuh"

namespace bq {

struct PagedWideParams {
    CUtensorMap qmap, kmap, vmap;  // (D, then slot, head and page in order of stride); boxes of 64 dims x positions of one page
    PagedWork w;
    int32_t box;                          // positions per box: min(page size, 128)
    int32_t k_slot, k_head, v_slot, v_head;  // which of coordinates 1 .. 3 is the slot, the head (the third is the page)
    int32_t q_tma;                        // the queries come by TMA: qmap is (D, heads, rows), boxes of 64 dims x 128 rows
    uint32_t idesc_qk, idesc_pv;
    long long wait_cycles;
};

namespace {

constexpr int kThreads = 384;
// Registers: the CTA starts with 384 x 168; the third warpgroup gives up what the softmax warps, a row of 128
// scores per thread, need more (256 x 216 + 128 x 72). The file is compiled as a whole program, since relocatable
// code may not move registers.
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
constexpr int kRows = kWideRows, kUnit = kWideUnit;
constexpr uint32_t kCols = 512;

template <int D>
struct WideSmem {
    static constexpr uint32_t kTile = 128 * D * 2;                   // one k or v tile, one half of the queries
    static constexpr int kStages = D == 128 ? 4 : 8;
    static constexpr uint32_t kRing = 2 * kTile;
    static constexpr uint32_t kBars = kRing + kStages * kTile;
    static constexpr uint32_t kTotal = kBars + 512 + 1024;           // + slack to align the tiles to 1024 bytes
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}

// Shared-memory matrix descriptors are a constant upper half and a lower half that
// only differs in the address.
// K-major tile (queries, keys): rows of 64 dims (128 B, 128-byte swizzle), groups
// of 8 rows 1024 B apart (stride offset; the leading offset is not used); version
// bit 46, layout type 2.
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kDescLoK = 1u << 16;
// v tile as the B operand with its dims (N) contiguous: one row of 64 dims per
// position, groups of 8 positions 1024 B apart (stride offset), the second 64 dims
// 128 rows further (leading offset).
constexpr uint32_t kDescLoV = uint32_t((128 * 128) >> 4) << 16;

// The products of a unit. One thread of the (converged) warp issues, by a predicate
// and not a branch, so that the operands can stay in uniform registers. Completion
// arrives on `bar`, and on `bar2` unless it is 0.
// S = Q K^T: D / 16 steps of 128 x 128 x 16, 32 B apart within a swizzled 64-dim row,
// then in the second 64 dims 128 rows on.
template <int D>
__device__ __forceinline__ void scores_product(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t bar, uint32_t bar2) {
    if constexpr (D == 128) {
    asm volatile(
        "{\n\t.reg .pred e, no, yes;\n\t.reg .b32 x, y;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 no, 0, 0;\n\tsetp.eq.b32 yes, 0, 0;\n\t"
        "add.u32 x, %1, 0;\n\tadd.u32 y, %2, 0;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, no;\n\t"
        "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "add.u32 x, %1, 1024;\n\tadd.u32 y, %2, 1024;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "add.u32 x, %1, 1026;\n\tadd.u32 y, %2, 1026;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "add.u32 x, %1, 1028;\n\tadd.u32 y, %2, 1028;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "add.u32 x, %1, 1030;\n\tadd.u32 y, %2, 1030;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t"
        "setp.ne.and.b32 e, %7, 0, e;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(0), "r"(bar), "r"(bar2)
        : "memory");
    } else {
    asm volatile(
        "{\n\t.reg .pred e, no, yes;\n\t.reg .b32 x, y;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 no, 0, 0;\n\tsetp.eq.b32 yes, 0, 0;\n\t"
        "add.u32 x, %1, 0;\n\tadd.u32 y, %2, 0;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, no;\n\t"
        "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, yes;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t"
        "setp.ne.and.b32 e, %7, 0, e;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(0), "r"(bar), "r"(bar2)
        : "memory");
    }
}
// O (+)= P V: 8 steps of 128 x D x 16, 16 positions (2048 B) and 8 columns of P apart.
__device__ __forceinline__ void output_product(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool accumulate,
                                               uint32_t bar, uint32_t bar2) {
    asm volatile(
        "{\n\t.reg .pred e, first, yes;\n\t.reg .b32 x, y;\n\t.reg .b64 b;\n\t"
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 first, %5, 0;\n\tsetp.eq.b32 yes, 0, 0;\n\t"
        "add.u32 x, %1, 0;\n\tadd.u32 y, %2, 0;\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, first;\n\t"
        "add.u32 x, %1, 8;\n\tadd.u32 y, %2, 128;\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, yes;\n\t"
        "add.u32 x, %1, 16;\n\tadd.u32 y, %2, 256;\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, yes;\n\t"
        "add.u32 x, %1, 24;\n\tadd.u32 y, %2, 384;\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, yes;\n\t"
        "add.u32 x, %1, 32;\n\tadd.u32 y, %2, 512;\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, yes;\n\t"
        "add.u32 x, %1, 40;\n\tadd.u32 y, %2, 640;\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, yes;\n\t"
        "add.u32 x, %1, 48;\n\tadd.u32 y, %2, 768;\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, yes;\n\t"
        "add.u32 x, %1, 56;\n\tadd.u32 y, %2, 896;\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, yes;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t"
        "setp.ne.and.b32 e, %7, 0, e;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(uint32_t(accumulate)), "r"(bar), "r"(bar2)
        : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
// The rest of a wait whose first look failed, out of line: the roles' registers are few.
__device__ __noinline__ bool wide_wait(uint32_t bar, uint32_t parity, volatile int* abort, long long limit, unsigned int* errors) {
    return tc_wait(bar, parity, abort, limit, errors);
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {  // completes at tmem_wait_ld
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A tile as warp 11 passes it on: units k0 .. k0 + nu of the rows r0 .. r0 + nrows of a sequence and kv head j.
struct WideTile {
    PagedSeq s;
    int j, r0, nrows, k0, nu, p0, p1;
    int whole, parts;  // one CTA has all of it; CTAs that share it when it begins here
    int ring;          // ring stages before it
    int seen;          // positions that every row sees (wide_seen)
    int valid;         // 0: the share has ended
};
constexpr int kTiles = 4;  // tiles on their way

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool full) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}

// Two fp32 values in a register pair: one instruction for both.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unf2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Eight fp32 values, 32-byte aligned: a row's lane writes whole sectors.
__device__ __forceinline__ void store8(float* dst, const float* v) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                 "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
                 : "memory");
}

// Positions that every row of a tile sees (one warp). The rows of a sequence see ascending
// numbers of positions. In the prefix pass, rows of many sequences, a row may see less of the
// prefix than the one before it: the least of all of them, but for rows that see nothing, of
// which the join takes nothing (mostly every row of the batch sees it all).
template <bool PREFIX>
__device__ __forceinline__ int wide_seen(const PagedWork& w, const PagedPrefix& prefix, const PagedSeq& s, int r0, int nrows, int lane) {
    if (!PREFIX) return paged_row_limit<PREFIX>(w, s, r0);
    if (prefix.seen >= prefix.len) return prefix.len;
    const int last = w.by_G(r0 + nrows - 1);
    int least = INT_MAX;
#pragma unroll 1
    for (int tok = w.by_G(r0) + lane; tok <= last; tok += 32) {
        const int limit = paged_row_limit<PREFIX>(w, s, tok * w.G);
        if (limit > 0) least = min(least, limit);
    }
    return __reduce_min_sync(0xffffffffu, least);
}

// Queries of half h of tile t into shared memory (one warp), in the
// 128-byte-swizzled K-major layout, arriving on `bar`. By TMA the box may reach
// into rows of other sequences or behind the last: those rows are not looked at.
template <typename E, int D>
__device__ __forceinline__ void wide_queries(const PagedWideParams& p, const WideTile& t, int h, int lane, uint32_t dst, uint32_t bar) {
    constexpr int CH = D / 8;
    const PagedWork& w = p.w;
    const int first = t.r0 + 128 * h;
    if (p.q_tma) {
        if (lane == 0) {
            mbar_arrive_expect_tx(bar, 128 * D * 2);
#pragma unroll
            for (int half = 0; half < D / 64; ++half)
                tma_load_3d(dst + half * (128 * 128), &p.qmap, half * 64, t.j * w.G, t.s.begin + w.by_G(first), bar);
        }
        __syncwarp();
        return;
    }
    const int ch = lane % CH, last = t.r0 + t.nrows - 1;
    const E* base = static_cast<const E*>(w.q) + t.j * w.G * D + ch * 8;
#pragma unroll 4
    for (int r = lane / CH; r < 128; r += 32 / CH) {
        const int rr = min(first + r, last), tok = w.by_G(rr);
        cp_async16_zfill(dst + (ch >> 3) * (128 * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4),
                         base + int64_t(t.s.begin + tok) * w.ldq + (rr - tok * w.G) * D, first + r <= last);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

template <bool PREFIX, typename E, int D>
__global__ void __launch_bounds__(kThreads, 1) paged_wide_kernel(const __grid_constant__ PagedWideParams p) {
    using SM = WideSmem<D>;
    constexpr int ST = SM::kStages, CH = D / 8;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ PagedPrefix s_prefix;
    __shared__ WideTile s_tile[kTiles];
    __shared__ volatile int s_bad[kTiles];  // n + 1: entries of v were cleared from tile n
    const uint32_t sraw = smem_u32(smem_raw), sb = (sraw + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (sb - sraw);
    const PagedWork& w = p.w;
    const PagedKV& kv = w.kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort = &s_abort;
    const long long lim = p.wait_cycles;
    // full / empty per ring stage; per half: queries staged, scores ready, probabilities written, second product
    // complete, queries used; scores read; per tile in s_tile: written, read by all eleven other warps
    const uint32_t bar_full = sb + SM::kBars, bar_empty = bar_full + 64, bar_q = bar_full + 128, bar_s = bar_full + 144,
                   bar_p = bar_full + 160, bar_pv = bar_full + 176, bar_read = bar_full + 192, bar_done = bar_full + 200,
                   bar_used = bar_full + 216, bar_tile = bar_full + 232, bar_free = bar_full + 264;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(bar_full + 8 * i, 1);
            mbar_init(bar_empty + 8 * i, 1);
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(bar_q + 8 * h, 1);
            mbar_init(bar_used + 8 * h, 1);
            mbar_init(bar_s + 8 * h, 1);
            mbar_init(bar_p + 8 * h, 4);  // an arrival per warp
            mbar_init(bar_pv + 8 * h, 1);
        }
        mbar_init(bar_read, 4);
        mbar_init(bar_done, 1);
        mbar_init(bar_done + 8, 1);
        for (int i = 0; i < kTiles; ++i) {
            s_bad[i] = 0;
            mbar_init(bar_tile + 8 * i, 1);
            mbar_init(bar_free + 8 * i, 11);
        }
        s_abort = 0;
        fence_barrier_init();
    }
    pdl_wait();  // before the tensor memory is taken: a kernel before this one may still need its own
    PagedCursor c = paged_find<PREFIX, kRows, kUnit, kWideOverhead, kThreads>(w, blockIdx.x, gridDim.x, s_prefix);
    if (warp == 9) tmem_alloc(smem_u32(&s_tmem), kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = s_tmem;  // scores at columns 0, probabilities of half h at 128 + 64 h, outputs at 256 + 128 h

    bool ok = true;
    // warp-wide; clears ok when the wait gave up (the softmax warps wait in line: a call would cost them registers)
    auto wait = [&](uint32_t bar, int phase) {
        if (!__all_sync(0xffffffffu, mbar_try_wait(bar, phase & 1)))
            ok = __all_sync(0xffffffffu, wide_wait(bar, phase & 1, abort, lim, kv.errors));
    };

    // The n-th tile of the share, and having read it.
    auto tile = [&](int n) -> const WideTile& { return s_tile[n % kTiles]; };
    auto release = [&](int n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_free + 8 * (n % kTiles));
    };

    if (warp < 8) {
        // ------------------------------------------------------------ softmax of one half
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int h = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
        const uint32_t t_p = lanes + 128 + 64 * h, t_o = lanes + 256 + 128 * h;
        int done_units = 0;  // units of this half (phases of bar_s, bar_p, bar_pv)
        for (int n = 0;; ++n) {
            ok = __all_sync(0xffffffffu, tc_wait(bar_tile + 8 * (n % kTiles), (n / kTiles) & 1, abort, lim, kv.errors));
            if (!ok) break;
            const WideTile& t = tile(n);
            if (!t.valid) break;
            const int hrows = t.nrows - 128 * h;  // valid rows of this half
            if (hrows <= 0) {
                release(n);
                continue;
            }
            const int myrow = t.r0 + 128 * h + row, units = t.nu, p0 = t.p0, p1 = t.p1;
            const bool idle = (warp & 3) * 32 >= hrows;  // no row of this warp exists
            const int limit = row < hrows ? paged_row_limit<PREFIX>(w, t.s, myrow) : 0;
            const int seen = t.seen;
            float mref = -INFINITY, l = 0.f;
            __syncwarp();  // tensor-memory instructions below are warp-wide
            for (int u = 0; u < units; ++u) {
                ok = __all_sync(0xffffffffu, tc_wait(bar_s + 8 * h, done_units & 1, abort, lim, kv.errors));
                if (!ok) break;
                tc_fence_after();
                const int base = p0 + u * kUnit;
                float s[128];
                if (!idle) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) tmem_ld32(lanes + 32 * q, s + 32 * q);
                    tmem_wait_ld();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_read);  // the score buffer may be written again
                if (!idle && base + kUnit > limit) {
                    const int sees = limit - base;
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = i < sees ? s[i] : -INFINITY;
                }
                if (!idle && u == 0) {  // the tile's first reference
                    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int i = 4; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
                    mref = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * w.scale_log2;
                }
                __syncwarp();
                // A warp without rows arrives with the others all the same, and never a unit ahead of them: it, too, waits
                // for the product before (its early arrival would count as another warp's).
                if (idle && u > 0) ok = __all_sync(0xffffffffu, tc_wait(bar_pv + 8 * h, (done_units - 1) & 1, abort, lim, kv.errors));
                if (!ok) break;
                // Probabilities against the reference as it stands, and the maximum beside them; only where a
                // maximum turns out to have moved by more than the allowance are they computed once more.
                bool again = !idle, first = u > 0;
                while (again) {
                    const float off = mref == -INFINITY ? 0.f : -mref;
                    const uint64_t sc2 = f2(w.scale_log2, w.scale_log2), off2 = f2(off, off);
                    uint64_t sum[2] = {0, 0};
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    // The first kHeld quarters wait in registers for the product before, which still reads its probabilities.
                    constexpr int kHeld = 2;
                    uint32_t held[kHeld][16], now[16];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t(&pk)[16] = q < kHeld ? held[q < kHeld ? q : 0] : now;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float x = s[32 * q + 2 * i], y = s[32 * q + 2 * i + 1];
                            mx[i & 3] = max3(mx[i & 3], x, y);
                            float a, b;
                            unf2(fma2(f2(x, y), sc2, off2), a, b);
                            a = ex2(a);
                            b = ex2(b);
                            sum[i & 1] = add2(sum[i & 1], f2(a, b));
                            pk[i] = pack2<E>(a, b);
                        }
                        if (q == kHeld - 1 && first) {  // it has read its probabilities and written its outputs
                            ok = __all_sync(0xffffffffu, tc_wait(bar_pv + 8 * h, (done_units - 1) & 1, abort, lim, kv.errors));
                            if (!ok) break;
                            tc_fence_after();
                            first = false;
                        }
                        if (q == kHeld - 1) {
#pragma unroll
                            for (int e = 0; e < kHeld; ++e) tmem_st16(t_p + 16 * e, held[e]);
                        } else if (q >= kHeld) {
                            tmem_st16(t_p + 16 * q, now);
                        }
                    }
                    if (!ok) break;
                    const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * w.scale_log2;
                    const bool move = m > mref + 8.f;  // also the first finite maximum
                    again = __any_sync(0xffffffffu, move);
                    if (again) {
                        tmem_wait_st();  // the probabilities are about to be written again, and stores have no order of their own
                        const float f = move ? ex2(mref - m) : 1.f;
                        mref = move ? m : mref;
                        l *= f;
                        if (u > 0) {
#pragma unroll 1
                            for (int q = 0; q < D / 16; ++q) {
                                float o[16];
                                tmem_ld16(t_o + 16 * q, o);
                                uint32_t o2[16];
#pragma unroll
                                for (int i = 0; i < 16; ++i) o2[i] = __float_as_uint(o[i] * f);
                                tmem_st16(t_o + 16 * q, o2);
                            }
                        }
                    } else {
                        float l0, l1;
                        unf2(add2(sum[0], sum[1]), l0, l1);
                        l += l0 + l1;
                        tmem_wait_st();
                    }
                }
                if (!ok) break;
                if (h == 0 && base + kUnit > min(p1, seen)) {  // rows of v that no position owns, or not every row sees
                    const int ring = t.ring + 2 * u + 1, st = ring % ST, from = max(0, p1 - base);
                    ok = __all_sync(0xffffffffu, tc_wait(bar_full + 8 * st, (ring / ST) & 1, abort, lim, kv.errors));
                    if (!ok) break;
                    const int some = max(0, min(from, seen - base));
#pragma unroll 1
                    for (int idx = row; idx < (128 - some) * CH; idx += 128) {
                        const int r = some + idx / CH, ch = idx % CH;
                        uint4* at = reinterpret_cast<uint4*>(smem + SM::kRing + st * SM::kTile + (ch >> 3) * (128 * 128) + r * 128 +
                                                             ((ch & 7) << 4));
                        if (r >= from) {
                            *at = make_uint4(0, 0, 0, 0);
                        } else {
                            const uint4 x = *at;
                            const uint4 bad = make_uint4(nonfinite2<E>(x.x), nonfinite2<E>(x.y), nonfinite2<E>(x.z), nonfinite2<E>(x.w));
                            if (bad.x | bad.y | bad.z | bad.w) {
                                *at = make_uint4(x.x & ~bad.x, x.y & ~bad.y, x.z & ~bad.z, x.w & ~bad.w);
                                s_bad[n % kTiles] = n + 1;
                            }
                        }
                    }
                    fence_async_smem();
                    __syncwarp();
                }
                ++done_units;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_p + 8 * h);
            }
            if (!ok) break;
            ok = __all_sync(0xffffffffu, tc_wait(bar_pv + 8 * h, (done_units - 1) & 1, abort, lim, kv.errors));
            if (!ok) break;
            tc_fence_after();
            if (!idle) {
                const bool whole = t.whole, final = whole && !w.row_o;
                const int tok = w.by_G(myrow), head = t.j * w.G + myrow - tok * w.G;
                const int64_t orow = t.s.begin + tok;
                const int64_t at = whole ? orow * kv.HQ + head
                                         : int64_t(2 * blockIdx.x + (t.k0 == 0 ? 1 : 0)) * kRows + 128 * h + row;
                if (l == 0.f && min(limit, p1) > p0) mref = kLowest;  // no score but -inf
                const float inv = paged_inverse(mref, l);
#pragma unroll
                for (int q = 0; q < D / 32; ++q) {
                    float o[32];
                    __syncwarp();
                    tmem_ld32(t_o + 32 * q, o);
                    tmem_wait_ld();
                    if (row < hrows && final) {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<E*>(w.out) + orow * w.ldo + head * D + 32 * q);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            dst[i] = make_uint4(pack2<E>(o[8 * i] * inv, o[8 * i + 1] * inv), pack2<E>(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                                pack2<E>(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack2<E>(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                    } else if (row < hrows) {
                        float* dst = (whole ? w.row_o : w.part_o) + at * D + 32 * q;
#pragma unroll
                        for (int i = 0; i < 4; ++i) store8(dst + 8 * i, o + 8 * i);
                    }
                }
                if (row < hrows) {
                    if (!final) {
                        (whole ? w.row_ml : w.part_ml)[at] = make_float2(mref, l);
                        if (w.row_at && t.k0 == 0)
                            w.row_at[orow * kv.HQ + head] = paged_row_at(blockIdx.x, t.parts, 128 * h + row);
                    } else if (w.lse) {
                        w.lse[orow * w.ldl + head] = l != 0.f ? (mref + log2f(l)) * kLn2 : -INFINITY;
                    }
                }
            }
            if (s_bad[n % kTiles] == n + 1 && row < hrows) {
                const int tok = w.by_G(myrow), head = t.j * w.G + myrow - tok * w.G;
                const int64_t orow = t.s.begin + tok;
                const bool final = t.whole && !w.row_o;
                const int64_t at = t.whole ? orow * kv.HQ + head
                                           : int64_t(2 * blockIdx.x + (t.k0 == 0 ? 1 : 0)) * kRows + 128 * h + row;
                bool page_ok = true;
#pragma unroll 1
                for (int pos = max(p0, seen); pos < min(p1, limit); ++pos) {
                    const E* v = static_cast<const E*>(kv.v) + paged_page(kv, t.s.table, pos, page_ok) * kv.vs_page + t.j * kv.vs_head +
                                 int64_t(pos & kv.page_mask) * kv.vs_slot;
#pragma unroll 1
                    for (int d = 0; d < D; d += 2) {
                        const uint32_t x = *reinterpret_cast<const uint32_t*>(v + d);
                        float a, b;
                        unpack2<E>(x & nonfinite2<E>(x), a, b);
                        if (final) {
                            uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<E*>(w.out) + orow * w.ldo + head * D + d);
                            float oa, ob;
                            unpack2<E>(*o, oa, ob);
                            *o = pack2<E>(oa + a, ob + b);
                        } else {
                            float* o = (t.whole ? w.row_o : w.part_o) + at * D + d;
                            o[0] += a;
                            o[1] += b;
                        }
                    }
                }
            }
            __syncwarp();
            tc_fence_before();  // ordered before the next tile's first product by its bar_p arrivals
            release(n);
        }
    } else {
        // One instruction for the whole warpgroup, under a condition that its warps share: executed from different
        // places by its warps, it would be undefined.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 8) {
            // -------------------------------------------------------- k / v loads
            int it = 0;
            bool pages_ok = true;
            for (int n = 0;; ++n) {
                wait(bar_tile + 8 * (n % kTiles), n / kTiles);
                if (!ok || !tile(n).valid) break;
                const int units = tile(n).nu, p0 = tile(n).p0, p1 = tile(n).p1, seq = tile(n).s.table, j = tile(n).j;
                release(n);
                for (int u = 0; ok && u < units; ++u) {
                    const int base = p0 + u * kUnit;
                    const int nb = max(0, (min(kUnit, p1 - base) + p.box - 1) / p.box);  // boxes that hold positions
                    int page = 0;
                    if (lane < nb) page = paged_page(kv, seq, base + lane * p.box, pages_ok);
                    const int slot = (base + lane * p.box) & kv.page_mask;
    #pragma unroll
                    for (int x = 0; x < 2; ++x, ++it) {
                        const int st = it % ST;
                        const uint32_t bar = bar_full + 8 * st;
                        if (it >= ST) wait(bar_empty + 8 * st, it / ST + 1);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(bar, uint32_t(nb * p.box) * (D * 2));
                        __syncwarp();
                        if (lane < nb) {
                            const CUtensorMap* map = x ? &p.vmap : &p.kmap;
                            const int ps = x ? p.v_slot : p.k_slot, ph = x ? p.v_head : p.k_head;
                            const int c1 = ps == 1 ? slot : ph == 1 ? j : page, c2 = ps == 2 ? slot : ph == 2 ? j : page,
                                      c3 = ps == 3 ? slot : ph == 3 ? j : page;
                            const uint32_t dst = sb + SM::kRing + st * SM::kTile + uint32_t(lane * p.box) * 128u;
    #pragma unroll
                            for (int half = 0; half < D / 64; ++half)
                                tma_load_4d(dst + half * (128 * 128), map, half * 64, c1, c2, c3, bar);
                        }
                    }
                }
            }
            if (!pages_ok) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
            // no tile may still be landing when the CTA leaves (an abort skips the products)
            for (int i = max(0, it - ST); i < it; ++i) tc_wait(bar_full + 8 * (i % ST), (i / ST) & 1, nullptr, lim, kv.errors);
            __syncwarp();
        } else {
            // -------------------------------------------------------- products
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            if (warp == 9) {
                int tiles0 = 0, tiles1 = 0, scored = 0;  // tiles of each half, score tiles so far
                for (int n = 0;; ++n) {
                    wait(bar_tile + 8 * (n % kTiles), n / kTiles);
                    if (!ok || !tile(n).valid) break;
                    const int both = __shfl_sync(0xffffffffu, tile(n).nrows > 128 ? 1 : 0, 0);
                    const int nu = __shfl_sync(0xffffffffu, tile(n).nu, 0), it = __shfl_sync(0xffffffffu, tile(n).ring, 0);
                    release(n);
                    wait(bar_q, tiles0++);
                    if (ok && both) wait(bar_q + 8, tiles1++);
                    for (int u = 0; ok && u < nu; ++u) {
                        const int ring = it + 2 * u, st = ring % ST;
                        const uint32_t k_lo = ((sb + SM::kRing + st * SM::kTile) >> 4) | kDescLoK;
                        wait(bar_full + 8 * st, ring / ST);
                        for (int h = 0; ok && h <= both; ++h, ++scored) {
                            if (scored > 0) wait(bar_read, scored - 1);
                            if (!ok) break;
                            tc_fence_after();
                            scores_product<D>(tm, ((sb + h * SM::kTile) >> 4) | kDescLoK, k_lo, p.idesc_qk, bar_s + 8 * h,
                                              h == both ? bar_empty + 8 * st : 0u);
                            if (u + 1 == nu && elect_one()) tc_commit(bar_used + 8 * h);
                            __syncwarp();
                        }
                    }
                    if (!ok) break;
                }
            } else if (warp == 10) {
                int units0 = 0, units1 = 0;  // units of each half before the tile
                for (int n = 0;; ++n) {
                    wait(bar_tile + 8 * (n % kTiles), n / kTiles);
                    if (!ok || !tile(n).valid) break;
                    const int both = __shfl_sync(0xffffffffu, tile(n).nrows > 128 ? 1 : 0, 0);
                    const int nu = __shfl_sync(0xffffffffu, tile(n).nu, 0), it = __shfl_sync(0xffffffffu, tile(n).ring, 0);
                    release(n);
                    for (int u = 0; ok && u < nu; ++u) {
                        const int ring = it + 2 * u + 1, st = ring % ST;
                        const uint32_t v_lo = ((sb + SM::kRing + st * SM::kTile) >> 4) | kDescLoV;
                        wait(bar_full + 8 * st, ring / ST);
                        for (int h = 0; ok && h <= both; ++h) {
                            wait(bar_p + 8 * h, (h ? units1 : units0) + u);
                            if (!ok) break;
                            tc_fence_after();
                            output_product(tm + 256 + 128 * h, tm + 128 + 64 * h, v_lo, p.idesc_pv, u > 0, bar_pv + 8 * h,
                                           h == both ? bar_empty + 8 * st : 0u);
                        }
                    }
                    if (!ok) break;
                    units0 += nu;
                    units1 += both ? nu : 0;
                }
            } else {
                // -------------------------------------------------------- tiles and queries
                int used0 = 0, used1 = 0, ring = 0;  // tiles of each half, ring stages so far
                bool shares = false;                 // the last tile goes on in the next CTA
                const int sequences = PREFIX ? 1 : kv.B;
                for (int n = 0; ok; ++n) {
                    if (n >= kTiles) wait(bar_free + 8 * (n % kTiles), n / kTiles - 1);
                    if (!ok) break;
                    WideTile t;
                    t.valid = 0;
                    while (c.u < c.hi && c.b < sequences) {  // past tiles of which this share holds only overhead
                        bool cut;
                        t.s = paged_seq<PREFIX>(w, s_prefix, c.b, cut);
                        const PagedSegment<PREFIX, kRows, kUnit, kWideOverhead> g(w, t.s, c);
                        if (g.nu > 0) {
                                t.j = c.j;
                            t.r0 = c.i * kRows;
                            t.nrows = min(kRows, t.s.rows - t.r0);
                            t.k0 = g.k0;
                            t.nu = g.nu;
                            t.p0 = (PREFIX ? 0 : w.prefix_len) + g.k0 * kUnit;
                            t.p1 = min(t.p0 + g.nu * kUnit, paged_tile_limit<PREFIX, kRows>(w, t.s, c.i));
                            t.whole = g.whole();
                            t.parts = g.parts(c, blockIdx.x);
                            t.ring = ring;
                            t.seen = wide_seen<PREFIX>(w, s_prefix, t.s, t.r0, t.nrows, lane);
                            t.valid = 1;
                            paged_next<PREFIX, kRows>(w, s_prefix, c, g.cost);
                            break;
                        }
                        paged_next<PREFIX, kRows>(w, s_prefix, c, g.cost);
                    }
                    if (lane == 0) {
                        s_tile[n % kTiles] = t;
                        mbar_arrive(bar_tile + 8 * (n % kTiles));
                    }
                    __syncwarp();
                    if (!t.valid) break;
                    ring += 2 * t.nu;
                    if (t.parts) {
                        shares = true;
                        if (lane == 0) w.shared[blockIdx.x] = PagedShared{t.parts, t.nrows, t.r0, t.s.begin, t.j};
                    }
                    for (int h = 0; ok && h <= (t.nrows > 128 ? 1 : 0); ++h) {
                        int& used = h ? used1 : used0;
                        if (used > 0) wait(bar_used + 8 * h, used - 1);  // the tile before it has been multiplied
                        if (!ok) break;
                        wide_queries<E, D>(p, t, h, lane, sb + h * SM::kTile, bar_q + 8 * h);
                        ++used;
                    }
                }
                if (lane == 0 && !shares) w.shared[blockIdx.x].parts = 0;
                // no queries may still be landing when the CTA leaves
                if (used0 > 0) tc_wait(bar_q, (used0 - 1) & 1, nullptr, lim, kv.errors);
                if (used1 > 0) tc_wait(bar_q + 8, (used1 - 1) & 1, nullptr, lim, kv.errors);
                __syncwarp();
            }
            if (warp <= 10) {  // every product issued above has finished once this completes
                const uint32_t done = bar_done + 8 * (warp - 9);
                if (elect_one()) tc_commit(done);
                __syncwarp();
                tc_wait(done, 0, nullptr, lim, kv.errors);
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_dealloc(tmem, kCols);
}

// Tensor map of pages (element strides st: page, head, slot): dims are D, then
// the other three in order of their strides; `slot` and `head` receive the
// coordinate (1 .. 3) of each.
int encode_pages(const bq_paged_kv* kv, const void* base, const int64_t* st, int box, CUtensorMap* map, int32_t* slot,
                 int32_t* head) {
    EncodeTiledFn enc = tensor_map_encoder();
    if (!enc) return set_error(BQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    struct Dim {
        int64_t stride, size;
        int what;  // 0 page, 1 head, 2 slot
    } d[3] = {{st[0], kv->num_pages, 0}, {st[1], kv->HKV, 1}, {st[2], kv->page_size, 2}};
    std::stable_sort(d, d + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    cuuint64_t dims[4] = {cuuint64_t(kv->D)}, strides[3];
    cuuint32_t boxes[4] = {64};
    const cuuint32_t es[4] = {1, 1, 1, 1};
    for (int i = 0; i < 3; ++i) {
        dims[i + 1] = cuuint64_t(d[i].size);
        strides[i] = cuuint64_t(d[i].size == 1 ? kv->D : d[i].stride) * 2;  // of one element: any that the encoder takes
        boxes[i + 1] = d[i].what == 2 ? cuuint32_t(box) : 1u;
        if (d[i].what == 2) *slot = i + 1;
        if (d[i].what == 1) *head = i + 1;
    }
    const CUresult r = enc(map, kv->dtype == BQ_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                           const_cast<void*>(base), dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(BQ_ERR_CUDA, "cuTensorMapEncodeTiled (pages) failed (%d)", int(r));
    return BQ_OK;
}

// Tensor map of the query rows, (D, heads, rows): a box is 64 dims of the G heads of
// a kv head and of 128 / G tokens, which are 128 rows of a tile in their order.
int encode_queries(const PagedWork& w, const bq_paged_kv* kv, CUtensorMap* map) {
    EncodeTiledFn enc = tensor_map_encoder();
    if (!enc) return set_error(BQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[3] = {cuuint64_t(kv->D), cuuint64_t(w.kv.HQ), cuuint64_t(w.kv.T)};
    const cuuint64_t strides[2] = {cuuint64_t(kv->D) * 2, cuuint64_t(w.ldq) * 2};
    const cuuint32_t box[3] = {64, cuuint32_t(w.G), cuuint32_t(128 / w.G)};
    const cuuint32_t es[3] = {1, 1, 1};
    const CUresult r = enc(map, kv->dtype == BQ_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                           const_cast<void*>(w.q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(BQ_ERR_CUDA, "cuTensorMapEncodeTiled (queries) failed (%d)", int(r));
    return BQ_OK;
}

template <bool PREFIX>
const void* wide_kernel(int dtype, int D) {
    return D == 128 ? (dtype == BQ_DT_BF16 ? reinterpret_cast<const void*>(&paged_wide_kernel<PREFIX, __nv_bfloat16, 128>)
                                           : reinterpret_cast<const void*>(&paged_wide_kernel<PREFIX, __half, 128>))
                    : (dtype == BQ_DT_BF16 ? reinterpret_cast<const void*>(&paged_wide_kernel<PREFIX, __nv_bfloat16, 64>)
                                           : reinterpret_cast<const void*>(&paged_wide_kernel<PREFIX, __half, 64>));
}

}  // namespace

int paged_launch_wide(const PagedWork& w, const bq_paged_kv* kv, int grid, uint32_t flags, void* stream) {
    PagedWideParams p;
    std::memset(&p, 0, sizeof(p));
    p.w = w;
    p.box = std::min(kv->page_size, 128);
    int rc = encode_pages(kv, kv->k_pages, kv->k_stride, p.box, &p.kmap, &p.k_slot, &p.k_head);
    if (!rc) rc = encode_pages(kv, kv->v_pages, kv->v_stride, p.box, &p.vmap, &p.v_slot, &p.v_head);
    if (rc) return rc;
    if (128 % w.G == 0) {
        rc = encode_queries(w, kv, &p.qmap);
        if (rc) return rc;
        p.q_tma = 1;
    }
    // kind::f16, fp32 accumulate; A and B of the pages' type; M = 128; N = 128 positions / D dims (B dims-contiguous)
    const uint32_t type = kv->dtype == BQ_DT_BF16 ? 1u : 0u;
    const uint32_t common = (1u << 4) | (type << 7) | (type << 10) | (uint32_t(128 >> 4) << 24);
    p.idesc_qk = common | (uint32_t(128 >> 3) << 17);
    p.idesc_pv = common | (1u << 16) | (uint32_t(kv->D >> 3) << 17);
    p.wait_cycles = kWaitCycles;
    const void* fn = w.prefix_pass ? wide_kernel<true>(kv->dtype, kv->D) : wide_kernel<false>(kv->dtype, kv->D);
    const uint32_t smem = kv->D == 128 ? WideSmem<128>::kTotal : WideSmem<64>::kTotal;
    rc = ensure_smem_attr(fn, smem);
    if (rc) return rc;
    void* args[] = {&p};
    return paged_launch(fn, dim3(grid), dim3(kThreads), smem, args, flags, stream, "paged attention");
}

}  // namespace bq
