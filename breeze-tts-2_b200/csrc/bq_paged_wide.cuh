// Shared pieces of the attention kernels for tiles of many rows (bq_paged_wide.cu,
// bq_paged8_wide.cu): the products on the tcgen05 tensor cores and the queries' way
// into shared memory. Both are compiled as whole programs.
#pragma once

#include <algorithm>
#include <climits>
#include <cstring>

#include "bq_host.h"
#include "bq_paged.cuh"
#include "bq_paged_host.h"
#include "bq_tmem.cuh"

namespace bq {
namespace {

constexpr int kRows = kWideRows, kUnit = kWideUnit;
constexpr uint32_t kCols = 512;

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

// Queries of half h of tile t into shared memory (one warp), in the
// 128-byte-swizzled K-major layout, arriving on `bar`. By TMA the box may reach
// into rows of other sequences or behind the last: those rows are not looked at.
template <typename E, int D>
__device__ __forceinline__ void wide_queries(const PagedWork& w, const CUtensorMap* qmap, bool by_tma, const WideTile& t, int h, int lane,
                                             uint32_t dst, uint32_t bar) {
    constexpr int CH = D / 8;
    const int first = t.r0 + 128 * h;
    if (by_tma) {
        if (lane == 0) {
            mbar_arrive_expect_tx(bar, 128 * D * 2);
#pragma unroll
            for (int half = 0; half < D / 64; ++half)
                tma_load_3d(dst + half * (128 * 128), qmap, half * 64, t.j * w.G, t.s.begin + w.by_G(first), bar);
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

// Tensor map of the query rows, (D, heads, rows): a box is 64 dims of the G heads of
// a kv head and of 128 / G tokens, which are 128 rows of a tile in their order.
int encode_queries(const PagedWork& w, int dtype, int D, CUtensorMap* map) {
    EncodeTiledFn enc = tensor_map_encoder();
    if (!enc) return set_error(BQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(w.kv.HQ), cuuint64_t(w.kv.T)};
    const cuuint64_t strides[2] = {cuuint64_t(D) * 2, cuuint64_t(w.ldq) * 2};
    const cuuint32_t box[3] = {64, cuuint32_t(w.G), cuuint32_t(128 / w.G)};
    const cuuint32_t es[3] = {1, 1, 1};
    const CUresult r = enc(map, dtype == BQ_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                           const_cast<void*>(w.q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(BQ_ERR_CUDA, "cuTensorMapEncodeTiled (queries) failed (%d)", int(r));
    return BQ_OK;
}

}  // namespace
}  // namespace bq
