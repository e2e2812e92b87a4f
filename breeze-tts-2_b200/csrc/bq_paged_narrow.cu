// Paged attention for tiles of at most 16 rows (a decode step, a few drafted
// tokens): one pass over the cached keys and values with a running maximum and
// sum, on mma.sync m16n8k16 tiles.
//
// Bound: HBM. Every cached row is read once per 16 query rows that share its
// kv head, 4 flops per element and row, far under what the tensor cores need
// to be busy; what counts is bytes in flight. Four warps per CTA take every
// fourth block of 16 positions of the CTA's share, each through a ring of its
// own (cp.async, 8 KB of k and v per stage, no barrier between warps), so two
// CTAs per SM keep 128 KB of loads in flight. Blocks of 16 never straddle a
// page. Rows of a page are stored 16-byte chunk ^ (row & 7), so that the
// ldmatrix reads of eight rows fall on different banks. Positions behind the
// share are zero-filled by the copy (0 bytes read): what lies behind a
// sequence's last position, NaN or not, never enters a product. Where some rows
// see a position and others do not, its probabilities are zero for the latter, but
// zero times an infinite or NaN v is NaN: such entries are taken out of the product
// and added to the rows that see them (narrow_nonfinite).
//
// Scores, statistics and outputs are fp32; the probabilities are rounded to the
// element type for the second product (relative error of half a step of that
// type each, as the values they weight). Over long caches that is the larger part
// of what the result is off: 0.0020 of its size in bf16 where probabilities in fp32
// leave 0.0017, the output's own rounding.
//
// Measured, join included (B200, copies run at 6554 GB/s): 8 sequences of 24 to 32
// thousand positions, 8 kv heads of 128, 881 MB in 145 to 150 us (6.0 TB/s); 48 of 17 to
// 6000, 184 MB in 39 us (4.7 TB/s), where finding the shares (2 us), each tile's
// start and end and the join (5 us) show. The shares are equal, the SMs' speeds are
// not: on average an SM is done after 87 % of the time. Two, four and eight times
// as many smaller shares, dealt out as CTAs end, cost more in starts than they
// gain (158, 160, 174 us against then 156); fetching the next tile's first 128 positions into L2
// meanwhile changes nothing (43 / 42 us).
#include "bq_host.h"
#include "bq_paged.cuh"
#include "bq_paged_host.h"

namespace bq {
namespace {

constexpr int kThreads = 32 * kNarrowWarps;
constexpr int kMaxRanks = kNarrowRanks;

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool full) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void lds128(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename E>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16(c, a[0], a[1], a[2], a[3], b0, b1);
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_f16(c, a[0], a[1], a[2], a[3], b0, b1);
}

// Shared memory: per warp a ring of kStages (k block, v block), then the query tile.
// After a tile's positions the rings hold the warps' outputs (fp32, rows padded by 8).
template <int D>
struct NarrowSmem {
    static constexpr int kBlock = 16 * D * 2;                      // bytes of 16 rows
    static constexpr int kStages = D == 128 ? 3 : 6;               // 24 KB of ring per warp
    static constexpr int kRing = kStages * 2 * kBlock;             // per warp
    static constexpr int kQ = kNarrowWarps * kRing;                // offset of the query tile
    static constexpr int kTotal = kQ + kBlock;
    static constexpr int kPitch = D + 8;                           // floats per output row
    static_assert(kNarrowWarps * 16 * kPitch * 4 <= kQ, "the warps' outputs fit the rings");
};

// Positions [p0, p1) of rows r0 .. r0 + nrows of a sequence and kv head j.
struct NarrowTile {
    PagedSeq s;
    int j, r0, nrows, p0, p1;
};

// Infinite and NaN entries of the v block at vb (positions pb .. pb + 15): added to
// the outputs of the rows that see their position, then cleared. A warp calls it.
template <typename E, int D>
__device__ __forceinline__ void narrow_nonfinite(uint32_t vb, int pb, int lim0, int lim1, float (&o)[D / 8][4]) {
    constexpr int CH = D / 8;
    const int lane = threadIdx.x & 31;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 16 * CH / 32; ++i) {
        uint32_t x[4];
        lds128(x, vb + (lane + 32 * i) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= nonfinite2<E>(x[e]);
    }
    if (!__any_sync(0xffffffffu, bad)) return;
#pragma unroll 1
    for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int n = 0; n < CH; ++n) {
            uint32_t x;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(vb + r * (D * 2) + ((n ^ (r & 7)) << 4) + (lane & 3) * 4));
            float a, b;
            unpack2<E>(x & nonfinite2<E>(x), a, b);  // 0 for the finite ones
            if (pb + r < lim0) o[n][0] += a, o[n][1] += b;
            if (pb + r < lim1) o[n][2] += a, o[n][3] += b;
        }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16 * CH / 32; ++i) {
        uint32_t x[4];
        lds128(x, vb + (lane + 32 * i) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] &= ~nonfinite2<E>(x[e]);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(vb + (lane + 32 * i) * 16), "r"(x[0]), "r"(x[1]), "r"(x[2]),
                     "r"(x[3])
                     : "memory");
    }
    __syncwarp();
}

// One tile with the whole CTA: emit(r, d, m, l, o) receives dims d .. d + 3 of row r,
// unnormalized, with the row's largest score (base 2) and sum of exponentials.
template <bool PREFIX, typename E, int D, typename Emit>
__device__ __forceinline__ void narrow_tile(const PagedWork& p, const NarrowTile& t, unsigned char* smem, int* s_lim,
                                            float2 (*s_ml)[kNarrowRows], const Emit& emit) {
    using SM = NarrowSmem<D>;
    constexpr int ROWS = kNarrowRows, CH = D / 8, ST = SM::kStages;
    const uint32_t sb = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const PagedKV& kv = p.kv;
    const uint32_t ring = sb + warp * SM::kRing;
    const PagedSeq& s = t.s;
    const int p0 = t.p0, p1 = t.p1, r0 = t.r0, nrows = t.nrows;
    bool pages_ok = true;
    const int blocks = max(0, (p1 - p0 + 15) >> 4);
    const int steps = (blocks - warp + kNarrowWarps - 1) / kNarrowWarps;
    const E* kh = static_cast<const E*>(kv.k) + t.j * kv.ks_head;
    const E* vh = static_cast<const E*>(kv.v) + t.j * kv.vs_head;

    // query tile: row r0 + r is head j G + (r0 + r) % G of token (r0 + r) / G
    for (int idx = threadIdx.x; idx < ROWS * CH; idx += kThreads) {
        const int r = idx / CH, ch = idx - r * CH, rr = r0 + min(r, nrows - 1), tok = p.by_G(rr);
        const E* src = static_cast<const E*>(p.q) + int64_t(s.begin + tok) * p.ldq + (t.j * p.G + rr - tok * p.G) * D + ch * 8;
        cp_async16_zfill(sb + SM::kQ + r * (D * 2) + ((ch ^ (r & 7)) << 4), src, r < nrows);
    }
    cp_commit();

    int pages = 0;  // lane i: page of the warp's step (32 n + i)
    auto issue = [&](int st) {
        if ((st & 31) == 0) {
            const int mine = st + lane;
            pages = mine < steps ? paged_page(kv, s.table, p0 + 16 * (warp + kNarrowWarps * mine), pages_ok) : 0;
        }
        const int page = __shfl_sync(0xffffffffu, pages, st & 31);
        if (st < steps) {
            const int pb = p0 + 16 * (warp + kNarrowWarps * st), slot = pb & kv.page_mask;
            const E* kp = kh + page * kv.ks_page + slot * kv.ks_slot;
            const E* vp = vh + page * kv.vs_page + slot * kv.vs_slot;
            const uint32_t dst = ring + (st % ST) * (2 * SM::kBlock);
#pragma unroll
            for (int i = 0; i < 16 * CH / 32; ++i) {
                const int idx = lane + 32 * i, r = idx / CH, ch = idx % CH;
                const uint32_t at = r * (D * 2) + ((ch ^ (r & 7)) << 4);
                cp_async16_zfill(dst + at, kp + r * kv.ks_slot + ch * 8, pb + r < p1);
                cp_async16_zfill(dst + SM::kBlock + at, vp + r * kv.vs_slot + ch * 8, pb + r < p1);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int st = 0; st < ST - 1; ++st) issue(st);
    if (threadIdx.x < ROWS) s_lim[threadIdx.x] = int(threadIdx.x) < nrows ? paged_row_limit<PREFIX>(p, s, r0 + threadIdx.x) : 0;
    cp_wait<ST - 1>();  // the query tile
    __syncthreads();
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        const int r = (lane & 7) + (lane & 8), ch = 2 * ks + (lane >> 4);
        ldsm4(qf[ks], sb + SM::kQ + r * (D * 2) + ((ch ^ (r & 7)) << 4));
    }
    const int lim0 = s_lim[g], lim1 = s_lim[g + 8];
    const int seen = __reduce_min_sync(0xffffffffu, min(g < nrows ? lim0 : p1, g + 8 < nrows ? lim1 : p1));  // by every row
    float o[D / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    for (int st = 0; st < steps; ++st) {
        cp_wait<ST - 2>();
        __syncwarp();  // every lane's copies of this stage have landed, and every lane is done with the one before
        issue(st + ST - 1);
        const uint32_t kb = ring + (st % ST) * (2 * SM::kBlock), vb = kb + SM::kBlock;
        float sc[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t bf[4];
            const int r = (lane & 7) + ((lane >> 4) << 3), ch = 2 * ks + ((lane >> 3) & 1);
            ldsm4(bf, kb + r * (D * 2) + ((ch ^ (r & 7)) << 4));
            mma<E>(sc[0], qf[ks], bf[0], bf[1]);
            mma<E>(sc[1], qf[ks], bf[2], bf[3]);
        }
        const int pb = p0 + 16 * (warp + kNarrowWarps * st) + 2 * tq;
        float n0 = m0, n1 = m1;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int pos = pb + 8 * n + e;
                sc[n][e] = pos < lim0 ? sc[n][e] * p.scale_log2 : -INFINITY;
                sc[n][2 + e] = pos < lim1 ? sc[n][2 + e] * p.scale_log2 : -INFINITY;
                n0 = fmaxf(n0, sc[n][e]);
                n1 = fmaxf(n1, sc[n][2 + e]);
            }
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 1));
        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 1));
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 2));
        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 2));
        if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {  // a maximum moved: rescale what was summed
            const float a0 = n0 == m0 ? 1.f : ex2(m0 - n0), a1 = n1 == m1 ? 1.f : ex2(m1 - n1);
            l0 *= a0;
            l1 *= a1;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
                o[n][0] *= a0;
                o[n][1] *= a0;
                o[n][2] *= a1;
                o[n][3] *= a1;
            }
            m0 = n0;
            m1 = n1;
        }
        const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;  // rows that see nothing yet
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sc[n][e] = ex2(sc[n][e] - u0);
                sc[n][2 + e] = ex2(sc[n][2 + e] - u1);
                l0 += sc[n][e];
                l1 += sc[n][2 + e];
            }
        const int blk = p0 + 16 * (warp + kNarrowWarps * st);
        if (min(blk + 16, p1) > seen) narrow_nonfinite<E, D>(vb, blk, lim0, lim1, o);
        const uint32_t pf[4] = {pack2<E>(sc[0][0], sc[0][1]), pack2<E>(sc[0][2], sc[0][3]),
                                pack2<E>(sc[1][0], sc[1][1]), pack2<E>(sc[1][2], sc[1][3])};
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
            uint32_t bf[4];
            const int r = (lane & 7) + (lane & 8), ch = 2 * dt + (lane >> 4);
            ldsm4t(bf, vb + r * (D * 2) + ((ch ^ (r & 7)) << 4));
            mma<E>(o[2 * dt], pf, bf[0], bf[1]);
            mma<E>(o[2 * dt + 1], pf, bf[2], bf[3]);
        }
    }
    cp_wait<0>();
    if (!pages_ok) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    __syncthreads();  // every warp is done with its ring: it now takes the warps' outputs
    float* red = reinterpret_cast<float*>(smem);
    if (g < nrows) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(red + (warp * 16 + g) * SM::kPitch + 8 * n + 2 * tq) = make_float2(o[n][0], o[n][1]);
        if (tq == 0) s_ml[warp][g] = make_float2(m0, l0);
    }
    if (g + 8 < nrows) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(red + (warp * 16 + g + 8) * SM::kPitch + 8 * n + 2 * tq) =
                make_float2(o[n][2], o[n][3]);
        if (tq == 0) s_ml[warp][g + 8] = make_float2(m1, l1);
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < nrows * (D / 4); idx += kThreads) {
        const int r = idx / (D / 4), d = (idx - r * (D / 4)) * 4;
        float mm = -INFINITY, ll = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kNarrowWarps; ++w) mm = fmaxf(mm, s_ml[w][r].x);
        const float u = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int w = 0; w < kNarrowWarps; ++w) {
            const float f = ex2(s_ml[w][r].x - u);
            const float4 v = *reinterpret_cast<const float4*>(red + (w * 16 + r) * SM::kPitch + d);
            ll = fmaf(f, s_ml[w][r].y, ll);
            a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
        }
        if (ll == 0.f && min(s_lim[r], p1) > p0) mm = kLowest;  // no score but -inf
        emit(r, d, mm, ll, a);
    }
    __syncthreads();  // the rings are free again
}

template <bool PREFIX, typename E, int D>
__global__ void __launch_bounds__(kThreads, 2) paged_narrow_kernel(const __grid_constant__ PagedWork p) {
    constexpr int ROWS = kNarrowRows, UNIT = kNarrowUnit;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_lim[ROWS];
    __shared__ float2 s_ml[kNarrowWarps][ROWS];
    __shared__ PagedPrefix s_prefix;
    const PagedKV& kv = p.kv;
    pdl_launch_dependents();
    pdl_wait();
    PagedCursor c = paged_find<PREFIX, ROWS, UNIT, kNarrowOverhead, kThreads>(p, blockIdx.x, gridDim.x, s_prefix);
    bool shares = false;  // the last tile goes on in the next CTA
    const int kv_lo = PREFIX ? 0 : p.prefix_len, sequences = PREFIX ? 1 : kv.B;
    while (c.u < c.hi && c.b < sequences) {
        bool cut;
        NarrowTile t;
        t.s = paged_seq<PREFIX>(p, s_prefix, c.b, cut);
        const PagedSegment<PREFIX, ROWS, UNIT, kNarrowOverhead> sg(p, t.s, c);
        if (sg.nu == 0) {
            paged_next<PREFIX, ROWS>(p, s_prefix, c, sg.cost);
            continue;
        }
        t.j = c.j;
        t.p0 = kv_lo + sg.k0 * UNIT;
        t.p1 = min(t.p0 + sg.nu * UNIT, paged_tile_limit<PREFIX, ROWS>(p, t.s, c.i));
        t.r0 = c.i * ROWS;
        t.nrows = min(ROWS, t.s.rows - t.r0);
        const bool whole = sg.whole();
        const int slot = 2 * blockIdx.x + (sg.k0 == 0 ? 1 : 0), parts = sg.parts(c, blockIdx.x);
        if (parts) {
            shares = true;
            if (threadIdx.x == 0) p.shared[blockIdx.x] = PagedShared{parts, t.nrows, t.r0, t.s.begin, c.j};
        }
        narrow_tile<PREFIX, E, D>(p, t, smem, s_lim, s_ml, [&](int r, int d, float mm, float ll, const float4& a) {
            const int rr = t.r0 + r, tok = p.by_G(rr), head = c.j * p.G + rr - tok * p.G;
            const int64_t row = t.s.begin + tok;
            if (whole && !p.row_o) {
                const float inv = paged_inverse(mm, ll);
                *reinterpret_cast<uint2*>(static_cast<E*>(p.out) + row * p.ldo + head * D + d) =
                    pack4<E>(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
                if (p.lse && d == 0) p.lse[row * p.ldl + head] = ll != 0.f ? (mm + log2f(ll)) * kLn2 : -INFINITY;
            } else {
                const int64_t at = whole ? row * kv.HQ + head : int64_t(slot) * ROWS + r;
                *reinterpret_cast<float4*>((whole ? p.row_o : p.part_o) + at * D + d) = a;
                if (d == 0) {
                    (whole ? p.row_ml : p.part_ml)[at] = make_float2(mm, ll);
                    if (p.row_at && sg.k0 == 0) p.row_at[row * kv.HQ + head] = paged_row_at(blockIdx.x, parts, r);
                }
            }
        });
        paged_next<PREFIX, ROWS>(p, s_prefix, c, sg.cost);
    }
    if (!shares && threadIdx.x == 0) p.shared[blockIdx.x].parts = 0;
}

// Few (sequence, kv head) pairs and a short cache: a cluster of CTAs per pair takes
// equal pieces of its positions and joins them through distributed shared memory
// (rank order, deterministic). No schedule to work out, no partials in memory and
// no second kernel. A shared prefix is read by each pair, mostly from L2. Bound:
// latency (length, page, keys, cluster barrier, output). Two sequences of 16 heads
// of 128, 300 to 700 positions: 6.0 us in a graph (equal shares and join: 10.6 us); four
// that share 512 of 520 to 800 positions: 7.6 us (two passes and join: 16.7 us).
template <typename E, int D>
__global__ void __launch_bounds__(kThreads, 2) paged_cluster_kernel(const __grid_constant__ PagedWork p, int ranks) {
    using SM = NarrowSmem<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_lim[kNarrowRows];
    __shared__ float2 s_ml[kNarrowWarps][kNarrowRows];
    __shared__ float2 s_row[kNarrowRows];
    constexpr int kOut = 40960;  // of the rings, behind the warps' outputs: this CTA's rows
    static_assert(kNarrowWarps * 16 * SM::kPitch * 4 <= kOut && kOut + 16 * D * 4 <= SM::kQ, "the rows fit the rings");
    float* out = reinterpret_cast<float*>(smem + kOut);
    pdl_launch_dependents();
    pdl_wait();
    const int pair = blockIdx.x / ranks, rank = blockIdx.x - pair * ranks;
    NarrowTile t;
    const int b = pair / p.kv.HKV;
    t.j = pair - b * p.kv.HKV;
    bool cut;
    t.s = paged_seq<false>(p, PagedPrefix{0, 0, 0}, b, cut);
    if (cut && rank == 0 && t.j == 0 && threadIdx.x == 0) atomicOr(p.kv.errors, BQ_DEVERR_POSITION_BIT);
    for (int i = 0; i * kNarrowRows < t.s.rows; ++i) {  // one tile, unless max_q was told too low
        t.r0 = i * kNarrowRows;
        t.nrows = min(kNarrowRows, t.s.rows - t.r0);
        const int limit = paged_tile_limit<false, kNarrowRows>(p, t.s, i), units = (limit + kNarrowUnit - 1) / kNarrowUnit;
        t.p0 = rank * units / ranks * kNarrowUnit;
        t.p1 = min((rank + 1) * units / ranks * kNarrowUnit, limit);
        narrow_tile<false, E, D>(p, t, smem, s_lim, s_ml, [&](int r, int d, float mm, float ll, const float4& a) {
            *reinterpret_cast<float4*>(out + r * D + d) = a;
            if (d == 0) s_row[r] = make_float2(mm, ll);
        });
        __syncwarp();        // (the barriers below want whole warps)
        cluster_sync_all();  // every rank's rows are in its shared memory
        for (int idx = rank * kThreads + threadIdx.x; idx < t.nrows * (D / 4); idx += ranks * kThreads) {
            const int r = idx / (D / 4), d = (idx - r * (D / 4)) * 4;
            const uint32_t a_out = smem_u32(out + r * D + d), a_row = smem_u32(&s_row[r]);
            float m[kMaxRanks], l[kMaxRanks], mm = -INFINITY, ll = 0.f;
            float4 o[kMaxRanks], a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q = 0; q < kMaxRanks; ++q) {
                if (q < ranks) {
                    const uint32_t from = dsmem_addr(a_row, uint32_t(q));
                    m[q] = dsmem_ld_f32(from);
                    l[q] = dsmem_ld_f32(from + 4);
                    o[q] = dsmem_ld4(dsmem_addr(a_out, uint32_t(q)));
                    mm = fmaxf(mm, m[q]);
                }
            }
            const float u = mm == -INFINITY ? 0.f : mm;
#pragma unroll
            for (int q = 0; q < kMaxRanks; ++q) {
                if (q < ranks) {
                    const float f = ex2(m[q] - u);
                    ll = fmaf(f, l[q], ll);
                    a.x = fmaf(f, o[q].x, a.x), a.y = fmaf(f, o[q].y, a.y), a.z = fmaf(f, o[q].z, a.z), a.w = fmaf(f, o[q].w, a.w);
                }
            }
            const int rr = t.r0 + r, tok = p.by_G(rr), head = t.j * p.G + rr - tok * p.G;
            const int64_t row = t.s.begin + tok;
            const float inv = paged_inverse(mm, ll);
            *reinterpret_cast<uint2*>(static_cast<E*>(p.out) + row * p.ldo + head * D + d) =
                pack4<E>(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
            if (p.lse && d == 0) p.lse[row * p.ldl + head] = ll != 0.f ? (mm + log2f(ll)) * kLn2 : -INFINITY;
        }
        __syncwarp();
        if ((i + 1) * kNarrowRows < t.s.rows)
            cluster_sync_all();  // the next tile's rows are written after every rank has read these
        else
            cluster_sync_relaxed();  // no rank leaves while another reads its rows (the reads were consumed by the stores)
    }
}

template <bool PREFIX>
const void* narrow_kernel(int dtype, int D) {
    return D == 128 ? (dtype == BQ_DT_BF16 ? reinterpret_cast<const void*>(&paged_narrow_kernel<PREFIX, __nv_bfloat16, 128>)
                                           : reinterpret_cast<const void*>(&paged_narrow_kernel<PREFIX, __half, 128>))
                    : (dtype == BQ_DT_BF16 ? reinterpret_cast<const void*>(&paged_narrow_kernel<PREFIX, __nv_bfloat16, 64>)
                                           : reinterpret_cast<const void*>(&paged_narrow_kernel<PREFIX, __half, 64>));
}

}  // namespace

int paged_launch_narrow(const PagedWork& w, int dtype, int D, int grid, uint32_t flags, void* stream) {
    const void* fn = w.prefix_pass ? narrow_kernel<true>(dtype, D) : narrow_kernel<false>(dtype, D);
    const uint32_t smem = D == 128 ? NarrowSmem<128>::kTotal : NarrowSmem<64>::kTotal;
    const int rc = ensure_smem_attr(fn, smem);
    if (rc) return rc;
    void* args[] = {const_cast<PagedWork*>(&w)};
    return paged_launch(fn, dim3(grid), dim3(kThreads), smem, args, flags, stream, "paged attention");
}

int paged_launch_cluster(const PagedWork& w, int dtype, int D, int ranks, uint32_t flags, void* stream) {
    const void* fn = D == 128 ? (dtype == BQ_DT_BF16 ? reinterpret_cast<const void*>(&paged_cluster_kernel<__nv_bfloat16, 128>)
                                                     : reinterpret_cast<const void*>(&paged_cluster_kernel<__half, 128>))
                              : (dtype == BQ_DT_BF16 ? reinterpret_cast<const void*>(&paged_cluster_kernel<__nv_bfloat16, 64>)
                                                     : reinterpret_cast<const void*>(&paged_cluster_kernel<__half, 64>));
    const uint32_t smem = D == 128 ? NarrowSmem<128>::kTotal : NarrowSmem<64>::kTotal;
    const int rc = ensure_smem_attr(fn, smem);
    if (rc) return rc;
    void* args[] = {const_cast<PagedWork*>(&w), &ranks};
    return paged_launch(fn, dim3(unsigned(w.kv.B) * w.kv.HKV * ranks), dim3(kThreads), smem, args, flags, stream, "paged attention",
                        ranks);
}

}  // namespace bq
