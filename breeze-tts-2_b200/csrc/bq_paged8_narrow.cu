// Attention over an 8-bit paged cache for tiles of at most 16 rows (a decode step, a
// few drafted tokens): one pass over the codes with a running maximum and sum, on
// mma.sync m16n8k16 tiles in f16, which holds every e4m3 code exactly.
//
// Bound: HBM, at half the bytes per position of a 16-bit cache; so the instructions
// between the loads and the products count, and the warps that cover their latencies:
// two for each scheduler, by the registers of the accumulators. Four warps per CTA take every fourth
// block of 32 positions of the CTA's share, each through a ring of its own (cp.async,
// no barrier between warps). The products' inner dimensions may be in any order, so a
// lane reads codes of neighbouring dims of its position by 16 bytes at a time and
// converts them in place: dims 4 i .. 4 i + 3 of its D / 4 are its entries of step i of
// q k^T, and v enters with positions 2 t, 2 t + 1 of neighbouring dims, two byte
// permutations per four pairs. Nothing is transposed or written back.
//
// Scales cost nothing per code. Those of k multiply the 16 scores of a block. Those of
// v go into the exponent of the probabilities: with base-2 scores s and v = code 2^e
// the weights are 2^(s + e - M), M a running maximum of s + e, so that the largest
// weight times code is what decides the range, whatever the scales are; the sum of
// exponentials takes the weights back times 2^-e.
//
// Rounding: q enters as f16 (bf16 rows scaled by a power of two that brings the row's
// largest entry to at least 2^14: exact but for entries under 2^-28 of it), the
// weights as f16 times 2^15 (half a step, 2^-11, and what is under 2^-29 of the
// largest loses less than 2^-40 of it). Scores, statistics and outputs are fp32.
//
// Measured (bf16, 32 query and 8 kv heads of 128, in a graph, join included): 6 sequences
// of 40 to 60 thousand positions, 581 MB, 103 us (5.6 TB/s; 114 when run for a second on
// end, at lower clocks); 64 sequences of 11 to 7000 positions, 168 MB, 44 us (3.8 TB/s:
// 5 to 7 us of shares and join, and each tile's start and end). The schedulers issue in
// 41 % of cycles, HBM is busy in 64 %, the ALU pipe (conversion, masks, exponents) in 39 %;
// a warp waits longest for its own last instruction (1.7 cycles an issue; 0.3 for loads),
// with eight warps on an SM too few to fill in. The products' 16 rows are half empty or
// more in a decode step. Not kept: a share per warp instead of per CTA (no
// sum over warps at a tile's end, but four times the parts to join: 47 us for the
// 64 sequences), finding the next tile's place and pages ahead (44.3 against 43.7).
#include "bq_host.h"
#include "bq_paged8.cuh"
#include "bq_paged8_host.h"

namespace bq {
namespace {

constexpr int kWarps = kNarrowWarps, kThreads = 32 * kWarps;
constexpr int kRows = kNarrowRows, kUnit = kNarrowUnit, kOverhead = kNarrow8Overhead;
constexpr int kStep = 32;              // positions of a warp's step
constexpr int kBatch = 32 * 16 / kStep;  // steps whose pages the lanes hold, one block of 16 positions each
// Weights are kept times 2^15, as they enter the product: relative to a reference 15 below the largest score. With
// exponents of v up to kSpread apart, what fp32 flushes of them is less than 2^-41 of the largest term of the sum of
// exponentials each. Exponents may lie 120 apart: then the sum takes what is flushed times 2^kFarLift. (Beside the masks,
// under a condition that both share: one of its own costs 6 sequences of 50 thousand positions 104.8 instead of 102.5 us.)
constexpr int kLift = 15, kSpread = 100, kFarLift = 64;
// Rounded up, so that no weight passes 2^15 however large the scores are (from 2^24 on fp32 does not hold m - 15, and
// fp16 ends at 2^16); sums and outputs are relative to what came out, so that nothing else depends on it.
__device__ __forceinline__ float reference(float m) { return __fadd_ru(m, -float(kLift)); }

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool full) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// N words (4 or 2) of shared memory.
template <int N>
__device__ __forceinline__ void lds(uint32_t* r, uint32_t a) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
    else
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a) : "memory");
}

// Shared memory: per warp a ring of kStages (k block, v block). After a tile's
// positions it holds the warps' outputs (fp32).
template <int D>
struct Smem8 {
    static constexpr int kBlock = kStep * D;                       // bytes of 32 rows
    static constexpr int kStages = D == 128 ? 3 : 6;               // 24 KB of ring per warp
    static constexpr int kRing = kStages * 2 * kBlock;
    static constexpr int kTotal = kWarps * kRing;
    // An output row: a lane's D / 4 dims, four floats of room, then the next lane's: eight lanes that store 16 bytes
    // each fall on different banks.
    static constexpr int kSeg = D / 4 + 4, kPitch = 4 * kSeg;      // floats
    static constexpr int kOut = kWarps * kRows * kPitch * 4;       // bytes of the warps' outputs
    static_assert(kOut + kRows * D * 4 <= kTotal, "the warps' outputs and the CTA's rows fit the rings");
    __device__ static int out_at(int warp, int r, int d) { return (warp * kRows + r) * kPitch + d / (D / 4) * kSeg + d % (D / 4); }
};

// 16-byte chunk c of row r of a block lies at chunk c ^ swizzle: lanes that read different rows at once read
// different banks (D = 128: 8 chunks a row; 64: two rows in 128 bytes).
template <int D>
__device__ __forceinline__ int chunk_at(int r, int c) {
    return D == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3);
}

// Positions [p0, p1) of rows r0 .. r0 + nrows of a sequence and kv head j.
struct Tile8 {
    PagedSeq s;
    int j, r0, nrows, p0, p1;
};

// NaN among four codes: 0xff in its byte.
__device__ __forceinline__ uint32_t nan4(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// NaN codes of the 16 rows of v at vb (positions pb ..): the rows that see their position become NaN, the codes are
// cleared (a zero weight times NaN is NaN, too). A warp calls it.
template <int D>
__device__ __forceinline__ void clear_nan(uint32_t vb, int r0, int pb, int lim0, int lim1, float (&o)[D / 8][4]) {
    constexpr int CH = D / 16, W = D / 16;  // chunks of a row; words of a lane's D / 4 dims
    const int lane = threadIdx.x & 31, tq = lane & 3;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 16 * CH / 32; ++i) {
        uint32_t x[4];
        lds<4>(x, vb + r0 * D + (lane + 32 * i) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= nan4(x[e]);
    }
    if (!__any_sync(0xffffffffu, bad)) return;
    const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll 1
    for (int r = 0; r < 16; ++r) {
        uint32_t x[W];
#pragma unroll
        for (int q = 0; q < W / 4; ++q) lds<4>(x + 4 * q, vb + (r0 + r) * D + (chunk_at<D>(r0 + r, tq * (W / 4) + q) << 4));
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const uint32_t n = nan4(x[w]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // dim 4 w + e of the lane's: n-tile (4 w + e) % (D / 8), column 2 tq or 2 tq + 1
                constexpr int T = D / 8;
                const int d = 4 * w + e;
                if ((n >> (8 * e)) & 1) {
                    if (pb + r < lim0) o[d % T][d / T] = nan;
                    if (pb + r < lim1) o[d % T][2 + d / T] = nan;
                }
            }
        }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16 * CH / 32; ++i) {
        const uint32_t a = vb + r0 * D + (lane + 32 * i) * 16;
        uint32_t x[4];
        lds<4>(x, a);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] &= ~nan4(x[e]);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
    }
    __syncwarp();
}

// The queries of one row as the A operand holds them (D / 16 steps of two pairs), and what its scores are to be
// multiplied with.
template <typename E, int D>
__device__ __forceinline__ void query_row(const PagedWork& p, const Tile8& t, int r, uint32_t (&q)[D / 16][2], float& factor) {
    constexpr int W = D / 8;  // words of a lane's D / 4 dims
    const int tq = threadIdx.x & 3;
    uint32_t x[W];
    const int rr = t.r0 + min(r, t.nrows - 1), tok = p.by_G(rr);
    const E* src = static_cast<const E*>(p.q) + int64_t(t.s.begin + tok) * p.ldq + (t.j * p.G + rr - tok * p.G) * D + tq * (D / 4);
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        const uint4 v = r < t.nrows ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
        x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
    }
    factor = p.scale_log2;
    if constexpr (std::is_same_v<E, __nv_bfloat16>) {
        uint32_t top = 0;  // largest finite magnitude of the row, as bits
#pragma unroll
        for (int i = 0; i < W; ++i) top = __vmaxu2(top, x[i] & 0x7fff7fffu & ~nonfinite2<E>(x[i]));
        top = max(top >> 16, top & 0xffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int k = top ? max(int(top >> 7) - 127 - 14, -126) : 0;  // the largest becomes 2^14 .. 2^15
        const float down = exp_scale(-k);
        factor *= exp_scale(k);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            float a, b;
            unpack2<E>(x[i], a, b);
            x[i] = pack_half2(a * down, b * down);
        }
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) q[i][0] = x[2 * i], q[i][1] = x[2 * i + 1];
}

// One tile with the whole CTA: emit(r, d, m, l, o) receives dims d .. d + 3 of row r,
// unnormalized, with the row's reference score (base 2) and sum of exponentials.
template <typename E, int D, typename Emit>
__device__ __forceinline__ void tile8(const PagedWork& p, const Paged8Scales& sc, const Tile8& t, unsigned char* smem,
                                      float2 (*s_ml)[kRows], const Emit& emit) {
    using SM = Smem8<D>;
    constexpr int CH = D / 16, ST = SM::kStages, T = D / 8;
    const uint32_t sb = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const PagedKV& kv = p.kv;
    const uint32_t ring = sb + warp * SM::kRing;
    const PagedSeq& s = t.s;
    const int p0 = t.p0, p1 = t.p1;
    bool pages_ok = true;
    const int steps = (max(0, (p1 - p0 + kStep - 1) / kStep) - warp + kWarps - 1) / kWarps;
    const uint8_t* kh = static_cast<const uint8_t*>(kv.k) + t.j * kv.ks_head;
    const uint8_t* vh = static_cast<const uint8_t*>(kv.v) + t.j * kv.vs_head;

    // Lane i looks up block i of 16 positions of a batch of steps: pages two batches ahead, scale bytes (k, v << 8)
    // one batch ahead, so that no step waits for either.
    auto position = [&](int batch) { return p0 + kStep * (warp + kWarps * (kBatch * batch + (lane >> 1))) + 16 * (lane & 1); };
    auto page_of = [&](int batch) {
        const int pos = position(batch);
        return pos < p1 ? paged_page(kv, s.table, pos, pages_ok) : 0;
    };
    auto scales_of = [&](int batch, int page) {
        const int pos = position(batch), blk = (pos & kv.page_mask) >> sc.block_shift;
        return pos < p1 ? uint32_t(*k_scale(sc, page, t.j, blk)) | uint32_t(*v_scale(sc, page, t.j, blk)) << 8
                        : uint32_t(kExpBias | kExpBias << 8);
    };
    int page_now = page_of(0), page_next = page_of(1), page_third = 0;
    uint32_t exp_issue = 0, exp_next = 0, exp_now = 0;
    auto issue = [&](int st) {
        if (st > 0 && st % kBatch == 0) {
            page_now = page_next;
            exp_issue = exp_next;
            page_next = page_third;
            exp_next = scales_of(st / kBatch + 1, page_next);
            page_third = page_of(st / kBatch + 2);
        }
        const int pages[2] = {__shfl_sync(0xffffffffu, page_now, 2 * st % 32), __shfl_sync(0xffffffffu, page_now, 2 * st % 32 + 1)};
        if (st < steps) {
            const int pb = p0 + kStep * (warp + kWarps * st);
            const uint32_t dst = ring + (st % ST) * (2 * SM::kBlock);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int slot = (pb + 16 * b) & kv.page_mask;
                const uint8_t* kp = kh + pages[b] * kv.ks_page + slot * kv.ks_slot;
                const uint8_t* vp = vh + pages[b] * kv.vs_page + slot * kv.vs_slot;
                const int r0 = lane / CH, c = lane % CH;  // rows r0 + 32 / CH i
                kp += r0 * kv.ks_slot + c * 16;
                vp += r0 * kv.vs_slot + c * 16;
                constexpr int RS = 32 / CH;
                if (pb + 16 * b + 16 <= p1) {
#pragma unroll
                    for (int i = 0; i < 16 / RS; ++i) {
                        const int rr = 16 * b + r0 + RS * i;
                        const uint32_t at = rr * D + (chunk_at<D>(rr, c) << 4);
                        cp_async16(dst + at, kp + i * (RS * kv.ks_slot));
                        cp_async16(dst + SM::kBlock + at, vp + i * (RS * kv.vs_slot));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16 / RS; ++i) {
                        const int rr = 16 * b + r0 + RS * i;
                        const uint32_t at = rr * D + (chunk_at<D>(rr, c) << 4);
                        cp_async16_zfill(dst + at, kp + i * (RS * kv.ks_slot), pb + rr < p1);
                        cp_async16_zfill(dst + SM::kBlock + at, vp + i * (RS * kv.vs_slot), pb + rr < p1);
                    }
                }
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int st = 0; st < ST - 1; ++st) issue(st);
    exp_issue = scales_of(0, page_now);
    exp_next = scales_of(1, page_next);
    page_third = page_of(2);
    uint32_t qf[D / 16][4];
    float f0, f1;
    {
        uint32_t a[D / 16][2], b[D / 16][2];
        query_row<E, D>(p, t, g, a, f0);
        query_row<E, D>(p, t, g + 8, b, f1);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) qf[i][0] = a[i][0], qf[i][1] = b[i][0], qf[i][2] = a[i][1], qf[i][3] = b[i][1];
    }
    const int lim0 = g < t.nrows ? paged_row_limit<false>(p, s, t.r0 + g) : 0;
    const int lim1 = g + 8 < t.nrows ? paged_row_limit<false>(p, s, t.r0 + g + 8) : 0;
    const int seen = __reduce_min_sync(0xffffffffu, min(g < t.nrows ? lim0 : p1, g + 8 < t.nrows ? lim1 : p1));  // by every row
    float o[T][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int n = 0; n < T; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    // TWO: the tile has more than 8 rows; else rows g + 8 are left out of the softmax.
    auto stream = [&](auto two) {
    constexpr bool TWO = decltype(two)::value;
    int top = -kExpMost;  // largest exponent of v so far
    bool far = false;
    for (int st = 0; st < steps; ++st) {
        cp_wait<ST - 2>();
        __syncwarp();  // every lane's copies of this stage have landed, and every lane is done with the one before
        issue(st + ST - 1);
        if (st % kBatch == 0) {
            exp_now = exp_issue;
            const int ev = scale_exp(exp_now >> 8);  // (0 where there is no block: not far from both ends)
            top = max(top, __reduce_max_sync(0xffffffffu, ev));
            far = top - __reduce_min_sync(0xffffffffu, ev) > kSpread;
        }
        const uint32_t kb = ring + (st % ST) * (2 * SM::kBlock), vb = kb + SM::kBlock;
        const int blk = p0 + kStep * (warp + kWarps * st), pb = blk + 2 * tq;
        float x[4][4] = {};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            uint32_t w[D / 16];
#pragma unroll
            for (int q = 0; q < D / 64; ++q) lds<4>(w + 4 * q, kb + (8 * n + g) * D + (chunk_at<D>(8 * n + g, tq * (D / 64) + q) << 4));
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                uint32_t lo, hi;
                codes_f16(w[i], lo, hi);
                mma_f16(x[n], qf[i][0], qf[i][1], qf[i][2], qf[i][3], lo, hi);
            }
        }
        float n0 = m0, n1 = m1, back[2];
        const bool cut = min(blk + kStep, p1) > seen || blk + kStep > p1;  // some row does not see all of it
        const bool unusual = cut || far;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t ee = __shfl_sync(0xffffffffu, exp_now, 2 * st % 32 + b);
            const int ev = scale_exp(ee >> 8);
            const float ks = exp_scale(scale_exp(ee & 255)), a0 = f0 * ks, a1 = f1 * ks, y = float(ev);
            back[b] = exp_scale(-ev);
#pragma unroll
            for (int n = 2 * b; n < 2 * b + 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    x[n][e] = fmaf(x[n][e], a0, y);
                    if constexpr (TWO) x[n][2 + e] = fmaf(x[n][2 + e], a1, y);
                }
        }
        if (cut) {
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (pb + 8 * n + e >= lim0) x[n][e] = -INFINITY;
                    if constexpr (TWO)
                        if (pb + 8 * n + e >= lim1) x[n][2 + e] = -INFINITY;
                }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            n0 = fmaxf(n0, fmaxf(x[n][0], x[n][1]));
            if constexpr (TWO) n1 = fmaxf(n1, fmaxf(x[n][2], x[n][3]));
        }
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 1));
        if constexpr (TWO) n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 1));
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 2));
        if constexpr (TWO) n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 2));
        if (__any_sync(0xffffffffu, n0 != m0 || (TWO && n1 != m1))) {  // a maximum moved: rescale what was summed
            const float a0 = n0 == m0 ? 1.f : ex2(0.5f * (reference(m0) - reference(n0)));  // in two steps: l may be as far from 1
            l0 = l0 * a0 * a0;
#pragma unroll
            for (int n = 0; n < T; ++n) o[n][0] *= a0 * a0, o[n][1] *= a0 * a0;
            m0 = n0;
            if constexpr (TWO) {
                const float a1 = n1 == m1 ? 1.f : ex2(0.5f * (reference(m1) - reference(n1)));
                l1 = l1 * a1 * a1;
#pragma unroll
                for (int n = 0; n < T; ++n) o[n][2] *= a1 * a1, o[n][3] *= a1 * a1;
                m1 = n1;
            }
        }
        const float u0 = m0 == -INFINITY ? 0.f : reference(m0), u1 = m1 == -INFINITY ? 0.f : reference(m1);  // (rows that see nothing yet)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if (unusual) {
                if (far) {
                    const float z = back[b] * exp_scale(-kFarLift);
                    auto flushed = [&](float d) { return d < -126.f ? ex2(d + kFarLift) * z : 0.f; };
#pragma unroll
                    for (int n = 2 * b; n < 2 * b + 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            l0 += flushed(x[n][e] - u0);
                            if constexpr (TWO) l1 += flushed(x[n][2 + e] - u1);
                        }
                }
                if (min(blk + 16 * b + 16, p1) > seen) clear_nan<D>(vb, 16 * b, blk + 16 * b, lim0, lim1, o);
            }
#pragma unroll
            for (int n = 2 * b; n < 2 * b + 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    x[n][e] = ex2(x[n][e] - u0);
                    l0 = fmaf(x[n][e], back[b], l0);
                    if constexpr (TWO) {
                        x[n][2 + e] = ex2(x[n][2 + e] - u1);
                        l1 = fmaf(x[n][2 + e], back[b], l1);
                    }
                }
            uint32_t pf[4] = {pack_half2(x[2 * b][0], x[2 * b][1]), 0, pack_half2(x[2 * b + 1][0], x[2 * b + 1][1]), 0};
            if constexpr (TWO) {
                pf[1] = pack_half2(x[2 * b][2], x[2 * b][3]);
                pf[3] = pack_half2(x[2 * b + 1][2], x[2 * b + 1][3]);
            }
            // the lane's positions 2 tq, 2 tq + 1, 8 + 2 tq, 9 + 2 tq; its D / 8 dims from g D / 8 on
            constexpr int W = D / 32;
            uint32_t v[4][W];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * b + 8 * (i >> 1) + 2 * tq + (i & 1);
                if constexpr (D == 128)
                    lds<4>(v[i], vb + r * D + (chunk_at<D>(r, g) << 4));
                else
                    lds<2>(v[i], vb + r * D + (chunk_at<D>(r, g >> 1) << 4) + (g & 1) * 8);
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                uint32_t a[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    codes_f16(prmt(v[2 * h][w], v[2 * h + 1][w], 0x5140), a[h][0], a[h][1]);
                    codes_f16(prmt(v[2 * h][w], v[2 * h + 1][w], 0x7362), a[h][2], a[h][3]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) mma_f16(o[4 * w + e], pf[0], pf[1], pf[2], pf[3], a[0][e], a[1][e]);
            }
        }
    }
    };
    if (t.nrows > 8)
        stream(std::true_type());
    else
        stream(std::false_type());
    cp_wait<0>();
    if (!pages_ok) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    // From here on a part's reference is near its sum, so that parts are weighed by what they hold of the row.
    auto settle = [&](float& m, float& l) {
        m = reference(m);
        return settle_part(m, l);
    };
    const float z0 = settle(m0, l0), z1 = settle(m1, l1);
    __syncthreads();  // every warp is done with its ring: it now takes the warps' outputs
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h;
        const float z = h ? z1 : z0;
        if (r < t.nrows) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {  // dims 4 i .. 4 i + 3 of the lane's D / 4
                const int c = 4 * i / T, n = 4 * i % T;
                *reinterpret_cast<float4*>(red + SM::out_at(warp, r, tq * (D / 4) + 4 * i)) =
                    make_float4(o[n][2 * h + c] * z, o[n + 1][2 * h + c] * z, o[n + 2][2 * h + c] * z, o[n + 3][2 * h + c] * z);
            }
            if (tq == 0) s_ml[warp][r] = h ? make_float2(m1, l1) : make_float2(m0, l0);
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < t.nrows * (D / 4); idx += kThreads) {
        const int r = idx / (D / 4), d = (idx - r * (D / 4)) * 4;
        float mm = -INFINITY, ll = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_ml[w][r].x);
        const float u = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(s_ml[w][r].x - u);
            const float4 v = *reinterpret_cast<const float4*>(red + SM::out_at(w, r, d));
            ll = fmaf(f, s_ml[w][r].y, ll);
            a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
        }
        if (ll == 0.f && min(paged_row_limit<false>(p, s, t.r0 + r), p1) > p0) mm = kLowest;  // no score but -inf
        emit(r, d, mm, ll, a);
    }
    __syncthreads();  // the rings are free again
}

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, 2) paged8_narrow_kernel(const __grid_constant__ PagedWork p,
                                                                    const __grid_constant__ Paged8Scales sc) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float2 s_ml[kWarps][kRows];
    __shared__ PagedPrefix s_prefix;  // (none: the shared pieces want one)
    const PagedKV& kv = p.kv;
    pdl_launch_dependents();
    pdl_wait();
    PagedCursor c = paged_find<false, kRows, kUnit, kOverhead, kThreads>(p, blockIdx.x, gridDim.x, s_prefix);
    bool shares = false;  // the last tile goes on in the next CTA
    while (c.u < c.hi && c.b < kv.B) {
        bool cut;
        Tile8 t;
        t.s = paged_seq<false>(p, s_prefix, c.b, cut);
        const PagedSegment<false, kRows, kUnit, kOverhead> sg(p, t.s, c);
        if (sg.nu == 0) {
            paged_next<false, kRows>(p, s_prefix, c, sg.cost);
            continue;
        }
        t.j = c.j;
        t.p0 = sg.k0 * kUnit;
        t.p1 = min(t.p0 + sg.nu * kUnit, paged_tile_limit<false, kRows>(p, t.s, c.i));
        t.r0 = c.i * kRows;
        t.nrows = min(kRows, t.s.rows - t.r0);
        const bool whole = sg.whole();
        const int slot = 2 * blockIdx.x + (sg.k0 == 0 ? 1 : 0), parts = sg.parts(c, blockIdx.x);
        if (parts) {
            shares = true;
            if (threadIdx.x == 0) p.shared[blockIdx.x] = PagedShared{parts, t.nrows, t.r0, t.s.begin, c.j};
        }
        tile8<E, D>(p, sc, t, smem, s_ml, [&](int r, int d, float mm, float ll, const float4& a) {
            if (whole) {
                const int rr = t.r0 + r, tok = p.by_G(rr), head = c.j * p.G + rr - tok * p.G;
                const int64_t row = t.s.begin + tok;
                const float inv = paged_inverse(mm, ll);
                *reinterpret_cast<uint2*>(static_cast<E*>(p.out) + row * p.ldo + head * D + d) =
                    pack4<E>(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
                if (p.lse && d == 0) p.lse[row * p.ldl + head] = ll != 0.f ? (mm + log2f(ll)) * kLn2 : -INFINITY;
            } else {
                const int64_t at = int64_t(slot) * kRows + r;
                *reinterpret_cast<float4*>(p.part_o + at * D + d) = a;
                if (d == 0) p.part_ml[at] = make_float2(mm, ll);
            }
        });
        paged_next<false, kRows>(p, s_prefix, c, sg.cost);
    }
    if (!shares && threadIdx.x == 0) p.shared[blockIdx.x].parts = 0;
}

// Few (sequence, kv head) pairs and a short cache: a cluster of CTAs per pair takes
// equal pieces of its positions and joins them through distributed shared memory
// (rank order, deterministic). No schedule to work out, no partials in memory and
// no second kernel. Bound: latency (length, page, codes, cluster barrier, output).
template <typename E, int D>
__global__ void __launch_bounds__(kThreads, 2) paged8_cluster_kernel(const __grid_constant__ PagedWork p,
                                                                     const __grid_constant__ Paged8Scales sc, int ranks) {
    using SM = Smem8<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float2 s_ml[kWarps][kRows];
    __shared__ float2 s_row[kRows];
    float* out = reinterpret_cast<float*>(smem + SM::kOut);  // of the rings, behind the warps' outputs: this CTA's rows
    pdl_launch_dependents();
    pdl_wait();
    const int pair = blockIdx.x / ranks, rank = blockIdx.x - pair * ranks;
    Tile8 t;
    const int b = pair / p.kv.HKV;
    t.j = pair - b * p.kv.HKV;
    bool cut;
    t.s = paged_seq<false>(p, PagedPrefix{0, 0, 0}, b, cut);
    if (cut && rank == 0 && t.j == 0 && threadIdx.x == 0) atomicOr(p.kv.errors, BQ_DEVERR_POSITION_BIT);
    for (int i = 0; i * kRows < t.s.rows; ++i) {  // one tile, unless max_q was told too low
        t.r0 = i * kRows;
        t.nrows = min(kRows, t.s.rows - t.r0);
        const int limit = paged_tile_limit<false, kRows>(p, t.s, i), units = (limit + kUnit - 1) / kUnit;
        t.p0 = rank * units / ranks * kUnit;
        t.p1 = min((rank + 1) * units / ranks * kUnit, limit);
        tile8<E, D>(p, sc, t, smem, s_ml, [&](int r, int d, float mm, float ll, const float4& a) {
            *reinterpret_cast<float4*>(out + r * D + d) = a;
            if (d == 0) s_row[r] = make_float2(mm, ll);
        });
        __syncwarp();        // (the barriers below want whole warps)
        cluster_sync_all();  // every rank's rows are in its shared memory
        for (int idx = rank * kThreads + threadIdx.x; idx < t.nrows * (D / 4); idx += ranks * kThreads) {
            const int r = idx / (D / 4), d = (idx - r * (D / 4)) * 4;
            const uint32_t a_out = smem_u32(out + r * D + d), a_row = smem_u32(&s_row[r]);
            float m[kNarrowRanks], l[kNarrowRanks], mm = -INFINITY, ll = 0.f;
            float4 o[kNarrowRanks], a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q = 0; q < kNarrowRanks; ++q) {
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
            for (int q = 0; q < kNarrowRanks; ++q) {
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
        if ((i + 1) * kRows < t.s.rows)
            cluster_sync_all();  // the next tile's rows are written after every rank has read these
        else
            cluster_sync_relaxed();  // no rank leaves while another reads its rows (the reads were consumed by the stores)
    }
}

}  // namespace

int paged8_launch_narrow(const PagedWork& w, const Paged8Scales& sc, int dtype, int D, int grid, uint32_t flags, void* stream) {
    const bool bf = dtype == BQ_DT_BF16;
    const void* fn = D == 128 ? (bf ? reinterpret_cast<const void*>(&paged8_narrow_kernel<__nv_bfloat16, 128>)
                                    : reinterpret_cast<const void*>(&paged8_narrow_kernel<__half, 128>))
                              : (bf ? reinterpret_cast<const void*>(&paged8_narrow_kernel<__nv_bfloat16, 64>)
                                    : reinterpret_cast<const void*>(&paged8_narrow_kernel<__half, 64>));
    const uint32_t smem = D == 128 ? Smem8<128>::kTotal : Smem8<64>::kTotal;
    const int rc = ensure_smem_attr(fn, smem);
    if (rc) return rc;
    void* args[] = {const_cast<PagedWork*>(&w), const_cast<Paged8Scales*>(&sc)};
    return paged_launch(fn, dim3(grid), dim3(kThreads), smem, args, flags, stream, "paged attention");
}

int paged8_launch_cluster(const PagedWork& w, const Paged8Scales& sc, int dtype, int D, int ranks, uint32_t flags, void* stream) {
    const bool bf = dtype == BQ_DT_BF16;
    const void* fn = D == 128 ? (bf ? reinterpret_cast<const void*>(&paged8_cluster_kernel<__nv_bfloat16, 128>)
                                    : reinterpret_cast<const void*>(&paged8_cluster_kernel<__half, 128>))
                              : (bf ? reinterpret_cast<const void*>(&paged8_cluster_kernel<__nv_bfloat16, 64>)
                                    : reinterpret_cast<const void*>(&paged8_cluster_kernel<__half, 64>));
    const uint32_t smem = D == 128 ? Smem8<128>::kTotal : Smem8<64>::kTotal;
    const int rc = ensure_smem_attr(fn, smem);
    if (rc) return rc;
    void* args[] = {const_cast<PagedWork*>(&w), const_cast<Paged8Scales*>(&sc), &ranks};
    return paged_launch(fn, dim3(unsigned(w.kv.B) * w.kv.HKV * ranks), dim3(kThreads), smem, args, flags, stream, "paged attention",
                        ranks);
}

}  // namespace bq
