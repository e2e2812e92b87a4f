// Attention over an 8-bit paged cache for tiles of many rows (prompts) on the tcgen05
// tensor cores: 256 rows per CTA in two halves of 128, keys and values in units of 128
// positions, laid out as in the 16-bit kernel (bq_paged_wide.cu): the halves take turns
// in one score buffer, probabilities and outputs stay in tensor memory, roles walk
// ahead. What differs is how k and v come in, and the scales.
//
// The tensor cores take both operands in one type, so codes are converted: a warp
// fetches them by TMA, a unit ahead, four others write them as 16-bit tiles in the
// swizzled layout of the products, once for the 256 rows. Keys become the queries' type,
// values fp16; either holds every code exactly. Queries split into e4m3 terms would leave
// the keys as they are, but probabilities need more range than e4m3 has, so values have
// to be converted all the same.
//
// Scales: 2^ek multiplies the scores of a block, 2^ev goes into the exponent of its
// probabilities, as in the kernel for few rows: the weights are 2^(s + ev - M + 7), M a
// reference that may lag behind the largest s + ev by up to 8, so at most 2^15 in fp16.
// The fetching warp leaves each unit's eight sets of factors in shared memory. Where
// the ev of a unit lie more than 100 below one of the tile so far, weights that fp32
// flushes might still count in the sum of exponentials, which is then computed on its own.
//
// Measured: a prompt of 6500 tokens, 16 heads over 8 of 128, 173 GFLOP in 245 us (0.71
// PFLOP/s; tensor cores and exponential units busy in 37 % of cycles each), 229 us on
// values without large maxima; the 16-bit kernel takes 214 and 186 us for the same values
// (64 dims: 213 and 196, 200 and 182), so the smaller cache costs prompts 7 to 23 %. What
// bounds it is the instructions around the products, codes converted once for each tile of
// rows among them: softmax, conversion and the roles' loops share the instruction cache, which a
// conversion unrolled over a tile already overruns (314 us; rolled, one 16-byte piece at a
// time, 246 then). Not kept: exponentials against the maximum so far while the new one is found,
// as the 16-bit kernel has it (257 us on even data, 285 on data whose maxima move; with the
// maximum first 257 and 267); scores read from tensor memory in pieces of 32, with a
// buffer for each half (308); two threads per row (253); codes fetched by the converting
// warps themselves (435).
//
// Roles (one CTA per SM, all 512 tensor-memory columns): warps 0-3, 4-7 softmax of half
// 0 / 1; 8 issues the scores' products, 9 the outputs'; 10 walks the tiles and fetches
// their queries; 11 fetches codes and scales; 12-15 convert.
#include "bq_paged8.cuh"
#include "bq_paged8_host.h"
#include "bq_paged_wide.cuh"

namespace bq {

struct Wide8Params {
    CUtensorMap qmap, kmap, vmap;  // queries: (D, heads, rows), boxes of 64 dims x 128 rows; codes: (D, then slot, head and
                                   // page in order of stride), boxes of positions of one page
    PagedWork w;
    Paged8Scales sc;
    int32_t q_tma;                           // the queries come by TMA
    int32_t box;                             // positions per box: min(page size, 128)
    int32_t k_slot, k_head, v_slot, v_head;  // which of coordinates 1 .. 3 is the slot, the head (the third is the page)
    uint32_t idesc_qk, idesc_pv;
    long long wait_cycles;
};

namespace {

constexpr int kThreads = 512;
// Registers: the CTA starts with 512 x 128; the third and fourth warpgroup give up what the softmax warps, a row of
// 128 scores per thread, need more (256 x 200 + 256 x 56). The file is compiled as a whole program, since relocatable
// code may not move registers.
constexpr int kSoftmaxRegs = 200, kOtherRegs = 56;
constexpr int kScores = 8, kOutputs = 9, kWalker = 10, kFetch = 11, kConvert = 12;  // warps of the roles behind the softmax
constexpr int kReaders = 15;      // warps that read a tile of the walker's
constexpr int kBlocks = kUnit / 16;
constexpr int kLift = 7, kFarLift = 64;  // weights are kept times 2^7; where that is not enough, their sum is of 2^64 times
constexpr int kSpread = 100;
// Rows with maxima of this size and more are computed again at the tile's end (large_row). Below, the exponent of a
// weight, s x + (y + 7 - M), is at most 15 for a score 8 above the reference M, and its roundings (half a unit of M's last
// place, three times) are less than 0.1; from 2^23 on they would take it past fp16's range, and further on under it. Taking
// the score's distance from the reference first, for all scores, costs prompts 257 us instead of 245, under a condition
// behind the maximum 255 to 262, before it 269, in an instance of the loop of its own 370 (registers spill).
constexpr float kLargeScore = 1048576.f;  // 2^20
constexpr long long kLargeCycles = 60000;  // twice what a position takes a warp there

template <int D>
struct Wide8Smem {
    static constexpr uint32_t kTile = 128 * D * 2;                   // one k or v tile, one half of the queries
    static constexpr int kStages = D == 128 ? 4 : 8;
    // Units whose factors are kept. When those of unit U are written, the keys of U - 1 have been converted, so their
    // stage was free: the scores of U - 1 - kStages / 2 have been multiplied, both halves have read those of the unit
    // before, and are done with all before that.
    static constexpr int kTables = kStages / 2 + 3;
    static constexpr uint32_t kRing = 2 * kTile;
    static constexpr uint32_t kCodes = kRing + kStages * kTile;      // the codes of a k and a v tile on their way
    static constexpr uint32_t kBars = kCodes + kTile;
    static constexpr uint32_t kTotal = kBars + 512 + 1024;           // + slack to align the tiles to 1024 bytes
};

// NaN among four codes: 0xff in its byte.
__device__ __forceinline__ uint32_t nan4(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

__device__ __forceinline__ void lds128(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t t) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(t) : "memory");
}

// Four codes -> four elements (exact).
template <typename E>
__device__ __forceinline__ uint2 codes_to(uint32_t w) {
    uint32_t lo, hi;
    codes_f16(w, lo, hi);
    if constexpr (std::is_same_v<E, __half>) {
        return make_uint2(lo, hi);
    } else {
        float a, b, c, d;
        unpack2<__half>(lo, a, b);
        unpack2<__half>(hi, c, d);
        return make_uint2(pack_bf162(a, b), pack_bf162(c, d));
    }
}

// A lane's 16-byte pieces of a 128-position tile: codes 16 c .. 16 c + 15 of rows row(k). Eight neighbouring lanes have
// two rows that differ in bit 0, so that their chunks of the converted tile fall on different banks, and, with rows of
// 128 bytes, in bit 2, so that those of the codes (128-byte swizzle, too) do.
template <int D>
struct Piece {
    static constexpr int kCount = D == 128 ? 8 : 4, kStep = D == 128 ? 2 : 1;  // rows k and k + kStep are 32 apart
    int first, c;
    __device__ __forceinline__ Piece(int warp, int lane) {
        const int sub = lane >> 2;
        first = 8 * warp + (D == 128 ? (sub & 2) | (sub & 1) * 5 : sub);
        c = (lane & 3) + (D == 128 ? (lane >> 4) * 4 : 0);
    }
    __device__ __forceinline__ int row(int k) const { return 32 * (k / kStep) + (first ^ (k % kStep)); }
    __device__ __forceinline__ uint32_t from(int k) const {  // in the codes
        const int r = row(k);
        return r * D + ((D == 128 ? c ^ (r & 7) : c) << 4);
    }
    __device__ __forceinline__ uint32_t to(int k) const {  // of its first chunk in the tile; the second is at ^ 16
        const int r = row(k);
        return (c >> 2) * (128 * 128) + r * 128 + ((((c & 3) * 2) ^ (r & 7)) << 4);
    }
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}

// Row `row` of a tile over positions [t.p0, end) in fp32, by one thread (slow, and little code: unrolled by two it would
// cost every prompt 12 us), to where the tile's rows go:
// `at` of the parts. Not a call: its registers would cost every tile (prompts 254 us instead of 245).
template <typename E, int D>
__device__ __forceinline__ void large_row(const PagedWork& w, const Paged8Scales& sc, const WideTile& t, int row, int end, int64_t at) {
    const PagedKV& kv = w.kv;
    const int tok = w.by_G(row), head = t.j * w.G + row - tok * w.G;
    const E* q = static_cast<const E*>(w.q) + int64_t(t.s.begin + tok) * w.ldq + head * D;
    bool page_ok = true;  // (a bad page has been reported by the warp that fetched it)
    auto score = [&](int pos) {
        const int page = paged_page(kv, t.s.table, pos, page_ok), slot = pos & kv.page_mask;
        const uint8_t* k = static_cast<const uint8_t*>(kv.k) + page * kv.ks_page + t.j * kv.ks_head + int64_t(slot) * kv.ks_slot;
        float s = 0.f;
#pragma unroll 1
        for (int d = 0; d < D; d += 8) {
            const uint2 codes = *reinterpret_cast<const uint2*>(k + d);
            float x[8], c[4];
            unpack8<E>(*reinterpret_cast<const uint4*>(q + d), x);
            codes_f32(codes.x, c);
#pragma unroll
            for (int i = 0; i < 4; ++i) s = fmaf(x[i], c[i], s);
            codes_f32(codes.y, c);
#pragma unroll
            for (int i = 0; i < 4; ++i) s = fmaf(x[4 + i], c[i], s);
        }
        // (rounded: as part of the difference below the product would not be, and its maximum is)
        return __fmul_rn(s, w.scale_log2 * exp_scale(scale_exp(*k_scale(sc, page, t.j, slot >> sc.block_shift))));
    };
    float top = -INFINITY, sum = 0.f, o[D];
#pragma unroll 1
    for (int pos = t.p0; pos < end; ++pos) top = fmaxf(top, score(pos));
#pragma unroll 1
    for (int d = 0; d < D; ++d) o[d] = 0.f;
#pragma unroll 1
    for (int pos = t.p0; pos < end; ++pos) {
        const float p = ex2(score(pos) - top);
        sum += p;
        const int page = paged_page(kv, t.s.table, pos, page_ok), slot = pos & kv.page_mask;
        const uint8_t* v = static_cast<const uint8_t*>(kv.v) + page * kv.vs_page + t.j * kv.vs_head + int64_t(slot) * kv.vs_slot;
        const float f = p * exp_scale(scale_exp(*v_scale(sc, page, t.j, slot >> sc.block_shift)));
#pragma unroll 1
        for (int d = 0; d < D; d += 4) {
            float c[4];
            codes_f32(*reinterpret_cast<const uint32_t*>(v + d), c);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d + i] = fmaf(f, c[i], o[d + i]);
        }
    }
    const int64_t orow = t.s.begin + tok;
    const float inv = t.whole ? 1.f / sum : 1.f;
#pragma unroll 1
    for (int d = 0; d < D; d += 2) {
        if (t.whole)
            *reinterpret_cast<uint32_t*>(static_cast<E*>(w.out) + orow * w.ldo + head * D + d) = pack2<E>(o[d] * inv, o[d + 1] * inv);
        else
            *reinterpret_cast<float2*>(w.part_o + at * D + d) = make_float2(o[d], o[d + 1]);
    }
    if (!t.whole)
        w.part_ml[at] = make_float2(top, sum);
    else if (w.lse)
        w.lse[orow * w.ldl + head] = (top + log2f(sum)) * kLn2;
}

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, 1) paged8_wide_kernel(const __grid_constant__ Wide8Params p) {
    using SM = Wide8Smem<D>;
    constexpr int ST = SM::kStages, kTables = SM::kTables;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ PagedPrefix s_prefix;  // (none: the shared pieces want one)
    __shared__ WideTile s_tile[kTiles];
    __shared__ volatile int s_bad[kTiles];   // n + 1: NaN entries of v were cleared from tile n
    __shared__ float4 s_factor[kTables][kBlocks];  // per block: scores times x, plus y, in base 2; sums times z
    __shared__ int s_far[kTables];           // the unit's sum of exponentials needs the longer way
    const uint32_t sraw = smem_u32(smem_raw), sb = (sraw + 1023u) & ~1023u;
    const PagedWork& w = p.w;
    const PagedKV& kv = w.kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort = &s_abort;
    const long long lim = p.wait_cycles;
    // full / empty per ring stage; per half: queries staged, scores ready, probabilities written, second product
    // complete, queries used; scores read; per tile in s_tile: written, read by all its readers; codes of keys / values
    // there, converted
    const uint32_t bar_full = sb + SM::kBars, bar_empty = bar_full + 64, bar_q = bar_full + 128, bar_s = bar_full + 144,
                   bar_p = bar_full + 160, bar_pv = bar_full + 176, bar_read = bar_full + 192, bar_done = bar_full + 200,
                   bar_used = bar_full + 216, bar_tile = bar_full + 232, bar_free = bar_full + 264, bar_codes = bar_full + 296,
                   bar_taken = bar_full + 312;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(bar_full + 8 * i, 4);  // an arrival per converting warp
            mbar_init(bar_empty + 8 * i, 1);
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(bar_q + 8 * h, 1);
            mbar_init(bar_used + 8 * h, 1);
            mbar_init(bar_s + 8 * h, 1);
            mbar_init(bar_p + 8 * h, 4);  // an arrival per warp
            mbar_init(bar_pv + 8 * h, 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(bar_codes + 8 * x, 1);
            mbar_init(bar_taken + 8 * x, 4);
        }
        mbar_init(bar_read, 4);
        mbar_init(bar_done, 1);
        mbar_init(bar_done + 8, 1);
        for (int i = 0; i < kTiles; ++i) {
            s_bad[i] = 0;
            mbar_init(bar_tile + 8 * i, 1);
            mbar_init(bar_free + 8 * i, kReaders);
        }
        s_abort = 0;
        fence_barrier_init();
    }
    pdl_wait();  // before the tensor memory is taken: a kernel before this one may still need its own
    PagedCursor c = paged_find<false, kRows, kUnit, kWide8Overhead, kThreads>(w, blockIdx.x, gridDim.x, s_prefix);
    if (warp == kScores) tmem_alloc(smem_u32(&s_tmem), kCols);
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
            const int myrow = t.r0 + 128 * h + row, units = t.nu, p0 = t.p0, p1 = t.p1, table = t.ring >> 1, seen = t.seen;
            const bool idle = (warp & 3) * 32 >= hrows;  // no row of this warp exists
            const int limit = row < hrows ? paged_row_limit<false>(w, t.s, myrow) : 0;
            float mref = -INFINITY, l = 0.f;
            bool again = false;  // the row is one for large_row
            __syncwarp();  // tensor-memory instructions below are warp-wide
            for (int u = 0; u < units; ++u) {
                ok = __all_sync(0xffffffffu, tc_wait(bar_s + 8 * h, done_units & 1, abort, lim, kv.errors));
                if (!ok) break;
                tc_fence_after();
                const int base = p0 + u * kUnit;
                const float4* factor = s_factor[(table + u) % kTables];
                float s[128];
                if (!idle) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) tmem_ld32(lanes + 32 * q, s + 32 * q);
                    tmem_wait_ld();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_read);  // the score buffer may be written again
                if (__builtin_expect(!idle && base + kUnit > seen, 0)) {  // some row of the tile does not see all
                    const int sees = limit - base;
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = i < sees ? s[i] : -INFINITY;
                }
                __syncwarp();
                if (!idle) {
                    // The largest s + ev, and a new reference where it is more than 8 above. The maximum beside the weights,
                    // which are then computed twice where it moved, is no faster for even data and slower for keys with
                    // uneven channels and levels, whose maxima move (6500 positions, at an earlier stage: 255 and 285 us,
                    // so 257 and 267).
                    float m = -INFINITY;
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) {
                        const float4 fb = factor[b];
                        float mx[2] = {s[16 * b], s[16 * b + 1]};
#pragma unroll
                        for (int i = 1; i < 8; ++i) mx[i & 1] = max3(mx[i & 1], s[16 * b + 2 * i], s[16 * b + 2 * i + 1]);
                        m = fmaxf(m, fmaf(fmaxf(mx[0], mx[1]), fb.x, fb.y));
                    }
                    const bool move = u == 0 || m > mref + 8.f;
                    if (__builtin_expect(u > 0 && __any_sync(0xffffffffu, move), 0)) {
                        ok = __all_sync(0xffffffffu, tc_wait(bar_pv + 8 * h, (done_units - 1) & 1, abort, lim, kv.errors));
                        if (!ok) break;
                        tc_fence_after();
                        const float f = move ? ex2(0.5f * (mref - m)) : 1.f;  // in two steps: l may be as far from 1
                        l = l * f * f;
#pragma unroll 1
                        for (int q = 0; q < D / 16; ++q) {
                            float o[16];
                            tmem_ld16(t_o + 16 * q, o);
                            uint32_t o2[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) o2[i] = __float_as_uint(o[i] * f * f);
                            tmem_st16(t_o + 16 * q, o2);
                        }
                    }
                    if (move) mref = m;
                    again |= fabsf(mref) >= kLargeScore && mref != -INFINITY;
                    const float off = (mref == -INFINITY ? 0.f : -mref) + kLift;
                    const bool far = s_far[(table + u) % kTables];
                    if (__builtin_expect(far, 0)) {  // (before the weights, which let go of the scores)
                        const float up = off + (kFarLift - kLift);
                        float all = 0.f;
#pragma unroll
                        for (int b = 0; b < kBlocks; ++b) {
                            const float4 fb = factor[b];
                            float part = 0.f;
#pragma unroll
                            for (int i = 0; i < 16; ++i) part += ex2(fmaf(s[16 * b + i], fb.x, fb.y + up));
                            all = fmaf(part, fb.z * exp_scale(kLift - kFarLift), all);
                        }
                        l += all;
                    }
                    float sum = 0.f;
                    // The first kHeld quarters wait in registers for the product before, which still reads its weights.
                    constexpr int kHeld = 2;
                    uint32_t held[kHeld][16], now[16];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t(&pk)[16] = q < kHeld ? held[q < kHeld ? q : 0] : now;
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const float4 fb = factor[2 * q + b];
                            const uint64_t sc2 = f2(fb.x, fb.x), off2 = f2(fb.y + off, fb.y + off);
                            uint64_t part = 0;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float x = s[32 * q + 16 * b + 2 * i], y = s[32 * q + 16 * b + 2 * i + 1];
                                float a, d;
                                unf2(fma2(f2(x, y), sc2, off2), a, d);
                                a = ex2(a);
                                d = ex2(d);
                                part = add2(part, f2(a, d));
                                pk[8 * b + i] = pack_half2(a, d);
                            }
                            float a, d;
                            unf2(part, a, d);
                            sum = fmaf(a + d, fb.z, sum);
                        }
                        if (q == kHeld - 1 && u > 0) {  // it has read its weights and written its outputs
                            ok = __all_sync(0xffffffffu, tc_wait(bar_pv + 8 * h, (done_units - 1) & 1, abort, lim, kv.errors));
                            if (!ok) break;
                            tc_fence_after();
                        }
                        if (q == kHeld - 1) {
#pragma unroll
                            for (int e = 0; e < kHeld; ++e) tmem_st16(t_p + 16 * e, held[e]);
                        } else if (q >= kHeld) {
                            tmem_st16(t_p + 16 * q, now);
                        }
                    }
                    if (!ok) break;
                    if (!far) l += sum;
                    tmem_wait_st();
                } else if (u > 0) {
                    // A warp without rows arrives with the others all the same, and never a unit ahead of them: it, too, waits
                    // for the product before (its early arrival would count as another warp's).
                    ok = __all_sync(0xffffffffu, tc_wait(bar_pv + 8 * h, (done_units - 1) & 1, abort, lim, kv.errors));
                }
                if (!ok) break;
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
                const bool whole = t.whole;
                const int tok = w.by_G(myrow), head = t.j * w.G + myrow - tok * w.G;
                const int64_t orow = t.s.begin + tok;
                const int64_t at = int64_t(2 * blockIdx.x + (t.k0 == 0 ? 1 : 0)) * kRows + 128 * h + row;
                if (l == 0.f && min(limit, p1) > p0) mref = kLowest;  // no score but -inf
                // A part's reference is to be near its sum, so that parts are weighed by what they hold of the row: the
                // exponent of l goes into it, and out of l and the outputs.
                const int k = l > 0.f && l < INFINITY ? int(__float_as_uint(l) >> 23) - 127 : 0;
                mref += float(k);
                l *= exp_scale(-k);
                const float z = exp_scale(-k - kLift), inv = whole ? paged_inverse(mref, l) * z : z;
#pragma unroll
                for (int q = 0; q < D / 32; ++q) {
                    float o[32];
                    __syncwarp();
                    tmem_ld32(t_o + 32 * q, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= inv;
                    if (row < hrows && whole && !again) {  // (large_row reads the query, which may be where its output goes)
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<E*>(w.out) + orow * w.ldo + head * D + 32 * q);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            dst[i] = make_uint4(pack2<E>(o[8 * i], o[8 * i + 1]), pack2<E>(o[8 * i + 2], o[8 * i + 3]),
                                                pack2<E>(o[8 * i + 4], o[8 * i + 5]), pack2<E>(o[8 * i + 6], o[8 * i + 7]));
                    } else if (row < hrows && !whole) {
                        float* dst = w.part_o + at * D + 32 * q;
#pragma unroll
                        for (int i = 0; i < 4; ++i) store8(dst + 8 * i, o + 8 * i);
                    }
                }
                if (row < hrows) {
                    if (!whole)
                        w.part_ml[at] = make_float2(mref, l);
                    else if (w.lse)
                        w.lse[orow * w.ldl + head] = l != 0.f ? (mref + log2f(l)) * kLn2 : -INFINITY;
                }
            }
            if (__builtin_expect(again && row < hrows, 0))
                large_row<E, D>(w, p.sc, t, myrow, min(limit, p1), int64_t(2 * blockIdx.x + (t.k0 == 0 ? 1 : 0)) * kRows + 128 * h + row);
            if (s_bad[n % kTiles] == n + 1 && row < hrows) {  // the rows that see a NaN value
                const int tok = w.by_G(myrow), head = t.j * w.G + myrow - tok * w.G;
                const int64_t orow = t.s.begin + tok;
                const int64_t at = int64_t(2 * blockIdx.x + (t.k0 == 0 ? 1 : 0)) * kRows + 128 * h + row;
                bool page_ok = true;
#pragma unroll 1
                for (int pos = max(p0, t.seen); pos < min(p1, limit); ++pos) {
                    const uint8_t* v = static_cast<const uint8_t*>(kv.v) + paged_page(kv, t.s.table, pos, page_ok) * kv.vs_page +
                                       t.j * kv.vs_head + int64_t(pos & kv.page_mask) * kv.vs_slot;
#pragma unroll 1
                    for (int d = 0; d < D; ++d)
                        if ((v[d] & 0x7f) == 0x7f) {
                            if (t.whole)
                                reinterpret_cast<uint16_t*>(w.out)[orow * w.ldo + head * D + d] = 0x7fff;  // NaN in either type
                            else
                                w.part_o[at * D + d] = __uint_as_float(0x7fc00000u);
                        }
                }
            }
            __syncwarp();
            tc_fence_before();  // ordered before the next tile's first product by its bar_p arrivals
            release(n);
        }
    } else {
        // One instruction for each whole warpgroup, under a condition that its warps share: executed from different
        // places by its warps, it would be undefined.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp >= kConvert) {
            // -------------------------------------------------------- codes -> tiles
            const Piece<D> piece(warp - kConvert, lane);
            int it = 0;
            for (int n = 0;; ++n) {
                wait(bar_tile + 8 * (n % kTiles), n / kTiles);
                if (!ok || !tile(n).valid) break;
                const int units = tile(n).nu, p0 = tile(n).p0, p1 = tile(n).p1, seen = min(p1, tile(n).seen);
                release(n);
                for (int u = 0; ok && u < units; ++u) {
                    const int base = p0 + u * kUnit;
                    auto convert = [&](auto type, int x) {
                        using T = decltype(type);
                        const int st = it % ST;
                        wait(bar_codes + 8 * x, it >> 1);
                        if (ok && it >= ST) wait(bar_empty + 8 * st, it / ST + 1);
                        if (!ok) return;
                        const uint32_t src = sb + SM::kCodes + x * (SM::kTile / 2), dst = sb + SM::kRing + st * SM::kTile;
                        if (x == 1 && base + kUnit > seen) {  // rows of v that no position owns, or, where they are NaN, not every row sees
#pragma unroll 1
                            for (int k = 0; k < Piece<D>::kCount; ++k) {
                                const int pos = base + piece.row(k);
                                if (pos < seen) continue;
                                uint32_t q[4], bad = 0;
                                lds128(q, src + piece.from(k));
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint32_t out = pos < p1 ? nan4(q[e]) : 0xffffffffu;
                                    bad |= out;
                                    q[e] &= ~out;
                                }
                                if (bad) sts128(src + piece.from(k), q[0], q[1], q[2], q[3]);
                                if (bad && pos < p1) s_bad[n % kTiles] = n + 1;
                            }
                        }
                        // Rolled: with the pieces unrolled the roles' loops exceed the instruction cache, and every phase behind
                        // a wait begins with its misses (prompt of 6500 positions: all unrolled 314 us, pairs 260, so 251).
#pragma unroll 1
                        for (int k = 0; k < Piece<D>::kCount; ++k) {
                            uint32_t q[4];
                            lds128(q, src + piece.from(k));
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const uint2 lo = codes_to<T>(q[2 * half]), hi = codes_to<T>(q[2 * half + 1]);
                                sts128(dst + (piece.to(k) ^ (half << 4)), lo.x, lo.y, hi.x, hi.y);
                            }
                        }
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(bar_full + 8 * st);
                            mbar_arrive(bar_taken + 8 * x);
                        }
                        ++it;
                    };
                    convert(E(), 0);
                    if (ok) convert(__half(), 1);
                }
                if (!ok) break;
            }
        } else {
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            if (warp == kScores) {
                // ---------------------------------------------------- S = Q K^T
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
            } else if (warp == kOutputs) {
                // ---------------------------------------------------- O += P V
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
            } else if (warp == kWalker) {
                // ---------------------------------------------------- tiles and queries
                int used0 = 0, used1 = 0, ring = 0;  // tiles of each half, ring stages so far
                bool shares = false;                 // the last tile goes on in the next CTA
                for (int n = 0; ok; ++n) {
                    if (n >= kTiles) wait(bar_free + 8 * (n % kTiles), n / kTiles - 1);
                    if (!ok) break;
                    WideTile t;
                    t.valid = 0;
                    while (c.u < c.hi && c.b < kv.B) {  // past tiles of which this share holds only overhead
                        bool cut;
                        t.s = paged_seq<false>(w, s_prefix, c.b, cut);
                        const PagedSegment<false, kRows, kUnit, kWide8Overhead> g(w, t.s, c);
                        if (g.nu > 0) {
                            t.j = c.j;
                            t.r0 = c.i * kRows;
                            t.nrows = min(kRows, t.s.rows - t.r0);
                            t.k0 = g.k0;
                            t.nu = g.nu;
                            t.p0 = g.k0 * kUnit;
                            t.p1 = min(t.p0 + g.nu * kUnit, paged_tile_limit<false, kRows>(w, t.s, c.i));
                            t.whole = g.whole();
                            t.parts = g.parts(c, blockIdx.x);
                            t.ring = ring;
                            t.seen = paged_row_limit<false>(w, t.s, t.r0);
                            t.valid = 1;
                            paged_next<false, kRows>(w, s_prefix, c, g.cost);
                            break;
                        }
                        paged_next<false, kRows>(w, s_prefix, c, g.cost);
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
                        wide_queries<E, D>(w, &p.qmap, p.q_tma, t, h, lane, sb + h * SM::kTile, bar_q + 8 * h);
                        ++used;
                    }
                }
                if (lane == 0 && !shares) w.shared[blockIdx.x].parts = 0;
                // no queries may still be landing when the CTA leaves
                if (used0 > 0) tc_wait(bar_q, (used0 - 1) & 1, nullptr, lim, kv.errors);
                if (used1 > 0) tc_wait(bar_q + 8, (used1 - 1) & 1, nullptr, lim, kv.errors);
                __syncwarp();
            } else if (warp == kFetch) {
                // ---------------------------------------------------- codes and factors
                int unit = 0, values = 0, next = 0, nu = 0, u = 0, p0 = 0, p1 = 0, j = 0, page = 0, top = 0;
                uint32_t byte = 0;
                bool pages_ok = true;
                auto open = [&]() {  // the tile `next`; without one, nu = 0
                    nu = u = 0;
                    wait(bar_tile + 8 * (next % kTiles), next / kTiles);
                    if (!ok) return;
                    const WideTile& t = tile(next);
                    if (t.valid) nu = t.nu, p0 = t.p0, p1 = t.p1, j = t.j;
                };
                // Of its unit u: pages of the boxes, a lane each; then scales of its blocks, of k in lanes 0 .. 7, of v in
                // 8 .. 15. Asked for a unit ahead, between the waits for the converting warps.
                auto pages = [&]() {
                    const int at = p0 + u * kUnit + lane * p.box;
                    page = 0;
                    if (lane * p.box < kUnit && at < p1) page = paged_page(kv, tile(next).s.table, at, pages_ok);
                };
                auto scales = [&]() {
                    const int b = lane & 7, pos = p0 + u * kUnit + 16 * b, blk = (pos & kv.page_mask) >> p.sc.block_shift;
                    const int pg = __shfl_sync(0xffffffffu, page, 16 * b / p.box);
                    byte = kExpBias;
                    if (lane < 16 && pos < p1) byte = lane < 8 ? *k_scale(p.sc, pg, j, blk) : *v_scale(p.sc, pg, j, blk);
                };
                open();
                if (ok && nu > 0) {
                    pages();
                    scales();
                }
                while (ok && nu > 0) {
                    const int base = p0 + u * kUnit, slot = (base + lane * p.box) & kv.page_mask, here = page, end = p1, head = j;
                    const int nb = max(0, (min(kUnit, end - base) + p.box - 1) / p.box);  // boxes that hold positions
                    auto fetch = [&](int x) {
                        const uint32_t bar = bar_codes + 8 * x;
                        if (lane == 0) mbar_arrive_expect_tx(bar, uint32_t(nb * p.box) * D);
                        __syncwarp();
                        if (lane < nb) {
                            const int ps = x ? p.v_slot : p.k_slot, ph = x ? p.v_head : p.k_head;
                            const int c1 = ps == 1 ? slot : ph == 1 ? head : here, c2 = ps == 2 ? slot : ph == 2 ? head : here,
                                      c3 = ps == 3 ? slot : ph == 3 ? head : here;
                            tma_load_4d(sb + SM::kCodes + x * (SM::kTile / 2) + uint32_t(lane * p.box) * D, x ? &p.vmap : &p.kmap, 0, c1, c2, c3,
                                        bar);
                        }
                    };
                    if (unit > 0) wait(bar_taken, unit - 1);
                    if (!ok) break;
                    // the unit's factors, for which the arrival for its keys speaks, too
                    const int e = scale_exp(byte), ev = __shfl_down_sync(0xffffffffu, e, 8);
                    const bool live = lane < kBlocks && base + 16 * lane < end;
                    if (u == 0) top = -kExpMost;
                    top = max(top, __reduce_max_sync(0xffffffffu, live ? ev : -kExpMost));
                    const int least = __reduce_min_sync(0xffffffffu, live ? ev : kExpMost), y = live ? ev : 0;
                    if (lane < kBlocks)  // (a factor of zero would make NaN of a masked score)
                        s_factor[unit % kTables][lane] =
                            make_float4(fmaxf(w.scale_log2 * exp_scale(e), 0x1p-149f), float(y), exp_scale(-y - kLift), 0.f);
                    if (lane == 0) s_far[unit % kTables] = top - least > kSpread;
                    __syncwarp();
                    fetch(0);
                    if (++u == nu) {
                        release(next);
                        ++next;
                        open();
                        if (!ok) nu = 0;  // (the keys are on their way: the end below waits for them)
                    }
                    if (nu > 0) pages();
                    ++unit;
                    if (ok && unit > 1) wait(bar_taken + 8, unit - 2);
                    if (!ok) break;
                    fetch(1);
                    ++values;
                    if (nu > 0) scales();
                }
                if (!pages_ok) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
                // no codes may still be landing when the CTA leaves
                if (unit > 0) tc_wait(bar_codes, (unit - 1) & 1, nullptr, lim, kv.errors);
                if (values > 0) tc_wait(bar_codes + 8, (values - 1) & 1, nullptr, lim, kv.errors);
                __syncwarp();
            }
            if (warp <= kOutputs) {  // every product issued above has finished once this completes
                const uint32_t done = bar_done + 8 * (warp - kScores);
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
    if (warp == kScores) tmem_dealloc(tmem, kCols);
}

// Tensor map of pages of codes (strides st: page, head, slot): dims are D, then the other three in order of their
// strides; `slot` and `head` receive the coordinate (1 .. 3) of each.
int encode_codes(const bq_paged8_kv* kv, const void* base, const int64_t* st, int box, CUtensorMap* map, int32_t* slot, int32_t* head) {
    EncodeTiledFn enc = tensor_map_encoder();
    if (!enc) return set_error(BQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    struct Dim {
        int64_t stride, size;
        int what;  // 0 page, 1 head, 2 slot
    } d[3] = {{st[0], kv->num_pages, 0}, {st[1], kv->HKV, 1}, {st[2], kv->page_size, 2}};
    std::stable_sort(d, d + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    cuuint64_t dims[4] = {cuuint64_t(kv->D)}, strides[3];
    cuuint32_t boxes[4] = {cuuint32_t(kv->D)};
    const cuuint32_t es[4] = {1, 1, 1, 1};
    for (int i = 0; i < 3; ++i) {
        dims[i + 1] = cuuint64_t(d[i].size);
        strides[i] = cuuint64_t(d[i].size == 1 ? kv->D : d[i].stride);  // of one element: any that the encoder takes
        boxes[i + 1] = d[i].what == 2 ? cuuint32_t(box) : 1u;
        if (d[i].what == 2) *slot = i + 1;
        if (d[i].what == 1) *head = i + 1;
    }
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, boxes, es,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, kv->D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(BQ_ERR_CUDA, "cuTensorMapEncodeTiled (codes) failed (%d)", int(r));
    return BQ_OK;
}

}  // namespace

int paged8_launch_wide(const PagedWork& w, const Paged8Scales& sc, const bq_paged8_kv* kv, int grid, uint32_t flags, void* stream) {
    const int dtype = kv->dtype, D = kv->D;
    Wide8Params p;
    std::memset(&p, 0, sizeof(p));
    p.w = w;
    p.sc = sc;
    int rc;
    if (128 % w.G == 0) {
        rc = encode_queries(w, dtype, D, &p.qmap);
        if (rc) return rc;
        p.q_tma = 1;
    }
    p.box = std::min(kv->page_size, 128);
    rc = encode_codes(kv, kv->k_pages, kv->k_stride, p.box, &p.kmap, &p.k_slot, &p.k_head);
    if (!rc) rc = encode_codes(kv, kv->v_pages, kv->v_stride, p.box, &p.vmap, &p.v_slot, &p.v_head);
    if (rc) return rc;
    // kind::f16, fp32 accumulate; queries and keys of the rows' type, weights and values fp16; M = 128; N = 128 positions
    // / D dims (B dims-contiguous)
    const uint32_t type = dtype == BQ_DT_BF16 ? 1u : 0u, common = (1u << 4) | (uint32_t(128 >> 4) << 24);
    p.idesc_qk = common | (type << 7) | (type << 10) | (uint32_t(128 >> 3) << 17);
    p.idesc_pv = common | (1u << 16) | (uint32_t(D >> 3) << 17);
    // (a wait may have to outlast large_row for all positions of a share: 15 us each, and as much again; more than 2^20 of
    // them, all of rows that need it, end with the error bit of a wait that gave up)
    p.wait_cycles = kWaitCycles + std::min<int64_t>(int64_t(kv->max_pages) * kv->page_size, 1 << 20) * kLargeCycles;
    const bool bf = dtype == BQ_DT_BF16;
    const void* fn = D == 128 ? (bf ? reinterpret_cast<const void*>(&paged8_wide_kernel<__nv_bfloat16, 128>)
                                    : reinterpret_cast<const void*>(&paged8_wide_kernel<__half, 128>))
                              : (bf ? reinterpret_cast<const void*>(&paged8_wide_kernel<__nv_bfloat16, 64>)
                                    : reinterpret_cast<const void*>(&paged8_wide_kernel<__half, 64>));
    const uint32_t smem = D == 128 ? Wide8Smem<128>::kTotal : Wide8Smem<64>::kTotal;
    rc = ensure_smem_attr(fn, smem);
    if (rc) return rc;
    void* args[] = {&p};
    return paged_launch(fn, dim3(grid), dim3(kThreads), smem, args, flags, stream, "paged attention");
}

}  // namespace bq
