// Attention over an 8-bit paged cache for tiles of many rows (prompts) on the tcgen05
// tensor cores: 256 rows per CTA in two halves of 128, keys and values in units of 128
// positions, laid out as in the 16-bit kernel (bq_paged_wide.cu): the halves take turns
// in one score buffer, probabilities and outputs stay in tensor memory, roles walk
// ahead. What differs is how k and v come in, and the scales.
//
// The tensor cores take both operands in one type, so codes are converted: four warps
// copy them (cp.async, one unit ahead, each lane what it will convert itself) and write
// them as 16-bit tiles in the swizzled layout of the products, once for the 256 rows.
// Keys become the queries' type, values fp16; either holds every code exactly. Queries
// split into e4m3 terms would leave the keys as they are, but probabilities need more
// range than e4m3 has, so values have to be converted all the same.
//
// Scales: 2^ek multiplies the scores of a block, 2^ev goes into the exponent of its
// probabilities, as in the kernel for few rows: the weights are 2^(s + ev - M + 7), M a
// reference that may lag behind the largest s + ev by up to 8, so at most 2^15 in fp16.
// The converting warps leave each unit's eight pairs of factors in shared memory. Where
// the ev of a unit lie more than 100 below one of the tile so far, weights that fp32
// flushes might still count in the sum of exponentials, which is then computed on its own.
//
// Roles (one CTA per SM, all 512 tensor-memory columns): warps 0-3, 4-7 softmax of half
// 0 / 1; 8 issues the scores' products, 9 the outputs'; 10 walks the tiles and fetches
// their queries; 12-15 convert.
#include "bq_paged8.cuh"
#include "bq_paged8_host.h"
#include "bq_paged_wide.cuh"

namespace bq {

struct Wide8Params {
    CUtensorMap qmap;  // (D, heads, rows), boxes of 64 dims x 128 rows
    PagedWork w;
    Paged8Scales sc;
    int32_t q_tma;     // the queries come by TMA
    uint32_t idesc_qk, idesc_pv;
    long long wait_cycles;
};

namespace {

constexpr int kThreads = 512;
// Registers: the CTA starts with 512 x 128; the third and fourth warpgroup give up what the softmax warps, a row of
// 128 scores per thread, need more (256 x 208 + 256 x 48). The file is compiled as a whole program, since relocatable
// code may not move registers.
constexpr int kSoftmaxRegs = 208, kOtherRegs = 48;
constexpr int kScores = 8, kOutputs = 9, kWalker = 10, kConvert = 12;  // warps of the roles behind the softmax
constexpr int kReaders = 14;      // warps that read a tile of the walker's
constexpr int kBlocks = kUnit / 16;
constexpr int kLift = 7, kFarLift = 64;  // weights are kept times 2^7; where that is not enough, their sum is of 2^64 times
constexpr int kSpread = 100;

template <int D>
struct Wide8Smem {
    static constexpr uint32_t kTile = 128 * D * 2;                   // one k or v tile, one half of the queries
    static constexpr int kStages = D == 128 ? 4 : 8;
    // Units whose factors are kept. When those of unit U are written, its keys' stage is free: the scores of unit
    // U - kStages / 2 have been multiplied, so that both halves have read those of the unit before and are done with
    // all before that.
    static constexpr int kTables = kStages / 2 + 2;
    static constexpr uint32_t kRing = 2 * kTile;
    static constexpr uint32_t kCodes = kRing + kStages * kTile;      // the codes of a k and a v tile on their way
    static constexpr uint32_t kBars = kCodes + kTile;
    static constexpr uint32_t kTotal = kBars + 512 + 1024;           // + slack to align the tiles to 1024 bytes
};

// NaN among four codes: 0xff in its byte.
__device__ __forceinline__ uint32_t nan4(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

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

// A lane's 16-byte pieces of a 128-position tile: rows row(k), codes 16 c .. 16 c + 15. Eight neighbouring lanes have
// two rows that differ in bit 0, so that their swizzled chunks fall on different banks.
template <int D>
struct Piece {
    static constexpr int kRowsPerWarp = D == 128 ? 4 : 8, kCount = 128 / (4 * kRowsPerWarp);
    int warp, first, c;
    __device__ __forceinline__ Piece(int warp_, int lane)
        : warp(warp_), first(kRowsPerWarp * warp_ + (lane >> 2) % kRowsPerWarp), c((lane & 3) + (D == 128 ? (lane >> 4) * 4 : 0)) {}
    __device__ __forceinline__ int row(int k) const { return 4 * kRowsPerWarp * k + first; }
    __device__ __forceinline__ int block(int k) const { return D == 128 ? k : 2 * k + (warp >> 1); }  // of 16 positions
    // of the first of its two chunks in a tile; the second is at ^ 16
    __device__ __forceinline__ uint32_t at(int k) const {
        const int r = row(k);
        return (c >> 2) * (128 * 128) + r * 128 + ((((c & 3) * 2) ^ (r & 7)) << 4);
    }
};

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, 1) paged8_wide_kernel(const __grid_constant__ Wide8Params p) {
    using SM = Wide8Smem<D>;
    constexpr int ST = SM::kStages, kTables = SM::kTables;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ PagedPrefix s_prefix;  // (none: the shared pieces want one)
    __shared__ WideTile s_tile[kTiles];
    __shared__ volatile int s_bad[kTiles];   // n + 1: NaN entries of v were cleared from tile n
    __shared__ float2 s_factor[kTables][kBlocks];  // per block: scores times x, plus y, in base 2
    __shared__ int s_far[kTables];           // the unit's sum of exponentials needs the longer way
    const uint32_t sraw = smem_u32(smem_raw), sb = (sraw + 1023u) & ~1023u;
    const PagedWork& w = p.w;
    const PagedKV& kv = w.kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort = &s_abort;
    const long long lim = p.wait_cycles;
    // full / empty per ring stage; per half: queries staged, scores ready, probabilities written, second product
    // complete, queries used; scores read; per tile in s_tile: written, read by all its readers
    const uint32_t bar_full = sb + SM::kBars, bar_empty = bar_full + 64, bar_q = bar_full + 128, bar_s = bar_full + 144,
                   bar_p = bar_full + 160, bar_pv = bar_full + 176, bar_read = bar_full + 192, bar_done = bar_full + 200,
                   bar_used = bar_full + 216, bar_tile = bar_full + 232, bar_free = bar_full + 264;
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
            const int myrow = t.r0 + 128 * h + row, units = t.nu, p0 = t.p0, p1 = t.p1, table = t.ring >> 1;
            const bool idle = (warp & 3) * 32 >= hrows;  // no row of this warp exists
            const int limit = row < hrows ? paged_row_limit<false>(w, t.s, myrow) : 0;
            float mref = -INFINITY, l = 0.f;
            __syncwarp();  // tensor-memory instructions below are warp-wide
            for (int u = 0; u < units; ++u) {
                ok = __all_sync(0xffffffffu, tc_wait(bar_s + 8 * h, done_units & 1, abort, lim, kv.errors));
                if (!ok) break;
                tc_fence_after();
                const int base = p0 + u * kUnit;
                const float2* factor = s_factor[(table + u) % kTables];
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
                    mref = -INFINITY;
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) {
                        float mx = s[16 * b];
#pragma unroll
                        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[16 * b + i]);
                        mref = fmaxf(mref, fmaf(mx, factor[b].x, factor[b].y));
                    }
                }
                __syncwarp();
                // A warp without rows arrives with the others all the same, and never a unit ahead of them: it, too, waits
                // for the product before (its early arrival would count as another warp's).
                if (idle && u > 0) ok = __all_sync(0xffffffffu, tc_wait(bar_pv + 8 * h, (done_units - 1) & 1, abort, lim, kv.errors));
                if (!ok) break;
                // Weights against the reference as it stands, and the maximum beside them; only where a
                // maximum turns out to have moved by more than the allowance are they computed once more.
                bool again = !idle, first = u > 0;
                while (again) {
                    const float off = (mref == -INFINITY ? 0.f : -mref) + kLift;
                    float m = -INFINITY, sum = 0.f;
                    // The first kHeld quarters wait in registers for the product before, which still reads its weights.
                    constexpr int kHeld = 2;
                    uint32_t held[kHeld][16], now[16];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t(&pk)[16] = q < kHeld ? held[q < kHeld ? q : 0] : now;
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const float2 fb = factor[2 * q + b];
                            const uint64_t sc2 = f2(fb.x, fb.x), off2 = f2(fb.y + off, fb.y + off);
                            uint64_t part = 0;
                            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float x = s[32 * q + 16 * b + 2 * i], y = s[32 * q + 16 * b + 2 * i + 1];
                                mx[i & 1] = max3(mx[i & 1], x, y);
                                float a, d;
                                unf2(fma2(f2(x, y), sc2, off2), a, d);
                                a = ex2(a);
                                d = ex2(d);
                                part = add2(part, f2(a, d));
                                pk[8 * b + i] = pack_half2(a, d);
                            }
                            float a, d;
                            unf2(part, a, d);
                            sum = fmaf(a + d, exp_scale(-int(fb.y) - kLift), sum);
                            m = fmaxf(m, fmaf(fmaxf(mx[0], mx[1]), fb.x, fb.y));
                        }
                        if (q == kHeld - 1 && first) {  // it has read its weights and written its outputs
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
                    const bool move = m > mref + 8.f;  // also the first finite maximum
                    again = __any_sync(0xffffffffu, move);
                    if (again) {
                        tmem_wait_st();  // the weights are about to be written again, and stores have no order of their own
                        const float f = move ? ex2(0.5f * (mref - m)) : 1.f;  // in two steps: l may be as far from 1
                        mref = move ? m : mref;
                        l = l * f * f;
                        if (u > 0) {
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
                    } else {
                        if (s_far[(table + u) % kTables]) {
                            sum = 0.f;
                            const float far = (mref == -INFINITY ? 0.f : -mref) + kFarLift;
#pragma unroll
                            for (int b = 0; b < kBlocks; ++b) {
                                const float2 fb = factor[b];
                                float part = 0.f;
#pragma unroll
                                for (int i = 0; i < 16; ++i) part += ex2(fmaf(s[16 * b + i], fb.x, fb.y + far));
                                sum = fmaf(part, exp_scale(-int(fb.y) - kFarLift), sum);
                            }
                        }
                        l += sum;
                        tmem_wait_st();
                    }
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
                    if (row < hrows && whole) {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<E*>(w.out) + orow * w.ldo + head * D + 32 * q);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            dst[i] = make_uint4(pack2<E>(o[8 * i], o[8 * i + 1]), pack2<E>(o[8 * i + 2], o[8 * i + 3]),
                                                pack2<E>(o[8 * i + 4], o[8 * i + 5]), pack2<E>(o[8 * i + 6], o[8 * i + 7]));
                    } else if (row < hrows) {
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
            const uint32_t codes = sb + SM::kCodes + (threadIdx.x & 127) * 16;
            bool pages_ok = true;
            int next = 0, nu = 0, np0 = 0, np1 = 0, u_next = 0, page = 0, nj = 0;  // the unit to be copied: tile, units, ...
            auto open = [&]() {  // the tile `next`; without one, nu = 0
                wait(bar_tile + 8 * (next % kTiles), next / kTiles);
                nu = 0;
                u_next = 0;
                if (!ok) return;
                const WideTile& t = tile(next);
                if (!t.valid) return;
                nu = t.nu, np0 = t.p0, np1 = t.p1, nj = t.j;
            };
            auto look = [&]() {  // the pages of its blocks of 16 positions, a lane each
                const int pos = np0 + u_next * kUnit + 16 * lane;
                page = 0;
                if (nu > 0 && lane < kBlocks && pos < np1) page = paged_page(kv, tile(next).s.table, pos, pages_ok);
            };
            auto copy = [&](int x) {  // its keys (0) or values (1)
                if (nu > 0) {
                    const int base = np0 + u_next * kUnit;
                    const uint8_t* from = static_cast<const uint8_t*>(x ? kv.v : kv.k) + nj * (x ? kv.vs_head : kv.ks_head) + piece.c * 16;
                    const int64_t st_page = x ? kv.vs_page : kv.ks_page, st_slot = x ? kv.vs_slot : kv.ks_slot;
#pragma unroll
                    for (int k = 0; k < Piece<D>::kCount; ++k) {
                        const int pos = base + piece.row(k), pg = __shfl_sync(0xffffffffu, page, piece.block(k));
                        cp_async16_zfill(codes + x * (SM::kTile / 2) + k * 2048, from + pg * st_page + (pos & kv.page_mask) * st_slot,
                                         pos < np1);
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            open();
            look();
            int here = page;  // pages of the unit to be converted
            copy(0);
            copy(1);
            int it = 0, top = 0;
            for (int n = 0; ok && nu > 0;) {
                const int u = u_next, units = nu, p0 = np0, p1 = np1, j = nj, base = p0 + u * kUnit;
                const int seen = tile(n).seen;
                if (++u_next == nu) {
                    ++next;
                    open();
                    if (!ok) break;
                }
                look();
                uint32_t byte = kExpBias;  // lanes 0 .. 7: of k, 8 .. 15: of v
                if (piece.warp == 0) {
                    const int b = lane & 7, pg = __shfl_sync(0xffffffffu, here, b), pos = base + 16 * b,
                              blk = (pos & kv.page_mask) >> p.sc.block_shift;
                    if (lane < 16 && pos < p1) byte = lane < 8 ? *k_scale(p.sc, pg, j, blk) : *v_scale(p.sc, pg, j, blk);
                }
#pragma unroll 1
                for (int x = 0; ok && x < 2; ++x, ++it) {
                    const int st = it % ST;
                    if (it >= ST) wait(bar_empty + 8 * st, it / ST + 1);
                    if (!ok) break;
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    const uint32_t dst = sb + SM::kRing + st * SM::kTile;
#pragma unroll
                    for (int k = 0; k < Piece<D>::kCount; ++k) {
                        uint32_t q[4];
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3])
                                     : "r"(codes + x * (SM::kTile / 2) + k * 2048) : "memory");
                        if (x == 1 && base + piece.row(k) >= seen) {  // a value that not every row sees
                            uint32_t bad = 0;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t nan = nan4(q[e]);
                                bad |= nan;
                                q[e] &= ~nan;
                            }
                            if (bad) s_bad[n % kTiles] = n + 1;
                        }
                        const uint32_t a = dst + piece.at(k);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint2 lo = x ? codes_to<__half>(q[2 * half]) : codes_to<E>(q[2 * half]),
                                        hi = x ? codes_to<__half>(q[2 * half + 1]) : codes_to<E>(q[2 * half + 1]);
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a ^ (half << 4)), "r"(lo.x), "r"(lo.y), "r"(hi.x),
                                         "r"(hi.y) : "memory");
                        }
                    }
                    if (x == 0 && piece.warp == 0) {  // the unit's factors
                        const int e = scale_exp(byte), ev = __shfl_down_sync(0xffffffffu, e, 8);
                        const bool live = lane < kBlocks && base + 16 * lane < p1;
                        if (u == 0) top = -kExpMost;
                        top = max(top, __reduce_max_sync(0xffffffffu, live ? ev : -kExpMost));
                        const int least = __reduce_min_sync(0xffffffffu, live ? ev : kExpMost), slot = (it >> 1) % kTables;
                        if (lane < kBlocks) s_factor[slot][lane] = make_float2(fmaxf(w.scale_log2 * exp_scale(e), 1e-37f), live ? float(ev) : 0.f);
                        if (lane == 0) s_far[slot] = top - least > kSpread;
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_full + 8 * st);
                    copy(x);
                }
                if (!ok) break;
                here = page;
                if (u + 1 == units) {
                    release(n);
                    ++n;
                }
            }
            if (!pages_ok) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
            asm volatile("cp.async.wait_all;" ::: "memory");
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

}  // namespace

int paged8_launch_wide(const PagedWork& w, const Paged8Scales& sc, int dtype, int D, int grid, uint32_t flags, void* stream) {
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
    // kind::f16, fp32 accumulate; queries and keys of the rows' type, weights and values fp16; M = 128; N = 128 positions
    // / D dims (B dims-contiguous)
    const uint32_t type = dtype == BQ_DT_BF16 ? 1u : 0u, common = (1u << 4) | (uint32_t(128 >> 4) << 24);
    p.idesc_qk = common | (type << 7) | (type << 10) | (uint32_t(128 >> 3) << 17);
    p.idesc_pv = common | (1u << 16) | (uint32_t(D >> 3) << 17);
    p.wait_cycles = kWaitCycles;
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
