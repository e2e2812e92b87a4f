// Paged attention for tiles of many rows (prompts, a prefix shared by a batch)
// on the tcgen05 tensor cores: 256 rows per CTA in two halves of 128, keys and
// values in units of 128 positions.
//
// Bound: tensor cores and, as close, the exponentials: a half's unit is two
// products of 128 x 128 x D (512 cycles each at D = 128) and 128 x 128
// exponentials (1024 cycles on an SM's 16 lanes). So the two halves take turns:
// while one half's scores go through the softmax warps, the tensor cores
// multiply for the other. Both halves use the same k / v tiles, which halves
// what the tiles cost in L2 reads (32 bytes per cycle and SM).
//
// Roles (10 warps, one CTA per SM, all 512 tensor-memory columns):
//   warps 0-3, 4-7  softmax of half 0 / 1, one row per thread: the row's 128
//                   scores from tensor memory, running maximum and sum, the
//                   probabilities back to tensor memory in 16 bits over the
//                   scores' columns (they are the A operand of the second
//                   product). The output accumulator stays in tensor memory; a
//                   row's reference maximum may lag behind the true one by up
//                   to a factor 2^8 (probabilities up to 256 are exact enough
//                   in either type, and the factor cancels), so the accumulator
//                   is rescaled only when a maximum really moves.
//   warp 8          k and v by tiled TMA, one box per page (or 128 positions of
//                   one) and 64 dims, into a ring of 32 KB stages
//   warp 9          one thread issues the products: S = Q K^T (both operands in
//                   shared memory, K-major) and O += P V (A in tensor memory, V
//                   as stored, dims contiguous)
// Page slots behind the last position arrive with the last page, whatever they
// hold; before the product that would multiply them by zero probabilities the
// softmax warps of half 0 clear those rows of v. Scores there are never used.
#include <algorithm>
#include <cstring>

#include "bq_host.h"
#include "bq_paged.cuh"
#include "bq_paged_host.h"
#include "bq_tmem.cuh"

namespace bq {

struct PagedWideParams {
    CUtensorMap kmap, vmap;  // (D, then slot, head and page in order of stride); boxes of 64 dims x positions of one page
    PagedWork w;
    int32_t box;                          // positions per box: min(page size, 128)
    int32_t k_slot, k_head, v_slot, v_head;  // which of coordinates 1 .. 3 is the slot, the head (the third is the page)
    uint32_t idesc_qk, idesc_pv;
    long long wait_cycles;
};

namespace {

constexpr int kThreads = 320;
constexpr int kRows = kWideRows, kUnit = kWideUnit;
constexpr uint32_t kCols = 512;

template <int D>
struct WideSmem {
    static constexpr uint32_t kTile = 128 * D * 2;                   // one k or v tile, one half of the queries
    static constexpr int kStages = D == 128 ? 4 : 8;
    static constexpr uint32_t kRing = 2 * kTile;
    static constexpr uint32_t kBars = kRing + kStages * kTile;
    static constexpr uint32_t kTotal = kBars + 256 + 1024;           // + slack to align the tiles to 1024 bytes
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}

// D[tmem] (+)= A[smem] . B[smem]^T, one 128 x N x 16 step.
__device__ __forceinline__ void tc_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Descriptor of a v tile as the B operand with its dims (N) contiguous: rows of
// 64 dims (128 B, 128-byte swizzle), one row per position; groups of 8
// positions are 1024 B apart (stride offset), the second 64 dims 128 rows
// further (leading offset).
__device__ __forceinline__ uint64_t tc_vdesc(uint32_t saddr) {
    return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t((128 * 128) >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) |
           (uint64_t(2) << 61);
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

// What every role derives for the tile at the cursor.
struct WideTile {
    PagedSeq s;
    int units, nu, p0, p1, r0, nrows;
    __device__ __forceinline__ WideTile(const PagedWork& w, const PagedCursor& c) {
        bool cut;
        s = paged_seq(w, c.b, cut);
        const int limit = paged_tile_limit<kRows>(w, s, c.i);
        units = paged_tile_units<kRows, kUnit>(w, s, c.i);
        nu = int(min((long long)(units - c.k), c.hi - c.u));
        p0 = (w.prefix_pass ? 0 : w.prefix_len) + c.k * kUnit;
        p1 = min(p0 + nu * kUnit, limit);
        r0 = c.i * kRows;
        nrows = min(kRows, s.rows - r0);
    }
};

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, 1) paged_wide_kernel(const __grid_constant__ PagedWideParams p) {
    using SM = WideSmem<D>;
    constexpr int ST = SM::kStages, CH = D / 8;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    const uint32_t sraw = smem_u32(smem_raw), sb = (sraw + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (sb - sraw);
    const PagedWork& w = p.w;
    const PagedKV& kv = w.kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort = &s_abort;
    const long long lim = p.wait_cycles;
    // full / empty per ring stage; per half: queries staged, scores ready, probabilities written, output complete
    const uint32_t bar_full = sb + SM::kBars, bar_empty = bar_full + 64, bar_q = bar_full + 128, bar_s = bar_full + 144,
                   bar_p = bar_full + 160, bar_o = bar_full + 176, bar_done = bar_full + 192;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(bar_full + 8 * i, 1);
            mbar_init(bar_empty + 8 * i, 1);
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(bar_q + 8 * h, 128);
            mbar_init(bar_s + 8 * h, 1);
            mbar_init(bar_p + 8 * h, 128);
            mbar_init(bar_o + 8 * h, 1);
        }
        mbar_init(bar_done, 1);
        s_abort = 0;
        fence_barrier_init();
    }
    pdl_wait();  // before the tensor memory is taken: a kernel before this one may still need its own
    PagedCursor c = paged_find<kRows, kUnit, kThreads>(w, blockIdx.x, gridDim.x);
    if (warp == 9) tmem_alloc(smem_u32(&s_tmem), kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = s_tmem;  // scores / probabilities of half h at columns 128 h, outputs at 256 + 128 h
    const int sequences = w.prefix_pass ? 1 : kv.B;

    if (warp < 8) {
        // ------------------------------------------------------------ softmax of one half
        const int h = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
        const uint32_t t_s = lanes + 128 * h, t_o = lanes + 256 + 128 * h;
        int seg = 0, ph_s = 0, it = 0;  // tiles of this half done, score phases, ring stages passed
        bool ok = true, shares = false;  // shares: the last tile goes on in the next CTA
        for (; ok && c.u < c.hi && c.b < sequences;) {
            const WideTile t(w, c);
            const int hrows = t.nrows - 128 * h;  // valid rows of this half
            if (hrows > 0) {
                for (int idx = row; idx < 128 * CH; idx += 128) {
                    const int r = idx / CH, ch = idx - r * CH;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (r < hrows) {
                        const int rr = t.r0 + 128 * h + r, tok = w.by_G(rr);
                        v = *reinterpret_cast<const uint4*>(static_cast<const E*>(w.q) + int64_t(t.s.begin + tok) * w.ldq +
                                                            (c.j * w.G + rr - tok * w.G) * D + ch * 8);
                    }
                    *reinterpret_cast<uint4*>(smem + h * SM::kTile + (ch >> 3) * (128 * 128) + r * 128 +
                                              (((ch & 7) ^ (r & 7)) << 4)) = v;
                }
                fence_async_smem();
                mbar_arrive(bar_q + 8 * h);
                const int myrow = t.r0 + 128 * h + row;
                const int limit = row < hrows ? paged_row_limit(w, t.s, myrow) : 0;
                const bool idle = (warp & 3) * 32 >= hrows;  // no row of this warp exists
                __syncwarp();
                float mref = -INFINITY, l = 0.f;
                for (int u = 0; u < t.nu; ++u) {
                    ok = __all_sync(0xffffffffu, tc_wait(bar_s + 8 * h, ph_s & 1, abort, lim));
                    if (!ok) break;
                    ++ph_s;
                    tc_fence_after();
                    const int base = t.p0 + u * kUnit;
                    if (!idle) {
                        float s[128];
#pragma unroll
                        for (int q = 0; q < 4; ++q) tmem_ld32(t_s + 32 * q, s + 32 * q);
                        tmem_wait_ld();
                        if (base + kUnit > limit) {
                            const int n = limit - base;
#pragma unroll
                            for (int i = 0; i < 128; ++i) s[i] = i < n ? s[i] : -INFINITY;
                        }
                        __syncwarp();  // tensor-memory instructions below are warp-wide
                        float m = s[0];
#pragma unroll
                        for (int i = 1; i < 128; ++i) m = fmaxf(m, s[i]);
                        m *= w.scale_log2;
                        const bool move = m > mref + 8.f;  // also the first finite maximum
                        if (__any_sync(0xffffffffu, move)) {
                            const float f = move ? ex2(mref - m) : 1.f;
                            if (move) mref = m;
                            l *= f;
                            if (u > 0) {
#pragma unroll
                                for (int q = 0; q < D / 16; ++q) {
                                    float o[16];
                                    tmem_ld16(t_o + 16 * q, o);
                                    uint32_t o2[16];
#pragma unroll
                                    for (int i = 0; i < 16; ++i) o2[i] = __float_as_uint(o[i] * f);
                                    tmem_st16(t_o + 16 * q, o2);
                                }
                            }
                        }
                        const float off = mref == -INFINITY ? 0.f : mref;
                        float l0 = 0.f, l1 = 0.f;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint32_t pk[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float a = ex2(fmaf(s[32 * q + 2 * i], w.scale_log2, -off));
                                const float b = ex2(fmaf(s[32 * q + 2 * i + 1], w.scale_log2, -off));
                                l0 += a;
                                l1 += b;
                                pk[i] = pack2<E>(a, b);
                            }
                            tmem_st16(t_s + 16 * q, pk);
                        }
                        l += l0 + l1;
                        tmem_wait_st();
                    }
                    if (h == 0 && base + kUnit > t.p1) {  // rows of v that no position owns
                        const int st = (it + 1) % ST, from = max(0, t.p1 - base);
                        ok = __all_sync(0xffffffffu, tc_wait(bar_full + 8 * st, ((it + 1) / ST) & 1, abort, lim));
                        if (!ok) break;
                        const uint4 z = make_uint4(0, 0, 0, 0);
                        for (int idx = row; idx < (128 - from) * CH; idx += 128) {
                            const int r = from + idx / CH, ch = idx % CH;
                            *reinterpret_cast<uint4*>(smem + SM::kRing + st * SM::kTile + (ch >> 3) * (128 * 128) + r * 128 +
                                                      ((ch & 7) << 4)) = z;
                        }
                        fence_async_smem();
                        __syncwarp();
                    }
                    it += 2;
                    tc_fence_before();
                    mbar_arrive(bar_p + 8 * h);
                }
                if (ok) ok = __all_sync(0xffffffffu, tc_wait(bar_o + 8 * h, seg & 1, abort, lim));
                if (!ok) break;
                ++seg;
                tc_fence_after();
                const bool whole = c.k == 0 && t.nu == t.units, final = whole && !w.row_o;
                const int parts = whole || c.k ? 0 : c.share.owner(c.u + t.units - 1) - int(blockIdx.x) + 1;
                if (parts) {
                    shares = true;
                    if (threadIdx.x == 0) w.shared[blockIdx.x] = PagedShared{parts, t.nrows, t.r0, t.s.begin, c.j};
                }
                if (!idle) {
                    const int tok = w.by_G(myrow), head = c.j * w.G + myrow - tok * w.G;
                    const int64_t orow = t.s.begin + tok;
                    const int64_t at = whole ? orow * kv.HQ + head
                                             : int64_t(2 * blockIdx.x + (c.k == 0 ? 1 : 0)) * kRows + 128 * h + row;
                    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
                    for (int q = 0; q < D / 16; ++q) {
                        float o[16];
                        __syncwarp();
                        tmem_ld16(t_o + 16 * q, o);
                        if (row < hrows && final) {
                            uint4* dst = reinterpret_cast<uint4*>(static_cast<E*>(w.out) + orow * w.ldo + head * D + 16 * q);
                            uint4 a, b;
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] *= inv;
                            a = make_uint4(pack2<E>(o[0], o[1]), pack2<E>(o[2], o[3]), pack2<E>(o[4], o[5]), pack2<E>(o[6], o[7]));
                            b = make_uint4(pack2<E>(o[8], o[9]), pack2<E>(o[10], o[11]), pack2<E>(o[12], o[13]),
                                           pack2<E>(o[14], o[15]));
                            dst[0] = a;
                            dst[1] = b;
                        } else if (row < hrows) {
                            float4* dst = reinterpret_cast<float4*>((whole ? w.row_o : w.part_o) + at * D + 16 * q);
#pragma unroll
                            for (int i = 0; i < 4; ++i) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                    }
                    if (row < hrows) {
                        if (!final) {
                            (whole ? w.row_ml : w.part_ml)[at] = make_float2(mref, l);
                            if (w.row_at && c.k == 0)
                                w.row_at[orow * kv.HQ + head] = paged_row_at(blockIdx.x, parts, 128 * h + row);
                        } else if (w.lse) {
                            w.lse[orow * w.ldl + head] = l > 0.f ? (mref + log2f(l)) * kLn2 : -INFINITY;
                        }
                    }
                }
                __syncwarp();
                tc_fence_before();  // ordered before the next tile's first product by its bar_p arrivals
            } else {
                it += 2 * t.nu;
            }
            c.u += t.nu;
            paged_next<kRows, kUnit>(w, c);
        }
        if (threadIdx.x == 0 && !shares) w.shared[blockIdx.x].parts = 0;
    } else if (warp == 8) {
        // ------------------------------------------------------------ k / v loads
        int it = 0;
        bool ok = true, pages_ok = true;
        for (; ok && c.u < c.hi && c.b < sequences;) {
            const WideTile t(w, c);
            for (int u = 0; ok && u < t.nu; ++u) {
                const int base = t.p0 + u * kUnit;
                const int nb = max(0, (min(kUnit, t.p1 - base) + p.box - 1) / p.box);  // boxes that hold positions
                int page = 0;
                if (lane < nb) page = paged_page(kv, c.b, base + lane * p.box, pages_ok);
                const int slot = (base + lane * p.box) & kv.page_mask;
#pragma unroll
                for (int x = 0; x < 2; ++x, ++it) {
                    const int st = it % ST;
                    const uint32_t bar = bar_full + 8 * st;
                    if (it >= ST) ok = __all_sync(0xffffffffu, tc_wait(bar_empty + 8 * st, ((it / ST) + 1) & 1, abort, lim));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(bar, uint32_t(nb * p.box) * (D * 2));
                    __syncwarp();
                    if (lane < nb) {
                        const CUtensorMap* map = x ? &p.vmap : &p.kmap;
                        const int ps = x ? p.v_slot : p.k_slot, ph = x ? p.v_head : p.k_head;
                        const int c1 = ps == 1 ? slot : ph == 1 ? c.j : page, c2 = ps == 2 ? slot : ph == 2 ? c.j : page,
                                  c3 = ps == 3 ? slot : ph == 3 ? c.j : page;
                        const uint32_t dst = sb + SM::kRing + st * SM::kTile + uint32_t(lane * p.box) * 128u;
#pragma unroll
                        for (int half = 0; half < D / 64; ++half)
                            tma_load_4d(dst + half * (128 * 128), map, half * 64, c1, c2, c3, bar);
                    }
                }
            }
            c.u += t.nu;
            paged_next<kRows, kUnit>(w, c);
        }
        if (!pages_ok) atomicOr(&g_device_error, BQ_DEVERR_PAGE_BIT);
        // no tile may still be landing when the CTA leaves (an abort skips the products)
        for (int i = max(0, it - ST); i < it; ++i) tc_wait(bar_full + 8 * (i % ST), (i / ST) & 1, nullptr, lim);
        __syncwarp();
    } else {
        // ------------------------------------------------------------ products
        if (lane == 0) {
            int it = 0, ph_q[2] = {0, 0}, ph_p[2] = {0, 0};
            bool ok = true;
            auto scores = [&](int h, int st) {  // S(h) = Q(h) K^T
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t at = (k >> 2) * (128 * 128) + 32 * (k & 3);
                    tc_mma_ss(tmem + 128 * h, tc_bdesc(sb + h * SM::kTile + at), tc_bdesc(sb + SM::kRing + st * SM::kTile + at),
                              p.idesc_qk, k > 0);
                }
                tc_commit(bar_s + 8 * h);
            };
            for (; ok && c.u < c.hi && c.b < sequences;) {
                const WideTile t(w, c);
                const int halves = t.nrows > 128 ? 2 : 1;
                ok = tc_wait(bar_full + 8 * (it % ST), (it / ST) & 1, abort, lim);
                for (int h = 0; ok && h < halves; ++h) {
                    ok = tc_wait(bar_q + 8 * h, ph_q[h]++ & 1, abort, lim);
                    if (!ok) break;
                    tc_fence_after();
                    scores(h, it % ST);
                }
                if (ok) tc_commit(bar_empty + 8 * (it % ST));
                for (int u = 0; ok && u < t.nu; ++u, it += 2) {
                    const int vs = (it + 1) % ST, ks = (it + 2) % ST;
                    const bool more = u + 1 < t.nu;
                    for (int h = 0; h < halves; ++h) {
                        ok = tc_wait(bar_p + 8 * h, ph_p[h]++ & 1, abort, lim);
                        if (ok && h == 0) ok = tc_wait(bar_full + 8 * vs, ((it + 1) / ST) & 1, abort, lim);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int k = 0; k < 8; ++k)  // O(h) += P(h) V, 16 positions per step
                            tc_mma(tmem + 256 + 128 * h, tmem + 128 * h + 8 * k,
                                   tc_vdesc(sb + SM::kRing + vs * SM::kTile + 2048 * k), p.idesc_pv, (u > 0 || k > 0) ? 1u : 0u);
                        if (h == halves - 1) tc_commit(bar_empty + 8 * vs);
                        if (more) {
                            if (h == 0) ok = tc_wait(bar_full + 8 * ks, ((it + 2) / ST) & 1, abort, lim);
                            if (!ok) break;
                            scores(h, ks);
                            if (h == halves - 1) tc_commit(bar_empty + 8 * ks);
                        } else {
                            tc_commit(bar_o + 8 * h);
                        }
                    }
                }
                c.u += t.nu;
                paged_next<kRows, kUnit>(w, c);
            }
            tc_commit(bar_done);  // every product issued above has finished once this completes
            tc_wait(bar_done, 0, nullptr, lim);
        }
        __syncwarp();
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
        strides[i] = cuuint64_t(d[i].stride) * 2;
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

}  // namespace

int paged_launch_wide(const PagedWork& w, const bq_paged_kv* kv, int grid, uint32_t flags, void* stream) {
    PagedWideParams p;
    std::memset(&p, 0, sizeof(p));
    p.w = w;
    p.box = std::min(kv->page_size, 128);
    int rc = encode_pages(kv, kv->k_pages, kv->k_stride, p.box, &p.kmap, &p.k_slot, &p.k_head);
    if (!rc) rc = encode_pages(kv, kv->v_pages, kv->v_stride, p.box, &p.vmap, &p.v_slot, &p.v_head);
    if (rc) return rc;
    // kind::f16, fp32 accumulate; A and B of the pages' type; M = 128; N = 128 positions / D dims (B dims-contiguous)
    const uint32_t type = kv->dtype == BQ_DT_BF16 ? 1u : 0u;
    const uint32_t common = (1u << 4) | (type << 7) | (type << 10) | (uint32_t(128 >> 4) << 24);
    p.idesc_qk = common | (uint32_t(128 >> 3) << 17);
    p.idesc_pv = common | (1u << 16) | (uint32_t(kv->D >> 3) << 17);
    p.wait_cycles = kWaitCycles;
    const bool bf = kv->dtype == BQ_DT_BF16;
    const void* fn = kv->D == 128 ? (bf ? reinterpret_cast<const void*>(&paged_wide_kernel<__nv_bfloat16, 128>)
                                        : reinterpret_cast<const void*>(&paged_wide_kernel<__half, 128>))
                                  : (bf ? reinterpret_cast<const void*>(&paged_wide_kernel<__nv_bfloat16, 64>)
                                        : reinterpret_cast<const void*>(&paged_wide_kernel<__half, 64>));
    const uint32_t smem = kv->D == 128 ? WideSmem<128>::kTotal : WideSmem<64>::kTotal;
    rc = ensure_smem_attr(fn, smem);
    if (rc) return rc;
    void* args[] = {&p};
    return paged_launch(fn, dim3(grid), dim3(kThreads), smem, args, flags, stream, "paged attention");
}

}  // namespace bq
