// bq_paged8_append: the new tokens' q / k / v rows of a projection into an 8-bit
// paged cache. Per head
//   h = x * rsqrt(mean(x^2) + eps) * gain        (when norm weights are given)
//   y = h * cos[pos] + rotate_half(h) * sin[pos]  (q and k heads; y = x for v)
// in fp32; q is rounded once to its type. k and v per block of positions and head:
// e = least with max |y| <= 448 * 2^e over the new tokens, not below the block's e
// so far where it holds older positions of the sequence (their codes follow when it
// grows), codes = e4m3(y * 2^-e).
//
// Bound: HBM for prompts (2 bytes read and 1 or 2 written per element), the latency
// of the dependent loads (row -> sequence -> length -> page -> scale -> store) for a
// decode step's handful of rows. A head of a row is a group of D / 8 lanes with 16
// bytes each, as in the 16-bit append: the norm and the largest magnitude are
// shuffles inside the group.
//
// Two forms. One new token per sequence: a group per head, its block's older codes
// (rarely) rescaled by the same group. Ragged rows: the tokens of a block share a
// scale, so a CTA takes all new tokens of a block of as many heads as its lanes hold in
// registers between the maximum and the codes; queries go to CTAs of their own.
//
// Measured in a graph: 2 rows of 48 heads 2.0 us, 160 rows of 48 heads 3.0 us (both the
// chain of loads) where no scale grows; a block whose scale does is rescaled position by
// position, each waiting for the one before, and the fullest such block sets the call's
// time: up to 8.3 us with blocks of 32, 14 with 64, 27 with 128. A few drafted rows of two
// streams of 48 heads 4.8 us; seven prompts of 28 heads of
// 64, blocks of 16, 26.9 MB in 11.5 us (2.3 TB/s: waves of short CTAs, each with its search
// for the sequence, its loads, one barrier and its stores). cos and sin are loaded a row
// ahead: loaded where they are used, each row waited for its own (prompts 15.0 us).
#include <algorithm>
#include <cstring>

#include "bq_host.h"
#include "bq_paged8.cuh"
#include "bq_paged8_host.h"

namespace bq {
namespace {

constexpr int kRowThreads = 128;    // one token per sequence
constexpr int kBlockThreads = 256;  // ragged rows
constexpr int kMostBlock = 128;
constexpr int kQueryHeads = 4;      // of a CTA of queries

struct Append8Params {
    PagedKV kv;
    Paged8Scales sc;
    int32_t rope_rows, has_norm;
    int32_t window, kv_ctas;  // rows of a CTA; CTAs along y of the k and v heads
    int32_t q_parts, q_sets;  // CTAs among which a window's queries are divided; a CTA's query heads / kQueryHeads
    float eps;
    const void* qkv;
    int64_t ldqkv;
    const void* cos;
    const void* sin;
    int64_t ldcs;
    const void* qn;
    const void* kn;
    void* q_out;
    int64_t ldq;
};

// Eight entries each of a position's cos and sin row, as they are in memory: loaded well
// before they are needed.
template <typename C>
struct Angle {
    static constexpr int N = sizeof(C) / 2;
    uint4 c[N], s[N];
    __device__ __forceinline__ void load(const Append8Params& p, int pos, int l) {
        const uint4* a = reinterpret_cast<const uint4*>(static_cast<const C*>(p.cos) + int64_t(pos) * p.ldcs + l * 8);
        const uint4* b = reinterpret_cast<const uint4*>(static_cast<const C*>(p.sin) + int64_t(pos) * p.ldcs + l * 8);
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = a[i], s[i] = b[i];
    }
    __device__ static __forceinline__ void unpack(const uint4 (&w)[N], float (&v)[8]) {
        if constexpr (N == 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[4 * i] = __uint_as_float(w[i].x), v[4 * i + 1] = __uint_as_float(w[i].y);
                v[4 * i + 2] = __uint_as_float(w[i].z), v[4 * i + 3] = __uint_as_float(w[i].w);
            }
        } else {
            unpack8<C>(w[0], v);
        }
    }
};

// Norm and rotation of one head: lane l of its group holds dims 8 l .. 8 l + 7. Every
// lane of the warp calls it (the shuffles are the warp's).
template <typename E, typename C, int D>
__device__ __forceinline__ void turn(const Append8Params& p, const Angle<C>& at, int l, const uint4& gain, float (&v)[8]) {
    constexpr int LG = D / 8;
    float c[8], s[8];
    Angle<C>::unpack(at.c, c);
    Angle<C>::unpack(at.s, s);
    if (p.has_norm) {
        float g[8], ss = 0.f;
        unpack8<E>(gain, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
        for (int m = LG / 2; m; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        const float inv = rsqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * g[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float other = __shfl_xor_sync(0xffffffffu, v[i], LG / 2);
        v[i] = v[i] * c[i] + (l < LG / 2 ? -other : other) * s[i];
    }
}

template <typename E>
__device__ __forceinline__ uint4 gain_of(const Append8Params& p, const void* gain, int l) {
    return p.has_norm ? *reinterpret_cast<const uint4*>(static_cast<const E*>(gain) + l * 8) : make_uint4(0, 0, 0, 0);
}

// Largest finite magnitude, as its bits (they order as the values do).
__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
        if (a < 0x7f800000u) t = max(t, a);
    }
    return t;
}
// Least e from -60 to 60 with top <= 448 * 2^e; 448 is 1.75 * 2^8.
__device__ __forceinline__ int need_exp(uint32_t top) {
    const int e = int(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, -kExpMost), kExpMost);
}
__device__ __forceinline__ uint2 encode8(const float (&v)[8], int e) {
    const float r = exp_scale(-e);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (__float_as_uint(v[i]) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : v[i] * r;
    return make_uint2(f32_codes(x[0], x[1]) | f32_codes(x[2], x[3]) << 16, f32_codes(x[4], x[5]) | f32_codes(x[6], x[7]) << 16);
}
// Codes times 2^d, d <= 0.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float r) {
    float v[4];
    codes_f32(w, v);
    return f32_codes(v[0] * r, v[1] * r) | f32_codes(v[2] * r, v[3] * r) << 16;
}

// The codes and the scale of one head's block: `at` and `scale` point to slot 0 and to
// the block's byte.
struct BlockAt {
    uint8_t* codes;
    int64_t slot;  // stride
    uint8_t* scale;
};
// Head h counts k heads, then v heads.
__device__ __forceinline__ BlockAt block_at(const Append8Params& p, int h, int page, int slot0) {
    const PagedKV& kv = p.kv;
    const int blk = slot0 >> p.sc.block_shift;
    BlockAt a;
    if (h < kv.HKV) {
        a.codes = static_cast<uint8_t*>(kv.k) + page * kv.ks_page + h * kv.ks_head + slot0 * kv.ks_slot;
        a.slot = kv.ks_slot;
        a.scale = const_cast<uint8_t*>(k_scale(p.sc, page, h, blk));
    } else {
        a.codes = static_cast<uint8_t*>(kv.v) + page * kv.vs_page + (h - kv.HKV) * kv.vs_head + slot0 * kv.vs_slot;
        a.slot = kv.vs_slot;
        a.scale = const_cast<uint8_t*>(v_scale(p.sc, page, h - kv.HKV, blk));
    }
    return a;
}

// ---------------------------------------------------------------- one new token per sequence
template <typename E, typename C, int D>
__global__ void __launch_bounds__(kRowThreads) append8_rows_kernel(const __grid_constant__ Append8Params p) {
    constexpr int LG = D / 8;  // lanes per head
    constexpr int HEADS = kRowThreads / LG;
    pdl_launch_dependents();
    pdl_wait();
    const PagedKV& kv = p.kv;
    const int b = blockIdx.x;
    const int l = threadIdx.x % LG;
    const int h = blockIdx.y * HEADS + threadIdx.x / LG;
    const int heads = kv.HQ + 2 * kv.HKV;
    const bool live = h < heads;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live) raw = *reinterpret_cast<const uint4*>(static_cast<const E*>(p.qkv) + int64_t(b) * p.ldqkv + h * D + l * 8);
    const uint4 gain = gain_of<E>(p, h < kv.HQ ? p.qn : p.kn, l);
    const int pos = max(kv.lens[b], 0) - 1;
    if (pos < 0) return;  // an unused batch slot
    bool ok = pos < p.rope_rows && (pos >> kv.page_shift) < kv.max_pages;
    if (!ok) {
        if (threadIdx.x == 0) atomicOr(kv.errors, BQ_DEVERR_POSITION_BIT);
        return;
    }
    const bool turns = blockIdx.y * HEADS < kv.HQ + kv.HKV;  // block-uniform: some head of this block is a q or k head
    Angle<C> angle;
    if (turns) angle.load(p, pos, l);
    const int page = paged_page(kv, b, pos, ok);
    if (!ok) {
        if (threadIdx.x == 0) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
        return;
    }
    const int slot = pos & kv.page_mask, kept = slot & ((1 << p.sc.block_shift) - 1);
    const bool cached = live && h >= kv.HQ;
    BlockAt at;
    int was = -kExpMost;
    if (cached) {
        at = block_at(p, h - kv.HQ, page, slot - kept);
        if (kept) was = scale_exp(*at.scale);
    }
    float v[8];
    unpack8<E>(raw, v);
    if (turns) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = v[i];
        turn<E, C, D>(p, angle, l, gain, y);
        if (h < kv.HQ + kv.HKV) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = y[i];
        }
    }
    uint32_t top = top_of(v);
#pragma unroll
    for (int m = LG / 2; m; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
    if (!live) return;
    if (!cached) {
        *reinterpret_cast<uint4*>(static_cast<E*>(p.q_out) + int64_t(b) * p.ldq + h * D + l * 8) = pack8<E>(v);
        return;
    }
    const int need = need_exp(top), e = kept ? max(was, need) : need;
    if (e > was && kept) {  // the block's older codes follow
        const float r = exp_scale(was - e);
#pragma unroll 4
        for (int s = 0; s < kept; ++s) {
            uint2* c = reinterpret_cast<uint2*>(at.codes + s * at.slot + l * 8);
            const uint2 w = *c;
            *c = make_uint2(rescale4(w.x, r), rescale4(w.y, r));
        }
    }
    *reinterpret_cast<uint2*>(at.codes + kept * at.slot + l * 8) = encode8(v, e);
    if (l == 0) *at.scale = uint8_t(e + kExpBias);
}

// ---------------------------------------------------------------- ragged rows
// The part of a sequence in a window of rows.
struct Segment {
    int lo, hi;      // rows of the window that are its
    int begin, end;  // all its rows
    int pos;         // position of row `begin` (negative: rows before the first position)
    int b;
};

// All threads: the sequences that have rows in [w0, w1), in any order.
__device__ __forceinline__ int find_segments(const PagedKV& kv, int w0, int w1, Segment* seg, int* count) {
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
    for (int b = threadIdx.x; b < kv.B; b += kBlockThreads) {
        int begin, n;
        paged_rows(kv, b, begin, n);
        const int lo = max(begin, w0), hi = min(begin + n, w1);
        if (lo >= hi) continue;
        const int i = atomicAdd(count, 1);
        if (i < kMostBlock) seg[i] = Segment{lo, hi, begin, begin + n, max(kv.lens[b], 0) - n, b};
    }
    __syncthreads();
    return min(*count, kMostBlock);  // (more only where starts are out of order)
}

// R: rows of a block that each group of lanes holds: block / R groups take a head's block, GROUPS R / block heads the CTA.
// As few as give each CTA one head, but for short blocks, of which it takes several heads (blocks of 16 rows of 64 dims:
// 1 row 13.1 us, 2 rows 11.5, 4 rows 12.9). With two rows three CTAs run on an SM (80 registers, up to 88 bytes of them
// spilled with fp32 tables), with more two (three, spilling: 400 rows of 16 kv heads 11.0 against 7.0 us). Eight rows
// (blocks of 128 positions of 128 dims) spill 180 to 344 bytes at two, too: 2020 rows of 48 heads take 16.0 us in blocks
// of 64 and 20.9 in blocks of 128.
template <typename E, typename C, int D, int R>
__global__ void __launch_bounds__(kBlockThreads, R == 2 ? 3 : 2) append8_blocks_kernel(const __grid_constant__ Append8Params p) {
    constexpr int LG = D / 8, GROUPS = kBlockThreads / LG;
    __shared__ Segment seg[kMostBlock];
    __shared__ int s_count, s_pos[kMostBlock];
    __shared__ uint32_t s_top[2][kBlockThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const PagedKV& kv = p.kv;
    const int l = threadIdx.x % LG, g = threadIdx.x / LG;
    int w0 = blockIdx.x * p.window, w1 = min(w0 + p.window, kv.T), h0 = 0;
    const bool queries = int(blockIdx.y) >= p.kv_ctas;
    if (queries) {  // of some heads and a part of the window
        const int y = blockIdx.y - p.kv_ctas, part = y % p.q_parts;
        h0 = y / p.q_parts * (p.q_sets * kQueryHeads);
        w0 += part * (p.window / p.q_parts);
        w1 = min(w1, w0 + p.window / p.q_parts);
        if (w0 >= w1) return;
    }
    const int n_seg = find_segments(kv, w0, w1, seg, &s_count);
    const int block = 1 << p.sc.block_shift;

    if (queries) {
        for (int r = threadIdx.x; r < w1 - w0; r += kBlockThreads) {
            int pos = -1;
            for (int i = 0; i < n_seg; ++i)
                if (w0 + r >= seg[i].lo && w0 + r < seg[i].hi) {
                    pos = seg[i].pos + (w0 + r - seg[i].begin);
                    bool ok = pos < p.rope_rows && (pos >> kv.page_shift) < kv.max_pages;
                    if (ok && pos >= 0) paged_page(kv, seg[i].b, pos, ok);  // a token that has no page is skipped whole
                    if (!ok) pos = -1;                                      // (its k and v set the error bit)
                }
            s_pos[r] = pos;
        }
        __syncthreads();
        // A group takes the heads of one row at a time, the next row's on their way meanwhile. (q may be written where qkv
        // is read: the next row is another one.)
        const uint4 gain = gain_of<E>(p, p.qn, l);
        uint4 raw[kQueryHeads];
        Angle<C> angle;
        auto row_at = [&](int r) { return static_cast<const E*>(p.qkv) + int64_t(w0 + r) * p.ldqkv + l * 8; };
        auto load = [&](const E* row, int q) { raw[q] = *reinterpret_cast<const uint4*>(row + min(h0 + q, kv.HQ - 1) * D); };
        const int per = GROUPS / p.q_sets;  // rows at a time; the sets of heads beside one another
        h0 += g / per * kQueryHeads;
        int next = min(g % per, w1 - w0 - 1);
        angle.load(p, max(s_pos[next], 0), l);
#pragma unroll
        for (int q = 0; q < kQueryHeads; ++q) load(row_at(next), q);
        for (int r0 = 0; r0 < w1 - w0; r0 += per) {  // all lanes of a warp stay for the shuffles
            const int r = r0 + g % per;
            const bool here = r < w1 - w0 && s_pos[r] >= 0;
            const Angle<C> at = angle;
            next = min(r + per, w1 - w0 - 1);
            angle.load(p, max(s_pos[next], 0), l);
#pragma unroll
            for (int q = 0; q < kQueryHeads; ++q) {
                float v[8];
                unpack8<E>(raw[q], v);
                load(row_at(next), q);
                turn<E, C, D>(p, at, l, gain, v);
                if (here && h0 + q < kv.HQ)
                    *reinterpret_cast<uint4*>(static_cast<E*>(p.q_out) + int64_t(w0 + r) * p.ldq + (h0 + q) * D + l * 8) = pack8<E>(v);
            }
        }
        return;
    }

    const int mine = block / R, item = g / mine, gi = g - item * mine;  // groups of a head; its index and the group's in it
    const int h = min(int(blockIdx.y) * (GROUPS / mine) + item, 2 * kv.HKV - 1);  // k heads, then v heads
    const bool live = int(blockIdx.y) * (GROUPS / mine) + item < 2 * kv.HKV, is_k = h < kv.HKV;
    const int warp0 = item * mine * LG / 32, warps = mine * LG / 32;  // the head's warps
    const uint4 gain = gain_of<E>(p, p.kn, l);
    int turnover = 0;
    for (int i = 0; i < n_seg; ++i) {
        const Segment s = seg[i];
        // blocks whose first new token lies in the window: the sequence's first one, and those at a block's start
        int r0 = s.lo, p0 = s.pos + (r0 - s.begin);
        if (p0 < 0) {
            r0 -= p0;
            p0 = 0;
        }
        if (r0 != s.begin && (p0 & (block - 1))) {
            const int skip = block - (p0 & (block - 1));
            r0 += skip;
            p0 += skip;
        }
        while (r0 < s.hi) {
            const int kept = p0 & (block - 1), rows = min(s.end - r0, block - kept);
            const int n = min(rows, max(0, p.rope_rows - p0));
            bool ok = (p0 >> kv.page_shift) < kv.max_pages;
            if ((!ok || n < rows) && threadIdx.x == 0) atomicOr(kv.errors, BQ_DEVERR_POSITION_BIT);
            ok = ok && n > 0;
            int page = 0;
            uint4 raw[R];
            Angle<C> angle;  // of the group's next row
            if (ok) {
                const E* src = static_cast<const E*>(p.qkv) + int64_t(r0) * p.ldqkv + (kv.HQ + h) * D + l * 8;
#pragma unroll
                for (int q = 0; q < R; ++q) {
                    raw[q] = make_uint4(0, 0, 0, 0);
                    if (gi + q * mine < n) raw[q] = *reinterpret_cast<const uint4*>(src + int64_t(gi + q * mine) * p.ldqkv);
                }
                if (is_k) angle.load(p, p0 + min(gi, n - 1), l);  // (the same for a warp)
                page = paged_page(kv, s.b, p0, ok);
                if (!ok && threadIdx.x == 0) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
            }
            if (ok) {  // (the same for all threads)
                const int slot = p0 & kv.page_mask;
                const BlockAt at = block_at(p, h, page, slot - kept);
                const int was = kept ? scale_exp(*at.scale) : -kExpMost;
                float v[R][8];
                uint32_t top = 0;
#pragma unroll
                for (int q = 0; q < R; ++q) {
                    if (q * mine >= n) continue;  // (the same for all threads)
                    unpack8<E>(raw[q], v[q]);
                    if (is_k) {
                        const Angle<C> now = angle;
                        if (q + 1 < R) angle.load(p, p0 + min(gi + (q + 1) * mine, n - 1), l);
                        turn<E, C, D>(p, now, l, gain, v[q]);
                    }
                    if (gi + q * mine < n) top = max(top, top_of(v[q]));
                }
                top = __reduce_max_sync(0xffffffffu, top);
                if ((threadIdx.x & 31) == 0) s_top[turnover][threadIdx.x >> 5] = top;
                __syncthreads();
                for (int w = 0; w < warps; ++w) top = max(top, s_top[turnover][warp0 + w]);
                turnover ^= 1;  // the next block's maxima go elsewhere: one barrier per block is enough
                const int need = need_exp(top), e = kept ? max(was, need) : need;
                if (live && kept && e > was) {  // the block's older codes follow
                    const float r = exp_scale(was - e);
                    for (int q = gi; q < kept; q += mine) {
                        uint2* c = reinterpret_cast<uint2*>(at.codes + q * at.slot + l * 8);
                        const uint2 w = *c;
                        *c = make_uint2(rescale4(w.x, r), rescale4(w.y, r));
                    }
                }
                if (live) {
#pragma unroll
                    for (int q = 0; q < R; ++q)
                        if (gi + q * mine < n)
                            *reinterpret_cast<uint2*>(at.codes + (kept + gi + q * mine) * at.slot + l * 8) = encode8(v[q], e);
                    if (gi == 0 && l == 0) *at.scale = uint8_t(e + kExpBias);
                }
            }
            r0 += rows;
            p0 += rows;
        }
    }
}

template <typename E, typename C, int D>
const void* blocks_kernel(int r) {
    if constexpr (kMostBlock * (D / 8) == 8 * kBlockThreads)  // blocks of 128 positions of 128 dims
        if (r == 8) return reinterpret_cast<const void*>(&append8_blocks_kernel<E, C, D, 8>);
    return r == 2 ? reinterpret_cast<const void*>(&append8_blocks_kernel<E, C, D, 2>)
                  : reinterpret_cast<const void*>(&append8_blocks_kernel<E, C, D, 4>);
}
template <typename E, typename C>
const void* append_kernel(int D, bool rows, int r) {
    if (rows)
        return D == 128 ? reinterpret_cast<const void*>(&append8_rows_kernel<E, C, 128>)
                        : reinterpret_cast<const void*>(&append8_rows_kernel<E, C, 64>);
    return D == 128 ? blocks_kernel<E, C, 128>(r) : blocks_kernel<E, C, 64>(r);
}

}  // namespace
}  // namespace bq

using namespace bq;

extern "C" int32_t bq_paged8_append(const bq_paged8_append_desc* d, void* stream) {
    if (!d) return set_error(BQ_ERR_INVALID_ARG, "desc is NULL");
    int rc = paged8_validate(&d->kv, d->T, d->HQ);
    if (rc) return rc;
    if (d->T == 0) return BQ_OK;
    const int width = (d->HQ + 2 * d->kv.HKV) * d->kv.D;
    if (d->cs_dtype != d->kv.dtype && d->cs_dtype != BQ_DT_F32)
        return set_error(BQ_ERR_INVALID_ARG, "cos / sin must have the rows' dtype or fp32 (dtype %d)", d->cs_dtype);
    if (!d->qkv || !d->cos || !d->sin || !d->q_out)
        return set_error(BQ_ERR_INVALID_ARG, "qkv, cos, sin and q_out must be non-NULL");
    if ((d->q_norm == nullptr) != (d->k_norm == nullptr))
        return set_error(BQ_ERR_INVALID_ARG, "q_norm and k_norm must be given together");
    if (d->ldqkv < width) return set_error(BQ_ERR_SHAPE, "ldqkv=%lld < %d", (long long)d->ldqkv, width);
    if (d->ldq < d->HQ * d->kv.D) return set_error(BQ_ERR_SHAPE, "ldq=%lld < %d", (long long)d->ldq, d->HQ * d->kv.D);
    if (d->rope_rows < 1 || d->ldcs < d->kv.D)
        return set_error(BQ_ERR_SHAPE, "cos / sin need rows of %d elements (got %d rows of stride %lld)", d->kv.D,
                         d->rope_rows, (long long)d->ldcs);
    const int cs = dtype_size(d->cs_dtype);
    if (!paged_aligned(d->qkv, d->ldqkv, 2) || !paged_aligned(d->q_out, d->ldq, 2) || !paged_aligned(d->cos, d->ldcs, cs) ||
        !paged_aligned(d->sin, d->ldcs, cs) || !paged_aligned(d->q_norm, 0, 2) || !paged_aligned(d->k_norm, 0, 2))
        return set_error(BQ_ERR_ALIGN, "qkv, cos, sin, q_out and norm rows must be 16-byte aligned");
    if (2 * d->kv.HKV + (d->HQ + kQueryHeads - 1) / kQueryHeads * 8 > 65535)
        return set_error(BQ_ERR_SHAPE, "%d query and %d kv heads are too many", d->HQ, d->kv.HKV);
    rc = paged_check_device();
    if (rc) return rc;
    Append8Params p;
    std::memset(&p, 0, sizeof(p));
    rc = paged8_fill(&p.kv, &p.sc, &d->kv, d->T, d->HQ);
    if (rc) return rc;
    p.rope_rows = d->rope_rows;
    p.has_norm = d->q_norm != nullptr;
    p.eps = d->eps;
    p.qkv = d->qkv;
    p.ldqkv = d->ldqkv;
    p.cos = d->cos;
    p.sin = d->sin;
    p.ldcs = d->ldcs;
    p.qn = d->q_norm;
    p.kn = d->k_norm;
    p.q_out = d->q_out;
    p.ldq = d->ldq;
    const bool f32 = d->cs_dtype == BQ_DT_F32, bf = d->kv.dtype == BQ_DT_BF16, rows = !d->kv.q_starts;
    const int lanes = d->kv.D / 8, r = std::max(2, d->kv.block * lanes / kBlockThreads);
    const void* fn = bf ? (f32 ? append_kernel<__nv_bfloat16, float>(d->kv.D, rows, r)
                               : append_kernel<__nv_bfloat16, __nv_bfloat16>(d->kv.D, rows, r))
                        : (f32 ? append_kernel<__half, float>(d->kv.D, rows, r) : append_kernel<__half, __half>(d->kv.D, rows, r));
    void* args[] = {&p};
    if (rows) {
        const int heads = d->HQ + 2 * d->kv.HKV, per = kRowThreads / lanes;
        return paged_launch(fn, dim3(d->T, (heads + per - 1) / per), dim3(kRowThreads), 0, args, d->flags, stream, "paged append");
    }
    p.window = paged8_window(&d->kv, d->T, d->kv.block);
    const int heads = kBlockThreads / lanes * r / d->kv.block;  // of a CTA
    p.kv_ctas = (2 * d->kv.HKV + heads - 1) / heads;
    // Queries: a short window's rows do not fill a CTA, which takes several sets of heads then (prompts with blocks of 16:
    // 14.7 -> 11.5 us). A long one's are divided among CTAs until there are three for every SM (400 rows of 16 heads: undivided
    // 8.0 us, in four 7.0; 8000 of 32: 60 and 74 us).
    const DeviceInfo* di = device_info();
    if (!di) return BQ_ERR_CUDA;
    p.q_parts = p.q_sets = 1;
    while (2 * p.q_sets * p.window * lanes <= kBlockThreads) p.q_sets *= 2;
    const int windows = (d->T + p.window - 1) / p.window, q_heads = (d->HQ + p.q_sets * kQueryHeads - 1) / (p.q_sets * kQueryHeads);
    while (2 * p.q_parts * kBlockThreads <= p.window * lanes && int64_t(windows) * q_heads * p.q_parts < 3 * di->sm_count) p.q_parts *= 2;
    return paged_launch(fn, dim3(windows, p.kv_ctas + q_heads * p.q_parts),
                        dim3(kBlockThreads), 0, args, d->flags, stream, "paged append");
}
