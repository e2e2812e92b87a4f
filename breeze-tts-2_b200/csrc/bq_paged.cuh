// Shared pieces of the paged KV-cache operators (bq_paged_append,
// bq_paged_attention): the cache as the kernels see it, bounds-checked page
// lookup, and 16-byte vector conversions of the two element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "bq_device.cuh"

namespace bq {

// A paged cache and the batch that uses it. Strides are in elements; every
// offset that contains a page index is formed in 64 bits.
struct PagedKV {
    int32_t B, HKV, page_shift, page_mask, num_pages, max_pages, T, HQ;
    void* k;
    int64_t ks_page, ks_head, ks_slot;
    void* v;
    int64_t vs_page, vs_head, vs_slot;
    const int32_t* table;
    int64_t ld_table;
    const int32_t* lens;
    const int32_t* starts;  // NULL: one new token per sequence
    unsigned int* errors;   // the device error word
};

// Rows [begin, begin + count) of the new tokens belong to sequence b. Values
// outside [0, T] or out of order are cut to rows that exist.
__device__ __forceinline__ void paged_rows(const PagedKV& kv, int b, int& begin, int& count) {
    if (!kv.starts) {
        begin = b;
        count = 1;
        return;
    }
    begin = min(max(kv.starts[b], 0), kv.T);
    const int end = min(max(kv.starts[b + 1], 0), kv.T);
    count = max(end - begin, 0);
}

// Cache length of sequence b, cut to what the page table can hold.
__device__ __forceinline__ int paged_len(const PagedKV& kv, int b, bool& cut) {
    const int len = kv.lens[b];
    const int64_t cap = int64_t(kv.max_pages) * (kv.page_mask + 1);
    cut = len > cap;
    return cut ? int(cap) : len;
}

// Page of position pos of sequence b (pos < max_pages * page size); an entry
// outside [0, num_pages) clears `ok` and reads page 0 instead, so no address
// leaves the cache.
__device__ __forceinline__ int paged_page(const PagedKV& kv, int b, int pos, bool& ok) {
    const int page = kv.table[int64_t(b) * kv.ld_table + (pos >> kv.page_shift)];
    const bool good = page >= 0 && page < kv.num_pages;
    ok = ok && good;
    return good ? page : 0;
}

// Division of 0 <= n < 2^31 by a constant of the launch: the round-up multiplier
// of Granlund and Montgomery ("Division by invariant integers using
// multiplication"), so that walking tiles and rows costs no integer division.
struct FastDiv {
    uint32_t mul, shift;
    __host__ void set(uint32_t d) {
        shift = 0;
        while ((uint64_t(1) << shift) < d) ++shift;
        mul = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ int operator()(int n) const {
        return int((__umulhi(mul, uint32_t(n)) + uint32_t(n)) >> shift);
    }
};

// ---------------------------------------------------------------- schedule
// The attention kernels cut the batch into tiles of ROWS rows -- row r of
// sequence b and kv head j is query head j * G + r % G of token r / G, so the
// query heads that share a kv head share a tile -- and each tile's positions
// into units of UNIT. All units of the batch, in (sequence, kv head, tile,
// position) order, are dealt to the CTAs in equal contiguous shares: however
// uneven the lengths, every CTA has the same work. A tile costs its units plus
// OVERHEAD more for its start and end (queries in, outputs out): the CTA whose
// share holds only those does nothing for the tile. A tile
// that ends up in several CTAs leaves one partial (largest score, sum of
// exponentials, unnormalized output) per CTA; a CTA can only share its first
// and its last tile, so two partial slots per CTA hold them all, and a second
// kernel joins them in CTA order (deterministic; no counters, no atomics).
//
// With a shared prefix there are two such schedules: the prefix over all rows
// of the batch at once (one pseudo-sequence), and each sequence's own positions
// from prefix_len on. The prefix's pages are those of the longest sequence that
// has new rows, as far as it goes (PagedPrefix): an unused slot's table entries
// are not looked at.
struct PagedShared {
    int32_t parts, rows, r0, begin, j;  // CTAs that hold it (0: none), its rows, first row, first token of the sequence, kv head
};

struct PagedWork {
    PagedKV kv;
    int32_t G, causal, prefix_len, prefix_pass;  // prefix_pass: this launch handles [0, prefix_len) for all rows
    FastDiv by_G;
    float scale_log2;                            // scale * log2(e): scores are kept in base 2
    const void* q;
    int64_t ldq;
    void* out;
    int64_t ldo;
    float* lse;
    int64_t ldl;
    float* part_o;     // [2 grid][ROWS][D] unnormalized outputs of shared tiles
    float2* part_ml;   // [2 grid][ROWS] (largest score, sum of exponentials)
    PagedShared* shared;  // [grid] the shared tile that begins in each CTA
    // with a prefix every row is joined from both passes' parts:
    float* row_o;      // [T][HQ][D] parts of tiles that one CTA holds
    float2* row_ml;    // [T][HQ]
    int2* row_at;      // [T][HQ] where the row's parts are (paged_row_at)
};

// A part of a row is its largest score m, its sum of exponentials l and its unnormalized outputs. A part that saw no
// position has m = -inf, l = 0; one that saw nothing but scores of -inf has m = kLowest, l = 0. A row of which no part
// saw any position is zeros, a row of which all scores are -inf is 0 / 0.
constexpr float kLowest = -3.402823466e38f;
__device__ __forceinline__ float paged_inverse(float m, float l) { return l != 0.f || m != -INFINITY ? 1.f / l : 0.f; }

// Where a row's parts of one pass are: x = CTA of the first, y = parts << 8 | row
// within the tile; no parts: in the row buffers.
__device__ __forceinline__ int2 paged_row_at(int cta, int parts, int row) { return make_int2(cta, parts << 8 | row); }

struct PagedSeq {
    int begin, count, rows, len, off;  // first row, new rows, rows * G, positions, position of the first new row
    int table;                         // its row of the page table
};

// The prefix pass's sequence: the row of the table that it reads, the positions that any row sees, those that
// every row sees (rows that see nothing aside).
struct PagedPrefix {
    int table, len, seen;
};

// PREFIX: the launch handles the prefix. A parameter of the kernels, since as a flag that they look at it takes the
// few-row kernel without a prefix from 38.7 to 45 us (48 sequences of 17 to 6000 positions).

template <bool PREFIX>
__device__ __forceinline__ PagedSeq paged_seq(const PagedWork& p, const PagedPrefix& prefix, int b, bool& cut) {
    PagedSeq s;
    cut = false;
    s.table = b;
    if (PREFIX) {
        s.begin = 0;
        s.count = p.kv.starts ? min(max(p.kv.starts[p.kv.B], 0), p.kv.T) : p.kv.T;
        s.len = prefix.len;
        s.off = 0;
        s.table = prefix.table;
    } else {
        paged_rows(p.kv, b, s.begin, s.count);
        s.len = max(paged_len(p.kv, b, cut), 0);
        s.off = max(p.kv.lens[b], 0) - s.count;
    }
    s.rows = s.count * p.G;
    return s;
}

// Positions that the last row of tile i sees (all that any row of it sees).
template <bool PREFIX, int ROWS>
__device__ __forceinline__ int paged_tile_limit(const PagedWork& p, const PagedSeq& s, int i) {
    if (PREFIX || !p.causal) return s.len;
    const int tok = p.by_G(min(s.rows, (i + 1) * ROWS) - 1);
    return max(0, min(s.len, s.off + tok + 1));
}

// Units of tile i: at least one, so that rows that see nothing are written too.
template <bool PREFIX, int ROWS, int UNIT>
__device__ __forceinline__ int paged_tile_units(const PagedWork& p, const PagedSeq& s, int i) {
    const int n = paged_tile_limit<PREFIX, ROWS>(p, s, i) - (PREFIX ? 0 : p.prefix_len);
    return max(1, (n + UNIT - 1) / UNIT);
}

// Cost of the tiles of one kv head, in units.
template <bool PREFIX, int ROWS, int UNIT, int OVERHEAD>
__device__ __forceinline__ long long paged_head_cost(const PagedWork& p, const PagedSeq& s, int tiles) {
    long long n = (long long)tiles * OVERHEAD;
    for (int i = 0; i < tiles; ++i) n += paged_tile_units<PREFIX, ROWS, UNIT>(p, s, i);
    return n;
}

// Share of CTA c: units [c q + min(c, r), ...) with q = U / grid, r = U % grid.
struct PagedShare {
    long long q;
    int r;
    PagedShare() = default;
    __device__ __forceinline__ PagedShare(long long U, int grid) {
        if (U >> 32) {
            q = U / grid;
            r = int(U - q * grid);
        } else {  // one 32-bit division
            const uint32_t u = uint32_t(U), d = u / uint32_t(grid);
            q = d;
            r = int(u - d * uint32_t(grid));
        }
    }
    __device__ __forceinline__ long long lo(int c) const { return q * c + min(c, r); }
    __device__ __forceinline__ int owner(long long u) const {
        const long long head = (q + 1) * r;
        if (u < head) return (head >> 32) ? int(u / (q + 1)) : int(uint32_t(u) / uint32_t(q + 1));
        return (u >> 32) || (q >> 32) ? r + int((u - head) / q) : r + int(uint32_t(u - head) / uint32_t(q));
    }
};

// All NT threads, in the prefix pass: the longest sequence that has rows, of several the first.
template <int NT>
__device__ __forceinline__ PagedPrefix paged_prefix(const PagedWork& p) {
    __shared__ unsigned long long s_key[NT / 32];
    __shared__ int s_seen[NT / 32];
    unsigned long long key = 0;  // length, then the smallest index
    int seen = p.prefix_len;
    for (int b = threadIdx.x; b < p.kv.B; b += NT) {
        int begin, count;
        paged_rows(p.kv, b, begin, count);
        bool cut;
        const int len = paged_len(p.kv, b, cut);
        if (count == 0 || len <= 0) continue;
        key = max(key, (unsigned long long)len << 32 | (0x7fffffffu - unsigned(b)));
        seen = min(seen, p.causal ? min(len, max(1, p.kv.lens[b] - count + 1)) : len);  // its first row that sees any
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    seen = __reduce_min_sync(0xffffffffu, seen);
    if ((threadIdx.x & 31) == 0) {
        s_key[threadIdx.x >> 5] = key;
        s_seen[threadIdx.x >> 5] = seen;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        key = max(key, s_key[w]);
        seen = min(seen, s_seen[w]);
    }
    const int len = int(key >> 32);
    return PagedPrefix{len ? int(0x7fffffffu - unsigned(key)) : 0, min(len, p.prefix_len), seen};
}

// Place in a CTA's share.
struct PagedCursor {
    int b, j, i, k;   // sequence, kv head, tile, cost units of the tile that lie before
    int tiles;        // of sequence b
    long long u, hi;  // cost units of the batch that lie before, end of the share
    PagedShare share;
};

// The part of the tile at the cursor that lies in the share: units [k0, k0 + nu)
// of `units`; nu = 0: only overhead.
template <bool PREFIX, int ROWS, int UNIT, int OVERHEAD>
struct PagedSegment {
    int units, k0, nu, cost;
    PagedSegment() = default;
    __device__ __forceinline__ PagedSegment(const PagedWork& p, const PagedSeq& s, const PagedCursor& c) {
        units = paged_tile_units<PREFIX, ROWS, UNIT>(p, s, c.i);
        cost = int(min((long long)(units + OVERHEAD - c.k), c.hi - c.u));
        k0 = max(0, c.k - OVERHEAD);
        nu = max(0, c.k + cost - OVERHEAD) - k0;
    }
    __device__ __forceinline__ bool whole() const { return nu == units; }
    // CTAs that hold the tile when it begins in this one and goes on, else 0
    __device__ __forceinline__ int parts(const PagedCursor& c, int cta) const {
        return whole() || k0 > 0 ? 0 : c.share.owner(c.u - c.k + units + OVERHEAD - 1) - cta + 1;
    }
};

// All NT threads: finds the share of CTA `cta` and, in the prefix pass, what `s_prefix` (shared memory) says. The thread whose sequences hold its
// first unit finds the place with what it has read and tells the others (when every
// thread read the sequence once more and divided for itself, 48 sequences of 17 to
// 6000 positions took 42.1 us instead of 38.4, 8 of 24 to 32 thousand 158 instead of
// 146).
template <bool PREFIX, int ROWS, int UNIT, int OVERHEAD, int NT>
__device__ __forceinline__ PagedCursor paged_find(const PagedWork& p, int cta, int grid, PagedPrefix& s_prefix) {
    __shared__ long long s_sum[NT / 32];
    __shared__ int s_at[5];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    PagedPrefix prefix = {0, 0, 0};
    if (PREFIX) {
        prefix = paged_prefix<NT>(p);
        if (threadIdx.x == 0) s_prefix = prefix;
    }
    const int B = PREFIX ? 1 : p.kv.B;
    const int per = (B + NT - 1) / NT, b0 = min(int(threadIdx.x) * per, B), b1 = min(b0 + per, B);
    PagedSeq s;
    int tiles = 0;
    long long head = 0, mine = 0;
    auto read = [&](int b) {
        bool cut;
        s = paged_seq<PREFIX>(p, prefix, b, cut);
        tiles = (s.rows + ROWS - 1) / ROWS;
        head = paged_head_cost<PREFIX, ROWS, UNIT, OVERHEAD>(p, s, tiles);
        return cut;
    };
    for (int b = b0; b < b1; ++b) {
        if (read(b) && cta == 0) atomicOr(p.kv.errors, BQ_DEVERR_POSITION_BIT);
        mine += head * p.kv.HKV;
    }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) s_sum[warp] = incl;
    if (threadIdx.x == 0) s_at[0] = -1;
    __syncthreads();
    long long before = incl - mine, U = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) before += s_sum[w];
        U += s_sum[w];
    }
    PagedCursor c;
    c.share = PagedShare(U, grid);
    c.u = c.share.lo(cta);
    c.hi = c.share.lo(cta + 1);
    if (c.u < c.hi && c.u >= before && c.u < before + mine) {
        int b = b0;
        if (per > 1)
            for (;; ++b) {
                read(b);
                if (c.u < before + head * p.kv.HKV) break;
                before += head * p.kv.HKV;
            }
        const long long rem = c.u - before;
        const int j = (rem >> 32) || (head >> 32) ? int(rem / head) : int(uint32_t(rem) / uint32_t(head));
        long long left = rem - j * head;
        int i = 0;
        for (;; ++i) {
            const int n = paged_tile_units<PREFIX, ROWS, UNIT>(p, s, i) + OVERHEAD;
            if (left < n) break;
            left -= n;
        }
        s_at[0] = b;
        s_at[1] = j;
        s_at[2] = i;
        s_at[3] = int(left);
        s_at[4] = tiles;
    }
    __syncthreads();
    c.b = s_at[0];
    c.j = c.i = c.k = c.tiles = 0;
    if (c.b < 0) {
        c.hi = c.u;  // nothing for this CTA
        return c;
    }
    c.j = s_at[1];
    c.i = s_at[2];
    c.k = s_at[3];
    c.tiles = s_at[4];
    return c;
}

// To the tile after the cursor's, `cost` units on (sequences without rows have none).
template <bool PREFIX, int ROWS>
__device__ __forceinline__ void paged_next(const PagedWork& p, const PagedPrefix& prefix, PagedCursor& c, int cost) {
    c.u += cost;
    c.k = 0;
    if (++c.i < c.tiles) return;
    c.i = 0;
    if (++c.j < p.kv.HKV) return;
    c.j = 0;
    const int B = PREFIX ? 1 : p.kv.B;
    for (++c.b; c.b < B; ++c.b) {
        bool cut;
        const PagedSeq s = paged_seq<PREFIX>(p, prefix, c.b, cut);
        c.tiles = (s.rows + ROWS - 1) / ROWS;
        if (c.tiles > 0) return;
    }
}

// Positions [0, limit) are seen by row r (of sequence s; in the prefix pass, of all rows).
template <bool PREFIX>
__device__ __forceinline__ int paged_row_limit(const PagedWork& p, const PagedSeq& s, int r) {
    const int tok = p.by_G(r);
    if (!PREFIX) return p.causal ? max(0, min(s.len, s.off + tok + 1)) : s.len;
    int b = tok;
    if (p.kv.starts) {  // the sequence of row tok: starts[b] <= tok < starts[b + 1]
        int lo = 0, hi = p.kv.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.kv.starts[mid] <= tok) lo = mid; else hi = mid;
        }
        b = lo;
    }
    int begin, count;
    paged_rows(p.kv, b, begin, count);
    bool cut;
    const int len = max(paged_len(p.kv, b, cut), 0);
    const int lim = p.causal ? min(len, max(p.kv.lens[b], 0) - count + (tok - begin) + 1) : len;
    return max(0, min(lim, p.prefix_len));
}

// What is infinite or NaN among two packed elements: 0xffff in its half.
template <typename E>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t x) {
    constexpr uint32_t exps = std::is_same_v<E, __half> ? 0x7C007C00u : 0x7F807F80u;
    return __vcmpeq2(x & exps, exps);
}

// Two or eight elements <-> fp32.
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
    if constexpr (std::is_same_v<T, __half>) {
        __half2 h;
        memcpy(&h, &w, 4);
        const float2 f = __half22float2(h);
        lo = f.x;
        hi = f.y;
    } else {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xFFFF0000u);
    }
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& r, float (&v)[8]) {
    unpack2<T>(r.x, v[0], v[1]);
    unpack2<T>(r.y, v[2], v[3]);
    unpack2<T>(r.z, v[4], v[5]);
    unpack2<T>(r.w, v[6], v[7]);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    return pack_bf162(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    return pack_half2(lo, hi);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}


// Four fp32 values as elements, 8 bytes.
template <typename T>
__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
    return make_uint2(pack2<T>(a, b), pack2<T>(c, d));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLn2 = 0.6931471805599453f;

}  // namespace bq
