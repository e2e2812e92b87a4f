// Paged KV-cache operators: descriptor checks, launch helper and
// bq_paged_attention (attention of the new tokens of a ragged batch over
// their paged caches).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "bq_host.h"
#include "bq_paged.cuh"
#include "bq_paged_host.h"

namespace bq {

int paged_validate(const bq_paged_kv* kv, int T, int HQ) {
    if (kv->dtype != BQ_DT_BF16 && kv->dtype != BQ_DT_F16)
        return set_error(BQ_ERR_FORMAT, "paged caches are bf16 or fp16 (dtype %d)", kv->dtype);
    if (kv->D != 64 && kv->D != 128) return set_error(BQ_ERR_SHAPE, "head dim must be 64 or 128 (got %d)", kv->D);
    if (kv->page_size < 16 || kv->page_size > 1024 || (kv->page_size & (kv->page_size - 1)))
        return set_error(BQ_ERR_SHAPE, "page size must be a power of two from 16 to 1024 (got %d)", kv->page_size);
    if (kv->B < 1 || kv->num_pages < 1 || kv->max_pages < 1 || T < 0)
        return set_error(BQ_ERR_SHAPE, "bad batch (B=%d, pages=%d, table columns=%d, rows=%d)", kv->B, kv->num_pages,
                         kv->max_pages, T);
    if (kv->HKV < 1 || HQ < 1 || HQ % kv->HKV || int64_t(HQ) * kv->D > (1 << 20))
        return set_error(BQ_ERR_SHAPE, "HQ=%d must be a multiple of HKV=%d", HQ, kv->HKV);
    if (int64_t(T) * (HQ + 2 * kv->HKV) > 0x7FFFFFFF)
        return set_error(BQ_ERR_SHAPE, "%d rows of %d heads are too many for one call", T, HQ);
    if (int64_t(kv->max_pages) * kv->page_size > 0x3FFFFFFF)
        return set_error(BQ_ERR_SHAPE, "the page table covers more than 2^30 positions");
    if (!kv->k_pages || !kv->v_pages || !kv->page_table || !kv->seq_lens)
        return set_error(BQ_ERR_INVALID_ARG, "pages, page_table and seq_lens must be non-NULL");
    if (!kv->q_starts && T != kv->B)
        return set_error(BQ_ERR_SHAPE, "%d rows for %d sequences: ragged rows need q_starts", T, kv->B);
    if (kv->ld_table < kv->max_pages)
        return set_error(BQ_ERR_SHAPE, "page table stride %lld < %d columns", (long long)kv->ld_table, kv->max_pages);
    const int size[3] = {kv->num_pages, kv->HKV, kv->page_size};
    for (int i = 0; i < 3; ++i) {
        if (size[i] == 1) continue;  // its stride is never taken
        if (kv->k_stride[i] < kv->D || kv->v_stride[i] < kv->D)
            return set_error(BQ_ERR_SHAPE, "page strides must be at least the head dim");
        if (kv->k_stride[i] % 8 || kv->v_stride[i] % 8) return set_error(BQ_ERR_ALIGN, "page strides must be multiples of 8");
    }
    if (!paged_aligned(kv->k_pages, 0, 2) || !paged_aligned(kv->v_pages, 0, 2))
        return set_error(BQ_ERR_ALIGN, "pages must be 16-byte aligned");
    return BQ_OK;
}

int paged_check_device() {
    const DeviceInfo* di = device_info();
    if (!di) return BQ_ERR_CUDA;
    if (di->major != 10)
        return set_error(BQ_ERR_DEVICE, "sm_%d%d device: this library is built for sm_100a", di->major, di->minor);
    return BQ_OK;
}

int paged_fill(PagedKV* o, const bq_paged_kv* kv, int T, int HQ) {
    o->B = kv->B;
    o->HKV = kv->HKV;
    o->page_shift = __builtin_ctz(unsigned(kv->page_size));
    o->page_mask = kv->page_size - 1;
    o->num_pages = kv->num_pages;
    o->max_pages = kv->max_pages;
    o->T = T;
    o->HQ = HQ;
    o->k = kv->k_pages;
    o->ks_page = kv->k_stride[0];
    o->ks_head = kv->k_stride[1];
    o->ks_slot = kv->k_stride[2];
    o->v = kv->v_pages;
    o->vs_page = kv->v_stride[0];
    o->vs_head = kv->v_stride[1];
    o->vs_slot = kv->v_stride[2];
    o->table = kv->page_table;
    o->ld_table = kv->ld_table;
    o->lens = kv->seq_lens;
    o->starts = kv->q_starts;
    o->errors = device_error_word();
    return o->errors ? BQ_OK : BQ_ERR_CUDA;
}

int paged_launch(const void* fn, dim3 grid, dim3 block, uint32_t smem, void** args, uint32_t flags, void* stream,
                 const char* what, int cluster) {
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (flags & BQ_FLAG_PDL) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = unsigned(cluster);
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
    if (e != cudaSuccess) return set_error(BQ_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    return BQ_OK;
}

namespace {

constexpr int kJoinWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;

// One pass's parts, as the joining kernel reads them.
struct PagedParts {
    const float* part_o;
    const float2* part_ml;
    const float* row_o;
    const float2* row_ml;
    const int2* row_at;
    int32_t rows, grid;
};

struct PagedJoin {
    PagedParts pass[2];  // own positions; the shared prefix (grid 0: none)
    const PagedShared* shared;
    const int32_t* starts;
    void* out;
    int64_t ldo;
    float* lse;
    int64_t ldl;
    int32_t B, T, HQ, G;
    FastDiv by_G, by_HQ;
};

// The parts of one output row in one pass.
struct RowParts {
    const float* o;
    const float2* ml;
    int64_t first, step;  // row of the first part (slot 2 c + 1), and from each CTA's slot 2 c to the next CTA's
    int64_t head;         // row of slot 2 c of the first CTA
    int32_t n;
    __device__ __forceinline__ int64_t at(int i) const { return i == 0 ? first : head + i * step; }
};

__device__ __forceinline__ RowParts shared_row(const PagedParts& p, int cta, int parts, int r) {
    RowParts x;
    x.o = p.part_o;
    x.ml = p.part_ml;
    x.head = int64_t(2 * cta) * p.rows + r;
    x.first = x.head + p.rows;
    x.step = int64_t(2) * p.rows;
    x.n = parts;
    return x;
}

// Running join of parts of one row: largest score, sum of exponentials, and this
// lane's outputs.
template <int DPL>
struct JoinRow {
    float m, l, acc[DPL];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < DPL; ++e) acc[e] = 0.f;
    }
    __device__ __forceinline__ void add(float m2, float l2, const float (&o)[DPL]) {
        if (l2 == 0.f && m2 == -INFINITY) return;  // saw nothing (its outputs are zeros, or zeros times what it did not see)
        const float nm = fmaxf(m, m2), u = nm == -INFINITY ? 0.f : nm, f = ex2(m - u), g = ex2(m2 - u);
        m = nm;
        l = l * f + l2 * g;
#pragma unroll
        for (int e = 0; e < DPL; ++e) acc[e] = acc[e] * f + o[e] * g;
    }
};

template <int DPL>
__device__ __forceinline__ void load_lane(const float* src, float (&o)[DPL]) {
    if constexpr (DPL == 4) {
        const float4 v = *reinterpret_cast<const float4*>(src);
        o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    } else {
        const float2 v = *reinterpret_cast<const float2*>(src);
        o[0] = v.x, o[1] = v.y;
    }
}

// One output row (R = 1) or R neighbouring rows of a tile: WPR warps, each on every
// WPR-th part, kParts parts of each row in flight. Every thread of the block calls
// it. `place` gives row r's output row and head.
constexpr int kFewParts = 8, kFewRows = 32;

template <typename E, int D, int WPR, int R, int kParts, typename Place>
__device__ __forceinline__ void join_rows(const PagedJoin& p, const RowParts (&part)[2], int rows, const Place& place) {
    constexpr int DPL = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WPR;
    JoinRow<DPL> row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) row[r].clear();
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        for (int i0 = sub; i0 < part[a].n; i0 += WPR * kParts) {
            float2 ml[kParts][R];
            float o[kParts][R][DPL];
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                const int64_t at = part[a].at(min(i0 + i * WPR, part[a].n - 1));
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int64_t from = at + min(r, rows - 1);  // rows of a slot follow one another
                    ml[i][r] = part[a].ml[from];
                    load_lane<DPL>(part[a].o + from * D + lane * DPL, o[i][r]);
                }
            }
#pragma unroll
            for (int i = 0; i < kParts; ++i)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (i0 + i * WPR < part[a].n) row[r].add(ml[i][r].x, ml[i][r].y, o[i][r]);
        }
    }
    if constexpr (WPR > 1) {
        __shared__ float s_acc[kJoinWarps][D];
        __shared__ float2 s_ml[kJoinWarps];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < DPL; ++e) s_acc[warp][lane * DPL + e] = row[0].acc[e];
        if (lane == 0) s_ml[warp] = make_float2(row[0].m, row[0].l);
        __syncthreads();
        if (sub == 0) {
#pragma unroll
            for (int q = 1; q < WPR; ++q) {
                float o[DPL];
#pragma unroll
                for (int e = 0; e < DPL; ++e) o[e] = s_acc[warp + q][lane * DPL + e];
                row[0].add(s_ml[warp + q].x, s_ml[warp + q].y, o);
            }
        }
    }
    if (sub != 0) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= rows) break;
        int t, h;
        place(r, t, h);
        const float l = row[r].l, inv = paged_inverse(row[r].m, l);
        const float (&acc)[DPL] = row[r].acc;
        E* dst = static_cast<E*>(p.out) + int64_t(t) * p.ldo + h * D + lane * DPL;
        if constexpr (DPL == 4)
            *reinterpret_cast<uint2*>(dst) = pack4<E>(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
        else
            *reinterpret_cast<uint32_t*>(dst) = pack2<E>(acc[0] * inv, acc[1] * inv);
        if (p.lse && lane == 0) p.lse[int64_t(t) * p.ldl + h] = l != 0.f ? (row[r].m + log2f(l)) * kLn2 : -INFINITY;
    }
}

// Joins the tiles that CTAs share: block (c, y) takes rows of the one that begins in
// CTA c (tiles that one CTA held are finished already), R per warp; where the tile
// is spread over more than kFewParts CTAs, one per warp, or, with few rows, one at a
// time with all its warps. Parts are added in CTA order within a warp, warps in
// order: deterministic. (A prompt of 1655 positions, one kv head of 64: 24 us; 38 us
// with a row per block there. One row per warp throughout costs a prompt of 7000
// tokens 213 instead of 207 us, eight parts in flight 211.)
// Bound: latency of two rounds of loads (a record, then the parts), or L2 for the
// prompts' tiles.
template <typename E, int D, int R>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_join_kernel(const __grid_constant__ PagedJoin p) {
    pdl_launch_dependents();
    pdl_wait();
    const PagedShared sh = p.shared[blockIdx.x];
    if (sh.parts == 0) return;
    const bool few = sh.parts <= kFewParts, each = few || sh.rows > kFewRows;
    const int mine = few ? R : 1;                // rows of a warp, or of the block
    const int per = each ? kJoinWarps * mine : 1;  // rows of a block at a time
    for (int r0 = blockIdx.y * per; r0 < sh.rows; r0 += gridDim.y * per) {
        const int idx = each ? r0 + (threadIdx.x >> 5) * mine : r0;
        RowParts part[2];
        part[0].n = part[1].n = 0;
        if (idx < sh.rows) part[1] = shared_row(p.pass[0], blockIdx.x, sh.parts, idx);
        auto place = [&](int r, int& t, int& h) {
            const int rr = sh.r0 + idx + r, tok = p.by_G(rr);
            t = sh.begin + tok;
            h = sh.j * p.G + rr - tok * p.G;
        };
        if (few)
            join_rows<E, D, 1, R, R == 1 ? 4 : 2>(p, part, max(0, min(R, sh.rows - idx)), place);
        else if (each)
            join_rows<E, D, 1, 1, 4>(p, part, max(0, min(1, sh.rows - idx)), place);
        else
            join_rows<E, D, kJoinWarps, 1, 4>(p, part, 1, place);
    }
}

// Joins every row from the prefix's parts and its own: WPR warps per row.
template <typename E, int D, int WPR>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_join_prefix_kernel(const __grid_constant__ PagedJoin p) {
    constexpr int RPB = kJoinWarps / WPR;
    pdl_launch_dependents();
    pdl_wait();
    int row_lo = 0, row_hi = p.T;  // rows of sequences
    if (p.starts) {
        row_lo = p.starts[0];
        row_hi = p.starts[p.B];
    }
    const int total = p.T * p.HQ;
    for (int r0 = blockIdx.x * RPB; r0 < total; r0 += gridDim.x * RPB) {
        const int idx = r0 + (threadIdx.x >> 5) / WPR;
        const int t = p.by_HQ(min(idx, total - 1));
        const bool live = idx < total && t >= row_lo && t < row_hi;
        RowParts part[2];
        part[0].n = part[1].n = 0;
        if (live) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {  // a = 0: the prefix, which comes first
                const PagedParts& ps = p.pass[1 - a];
                const int2 at = ps.row_at[idx];
                const int n = at.y >> 8;
                if (n > 0) {  // clamped: a row that ill-ordered starts left out reads no address outside
                    const int cta = min(max(at.x, 0), ps.grid - 1);
                    part[a] = shared_row(ps, cta, min(n, ps.grid - cta), min(at.y & 255, ps.rows - 1));
                } else {
                    part[a].o = ps.row_o;
                    part[a].ml = ps.row_ml;
                    part[a].first = idx;
                    part[a].n = 1;
                }
            }
        }
        join_rows<E, D, WPR, 1, 4>(p, part, live ? 1 : 0, [&](int, int& tt, int& h) {
            tt = t;
            h = idx - t * p.HQ;
        });
    }
}

constexpr int kJoinRows = 2;  // rows of a warp where tiles have many

template <typename E, int D>
const void* join_kernel(bool prefix, bool many) {
    if (prefix)
        return many ? reinterpret_cast<const void*>(&paged_join_prefix_kernel<E, D, 1>)
                    : reinterpret_cast<const void*>(&paged_join_prefix_kernel<E, D, kJoinWarps>);
    return many ? reinterpret_cast<const void*>(&paged_join_kernel<E, D, kJoinRows>)
                : reinterpret_cast<const void*>(&paged_join_kernel<E, D, 1>);
}

// Most positions per CTA of a cluster that the page table may hold. Clusters against
// equal shares, 128 dims, all sequences of the table's length: two sequences of 16
// heads, 256 / 1024 / 4096 positions 5.4 / 6.4 / 11.8 us and 8.4 / 10.7 / 17.2 us; 9
// sequences of 8 (four CTAs per pair), 1024 / 2048 positions 13.2 / 19.0 and 14.2 /
// 18.7 us. Uneven lengths cost a cluster its longest, hence the limit.
constexpr int kClusterPositions = 512;

// Bytes of repeated reads that a shared prefix must save for its second pass and
// the join of every row to pay. Shared against not, 128 dims, 64 positions of their
// own, prefix of 1024 / 2048 / 4096 (MB saved; us, in a graph):
//                             one new token, 4 rows per kv head   8 tokens, 32 rows (256-row kernel)
//   16 sequences of 8 kv heads, 60 / 120 / 240 MB
//                             23 / 24 / 25 and 16 / 23 / 36       34 / 37 / 40 and 26 / 36 / 56
//   48 of 2, 47 / 94 / 188    23 / 23 / 24 and 14 / 19 / 29       30 / 34 / 36 and 24 / 31 / 46
//   96 of 8, 380 / 760 / 1520 32 / 34 / 37 and 55 / 93 / 168      88 / 98 / 119 and 104 / 155 / 265
// 64 dims break even at 60 to 110 MB. Bytes alone misjudge many rows behind a short
// prefix, where joining them costs most: 96 sequences of 64 rows per kv head behind 512
// or 1024 positions (190 / 380 MB) take 116 / 128 us shared, 81 / 105 not.
constexpr int64_t kSharedBytes = 96ll << 20;

// One pass over positions: its kernel and its CTAs.
struct PagedPass {
    bool wide;
    int rows, unit, grid;
};

// Scratch of one pass: the shared tiles' partials and records, then, with a
// prefix, the row buffers.
struct PagedScratch {
    size_t part_o, part_ml, shared, row_o, row_ml, row_at;
};
struct PagedPlan {
    PagedPass pass[2];  // own positions, the prefix
    PagedScratch at[2];
    int64_t tile_rows;  // rows of one own tile as far as is known
    int ranks;          // > 0: one cluster of so many CTAs per (sequence, kv head) instead
    int prefix;         // shared positions that get a pass of their own
    size_t total;
};

// rows: rows that share a kv head as far as is known. Up to 16 take the kernel for
// few rows (two CTAs per SM), and up to 32 of 64 dims, though it then reads the
// cache twice, the second time from L2 (24 rows: 32 sequences of 700 and 6000
// positions 26 and 63 us, against 46 and 90 us with the 256-row kernel; of 128
// dims 38 and 135 us against 55 and 94 us, where they take the latter). More go to
// the 256-row kernel, one CTA per SM (48 rows of 64 dims, 6000 positions: 112 / 90 us).
PagedPass paged_pass(int64_t rows, int D, int sms) {
    if (rows <= kNarrowRows * (D == 64 ? 2 : 1)) return PagedPass{false, kNarrowRows, kNarrowUnit, 2 * sms};
    return PagedPass{true, kWideRows, kWideUnit, sms};
}

int plan_paged(const bq_paged_attn_desc* d, PagedPlan* pl) {
    const DeviceInfo* di = device_info();
    if (!di) return BQ_ERR_CUDA;
    const int G = d->HQ / d->kv.HKV;
    *pl = PagedPlan{};
    const int64_t most = !d->kv.q_starts ? 1 : d->max_q > 0 ? d->max_q : (int64_t(d->T) + d->kv.B - 1) / d->kv.B;
    pl->tile_rows = most * G;
    const bool share = d->prefix_len > 0 && (d->flags & BQ_PAGED_SHARE);
    if (most * G <= kNarrowRows && !share) {
        const int64_t pairs = int64_t(d->kv.B) * d->kv.HKV, room = int64_t(d->kv.max_pages) * d->kv.page_size;
        int ranks = kNarrowRanks;
        while (ranks > 1 && pairs * ranks > 2 * di->sm_count) ranks >>= 1;
        if (ranks > 1 && room <= int64_t(kClusterPositions) * ranks) {
            pl->ranks = ranks;
            return BQ_OK;
        }
    }
    const int64_t saved = int64_t(d->kv.B - 1) * d->prefix_len * d->kv.HKV * d->kv.D * 4;
    pl->prefix = share || saved >= kSharedBytes ? d->prefix_len : 0;
    pl->pass[0] = paged_pass(most * G, d->kv.D, di->sm_count);
    pl->pass[1] = paged_pass(int64_t(d->T) * G, d->kv.D, di->sm_count);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~size_t(255);
        return here;
    };
    for (int i = 0; i < (pl->prefix > 0 ? 2 : 1); ++i) {
        const size_t slots = size_t(2) * pl->pass[i].grid * pl->pass[i].rows, rows = size_t(d->T) * d->HQ;
        PagedScratch& s = pl->at[i];
        s.part_o = take(slots * d->kv.D * 4);
        s.part_ml = take(slots * 8);
        s.shared = take(size_t(pl->pass[i].grid) * sizeof(PagedShared));
        if (pl->prefix > 0) {
            s.row_o = take(rows * d->kv.D * 4);
            s.row_ml = take(rows * 8);
            s.row_at = take(rows * 8);
        }
    }
    pl->total = at;
    return BQ_OK;
}

int launch_pass(const PagedPass& ps, const PagedWork& w, const bq_paged_attn_desc* d, void* stream) {
    return ps.wide ? paged_launch_wide(w, &d->kv, ps.grid, d->flags, stream)
                   : paged_launch_narrow(w, d->kv.dtype, d->kv.D, ps.grid, d->flags, stream);
}

int validate_attention(const bq_paged_attn_desc* d) {
    if (!d) return set_error(BQ_ERR_INVALID_ARG, "desc is NULL");
    const int rc = paged_validate(&d->kv, d->T, d->HQ);
    if (rc) return rc;
    const int width = d->HQ * d->kv.D;
    if (d->T && (!d->q || !d->out)) return set_error(BQ_ERR_INVALID_ARG, "q and out must be non-NULL");
    if (d->ldq < width || d->ldo < width)
        return set_error(BQ_ERR_SHAPE, "row strides %lld / %lld < %d", (long long)d->ldq, (long long)d->ldo, width);
    if (d->lse && d->ldl < d->HQ) return set_error(BQ_ERR_SHAPE, "lse row stride %lld < %d", (long long)d->ldl, d->HQ);
    if (!paged_aligned(d->q, d->ldq, 2) || !paged_aligned(d->out, d->ldo, 2))
        return set_error(BQ_ERR_ALIGN, "q and out rows must be 16-byte aligned");
    if (!(d->scale > 0.f) || !std::isfinite(d->scale * kLog2e))  // the kernels' factor: scores are kept in base 2
        return set_error(BQ_ERR_INVALID_ARG, "scale must be positive and finite (times log2(e), too)");
    if (d->max_q < 0) return set_error(BQ_ERR_INVALID_ARG, "max_q=%d is negative", d->max_q);
    if (d->prefix_len < 0 || d->prefix_len % d->kv.page_size)
        return set_error(BQ_ERR_SHAPE, "prefix_len=%d must be a multiple of the page size %d", d->prefix_len,
                         d->kv.page_size);
    if (d->prefix_len / d->kv.page_size > d->kv.max_pages)
        return set_error(BQ_ERR_SHAPE, "prefix_len=%d exceeds the page table", d->prefix_len);
    return BQ_OK;
}

}  // namespace
}  // namespace bq

using namespace bq;

extern "C" {

int32_t bq_paged_attention_workspace_bytes(const bq_paged_attn_desc* d, size_t* bytes) {
    if (!bytes) return set_error(BQ_ERR_INVALID_ARG, "bytes is NULL");
    int rc = validate_attention(d);
    if (rc) return rc;
    PagedPlan pl;
    rc = plan_paged(d, &pl);
    if (rc) return rc;
    *bytes = d->T ? pl.total : 0;
    return BQ_OK;
}

int32_t bq_paged_attention(const bq_paged_attn_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = validate_attention(d);
    if (rc) return rc;
    if (d->T == 0) return BQ_OK;
    rc = paged_check_device();
    if (rc) return rc;
    PagedPlan pl;
    rc = plan_paged(d, &pl);
    if (rc) return rc;
    if (pl.total && (!workspace || workspace_bytes < pl.total))
        return set_error(BQ_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", workspace_bytes, pl.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return set_error(BQ_ERR_ALIGN, "workspace must be 256-byte aligned");
    char* ws = static_cast<char*>(workspace);
    PagedWork w;
    std::memset(&w, 0, sizeof(w));
    rc = paged_fill(&w.kv, &d->kv, d->T, d->HQ);
    if (rc) return rc;
    w.G = d->HQ / d->kv.HKV;
    w.by_G.set(uint32_t(w.G));
    w.causal = (d->flags & BQ_PAGED_FULL) ? 0 : 1;
    w.prefix_len = pl.prefix;
    w.scale_log2 = d->scale * kLog2e;
    w.q = d->q;
    w.ldq = d->ldq;
    w.out = d->out;
    w.ldo = d->ldo;
    w.lse = d->lse;
    w.ldl = d->ldl;
    if (pl.ranks) return paged_launch_cluster(w, d->kv.dtype, d->kv.D, pl.ranks, d->flags, stream);
    PagedJoin p;
    std::memset(&p, 0, sizeof(p));
    const bool prefix = pl.prefix > 0;
    for (int i = prefix ? 1 : 0; i >= 0; --i) {  // the prefix first
        const PagedScratch& s = pl.at[i];
        w.prefix_pass = i;
        w.part_o = reinterpret_cast<float*>(ws + s.part_o);
        w.part_ml = reinterpret_cast<float2*>(ws + s.part_ml);
        w.shared = reinterpret_cast<PagedShared*>(ws + s.shared);
        if (prefix) {
            w.row_o = reinterpret_cast<float*>(ws + s.row_o);
            w.row_ml = reinterpret_cast<float2*>(ws + s.row_ml);
            w.row_at = reinterpret_cast<int2*>(ws + s.row_at);
        }
        rc = launch_pass(pl.pass[i], w, d, stream);
        if (rc) return rc;
        p.pass[i] = PagedParts{w.part_o, w.part_ml, w.row_o, w.row_ml, w.row_at, pl.pass[i].rows, pl.pass[i].grid};
    }
    p.shared = w.shared;
    p.starts = w.kv.starts;
    p.out = w.out;
    p.ldo = w.ldo;
    p.lse = w.lse;
    p.ldl = w.ldl;
    p.B = w.kv.B;
    p.T = d->T;
    p.HQ = d->HQ;
    p.G = w.G;
    p.by_G = w.by_G;
    p.by_HQ.set(uint32_t(d->HQ));
    // With a prefix, 1024 rows give every SM a row per warp; fewer are shared among a block's warps.
    const int64_t rows = int64_t(d->T) * d->HQ;
    const bool many = prefix ? rows >= 1024 : pl.pass[0].wide;
    const int per = prefix ? (many ? kJoinWarps : 1) : kJoinWarps * (many ? kJoinRows : 1);
    const int64_t tile = std::min<int64_t>(pl.pass[0].rows, pl.tile_rows);  // (a tile spread over many CTAs: a block per row)
    const dim3 grid = prefix ? dim3(unsigned(std::min<int64_t>((rows + per - 1) / per, 1 << 20)))
                             : dim3(pl.pass[0].grid, unsigned(std::max((tile + per - 1) / per, std::min<int64_t>(tile, 4))));
    const bool bf = d->kv.dtype == BQ_DT_BF16;
    const void* fn = d->kv.D == 128 ? (bf ? join_kernel<__nv_bfloat16, 128>(prefix, many) : join_kernel<__half, 128>(prefix, many))
                                    : (bf ? join_kernel<__nv_bfloat16, 64>(prefix, many) : join_kernel<__half, 64>(prefix, many));
    void* args[] = {&p};
    return paged_launch(fn, grid, dim3(32 * kJoinWarps), 0, args, d->flags, stream, "paged attention join");
}

}  // extern "C"
