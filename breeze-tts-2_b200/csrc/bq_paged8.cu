// 8-bit paged KV cache: descriptor checks and bq_paged8_attention (attention of the
// new tokens of a ragged batch over their caches).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "bq_host.h"
#include "bq_paged8.cuh"
#include "bq_paged8_host.h"

namespace bq {

int paged8_validate(const bq_paged8_kv* kv, int T, int HQ, bool f32) {
    if (kv->dtype != BQ_DT_BF16 && kv->dtype != BQ_DT_F16 && !(f32 && kv->dtype == BQ_DT_F32))
        return set_error(BQ_ERR_FORMAT, "rows are bf16 or fp16%s (dtype %d)", f32 ? ", or fp32 read back" : "", kv->dtype);
    if (kv->D != 64 && kv->D != 128) return set_error(BQ_ERR_SHAPE, "head dim must be 64 or 128 (got %d)", kv->D);
    if (kv->page_size < 16 || kv->page_size > 1024 || (kv->page_size & (kv->page_size - 1)))
        return set_error(BQ_ERR_SHAPE, "page size must be a power of two from 16 to 1024 (got %d)", kv->page_size);
    if (kv->block < 16 || kv->block > 128 || (kv->block & (kv->block - 1)) || kv->block > kv->page_size)
        return set_error(BQ_ERR_SHAPE, "positions per scale must be 16, 32, 64 or 128, and at most the page size (got %d)", kv->block);
    if (kv->B < 1 || kv->num_pages < 1 || kv->max_pages < 1 || T < 0)
        return set_error(BQ_ERR_SHAPE, "bad batch (B=%d, pages=%d, table columns=%d, rows=%d)", kv->B, kv->num_pages,
                         kv->max_pages, T);
    if (kv->HKV < 1 || int64_t(kv->HKV) * kv->D > (1 << 20)) return set_error(BQ_ERR_SHAPE, "bad number of kv heads (%d)", kv->HKV);
    if (!f32 && (HQ < 1 || HQ % kv->HKV || int64_t(HQ) * kv->D > (1 << 20)))
        return set_error(BQ_ERR_SHAPE, "HQ=%d must be a multiple of HKV=%d", HQ, kv->HKV);
    if (int64_t(T) * (HQ + 2 * kv->HKV) > 0x7FFFFFFF)
        return set_error(BQ_ERR_SHAPE, "%d rows of %d heads are too many for one call", T, HQ);
    if (int64_t(kv->max_pages) * kv->page_size > 0x3FFFFFFF)
        return set_error(BQ_ERR_SHAPE, "the page table covers more than 2^30 positions");
    if (!kv->k_pages || !kv->v_pages || !kv->k_scales || !kv->v_scales || !kv->page_table || !kv->seq_lens)
        return set_error(BQ_ERR_INVALID_ARG, "pages, scales, page_table and seq_lens must be non-NULL");
    if (!kv->q_starts && T != kv->B)
        return set_error(BQ_ERR_SHAPE, "%d rows for %d sequences: ragged rows need q_starts", T, kv->B);
    if (kv->ld_table < kv->max_pages)
        return set_error(BQ_ERR_SHAPE, "page table stride %lld < %d columns", (long long)kv->ld_table, kv->max_pages);
    const int size[3] = {kv->num_pages, kv->HKV, kv->page_size};
    for (int i = 0; i < 3; ++i) {
        if (size[i] == 1) continue;  // its stride is never taken
        if (kv->k_stride[i] < kv->D || kv->v_stride[i] < kv->D)
            return set_error(BQ_ERR_SHAPE, "page strides must be at least the head dim");
        if (kv->k_stride[i] % 16 || kv->v_stride[i] % 16) return set_error(BQ_ERR_ALIGN, "page strides must be multiples of 16");
        if (i < 2 && (kv->k_scale_stride[i] < kv->page_size / kv->block || kv->v_scale_stride[i] < kv->page_size / kv->block))
            return set_error(BQ_ERR_SHAPE, "scale strides must be at least the scales of a page and head");
    }
    if (!paged_aligned(kv->k_pages, 0, 1) || !paged_aligned(kv->v_pages, 0, 1))
        return set_error(BQ_ERR_ALIGN, "pages must be 16-byte aligned");
    return BQ_OK;
}

int paged8_fill(PagedKV* o, Paged8Scales* sc, const bq_paged8_kv* kv, int T, int HQ) {
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
    sc->k = kv->k_scales;
    sc->ks_page = kv->k_scale_stride[0];
    sc->ks_head = kv->k_scale_stride[1];
    sc->v = kv->v_scales;
    sc->vs_page = kv->v_scale_stride[0];
    sc->vs_head = kv->v_scale_stride[1];
    sc->block_shift = __builtin_ctz(unsigned(kv->block));
    return o->errors ? BQ_OK : BQ_ERR_CUDA;
}

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Most positions per CTA of a cluster that the page table may hold, as for 16-bit caches: a cluster costs its longest
// sequence, so a roomy table, which may hold uneven ones, takes equal shares. Clusters against equal shares, all sequences
// of the table's length, 128 dims, us:
//   2 of 16 heads   256 / 1024 / 4096 positions    6.2 / 6.8 / 11.3   and    9.0 / 11.2 / 15.3
//   9 of 8          128 /  512 / 1024 (2 CTAs)     5.8 / 7.7 / 10.6   and    9.5 / 11.0 / 12.8
//   18 of 8         512 / 1024        (2 CTAs)     8.2 / 11.2         and   13.5 / 16.7
//   64 of 8         128 /  512        (1 CTA)     10.9 / 19.8         and   14.4 / 24.6   (200 of 8: no difference)
// and 64 dims:
//   2 of 16 heads   256 / 1024 / 4096 positions    5.6 / 6.0 /  9.3   and    8.5 / 10.4 / 12.8
//   9 of 8          128 /  512 / 1024              5.4 / 6.9 /  9.0   and    8.7 /  9.9 / 11.0
//   64 of 8         128 /  512                     9.8 / 16.3         and   12.8 / 20.4
constexpr int kClusterPositions = 512;

// Rows that share a kv head up to which they go to the kernel for few rows, in tiles of 16. Two tiles take less than one
// of the 256-row kernel; with three, long batches of 64 dims still do, and short or single ones do not. Few / many, us:
//                                        24 rows      32          48          64          96
//   128 dims, 8 kv heads, 32 x 6000    160 / 197   146 / 198   211 / 204   278 / 208   409 / 223
//             4 heads,    4 x 20000     44 / 53     43 / 55     51 / 53     64 / 55     88 / 57
//             4 heads,    8 x 2000      18 / 22     19 / 23     28 / 23     38 / 24     55 / 25
//             1 head,     1 x 300       12 / 14     12 / 14     18 / 15     24 / 15     35 / 15
//   64 dims,  8 heads,    32 x 6000    103 / 173   105 / 173   151 / 174   196 / 176   285 / 179
//             4 heads,    8 x 2000      15 / 20     15 / 21     22 / 21     30 / 21     44 / 22
//             1 head,     1 x 300       10 / 12     10 / 12     15 / 13     20 / 13     29 / 13
constexpr int kFewRows = 32;

// How a call is divided: clusters of `ranks` CTAs per (sequence, kv head), or equal shares of all positions for
// `grid` CTAs with scratch for the tiles (of `rows` rows) that they share.
struct Plan8 {
    int ranks, grid, rows;
    bool wide;
    int64_t tile_rows;  // rows of a tile as far as is known
    size_t part_o, part_ml, shared, total;
};

int plan8(const bq_paged8_attn_desc* d, Plan8* pl) {
    const DeviceInfo* di = device_info();
    if (!di) return BQ_ERR_CUDA;
    *pl = Plan8{};
    const int64_t most = !d->kv.q_starts ? 1 : d->max_q > 0 ? d->max_q : (int64_t(d->T) + d->kv.B - 1) / d->kv.B;
    pl->tile_rows = most * (d->HQ / d->kv.HKV);
    if (pl->tile_rows <= kNarrowRows) {
        const int64_t pairs = int64_t(d->kv.B) * d->kv.HKV, room = int64_t(d->kv.max_pages) * d->kv.page_size;
        // Two CTAs per SM. Clusters of more than two do not find places for that many, since a cluster stays within a part
        // of the GPU: 72 clusters of 4, 128 positions each, take 10.1 us in two waves, 72 of 2 5.8.
        auto fits = [&](int ranks) { return pairs * ranks * 4 <= (ranks > 2 ? 7 : 8) * di->sm_count; };
        int ranks = kNarrowRanks;
        while (ranks > 1 && !fits(ranks)) ranks >>= 1;
        if ((fits(ranks) || pairs <= 4 * di->sm_count) && room <= int64_t(kClusterPositions) * ranks) {
            pl->ranks = ranks;
            return BQ_OK;
        }
    }
    pl->wide = pl->tile_rows > kFewRows;
    pl->rows = pl->wide ? kWideRows : kNarrowRows;
    pl->grid = (pl->wide ? 1 : 2) * di->sm_count;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~size_t(255);
        return here;
    };
    const size_t slots = size_t(2) * pl->grid * pl->rows;
    pl->part_o = take(slots * d->kv.D * 4);
    pl->part_ml = take(slots * 8);
    pl->shared = take(size_t(pl->grid) * sizeof(PagedShared));
    pl->total = at;
    return BQ_OK;
}

int validate_attention(const bq_paged8_attn_desc* d) {
    if (!d) return set_error(BQ_ERR_INVALID_ARG, "desc is NULL");
    const int rc = paged8_validate(&d->kv, d->T, d->HQ);
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
    return BQ_OK;
}

}  // namespace
}  // namespace bq

using namespace bq;

extern "C" {

int32_t bq_paged8_attention_workspace_bytes(const bq_paged8_attn_desc* d, size_t* bytes) {
    if (!bytes) return set_error(BQ_ERR_INVALID_ARG, "bytes is NULL");
    int rc = validate_attention(d);
    if (rc) return rc;
    Plan8 pl;
    rc = plan8(d, &pl);
    if (rc) return rc;
    *bytes = d->T ? pl.total : 0;
    return BQ_OK;
}

int32_t bq_paged8_attention(const bq_paged8_attn_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = validate_attention(d);
    if (rc) return rc;
    if (d->T == 0) return BQ_OK;
    rc = paged_check_device();
    if (rc) return rc;
    Plan8 pl;
    rc = plan8(d, &pl);
    if (rc) return rc;
    if (pl.total && (!workspace || workspace_bytes < pl.total))
        return set_error(BQ_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", workspace_bytes, pl.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return set_error(BQ_ERR_ALIGN, "workspace must be 256-byte aligned");
    char* ws = static_cast<char*>(workspace);
    PagedWork w;
    Paged8Scales sc;
    std::memset(&w, 0, sizeof(w));
    std::memset(&sc, 0, sizeof(sc));
    rc = paged8_fill(&w.kv, &sc, &d->kv, d->T, d->HQ);
    if (rc) return rc;
    w.G = d->HQ / d->kv.HKV;
    w.by_G.set(uint32_t(w.G));
    w.causal = (d->flags & BQ_PAGED_FULL) ? 0 : 1;
    w.scale_log2 = d->scale * kLog2e;
    w.q = d->q;
    w.ldq = d->ldq;
    w.out = d->out;
    w.ldo = d->ldo;
    w.lse = d->lse;
    w.ldl = d->ldl;
    if (pl.ranks) return paged8_launch_cluster(w, sc, d->kv.dtype, d->kv.D, pl.ranks, d->flags, stream);
    w.part_o = reinterpret_cast<float*>(ws + pl.part_o);
    w.part_ml = reinterpret_cast<float2*>(ws + pl.part_ml);
    w.shared = reinterpret_cast<PagedShared*>(ws + pl.shared);
    rc = pl.wide ? paged8_launch_wide(w, sc, &d->kv, pl.grid, d->flags, stream)
                 : paged8_launch_narrow(w, sc, d->kv.dtype, d->kv.D, pl.grid, d->flags, stream);
    if (rc) return rc;
    return paged_launch_join(w, d->kv.dtype, d->kv.D, pl.rows, pl.grid, pl.wide, pl.tile_rows, d->flags, stream);
}

}  // extern "C"
