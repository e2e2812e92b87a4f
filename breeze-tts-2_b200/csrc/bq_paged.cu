// Paged KV-cache operators: descriptor checks, launch helper and
// bq_paged_attention (attention of the new tokens of a ragged batch over
// their paged caches).
#include <algorithm>
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
    for (int i = 0; i < 3; ++i) {
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

void paged_fill(PagedKV* o, const bq_paged_kv* kv, int T, int HQ) {
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
}

int paged_launch(const void* fn, dim3 grid, dim3 block, uint32_t smem, void** args, uint32_t flags, void* stream,
                 const char* what) {
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    if (flags & BQ_FLAG_PDL) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
    if (e != cudaSuccess) return set_error(BQ_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    return BQ_OK;
}

namespace {

constexpr int kJoinThreads = 128;

// What the joining kernel needs of the prefix pass.
struct PagedPrefixParts {
    const float* part_o;
    const float2* part_ml;
    const float* row_o;
    const float2* row_ml;
    int32_t rows, unit, grid;  // ROWS and UNIT of the pass, its CTAs
};

struct PagedJoin {
    PagedWork own;
    int32_t own_grid;
    PagedPrefixParts pre;
};

// Parts of one output row: either the row buffer (a tile that one CTA held) or
// the slots of CTAs c0 .. c1.
struct PagedParts {
    const float* part_o;
    const float2* part_ml;
    const float* row_o;
    const float2* row_ml;
    int64_t row;            // index into the row buffers
    int32_t rows, r, c0, n; // rows per slot, row within the tile, first CTA, parts
    long long u0, q;        // first unit of the tile; share
    int32_t rem;
    __device__ __forceinline__ int64_t at(int i) const {
        const long long lo = q * (c0 + i) + min(c0 + i, rem);
        return int64_t(paged_slot(c0 + i, u0, lo)) * rows + r;
    }
};

__device__ __forceinline__ PagedParts paged_parts(const PagedShare& sh, long long u0, int units, int rows, int r) {
    PagedParts t;
    t.u0 = u0;
    t.q = sh.q;
    t.rem = sh.r;
    t.rows = rows;
    t.r = r;
    t.c0 = sh.owner(u0);
    t.n = sh.owner(u0 + units - 1) - t.c0 + 1;
    return t;
}

// Joins the parts of one output row (grid (T, HQ)): out = sum f_i o_i / sum f_i
// l_i with f_i = 2^(m_i - max m), over the prefix's parts, then the sequence's
// own, in CTA order. A row whose tile one CTA held, and that has no prefix, is
// finished already. The statistics of up to 32 parts are read at once, one per
// lane; the four warps then take every fourth part's output row.
template <typename E, int D, int ROWS, int UNIT>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedJoin p) {
    constexpr int DPL = D / 32;
    __shared__ float s_acc[4][D];
    pdl_launch_dependents();
    pdl_wait();
    const PagedWork& w = p.own;
    const PagedKV& kv = w.kv;
    const int t = blockIdx.x, h = blockIdx.y, j = h / w.G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int b = t;
    if (kv.starts) {
        int n = 0;
        for (int i0 = 0; i0 < kv.B; i0 += kJoinThreads) {
            const int i = i0 + int(threadIdx.x);
            n += __syncthreads_count(i < kv.B && kv.starts[i + 1] <= t);
        }
        b = n;
        if (b >= kv.B) return;  // a row behind the last sequence
    }
    bool cut;
    const PagedSeq s = paged_seq(w, b, cut);
    if (t < s.begin || t >= s.begin + s.count) return;
    const int r = (t - s.begin) * w.G + (h - j * w.G), tile = r / ROWS;
    const long long base = w.bases[b];
    const int head_units = int((w.bases[b + 1] - base) / kv.HKV);
    long long u0 = base + (long long)j * head_units;
    for (int i = 0; i < tile; ++i) u0 += paged_tile_units<ROWS, UNIT>(w, s, i);
    const PagedShare sh(w.bases[kv.B], p.own_grid);
    PagedParts part[2];
    int np = 1;
    part[0] = paged_parts(sh, u0, paged_tile_units<ROWS, UNIT>(w, s, tile), ROWS, r - tile * ROWS);
    part[0].part_o = w.part_o, part[0].part_ml = w.part_ml, part[0].row_o = w.row_o, part[0].row_ml = w.row_ml;
    part[0].row = int64_t(t) * kv.HQ + h;
    if (p.pre.grid) {
        const int rows = (kv.starts ? min(max(kv.starts[kv.B], 0), kv.T) : kv.T) * w.G;
        const int tiles = (rows + p.pre.rows - 1) / p.pre.rows, units = (w.prefix_len + p.pre.unit - 1) / p.pre.unit;
        const int pr = t * w.G + (h - j * w.G), pt = pr / p.pre.rows;
        const PagedShare ps((long long)tiles * units * kv.HKV, p.pre.grid);
        part[1] = part[0];
        part[0] = paged_parts(ps, ((long long)j * tiles + pt) * units, units, p.pre.rows, pr - pt * p.pre.rows);
        part[0].part_o = p.pre.part_o, part[0].part_ml = p.pre.part_ml;
        part[0].row_o = p.pre.row_o, part[0].row_ml = p.pre.row_ml;
        part[0].row = part[1].row;
        np = 2;
    } else if (part[0].n == 1) {
        return;
    }
    float M = -INFINITY;
    for (int k = 0; k < np; ++k)
        for (int i = lane; i < part[k].n; i += 32)
            M = fmaxf(M, part[k].n == 1 ? part[k].row_ml[part[k].row].x : part[k].part_ml[part[k].at(i)].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float u = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc[DPL] = {};
    for (int k = 0; k < np; ++k) {
        for (int i0 = 0; i0 < part[k].n; i0 += 32) {
            const int i = i0 + lane;
            float f = 0.f, l = 0.f;
            if (i < part[k].n) {
                const float2 ml = part[k].n == 1 ? part[k].row_ml[part[k].row] : part[k].part_ml[part[k].at(i)];
                f = ex2(ml.x - u);
                l = f * ml.y;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            L += l;
#pragma unroll 4
            for (int a = warp; a < min(32, part[k].n - i0); a += 4) {
                const float fa = __shfl_sync(0xffffffffu, f, a);
                const float* src = (part[k].n == 1 ? part[k].row_o + part[k].row * D : part[k].part_o + part[k].at(i0 + a) * D) + lane * DPL;
#pragma unroll
                for (int e = 0; e < DPL; ++e) acc[e] = fmaf(fa, src[e], acc[e]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < DPL; ++e) s_acc[warp][lane * DPL + e] = acc[e];
    __syncthreads();
    const int d = threadIdx.x;
    const float inv = L > 0.f ? 1.f / L : 0.f;
    if (d < D)
        static_cast<E*>(w.out)[int64_t(t) * w.ldo + h * D + d] = E((s_acc[0][d] + s_acc[1][d] + s_acc[2][d] + s_acc[3][d]) * inv);
    if (w.lse && d == 0) w.lse[int64_t(t) * w.ldl + h] = L > 0.f ? (M + log2f(L)) * kLn2 : -INFINITY;
}

template <typename E, int D>
const void* join_kernel(bool wide) {
    return wide ? reinterpret_cast<const void*>(&paged_join_kernel<E, D, kWideRows, kWideUnit>)
                : reinterpret_cast<const void*>(&paged_join_kernel<E, D, kNarrowRows, kNarrowUnit>);
}

// One pass over positions: its kernel and its CTAs.
struct PagedPass {
    bool wide;
    int rows, unit, grid;
};

// Scratch of a call, in order: first units of the sequences, then per pass the
// shared tiles' partials, then, with a prefix, both passes' row buffers.
struct PagedPlan {
    PagedPass own, pre;
    size_t bases, own_o, own_ml, pre_o, pre_ml, row_o, row_ml, pre_row_o, pre_row_ml, total;
};

// rows: rows of one tile as far as is known. Tiles of up to 16 rows take the
// kernel for few rows, two CTAs per SM; larger ones the 256-row kernel, one per SM.
PagedPass paged_pass(int64_t rows, int sms) {
    if (rows <= kNarrowRows) return PagedPass{false, kNarrowRows, kNarrowUnit, 2 * sms};
    return PagedPass{true, kWideRows, kWideUnit, sms};
}

int plan_paged(const bq_paged_attn_desc* d, PagedPlan* pl) {
    const DeviceInfo* di = device_info();
    if (!di) return BQ_ERR_CUDA;
    const int G = d->HQ / d->kv.HKV;
    const int64_t most = !d->kv.q_starts ? 1 : d->max_q > 0 ? d->max_q : (int64_t(d->T) + d->kv.B - 1) / d->kv.B;
    pl->own = paged_pass(most * G, di->sm_count);
    pl->pre = paged_pass(int64_t(d->T) * G, di->sm_count);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~size_t(255);
        return here;
    };
    const size_t own = size_t(2) * pl->own.grid * pl->own.rows, pre = size_t(2) * pl->pre.grid * pl->pre.rows;
    pl->bases = take((size_t(d->kv.B) + 1) * 8);
    pl->own_o = take(own * d->kv.D * 4);
    pl->own_ml = take(own * 8);
    if (d->prefix_len > 0) {
        const size_t rows = size_t(d->T) * d->HQ;
        pl->pre_o = take(pre * d->kv.D * 4);
        pl->pre_ml = take(pre * 8);
        pl->row_o = take(rows * d->kv.D * 4);
        pl->row_ml = take(rows * 8);
        pl->pre_row_o = take(rows * d->kv.D * 4);
        pl->pre_row_ml = take(rows * 8);
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
    if (!d->q || !d->out) return set_error(BQ_ERR_INVALID_ARG, "q and out must be non-NULL");
    if (d->ldq < width || d->ldo < width)
        return set_error(BQ_ERR_SHAPE, "row strides %lld / %lld < %d", (long long)d->ldq, (long long)d->ldo, width);
    if (d->lse && d->ldl < d->HQ) return set_error(BQ_ERR_SHAPE, "lse row stride %lld < %d", (long long)d->ldl, d->HQ);
    if (!paged_aligned(d->q, d->ldq, 2) || !paged_aligned(d->out, d->ldo, 2))
        return set_error(BQ_ERR_ALIGN, "q and out rows must be 16-byte aligned");
    if (!(d->scale > 0.f) || d->scale > 3.0e38f) return set_error(BQ_ERR_INVALID_ARG, "scale must be positive and finite");
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
    if (!workspace || workspace_bytes < pl.total)
        return set_error(BQ_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", workspace_bytes, pl.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return set_error(BQ_ERR_ALIGN, "workspace must be 256-byte aligned");
    char* ws = static_cast<char*>(workspace);
    auto f32 = [&](size_t at) { return reinterpret_cast<float*>(ws + at); };
    auto f32x2 = [&](size_t at) { return reinterpret_cast<float2*>(ws + at); };
    PagedJoin p;
    std::memset(&p, 0, sizeof(p));
    PagedWork& w = p.own;
    paged_fill(&w.kv, &d->kv, d->T, d->HQ);
    w.G = d->HQ / d->kv.HKV;
    w.causal = (d->flags & BQ_PAGED_FULL) ? 0 : 1;
    w.prefix_len = d->prefix_len;
    w.scale_log2 = d->scale * 1.4426950408889634f;
    w.q = d->q;
    w.ldq = d->ldq;
    w.out = d->out;
    w.ldo = d->ldo;
    w.lse = d->lse;
    w.ldl = d->ldl;
    w.bases = reinterpret_cast<long long*>(ws + pl.bases);
    w.part_o = f32(pl.own_o);
    w.part_ml = f32x2(pl.own_ml);
    p.own_grid = pl.own.grid;
    if (d->prefix_len > 0) {
        w.row_o = f32(pl.row_o);
        w.row_ml = f32x2(pl.row_ml);
        PagedWork pre = w;
        pre.prefix_pass = 1;
        pre.bases = nullptr;
        pre.part_o = f32(pl.pre_o);
        pre.part_ml = f32x2(pl.pre_ml);
        pre.row_o = f32(pl.pre_row_o);
        pre.row_ml = f32x2(pl.pre_row_ml);
        rc = launch_pass(pl.pre, pre, d, stream);
        if (rc) return rc;
        p.pre = PagedPrefixParts{pre.part_o, pre.part_ml, pre.row_o, pre.row_ml, pl.pre.rows, pl.pre.unit, pl.pre.grid};
    }
    rc = launch_pass(pl.own, w, d, stream);
    if (rc) return rc;
    const bool bf = d->kv.dtype == BQ_DT_BF16;
    const void* fn = d->kv.D == 128 ? (bf ? join_kernel<__nv_bfloat16, 128>(pl.own.wide) : join_kernel<__half, 128>(pl.own.wide))
                                    : (bf ? join_kernel<__nv_bfloat16, 64>(pl.own.wide) : join_kernel<__half, 64>(pl.own.wide));
    void* args[] = {&p};
    return paged_launch(fn, dim3(d->T, d->HQ), dim3(kJoinThreads), 0, args, d->flags, stream, "paged attention join");
}

}  // extern "C"
