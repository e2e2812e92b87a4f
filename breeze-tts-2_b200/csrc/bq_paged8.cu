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

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

struct Attn8Params {
    PagedKV kv;
    Paged8Scales sc;
    int32_t G, causal;
    float scale_log2;
    const void* q;
    int64_t ldq;
    void* out;
    int64_t ldo;
    float* lse;
    int64_t ldl;
};

// One warp per row and query head, position by position with a running maximum.
template <typename E, int D>
__global__ void __launch_bounds__(32 * kWarps) attend8_kernel(const __grid_constant__ Attn8Params p) {
    constexpr int DPL = D / 32;
    pdl_launch_dependents();
    pdl_wait();
    const PagedKV& kv = p.kv;
    const int lane = threadIdx.x & 31, h = blockIdx.y * kWarps + (threadIdx.x >> 5), t = blockIdx.x, j = h / p.G;
    if (h >= kv.HQ) return;
    int b = t;
    if (kv.starts) {
        if (t < kv.starts[0] || t >= kv.starts[kv.B]) return;
        int lo = 0, hi = kv.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (kv.starts[mid] <= t) lo = mid; else hi = mid;
        }
        b = lo;
    }
    int begin, count;
    paged_rows(kv, b, begin, count);
    bool cut;
    const int len = max(paged_len(kv, b, cut), 0);
    const int limit = p.causal ? max(0, min(len, max(kv.lens[b], 0) - count + (t - begin) + 1)) : len;
    if (cut && lane == 0) atomicOr(kv.errors, BQ_DEVERR_POSITION_BIT);
    float q[DPL], o[DPL] = {}, m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < DPL; ++i) {
        const E x = static_cast<const E*>(p.q)[int64_t(t) * p.ldq + h * D + lane * DPL + i];
        q[i] = float(x);
    }
    for (int pos = 0; pos < limit; ++pos) {
        const int page = paged_page(kv, b, pos, ok), slot = pos & kv.page_mask, blk = slot >> p.sc.block_shift;
        const uint8_t* kc = static_cast<const uint8_t*>(kv.k) + page * kv.ks_page + j * kv.ks_head + slot * kv.ks_slot + lane * DPL;
        const uint8_t* vc = static_cast<const uint8_t*>(kv.v) + page * kv.vs_page + j * kv.vs_head + slot * kv.vs_slot + lane * DPL;
        uint32_t kw, vw;
        if (DPL == 4) {
            kw = *reinterpret_cast<const uint32_t*>(kc);
            vw = *reinterpret_cast<const uint32_t*>(vc);
        } else {
            kw = *reinterpret_cast<const uint16_t*>(kc);
            vw = *reinterpret_cast<const uint16_t*>(vc);
        }
        float k[4], v[4], s = 0.f;
        codes_f32(kw, k);
        codes_f32(vw, v);
        for (int i = 0; i < DPL; ++i) s = fmaf(q[i], k[i], s);
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= p.scale_log2 * exp_scale(scale_exp(*k_scale(p.sc, page, j, blk)));
        const float nm = fmaxf(m, s), u = nm == -INFINITY ? 0.f : nm, f = exp2f(m - u), w = exp2f(s - u);
        const float sv = exp_scale(scale_exp(*v_scale(p.sc, page, j, blk)));
        m = nm;
        l = l * f + w;
        for (int i = 0; i < DPL; ++i) o[i] = o[i] * f + w * (v[i] * sv);
    }
    if (!ok && lane == 0) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
    const float inv = limit ? 1.f / l : 0.f;
    for (int i = 0; i < DPL; ++i) static_cast<E*>(p.out)[int64_t(t) * p.ldo + h * D + lane * DPL + i] = E(o[i] * inv);
    if (p.lse && lane == 0) p.lse[int64_t(t) * p.ldl + h] = l != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
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
    const int rc = validate_attention(d);
    if (rc) return rc;
    *bytes = 0;
    return BQ_OK;
}

int32_t bq_paged8_attention(const bq_paged8_attn_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = validate_attention(d);
    if (rc) return rc;
    if (d->T == 0) return BQ_OK;
    rc = paged_check_device();
    if (rc) return rc;
    Attn8Params p;
    std::memset(&p, 0, sizeof(p));
    rc = paged8_fill(&p.kv, &p.sc, &d->kv, d->T, d->HQ);
    if (rc) return rc;
    p.G = d->HQ / d->kv.HKV;
    p.causal = (d->flags & BQ_PAGED_FULL) ? 0 : 1;
    p.scale_log2 = d->scale * kLog2e;
    p.q = d->q;
    p.ldq = d->ldq;
    p.out = d->out;
    p.ldo = d->ldo;
    p.lse = d->lse;
    p.ldl = d->ldl;
    (void)workspace, (void)workspace_bytes;
    const bool bf = d->kv.dtype == BQ_DT_BF16;
    const void* fn = d->kv.D == 128 ? (bf ? reinterpret_cast<const void*>(&attend8_kernel<__nv_bfloat16, 128>)
                                          : reinterpret_cast<const void*>(&attend8_kernel<__half, 128>))
                                    : (bf ? reinterpret_cast<const void*>(&attend8_kernel<__nv_bfloat16, 64>)
                                          : reinterpret_cast<const void*>(&attend8_kernel<__half, 64>));
    void* args[] = {&p};
    return paged_launch(fn, dim3(d->T, (d->HQ + kWarps - 1) / kWarps), dim3(32 * kWarps), 0, args, d->flags, stream, "paged attention");
}

}  // extern "C"
