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

constexpr int kThreads = 128;

struct PagedAttnParams {
    PagedKV kv;
    int32_t causal;
    float scale;
    const void* q;
    int64_t ldq;
    void* out;
    int64_t ldo;
    float* lse;
    int64_t ldl;
};

// One CTA per (row, query head): warps take every fourth cached position, the
// lanes of a warp the head's dimensions, with a running maximum and sum per
// warp; the four are joined at the end.
template <typename E, int D>
__global__ void __launch_bounds__(kThreads) paged_attention_rows_kernel(const __grid_constant__ PagedAttnParams p) {
    constexpr int DPL = D / 32;
    __shared__ float s_acc[4][D + 2];
    pdl_launch_dependents();
    pdl_wait();
    const PagedKV& kv = p.kv;
    const int t = blockIdx.x, h = blockIdx.y, j = h / (kv.HQ / kv.HKV);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int b = t;
    if (kv.starts) {
        int n = 0;
        for (int i0 = 0; i0 < kv.B; i0 += kThreads) {
            const int i = i0 + int(threadIdx.x);
            n += __syncthreads_count(i < kv.B && kv.starts[i + 1] <= t);
        }
        b = n;
        if (b >= kv.B) return;
    }
    int begin, count;
    paged_rows(kv, b, begin, count);
    if (t < begin || t >= begin + count) return;
    bool cut, ok = true;
    const int len = paged_len(kv, b, cut);
    const int limit = p.causal ? min(len, kv.lens[b] - count + (t - begin) + 1) : len;
    float qv[DPL], acc[DPL], m = -INFINITY, l = 0.f;
    const E* q = static_cast<const E*>(p.q) + int64_t(t) * p.ldq + h * D + lane * DPL;
#pragma unroll
    for (int e = 0; e < DPL; ++e) {
        qv[e] = float(q[e]) * p.scale;
        acc[e] = 0.f;
    }
    for (int s = warp; s < limit; s += 4) {
        const int64_t page = paged_page(kv, b, s, ok);
        const E* k = static_cast<const E*>(kv.k) + page * kv.ks_page + j * kv.ks_head + (s & kv.page_mask) * kv.ks_slot;
        const E* v = static_cast<const E*>(kv.v) + page * kv.vs_page + j * kv.vs_head + (s & kv.page_mask) * kv.vs_slot;
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < DPL; ++e) d = fmaf(qv[e], float(k[lane * DPL + e]), d);
#pragma unroll
        for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        const float nm = fmaxf(m, d), a = __expf(m - nm), w = __expf(d - nm);
        l = l * a + w;
#pragma unroll
        for (int e = 0; e < DPL; ++e) acc[e] = fmaf(w, float(v[lane * DPL + e]), acc[e] * a);
        m = nm;
    }
#pragma unroll
    for (int e = 0; e < DPL; ++e) s_acc[warp][lane * DPL + e] = acc[e];
    if (lane == 0) {
        s_acc[warp][D] = m;
        s_acc[warp][D + 1] = l;
        if (!ok) atomicOr(&g_device_error, BQ_DEVERR_PAGE_BIT);
        if (cut) atomicOr(&g_device_error, BQ_DEVERR_POSITION_BIT);
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    float mm = -INFINITY, ll = 0.f, aa = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, s_acc[w][D]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = s_acc[w][D + 1] > 0.f ? __expf(s_acc[w][D] - mm) : 0.f;
        ll += f * s_acc[w][D + 1];
        aa += f * s_acc[w][d];
    }
    static_cast<E*>(p.out)[int64_t(t) * p.ldo + h * D + d] = E(ll > 0.f ? aa / ll : 0.f);
    if (p.lse && d == 0) p.lse[int64_t(t) * p.ldl + h] = ll > 0.f ? mm + logf(ll) : -INFINITY;
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
    const int rc = validate_attention(d);
    if (rc) return rc;
    *bytes = 0;
    return BQ_OK;
}

int32_t bq_paged_attention(const bq_paged_attn_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = validate_attention(d);
    if (rc) return rc;
    (void)workspace;
    (void)workspace_bytes;
    if (d->T == 0) return BQ_OK;
    rc = paged_check_device();
    if (rc) return rc;
    PagedAttnParams p;
    std::memset(&p, 0, sizeof(p));
    paged_fill(&p.kv, &d->kv, d->T, d->HQ);
    p.causal = (d->flags & BQ_PAGED_FULL) ? 0 : 1;
    p.scale = d->scale;
    p.q = d->q;
    p.ldq = d->ldq;
    p.out = d->out;
    p.ldo = d->ldo;
    p.lse = d->lse;
    p.ldl = d->ldl;
    const bool bf = d->kv.dtype == BQ_DT_BF16;
    const void* fn = d->kv.D == 128 ? (bf ? reinterpret_cast<const void*>(&paged_attention_rows_kernel<__nv_bfloat16, 128>)
                                          : reinterpret_cast<const void*>(&paged_attention_rows_kernel<__half, 128>))
                                    : (bf ? reinterpret_cast<const void*>(&paged_attention_rows_kernel<__nv_bfloat16, 64>)
                                          : reinterpret_cast<const void*>(&paged_attention_rows_kernel<__half, 64>));
    void* args[] = {&p};
    return paged_launch(fn, dim3(d->T, d->HQ), dim3(kThreads), 0, args, d->flags, stream, "paged attention");
}

}  // extern "C"
