// bq_paged_append: the new tokens' q / k / v rows of a projection, per head
//   h = x * rsqrt(mean(x^2) + eps) * gain        (when norm weights are given)
//   y = h * cos[pos] + rotate_half(h) * sin[pos]  (q and k heads)
// in fp32, rounded once to the element type; q rows go to q_out, k and v rows
// into slot pos % page_size of page table[b][pos / page_size].
//
// Bound: HBM (every row is read once and written once, ~8 flops per element);
// for a decode step's handful of rows, the latency of the dependent loads
// (row -> sequence -> length -> page -> store). A head is one group of D / 8
// lanes holding 16 bytes each, so a row is read and written in full 128-byte
// lines, the norm is a shuffle reduction inside the group, and the rotation's
// partner (dim +- D / 2) is the lane half a group away.
//
// Measured (B200, in a graph): 2 rows of 48 heads of 128 in 1.9 us, 200 rows (5 MB) in
// 2.7 us, 2751 ragged rows of 40 heads of 64 (29 MB) in 10.2 us from L2, 12.4 us with
// other rows each call, 2.3 TB/s. Blocks of 64, 256
// and 512 threads, several rows per block and several heads per lane group were no
// faster.
#include <cstring>

#include "bq_host.h"
#include "bq_paged.cuh"
#include "bq_paged_host.h"

namespace bq {
namespace {

constexpr int kAppendThreads = 128;

struct AppendParams {
    PagedKV kv;
    int32_t rope_rows, has_norm;
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

template <typename C>
__device__ __forceinline__ void load8(const C* p, float (&v)[8]) {
    if constexpr (sizeof(C) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        unpack8<C>(*reinterpret_cast<const uint4*>(p), v);
    }
}

// E: element type, C: type of cos / sin (E or float).
template <typename E, typename C, int D>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int LG = D / 8;  // lanes per head
    constexpr int HEADS = kAppendThreads / LG;
    pdl_launch_dependents();
    pdl_wait();
    const PagedKV& kv = p.kv;
    const int t = blockIdx.x;
    const int l = threadIdx.x % LG;
    const int h = blockIdx.y * HEADS + threadIdx.x / LG;
    const int heads = kv.HQ + 2 * kv.HKV;
    const bool live = h < heads;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live) raw = *reinterpret_cast<const uint4*>(static_cast<const E*>(p.qkv) + int64_t(t) * p.ldqkv + h * D + l * 8);

    // Sequence of row t. With ragged rows every thread looks at some sequences, and the one that finds the row's
    // passes on what it read: one round of loads and a barrier, whatever the batch.
    int b = t, pos;
    if (kv.starts) {
        __shared__ int s_seq, s_pos;
        if (threadIdx.x == 0) s_seq = -1;
        __syncthreads();
        for (int i = threadIdx.x; i < kv.B; i += kAppendThreads) {
            const int begin = kv.starts[i], end = kv.starts[i + 1], len = max(kv.lens[i], 0);
            if (t >= begin && t < end) {
                s_seq = i;
                s_pos = len - (min(end, kv.T) - max(begin, 0)) + (t - max(begin, 0));
            }
        }
        __syncthreads();
        b = s_seq;
        if (b < 0) return;  // a row of no sequence
        pos = s_pos;
    } else {
        pos = max(kv.lens[b], 0) - 1;
    }
    if (pos < 0) return;  // an unused batch slot
    bool ok = pos < p.rope_rows && (pos >> kv.page_shift) < kv.max_pages;
    if (!ok) {
        if (threadIdx.x == 0) atomicOr(kv.errors, BQ_DEVERR_POSITION_BIT);
        return;
    }
    const int page = paged_page(kv, b, pos, ok);
    if (!ok) {
        if (threadIdx.x == 0) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
        return;
    }
    const int slot = pos & kv.page_mask;
    uint4 res = raw;
    if (blockIdx.y * HEADS < kv.HQ + kv.HKV) {  // block-uniform: some head of this block is a q or k head
        const bool rot = h < kv.HQ + kv.HKV;
        float v[8], c[8], s[8], o[8];
        unpack8<E>(raw, v);
        load8<C>(static_cast<const C*>(p.cos) + int64_t(pos) * p.ldcs + l * 8, c);
        load8<C>(static_cast<const C*>(p.sin) + int64_t(pos) * p.ldcs + l * 8, s);
        if (p.has_norm) {
            float g[8], ss = 0.f;
            load8<E>(static_cast<const E*>(h < kv.HQ ? p.qn : p.kn) + l * 8, g);
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
            o[i] = v[i] * c[i] + (l < LG / 2 ? -other : other) * s[i];
        }
        if (rot) res = pack8<E>(o);
    }
    if (!live) return;
    E* dst;
    if (h < kv.HQ)
        dst = static_cast<E*>(p.q_out) + int64_t(t) * p.ldq + h * D;
    else if (h < kv.HQ + kv.HKV)
        dst = static_cast<E*>(kv.k) + page * kv.ks_page + (h - kv.HQ) * kv.ks_head + slot * kv.ks_slot;
    else
        dst = static_cast<E*>(kv.v) + page * kv.vs_page + (h - kv.HQ - kv.HKV) * kv.vs_head + slot * kv.vs_slot;
    *reinterpret_cast<uint4*>(dst + l * 8) = res;
}

template <typename E>
const void* append_kernel(int D, bool cs_f32) {
    if (D == 128)
        return cs_f32 ? reinterpret_cast<const void*>(&paged_append_kernel<E, float, 128>)
                      : reinterpret_cast<const void*>(&paged_append_kernel<E, E, 128>);
    return cs_f32 ? reinterpret_cast<const void*>(&paged_append_kernel<E, float, 64>)
                  : reinterpret_cast<const void*>(&paged_append_kernel<E, E, 64>);
}

}  // namespace
}  // namespace bq

using namespace bq;

extern "C" int32_t bq_paged_append(const bq_paged_append_desc* d, void* stream) {
    if (!d) return set_error(BQ_ERR_INVALID_ARG, "desc is NULL");
    int rc = paged_validate(&d->kv, d->T, d->HQ);
    if (rc) return rc;
    if (d->T == 0) return BQ_OK;
    const int width = (d->HQ + 2 * d->kv.HKV) * d->kv.D;
    if (d->cs_dtype != d->kv.dtype && d->cs_dtype != BQ_DT_F32)
        return set_error(BQ_ERR_INVALID_ARG, "cos / sin must have the cache's dtype or fp32 (dtype %d)", d->cs_dtype);
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
    rc = paged_check_device();
    if (rc) return rc;
    AppendParams p;
    std::memset(&p, 0, sizeof(p));
    rc = paged_fill(&p.kv, &d->kv, d->T, d->HQ);
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
    const bool f32 = d->cs_dtype == BQ_DT_F32;
    const void* fn = d->kv.dtype == BQ_DT_BF16 ? append_kernel<__nv_bfloat16>(d->kv.D, f32)
                                               : append_kernel<__half>(d->kv.D, f32);
    const int heads = d->HQ + 2 * d->kv.HKV, per = kAppendThreads / (d->kv.D / 8);
    void* args[] = {&p};
    return paged_launch(fn, dim3(d->T, (heads + per - 1) / per), dim3(kAppendThreads), 0, args, d->flags, stream,
                        "paged append");
}
