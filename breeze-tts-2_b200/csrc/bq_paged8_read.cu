// bq_paged8_read: the last positions of each sequence of an 8-bit paged cache as
// rows of bf16, fp16 or fp32: code * 2^e, one rounding (none in bf16 and fp32, whose
// exponents reach further than the cache's).
//
// Bound: HBM, 1 byte read and 2 (4) written per element. A CTA takes a window of
// rows and some heads of k or of v; a thread turns 16 codes at a time (32 bytes out),
// several of them in flight. Measured: 96925 rows of 8 heads of 128 to bf16, 595 MB in
// 105 us (5.7 TB/s), to fp32 178 us (991 MB, 5.6 TB/s); 410 rows of 16 heads 4.4 us. Two
// stores of 16 bytes instead of one of 32 cost the long case 5 %.
#include <cstring>

#include "bq_host.h"
#include "bq_paged8.cuh"
#include "bq_paged8_host.h"

namespace bq {
namespace {

constexpr int kThreads = 256, kMostRows = 64, kMostHeads = 8;

struct Read8Params {
    PagedKV kv;
    Paged8Scales sc;
    int32_t window, head_shift;  // rows and 2^x heads of a CTA
    int32_t aligned;             // outputs are 32-byte aligned
    void* k_out;
    int64_t ko_row, ko_head;
    void* v_out;
    int64_t vo_row, vo_head;
};

// 32 bytes by one instruction where they are aligned: a warp then writes whole sectors.
__device__ __forceinline__ void store32(void* dst, const uint4& a, const uint4& b, bool aligned) {
    if (aligned) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x),
                     "r"(b.y), "r"(b.z), "r"(b.w)
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(dst)[0] = a;
        reinterpret_cast<uint4*>(dst)[1] = b;
    }
}
template <typename T>
__device__ __forceinline__ void store16(T* dst, const float (&v)[16], bool aligned) {
    if constexpr (sizeof(T) == 4) {
        uint4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                              __float_as_uint(v[4 * i + 3]));
        store32(dst, x[0], x[1], aligned);
        store32(dst + 8, x[2], x[3], aligned);
    } else {
        float a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = v[i], b[i] = v[8 + i];
        store32(dst, pack8<T>(a), pack8<T>(b), aligned);
    }
}

// FLIGHT: pieces that a thread has on their way. Four where all CTAs run at once (they fit an SM four times); two where
// more CTAs come after one another, eight on an SM then (96925 rows of 8 heads of 128: 122 us with four, 105 with two;
// 410 rows of 16 heads: 4.4 and 5.0; 6500 rows of 8: 9.6 and 16).
template <typename T, int D, int FLIGHT>
__global__ void __launch_bounds__(kThreads, FLIGHT == 2 ? 8 : 1) read8_kernel(const __grid_constant__ Read8Params p) {
    constexpr int CH = D / 16;  // pieces of a head
    __shared__ int s_page[kMostRows], s_slot[kMostRows];
    pdl_launch_dependents();
    pdl_wait();
    const PagedKV& kv = p.kv;
    const int w0 = blockIdx.x * p.window, rows = min(p.window, kv.T - w0);
    const int half = gridDim.y / 2, h0 = int(blockIdx.y) % half << p.head_shift;
    const bool is_k = int(blockIdx.y) < half;
    const int CHH = CH << p.head_shift;  // pieces of a row
    const int row_shift = p.head_shift + (D == 128 ? 3 : 2);

    // page (-1: leave the row) and slot of every row of the window
    auto place = [&](int r, int b, int pos) {
        bool ok = (pos >> kv.page_shift) < kv.max_pages;
        if (pos < 0) {
            s_page[r] = -1;
            return;
        }
        if (!ok) {
            if (blockIdx.y == 0) atomicOr(kv.errors, BQ_DEVERR_POSITION_BIT);
            s_page[r] = -1;
            return;
        }
        const int page = paged_page(kv, b, pos, ok);
        if (!ok && blockIdx.y == 0) atomicOr(kv.errors, BQ_DEVERR_PAGE_BIT);
        s_page[r] = ok ? page : -1;
        s_slot[r] = pos & kv.page_mask;
    };
    if (!kv.starts) {
        if (int(threadIdx.x) < rows) place(threadIdx.x, w0 + threadIdx.x, max(kv.lens[w0 + threadIdx.x], 0) - 1);
    } else {
        if (threadIdx.x < kMostRows) s_page[threadIdx.x] = -1;
        __shared__ int s_end[kMostRows], s_pos[kMostRows], s_seq[kMostRows];  // of the sequence whose first row in the window is r
        if (threadIdx.x < kMostRows) s_seq[threadIdx.x] = -1;
        __syncthreads();
        for (int b = threadIdx.x; b < kv.B; b += kThreads) {
            int begin, n;
            paged_rows(kv, b, begin, n);
            const int lo = max(begin, w0), hi = min(begin + n, w0 + rows);
            if (lo >= hi) continue;
            s_seq[lo - w0] = b;
            s_end[lo - w0] = hi - w0;
            s_pos[lo - w0] = max(kv.lens[b], 0) - n + (lo - begin);
        }
        __syncthreads();
        if (int(threadIdx.x) < rows)
            for (int r = threadIdx.x; r >= 0; --r)
                if (s_seq[r] >= 0) {
                    if (int(threadIdx.x) < s_end[r]) place(threadIdx.x, s_seq[r], s_pos[r] + (int(threadIdx.x) - r));
                    break;
                }
    }
    __syncthreads();

    const uint8_t* pages = static_cast<const uint8_t*>(is_k ? kv.k : kv.v);
    const int64_t st_page = is_k ? kv.ks_page : kv.vs_page, st_head = is_k ? kv.ks_head : kv.vs_head,
                  st_slot = is_k ? kv.ks_slot : kv.vs_slot;
    T* out = static_cast<T*>(is_k ? p.k_out : p.v_out);
    const int64_t o_row = is_k ? p.ko_row : p.vo_row, o_head = is_k ? p.ko_head : p.vo_head;
    const int total = rows * CHH;
    for (int i0 = threadIdx.x; i0 < total; i0 += kThreads * FLIGHT) {
        uint4 w[FLIGHT];
        uint8_t e[FLIGHT];
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) {
            const int i = i0 + f * kThreads, r = i >> row_shift, h = h0 + (i & (CHH - 1)) / CH, c = i % CH;
            w[f] = make_uint4(0, 0, 0, 0);
            e[f] = kExpBias;
            if (i < total && h < kv.HKV && s_page[r] >= 0) {
                const int page = s_page[r], slot = s_slot[r], blk = slot >> p.sc.block_shift;
                w[f] = *reinterpret_cast<const uint4*>(pages + page * st_page + h * st_head + slot * st_slot + c * 16);
                e[f] = is_k ? *k_scale(p.sc, page, h, blk) : *v_scale(p.sc, page, h, blk);
            }
        }
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) {
            const int i = i0 + f * kThreads, r = i >> row_shift, h = h0 + (i & (CHH - 1)) / CH, c = i % CH;
            if (i >= total || h >= kv.HKV || s_page[r] < 0) continue;
            const float s = exp_scale(scale_exp(e[f]));
            const uint32_t words[4] = {w[f].x, w[f].y, w[f].z, w[f].w};
            float v[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float x[4];
                codes_f32(words[q], x);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[4 * q + k] = x[k] * s;
                    if constexpr (std::is_same_v<T, __half>)  // a finite entry stays finite
                        v[4 * q + k] = v[4 * q + k] > 65504.f ? 65504.f : v[4 * q + k] < -65504.f ? -65504.f : v[4 * q + k];
                }
            }
            store16<T>(out + (w0 + r) * o_row + h * o_head + c * 16, v, p.aligned);
        }
    }
}

template <int D, int FLIGHT>
const void* read_kernel(int dtype) {
    return dtype == BQ_DT_BF16  ? reinterpret_cast<const void*>(&read8_kernel<__nv_bfloat16, D, FLIGHT>)
           : dtype == BQ_DT_F16 ? reinterpret_cast<const void*>(&read8_kernel<__half, D, FLIGHT>)
                                : reinterpret_cast<const void*>(&read8_kernel<float, D, FLIGHT>);
}

}  // namespace
}  // namespace bq

using namespace bq;

extern "C" int32_t bq_paged8_read(const bq_paged8_read_desc* d, void* stream) {
    if (!d) return set_error(BQ_ERR_INVALID_ARG, "desc is NULL");
    int rc = paged8_validate(&d->kv, d->T, 0, true);
    if (rc) return rc;
    if (d->T == 0) return BQ_OK;
    if (!d->k_out || !d->v_out) return set_error(BQ_ERR_INVALID_ARG, "k_out and v_out must be non-NULL");
    const int elem = dtype_size(d->kv.dtype), size[2] = {d->T, d->kv.HKV};
    for (int i = 0; i < 2; ++i) {
        if (size[i] == 1) continue;  // its stride is never taken
        if (d->ko_stride[i] < d->kv.D || d->vo_stride[i] < d->kv.D)
            return set_error(BQ_ERR_SHAPE, "strides of k_out and v_out must be at least the head dim");
        if (d->ko_stride[i] * elem % 16 || d->vo_stride[i] * elem % 16)
            return set_error(BQ_ERR_ALIGN, "rows and heads of k_out and v_out must be 16-byte aligned");
    }
    if (!paged_aligned(d->k_out, 0, elem) || !paged_aligned(d->v_out, 0, elem))
        return set_error(BQ_ERR_ALIGN, "k_out and v_out must be 16-byte aligned");
    rc = paged_check_device();
    if (rc) return rc;
    Read8Params p;
    std::memset(&p, 0, sizeof(p));
    rc = paged8_fill(&p.kv, &p.sc, &d->kv, d->T, 0);
    if (rc) return rc;
    // A CTA's start (its rows' sequences, lengths and pages) takes as long as some 16 KB of codes do: large pieces (96925 rows
    // of 8 heads of 128: 32 rows of 2 / 4 / 8 heads 253 / 162 / 124 us, 64 of 8 122 us), but two CTAs for every SM, so that
    // enough is on its way (at least one / two / four for each: 5000 rows of 8 heads 15.7 / 9.6 / 10.8 us, 3000 rows 9.3 /
    // 6.5 / 7.2, 410 rows of 16 heads 4.5 / 4.4 / 4.5).
    const DeviceInfo* di = device_info();
    if (!di) return BQ_ERR_CUDA;
    int heads = 1;
    while (heads < d->kv.HKV && heads < kMostHeads) heads *= 2;
    p.window = paged8_window(&d->kv, d->T, kMostRows);
    while (int64_t((d->T + p.window - 1) / p.window) * 2 * ((d->kv.HKV + heads - 1) / heads) < 2 * di->sm_count) {
        if (p.window > 16 || (heads == 1 && p.window > 4))
            p.window /= 2;
        else if (heads > 1)
            heads /= 2;
        else
            break;
    }
    p.head_shift = __builtin_ctz(unsigned(heads));
    p.k_out = d->k_out;
    p.ko_row = d->ko_stride[0];
    p.ko_head = d->ko_stride[1];
    p.v_out = d->v_out;
    p.vo_row = d->vo_stride[0];
    p.vo_head = d->vo_stride[1];
    p.aligned = ((reinterpret_cast<uintptr_t>(d->k_out) | reinterpret_cast<uintptr_t>(d->v_out)) & 31) == 0;
    for (int i = 0; i < 2; ++i)
        if (size[i] > 1 && (d->ko_stride[i] * elem % 32 || d->vo_stride[i] * elem % 32)) p.aligned = 0;
    const dim3 grid((d->T + p.window - 1) / p.window, 2 * ((d->kv.HKV + heads - 1) / heads));
    const bool many = int64_t(grid.x) * grid.y > 4 * di->sm_count;
    const void* fn = d->kv.D == 128 ? (many ? read_kernel<128, 2>(d->kv.dtype) : read_kernel<128, 4>(d->kv.dtype))
                                    : (many ? read_kernel<64, 2>(d->kv.dtype) : read_kernel<64, 4>(d->kv.dtype));
    void* args[] = {&p};
    return paged_launch(fn, grid, dim3(kThreads), 0, args, d->flags, stream, "paged read");
}
