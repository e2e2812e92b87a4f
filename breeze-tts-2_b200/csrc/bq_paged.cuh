// Shared pieces of the paged KV-cache operators (bq_paged_append,
// bq_paged_attention): the cache as the kernels see it, bounds-checked page
// lookup, and 16-byte vector conversions of the two element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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

// Eight elements of a 16-byte vector <-> fp32.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& r, float (&v)[8]);
template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4& r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
template <>
__device__ __forceinline__ void unpack8<__half>(const uint4& r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __half2 h;
        memcpy(&h, &w[i], 4);
        const float2 f = __half22float2(h);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
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

}  // namespace bq
