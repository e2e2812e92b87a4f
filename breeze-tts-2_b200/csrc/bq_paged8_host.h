// Host-side helpers of the 8-bit paged KV cache.
#pragma once

#include "bq_paged_host.h"

namespace bq {

struct Paged8Scales;

// What a tile's start and end cost in units in the kernel for few rows (bq_paged8_narrow.cu), whose tile, unit and
// warps are those of its 16-bit counterpart.
constexpr int kNarrow8Overhead = 5;
int paged8_launch_narrow(const PagedWork& w, const Paged8Scales& sc, int dtype, int D, int grid, uint32_t flags, void* stream);
// The kernel for many rows (bq_paged8_wide.cu), with the tile and unit of its 16-bit counterpart.
constexpr int kWide8Overhead = 3;
int paged8_launch_wide(const PagedWork& w, const Paged8Scales& sc, const bq_paged8_kv* kv, int grid, uint32_t flags, void* stream);
// The form for few rows with a cluster of `ranks` CTAs per (sequence, kv head).
int paged8_launch_cluster(const PagedWork& w, const Paged8Scales& sc, int dtype, int D, int ranks, uint32_t flags, void* stream);

// Checks the cache part of a descriptor with T rows; HQ query heads (0: none).
int paged8_validate(const bq_paged8_kv* kv, int T, int HQ, bool f32 = false);
int paged8_fill(PagedKV* out, Paged8Scales* scales, const bq_paged8_kv* kv, int T, int HQ);
// Rows of a window of the kernels that walk ragged rows: a power of two of at most T / B and `most`, so that
// a window holds rows of few sequences.
inline int paged8_window(const bq_paged8_kv* kv, int T, int most) {
    int w = 1;
    while (2 * w <= most && int64_t(2 * w) * kv->B <= T) w *= 2;
    return w;
}

}  // namespace bq
