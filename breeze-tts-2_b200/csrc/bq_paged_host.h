// Host-side helpers of the paged KV-cache operators.
#pragma once

#include "bq_host.h"

namespace bq {

struct PagedKV;
struct PagedWork;

// Tile and unit of the kernel for few rows (bq_paged_narrow.cu), what a tile's
// start and end cost in units (with 0 / 1 / 2 / 4 units 48 streams of 17 to 6000
// positions take 66 / 48 / 44 / 44 us, two streams of 700 11.3 / 10.1 / 10.2 / 10.3 us),
// and its warps.
constexpr int kNarrowRows = 16, kNarrowUnit = 64, kNarrowOverhead = 2, kNarrowWarps = 4;
// The same of the kernel for many rows (bq_paged_wide.cu). Measured overheads: with 1 / 2 / 3 / 4 / 6 units a prompt
// of 7000 tokens takes 233 / 221 / 214 / 219 / 224 us, a chunk beside running streams 124 / 120 / 117 / 115 / 114 us.
constexpr int kWideRows = 256, kWideUnit = 128, kWideOverhead = 3;
int paged_launch_wide(const PagedWork& w, const bq_paged_kv* kv, int grid, uint32_t flags, void* stream);
int paged_launch_narrow(const PagedWork& w, int dtype, int D, int grid, uint32_t flags, void* stream);

// The form of the few-row kernel with a cluster of `ranks` CTAs per (sequence, kv head).
constexpr int kNarrowRanks = 8;
int paged_launch_cluster(const PagedWork& w, int dtype, int D, int ranks, uint32_t flags, void* stream);

// Checks the cache part of a descriptor with T new rows of HQ query heads.
int paged_validate(const bq_paged_kv* kv, int T, int HQ);
// BQ_OK when the current device is the one this library is built for.
int paged_check_device();
int paged_fill(PagedKV* out, const bq_paged_kv* kv, int T, int HQ);
// 16-byte aligned base and row stride (NULL counts as aligned).
inline bool paged_aligned(const void* p, int64_t ld, int elem) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * elem) % 16 == 0;
}
// cluster: CTAs per cluster along x (1: none).
int paged_launch(const void* fn, dim3 grid, dim3 block, uint32_t smem, void** args, uint32_t flags, void* stream,
                 const char* what, int cluster = 1);

}  // namespace bq
