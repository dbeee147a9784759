// paged.h -- the rotation table, the paged cache and the ragged batch as the
// kernels see them (rope.hip, paged_attention.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "lq8_internal.h"

struct lq8_rope {
    int device = 0;
    lq8_rope_config cfg{};
    void* table = nullptr;  // device: RopePair [rotary_dim / 2]
};

namespace lq8 {

// One pair's rotation: turns (full circles) per position, and its axis.
struct RopePair {
    double turns;
    int axis, pad;
};

constexpr int PAGE_MIN = 16, PAGE_MAX = 1024;
constexpr uint32_t MAX_KV_HEADS = 1024, MAX_HEADS = 16384, MAX_BATCH = 65536;
// a launch has at most 2^32 threads, and there may be 256 of a row, or of a row's head
constexpr uint32_t MAX_ROWS = 1u << 23, MAX_ROW_HEADS = 1u << 23;

// Element types of a call: rows in T, pages in C.
enum PagedTypes : int { PT_F32_F32 = 0, PT_F32_BF16 = 1, PT_BF16_BF16 = 2 };

struct PagesDev {
    void *k, *v;
    int num_pages, page_shift, kv_heads;
    size_t page_stride;  // elements
};

struct BatchDev {
    int batch, rows, max_rows, max_pages;
    const int32_t *row_begin, *lengths, *pages;
};

// Rows of sequence s, inside [0, rows] whatever row_begin says: `total` of
// them, of which the first `count` are worked on (max_rows).
struct RowRange {
    int first, total, count;
};
__device__ __forceinline__ RowRange rows_of(const BatchDev& b, int s) {
    if (!b.row_begin) return {s, 1, 1};
    const int lo = min(max(b.row_begin[s], 0), b.rows);
    const int hi = min(max(b.row_begin[s + 1], lo), b.rows);
    return {lo, hi - lo, min(hi - lo, b.max_rows)};
}

// Positions of a table with `length` of them that can exist.
__device__ __forceinline__ int held(int length, int max_pages, int page_shift) {
    return (int)min((int64_t)max(length, 0), (int64_t)max_pages << page_shift);
}

struct Bf16 {
    uint16_t bits;
};

// Restores the caller's current device.
struct DeviceGuard {
    int before = -1;
    lq8_status status = LQ8_OK;
    explicit DeviceGuard(int device) {
        hipError_t e = hipGetDevice(&before);
        if (e == hipSuccess && before != device) e = hipSetDevice(device);
        else if (e == hipSuccess) before = -1;
        if (e != hipSuccess) status = hip_fail(e, "device selection");
    }
    ~DeviceGuard() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// Host checks shared by the entry points (they need no device).
lq8_status check_pages(const lq8_kv_pages* kv, PagesDev* out);
lq8_status check_batch(const lq8_paged_batch* b, uint32_t page_size, BatchDev* out);
lq8_status check_types(int32_t rows, int32_t pages, PagedTypes* out);
lq8_status check_rows(const char* what, const void* p, size_t* stride, size_t width, size_t elem);

}  // namespace lq8
