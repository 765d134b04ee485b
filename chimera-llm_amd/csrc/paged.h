// What the kernels of the paged key/value cache share: the index arrays of a batch and the checks of the host structs.
#pragma once

#include "common.h"

namespace lcmhip {

// An index that no kernel of the call writes, read through the scalar path where its address is the same for a wave.
__host__ __device__ __forceinline__ int32_t read_index(const int32_t* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
#else
    return *p;
#endif
}

// A table of page ids as the kernels see it.  Nothing in the index arrays is trusted with an address: page() answers -1
// for an id outside the pool and for a position behind the table.
struct PageTable {
    const int32_t* ids;
    int max_pages;
    int page_shift;          // log2(page_size)
    uint32_t n_pages;
    __host__ __device__ __forceinline__ int page(int seq, int pos) const {   // pos >= 0
        const int p = pos >> page_shift;
        const int32_t id = read_index(ids + ((size_t)seq * max_pages + (p < max_pages ? p : max_pages - 1)));
        return p < max_pages && (uint32_t)id < n_pages ? id : -1;
    }
};

// Rows of sequence b in a batch of `rows` rows; starts == nullptr: row b.  The range is cut to [0, rows].
__host__ __device__ __forceinline__ void seq_rows(const int32_t* starts, int b, int64_t rows, int64_t& r0, int64_t& r1) {
    r0 = starts ? starts[b] : b;
    r1 = starts ? starts[b + 1] : b + 1;
    r0 = r0 < 0 ? 0 : (r0 < rows ? r0 : rows);
    r1 = r1 < r0 ? r0 : (r1 < rows ? r1 : rows);
}

// The number of entries of ends[0 .. n) that are <= t: for the non-falling ends of consecutive ranges, the range that holds
// t (n: none does).  One wave, every lane gets the answer; n / 64 independent loads.
__device__ __forceinline__ int wave_count_le(const int32_t* ends, int n, int64_t t) {
    const int lane = threadIdx.x & 63;
    int c = 0;
    for (int i = 0; i < n; i += 64) c += __popcll(__ballot(i + lane < n && ends[min(i + lane, n - 1)] <= t));
    return c;
}

constexpr int64_t kMaxBlocks = (1 << 24) - 1;   // workgroups of 256: a launch holds fewer than 2^32 work items
constexpr int kMaxKeys = 1 << 30;    // of one list: positions a few tiles behind the last are still int32

inline int check_pages(const lcmhip_kv_pages* p) {
    LCM_REQUIRE(p && p->k && p->v, "paged cache: null pages");
    LCM_REQUIRE(p->dtype == LCMHIP_F32 || p->dtype == LCMHIP_BF16, "paged cache: unknown dtype");
    LCM_REQUIRE(p->head_dim == 64 || p->head_dim == 128, "paged cache: head_dim must be 64 or 128");
    LCM_REQUIRE(p->page_size >= 16 && p->page_size <= 65536 && (p->page_size & (p->page_size - 1)) == 0,
                "paged cache: page_size must be a power of two in [16, 65536]");
    LCM_REQUIRE(p->n_kv_heads >= 1 && p->n_kv_heads <= 65535, "paged cache: n_kv_heads out of range");
    LCM_REQUIRE(p->n_pages >= 1 && p->n_pages <= INT32_MAX, "paged cache: n_pages out of range");
    LCM_REQUIRE(((uintptr_t)p->k | (uintptr_t)p->v) % 16 == 0, "paged cache: pages must be 16-byte aligned");
    return LCMHIP_OK;
}

inline int check_batch(const lcmhip_kv_pages* p, const lcmhip_paged_batch* b, int64_t rows) {
    LCM_REQUIRE(b && (b->n_seqs == 0 || (b->page_table && b->seq_lens)), "paged batch: null argument");
    LCM_REQUIRE(b->n_seqs >= 0 && b->n_seqs <= (1 << 24), "paged batch: n_seqs out of range");
    LCM_REQUIRE(b->max_pages >= 1, "paged batch: max_pages must be positive");
    LCM_REQUIRE(b->max_q >= 1, "paged batch: max_q must be positive");
    LCM_REQUIRE(b->max_keys >= 1 && b->max_keys <= kMaxKeys && b->max_keys <= (int64_t)b->max_pages * p->page_size,
                "paged batch: max_keys must be in [1, max_pages * page_size], at most 2^30");
    LCM_REQUIRE(rows >= 0 && rows <= (1 << 30), "paged batch: rows out of range");
    LCM_REQUIRE(b->q_starts || rows == b->n_seqs, "paged batch: without q_starts there is one row for every sequence");
    return LCMHIP_OK;
}

// Row tensors (rows, heads, head_dim): 16-byte pieces everywhere.
inline int check_rows(const void* x, int64_t row, int64_t head, int dtype, const char* what) {
    const int64_t unit = 16 / (int64_t)dtype_size(dtype);
    LCM_REQUIRE((uintptr_t)x % 16 == 0 && row % unit == 0 && head % unit == 0,
                std::string(what) + ": pointer and strides must be multiples of 16 bytes");
    return LCMHIP_OK;
}

// Whether two of the pieces of `d` values at t row + h head, t < rows, h < heads, share a value.  Strides of either sign: turning an
// axis round moves all pieces alike.
inline bool rows_overlap(int64_t rows, int64_t heads, int64_t row_stride, int64_t head_stride, int64_t d) {
    const __int128 row = row_stride < 0 ? -(__int128)row_stride : row_stride, head = head_stride < 0 ? -(__int128)head_stride : head_stride;
    if (heads <= 1) return rows > 1 && row < d;
    if (rows <= 1 || head < d) return head < d;
    if (row >= (heads - 1) * head + d) return false;       // rows one behind the other, the ordinary case
    if (row < d) return true;
    for (int64_t h = 1; h < heads; ++h) {                  // the rows t that begin next before and behind head h of row 0
        const __int128 t = h * head / row, before = h * head - t * row;
        if ((t < rows && before < d) || (t + 1 < rows && row - before < d)) return true;
    }
    return false;
}

inline int page_shift_of(const lcmhip_kv_pages* p) { return __builtin_ctz((unsigned)p->page_size); }

}  // namespace lcmhip
