// What the kernels on paged KV caches share.
#pragma once

#include "attention_device.h"
#include "../../include/wick_rocm_lfm2.h"

namespace wick_rocm {

// Pages that rows take.
__host__ __device__ inline uint32_t pages_of(uint64_t rows, uint32_t page_shift) { return (uint32_t)((rows + (1u << page_shift) - 1u) >> page_shift); }

// Where token j of those that are appended goes: the row of its sequence (WICK_ROCM_NO_ROW: it is dropped) and the page of that row (none of the pool's: the row is).
struct PagedRows {
    const uint32_t *table, *start, *first;  // first may be null: token j is sequence j's
    uint32_t n_seqs, max_pages, n_pages, page_shift;
};
__device__ __forceinline__ uint32_t paged_row(const PagedRows& p, uint32_t j, uint32_t& page) {
    uint32_t s = j, in = 0;
    page = WICK_ROCM_NO_PAGE;
    if (p.first) {  // the last sequence whose tokens begin at or before this one
        uint32_t low = 0, high = p.n_seqs;
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2u;
            (p.first[mid] <= j ? low : high) = mid;
        }
        s = low, in = j - p.first[s];
        if (j < p.first[s] || j >= p.first[s + 1]) return WICK_ROCM_NO_ROW;
    }
    const uint32_t start = p.start[s], row = start + in;
    if (start == WICK_ROCM_NO_ROW || row < start) return WICK_ROCM_NO_ROW;
    if (row >> p.page_shift < p.max_pages) page = p.table[(size_t)s * p.max_pages + (row >> p.page_shift)];
    return row;
}
// Elements in front of that row in a plane.
__device__ __forceinline__ size_t paged_at(const PagedRows& p, uint32_t page, uint32_t row, uint32_t n_kv_heads, uint32_t c, uint32_t head_dim) {
    return ((((size_t)page * n_kv_heads + c) << p.page_shift) + (row & ((1u << p.page_shift) - 1u))) * head_dim;
}

// Sum over a wave's lanes up to this one, without LDS: inside rows of 16 lanes, then the last of a row to the next one, and of a half to the other.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_moved_or_zero(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v) {
    v += lane_moved_or_zero<0x111, 0xf>(v), v += lane_moved_or_zero<0x112, 0xf>(v), v += lane_moved_or_zero<0x114, 0xf>(v), v += lane_moved_or_zero<0x118, 0xf>(v);
    v += lane_moved_or_zero<0x142, 0xa>(v), v += lane_moved_or_zero<0x143, 0xc>(v);
    return v;
}

}  // namespace wick_rocm
