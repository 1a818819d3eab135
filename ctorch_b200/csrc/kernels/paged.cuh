// Device view of paged keys and values whose pages may be shared (b200_kv_pages).
#pragma once

#include "common.cuh"

namespace b200 {

struct PagesView {
    void* pool[2];  // 0 = K, 1 = V
    const int32_t* table;
    int64_t pages;
    int sequences, pages_per_seq, page_size, kv_heads, head_dim, dtype;
    __device__ __forceinline__ int capacity() const { return pages_per_seq * page_size; }
};

// The page of a position of a sequence, -1 where the table names none.
__device__ __forceinline__ int page_of(const PagesView& v, int sequence, int logical) {
    const int page = __ldg(v.table + static_cast<int64_t>(sequence) * v.pages_per_seq + logical);
    return page >= 0 && page < v.pages ? page : -1;
}
// First element of one head's row in a page.
__device__ __forceinline__ int64_t page_row(const PagesView& v, int page, int head, int slot) {
    return ((static_cast<int64_t>(page) * v.kv_heads + head) * v.page_size + slot) * v.head_dim;
}

// Checks and converts the C struct; false (with the error text set) when it is inconsistent.
bool pages_view(const b200_kv_pages& pages, const char* who, PagesView& view);

}  // namespace b200
