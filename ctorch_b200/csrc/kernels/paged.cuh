// Device view of paged keys and values whose pages may be shared (b200_kv_pages).
#pragma once

#include "common.cuh"

namespace b200 {

// n / d for 0 <= n < 2^31 by a multiplication: with 2^k the power of two from d on and f = ceil(2^(31 + k) / d) < 2^32, f d - 2^(31 + k) < d <= 2^k, so
// n f / 2^(31 + k) exceeds n / d by less than n 2^k / (d 2^(31 + k)) < 1 / d.
struct Divider {
    uint32_t factor;
    int shift;   // -1: d = 1
};
inline Divider divider(int d) {
    int k = 0;
    while ((1 << k) < d) ++k;
    if (k == 0) return {0, -1};
    return {static_cast<uint32_t>(((uint64_t{1} << (31 + k)) + d - 1) / d), k - 1};
}
__device__ __forceinline__ int divide(int n, Divider d) { return d.shift < 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), d.factor) >> d.shift); }

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
// Pool rows of the positions from, from + stride, ... of a sequence, as a copying warp walks them.  Page numbers are asked for two steps before they are
// wanted, since the way to L2 and back is longer than a step; places in the table and the page move on without divisions.
struct PageStream {
    const PagesView& view;
    const int32_t* table;
    int index, place, whole, rest, position, stride, end;   // index and place of the position that is asked for next
    int number[2], at[2];
    __device__ __forceinline__ PageStream(const PagesView& view, int sequence, int from, int stride, int end)
        : view(view), table(view.table + static_cast<int64_t>(sequence) * view.pages_per_seq), index(from / view.page_size), place(from % view.page_size),
          whole(stride / view.page_size), rest(stride % view.page_size), position(from), stride(stride), end(end) {
        ask(0);
        ask(1);
    }
    __device__ __forceinline__ void ask(int i) {
        number[i] = position < end ? __ldg(table + index) : -1;
        at[i] = place;
        position += stride;
        index += whole;
        place += rest;
        if (place >= view.page_size) {
            place -= view.page_size;
            ++index;
        }
    }
    // Row of the pools' [pages * kv_heads * page_size] rows that holds the next position; `outside` where there is none.
    __device__ __forceinline__ int next(int head, int outside) {
        const int page = number[0], row = at[0];
        number[0] = number[1];
        at[0] = at[1];
        ask(1);
        return page >= 0 && page < view.pages ? (page * view.kv_heads + head) * view.page_size + row : outside;
    }
};
// First element of one head's row in a page.
__device__ __forceinline__ int64_t page_row(const PagesView& v, int page, int head, int slot) {
    return ((static_cast<int64_t>(page) * v.kv_heads + head) * v.page_size + slot) * v.head_dim;
}

// Checks and converts the C struct; false (with the error text set) when it is inconsistent.
bool pages_view(const b200_kv_pages& pages, const char* who, PagesView& view);

}  // namespace b200
