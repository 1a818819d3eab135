// Work items of the attention over a shared prefix and own tokens: what its kernels share.
#pragma once

#include "mma.cuh"
#include "paged.cuh"
#include "rows.cuh"

namespace b200 {

constexpr int kUnit = 64;   // keys of a step; splits are whole steps

struct PrefixParams {
    RowsView rows;
    PagesView own, prefix;
    int heads, group, dim, groups;
    int row_begin, row_end;    // of this launch: the rows of the pass from row_begin on, whose partial results begin there
    Divider by_group;
    const int32_t *group_first, *group_prefix, *prefix_length;
    const void* query;
    float scale;               // times log2(e)
    int prefix_splits, own_splits;
    int prefix_tiles;          // row tiles of all groups, at most
    int own_tiles;             // row tiles per sequence, at most
    int prefix_rows, own_rows; // pairs of a row tile
    int items;                 // of this launch
    int beside;                // 1: the prefix's items are another kernel's, launched just before, beside which this one runs
    int joined;                // 1: the own tokens' items go over the keys of their sequence's prefix first and leave results, not partial ones
    int planes;                // 1: weights as two bf16 planes
    int wide_out;              // results on 16-byte boundaries
    int32_t* status;
    float* part_o;             // [(row_end - row_begin) * heads][splits][dim]
    float* part_ml;            // [(row_end - row_begin) * heads][splits][2]
    float* out;
    __nv_bfloat16 *out_hi, *out_lo;
    int64_t out_stride;
};

struct KeySpan { int begin, end; };
// Split `index` of `total` keys.
__device__ __forceinline__ KeySpan split_span(int total, int splits, int index) {
    const int steps = (total + kUnit - 1) / kUnit, per = (steps + splits - 1) / splits;
    const int begin = min(total, index * per * kUnit);
    return {begin, min(total, begin + per * kUnit)};
}
// The splits of `total` keys that begin before key `seen`.
__device__ __forceinline__ int used_splits(int total, int splits, int seen) {
    const int steps = (total + kUnit - 1) / kUnit;
    if (steps == 0 || seen <= 0) return 0;
    const int per = (steps + splits - 1) / splits * kUnit;
    return (min(seen, total) + per - 1) / per;
}

// The weights of the softmax as the tensor cores take them.  What they are relative to, a running maximum, hangs on the split, the tile and the form, and these on
// the batch, so it is a whole number of powers of two (whole_maximum): another one shifts a weight's exponent and leaves its rounding alone.  (Rounded relative to
// the maximum itself, f32 results of peaked rows moved by up to 9e-3 from batch to batch, and a third of all bf16 results by a step.)
//   PLANES, for results in f32 or two planes: two bf16 planes, 15 bits.  The first is cut off, not rounded, and the second larger by 2^-23 of the weight, so that
//   both are positive where the weight is (down to 2^-109) and an infinite value stays one.
//   Otherwise, for bf16 results, one plane of 8 bits, and the sum is that of the rounded weights: rounding the largest ones cancels.  Half the products.
__device__ __forceinline__ float whole_maximum(float top) { return top == -INFINITY ? 0.0f : ceilf(top); }
__device__ __forceinline__ uint32_t first_plane(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }
__device__ __forceinline__ uint32_t second_plane(float a, float b) {
    const float high_a = __uint_as_float(__float_as_uint(a) & 0xffff0000u), high_b = __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    return pack_bf16(fmaf(a, 0x1.000002p0f, -high_a), fmaf(b, 0x1.000002p0f, -high_b));
}

// Keys of the prefix in a slot of its table.
__device__ __forceinline__ int prefix_keys(const PrefixParams& p, int slot) {
    if (slot < 0 || slot >= p.prefix.sequences) return 0;
    return max(0, min(__ldg(p.prefix_length + slot), p.prefix.capacity()));
}
__device__ __forceinline__ int own_keys(const PrefixParams& p, int slot, int count) {
    if (slot < 0 || slot >= p.own.sequences) return 0;
    return max(0, min(p.rows.lengths[slot] + count, p.own.capacity()));
}

// One item: the rows m_begin .. m_count - 1 of (row, head of the group) pairs from `row` on, and a span of keys.
struct Item {
    bool live, causal;
    int row, m_begin, m_count;   // first row of the group or sequence; pair m is row + m / group, head kv_head * group + m % group
    int kv_head, slot, split;    // split: which partial result
    int visible;                 // keys that pair 0 sees (causal: pair m sees m / group more)
    KeySpan keys;
    int shared_slot, shared;     // joined: the prefix and its keys, which are seen before `keys`
};

// Items are numbered split-major inside a kind; the prefix's, which are longer, come first.
__device__ __forceinline__ int prefix_items(const PrefixParams& p) { return p.prefix_tiles * p.own.kv_heads * p.prefix_splits; }

// Item `index` of the prefix, worked out by a whole warp.
__device__ __forceinline__ Item find_prefix_item(const PrefixParams& p, int index) {
    Item it{};
    const int kv_heads = p.own.kv_heads, lane = threadIdx.x & 31;
    it.kv_head = index % kv_heads;
    const int rest = index / kv_heads;
    int tile = rest % p.prefix_tiles;
    it.split = rest / p.prefix_tiles;
    // tile -> group: the groups' tile counts are added up 32 at a time
    for (int base = 0; base < p.groups; base += 32) {
        const int g = base + lane;
        int begin = 0, rows = 0, tiles = 0, slot = -1, keys = 0;
        if (g < p.groups) {   // two rounds of loads that do not wait for one another
            const int from = __ldg(p.group_first + g), to = __ldg(p.group_first + g + 1);
            slot = __ldg(p.group_prefix + g);
            begin = max(__ldg(p.rows.first + from), p.row_begin);
            rows = max(0, min(__ldg(p.rows.first + to), p.row_end) - begin);
            keys = prefix_keys(p, slot);
            tiles = (rows * p.group + p.prefix_rows - 1) / p.prefix_rows;
        }
        int up_to = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, up_to, o);
            if (lane >= o) up_to += other;
        }
        const unsigned found = __ballot_sync(0xffffffffu, up_to > tile);
        if (found) {
            const int from = __ffs(found) - 1;
            it.row = __shfl_sync(0xffffffffu, begin, from);
            it.m_count = __shfl_sync(0xffffffffu, rows, from) * p.group;
            it.m_begin = (tile - __shfl_sync(0xffffffffu, up_to - tiles, from)) * p.prefix_rows;
            it.slot = __shfl_sync(0xffffffffu, slot, from);
            keys = __shfl_sync(0xffffffffu, keys, from);
            it.keys = split_span(keys, p.prefix_splits, it.split);
            it.visible = keys;
            it.live = it.keys.begin < it.keys.end;
            return it;
        }
        tile -= __shfl_sync(0xffffffffu, up_to, 31);
    }
    return it;
}

// The group of sequence s, -1 for none: groups own consecutive sequences.
__device__ __forceinline__ int group_of(const PrefixParams& p, int s) {
    if (p.groups == 0 || s < __ldg(p.group_first)) return -1;
    int low = 0, high = p.groups;   // group_first[low] <= s, and s < group_first[high] unless high is the end
    while (high - low > 1) {
        const int middle = (low + high) / 2;
        if (__ldg(p.group_first + middle) <= s) low = middle;
        else high = middle;
    }
    return s < __ldg(p.group_first + low + 1) ? low : -1;
}

// Item `index` of the own tokens, by any one thread.
__device__ __forceinline__ Item find_own_item(const PrefixParams& p, int index) {
    Item it{};
    const int kv_heads = p.own.kv_heads;
    it.kv_head = index % kv_heads;
    int rest = index / kv_heads;
    const int tile = rest % p.own_tiles;
    rest /= p.own_tiles;
    const int s = rest % p.rows.sequences, split = rest / p.rows.sequences;
    it.split = p.prefix_splits + split;
    const int first = __ldg(p.rows.first + s), count = max(0, __ldg(p.rows.first + s + 1) - first);
    it.row = max(first, p.row_begin);
    it.m_count = max(0, min(first + count, p.row_end) - it.row) * p.group;
    it.m_begin = tile * p.own_rows;
    it.slot = __ldg(p.rows.slot + s);
    const int length = it.slot >= 0 && it.slot < p.own.sequences ? p.rows.lengths[it.slot] : INT32_MIN / 2;
    const int keys = max(0, min(length + count, p.own.capacity()));
    it.keys = split_span(keys, p.own_splits, split);
    it.causal = true;
    it.visible = length + 1 + it.row - first;
    // no further than the tile's last pair sees
    it.keys.end = min(it.keys.end, it.visible + divide(max(0, min(it.m_begin + p.own_rows, it.m_count) - 1), p.by_group));
    it.live = it.m_begin < it.m_count && it.keys.begin < it.keys.end;
    if (p.joined) {
        it.keys.end = max(0, it.keys.end);
        it.live = it.m_begin < it.m_count;
        const int g = group_of(p, s);
        if (g >= 0) {
            it.shared_slot = __ldg(p.group_prefix + g);
            it.shared = prefix_keys(p, it.shared_slot);
        }
    }
    return it;
}
__device__ __forceinline__ Item find_item(const PrefixParams& p, int index) {
    return index < prefix_items(p) ? find_prefix_item(p, index) : find_own_item(p, index - prefix_items(p));
}
__device__ __forceinline__ Item item_of_lane(const Item& it, int lane) {
    Item r;
    r.live = __shfl_sync(0xffffffffu, it.live, lane);
    r.causal = __shfl_sync(0xffffffffu, it.causal, lane);
    r.row = __shfl_sync(0xffffffffu, it.row, lane);
    r.m_begin = __shfl_sync(0xffffffffu, it.m_begin, lane);
    r.m_count = __shfl_sync(0xffffffffu, it.m_count, lane);
    r.kv_head = __shfl_sync(0xffffffffu, it.kv_head, lane);
    r.slot = __shfl_sync(0xffffffffu, it.slot, lane);
    r.split = __shfl_sync(0xffffffffu, it.split, lane);
    r.visible = __shfl_sync(0xffffffffu, it.visible, lane);
    r.keys.begin = __shfl_sync(0xffffffffu, it.keys.begin, lane);
    r.keys.end = __shfl_sync(0xffffffffu, it.keys.end, lane);
    r.shared_slot = __shfl_sync(0xffffffffu, it.shared_slot, lane);
    r.shared = __shfl_sync(0xffffffffu, it.shared, lane);
    return r;
}

// A kernel that runs beside the prefix's: that one let it start when everything before both was complete, so it need not wait to begin; its first CTA waits
// before it ends, so that the kernel is complete no earlier than the other and the merge can wait for this one alone.  This holds because the prefix's kernel is
// launched just before it on the same stream, and all its CTAs wait before they let it start.
__device__ __forceinline__ void begin_items(const PrefixParams& p) {
    if (!p.beside) grid_dependency_wait();
    grid_launch_dependents();
}
__device__ __forceinline__ void end_items(const PrefixParams& p) {
    if (p.beside && blockIdx.x == 0) grid_dependency_wait();
}
__device__ __forceinline__ int first_item(const PrefixParams& p) { return p.beside ? prefix_items(p) : 0; }

// Pair m of an item among the pass's rows * heads, and where it leaves its partial result, a row of [(row_end - row_begin) * heads][splits].
__device__ __forceinline__ int64_t pair_row(const PrefixParams& p, const Item& it, int m) {
    return static_cast<int64_t>(it.row) * p.heads + it.kv_head * p.group + static_cast<int64_t>(divide(m, p.by_group)) * (p.heads - p.group) + m;
}
// Where the results of a pair begin.
__device__ __forceinline__ int64_t result_at(const PrefixParams& p, const Item& it, int m) {
    const int of_row = divide(m, p.by_group);
    return (it.row + of_row) * p.out_stride + static_cast<int64_t>(it.kv_head * p.group + m - of_row * p.group) * p.dim;
}
// N adjacent results, 2 or 4, at a multiple of N values behind a pair's begin.
template <int N> __device__ __forceinline__ void store_results(const PrefixParams& p, int64_t at, const float (&v)[N]) {
    if (!p.wide_out) {
#pragma unroll
        for (int u = 0; u < N; ++u) store_forms(v[u], at + u, p.out, p.out_hi, p.out_lo);
        return;
    }
    if (p.out) {
        if constexpr (N == 4) *reinterpret_cast<float4*>(p.out + at) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<float2*>(p.out + at) = make_float2(v[0], v[1]);
    }
    if (p.out_hi) {
        uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
        for (int u = 0; u < N / 2; ++u) pack_planes(v[2 * u], v[2 * u + 1], hi[u], lo[u]);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __nv_bfloat16* to = which ? p.out_lo : p.out_hi;
            const uint32_t(&x)[N / 2] = which ? lo : hi;
            if (!to) continue;
            if constexpr (N == 4) *reinterpret_cast<uint2*>(to + at) = make_uint2(x[0], x[1]);
            else *reinterpret_cast<uint32_t*>(to + at) = x[0];
        }
    }
}
__device__ __forceinline__ int64_t partial_row(const PrefixParams& p, const Item& it, int m) {
    return (pair_row(p, it, m) - static_cast<int64_t>(p.row_begin) * p.heads) * (p.prefix_splits + p.own_splits) + it.split;
}

}  // namespace b200
