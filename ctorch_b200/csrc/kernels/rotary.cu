// Rotary positions: tables of cosines and sines, scaled for long contexts, and the rotation of the queries and keys of a packed pass with
// the append of its keys and values to paged caches.
#include "mma.cuh"
#include "paged.cuh"
#include "rows.cuh"

#include <algorithm>
#include <cmath>

namespace b200 {

bool pages_view(const b200_kv_pages& p, const char* who, PagesView& view) {
    if ((p.dtype != B200_F32 && p.dtype != B200_BF16) || p.kv_heads <= 0 || p.head_dim <= 0 || p.page_size <= 0 || p.sequences <= 0 || p.pages_per_sequence <= 0
        || p.pages <= 0 || p.pages > INT32_MAX || !p.key || !p.value || !p.table || static_cast<int64_t>(p.pages_per_sequence) * p.page_size > INT32_MAX / 2) {
        set_error("%s: inconsistent pages (b200_kv_pages)", who);
        return false;
    }
    view = PagesView{{p.key, p.value}, p.table, p.pages, p.sequences, p.pages_per_sequence, p.page_size, p.kv_heads, p.head_dim, p.dtype};
    return true;
}

namespace {

// ---- tables -----------------------------------------------------------------------------------------------------------------------------
struct TableParams {
    double log_base, factor, original, low, high, magnitude;
    int kind, half, run;
    int64_t first, positions;
    float *cosine, *sine;
};

// A thread owns one frequency and `run` consecutive positions: sine and cosine of the first angle and of the step, then one complex product per position
// (a few 2^-53 each).  Bound by the stores: 64 k positions and more x 64 frequencies at 5 TB/s (sines and cosines of every single angle: 2 TB/s).
__global__ void __launch_bounds__(256) rotary_tables_kernel(const TableParams p) {
    const int64_t at = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
    const int i = static_cast<int>(at % p.half);
    const int64_t begin = at / p.half * p.run, end = min(begin + p.run, p.positions);
    double frequency = exp(-static_cast<double>(i) / p.half * p.log_base);
    if (p.kind == B200_ROTARY_LINEAR) frequency /= p.factor;
    if (p.kind == B200_ROTARY_PARTS) {
        const double turns = p.original * frequency * 0.15915494309189535;
        const double kept = fmin(1.0, fmax(0.0, (turns - p.low) / (p.high - p.low)));
        frequency *= kept + (1.0 - kept) / p.factor;
    }
    double s, c, step_s, step_c;
    sincos(static_cast<double>(p.first + begin) * frequency, &s, &c);
    sincos(frequency, &step_s, &step_c);
    s *= p.magnitude;
    c *= p.magnitude;
    grid_dependency_wait();   // the tables may still be read
    grid_launch_dependents();
    for (int64_t q = begin; q < end; ++q) {
        p.cosine[q * p.half + i] = static_cast<float>(c);
        p.sine[q * p.half + i] = static_cast<float>(s);
        const double next = c * step_c - s * step_s;
        s = s * step_c + c * step_s;
        c = next;
    }
}

// ---- rotation and append ----------------------------------------------------------------------------------------------------------------
struct AppendParams {
    RowsView rows;
    PagesView cache;
    int heads, rot, pairs, positions;
    const float *cosine, *sine, *projected;
    const int32_t* offset;
    int64_t stride;
    int query_bf16;
    void* query;
    Divider by_head;   // items of a head
};

template <int V> __device__ __forceinline__ void store_values(void* base, int bf16, int64_t at, const Lanes<V>& v) {
    if (!bf16) {
        store_lanes<V>(static_cast<float*>(base) + at, v);
    } else if constexpr (V == 4) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.v[0], v.v[1]), b = __floats2bfloat162_rn(v.v[2], v.v[3]);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(base) + at) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(v.v[0]);
    }
}

// Where the two quarters of an item lie in its head: d .. d + V - 1 and e .. e + V - 1, which turn together in the rotating part.
template <int V> __device__ __forceinline__ void item_places(const AppendParams& p, int j, int& d, int& e) {
    d = j * 2 * V;
    e = d + V;
    if (!p.pairs && d < p.rot) {
        d = j * V;
        e = d + p.rot / 2;
    }
}

// Where a row's keys and values go, and the row of the tables that turns it; -1 for none.
struct AppendPlace { int page, entry, turn; };
__device__ __forceinline__ AppendPlace append_place(const AppendParams& p, int row) {
    AppendPlace at{-1, 0, -1};
    const int s = __ldg(p.rows.sequence + row), slot = __ldg(p.rows.slot + s);
    if (slot < 0 || slot >= p.cache.sequences) return at;
    const int position = p.rows.lengths[slot] + row - __ldg(p.rows.first + s);
    const int64_t turn = static_cast<int64_t>(position) + (p.offset ? __ldg(p.offset + s) : 0);
    if (p.rot > 0 && turn >= 0 && turn < p.positions) at.turn = static_cast<int>(turn);
    if (position >= 0 && position < p.cache.capacity()) {
        at.page = page_of(p.cache, slot, position / p.cache.page_size);
        at.entry = position % p.cache.page_size;
    }
    return at;
}

// Turns an item by its row's cosines and sines.
template <int V> __device__ __forceinline__ void turn_item(const AppendParams& p, int d, const float* cosine, const float* sine, Lanes<V>& a, Lanes<V>& b) {
    if (!p.pairs) {
        const Lanes<V> c = load_lanes<V>(cosine + d), s = load_lanes<V>(sine + d);
#pragma unroll
        for (int u = 0; u < V; ++u) {
            const float x = a.v[u], y = b.v[u];
            a.v[u] = x * c.v[u] - y * s.v[u];
            b.v[u] = y * c.v[u] + x * s.v[u];
        }
    } else if constexpr (V == 4) {
        const Lanes<4> c = load_lanes<4>(cosine + d / 2), s = load_lanes<4>(sine + d / 2);
        const float x[4] = {a.v[0], a.v[2], b.v[0], b.v[2]}, y[4] = {a.v[1], a.v[3], b.v[1], b.v[3]};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            Lanes<4>& to = u < 2 ? a : b;
            to.v[(u & 1) * 2] = x[u] * c.v[u] - y[u] * s.v[u];
            to.v[(u & 1) * 2 + 1] = y[u] * c.v[u] + x[u] * s.v[u];
        }
    } else {
        const float c = cosine[d / 2], s = sine[d / 2], x = a.v[0], y = b.v[0];
        a.v[0] = x * c - y * s;
        b.v[0] = y * c + x * s;
    }
}

template <int V> __device__ __forceinline__ void store_item(void* base, int bf16, int64_t to, int d, int e, const Lanes<V>& a, const Lanes<V>& b) {
    if (V == 4 && bf16 && e == d + V) {
        const uint4 x = make_uint4(pack_bf16(a.v[0], a.v[1 % V]), pack_bf16(a.v[2 % V], a.v[3 % V]), pack_bf16(b.v[0], b.v[1 % V]), pack_bf16(b.v[2 % V], b.v[3 % V]));
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + to + d) = x;
        return;
    }
    store_values<V>(base, bf16, to + d, a);
    store_values<V>(base, bf16, to + e, b);
}

// Turns the item j of a row's head and stores it.
template <int V> __device__ __forceinline__ void finish_item(const AppendParams& p, int row, const AppendPlace& at, int head, int d, int e, bool turns, const float* cosine,
                                                             const float* sine, Lanes<V>& a, Lanes<V>& b) {
    const int kv_heads = p.cache.kv_heads;
    if (turns) turn_item<V>(p, d, cosine, sine, a, b);
    if (head < p.heads) {
        store_item<V>(p.query, p.query_bf16, (static_cast<int64_t>(row) * p.heads + head) * p.cache.head_dim, d, e, a, b);
    } else if (at.page >= 0) {
        const bool value = head >= p.heads + kv_heads;
        store_item<V>(p.cache.pool[value], p.cache.dtype == B200_BF16, page_row(p.cache, at.page, head - p.heads - (value ? kv_heads : 0), at.entry), d, e, a, b);
    }
}

// An item is 2 V values of one head of one row.  grid (rows, blocks of items): a block has one or more whole rows where there are rows for every SM, since it
// walks from the row to its page (four dependent loads); it asks for the row's values before that, and before it knows whether the row is one of a sequence.
// Bound by this chain with few rows, by memory with many: 670 MB (18 k rows of 48 heads of 128 to bf16) in 118 - 125 us, 5.4 - 5.7 TB/s.
constexpr int kItemsHeld = 4;
template <int V> __global__ void __launch_bounds__(256) rotary_append_kernel(const AppendParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int row = blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= p.rows.rows) return;
    const int dim = p.cache.head_dim, per_head = dim / (2 * V), turning = p.heads + p.cache.kv_heads;
    const int items = (p.heads + 2 * p.cache.kv_heads) * per_head, stride = gridDim.y * blockDim.x;
    const float* source = p.projected + row * p.stride;
    const int live = __ldg(p.rows.first + p.rows.sequences);
    AppendPlace at{};
    bool placed = false;
    for (int first = blockIdx.y * blockDim.x + threadIdx.x; first < items; first += kItemsHeld * stride) {
        Lanes<V> a[kItemsHeld], b[kItemsHeld];
#pragma unroll
        for (int k = 0; k < kItemsHeld; ++k) {
            const int item = first + k * stride;
            if (item >= items) break;
            const int head = divide(item, p.by_head), j = item - head * per_head;
            int d = j * 2 * V, e = d + V;
            if (head < turning) item_places<V>(p, j, d, e);   // values do not turn
            a[k] = load_lanes<V>(source + head * dim + d);
            b[k] = load_lanes<V>(source + head * dim + e);
        }
        if (!placed) {
            placed = true;
            if (row >= live) return;
            at = append_place(p, row);
        }
        const int64_t table = static_cast<int64_t>(at.turn) * (p.rot / 2);
#pragma unroll
        for (int k = 0; k < kItemsHeld; ++k) {
            const int item = first + k * stride;
            if (item >= items) break;
            const int head = divide(item, p.by_head), j = item - head * per_head;
            int d = j * 2 * V, e = d + V;
            if (head < turning) item_places<V>(p, j, d, e);
            finish_item<V>(p, row, at, head, d, e, at.turn >= 0 && head < turning && j * 2 * V < p.rot, p.cosine + table, p.sine + table, a[k], b[k]);
        }
    }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_rotary_tables(const b200_rotary_scaling* s, int32_t rot_dims, int64_t first, int64_t positions, float* cosine, float* sine, void* stream) {
    if (!s || !cosine || !sine || rot_dims <= 0 || (rot_dims & 1) || first < 0 || positions < 0 || first > (int64_t{1} << 52) || positions > (int64_t{1} << 31)
        || s->kind < B200_ROTARY_PLAIN || s->kind > B200_ROTARY_PARTS || !(s->base > 0.0) || !std::isfinite(s->base) || !std::isfinite(s->magnitude)) {
        set_error("b200_rotary_tables: bad pointer, size, kind or base");
        return B200_BAD_ARGUMENT;
    }
    if (s->kind != B200_ROTARY_PLAIN && (!(s->factor > 0.0) || !std::isfinite(s->factor))) {
        set_error("b200_rotary_tables: the factor must be positive");
        return B200_BAD_ARGUMENT;
    }
    if (s->kind == B200_ROTARY_PARTS && !(s->original > 0.0 && s->low < s->high && std::isfinite(s->original) && std::isfinite(s->low) && std::isfinite(s->high))) {
        set_error("b200_rotary_tables: scaling by parts needs original > 0 and low < high");
        return B200_BAD_ARGUMENT;
    }
    if (positions == 0) return B200_OK;
    TableParams p{};
    p.log_base = std::log(s->base);
    // two entries have one frequency, f_0 = 1, whatever the base
    if (s->kind == B200_ROTARY_BASE && rot_dims > 2) p.log_base += std::log(s->factor) * rot_dims / (rot_dims - 2);
    p.factor = s->factor; p.original = s->original; p.low = s->low; p.high = s->high;
    p.magnitude = s->magnitude == 0.0 ? 1.0 : s->magnitude;
    p.kind = s->kind; p.half = rot_dims / 2;
    p.first = first; p.positions = positions; p.cosine = cosine; p.sine = sine;
    // enough threads for every SM before the runs get longer than a few positions; 32 positions make two pairs of sines and cosines cheap
    p.run = static_cast<int>(positions * p.half / (148 * 1024));
    p.run = p.run < 2 ? 2 : p.run > 32 ? 32 : p.run;
    const int64_t threads = (positions + p.run - 1) / p.run * p.half;
    if ((threads + 255) / 256 > INT32_MAX) { set_error("b200_rotary_tables: the tables are too large"); return B200_UNSUPPORTED; }
    return cuda_status(launch_dependent(rotary_tables_kernel, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, as_stream(stream), p),
                       "rotary_tables_kernel launch");
}

extern "C" int b200_rotary_append(const b200_rotary_append_args* a, const b200_rows* pass, void* stream) {
    AppendParams p{};
    if (!rows_view(pass, p.rows)) return B200_BAD_ARGUMENT;
    if (!a) { set_error("b200_rotary_append: no arguments"); return B200_BAD_ARGUMENT; }
    if (!pages_view(a->cache, "b200_rotary_append", p.cache)) return B200_BAD_ARGUMENT;
    const int dim = a->cache.head_dim;
    const int64_t width = (static_cast<int64_t>(a->heads) + 2 * a->cache.kv_heads) * dim;
    const int64_t stride = a->stride ? a->stride : width;
    if (a->heads <= 0 || (dim & 1) || a->rot_dims < 0 || (a->rot_dims & 1) || a->rot_dims > dim || !a->projected || !a->query || stride < width
        || width > INT32_MAX || (a->query_dtype != B200_F32 && a->query_dtype != B200_BF16)
        || (a->rot_dims > 0 && (!a->cosine || !a->sine || a->positions <= 0))) {
        set_error("b200_rotary_append: bad pointer, size or dtype");
        return B200_BAD_ARGUMENT;
    }
    p.heads = a->heads; p.rot = a->rot_dims; p.pairs = a->rotate_pairs != 0; p.positions = a->positions;
    p.cosine = a->cosine; p.sine = a->sine; p.projected = a->projected; p.offset = a->offset; p.stride = stride;
    p.query_bf16 = a->query_dtype == B200_BF16; p.query = a->query;
    // four values per access where every address allows it
    uintptr_t bits = reinterpret_cast<uintptr_t>(a->projected) | reinterpret_cast<uintptr_t>(a->query) | reinterpret_cast<uintptr_t>(a->cache.key)
                     | reinterpret_cast<uintptr_t>(a->cache.value);
    if (a->rot_dims) bits |= reinterpret_cast<uintptr_t>(a->cosine) | reinterpret_cast<uintptr_t>(a->sine);
    const bool wide = dim % 8 == 0 && a->rot_dims % 8 == 0 && stride % 4 == 0 && bits % 16 == 0;
    p.by_head = divider(dim / (wide ? 8 : 2));
    const int64_t items = width / (wide ? 8 : 2);
    // Many rows: four items per thread and no thread without, so that as many rows as there is room for have their values on the way.  18 k rows of 48 heads
    // of 128 (of 64, 10 heads of 128): 119 us (64, 31), with 256 threads for every 256 items of a row 197 (109, 52).  Short rows share blocks of up to 128 threads:
    // with rows of 3 heads of 64 11 us, with a block each 20.
    int64_t threads = 256, blocks = (items + 255) / 256, rows = 1;
    if (p.rows.rows >= 148) {
        threads = std::clamp<int64_t>((items + 32 * kItemsHeld - 1) / (32 * kItemsHeld) * 32, 32, 256);
        if (p.rows.rows >= 8 * 148) rows = std::max<int64_t>(1, 128 / threads);
        blocks = 1;
    }
    const dim3 grid(static_cast<unsigned>((p.rows.rows + rows - 1) / rows), static_cast<unsigned>(blocks < 65535 ? blocks : 65535));
    const dim3 block(static_cast<unsigned>(threads), static_cast<unsigned>(rows));
    return cuda_status(wide ? launch_dependent(rotary_append_kernel<4>, grid, block, 0, as_stream(stream), p)
                            : launch_dependent(rotary_append_kernel<1>, grid, block, 0, as_stream(stream), p),
                       "rotary_append_kernel launch");
}
