// Grouped-query attention of packed sequences over a prefix that groups of them share and over their own tokens (b200_prefix_attention).
//
// With G = heads / kv_heads, the rows of a group times the G heads of one KV head are the M side of the products with the prefix: every key and
// value of the prefix enters an SM once per tile of rows instead of once per sequence.  A sequence's own tokens are the same work with the rows
// of that sequence.  Items are (prefix tile or sequence tile, KV head, split of the keys); each leaves an unnormalised partial result (maximum,
// sum, accumulator) per row and head, and the merge kernel joins them under one softmax:
//   m = max m_i,  out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i      (scores in units of log2 e).
// Where the prefixes are short, an item is joined: the rows of a sequence tile with the prefix's keys and then the sequence's own, and it leaves the result.
#include "mma.cuh"
#include "prefix.cuh"
#include "prefix_tensor.cuh"

#include <algorithm>
#include <cmath>

namespace b200 {
namespace {

// ---- any type and head size: f32 products on the CUDA cores --------------------------------------------------------------------------------
constexpr int kPlainKeys = 32, kPlainThreads = 128;

__host__ __device__ constexpr int plain_width(int dim) { return (dim + 3) / 4 * 4; }
// Rows four floats longer than a multiple of 32 at most: neighbouring rows begin in other banks.
__host__ __device__ constexpr int plain_smem(int dim, int rows) {
    return ((rows + 2 * kPlainKeys) * (plain_width(dim) + 4) + rows * (kPlainKeys + 1)) * static_cast<int>(sizeof(float));
}

template <class T> __device__ __forceinline__ float4 load_four(const T* p);
template <> __device__ __forceinline__ float4 load_four(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <> __device__ __forceinline__ float4 load_four(const __nv_bfloat16* p) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    return make_float4(bf16_lo(x.x), bf16_hi(x.x), bf16_lo(x.y), bf16_hi(x.y));
}
// Values d .. d + 3 of a row, zeros past its end.  `whole`: head sizes of 4 n in aligned pools.
template <class T> __device__ __forceinline__ float4 load_piece(const T* row, int d, int dim, bool whole) {
    if (whole) return d < dim ? load_four<T>(row + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return make_float4(d < dim ? load_as_f32(row, d) : 0.0f, d + 1 < dim ? load_as_f32(row, d + 1) : 0.0f, d + 2 < dim ? load_as_f32(row, d + 2) : 0.0f,
                       d + 3 < dim ? load_as_f32(row, d + 3) : 0.0f);
}

// A tile of 16 ROWS pairs x 32 keys: thread (ty, tx) has the scores of rows ROWS ty .. + ROWS - 1 with the keys tx + 8 j, and the columns 4 tx + 32 c of their
// accumulators; it brings the same columns of the keys ty and ty + 16, up to 128 wide a step ahead.  Bound by the chain of a step (shared memory, f32
// products) with few CTAs, which the splits are for.
template <class T, int BLOCKS, int ROWS> __global__ void __launch_bounds__(kPlainThreads, BLOCKS == 2 ? 4 : BLOCKS == 4 ? 3 : 2) prefix_plain_kernel(const PrefixParams p, const bool whole) {
    extern __shared__ __align__(16) float plain_shared[];
    begin_items(p);
    const Item it = find_item(p, first_item(p) + blockIdx.x);
    if (!it.live) return end_items(p);
    const int width = plain_width(p.dim), pitch = width + 4;
    float* query = plain_shared;
    constexpr int kRows = 16 * ROWS;
    float* key = query + kRows * pitch;
    float* value = key + kPlainKeys * pitch;
    float* weight = value + kPlainKeys * pitch;
    const int thread = threadIdx.x, ty = thread / 8, tx = thread % 8;
    const PagesView& view = it.causal ? p.own : p.prefix;
    constexpr bool kAhead = BLOCKS <= 4;
    float4 next[2][2][BLOCKS];   // [key or value][row][columns]
    auto fetch = [&](int begin) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int position = begin + ty + 16 * r;
            int page = -1;
            if (position < it.keys.end) page = page_of(view, it.slot, position / view.page_size);
            const int64_t at = page >= 0 ? page_row(view, page, it.kv_head, position % view.page_size) : 0;
#pragma unroll
            for (int which = 0; which < 2; ++which)
#pragma unroll
                for (int c = 0; c < BLOCKS; ++c)
                    next[which][r][c] = page >= 0 ? load_piece(static_cast<const T*>(view.pool[which]) + at, 32 * c + 4 * tx, p.dim, whole) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    };
    if (kAhead) fetch(it.keys.begin);
    for (int i = thread; i < kRows * (width / 4); i += kPlainThreads) {
        const int r = i / (width / 4), m = it.m_begin + r, d = i % (width / 4) * 4;
        *reinterpret_cast<float4*>(query + r * pitch + d) =
            m < it.m_count ? load_piece(static_cast<const T*>(p.query) + pair_row(p, it, m) * p.dim, d, p.dim, whole) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float most[ROWS], sum[ROWS] = {}, acc[ROWS][BLOCKS][4] = {};
    int limit[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        most[r] = -INFINITY;
        limit[r] = it.causal ? min(it.keys.end, it.visible + divide(it.m_begin + ROWS * ty + r, p.by_group)) : it.keys.end;
    }
    for (int begin = it.keys.begin; begin < it.keys.end; begin += kPlainKeys) {
        __syncthreads();
        if (!kAhead) fetch(begin);
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < BLOCKS; ++c)
                if (32 * c + 4 * tx < width) {
                    *reinterpret_cast<float4*>(key + (ty + 16 * r) * pitch + 32 * c + 4 * tx) = next[0][r][c];
                    *reinterpret_cast<float4*>(value + (ty + 16 * r) * pitch + 32 * c + 4 * tx) = next[1][r][c];
                }
        if (kAhead && begin + kPlainKeys < it.keys.end) fetch(begin + kPlainKeys);
        __syncthreads();
        float score[ROWS][4] = {};
#pragma unroll 4
        for (int d = 0; d < width; d += 4) {
            float4 a[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) a[r] = *reinterpret_cast<const float4*>(query + (ROWS * ty + r) * pitch + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 k = *reinterpret_cast<const float4*>(key + (tx + 8 * j) * pitch + d);
#pragma unroll
                for (int r = 0; r < ROWS; ++r) score[r][j] += a[r].x * k.x + a[r].y * k.y + a[r].z * k.z + a[r].w * k.w;
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float top = most[r];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                score[r][j] = begin + tx + 8 * j < limit[r] ? score[r][j] * p.scale : -INFINITY;
                top = fmaxf(top, score[r][j]);
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float base = top == -INFINITY ? 0.0f : top, shrink = exp2f(most[r] - base);
            float here = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w = exp2f(score[r][j] - base);
                here += w;
                weight[(ROWS * ty + r) * (kPlainKeys + 1) + tx + 8 * j] = w;
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) here += __shfl_xor_sync(0xffffffffu, here, o);
            sum[r] = sum[r] * shrink + here;
            most[r] = top;
#pragma unroll
            for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[r][c][u] *= shrink;
        }
        __syncwarp();   // the weights of a row are written and read by the same eight lanes
        // A row sees no more than the next one; what a row does not see is not multiplied, since it may be no number.
        auto add_values = [&](int keys, auto&& sees) {
#pragma unroll 4
            for (int k = 0; k < keys; ++k) {
                float w[ROWS];
#pragma unroll
                for (int r = 0; r < ROWS; ++r) w[r] = weight[(ROWS * ty + r) * (kPlainKeys + 1) + k];
#pragma unroll
                for (int c = 0; c < BLOCKS; ++c) {
                    if (32 * c + 4 * tx >= width) continue;
                    const float4 v = *reinterpret_cast<const float4*>(value + k * pitch + 32 * c + 4 * tx);
#pragma unroll
                    for (int r = 0; r < ROWS; ++r)
                        if (sees(r, k)) { acc[r][c][0] += w[r] * v.x; acc[r][c][1] += w[r] * v.y; acc[r][c][2] += w[r] * v.z; acc[r][c][3] += w[r] * v.w; }
                }
            }
        };
        if (limit[0] >= begin + kPlainKeys) add_values(kPlainKeys, [](int, int) { return true; });
        else add_values(min(kPlainKeys, limit[ROWS - 1] - begin), [&](int r, int k) { return begin + k < limit[r]; });
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int m = it.m_begin + ROWS * ty + r;
        if (m >= it.m_count) continue;
        const int64_t at = partial_row(p, it, m);
        if (tx == 0) {
            p.part_ml[2 * at] = most[r];
            p.part_ml[2 * at + 1] = sum[r];
        }
#pragma unroll
        for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (32 * c + 4 * tx + u < p.dim) p.part_o[at * p.dim + 32 * c + 4 * tx + u] = acc[r][c][u];
    }
    end_items(p);
}

// ---- bf16, heads of 8 n <= 128 values: mma.sync ---------------------------------------------------------------------------------------------
constexpr int kMmaWarps = 4, kMmaThreads = (kMmaWarps + 1) * 32;   // four warps of products, one that copies

template <int HD> struct MmaShape {                              // HD: the head size rounded up to 64, 96 or 128
    static constexpr int blocks = HD <= 64 ? 1 : 2;              // of 64 values: rows of 128 bytes as TMA's swizzle lays them out
    static constexpr int block_bytes = kUnit * 128;
    static constexpr int tile_bytes = blocks * block_bytes;      // K or V of one step
    // What two CTAs per SM leave room for beside the area where warps' results are joined.
    static constexpr int stages(int parts) { return blocks == 1 ? 4 : parts > 1 ? 2 : 3; }
    static constexpr int join_bytes(int parts) { return parts > 1 ? 64 * (HD + 4) * 4 + 64 * 2 * 4 : 0; }
    static constexpr int smem_bytes(int parts) { return stages(parts) * 2 * tile_bytes + join_bytes(parts) + 1024 + 512; }   // slack of the 1024-byte alignment, control words
};
// Byte offset of 16-byte piece c of row r.
__device__ __forceinline__ uint32_t piece_offset(int r, int c) { return static_cast<uint32_t>((c >> 3) * kUnit * 128 + r * 128 + (((c ^ r) & 7) << 4)); }
__device__ __forceinline__ void mma_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kMmaWarps * 32) : "memory"); }
__device__ __forceinline__ bool mma_any(bool mine) {
    uint32_t any;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
                 : "=r"(any) : "r"(static_cast<uint32_t>(mine)), "n"(kMmaWarps * 32) : "memory");
    return any != 0;
}

// Between this thread's own stores to a stage and the copy that refills it.
__device__ __forceinline__ void own_writes_done() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Steps with keys that some pairs of the tile do not see: a weight of 0 does not cancel a value that is no number, so such values leave the tile
// before the products, and are added to the accumulators of the pairs that do see them.
template <int HD> __device__ __forceinline__ void guard_values(unsigned char* value, int pieces, int begin, int warp_key, int keys, const int (&seen)[2],
                                                               float (&acc)[HD / 8][4]) {
    constexpr int kThreads = kMmaWarps * 32;
    bool odd = false;
    for (int i = threadIdx.x; i < kUnit * pieces; i += kThreads) {
        const uint4 x = *reinterpret_cast<const uint4*>(value + piece_offset(i / pieces, i % pieces));
        const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) odd |= (words[u] & 0x7f80u) == 0x7f80u || (words[u] & 0x7f800000u) == 0x7f800000u;
    }
    if (!mma_any(odd)) return;
    const int quad = threadIdx.x & 3;
    for (int k = warp_key; k < warp_key + keys; ++k)
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
            if (n >= pieces) continue;
            const uint32_t two = *reinterpret_cast<const uint32_t*>(value + piece_offset(k, n) + 4 * quad);
            const float v[2] = {bf16_lo(two), bf16_hi(two)};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!isfinite(v[e & 1]) && begin + k < seen[e >> 1]) acc[n][e] += v[e & 1];
        }
    mma_barrier();
    for (int i = threadIdx.x; i < kUnit * pieces * 8; i += kThreads) {
        uint16_t* x = reinterpret_cast<uint16_t*>(value + piece_offset(i / (pieces * 8), i / 8 % pieces)) + i % 8;
        if ((*x & 0x7f80) == 0x7f80) *x = 0;
    }
    own_writes_done();
    mma_barrier();
}

struct MmaMaps { CUtensorMap own[2], prefix[2]; };   // K and V

// A tile has 64 / PARTS pairs, 16 per warp: PARTS warps share the 64 keys of a step, and their results are joined at the end.  Tiles of 16 pairs (PARTS 4) for
// single tokens, of 64 where there are as many pairs, so that no warp multiplies rows that are not there.  A CTA takes item after item; the copying warp finds
// them and runs ahead of the products, so that keys of the next item are on their way while the last one's results are written.
template <int HD, int PARTS, bool JOINED, bool PLANES> __global__ void __launch_bounds__(kMmaThreads, 2) prefix_mma_kernel(const __grid_constant__ MmaMaps maps, const PrefixParams p, const int box_rows) {
    using S = MmaShape<HD>;
    extern __shared__ unsigned char mma_shared[];
    constexpr int kStages = S::stages(PARTS);
    constexpr int kKeys = 64 / PARTS, kRowGroups = 4 / PARTS;   // keys per warp and step
    constexpr int kTiles = kKeys / 8, kSteps = HD / 16, kColumns = HD / 8;
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(mma_shared) + 1023) & ~static_cast<uintptr_t>(1023));
    float* joined = reinterpret_cast<float*>(ring + kStages * 2 * S::tile_bytes);
    uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(joined) + S::join_bytes(PARTS));
    uint64_t* empty = full + kStages;
    uint64_t* item_full = empty + kStages;   // [2] items found ahead
    uint64_t* item_empty = item_full + 2;
    Item* item_of = reinterpret_cast<Item*>(item_empty + 2);
    volatile int* alive = reinterpret_cast<volatile int*>(item_of + 2);
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    if (thread == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kMmaWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&item_full[i], 1);
            mbar_init(&item_empty[i], kMmaWarps);
        }
        *alive = 1;
        mbar_fence_init();
    }
    __syncthreads();
    begin_items(p);
    // after a wait that ran out every role goes through the rest of its item without waiting, and leaves
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (*alive && !mbar_wait(bar, parity)) {
            atomicExch(p.status, B200_DEVICE_TIMEOUT);
            *alive = 0;
        }
    };
    if (warp == kMmaWarps) {
        const int across = boxes_per_row(box_rows, p.dim), boxes = kUnit / box_rows * across;   // at most 16 per tensor
        const int which = lane / boxes, block = lane % across, row = lane % boxes / across * box_rows;
        int issued = 0, found = 0;
        const int shared_items = p.beside ? 0 : prefix_items(p), stride = static_cast<int>(gridDim.x);
        int index = blockIdx.x, batch = 0;   // own items are found 32 at a time, one per lane, from `batch` on
        unsigned waiting = 0;                // those of the batch that have work and are still to come
        Item mine{};
        while (true) {
            Item it{};
            bool any = false;
            for (; index < shared_items && !any; index += stride) {
                it = find_prefix_item(p, index);
                any = it.live;
            }
            while (!any) {
                if (!waiting) {
                    const int64_t at = index + static_cast<int64_t>(batch + lane) * stride;
                    if (index + static_cast<int64_t>(batch) * stride >= p.items) break;
                    mine.live = false;
                    if (at < p.items) mine = find_own_item(p, static_cast<int>(at) - shared_items);
                    waiting = __ballot_sync(0xffffffffu, mine.live);
                    batch += 32;
                    continue;
                }
                it = item_of_lane(mine, __ffs(waiting) - 1);
                waiting &= waiting - 1;
                any = true;
            }
            if (!any) it.m_count = -1;   // no more
            wait(&item_empty[found & 1], ((found >> 1) & 1) ^ 1);
            if (lane == 0) {
                item_of[found & 1] = it;
                mbar_arrive(&item_full[found & 1]);
            }
            ++found;
            if (!any || !__all_sync(0xffffffffu, *alive != 0)) break;
            // the prefix of a joined item, then the item's own span
            const int shared_steps = JOINED ? (it.shared + kUnit - 1) / kUnit : 0, end = issued + shared_steps + (it.keys.end - it.keys.begin + kUnit - 1) / kUnit;
            for (int span = shared_steps ? 0 : 1; span < 2; ++span) {
                const PagesView& view = span && it.causal ? p.own : p.prefix;
                const int outside = static_cast<int>(view.pages) * view.kv_heads * view.page_size;   // a row past the pools: zeros
                const CUtensorMap* map = span && it.causal ? &maps.own[which & 1] : &maps.prefix[which & 1];
                const int until = span ? end : issued + shared_steps, last_key = span ? it.keys.end : it.shared;
                if (issued >= until) break;
                PageStream pages(view, span ? it.slot : it.shared_slot, (span ? it.keys.begin : 0) + row, kUnit, which < 2 ? last_key : 0);
                for (; issued < until; ++issued) {
                    const int stage = issued % kStages, y = pages.next(it.kv_head, outside);
                    wait(&empty[stage], ((issued / kStages) & 1) ^ 1);
                    if (!__all_sync(0xffffffffu, *alive != 0)) break;
                    if (lane == 0) mbar_expect_tx(&full[stage], 2 * S::tile_bytes);
                    __syncwarp();
                    unsigned char* to = ring + (stage * 2 + which) * S::tile_bytes;
                    if (which < 2) {
                        if (across < S::blocks) tma_load_3d(to, map, 0, y, 0, &full[stage]);
                        else tma_load_2d(to + block * S::block_bytes + row * 128, map, block * 64, y, &full[stage]);
                    }
                }
                if (issued < until) break;
            }
            if (issued < end) break;
        }
        if (!*alive)   // no copy is in flight when the CTA leaves
            for (int j = max(0, issued - kStages); j < issued; ++j) mbar_wait(&full[j % kStages], (j / kStages) & 1);
        return end_items(p);
    }
    int taken = 0;   // steps of the items before
    for (int number = 0;; ++number) {
        wait(&item_full[number & 1], (number >> 1) & 1);
        const Item it = item_of[number & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[number & 1]);
        if (mma_any(!*alive) || it.m_count < 0) return end_items(p);
        const int shared_steps = JOINED ? (it.shared + kUnit - 1) / kUnit : 0, steps = shared_steps + (it.keys.end - it.keys.begin + kUnit - 1) / kUnit;
        // query fragments
        const int quad = lane & 3, row_group = warp % kRowGroups, m0 = it.m_begin + row_group * 16 + (lane >> 2);
        uint32_t q[kSteps][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int m = m0 + 8 * r;
            const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(p.query) + pair_row(p, it, m) * p.dim;
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = 16 * k + 8 * h + 2 * quad;
                    q[k][2 * h + r] = m < it.m_count && d < p.dim ? __ldg(reinterpret_cast<const uint32_t*>(row + d)) : 0u;
                }
        }
        int own_seen[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) own_seen[r] = it.causal ? min(it.keys.end, it.visible + divide(m0 + 8 * r, p.by_group)) : it.keys.end;
        float acc[kColumns][4] = {}, most[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
        const int warp_key = warp / kRowGroups * kKeys;
        const int first_limit = it.causal ? it.visible + divide(it.m_begin, p.by_group) : it.keys.end;   // keys that the tile's first pair sees
        for (int step = 0; step < steps; ++step) {
            const bool shared = JOINED && step < shared_steps;   // everyone sees these
            const int stage = (taken + step) % kStages, begin = shared ? step * kUnit : it.keys.begin + (step - shared_steps) * kUnit, end = shared ? it.shared : it.keys.end;
            const int seen[2] = {shared ? end : own_seen[0], shared ? end : own_seen[1]};
            wait(&full[stage], ((taken + step) / kStages) & 1);
            unsigned char* values = ring + (stage * 2 + 1) * S::tile_bytes;
            const uint32_t key = smem_u32(ring) + stage * 2 * S::tile_bytes, value = key + S::tile_bytes;
            if (begin + kUnit > end && end % box_rows) {
                // rows of the last box behind the keys may hold anything
                const int from = end - begin, behind = (from + box_rows - 1) / box_rows * box_rows - from;
                for (int i = thread; i < behind * 8 * S::blocks; i += kMmaWarps * 32)
                    *reinterpret_cast<uint4*>(values + i / (behind * 8) * S::block_bytes + from * 128 + i % (behind * 8) * 16) = make_uint4(0, 0, 0, 0);
                own_writes_done();
                mma_barrier();
            }
            float score[kTiles][4] = {};
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int n = 0; n < kTiles; n += 2) {
                    uint32_t b[4];   // keys n*8 .. +7 and +8 .. +15, both halves of the 16 values
                    ldsm_x4(b, key + piece_offset(warp_key + n * 8 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                    mma_16816(score[n], q[k], b[0], b[1]);
                    mma_16816(score[n + 1], q[k], b[2], b[3]);
                }
            const int first_key = begin + warp_key + 2 * quad;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float top = most[r];
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float& x = score[n][2 * r + u];
                        x = first_key + n * 8 + u < seen[r] ? x * p.scale : -INFINITY;
                        top = fmaxf(top, x);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float base = whole_maximum(top), shrink = exp2_fast(most[r] - base);
                float here = 0.0f;
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                    float &a = score[n][2 * r], &b = score[n][2 * r + 1];
                    a = exp2_fast(a - base);
                    b = exp2_fast(b - base);
                    if constexpr (!PLANES) {
                        const uint32_t rounded = pack_bf16(a, b);
                        a = bf16_lo(rounded);
                        b = bf16_hi(rounded);
                    }
                    here += a + b;
                }
                sum[r] = sum[r] * shrink + here;   // of this lane's keys; the quad's are added at the end
                if (top != -INFINITY) most[r] = base;
#pragma unroll
                for (int n = 0; n < kColumns; ++n) {
                    acc[n][2 * r] *= shrink;
                    acc[n][2 * r + 1] *= shrink;
                }
            }
            if (!shared && min(end, begin + kUnit) > first_limit) guard_values<HD>(values, p.dim / 8, begin, warp_key, kKeys, seen, acc);
#pragma unroll
            for (int k = 0; k < kKeys / 16; ++k) {
                uint32_t weights[2][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = score[2 * k + i / 2][2 * (i % 2)], b = score[2 * k + i / 2][2 * (i % 2) + 1];
                    weights[0][i] = first_plane(a, b);
                    if constexpr (PLANES) weights[1][i] = second_plane(a, b);
                }
#pragma unroll
                for (int n = 0; n < kColumns; n += 2) {
                    uint32_t b[4];
                    ldsm_x4_trans(b, value + piece_offset(warp_key + 16 * k + (lane & 15), n + (lane >> 4)));
#pragma unroll
                    for (int plane = 0; plane < 1 + PLANES; ++plane) {
                        mma_16816(acc[n], weights[plane], b[0], b[1]);
                        mma_16816(acc[n + 1], weights[plane], b[2], b[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
        }
        if constexpr (PARTS > 1) {
            // join the warps: [part][rows][HD] accumulators behind [part][rows][2] maxima and sums
            constexpr int kRows = 64 / PARTS, kPitch = HD + 4;
            float* rows_of = joined + 64 * 2;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int at = warp / kRowGroups * kRows + row_group * 16 + (lane >> 2) + 8 * r;
                if (quad == 0) {
                    joined[at * 2] = most[r];
                    joined[at * 2 + 1] = sum[r];
                }
#pragma unroll
                for (int n = 0; n < kColumns; ++n) *reinterpret_cast<float2*>(rows_of + at * kPitch + 8 * n + 2 * quad) = make_float2(acc[n][2 * r], acc[n][2 * r + 1]);
            }
            mma_barrier();
            const int live = min(kRows, it.m_count - it.m_begin);
            for (int i = thread; i < live * (HD / 4); i += kMmaWarps * 32) {
                const int m = i / (HD / 4), d = i % (HD / 4) * 4;
                float top = -INFINITY, total = 0.0f;
#pragma unroll
                for (int w = 0; w < PARTS; ++w) top = fmaxf(top, joined[(w * kRows + m) * 2]);
                const float base = top == -INFINITY ? 0.0f : top;
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < PARTS; ++w) {
                    const float f = exp2_fast(joined[(w * kRows + m) * 2] - base);
                    const float4 v = *reinterpret_cast<const float4*>(rows_of + (w * kRows + m) * kPitch + d);
                    total += f * joined[(w * kRows + m) * 2 + 1];
                    o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
                }
                if constexpr (JOINED) {
                    const float inverse = total == 0.0f ? 0.0f : 1.0f / total, v[4] = {o.x * inverse, o.y * inverse, o.z * inverse, o.w * inverse};
                    if (d < p.dim) store_results<4>(p, result_at(p, it, it.m_begin + m) + d, v);
                } else {
                    const int64_t to = partial_row(p, it, it.m_begin + m);
                    if (d == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * to) = make_float2(top, total);
                    if (d < p.dim) *reinterpret_cast<float4*>(p.part_o + to * p.dim + d) = o;
                }
            }
            mma_barrier();   // the next item's results may be written
        } else {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int m = m0 + 8 * r;
                if (m >= it.m_count) continue;
                if constexpr (JOINED) {
                    const float inverse = sum[r] == 0.0f ? 0.0f : 1.0f / sum[r];
                    const int64_t to = result_at(p, it, m);
#pragma unroll
                    for (int n = 0; n < kColumns; ++n) {
                        const float v[2] = {acc[n][2 * r] * inverse, acc[n][2 * r + 1] * inverse};
                        if (8 * n < p.dim) store_results<2>(p, to + 8 * n + 2 * quad, v);
                    }
                } else {
                    const int64_t to = partial_row(p, it, m);
                    if (quad == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * to) = make_float2(most[r], sum[r]);
#pragma unroll
                    for (int n = 0; n < kColumns; ++n)
                        if (8 * n < p.dim) *reinterpret_cast<float2*>(p.part_o + to * p.dim + 8 * n + 2 * quad) = make_float2(acc[n][2 * r], acc[n][2 * r + 1]);
                }
            }
        }
        taken += steps;
    }
}

// ---- merge ------------------------------------------------------------------------------------------------------------------------------
constexpr int kMergeWarps = 4, kMostSplits = 64;

// A warp per row and head, or, SPREAD, a block: with many splits of few rows its warps share the partial results (57 splits of 6 rows and heads: 11 us, 24 with a warp each).
// V = 4 (head sizes of 4 n): a group of `lanes` lanes reads one partial result at 16 bytes per lane, the warp's groups take
// turns over the splits and are added at the end.
// The pass's arrays were complete before the kernels that left the partial results began, so what is to be read is worked out while those still run.
template <int V, bool SPREAD> __global__ void __launch_bounds__(kMergeWarps * 32) prefix_merge_kernel(const PrefixParams p) {
    __shared__ Lanes<V> shares[SPREAD ? kMergeWarps : 1][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t index = SPREAD ? blockIdx.x : blockIdx.x * static_cast<int64_t>(kMergeWarps) + warp;
    const int64_t row_of = p.row_begin + index / p.heads;
    const int row = static_cast<int>(min(row_of, static_cast<int64_t>(p.row_end)));
    if (row >= p.row_end || row >= __ldg(p.rows.first + p.rows.sequences)) {
        grid_dependency_wait();
        return;
    }
    const int s = __ldg(p.rows.sequence + row);
    const int slot = __ldg(p.rows.slot + s), first = __ldg(p.rows.first + s), count = __ldg(p.rows.first + s + 1) - first;
    int g = -1;
    for (int base = 0; base < p.groups; base += 32) {
        const int c = base + lane;
        const unsigned found = __ballot_sync(0xffffffffu, c < p.groups && __ldg(p.group_first + c) <= s && s < __ldg(p.group_first + c + 1));
        if (found) {
            g = base + __ffs(found) - 1;
            break;
        }
    }
    const int shared = g < 0 ? 0 : prefix_keys(p, __ldg(p.group_prefix + g)), own = own_keys(p, slot, count);
    const int from_prefix = used_splits(shared, p.prefix_splits, shared);
    const int parts = from_prefix + (own > 0 ? used_splits(own, p.own_splits, p.rows.lengths[slot] + row - first + 1) : 0);
    const int64_t base = index * (p.prefix_splits + p.own_splits);
    const int skip = p.prefix_splits - from_prefix;
    grid_dependency_wait();
    grid_launch_dependents();
    constexpr int kHeld = 2 * kMostSplits / 32;
    float most[kHeld], weight[kHeld], top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int i = 32 * j + lane;
        const float2 ml = i < parts ? *reinterpret_cast<const float2*>(p.part_ml + 2 * (base + i + (i < from_prefix ? 0 : skip))) : make_float2(-INFINITY, 0.0f);
        most[j] = ml.x;
        weight[j] = ml.y;
        top = fmaxf(top, ml.x);
    }
    top = warp_max(top);
    const float zero = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const float f = exp2f(most[j] - zero);
        total += f * weight[j];
        weight[j] = f;
    }
    total = warp_sum(total);
    // a row that sees nothing gives zeros; one whose weights are no numbers gives no numbers
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    const int pieces = p.dim / V;
    const int lanes = pieces >= 32 ? 32 : pieces > 16 ? 32 : pieces > 8 ? 16 : 8, groups = 32 / lanes, turn = lane / lanes;
    const int64_t to = row * p.out_stride + index % p.heads * p.dim;
    for (int d = lane % lanes; d - lane % lanes < pieces; d += lanes) {
        Lanes<V> o{};
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            if constexpr (SPREAD) {
                for (int begin = 0; begin < 32; begin += 4 * groups) {   // partial results that are requested together
                    if (32 * j + begin >= parts) break;
                    if ((32 * j + begin) / (4 * groups) % kMergeWarps != warp) continue;
                    Lanes<V> v[4];
                    float f[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int i = begin + k * groups + turn, part = 32 * j + i;
                        f[k] = __shfl_sync(0xffffffffu, weight[j], i & 31);
                        if (i >= 32 || part >= parts || d >= pieces) f[k] = 0.0f;
                        v[k] = Lanes<V>{};
                        if (f[k] != 0.0f) v[k] = load_lanes<V>(p.part_o + (base + part + (part < from_prefix ? 0 : skip)) * p.dim + d * V);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int u = 0; u < V; ++u) o.v[u] += f[k] * v[k].v[u];
                }
            } else {
#pragma unroll 8
                for (int i = 0; i < 32; i += groups) {
                    if (32 * j + i >= parts) break;
                    const int part = 32 * j + i + turn;
                    const float f = __shfl_sync(0xffffffffu, weight[j], i + turn);
                    if (part < parts && d < pieces && f != 0.0f) {
                        const Lanes<V> v = load_lanes<V>(p.part_o + (base + part + (part < from_prefix ? 0 : skip)) * p.dim + d * V);
#pragma unroll
                        for (int u = 0; u < V; ++u) o.v[u] += f * v.v[u];
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < V; ++u)
            for (int x = lanes; x < 32; x *= 2) o.v[u] += __shfl_xor_sync(0xffffffffu, o.v[u], x);
        if constexpr (SPREAD) {
            __syncthreads();
            shares[warp][lane] = o;
            __syncthreads();
            if (warp) continue;
            for (int w = 1; w < kMergeWarps; ++w)
#pragma unroll
                for (int u = 0; u < V; ++u) o.v[u] += shares[w][lane].v[u];
        }
#pragma unroll
        for (int u = 0; u < V; ++u) {
            if (turn == 0 && d < pieces) store_forms(o.v[u] * inverse, to + d * V + u, p.out, p.out_hi, p.out_lo);
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------
constexpr int kMostDim = 256;

enum class Form { plain, mma };
struct Plan {
    Form form;
    int rows;                  // rows per launch
    bool aligned;              // 16-byte addresses, head sizes of 4 n
    bool tensor;               // the prefix's items are the tcgen05 kernel's
    bool joined;               // one item per tile of own rows goes over prefix and own tokens: no partial results
    int prefix_rows, own_rows, prefix_tiles, own_tiles, prefix_splits, own_splits;
    int own_ctas;              // beside the tcgen05 kernel, 0: as many as there are items for
};

bool mma_takes(const b200_kv_pages& pages) {
    return pages.head_dim % 8 == 0 && pages.head_dim <= 128 && pages.page_size % 8 == 0 && pages.pages * pages.kv_heads * pages.page_size < INT32_MAX;
}

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int kSms = 148;   // of a B200: plans are made from sizes alone, without asking a device, and so are the launches

// us that a step of prefix_mma_kernel takes an SM, measured, and a CTA that has an SM to itself.
double step_time(int rows, int dim) { return rows == 16 ? (dim > 64 ? 0.6 : 0.4) : rows == 32 ? (dim > 64 ? 1.0 : 0.65) : dim > 64 ? 1.7 : 0.9; }

// How the tcgen05 kernel and the own tokens' kernel share the SMs.  A CTA of the first has an SM to itself; the other's CTAs run on the SMs that its last wave
// leaves: few splits of the prefix leave more of them and fewer partial results, many shorten the prefix's own time.  Measured, in us: a CTA of the prefix takes
// 10 and 0.75 (heads of 64: 0.6) per step; partial results go out and back at 5 MB per us.
struct Share { int splits, own_ctas; double time; };   // own_ctas: 0: as many as there are items for
Share share_sms(int64_t items, int max_prefix, int most_splits, int dim, int own_rows, double own_steps, double part_bytes) {
    const int steps = ceil_div(max_prefix, kTensorKeys);
    const double step = dim > 64 ? 0.75 : 0.6;
    const double own = own_steps * step_time(own_rows, dim);
    Share best{1, 0, 1e30};
    for (int n = 1; n <= most_splits && n <= steps; ++n) {
        const int64_t ctas = items * n, waves = ceil_div64(ctas, kSms);
        const double wave = 10.0 + step * ceil_div(steps, n);
        const double rest = static_cast<double>(waves * kSms - ctas), prefix = static_cast<double>(waves) * wave;
        const double free_only = rest > 0 ? std::max(prefix, prefix - wave + own / rest) : 1e30, all = prefix + std::max(0.0, own - rest * wave) / kSms;
        const double time = std::min(free_only, all) + n * part_bytes / 5e6;
        if (time < best.time) best = {n, free_only <= all ? static_cast<int>(2 * rest) : 0, time};
    }
    return best;
}

// Partial results (a maximum, a sum and an accumulator of head_dim values for a row, head and split) that a call may leave, by sizes alone of which smaller ones
// never need more: a program that asks with its largest pass and bounds has enough for all others.  Up to 64 splits each of prefix and own tokens, as many as they
// have steps, in 2^16 partial results; four splits together in up to 2^19 (273 MB
// with heads of 128), in which the parts of longer passes are run one after the other.
constexpr int64_t kManySplits = 1 << 16, kMostPartial = 1 << 19;
int64_t partial_results(const b200_prefix_args& a, int64_t rows, int max_length, int max_prefix) {
    const int64_t pairs = rows * a.heads;
    const int prefix = a.groups > 0 ? std::min(ceil_div(max_prefix, kUnit), kMostSplits) : 0;
    const int64_t splits = prefix + std::min(ceil_div(max_length, kUnit), kMostSplits);
    return std::max(std::min(pairs * splits, kManySplits), std::min<int64_t>(pairs * std::min<int64_t>(splits, 4), std::max<int64_t>(kMostPartial, 2 * a.heads)));
}
// Rows whose partial results, one of the prefix and one of the own tokens, find room, in whole waves of the tcgen05 kernel's tiles.
int64_t rows_per_launch(const b200_prefix_args& a) {
    const int64_t most = std::max<int64_t>(1, kMostPartial / 2 / a.heads), kv_heads = a.cache.kv_heads, group = a.heads / kv_heads;
    const int64_t waves = most * group / kTensorRows * kv_heads / kSms, tiles = waves * kSms / kv_heads;
    return tiles > 0 ? tiles * kTensorRows / group : most;
}

Plan make_plan(const b200_prefix_args& a, const b200_rows& whole, int max_length, int max_prefix, bool may_join = true) {
    Plan plan{};
    b200_rows pass = whole;
    if (!may_join && pass.rows > rows_per_launch(a)) {   // a joined pass leaves no partial results
        pass.rows = rows_per_launch(a);
        pass.sequences = static_cast<int32_t>(std::min<int64_t>(pass.sequences, pass.rows));
        pass.max_count = static_cast<int32_t>(std::min<int64_t>(pass.max_count, pass.rows));
    }
    plan.rows = static_cast<int>(pass.rows);
    // splits of prefix and own tokens together
    const int64_t most = partial_results(a, pass.rows, max_length, max_prefix) / (pass.rows * a.heads);
    const int most_splits = static_cast<int>(std::clamp<int64_t>(most, 2, 2 * kMostSplits));
    const int kv_heads = a.cache.kv_heads, group = a.heads / kv_heads;
    uintptr_t bits = reinterpret_cast<uintptr_t>(a.query) | reinterpret_cast<uintptr_t>(a.cache.key) | reinterpret_cast<uintptr_t>(a.cache.value);
    if (a.groups) bits |= reinterpret_cast<uintptr_t>(a.prefix.key) | reinterpret_cast<uintptr_t>(a.prefix.value);
    const bool mma = a.cache.dtype == B200_BF16 && mma_takes(a.cache) && (!a.groups || mma_takes(a.prefix)) && bits % 16 == 0;
    plan.aligned = bits % 16 == 0 && a.cache.head_dim % 4 == 0;
    const int64_t pairs = pass.rows * group;
    const int groups = a.groups < pass.sequences ? a.groups : pass.sequences;
    const bool prefix = a.groups > 0 && max_prefix > 0;
    plan.form = mma ? Form::mma : Form::plain;
    plan.tensor = mma && prefix && pairs > 32 * static_cast<int64_t>(groups);
    // tiles of 16, 32 or 64 pairs: the smallest that holds the most that a sequence (or, with the prefix's items among them, a group) has
    const int64_t own_pairs = static_cast<int64_t>(pass.max_count) * group;
    const int64_t most_pairs = prefix && !plan.tensor ? std::max(own_pairs, ceil_div64(pairs, groups)) : own_pairs;
    plan.own_rows = !mma ? (most_pairs <= 16 ? 16 : 32) : most_pairs <= 16 ? 16 : most_pairs <= 32 ? 32 : 64;
    plan.prefix_rows = plan.tensor ? kTensorRows : plan.own_rows;
    plan.prefix_tiles = prefix ? static_cast<int>(pairs / plan.prefix_rows) + groups : 0;
    plan.own_tiles = ceil_div(own_pairs, plan.own_rows);
    auto splits = [&](int64_t items, int keys, int ctas, int room) {
        const int most = ceil_div(keys, mma ? 4 * kUnit : kUnit);   // the plain kernel takes longer over a step than a partial result costs
        const int64_t n = std::min<int64_t>(ctas / std::max<int64_t>(items, 1), std::min({most, room, kMostSplits}));
        return static_cast<int>(std::max<int64_t>(n, 1));
    };
    const int64_t own_items = static_cast<int64_t>(pass.sequences) * plan.own_tiles * kv_heads;
    plan.own_splits = splits(own_items, max_length, 2 * kSms, prefix ? most_splits / 2 : most_splits);
    const int room = std::min(kMostSplits, most_splits - plan.own_splits);
    const int prefix_steps = prefix ? ceil_div(max_prefix, kUnit) : 0, length_steps = ceil_div(max_length, kUnit);
    // tiles that the rows fill: the last tile of every group is half empty
    const int64_t filled = prefix ? std::max<int64_t>(ceil_div(pairs, plan.prefix_rows), groups) * kv_heads : 0;
    const int64_t own_filled = plan.own_tiles == 1 ? own_items : (ceil_div64(pairs, plan.own_rows) + pass.sequences / 2) * kv_heads;
    double time;   // of the split work, its launches and merge, in us
    if (plan.tensor) {
        const Share share = share_sms(filled, max_prefix, room, a.cache.head_dim, plan.own_rows, static_cast<double>(own_filled) * length_steps,
                                      static_cast<double>(pairs) * kv_heads * a.cache.head_dim * 8);
        plan.prefix_splits = share.splits;
        plan.own_ctas = share.own_ctas;
        time = 5.0 + share.time;
    } else {
        if (prefix) plan.prefix_splits = splits(filled, max_prefix, 2 * kSms, room);
        const double longest = std::max(prefix ? ceil_div(prefix_steps, plan.prefix_splits) : 0, ceil_div(length_steps, plan.own_splits));
        time = 10.0 + step_time(plan.own_rows, a.cache.head_dim) * std::max(longest, (static_cast<double>(filled) * prefix_steps + static_cast<double>(own_filled) * length_steps) / kSms);
    }
    if (!mma || !may_join) return plan;
    // Short prefixes, whose keys come from L2 each time: one item per tile of own rows goes over both and leaves the result.  Measured, 32 heads
    // of 64 over 8: 34 sequences of up to 5 tokens behind 329 keys 13.7 us joined, 16.4 split; 52 single tokens behind 165 12.5 and 13.0; 9 behind 5755 49 and 27.
    const int rows = own_pairs <= 16 ? 16 : own_pairs <= 32 ? 32 : 64, tiles = ceil_div(own_pairs, rows);
    const int64_t items = (tiles == 1 ? pass.sequences : ceil_div64(pairs, rows) + pass.sequences / 2) * kv_heads;
    const double step = step_time(rows, a.cache.head_dim);
    if (6.0 + step * (2.5 + (prefix_steps + length_steps) * std::max(1.0, static_cast<double>(items) / kSms)) > time) return plan;
    plan.joined = true;
    plan.tensor = false;
    plan.own_rows = plan.prefix_rows = rows;
    plan.own_tiles = tiles;
    plan.own_splits = 1;
    plan.prefix_tiles = plan.prefix_splits = plan.own_ctas = 0;
    return plan;
}

// Floats of the accumulators of `results` partial results: the maxima and sums behind them are read eight bytes at a time, and results * head_dim may be odd.
int64_t part_floats(int64_t results, int dim) { return (results * dim + 3) / 4 * 4; }

bool same_heads(const b200_kv_pages& a, const b200_kv_pages& b) { return a.dtype == b.dtype && a.kv_heads == b.kv_heads && a.head_dim == b.head_dim; }

int check_prefix(const b200_prefix_args* a, const b200_rows* pass, PrefixParams& p) {
    if (!rows_view(pass, p.rows)) return B200_BAD_ARGUMENT;
    if (!a) { set_error("b200_prefix_attention: no arguments"); return B200_BAD_ARGUMENT; }
    if (!pages_view(a->cache, "b200_prefix_attention", p.own)) return B200_BAD_ARGUMENT;
    if (a->groups < 0 || a->heads <= 0 || a->heads % a->cache.kv_heads || !a->query || !std::isfinite(a->scale)
        || (a->groups && (!a->group_first || !a->group_prefix || !a->prefix_length))) {
        set_error("b200_prefix_attention: bad pointer, size, scale or head grouping");
        return B200_BAD_ARGUMENT;
    }
    if (a->groups) {
        if (!pages_view(a->prefix, "b200_prefix_attention", p.prefix)) return B200_BAD_ARGUMENT;
        if (!same_heads(a->cache, a->prefix)) { set_error("b200_prefix_attention: prefix and cache differ in type or heads"); return B200_BAD_ARGUMENT; }
    }
    if (a->cache.head_dim > kMostDim) { set_error("b200_prefix_attention: head_dim above %d is not supported", kMostDim); return B200_UNSUPPORTED; }
    return B200_OK;
}

template <class T, int ROWS> cudaError_t launch_plain(const PrefixParams& p, unsigned items, bool whole, cudaStream_t stream) {
    auto kernel = p.dim <= 64 ? prefix_plain_kernel<T, 2, ROWS> : p.dim <= 128 ? prefix_plain_kernel<T, 4, ROWS> : prefix_plain_kernel<T, 8, ROWS>;
    // the kernel's limit is the same whatever the head size: a call beside this one may be between setting it and launching
    const int most = plain_smem(p.dim <= 64 ? 64 : p.dim <= 128 ? 128 : 256, 16 * ROWS);
    if (most > 48 * 1024) {
        const cudaError_t status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (status != cudaSuccess) return status;
    }
    return launch_dependent(kernel, dim3(items), dim3(kPlainThreads), static_cast<size_t>(plain_smem(p.dim, 16 * ROWS)), stream, p, whole);
}
template <class T> cudaError_t launch_plain(const PrefixParams& p, unsigned items, bool whole, cudaStream_t stream) {
    return p.own_rows == 16 ? launch_plain<T, 1>(p, items, whole, stream) : launch_plain<T, 2>(p, items, whole, stream);
}

template <int HD, bool JOINED, bool PLANES> int launch_mma(const PrefixParams& p, int ctas, cudaStream_t stream) {
    auto kernel = p.own_rows == 16 ? prefix_mma_kernel<HD, 4, JOINED, PLANES> : p.own_rows == 32 ? prefix_mma_kernel<HD, 2, JOINED, PLANES> : prefix_mma_kernel<HD, 1, JOINED, PLANES>;
    const int smem = MmaShape<HD>::smem_bytes(p.own_rows == 16 ? 4 : p.own_rows == 32 ? 2 : 1);
    MmaMaps maps;
    int box_rows = page_box_rows(p.own.page_size);
    if (p.groups && !p.beside) box_rows = std::min(box_rows, page_box_rows(p.prefix.page_size));   // powers of two
    int status = page_maps(p.own, box_rows, maps.own);
    if (status == B200_OK && p.groups && !p.beside) status = page_maps(p.prefix, box_rows, maps.prefix);
    if (status != B200_OK) return status;
    B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    return cuda_status(launch_dependent(kernel, dim3(static_cast<unsigned>(std::min(p.items, ctas))), dim3(kMmaThreads), static_cast<size_t>(smem), stream, maps, p, box_rows), "prefix_mma_kernel launch");
}

template <int HD> int launch_mma(const PrefixParams& p, int ctas, cudaStream_t stream) {
    if (p.joined) return p.planes ? launch_mma<HD, true, true>(p, ctas, stream) : launch_mma<HD, true, false>(p, ctas, stream);
    return p.planes ? launch_mma<HD, false, true>(p, ctas, stream) : launch_mma<HD, false, false>(p, ctas, stream);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" size_t b200_prefix_scratch_bytes(const b200_prefix_args* a, const b200_rows* pass, int32_t max_length, int32_t max_prefix) {
    PrefixParams p{};
    if (check_prefix(a, pass, p) != B200_OK || max_length <= 0 || max_prefix < 0) return 0;
    const int64_t results = partial_results(*a, pass->rows, max_length, max_prefix);
    return static_cast<size_t>(part_floats(results, a->cache.head_dim) + 2 * results) * sizeof(float) + 256;
}

extern "C" int b200_prefix_attention(const b200_prefix_args* a, const b200_rows* pass, int32_t max_length, int32_t max_prefix, void* scratch, size_t scratch_bytes,
                                     float* out, void* out_hi, void* out_lo, int64_t out_stride, void* stream) {
    PrefixParams p{};
    const int checked = check_prefix(a, pass, p);
    if (checked != B200_OK) return checked;
    const int64_t width = static_cast<int64_t>(a->heads) * a->cache.head_dim;
    if ((!out && !out_hi) || (out_lo && !out_hi) || max_length <= 0 || max_prefix < 0 || (out_stride && out_stride < width)) {
        set_error("b200_prefix_attention: bad result, stride or length");
        return B200_BAD_ARGUMENT;
    }
    const size_t need = b200_prefix_scratch_bytes(a, pass, max_length, max_prefix);
    if (!scratch || scratch_bytes < need || reinterpret_cast<uintptr_t>(scratch) % 32) {
        set_error("b200_prefix_attention: scratch of %zu bytes on a 32-byte boundary needed, %zu given", need, scratch_bytes);
        return B200_BAD_ARGUMENT;
    }
    Plan plan = make_plan(*a, *pass, max_length, max_prefix);
    if (!plan.joined) plan = make_plan(*a, *pass, max_length, max_prefix, false);
    p.heads = a->heads; p.group = a->heads / a->cache.kv_heads; p.by_group = divider(p.group); p.dim = a->cache.head_dim;
    p.groups = plan.prefix_splits || (plan.joined && max_prefix > 0) ? a->groups : 0;
    p.joined = plan.joined;
    p.planes = out || out_lo;
    p.group_first = a->group_first; p.group_prefix = a->group_prefix; p.prefix_length = a->prefix_length;
    p.query = a->query;
    p.scale = static_cast<float>(static_cast<double>(a->scale) * 1.4426950408889634);
    p.prefix_splits = plan.prefix_splits; p.own_splits = plan.own_splits; p.prefix_tiles = plan.prefix_tiles; p.own_tiles = plan.own_tiles;
    p.prefix_rows = plan.prefix_rows; p.own_rows = plan.own_rows;
    p.part_o = static_cast<float*>(scratch);
    p.part_ml = p.part_o + part_floats(static_cast<int64_t>(plan.rows) * a->heads * (plan.prefix_splits + plan.own_splits), p.dim);
    p.out = out; p.out_hi = static_cast<__nv_bfloat16*>(out_hi); p.out_lo = static_cast<__nv_bfloat16*>(out_lo);
    p.out_stride = out_stride ? out_stride : width;
    p.wide_out = (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_hi) | reinterpret_cast<uintptr_t>(out_lo)) % 16 == 0 && p.out_stride % 8 == 0 && p.dim % 8 == 0;
    const int64_t prefix_items = static_cast<int64_t>(plan.prefix_tiles) * plan.prefix_splits * a->cache.kv_heads;
    const int64_t own_items = static_cast<int64_t>(pass->sequences) * plan.own_tiles * plan.own_splits * a->cache.kv_heads;
    if (prefix_items + own_items > INT32_MAX || static_cast<int64_t>(pass->rows) * p.group > INT32_MAX / 2) {
        set_error("b200_prefix_attention: too many rows");
        return B200_UNSUPPORTED;
    }
    cudaStream_t s = as_stream(stream);
    if (plan.form == Form::mma) {
        int device = 0;
        B200_CUDA(cudaGetDevice(&device));
        p.status = device_status_word(device);
        if (!p.status) { set_error("b200_prefix_attention: the device status word could not be allocated"); return B200_NO_DEVICE; }
    }
    const bool spread = plan.prefix_splits + plan.own_splits > 8 && plan.rows * static_cast<int64_t>(a->heads) <= 8 * kSms;
    auto merge = spread ? (p.dim % 4 == 0 ? prefix_merge_kernel<4, true> : prefix_merge_kernel<1, true>)
                        : (p.dim % 4 == 0 ? prefix_merge_kernel<4, false> : prefix_merge_kernel<1, false>);
    for (int begin = 0; begin < p.rows.rows; begin += plan.rows) {
        p.row_begin = begin;
        p.row_end = std::min(p.rows.rows, begin + plan.rows);
        p.beside = 0;
        int ctas = 2 * kSms, status;
        if (plan.tensor) {
            status = launch_prefix_tensor(p, static_cast<int>(prefix_items), s);
            if (status != B200_OK) return status;
            p.beside = 1;
        }
        p.items = static_cast<int>(plan.tensor ? own_items : prefix_items + own_items);
        // beside the prefix: CTAs for the SMs that are free at once, or, where those do not suffice, two items per CTA, which begin as SMs become free
        if (plan.tensor) ctas = plan.own_ctas ? plan.own_ctas : std::max(ctas, (p.items + 1) / 2);
        const unsigned items = static_cast<unsigned>(p.items);
        if (plan.form == Form::plain)
            status = cuda_status(a->cache.dtype == B200_BF16 ? launch_plain<__nv_bfloat16>(p, items, plan.aligned, s) : launch_plain<float>(p, items, plan.aligned, s),
                                 "prefix_plain_kernel launch");
        else
            status = p.dim <= 64 ? launch_mma<64>(p, ctas, s) : p.dim <= 96 ? launch_mma<96>(p, ctas, s) : launch_mma<128>(p, ctas, s);
        if (status != B200_OK || plan.joined) return status;
        const int64_t pairs = static_cast<int64_t>(p.row_end - begin) * a->heads;
        status = cuda_status(launch_dependent(merge, dim3(static_cast<unsigned>(spread ? pairs : ceil_div64(pairs, kMergeWarps))), dim3(kMergeWarps * 32), 0, s, p),
                             "prefix_merge_kernel launch");
        if (status != B200_OK) return status;
    }
    return B200_OK;
}
