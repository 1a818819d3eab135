// The shared prefix of b200_prefix_attention on tcgen05: groups with many rows.
//
// A CTA has two tiles of 128 (row, head) pairs and a span of keys, 64 at a time.  Per tile and step: S = Q K^T into tensor memory (128 x 64 f32),
// a softmax warpgroup - a thread per pair - turns S into bf16 weights P in the same columns, O += P V with P read from tensor memory.  Each tile has two
// such buffers of scores, so that its softmax works on one while the products of the other are under way, and the two tiles share the tensor cores.
//   warps 0-3, 4-7   softmax of tile 0 and 1 (lane quarter = warp % 4), at the end the tile's partial result
//   warp 8           copies K and V steps through a ring of shared-memory slots with TMA, page by page
//   warps 9, 10      all products of tile 0 and 1 (a product keeps its issuing warp as long as the tensor cores); warp 9 also has the tensor memory
// O stays in tensor memory; it is rescaled only when a row's maximum has grown by more than 2^8 since the maximum its weights are relative to: they
// are relative to the same one in the sum and in O, so the quotient is the softmax all the same, and weights up to 2^8 lose nothing in f32 and bf16.
// With PLANES the second planes of the weights take the other half of the columns of S, and O += P V has twice the products.
#include "mma.cuh"
#include "prefix.cuh"
#include "prefix_tensor.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr int kTensorThreads = 352;
constexpr float kLazy = 8.0f;

// HD: the head size rounded up to 64 or 128; what is behind the head's end is zeros.
template <int HD> struct TensorShape {
    static constexpr int blocks = HD / 64;                          // 64 values: one swizzled row of 128 bytes
    static constexpr int query_block = 128 * 128, key_block = kTensorKeys * 128;
    static constexpr int query_bytes = blocks * query_block;        // a tile's queries
    static constexpr int step_bytes = blocks * key_block;           // K or V of a step
    static constexpr int slots = 10;
    static constexpr int smem_bytes = 2 * query_bytes + slots * step_bytes + 1024 + 1024;   // slack of the 1024-byte alignment, control words
    static constexpr uint32_t scores = mma_instruction_bf16(128, kTensorKeys);
    static constexpr uint32_t sums = mma_instruction_bf16(128, HD) | kTransposedB;
};
// The ring carries K0, K1, V0, K2, V1, ...: scores run ahead of the values by a step.
__device__ __forceinline__ int key_item(int step) { return step ? 2 * step - 1 : 0; }
__device__ __forceinline__ int value_item(int step, int steps) { return step + 1 < steps ? 2 * step + 2 : 2 * steps - 1; }

// 2^x for x <= 8 on the FMA units: 2^x = 2^n 2^f with n the nearest integer and |f| <= 1/2, 2^f by a polynomial whose relative error is the smallest one
// of degree 5 (fitted on Chebyshev points; 2.3e-7 as evaluated in f32), 2^n by its exponent.  Below 2^-126 the result is 2^-126.  `odd` becomes NaN where x is.
__device__ __forceinline__ Two exp2_polynomial(Two x, Two& odd) {
    float a, b;
    split(x, a, b);
    asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(a));   // -126
    asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(b));
    x = two(a, b);
    const Two rounded = add_two(x, two(12582912.0f, 12582912.0f));             // 1.5 * 2^23: the integer is in the low bits
    const Two n = add_two(rounded, two(-12582912.0f, -12582912.0f));
    const Two f = fma_two(n, two(-1.0f, -1.0f), x);
    Two r = fma_two(f, two(0.0013276472454890609f, 0.0013276472454890609f), two(0.009675541892647743f, 0.009675541892647743f));
    r = fma_two(r, f, two(0.05550713092088699f, 0.05550713092088699f));
    r = fma_two(r, f, two(0.24022120237350464f, 0.24022120237350464f));
    r = fma_two(r, f, two(0.6931469440460205f, 0.6931469440460205f));
    r = fma_two(r, f, two(1.0000001192092896f, 1.0000001192092896f));
    odd = fma_two(r, two(0.0f, 0.0f), odd);
    float whole_a, whole_b;
    split(rounded, whole_a, whole_b);
    split(r, a, b);
    return two(__uint_as_float(__float_as_uint(a) + (__float_as_uint(whole_a) << 23)), __uint_as_float(__float_as_uint(b) + (__float_as_uint(whole_b) << 23)));
}

// Scores behind the last key weigh nothing.
__device__ __forceinline__ void hide_scores(uint32_t (&s)[2][32], int live) {
    if (live >= kTensorKeys) return;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (32 * c + i >= live) s[c][i] = 0xff800000u;   // -inf
}

template <int HD, bool PLANES>
__global__ void __launch_bounds__(kTensorThreads, 1) prefix_tensor_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                                                                          const PrefixParams p, const int box_rows) {
    using S = TensorShape<HD>;
    extern __shared__ uint8_t tensor_shared[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tensor_shared) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* ring = smem + 2 * S::query_bytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + S::slots * S::step_bytes);
    uint64_t* empty = full + S::slots;
    uint64_t* q_ready = empty + S::slots;
    uint64_t* s_full = q_ready + 2;     // [tile][step & 1] S of a step is in tensor memory
    uint64_t* p_ready = s_full + 4;     // [tile][step & 1] the weights of a step are
    uint64_t* o_done = p_ready + 4;     // [tile][step & 1] a step's values are added to O
    uint64_t* tail = o_done + 4;        // what the last step's pages hold behind its keys is zeroed
    uint64_t* drained = tail + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
    volatile int* alive = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    begin_items(p);
    const Item it = find_prefix_item(p, blockIdx.x);
    if (!it.live) return;
    const int tiles = it.m_count - it.m_begin > 128 ? 2 : 1;
    const int steps = (it.keys.end - it.keys.begin + kTensorKeys - 1) / kTensorKeys;
    const int last_keys = it.keys.end - it.keys.begin - (steps - 1) * kTensorKeys;
    const bool has_tail = last_keys % box_rows != 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::slots; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], tiles);
        }
        for (int t = 0; t < 2; ++t) mbar_init(&q_ready[t], 4);
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_ready[i], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(tail, 1);
        for (int t = 0; t < 2; ++t) mbar_init(&drained[t], 1);
        *alive = 1;
        mbar_fence_init();
    }
    if (warp == 9) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // for whole warps; every wait ends: after a limit, or when another role has given up
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if (!mbar_wait(bar, parity)) {
            atomicExch(p.status, B200_DEVICE_TIMEOUT);
            *alive = 0;
        }
        return __all_sync(0xffffffffu, *alive != 0) != 0;
    };

    if (warp == 8) {
        const int outside = static_cast<int>(p.prefix.pages) * p.prefix.kv_heads * p.prefix.page_size;   // a row past the pools: zeros
        const int across = boxes_per_row(box_rows, p.dim), boxes = kTensorKeys / box_rows * across;   // at most 16
        const int block = lane % across, row = lane / across * box_rows;
        PageStream pages(p.prefix, it.slot, it.keys.begin + row, kTensorKeys, lane < boxes ? it.keys.end : 0);
        int issued = 0, key_row = outside, value_row = outside;
        for (int j = 0; j < 2 * steps; ++j, ++issued) {
            const int slot = j % S::slots;
            const bool values = j == 2 * steps - 1 || (j > 0 && j % 2 == 0);
            if (!values) {
                value_row = key_row;   // the values of a step come behind the keys of the next
                key_row = pages.next(it.kv_head, outside);
            }
            const int y = !values || j == 2 * steps - 1 ? key_row : value_row;
            if (!wait(&empty[slot], ((j / S::slots) & 1) ^ 1)) break;
            if (lane == 0) mbar_expect_tx(&full[slot], S::step_bytes);
            __syncwarp();
            uint8_t* to = ring + slot * S::step_bytes;
            const CUtensorMap* map = values ? &value_map : &key_map;
            if (across < S::blocks) {
                if (lane == 0) tma_load_3d(to, map, 0, y, 0, &full[slot]);
            } else if (lane < boxes) {
                tma_load_2d(to + block * S::key_block + row * 128, map, block * 64, y, &full[slot]);
            }
            __syncwarp();
        }
        if (issued == 2 * steps && has_tail) {
            // rows of the last box behind the keys may hold anything, and a weight of 0 does not cancel what is no number
            const int j = 2 * steps - 1, slot = j % S::slots;
            if (wait(&full[slot], (j / S::slots) & 1)) {
                const int behind = (last_keys + box_rows - 1) / box_rows * box_rows - last_keys;
                for (int i = lane; i < behind * 8 * S::blocks; i += 32)
                    *reinterpret_cast<uint4*>(ring + slot * S::step_bytes + i / (behind * 8) * S::key_block + last_keys * 128 + i % (behind * 8) * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(tail);
            }
        }
        if (*alive == 0)   // no copy is in flight when the CTA leaves
            for (int j = max(0, issued - S::slots); j < issued; ++j) mbar_wait(&full[j % S::slots], (j / S::slots) & 1);
    } else if (warp >= 9) {
        // The operands of the products come from uniform registers, which the compiler can only fill cheaply where it sees that a value is the same in
        // the whole warp: hence the broadcasts, and descriptors made outside the elected regions.
        const int t = __shfl_sync(0xffffffffu, warp - 9, 0), last = __shfl_sync(0xffffffffu, steps, 0) - 1;
        const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0), slots = __shfl_sync(0xffffffffu, smem_u32(ring), 0);
        const uint64_t query = operand_descriptor(__shfl_sync(0xffffffffu, smem_u32(smem), 0) + t * S::query_bytes);
        const uint32_t s_at = base + t * 128, o_at = base + 256 + t * HD;
        auto ready = [&](int item) { return wait(&full[item % S::slots], (item / S::slots) & 1); };
        auto key_of = [&](int item) { return operand_descriptor(slots + item % S::slots * S::step_bytes); };
        auto scores = [&](int buffer, int item, uint64_t key) {   // one lane
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
                tc_mma_bf16(s_at + buffer * 64, query + (k / 4 * S::query_block >> 4) + 2 * (k % 4), key + (k / 4 * S::key_block >> 4) + 2 * (k % 4), S::scores, k != 0);
            tc_commit(&s_full[2 * t + buffer]);
            tc_commit(&empty[item % S::slots]);
        };
        bool going = t < tiles && wait(&q_ready[t], 0);
        for (int step = 0; step < 2; ++step) {
            if (step > last || !going) break;
            const int k = key_item(step);
            going = ready(k);
            tc_fence_after_sync();
            const uint64_t key = key_of(k);
            if (going && elect_one()) scores(step, k, key);
        }
        for (int step = 0; step <= last; ++step) {
            if (!going) break;
            const int v = value_item(step, last + 1), k = key_item(step + 2), buffer = step & 1;
            const bool more = step + 2 <= last;
            going = ready(v) && (step < last || !has_tail || wait(tail, 0)) && (!more || ready(k)) && wait(&p_ready[2 * t + buffer], (step >> 1) & 1);
            tc_fence_after_sync();
            const uint64_t value = operand_descriptor_transposed(slots + v % S::slots * S::step_bytes, S::key_block), key = key_of(k);
            if (going && elect_one()) {
#pragma unroll
                for (int i = 0; i < (1 + PLANES) * (kTensorKeys / 16); ++i)   // the weights' first planes, then the second ones
                    tc_mma_bf16_tmem(o_at, s_at + buffer * 64 + 8 * i, value + i % (kTensorKeys / 16) * 128, S::sums, (step | i) != 0);
                tc_commit(&o_done[2 * t + buffer]);
                tc_commit(&empty[v % S::slots]);
                if (more) scores(buffer, k, key);
            }
        }
        if (*alive == 0) {   // nor a product
            if (elect_one()) tc_commit(&drained[t]);
            mbar_wait(&drained[t], 0);
        }
    } else if (warp / 4 < tiles) {
        const int t = warp / 4, row = threadIdx.x % 128;
        const int m_tile = it.m_begin + t * 128;
        // the tile's queries, as TMA would lay them out; a negative scale becomes one of the queries
        {
            const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
            constexpr int kPieces = 8 * S::blocks;
            uint4 x[kPieces];   // requested together; a row's pieces by neighbouring threads
            const int c = row % kPieces;
#pragma unroll
            for (int u = 0; u < kPieces; ++u) {
                const int m = m_tile + row / kPieces + u * (128 / kPieces);
                x[u] = make_uint4(0, 0, 0, 0);
                if (m < it.m_count && 8 * c < p.dim) x[u] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.query) + pair_row(p, it, m) * p.dim + 8 * c));
            }
#pragma unroll
            for (int u = 0; u < kPieces; ++u) {
                const int r = row / kPieces + u * (128 / kPieces);
                x[u].x ^= flip; x[u].y ^= flip; x[u].z ^= flip; x[u].w ^= flip;
                *reinterpret_cast<uint4*>(smem + t * S::query_bytes + c / 8 * S::query_block + r * 128 + (((c ^ r) & 7) << 4)) = x[u];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_ready[t]);
        }
        const float scale = fmaxf(fabsf(p.scale), 0x1p-149f);   // 0 times the -inf of hidden scores would be no number
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + t * 128, o_at = tmem + lanes + 256 + t * HD;
        float most = -INFINITY, sum = 0.0f;   // the maximum that the weights are relative to
        bool going = true;
        for (int step = 0; step < steps; ++step) {
            const int buffer = 2 * t + (step & 1);
            const uint32_t s_here = s_at + (step & 1) * 64;
            going = wait(&s_full[buffer], (step >> 1) & 1);
            if (!going) break;
            tc_fence_after_sync();
            uint32_t s[2][32];
#pragma unroll
            for (int c = 0; c < 2; ++c) tmem_load_32_async(s_here + 32 * c, s[c]);
            tmem_wait_loads();
#pragma unroll
            for (int c = 0; c < 2; ++c) tmem_loaded(s[c]);
            hide_scores(s, it.keys.end - it.keys.begin - step * kTensorKeys);
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 32; i += 2)
#pragma unroll
                for (int c = 0; c < 4; ++c) top[c] = fmaxf(top[c], __uint_as_float(s[c / 2][i + c % 2]));
            const float here = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
            const bool grows = here > most + kLazy;
            if (__any_sync(0xffffffffu, grows)) {
                const float base = whole_maximum(here), factor = grows ? exp2_fast(most - base) : 1.0f;
                if (grows) most = base;
                sum *= factor;
                if (step > 0) {
                    going = wait(&o_done[2 * t + ((step - 1) & 1)], ((step - 1) >> 1) & 1);
                    if (!going) break;
                    tc_fence_after_sync();
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t o[32];
                        tmem_load_32(o_at + 32 * c, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                        tmem_store_32(o_at + 32 * c, o);
                    }
                }
            }
            const float base = most == -INFINITY ? 0.0f : -most;
            // The exponential unit gives 16 results a cycle and SM: 1024 cycles for the two tiles' 128 x 64 weights, as long as their products take.  Every
            // fourth pair is computed on the FMA units instead.
            const Two scales = two(scale, scale), bases = two(base, base);
            float sums[4] = {};
            Two odd = two(0.0f, 0.0f);
            uint32_t weights[32], second[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                Two x = fma_two(two(__uint_as_float(s[i / 16][2 * (i % 16)]), __uint_as_float(s[i / 16][2 * (i % 16) + 1])), scales, bases);
                float a, b;
                if (i % 4 == 3) {
                    x = exp2_polynomial(x, odd);
                    split(x, a, b);
                } else {
                    split(x, a, b);
                    a = exp2_fast(a);
                    b = exp2_fast(b);
                }
                float &low = sums[2 * (i & 1)], &high = sums[2 * (i & 1) + 1];
                if constexpr (PLANES) {
                    weights[i] = first_plane(a, b);
                    second[i] = second_plane(a, b);
                    low += a;
                    high += b;
                } else {
                    weights[i] = pack_bf16(a, b);
                    add_bf16(weights[i], low, high);
                }
            }
            tmem_store_32(s_here, weights);
            if constexpr (PLANES) tmem_store_32(s_here + 32, second);
            {
                float a, b;
                split(odd, a, b);
                sum += a + b;   // (one after the other: 361 us for 2.2 k rows behind 8000 keys, in one expression 367)
                sum += (sums[0] + sums[1]) + (sums[2] + sums[3]);
            }
            tmem_wait_stores();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[buffer]);
        }
        if (going && wait(&o_done[2 * t + ((steps - 1) & 1)], ((steps - 1) >> 1) & 1)) {
            tc_fence_after_sync();
            // a thread has a row of O: through the tile's part of shared memory, whose queries nobody needs any more, so that the lanes of a store write
            // neighbouring pieces; 64 values of the warp's 32 rows at a time, pieces permuted against bank conflicts
            const int m = m_tile + row;
            const int64_t to = m < it.m_count ? partial_row(p, it, m) : -1;
            if (to >= 0) *reinterpret_cast<float2*>(p.part_ml + 2 * to) = make_float2(most, sum);
            uint8_t* rows = smem + t * S::query_bytes + (warp & 3) * (S::query_bytes / 4);
            constexpr int kPieces = S::query_bytes / 4 / 32 / 16;   // 16 (8) pieces of four values: 64 (32) values
#pragma unroll 1
            for (int first = 0; first < HD; first += 4 * kPieces) {
#pragma unroll
                for (int c = 0; c < kPieces / 8; ++c) {
                    uint32_t o[32];
                    tmem_load_32(o_at + first + 32 * c, o);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4*>(rows + lane * kPieces * 16 + (((8 * c + i) ^ (lane & 7)) << 4)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const int r = i * (32 / kPieces) + lane / kPieces, c = lane % kPieces;
                    const int64_t at = __shfl_sync(0xffffffffu, to, r);
                    if (at >= 0 && first + 4 * c < p.dim) *reinterpret_cast<uint4*>(p.part_o + at * p.dim + first + 4 * c) = *reinterpret_cast<const uint4*>(rows + r * kPieces * 16 + ((c ^ (r & 7)) << 4));
                }
                __syncwarp();
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

template <int HD, bool PLANES> int launch_tensor(const PrefixParams& p, int items, cudaStream_t stream) {
    const int box_rows = page_box_rows(p.prefix.page_size);
    CUtensorMap maps[2];
    const int status = page_maps(p.prefix, box_rows, maps);
    if (status != B200_OK) return status;
    auto kernel = prefix_tensor_kernel<HD, PLANES>;
    B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TensorShape<HD>::smem_bytes));
    return cuda_status(launch_dependent(kernel, dim3(static_cast<unsigned>(items)), dim3(kTensorThreads), TensorShape<HD>::smem_bytes, stream, maps[0], maps[1], p, box_rows),
                       "prefix_tensor_kernel launch");
}

}  // namespace

int page_box_rows(int page_size) {
    for (int rows = 64; rows >= 8; rows /= 2)
        if (page_size % rows == 0) return rows;
    return 0;
}

int page_maps(const PagesView& pages, int box_rows, CUtensorMap* maps) {
    encode_tiled_fn encode = tensor_map_encoder();
    if (!encode) { set_error("cuTensorMapEncodeTiled is not available from this driver"); return B200_NO_DEVICE; }
    const cuuint64_t rows = static_cast<cuuint64_t>(pages.pages) * pages.kv_heads * pages.page_size, bytes = static_cast<cuuint64_t>(pages.head_dim) * 2;
    const bool whole = boxes_per_row(box_rows, pages.head_dim) == 1 && pages.head_dim > 64;
    // [64 values][rows][blocks of 64 values], or [values][rows]
    const cuuint64_t dims[3] = {whole ? 64 : static_cast<cuuint64_t>(pages.head_dim), rows, static_cast<cuuint64_t>(pages.head_dim / 64)}, strides[2] = {bytes, 128};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(pages.head_dim / 64)}, ones[3] = {1, 1, 1};
    for (int which = 0; which < 2; ++which) {
        const CUresult result = encode(&maps[which], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, whole ? 3 : 2, pages.pool[which], dims, strides, box, ones,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (result != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled failed with %d", static_cast<int>(result)); return B200_BAD_ARGUMENT; }
    }
    return B200_OK;
}

int launch_prefix_tensor(const PrefixParams& p, int items, cudaStream_t stream) {
    if (p.planes) return p.dim > 64 ? launch_tensor<128, true>(p, items, stream) : launch_tensor<64, true>(p, items, stream);
    return p.dim > 64 ? launch_tensor<128, false>(p, items, stream) : launch_tensor<64, false>(p, items, stream);
}

}  // namespace b200
