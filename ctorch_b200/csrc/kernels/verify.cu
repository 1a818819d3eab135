// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Two launches.  verify_rows_kernel: for every row of target and draft logits the maximum and the sum of its weights exp((x - max) / T); a row is
// split over a cluster of CTAs that hold their part in shared memory, so the row is read once although the weights need the maximum first.
// verify_finish_kernel: one cluster per sequence walks the acceptance tests, then draws from the residual of the row that refused: running sums
// over segments of 128 values, in index order.  Sums are as good as f64 and added in an order that the row's alignment and the pass's sizes set.
#include "linear_common.cuh"
#include "mma.cuh"
#include "rows.cuh"

#include <algorithm>

#include <cmath>

namespace b200 {
namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kRowThreads = 128, kRowWarps = kRowThreads / 32;
constexpr int kPieceVectors = 1024, kTilePieces = 4;
constexpr int kTileVectors = kTilePieces * kPieceVectors;    // 16-byte vectors of a row that a CTA holds
constexpr int kSweeps = kPieceVectors / kRowThreads;         // of the block's threads over a piece
static_assert(kTileVectors / kRowThreads * 4 / 2 <= 64);     // see add_weights: values of a thread per half of its sums
constexpr int kVerifyMostParts = 8, kVerifyMostVocab = 1 << 23;

struct VerifyParams {
    RowsView rows;
    const float *logits, *draft;
    int64_t stride;
    int vocab, parts, chunk;      // CTAs per row, values per CTA (a multiple of 4)
    int draw_parts, draw_chunk;   // the same of the drawing clusters
    float inverse;
    const int64_t* ids;
    const double *accept, *draw;
    int32_t* accepted;
    int64_t* next;
    int advance;
    float* row_max;               // [2 * rows]: target and draft of each row
    double* row_sum;              // [2 * rows][parts]
    Candidate* best;              // greedy: [rows][parts]
    int32_t* status;
};

__device__ __forceinline__ float weight_of(float x, float most, float inverse) { return expf(__fmul_rn(__fsub_rn(x, most), inverse)); }

// A weight in f64 by its bits (conversions share the exponential's unit, at a quarter of the rate of these operations); weights below 2^-126 count as 0.
__device__ __forceinline__ double widen(float w) {
    const uint32_t bits = __float_as_uint(w);   // not negative
    return bits < 0x00800000u ? 0.0 : __hiloint2double(static_cast<int>((bits >> 3) + (bits < 0x7f800000u ? 0x38000000u : 0x70000000u)), static_cast<int>(bits << 29));
}

// Adds the weights of two values to a sum in three parts: multiples of 2^-17, of which the at most 64 that a thread adds are exact in f32; what is left of each
// weight, at most 2^-18, in multiples of 2^-36, exact as well; and what is left of that, at most 2^-37, to a sum below 2^-31, off by 2^-56 for each value.
// A row's sum is then off by 2^-38 for 2^18 values, as good as f64 sums of as many weights (2^-53 each), without conversions, which take the exponential's unit.
// With two parts it was off by up to 1.4e-7 (10^5 weights of 2^-18).
struct Parts { Two coarse, middle, fine; };
__device__ __forceinline__ void add_weights(Two x, Two minus_most, Two inverse, Parts& sum) {
    float a, b;
    split(mul_two(add_two(x, minus_most), inverse), a, b);
    const Two w = two(expf(a), expf(b)), minus_one = two(-1.0f, -1.0f);
    const Two high = add_two(add_two(w, two(96.0f, 96.0f)), two(-96.0f, -96.0f));
    const Two rest = fma_two(high, minus_one, w);
    const Two middle = add_two(add_two(rest, two(0x1.8p-13f, 0x1.8p-13f)), two(-0x1.8p-13f, -0x1.8p-13f));
    sum.coarse = add_two(sum.coarse, high);
    sum.middle = add_two(sum.middle, middle);
    sum.fine = add_two(sum.fine, fma_two(middle, minus_one, rest));
}
__device__ __forceinline__ double total_of(const Parts& sum) {
    float a, b;
    double total = 0.0;
    split(sum.fine, a, b);
    total += static_cast<double>(a) + static_cast<double>(b);
    split(sum.middle, a, b);
    total += static_cast<double>(a) + static_cast<double>(b);
    split(sum.coarse, a, b);
    return total + (static_cast<double>(a) + static_cast<double>(b));
}

// One CTA's part of a row, in vectors of four values on 16-byte boundaries: vector v holds the values 4 v - shift .. + 3 of the part.
struct RowPart {
    const float* base;
    int length, shift, vectors;
    __device__ __forceinline__ RowPart(int vocab, int chunk, const float* row, int part) {
        const int begin = min(vocab, part * chunk);
        base = row + begin;
        length = min(vocab, begin + chunk) - begin;
        shift = static_cast<int>((reinterpret_cast<uintptr_t>(base) >> 2) & 3);
        vectors = length > 0 ? (length + shift + 3) / 4 : 0;
    }
    // Values of vector v as seen with `by` in the place of the own shift; outside the part -inf, the value without weight.
    __device__ __forceinline__ float4 load(int v, int by) const {
        const int at = 4 * v - by;
        if (by == shift && at >= 0 && at + 4 <= length) return __ldcs(reinterpret_cast<const float4*>(base + at));
        float r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) r[u] = at + u >= 0 && at + u < length ? __ldcs(base + at + u) : -INFINITY;
        return make_float4(r[0], r[1], r[2], r[3]);
    }
    __device__ __forceinline__ float4 load(int v) const { return load(v, shift); }
    __device__ __forceinline__ float4 load_or_none(int v) const { return v < vectors ? load(v) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }
    // A vector as it lies in memory, without what lies outside the part.
    __device__ __forceinline__ float4 inside(float4 x, int v) const {
        const int at = 4 * v - shift;
        if (at >= 0 && at + 4 <= length) return x;
        x.x = at >= 0 && at < length ? x.x : -INFINITY;
        x.y = at + 1 >= 0 && at + 1 < length ? x.y : -INFINITY;
        x.z = at + 2 >= 0 && at + 2 < length ? x.z : -INFINITY;
        x.w = at + 3 >= 0 && at + 3 < length ? x.w : -INFINITY;
        return x;
    }
};

__device__ __forceinline__ int cluster_part() {
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    return static_cast<int>(rank);
}
__device__ __forceinline__ double load_cluster_double(uint32_t address) {
    double value;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(value) : "r"(address) : "memory");
    return value;
}

// Of a peer whose candidate is on an 8-byte boundary.
__device__ __forceinline__ Candidate load_cluster_candidate(uint32_t address) {
    Candidate c;
    asm volatile("ld.shared::cluster.v2.b32 {%0, %1}, [%2];" : "=f"(c.value), "=r"(c.index) : "r"(address) : "memory");
    return c;
}

__device__ __forceinline__ float most_of(float4 x) { return fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)); }

// grid: clusters of `parts` CTAs, two (target, draft) or one per row.  A part's first kTileVectors come to shared memory with bulk copies and stay for the
// second pass; longer parts are read twice.  Bound by the chain of a CTA (9 us: launch of the cluster, its row's place, copy, the cluster's barrier, 16 instructions
// per value), of which an SM holds three with 64 KB each: 710 rows of 128256 take 130 us, 2.8 TB/s.  What did not help: several rows per cluster with the next one's
// copies under way (+15%), a cluster per sequence that stops at the first refusal (+50%), 512 threads (+10%).
__global__ void __launch_bounds__(kRowThreads) verify_rows_kernel(const VerifyParams p) {
    extern __shared__ __align__(128) float4 tile[];
    __shared__ uint64_t full[kTilePieces];
    __shared__ float warp_max_of[kRowWarps];
    __shared__ double warp_sum_of[kRowWarps];
    __shared__ float part_max;
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    if (thread == 0) {
        for (int i = 0; i < kTilePieces; ++i) mbar_init(&full[i], 1);
        mbar_fence_init();
    }
    __syncthreads();
    grid_dependency_wait();
    grid_launch_dependents();
    const int part = cluster_part(), unit = blockIdx.x / p.parts;
    const int sides = p.draft ? 2 : 1;
    const int row = unit / sides, side = unit % sides;
    // (the whole cluster leaves together)
    if (row >= __ldg(p.rows.first + p.rows.sequences)) return;
    if (side == 1 && row + 1 == __ldg(p.rows.first + __ldg(p.rows.sequence + row) + 1)) return;
    const RowPart own(p.vocab, p.chunk, (side ? p.draft : p.logits) + row * p.stride, part);
    const int tiled = min(own.vectors, kTileVectors);
    if (thread == 0)
        for (int piece = 0; piece * kPieceVectors < tiled; ++piece) {
            int begin = piece * kPieceVectors, end = min(begin + kPieceVectors, tiled);
            // The vectors at the part's ends may reach into its neighbours, which are in the buffer but for the first row's begin and the last row's end.
            if (begin == 0 && own.shift && row == 0 && part == 0) {
                for (int u = own.shift; u < 4; ++u) reinterpret_cast<float*>(tile)[u] = u - own.shift < own.length ? __ldg(own.base + u - own.shift) : 0.0f;
                ++begin;
            }
            if (begin < end && 4 * end - own.shift > own.length && row == p.rows.rows - 1) {
                --end;
                for (int u = 0; u < 4; ++u) {
                    const int at = 4 * end - own.shift + u;
                    reinterpret_cast<float*>(tile + end)[u] = at >= 0 && at < own.length ? __ldg(own.base + at) : 0.0f;
                }
            }
            mbar_expect_tx(&full[piece], begin < end ? (end - begin) * 16 : 0);
            if (begin < end) bulk_load(tile + begin, own.base - own.shift + 4 * begin, (end - begin) * 16, &full[piece]);
        }
    float most = -INFINITY;
    bool gave_up = false;
    for (int v = kTileVectors + thread; v < own.vectors; v += kPieceVectors) {
        float4 x[kSweeps];
#pragma unroll
        for (int j = 0; j < kSweeps; ++j) x[j] = own.load_or_none(v + j * kRowThreads);
#pragma unroll
        for (int j = 0; j < kSweeps; ++j) most = fmaxf(most, most_of(x[j]));
    }
    const int sweeps = max(0, tiled - 1) / kRowThreads;   // whole ones, before the part's last vector
    const float4* mine = tile + thread;
    for (int piece = 0; piece * kPieceVectors < tiled; ++piece) {
        if (!mbar_wait(&full[piece], 0)) {
            atomicExch(p.status, B200_DEVICE_TIMEOUT);
            gave_up = true;
        }
        if (piece == 0 && thread == 0 && own.shift) tile[0] = own.inside(tile[0], 0);
        if (kSweeps * (piece + 1) <= sweeps) {
#pragma unroll
            for (int j = 0; j < kSweeps; ++j) most = fmaxf(most, most_of(mine[(kSweeps * piece + j) * kRowThreads]));
            continue;
        }
        for (int v = piece * kPieceVectors + thread; v < min(tiled, (piece + 1) * kPieceVectors); v += kRowThreads) {
            if (v == own.vectors - 1) tile[v] = own.inside(tile[v], v);
            most = fmaxf(most, most_of(tile[v]));
        }
    }
    most = warp_max(most);
    if (lane == 0) warp_max_of[warp] = most;
    __syncthreads();
    most = warp_max(lane < kRowWarps ? warp_max_of[lane] : -INFINITY);
    if (p.parts > 1) {
        if (thread == 0) part_max = most;
        cluster_sync_all();
        most = warp_max(lane < p.parts ? load_cluster_float(map_peer_shared(smem_u32(&part_max), static_cast<uint32_t>(lane))) : -INFINITY);
    }
    double sum = 0.0;
    const Two zero = two(0.0f, 0.0f), minus_most = two(-most, -most), inverse = two(p.inverse, p.inverse);
    Parts parts{zero, zero, zero};
    auto add = [&](float4 x) {
        add_weights(two(x.x, x.y), minus_most, inverse, parts);
        add_weights(two(x.z, x.w), minus_most, inverse, parts);
    };
    for (int sweep = 0; sweep + 4 <= sweeps; sweep += 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) add(mine[(sweep + j) * kRowThreads]);
    for (int v = sweeps / 4 * 4 * kRowThreads + thread; v < tiled; v += kRowThreads) add(tile[v]);
    sum += total_of(parts);
    for (int v = kTileVectors + thread; v < own.vectors; v += kPieceVectors) {
        float4 x[kSweeps];
#pragma unroll
        for (int j = 0; j < kSweeps; ++j) x[j] = own.load_or_none(v + j * kRowThreads);
        parts = {zero, zero, zero};
#pragma unroll
        for (int j = 0; j < kSweeps; ++j) add(x[j]);
        sum += total_of(parts);
    }
    // values outside the part weigh nothing; where the row's maximum is itself -inf every weight is NaN, as for the values inside
    sum = warp_sum(sum);
    if (lane == 0) warp_sum_of[warp] = sum;
    __syncthreads();
    if (thread == 0) {
        sum = 0.0;
        for (int w = 0; w < kRowWarps; ++w) sum += warp_sum_of[w];
        const int64_t at = 2 * static_cast<int64_t>(row) + side;
        p.row_sum[at * p.parts + part] = sum;
        if (part == 0) p.row_max[at] = most;
    }
    if (gave_up)   // no copy is in flight when the CTA leaves
        for (int piece = 0; piece * kPieceVectors < tiled; ++piece) mbar_wait(&full[piece], 0);
    if (p.parts > 1) cluster_sync_all();   // the peers have read this CTA's maximum
}

// Temperature 0: the first maximum of every row.  grid: rows * parts.
__global__ void __launch_bounds__(kVerifyThreads) verify_best_kernel(const VerifyParams p) {
    __shared__ Candidate warp_best[kVerifyWarps];
    grid_dependency_wait();
    grid_launch_dependents();
    const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    if (row >= __ldg(p.rows.first + p.rows.sequences)) return;
    const RowPart own(p.vocab, p.chunk, p.logits + row * p.stride, part);
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    constexpr int kBatch = 8;
    Candidate best{-INFINITY, INT32_MAX};
    for (int begin = thread; begin < own.vectors; begin += kBatch * kVerifyThreads) {
        float4 x[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) x[j] = own.load_or_none(begin + j * kVerifyThreads);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int at = 4 * (begin + j * kVerifyThreads) - own.shift;
            const float values[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const Candidate other{values[u], part * p.chunk + at + u};
                if (at + u >= 0 && at + u < own.length && preferred(other, best)) best = other;
            }
        }
    }
    for (int o = 16; o > 0; o >>= 1) {
        const Candidate other{__shfl_xor_sync(0xffffffffu, best.value, o), __shfl_xor_sync(0xffffffffu, best.index, o)};
        if (preferred(other, best)) best = other;
    }
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    if (thread == 0) {
        for (int w = 1; w < kVerifyWarps; ++w)
            if (preferred(warp_best[w], best)) best = warp_best[w];
        p.best[static_cast<int64_t>(row) * p.parts + part] = best;
    }
}

struct RowStats {
    float most;
    double sum;
    bool good;   // there are finite weights
};
__device__ __forceinline__ RowStats row_stats(const VerifyParams& p, int row, int side) {
    const int64_t at = 2 * static_cast<int64_t>(row) + side;
    RowStats r{p.row_max[at], 0.0, false};
    double part[kVerifyMostParts];
#pragma unroll
    for (int c = 0; c < kVerifyMostParts; ++c) part[c] = c < p.parts ? p.row_sum[at * p.parts + c] : 0.0;
#pragma unroll
    for (int c = 0; c < kVerifyMostParts; ++c) r.sum += part[c];
    r.good = r.sum > 0.0 && r.sum < INFINITY;
    return r;
}

// What is left of a value's probability: the target's share less the draft's.
struct Residual {
    float most, draft_most, inverse;
    double scale, draft_scale;   // one over the sums
    int without;                 // the draft that counts as certain, or -1
    bool minus;                  // the draft's probabilities are taken off
    __device__ __forceinline__ double value(float x, float y, int index) const {
        double left = widen(weight_of(x, most, inverse)) * scale;
        if (minus) left -= widen(weight_of(y, draft_most, inverse)) * draft_scale;
        return index == without || !(left > 0.0) ? 0.0 : left;
    }
};

// What the test of a row's draft needs besides the row's sums.
struct Test {
    bool valid;
    float target, draft;
    double accept;
};
__device__ __forceinline__ Test fetch_test(const VerifyParams& p, int row) {
    Test t{};
    const int64_t x = __ldg(p.ids + row + 1);
    t.accept = p.accept[row];
    t.valid = x >= 0 && x < p.vocab;
    if (t.valid) {
        t.target = __ldg(p.logits + row * p.stride + x);
        if (p.draft) t.draft = __ldg(p.draft + row * p.stride + x);
    }
    return t;
}

// The rows of a sequence whose tokens stand: its slot's length moves on.  A slot below 0 is none.
__device__ __forceinline__ void advance_slot(const VerifyParams& p, int s, int tokens) {
    const int slot = __ldg(p.rows.slot + s);
    if (p.advance && slot >= 0) atomicAdd(p.rows.lengths + slot, tokens);
}

// grid: a cluster of `draw_parts` CTAs per sequence.  Dynamic shared memory: the sums of the part's segments of 128 values.
__global__ void __launch_bounds__(kVerifyThreads) verify_finish_kernel(const VerifyParams p) {
    extern __shared__ double segment_sum[];
    __shared__ int stop_row;
    __shared__ double part_total;
    __shared__ Candidate warp_best[kVerifyWarps];
    __shared__ alignas(8) Candidate part_best;   // read by the peers as eight bytes
    const int part = cluster_part(), s = blockIdx.x / p.draw_parts;
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    // The pass's arrays and the logits were complete before verify_rows_kernel began: what the first tests need is fetched while that still runs.
    const int first = __ldg(p.rows.first + s), last = __ldg(p.rows.first + s + 1) - 1;
    const double draw = last >= first ? p.draw[s] : 0.0;
    Test test{};
    if (warp == 0 && first + lane < last) test = fetch_test(p, first + lane);
    grid_dependency_wait();
    grid_launch_dependents();
    if (last < first) {
        if (part == 0 && thread == 0) {
            p.accepted[s] = 0;
            p.next[s] = -1;
        }
        return;
    }
    // the first draft that is refused, else the last row
    if (warp == 0) {
        int stop = last;
        for (int base = first; base < last; base += 32) {
            const int row = base + lane;
            if (base > first && row < last) test = fetch_test(p, row);
            bool refused = false;
            if (row < last) {
                refused = true;
                if (test.valid) {
                    const RowStats t = row_stats(p, row, 0);
                    double q = 1.0;
                    if (p.draft) {
                        const RowStats d = row_stats(p, row, 1);
                        q = d.good ? widen(weight_of(test.draft, d.most, p.inverse)) / d.sum : NAN;
                    }
                    const double share = t.good ? widen(weight_of(test.target, t.most, p.inverse)) / t.sum : NAN;
                    refused = !(test.accept * q < share);
                }
            }
            const unsigned found = __ballot_sync(0xffffffffu, refused);
            if (found) {
                stop = base + __ffs(found) - 1;
                break;
            }
        }
        if (lane == 0) stop_row = stop;
    }
    __syncthreads();
    const int row = stop_row;
    const RowStats stats = row_stats(p, row, 0);
    Residual residual{stats.most, 0.0f, p.inverse, 1.0 / stats.sum, 0.0, -1, false};
    if (row < last) {
        const int64_t x = __ldg(p.ids + row + 1);
        if (x >= 0 && x < p.vocab) {
            if (p.draft) {
                const RowStats d = row_stats(p, row, 1);
                residual.minus = d.good;
                residual.draft_most = d.most;
                residual.draft_scale = 1.0 / d.sum;
            } else {
                residual.without = static_cast<int>(x);
            }
        }
    }
    const RowPart target(p.vocab, p.draw_chunk, p.logits + row * p.stride, part);
    const RowPart draft(p.vocab, p.draw_chunk, (p.draft ? p.draft : p.logits) + row * p.stride, part);
    const int begin = part * p.draw_chunk;
    if (!stats.good) {   // no distribution: the argmax, as b200_argmax has it
        Candidate best{-INFINITY, INT32_MAX};
        for (int i = thread; i < target.length; i += kVerifyThreads) {
            const Candidate other{target.base[i], begin + i};
            if (preferred(other, best)) best = other;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const Candidate other{__shfl_xor_sync(0xffffffffu, best.value, o), __shfl_xor_sync(0xffffffffu, best.index, o)};
            if (preferred(other, best)) best = other;
        }
        if (lane == 0) warp_best[warp] = best;
        __syncthreads();
        if (thread == 0) {
            for (int w = 1; w < kVerifyWarps; ++w)
                if (preferred(warp_best[w], best)) best = warp_best[w];
            part_best = best;
        }
        cluster_sync_all();
        if (part == 0 && thread == 0) {
            for (int c = 1; c < p.draw_parts; ++c) {
                const Candidate other = load_cluster_candidate(map_peer_shared(smem_u32(&part_best), static_cast<uint32_t>(c)));
                if (preferred(other, best)) best = other;
            }
            p.next[s] = best.index;
        }
        cluster_sync_all();
    } else {
        const int segments = (target.vectors + 31) / 32;
        const int run = (segments + 31) / 32;   // segments that a lane of the first warp adds up
        double total, before, lane_before, mine;
        while (true) {
            constexpr int kBatch = 4;   // segments of a warp whose values are requested together
            for (int begin_g = warp; begin_g < segments; begin_g += kBatch * kVerifyWarps) {
                float4 x[kBatch], y[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int v = (begin_g + k * kVerifyWarps) * 32 + lane;
                    x[k] = v < target.vectors ? target.load(v) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    y[k] = residual.minus && v < target.vectors ? draft.load(v, target.shift) : x[k];
                }
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int g = begin_g + k * kVerifyWarps, at = begin + 4 * (g * 32 + lane) - target.shift;
                    double sum = residual.value(x[k].x, y[k].x, at);
                    sum += residual.value(x[k].y, y[k].y, at + 1);
                    sum += residual.value(x[k].z, y[k].z, at + 2);
                    sum += residual.value(x[k].w, y[k].w, at + 3);
                    sum = warp_sum(sum);
                    if (lane == 0 && g < segments) segment_sum[g] = sum;
                }
            }
            __syncthreads();
            if (warp == 0) {
                mine = 0.0;
                for (int g = lane * run; g < min(segments, (lane + 1) * run); ++g) mine += segment_sum[g];
                double up_to = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double other = __shfl_up_sync(0xffffffffu, up_to, o);
                    if (lane >= o) up_to += other;
                }
                const double below = __shfl_up_sync(0xffffffffu, up_to, 1);
                lane_before = lane ? below : 0.0;
                if (lane == 31) part_total = up_to;
            }
            cluster_sync_all();
            total = before = 0.0;
            for (int c = 0; c < p.draw_parts; ++c) {
                if (c == part) before = total;
                total += load_cluster_double(map_peer_shared(smem_u32(&part_total), static_cast<uint32_t>(c)));
            }
            if (total > 0.0 || (!residual.minus && residual.without < 0)) break;
            // nothing is left by rounding: the target's own distribution (every CTA of the cluster comes to this together)
            residual.minus = false;
            residual.without = -1;
            cluster_sync_all();
        }
        const double wanted = draw * total;
        // the first part whose running sum exceeds what is wanted; by rounding there may be none, then the last with any weight
        int chosen = -1, heavy = 0;
        double running = 0.0;
        for (int c = 0; c < p.draw_parts; ++c) {
            const double here = load_cluster_double(map_peer_shared(smem_u32(&part_total), static_cast<uint32_t>(c)));
            running += here;
            if (here > 0.0) heavy = c;
            if (chosen < 0 && here > 0.0 && running > wanted) chosen = c;
        }
        if (chosen < 0) chosen = heavy;
        if (chosen == part && warp == 0) {
            // the same among the segments, then among the segment's values
            double sum = before + lane_before;
            int segment = -1, some = -1;
            for (int g = lane * run; g < min(segments, (lane + 1) * run); ++g) {
                if (segment_sum[g] > 0.0) some = g;
                if (segment_sum[g] > 0.0 && sum + segment_sum[g] > wanted) {
                    segment = g;
                    break;
                }
                sum += segment_sum[g];
            }
            const unsigned found = __ballot_sync(0xffffffffu, segment >= 0);
            if (found) {
                const int from = __ffs(found) - 1;
                segment = __shfl_sync(0xffffffffu, segment, from);
                sum = __shfl_sync(0xffffffffu, sum, from);
            } else {
                segment = warp_max_int(some);
                sum = -INFINITY;
            }
            const int v = segment * 32 + lane, at = begin + 4 * v - target.shift;
            double left[4] = {0.0, 0.0, 0.0, 0.0};
            if (v < target.vectors) {
                const float4 x = target.load(v), y = residual.minus ? draft.load(v, target.shift) : x;
                left[0] = residual.value(x.x, y.x, at);
                left[1] = residual.value(x.y, y.y, at + 1);
                left[2] = residual.value(x.z, y.z, at + 2);
                left[3] = residual.value(x.w, y.w, at + 3);
            }
            double up_to = left[0] + left[1] + left[2] + left[3];
            const double four = up_to;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double other = __shfl_up_sync(0xffffffffu, up_to, o);
                if (lane >= o) up_to += other;
            }
            sum += up_to - four;
            int index = -1, any = -1;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                sum += left[u];
                if (left[u] > 0.0) {
                    any = at + u;
                    if (index < 0 && sum > wanted) index = at + u;
                }
            }
            const unsigned hit = __ballot_sync(0xffffffffu, index >= 0);
            index = hit ? __shfl_sync(0xffffffffu, index, __ffs(hit) - 1) : warp_max_int(any);
            if (lane == 0) p.next[s] = index;
        }
        cluster_sync_all();   // the peers have read this CTA's total
    }
    if (part == 0 && thread == 0) {
        p.accepted[s] = row - first;
        advance_slot(p, s, row - first + 1);
    }
}

// Temperature 0: a warp per sequence.
__global__ void __launch_bounds__(128) verify_greedy_kernel(const VerifyParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int s = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (s >= p.rows.sequences) return;
    const int first = __ldg(p.rows.first + s), last = __ldg(p.rows.first + s + 1) - 1;
    int stop = last, token = -1;
    for (int base = first; base <= last; base += 32) {
        const int row = base + lane;
        Candidate best{-INFINITY, INT32_MAX};
        if (row <= last)
            for (int c = 0; c < p.parts; ++c) {
                const Candidate other = p.best[static_cast<int64_t>(row) * p.parts + c];
                if (preferred(other, best)) best = other;
            }
        const bool stops = row == last || (row < last && __ldg(p.ids + row + 1) != best.index);
        const unsigned found = __ballot_sync(0xffffffffu, stops);
        if (found) {
            const int from = __ffs(found) - 1;
            stop = base + from;
            token = __shfl_sync(0xffffffffu, best.index, from);
            break;
        }
    }
    if (lane == 0) {
        p.accepted[s] = last < first ? 0 : stop - first;
        p.next[s] = token;
        if (last >= first) advance_slot(p, s, stop - first + 1);
    }
}

// CTAs per row: parts that a CTA can hold, and more, of 2048 values at least, where there are fewer CTAs than wanted.  Parts of a size cost a cluster's launch and
// barriers each: a batch of 358 rows of 32000 takes 42 us with two parts per row, 50 with eight; 15 rows of 50257 take 18 us with four parts and 14 with eight.
int split_rows(int64_t vocab, int64_t rows, int64_t ctas) {
    constexpr int kLeast = 2048;
    int parts = 1;
    while (parts < kVerifyMostParts && (vocab > static_cast<int64_t>(parts) * (4 * kTileVectors - 8) || (rows * parts < ctas && vocab >= 2 * parts * kLeast))) parts *= 2;
    return parts;
}
// Shared memory of the drawing kernel for a part of `chunk` values.
size_t segment_bytes(int chunk) { return static_cast<size_t>((chunk + 3) / 4 + 1 + 31) / 32 * sizeof(double); }
int chunk_of(int vocab, int parts) { return ((vocab + parts - 1) / parts + 3) / 4 * 4; }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" size_t b200_verify_scratch_bytes(const b200_verify_args* a, const b200_rows* pass) {
    if (!a || !pass || pass->rows <= 0 || a->vocab <= 0) return 0;
    const size_t units = 2 * static_cast<size_t>(pass->rows);
    return units * kVerifyMostParts * sizeof(double) + units * sizeof(float) + 256;
}

extern "C" int b200_verify_drafts(const b200_verify_args* a, const b200_rows* pass, void* scratch, size_t scratch_bytes, void* stream) {
    VerifyParams p{};
    if (!rows_view(pass, p.rows)) return B200_BAD_ARGUMENT;
    if (!a || !a->logits || !a->ids || !a->accepted || !a->next || a->vocab <= 0 || !std::isfinite(a->temperature) || a->temperature < 0.0
        || (a->stride && a->stride < a->vocab) || (a->temperature > 0.0 && (!a->accept || !a->draw))) {
        set_error("b200_verify_drafts: bad pointer, size or temperature");
        return B200_BAD_ARGUMENT;
    }
    const float inverse = a->temperature > 0.0 ? static_cast<float>(1.0 / a->temperature) : 1.0f;
    if (!std::isfinite(inverse) || inverse == 0.0f) { set_error("b200_verify_drafts: temperature %g is out of range", a->temperature); return B200_BAD_ARGUMENT; }
    if (a->vocab > kVerifyMostVocab) { set_error("b200_verify_drafts: more than 2^23 values per row are not supported"); return B200_UNSUPPORTED; }
    const size_t need = b200_verify_scratch_bytes(a, pass);
    if (!scratch || scratch_bytes < need || reinterpret_cast<uintptr_t>(scratch) % 8) {
        set_error("b200_verify_drafts: scratch of %zu bytes on an 8-byte boundary needed, %zu given", need, scratch_bytes);
        return B200_BAD_ARGUMENT;
    }
    const bool greedy = a->temperature == 0.0;
    p.logits = a->logits; p.draft = greedy ? nullptr : a->draft_logits; p.stride = a->stride ? a->stride : a->vocab;
    p.vocab = static_cast<int>(a->vocab);
    p.parts = split_rows(p.vocab, static_cast<int64_t>(p.rows.rows) * (p.draft ? 2 : 1), 2 * 148);
    p.chunk = chunk_of(p.vocab, p.parts);
    p.draw_parts = split_rows(p.vocab, p.rows.sequences, 4 * 148);
    p.draw_chunk = chunk_of(p.vocab, p.draw_parts);
    p.inverse = inverse; p.ids = a->ids; p.accept = a->accept; p.draw = a->draw; p.accepted = a->accepted; p.next = a->next; p.advance = a->advance != 0;
    const size_t units = 2 * static_cast<size_t>(p.rows.rows);
    p.row_sum = static_cast<double*>(scratch);
    p.best = static_cast<Candidate*>(scratch);
    p.row_max = reinterpret_cast<float*>(p.row_sum + units * kVerifyMostParts);
    cudaStream_t st = as_stream(stream);
    const int64_t ctas = static_cast<int64_t>(p.rows.rows) * (p.draft ? 2 : 1) * p.parts;
    if (ctas > INT32_MAX) { set_error("b200_verify_drafts: too many rows"); return B200_UNSUPPORTED; }
    if (greedy) {
        const int status = cuda_status(launch_dependent(verify_best_kernel, dim3(static_cast<unsigned>(ctas)), dim3(kVerifyThreads), 0, st, p), "verify_best_kernel launch");
        if (status != B200_OK) return status;
        return cuda_status(launch_dependent(verify_greedy_kernel, dim3(static_cast<unsigned>((p.rows.sequences + 3) / 4)), dim3(128), 0, st, p),
                           "verify_greedy_kernel launch");
    }
    int device = 0;
    B200_CUDA(cudaGetDevice(&device));
    p.status = device_status_word(device);
    if (!p.status) { set_error("b200_verify_drafts: the device status word could not be allocated"); return B200_NO_DEVICE; }
    const size_t held = static_cast<size_t>(std::min((p.chunk + 6) / 4, kTileVectors)) * 16;
    B200_CUDA(cudaFuncSetAttribute(verify_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileVectors * 16));
    const int status = cuda_status(launch_dependent_cluster(verify_rows_kernel, dim3(static_cast<unsigned>(ctas)), dim3(kRowThreads), held, st,
                                                            dim3(static_cast<unsigned>(p.parts), 1, 1), p), "verify_rows_kernel launch");
    if (status != B200_OK) return status;
    const size_t smem = segment_bytes(p.draw_chunk);
    // the same limit for all vocabularies: a call beside this one may be between setting it and launching
    if (smem > 48 * 1024) B200_CUDA(cudaFuncSetAttribute(verify_finish_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(segment_bytes(kVerifyMostVocab / kVerifyMostParts))));
    return cuda_status(launch_dependent_cluster(verify_finish_kernel, dim3(static_cast<unsigned>(p.rows.sequences * p.draw_parts)), dim3(kVerifyThreads), smem, st,
                                                dim3(static_cast<unsigned>(p.draw_parts), 1, 1), p), "verify_finish_kernel launch");
}
