// Host side of the tcgen05 kernel for shared prefixes.
#pragma once

#include "prefix.cuh"

namespace b200 {

constexpr int kTensorRows = 256, kTensorKeys = 128;   // (row, head) pairs of a CTA, keys of a step

// Whether the kernel can take a prefix (16-byte aligned pools).
bool prefix_tensor_takes(const b200_kv_pages& prefix, float scale);
// Items of the prefix alone; p.prefix_rows is kTensorRows.
int launch_prefix_tensor(const PrefixParams& p, int items, cudaStream_t stream);

}  // namespace b200
