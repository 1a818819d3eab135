// Host side of the tcgen05 kernel for shared prefixes.
#pragma once

#include "prefix.cuh"

namespace b200 {

constexpr int kTensorRows = 256, kTensorKeys = 64;   // (row, head) pairs of a CTA, keys of a step

// Rows of a TMA box of a page: a part of it of at most 64 rows, at least 8; 0 where there is none.
int page_box_rows(int page_size);
// Tensor maps of the keys and the values: rows of a page's head in blocks of 64 values, box_rows at a time - one block, or, where boxes have 64 rows and
// whole blocks make up the row, all of them at once.
int page_maps(const PagesView& pages, int box_rows, CUtensorMap* maps);
__host__ __device__ inline int boxes_per_row(int box_rows, int dim) { return box_rows == 64 && dim % 64 == 0 ? 1 : (dim + 63) / 64; }

// Items of the prefix alone, of pages that prefix_mma_kernel takes; p.prefix_rows is kTensorRows.
int launch_prefix_tensor(const PrefixParams& p, int items, cudaStream_t stream);

}  // namespace b200
