// Attention over a paged cache for few rows (paged_short.cu); nt: rows of a tile / 8, 1 or 2.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>

namespace ftb {
struct PagedAttn;
size_t paged_short_scratch_bytes(int nt, int d);
int paged_short_launch(const PagedAttn& a, int d, int dtype, int nt, float* parts, cudaStream_t stream);
}  // namespace ftb
