// The two kernels of the attention over a paged cache.  Both leave partial tiles in scratch: two places for each of their pieces
// (part_floats numbers each), then a PagedCut for each piece.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>

namespace ftb {
struct PagedAttn;

// Shared memory of an SM for the kernel for few rows and the joining one: the same for both, since another division waits for the SM
// to be empty.
constexpr int kPagedCarveout = 76 * 1024;

// Few rows (paged_short.cu): tiles of 8 or 16.
int paged_short_pieces(int rows);
int paged_short_launch(const PagedAttn& a, int d, int dtype, int rows, void* scratch, cudaStream_t stream);

// Many rows (paged_tile.cu): tiles of 128 or 256.
int paged_tile_pieces();
int paged_tile_launch(const PagedAttn& a, int d, int dtype, int rows, void* scratch, cudaStream_t stream);
}  // namespace ftb
