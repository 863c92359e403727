// What the two kernels that add up attention weight over a paged cache share.
#pragma once
#include "paged_work.cuh"

namespace ftb {

struct Weigh {
  PagedAttn attn;  // (without results)
  float* weights;  // [pages, kv_heads, page_size]
  const float* lse;
};

// Sequences with few rows (paged_weigh.cu), many rows (paged_weigh_tile.cu); the latter with scratch memory.
size_t paged_weigh_tile_scratch(int T, int kv_heads, int group, int d);
int paged_weigh_tile_launch(const Weigh& x, int d, int dtype, void* scratch, cudaStream_t stream);

// The keys that some row of a sequence sees.
__device__ __forceinline__ PagedKeys all_keys(const PagedAttn& a, const PagedSeq& s) {
  return s.flats > 0 ? keys_of_rows(a, s.pos0, s.first, s.hi, 0, s.flats) : PagedKeys{0, 0};
}
// Blocks of n of them.
template <int kBlockKeys>
__device__ __forceinline__ int blocks_of(const PagedKeys& k) {
  return k.hi > k.lo ? (k.hi + kBlockKeys - 1) / kBlockKeys - k.lo / kBlockKeys : 0;
}

}  // namespace ftb
