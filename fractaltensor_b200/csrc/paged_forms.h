// The two kernels of the attention over a paged cache.  Both leave partial tiles in scratch: two places for each of their pieces
// (part_floats numbers each), then a PagedCut for each piece.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <cstdlib>

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

// Whether n numbers at o (16 bits) meet the numbers of some of T rows of heads at q.
inline bool over_rows(const void* o, long long n, const void* q, int T, long long q_row, int heads, long long q_head, long long d) {
  const long long span = (heads - 1) * q_head, lo = std::min(0ll, span), hi = std::max(0ll, span) + d;  // of a row
  const long long step = T > 1 ? std::abs(q_row) : 0, first = T > 1 && q_row < 0 ? (T - 1) * q_row : 0;
  // o's beginning, in numbers from where the lowest row is (both on 2-byte boundaries)
  const long long at = static_cast<long long>(reinterpret_cast<uintptr_t>(o) - reinterpret_cast<uintptr_t>(q)) / 2 - first;
  if (step == 0) return at < hi && at + n > lo;
  // rows r with r * step + hi > at and r * step + lo < at + n
  auto floor_div = [](long long x, long long y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
  const long long r0 = std::max(0ll, floor_div(at - hi, step) + 1), r1 = std::min(T - 1ll, floor_div(at + n - lo - 1, step));
  return r0 <= r1;
}
}  // namespace ftb
