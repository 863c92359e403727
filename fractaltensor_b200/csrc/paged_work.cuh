// How the attention kernels over a paged cache share out their work.
//
// A tile is up to R rows (token, head of a group) of one sequence and kv head; its cost is the number of units of kUnitKeys
// keys that it walks.  The units of all tiles, in the order sequence, kv head, tile, form one line that is cut into as many
// equal pieces as there are CTAs: ragged batches and single long sequences fill the device alike, and nothing about the
// lengths has to be known on the host, so that a captured call follows them.  A tile that a cut goes through leaves
// partial results (out of 32-bit sums, with the maximum that they refer to), which a second kernel joins in the order of the pieces:
// the same bits from call to call.
#pragma once
#include "paged_attn.cuh"

namespace ftb {

struct PagedSeq {
  long long pos0;  // position of row t: pos0 + t
  int first, n;    // rows
  int tiles, lo, hi, units;  // tiles of a kv head; keys lo .. hi - 1 are seen by some row; units of a tile
};

template <int R, int kUnitKeys>
__device__ __forceinline__ PagedSeq paged_sequence(const PagedAttn& a, int b) {
  PagedSeq s;
  const int end = a.batch.starts[b + 1];
  s.first = max(0, a.batch.starts[b]);
  s.n = min(end, a.T) - s.first;
  s.pos0 = static_cast<long long>(a.batch.lens[b]) - end;
  s.tiles = s.units = s.lo = s.hi = 0;
  if (s.n <= 0 || s.first >= a.T) return s;
  const long long room = static_cast<long long>(a.batch.W) << a.batch.page_shift;
  const long long last = s.pos0 + s.first + s.n - 1;
  if (last >= room) atomicCAS(a.status, 0, FTB_ERR_INDEX);  // a table too narrow for the length
  s.hi = static_cast<int>(max(0ll, min(min(last + 1, room), 0x7fffff00ll)));
  if (a.window > 0) s.lo = static_cast<int>(max(0ll, min(s.pos0 + s.first - a.window + 1, static_cast<long long>(s.hi))));
  s.tiles = static_cast<int>((static_cast<long long>(s.n) * a.group + R - 1) / R);
  s.units = s.hi > s.lo ? (s.hi + kUnitKeys - 1) / kUnitKeys - s.lo / kUnitKeys : 1;  // (1: zeros have to be written)
  return s;
}

// The line of all units, and where sequence `seq` begins on it.
struct PagedLine {
  long long total;
  int pieces;
};
constexpr int kLineThreads = 128;

__device__ __forceinline__ long long piece_begin(const PagedLine& line, int g) {
  return line.total / line.pieces * g + line.total % line.pieces * g / line.pieces;
}

// All kLineThreads threads of a block: the line's length, and the sequence that unit piece_begin(line, g) belongs to with that
// sequence's beginning.  at_least: units of a piece where there are few.
template <int R, int kUnitKeys>
__device__ __forceinline__ PagedLine paged_line(const PagedAttn& a, int g, int most_pieces, int at_least, int* seq, long long* begin) {
  __shared__ long long s_sum[kLineThreads / 32];
  __shared__ long long s_begin;
  __shared__ int s_seq;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.batch.B + kLineThreads - 1) / kLineThreads;
  const int b0 = min(a.batch.B, tid * per), b1 = min(a.batch.B, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const PagedSeq s = paged_sequence<R, kUnitKeys>(a, b);
    mine += static_cast<long long>(s.tiles) * a.kv_heads * s.units;
  }
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  if (lane == 31) s_sum[warp] = sum;
  if (tid == 0) s_seq = a.batch.B;
  __syncthreads();
  long long before = 0;
  PagedLine line{0, 1};
#pragma unroll
  for (int w = 0; w < kLineThreads / 32; ++w) {
    if (w < warp) before += s_sum[w];
    line.total += s_sum[w];
  }
  line.pieces = static_cast<int>(max(1ll, min(static_cast<long long>(most_pieces), line.total / at_least)));
  long long at = before + sum - mine;
  if (g < line.pieces) {
    const long long u = piece_begin(line, g);
    if (u >= at && u < at + mine) {
      for (int b = b0; b < b1; ++b) {
        const PagedSeq s = paged_sequence<R, kUnitKeys>(a, b);
        const long long c = static_cast<long long>(s.tiles) * a.kv_heads * s.units;
        if (u < at + c) {
          s_seq = b;
          s_begin = at;
          break;
        }
        at += c;
      }
    }
  }
  __syncthreads();
  *seq = s_seq;
  *begin = s_begin;
  return line;
}

}  // namespace ftb
