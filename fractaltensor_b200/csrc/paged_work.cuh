// How the attention kernels over a paged cache share out their work.
//
// A tile is up to R rows (token, head of a group) of one sequence and kv head; its cost is the number of units of
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
  int flats;       // rows (token, head of the group) of a kv head; 0: not this launch's
  int hi;          // keys 0 .. hi - 1 are seen by some row
};

__device__ __forceinline__ PagedSeq paged_sequence(const PagedAttn& a, int b) {
  PagedSeq s;
  const int end = a.batch.starts[b + 1];
  s.first = max(0, a.batch.starts[b]);
  s.n = min(end, a.T) - s.first;
  s.pos0 = static_cast<long long>(a.batch.lens[b]) - end;
  s.flats = s.hi = 0;
  if (s.n <= 0 || s.first >= a.T) return s;
  const int flats = s.n * a.group;  // T * group fits
  if (flats < a.least_rows || flats > a.most_rows) return s;
  s.flats = flats;
  const long long room = static_cast<long long>(a.batch.W) << a.batch.page_shift;
  const long long last = s.pos0 + s.first + s.n - 1;
  if (last >= room) atomicCAS(a.status, 0, FTB_ERR_INDEX);  // a table too narrow for the length
  s.hi = static_cast<int>(max(0ll, min(min(last + 1, room), 0x7fffff00ll)));
  return s;
}

// Rows flat0 .. + rows - 1 of a kv head: the keys that some of them see, lo .. hi - 1.
struct PagedKeys {
  int lo, hi;
};
__device__ __forceinline__ PagedKeys keys_of_rows(const PagedAttn& a, long long pos0, int first, int hi_all, int flat0, int rows) {
  const long long first_pos = pos0 + first + flat0 / a.group, last_pos = pos0 + first + (flat0 + rows - 1) / a.group;
  PagedKeys k;
  k.hi = static_cast<int>(min(static_cast<long long>(hi_all), max(0ll, last_pos + 1)));
  k.lo = a.window > 0 ? static_cast<int>(min(static_cast<long long>(k.hi), max(0ll, first_pos - a.window + 1))) : 0;
  return k;
}
// Units of kUnitKeys that a walk over them takes; a tile without keys costs one (zeros have to be written).
template <int kUnitKeys>
__device__ __forceinline__ int units_of(const PagedKeys& k) {
  return k.hi > k.lo ? (k.hi + kUnitKeys - 1) / kUnitKeys - k.lo / kUnitKeys : 1;
}
// The line's share of a sequence: tiles of R rows.
template <int R, int kUnitKeys>
__device__ __forceinline__ long long units_of_head(const PagedAttn& a, const PagedSeq& s) {
  long long sum = 0;
  for (int flat0 = 0; flat0 < s.flats; flat0 += R)
    sum += units_of<kUnitKeys>(keys_of_rows(a, s.pos0, s.first, s.hi, flat0, min(R, s.flats - flat0)));
  return sum;
}

struct PagedLine {
  long long total;
  int pieces;
};
constexpr int kLineThreads = 128;
struct PagedLineRoom {  // in shared memory
  long long sum[kLineThreads / 32], begin;
  int seq;
};

__device__ __forceinline__ long long piece_begin(const PagedLine& line, int g) {
  return line.total / line.pieces * g + line.total % line.pieces * g / line.pieces;
}

// All threads of a block, kLineThreads or more: the line, and the sequence that the first unit of piece g belongs to (B: none)
// with that sequence's beginning.  at_least: units of a piece where there are few.
template <int R, int kUnitKeys>
__device__ __forceinline__ PagedLine paged_line(const PagedAttn& a, int g, int most_pieces, int at_least, PagedLineRoom& room, int* seq, long long* begin) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.batch.B + kLineThreads - 1) / kLineThreads;
  const int b0 = min(a.batch.B, tid * per), b1 = tid < kLineThreads ? min(a.batch.B, b0 + per) : b0;
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += units_of_head<R, kUnitKeys>(a, paged_sequence(a, b)) * a.kv_heads;
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  if (lane == 31 && tid < kLineThreads) room.sum[warp] = sum;
  if (tid == 0) {
    room.seq = a.batch.B;
    room.begin = 0;
  }
  __syncthreads();
  long long before = 0;
  PagedLine line{0, 1};
#pragma unroll
  for (int w = 0; w < kLineThreads / 32; ++w) {
    if (w < warp) before += room.sum[w];
    line.total += room.sum[w];
  }
  line.pieces = static_cast<int>(max(1ll, min(static_cast<long long>(most_pieces), line.total / at_least)));
  if (mine > 0 && g < line.pieces) {
    const long long u = piece_begin(line, g);
    long long at = before + sum - mine;
    if (u >= at && u < at + mine) {
      for (int b = b0; b < b1; ++b) {
        const long long c = units_of_head<R, kUnitKeys>(a, paged_sequence(a, b)) * a.kv_heads;
        if (u < at + c) {
          room.seq = b;
          room.begin = at;
          break;
        }
        at += c;
      }
    }
  }
  __syncthreads();
  *seq = room.seq;
  *begin = room.begin;
  return line;
}

// A stretch of a tile that a piece works on: units r0 .. r1 - 1 of its `units`.
struct PagedTile {
  int b, h, flat0, rows;
  PagedKeys keys;
  int units, r0, r1;
  long long begin;  // of the tile on the line
};

// Walks the tiles of a piece in their order.
template <int R, int kUnitKeys>
struct PagedWalk {
  PagedLine line;
  long long u, u_end, at, per;  // at: the sequence's beginning, per: units of one of its kv heads
  int b;
  PagedSeq s;

  __device__ __forceinline__ void begin(const PagedAttn& a, const PagedLine& line_, int piece, int seq, long long seq_begin) {
    line = line_;
    u = piece_begin(line, piece);
    u_end = piece_begin(line, piece + 1);
    b = seq;
    at = seq_begin;
    per = 0;
    if (u < u_end && b < a.batch.B) {
      s = paged_sequence(a, b);
      per = units_of_head<R, kUnitKeys>(a, s);
    } else {
      u = u_end;
    }
  }
  __device__ __forceinline__ bool more() const { return u < u_end; }
  // The tile that unit u is in, as far as the piece has it; moves on behind it.
  __device__ __forceinline__ PagedTile next(const PagedAttn& a) {
    while (u >= at + per * a.kv_heads) {
      at += per * a.kv_heads;
      s = paged_sequence(a, ++b);
      per = units_of_head<R, kUnitKeys>(a, s);
    }
    PagedTile t;
    t.b = b;
    t.h = static_cast<int>((u - at) / per);
    t.begin = at + per * t.h;
    for (t.flat0 = 0;; t.flat0 += R) {
      t.rows = min(R, s.flats - t.flat0);
      t.keys = keys_of_rows(a, s.pos0, s.first, s.hi, t.flat0, t.rows);
      t.units = units_of<kUnitKeys>(t.keys);
      if (u < t.begin + t.units) break;
      t.begin += t.units;
    }
    t.r0 = static_cast<int>(u - t.begin);
    t.r1 = static_cast<int>(min(static_cast<long long>(t.units), u_end - t.begin));
    u = t.begin + t.r1;
    return t;
  }
};

// What joins the parts of a tile: left by the piece behind the first cut in it; `last` is the last piece that has a part.
struct PagedCut {
  int last;  // -1: nothing to join
  int b, first, flat0, rows, h, lo, hi;
  long long pos0;
};

// Whether cut `piece`, in front of that piece, is the first one in the tile, and the last piece with a part of it.
__device__ __forceinline__ int last_piece_of(const PagedLine& line, int piece, const PagedTile& t) {
  if (t.r0 == 0 || piece_begin(line, piece - 1) > t.begin) return -1;
  int last = piece;
  while (last + 1 < line.pieces && piece_begin(line, last + 1) < t.begin + t.units) ++last;
  return last;
}

// Parts: each piece has two places, for the end of a tile that began in front of it and for the beginning of one that ends behind
// it; a place is [R, d] sums and [R] pairs (maximum, sum of the weights).
template <int R, int D>
__host__ __device__ constexpr size_t part_floats() { return static_cast<size_t>(R) * (D + 2); }

// A piece without empties: line.total >= pieces * at_least, so that piece_begin grows from piece to piece.

}  // namespace ftb
