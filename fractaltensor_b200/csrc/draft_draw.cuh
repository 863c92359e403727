// A token drawn from a row of weights by a random number, by a CTA or a cluster of them: the first j with w_0 + .. + w_j > share * sum(w).
//
// Sums are kept in 64 bits: the chosen index follows from a comparison with a partial sum of up to V numbers, and in 32 bits the order
// of summation would decide it.  Every warp takes a stretch of the row: one pass for the stretches' sums, which the CTAs hand
// each other through distributed shared memory, and a second look at the one stretch (a 64th of the row or less) in which the limit is passed.
#pragma once
#include <climits>

#include "ptx.cuh"

namespace ftb {

// What is not positive and finite counts as 0, in the target's rows and in the draft's.
__device__ __forceinline__ double probability(float x) {
  x = fmaxf(x, 0.f);  // (0 of a NaN)
  return static_cast<double>(x < __int_as_float(0x7f800000) ? x : 0.f);
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
  double x;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(x) : "r"(addr) : "memory");
  return x;
}

template <int C, int kThreads>
struct DrawRoom {  // in shared memory
  double sums[kThreads / 32], totals[2];  // of the warps; of this CTA (in the two tries)
  double total[C];
  int found, heavy;
};

// The row: row.p(j) and row.q(j) load what row.weight(p, q, j) takes; a warp says row.look(j, n) before it weighs numbers of j .. j + n - 1;
// row.all() stops leaving out what it leaves out, for the case that nothing else weighs anything.  C: CTAs of a cluster; kAhead: the next numbers are on their way while
// some are weighed.  All threads; *share is read when it is needed (a register pair less while the row is read); one thread of one of the CTAs says put(token); -> sum(w),
// where it is 0 nothing is put.  A cluster meets once more before one of its CTAs leaves.
template <int C, int kThreads, bool kAhead, typename Row, typename Put>
__device__ __forceinline__ double draw_token(Row& row, int V, const float* share, int rank, DrawRoom<C, kThreads>& room, Put put) {
  constexpr int kWarps = kThreads / 32, kUnroll = 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // a warp's stretch of the row: whole groups of 32
  const int stretch = ((V + C * kThreads - 1) / (C * kThreads)) * 32;
  const int from = static_cast<int>(min(static_cast<long long>(V), static_cast<long long>(rank * kWarps + warp) * stretch)), to = min(V, from + stretch);
  double total = 0.0, before = 0.0;  // of the row; of the CTAs in front of this one
  for (int tries = 0; tries < 2; ++tries) {  // where p and q are the same, nothing is left of the difference: p itself
    double s = 0.0;
    float pv[kUnroll], qv[kUnroll];
    auto load = [&](int j) {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int at = j + k * 32 + lane;
        pv[k] = at < to ? row.p(at) : 0.f;
        qv[k] = at < to ? row.q(at) : 0.f;
      }
    };
    if (kAhead) load(from);
    for (int j = from; j < to; j += 32 * kUnroll) {
      float p[kUnroll], q[kUnroll];
      if (!kAhead) load(j);
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        p[k] = pv[k];
        q[k] = qv[k];
      }
      if (kAhead) load(j + 32 * kUnroll);
      row.look(j, 32 * kUnroll);
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) s += row.weight(p[k], q[k], j + k * 32 + lane);
    }
    s = warp_sum(s);
    if (lane == 0) room.sums[warp] = s;
    __syncthreads();
    double cta = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) cta += room.sums[w];
    if constexpr (C == 1) {
      total = cta;
      __syncthreads();
    } else {
      if (threadIdx.x == 0) room.totals[tries] = cta;
      cluster_sync_all();
      if (threadIdx.x < C) room.total[threadIdx.x] = ld_cluster_f64(map_to_cta(smem_u32(&room.totals[tries]), threadIdx.x));
      __syncthreads();
      total = before = 0.0;
#pragma unroll
      for (int r = 0; r < C; ++r) {
        if (r < rank) before += room.total[r];
        total += room.total[r];
      }
    }
    if (total > 0.0) break;
    row.all();
  }
  // The stretch in which the limit is passed: room.sums[] are this CTA's still.  (u of 1 or above, or sums that round down: the last
  // stretch that weighs anything.)
  const double limit = static_cast<double>(*share) * total;
  // Which CTA has it follows from the CTAs' sums alone, the same in all of them.
  const bool passed = total > limit;
  bool past = false, own = C == 1;
  if constexpr (C > 1) {
    double at = 0.0;
    int weighs = -1;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      at += room.total[r];
      if (passed && !past && at > limit) {
        past = true;
        own = r == rank;
      }
      if (room.total[r] > 0.0) weighs = r;
    }
    if (!passed) own = weighs == rank;
  }
  int first = -1, last = -1;
  double in_front = before, begin = before;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (first < 0 && begin + room.sums[w] > limit) {
      first = w;
      in_front = begin;
    }
    begin += room.sums[w];
    if (room.sums[w] > 0.0) last = w;
  }
  const bool heaviest = !passed || first < 0;  // (sums that round differently: the last one too)
  if (heaviest) first = last;
  // That stretch again, by all warps of the CTA, kUnroll numbers side by side a lane: one scan over the warps' sums for
  // kThreads * kUnroll of them.
  if (own && total > 0.0) {  // of all CTAs, one
    const int begin_at = static_cast<int>(min(static_cast<long long>(V), static_cast<long long>(rank * kWarps + first) * stretch)), end_at = min(V, begin_at + stretch);
    int found = INT_MAX, heavy = -1;
    double run = in_front;
    for (int j0 = begin_at; j0 < end_at && found == INT_MAX; j0 += kThreads * kUnroll) {
      const int j = j0 + static_cast<int>(threadIdx.x) * kUnroll;
      double w[kUnroll], sum = 0.0;
      float pv[kUnroll], qv[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        pv[k] = j + k < end_at ? row.p(j + k) : 0.f;
        qv[k] = j + k < end_at ? row.q(j + k) : 0.f;
      }
      row.look(j - lane * kUnroll, 32 * kUnroll);
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        w[k] = row.weight(pv[k], qv[k], j + k);
        sum += w[k];
      }
      double ends = sum;  // sum of the warp's lanes up to this one
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, ends, o);
        if (lane >= o) ends += y;
      }
      const double begins = __shfl_up_sync(0xffffffffu, ends, 1);
      __syncthreads();  // (sums, room.found and room.heavy have been read)
      if (lane == 31) room.sums[warp] = ends;
      if (threadIdx.x == 0) {
        room.found = INT_MAX;
        room.heavy = -1;
      }
      __syncthreads();
      double upto = run + (lane > 0 ? begins : 0.0);
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        if (v < warp) upto += room.sums[v];
        run += room.sums[v];
      }
      int here_found = INT_MAX, here_heavy = -1;
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        upto += w[k];
        if (w[k] > 0.0) {
          if (here_found == INT_MAX && !heaviest && upto > limit) here_found = j + k;
          here_heavy = j + k;
        }
      }
      here_found = __reduce_min_sync(0xffffffffu, here_found);
      here_heavy = __reduce_max_sync(0xffffffffu, here_heavy);
      if (lane == 0) {
        if (here_found != INT_MAX) atomicMin(&room.found, here_found);
        if (here_heavy >= 0) atomicMax(&room.heavy, here_heavy);
      }
      __syncthreads();
      found = room.found;
      if (room.heavy >= 0) heavy = room.heavy;
    }
    if (threadIdx.x == 0) put(found != INT_MAX ? found : heavy);
  }
  return total;
}

}  // namespace ftb
