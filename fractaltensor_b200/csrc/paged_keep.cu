// Which keys of a paged cache stay, and the moves of their rows.
//
// paged_choose: of a sequence of more than `keep` keys the last `recent` and, of those in front, the keep - recent with the largest
// weights stay, of equal weights those in front; for each kv head on its own.  The weight of the last one that stays is found digit by digit
// (radix selection on the weights' bits, put in the order of the numbers): a histogram of eight bits of what agrees with the digits
// so far, four times, then the positions in their order by counts of what lies in front.
//
// paged_move: row first + kept[i] goes to first + i, i < counts, of keys, values, exponents and weights.  Into other pages every step of rows
// is on its own.  In the same pages a chain of steps is one CTA's: kept ascends, so that kept[i] >= i, and what a step writes (up to
// row i) is never read by a later one (kept[j] > kept[i] >= i); within a step all rows are read before one is written.  Chains run side
// by side for the pieces of a row, which do not meet, and where there are few, a cluster of CTAs takes a step together.
//
// 48 sequences of 1500 to 9000 keys of 16 bits, 8 kv heads of 128, to 2048 of them in other pages: 156.8 us (194 with a table for 131 072 keys, whose room leaves one CTA an SM to the choice), of which the moves, bound by memory, are 131
// (6.2 TB/s) and the choice 26, trips and digits one behind the other.  One of 100 001 keys of 8 bits, 4 kv heads, to 8192 in its own pages 23.5 to 24.7 us
// (372 with chains of single CTAs that looked rows up one behind the other).  Its choice
// is bound by instructions, some 20 a key and digit, and by a cluster's barriers, 1 us each.  The paths of 128 trees 3.5 us, a launch.  Measured and not kept: lanes with
// the same digit adding as one (30 for 28 us), a bin for every second lane (31 for 28).
#include <algorithm>
#include <climits>

#include "../../include/ftb200.h"
#include "paged.cuh"
#include "tmap.h"

namespace ftb {
namespace {

// --------------------------------------------------------------------------------------------- choice
struct Choose {
  PagedBatch batch;
  const float* weights;  // [pages, kv_heads, page_size]
  int* kept;             // [B, kv_heads, keep]
  int* lens_out;
  int kv_heads, keep, recent;
  int* status;
};

constexpr int kBins = 256, kCopies = 4;

// Unsigned numbers in the order of the weights; NaN is below all of them.
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);  // (-0 is 0)
  if (w != w) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
  int x;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
  return x;
}

// C CTAs for each sequence and kv head, a stretch of the keys each, of which `room` stay in shared memory after they have been read.
template <int C, int kThreads>
__global__ void __launch_bounds__(kThreads, C == 1 ? 3 : 1)
paged_choose_kernel(const __grid_constant__ Choose a, int room) {
  constexpr int kWarps = kThreads / 32, kSweep = 4, kChooseAtOnce = C > 1 ? 8 : 4;  // (the last: 8 for one CTA 161 us for 159.6, 4 for a cluster 42 for 28)
  extern __shared__ uint32_t known_keys[];
  __shared__ int bins[2][kCopies][kBins], sums[2][kBins], above_of[kWarps], equal_of[kWarps], mine[2], of_warp[kBins / 32];
  __shared__ int s_digit, s_left, s_all;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0, head = blockIdx.x / C;
  const int b = head / a.kv_heads, h = head - b * a.kv_heads;
  grid_launch_dependents();
  grid_dependency_wait();
  const int asked = max(0, a.batch.lens[b]), L = static_cast<int>(min(static_cast<long long>(a.batch.W) << a.batch.page_shift, static_cast<long long>(asked)));
  if (threadIdx.x == 0 && rank == 0 && h == 0) {
    if (asked > L) atomicCAS(a.status, 0, FTB_ERR_INDEX);  // a table too narrow for the length
    a.lens_out[b] = min(L, a.keep);
  }
  int* kept = a.kept + static_cast<long long>(head) * a.keep;
  const int at = rank * kThreads + threadIdx.x;
  if (L <= a.keep) {
    for (int i = at; i < a.keep; i += C * kThreads) kept[i] = i < L ? i : -1;
    return;
  }
  const int old = L - a.recent, want = a.keep - a.recent;  // 0 <= want < old
  for (int i = at; i < a.recent; i += C * kThreads) kept[want + i] = old + i;
  if (want == 0) return;
  const int* table = a.batch.table + static_cast<long long>(b) * a.batch.W;
  const int shift = a.batch.page_shift, in_page = (1 << shift) - 1;
  auto key_at = [&](int i) -> uint32_t {
    const int page = table[i >> shift];
    if (page < 0 || page >= a.batch.pages) return 0u;  // (which is said where it is first read)
    return order_of(a.weights[(((static_cast<long long>(page) * a.kv_heads) + h) << shift) + (i & in_page)]);
  };
  // a warp's stretch: whole groups of 32
  const int stretch = (old + C * kThreads - 1) / (C * kThreads) * 32;
  const int from = static_cast<int>(min(static_cast<long long>(old), static_cast<long long>(rank * kWarps + warp) * stretch));
  const int to = static_cast<int>(min(static_cast<long long>(old), static_cast<long long>(from) + stretch));
  const int first = static_cast<int>(min(static_cast<long long>(old), static_cast<long long>(rank) * kWarps * stretch));  // of the CTA's
  // f(i, key) for this lane's keys and 0 behind them, all lanes of the warp at once; some of them loaded before one is looked at
  const int held = static_cast<int>(min(static_cast<long long>(to), static_cast<long long>(first) + room));
  auto each = [&](auto f) {
    int i0 = from;
    for (; i0 < held; i0 += 32 * kSweep) {
      uint32_t key[kSweep];
#pragma unroll
      for (int u = 0; u < kSweep; ++u) key[u] = i0 + u * 32 + lane < held ? known_keys[i0 + u * 32 + lane - first] : 0u;
      if (i0 + 32 * kSweep > held && held < to) break;  // (the others are not held)
#pragma unroll
      for (int u = 0; u < kSweep; ++u) f(i0 + u * 32 + lane, key[u]);
    }
    for (; i0 < to; i0 += 32) {
      const int i = i0 + lane;
      f(i, i < held ? known_keys[i - first] : i < to ? key_at(i) : 0u);
    }
  };
  uint32_t prefix = 0, known = 0;  // the digits so far, and which bits they are
  int left = want;
  bool all = false;  // whatever agrees with the digits stays
  for (int i = threadIdx.x; i < kCopies * kBins; i += kThreads) (&bins[0][0][0])[i] = 0;
  if (threadIdx.x == 0) s_digit = s_left = s_all = 0;
  __syncthreads();
  for (int d = 0; d < 4; ++d) {
    const int low = 24 - 8 * d;
    int* bin = bins[d & 1][warp % kCopies];
    for (int i = threadIdx.x; i < kCopies * kBins; i += kThreads) (&bins[(d & 1) ^ 1][0][0])[i] = 0;  // the next digit's
    if (d == 0) {
      for (int i0 = from; i0 < to; i0 += 32 * kChooseAtOnce) {
        int page[kChooseAtOnce];
        float w[kChooseAtOnce];
#pragma unroll
        for (int u = 0; u < kChooseAtOnce; ++u) {
          const int i = i0 + u * 32 + lane;
          page[u] = i < to ? table[i >> shift] : 0;
        }
#pragma unroll
        for (int u = 0; u < kChooseAtOnce; ++u) {  // (page 0 in a missing one's place, so that nothing stands between the loads)
          const int i = i0 + u * 32 + lane, there = page[u] >= 0 && page[u] < a.batch.pages ? page[u] : 0;
          w[u] = a.weights[(((static_cast<long long>(there) * a.kv_heads) + h) << shift) + (i & in_page)];
        }
#pragma unroll
        for (int u = 0; u < kChooseAtOnce; ++u) {
          const int i = i0 + u * 32 + lane;
          if (i >= to) continue;
          const bool there = page[u] >= 0 && page[u] < a.batch.pages;
          if (!there) atomicCAS(a.status, 0, FTB_ERR_INDEX);
          const uint32_t key = there ? order_of(w[u]) : 0u;
          if (i - first < room) known_keys[i - first] = key;
          atomicAdd(bin + (key >> low), 1);
        }
      }
    } else {
      each([&](int i, uint32_t key) {
        if (i < to && (key & known) == prefix) atomicAdd(bin + (key >> low & 255u), 1);
      });
    }
    __syncthreads();
    // thread i: bin 255 - i, and how many keys are in the bins above
    int* of_cta = sums[d & 1];  // (the other one may still be read by a CTA of the cluster)
    int count = 0, upto = 0;
    if (threadIdx.x < kBins) {
#pragma unroll
      for (int c = 0; c < kCopies; ++c) count += bins[d & 1][c][255 - threadIdx.x];
      of_cta[threadIdx.x] = count;
    }
    if constexpr (C > 1) {
      cluster_sync_all();
      if (threadIdx.x < kBins) {
        count = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) count += ld_cluster_s32(map_to_cta(smem_u32(&of_cta[threadIdx.x]), r));
      }
    }
    if (threadIdx.x < kBins) {
      upto = count;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (lane == 31) of_warp[warp] = upto;
    }
    __syncthreads();
    if (threadIdx.x < kBins) {
#pragma unroll
      for (int w = 0; w < kBins / 32; ++w) upto += w < warp ? of_warp[w] : 0;
      if (upto - count < left && upto >= left) {
        s_digit = 255 - threadIdx.x;
        s_left = left - (upto - count);
        s_all = upto == left;
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_digit) << low;
    known |= 255u << low;
    left = s_left;
    all = s_all != 0;
    if (all) break;  // mostly after three digits
  }
  // what is above stays, of what is equal the first `left`; where all of that stays, it counts as above
  const uint32_t least = all ? prefix : prefix + 1;
  int above = 0, equal = 0;
  if (all) {
    each([&](int i, uint32_t key) { above += i < to && (key & known) >= least; });
  } else {
    each([&](int i, uint32_t key) {
      above += i < to && key >= least;
      equal += i < to && key == prefix;
    });
  }
  above = __reduce_add_sync(0xffffffffu, above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) {
    above_of[warp] = above;
    equal_of[warp] = equal;
  }
  __syncthreads();
  const int its_above = lane < kWarps ? above_of[lane] : 0, its_equal = lane < kWarps ? equal_of[lane] : 0;
  above = __reduce_add_sync(0xffffffffu, lane < warp ? its_above : 0);  // in front of this warp's stretch
  equal = __reduce_add_sync(0xffffffffu, lane < warp ? its_equal : 0);
  if constexpr (C > 1) {
    if (warp == 0) {
      const int all_above = __reduce_add_sync(0xffffffffu, its_above), all_equal = __reduce_add_sync(0xffffffffu, its_equal);
      if (lane == 0) {
        mine[0] = all_above;
        mine[1] = all_equal;
      }
    }
    cluster_sync_all();
    above += __reduce_add_sync(0xffffffffu, lane < rank ? ld_cluster_s32(map_to_cta(smem_u32(&mine[0]), lane)) : 0);
    equal += __reduce_add_sync(0xffffffffu, lane < rank ? ld_cluster_s32(map_to_cta(smem_u32(&mine[1]), lane)) : 0);
  }
  // (weights that another stream changes meanwhile may give any counts: nothing is written behind the head's own)
  const unsigned in_front = (1u << lane) - 1u;
  if (all) {
    each([&](int i, uint32_t key) {
      const bool stays = i < to && (key & known) >= least;
      const unsigned those = __ballot_sync(0xffffffffu, stays);
      const unsigned to_at = above + __popc(those & in_front);
      if (stays && to_at < static_cast<unsigned>(want)) kept[to_at] = i;
      above += __popc(those);
    });
  } else {
    each([&](int i, uint32_t key) {
      const bool is_above = i < to && key >= least, is_equal = i < to && key == prefix;
      const unsigned those = __ballot_sync(0xffffffffu, is_above), equals = __ballot_sync(0xffffffffu, is_equal);
      const int before = equal + __popc(equals & in_front);
      const unsigned to_at = above + __popc(those & in_front) + min(left, before);
      if ((is_above || (is_equal && before < left)) && to_at < static_cast<unsigned>(want)) kept[to_at] = i;
      above += __popc(those);
      equal += __popc(equals);
    });
  }
  if constexpr (C > 1) cluster_sync_all();  // nobody leaves while its counts may be read
}

// ---------------------------------------------------------------------------------------------- moves
struct Move {
  PagedBatch batch;       // of what is read
  const int* into;        // the table of what is written, into_W wide
  int into_W;
  const int *kept, *counts, *first;  // first may be nullptr: 0
  long long kept_seq, kept_head;     // distances in numbers
  int most;               // rows of a sequence
  int kv_heads;
  unsigned char *k, *v, *k_exp, *v_exp;
  float* weights;
  int* status;
};

constexpr int kMostKept = 1 << 30;  // positions of a sequence: they are counted in 32 bits, some steps of all threads beyond the last one

constexpr int kMoveThreads = 256, kMoveAtOnce = 8, kMostRoom = 48 * 1024;

// Rows of cache planes that a kept row comes from and goes to; -1: none.
struct Rows {
  int from, to;
};
// The page at position pos of one of a sequence's tables as it stands there; -1 behind its width.
__device__ __forceinline__ int page_there(const int* table, int W, int shift, long long pos) {
  const long long i = pos >> shift;
  return i < W ? table[i] : -1;
}
__device__ __forceinline__ Rows rows_of(const Move& a, int h, int first, int k, int i, int from, int to) {
  const int shift = a.batch.page_shift, in_page = (1 << shift) - 1;
  const long long src = static_cast<long long>(first) + k, dst = static_cast<long long>(first) + i;
  if (src == dst && a.into == a.batch.table) return {-1, -1};  // where it is, page or not
  if (k < 0 || first < 0 || from < 0 || from >= a.batch.pages || to < 0 || to >= a.batch.pages) {
    atomicCAS(a.status, 0, FTB_ERR_INDEX);
    return {-1, -1};
  }
  return {((from * a.kv_heads + h) << shift) + static_cast<int>(src & in_page), ((to * a.kv_heads + h) << shift) + static_cast<int>(dst & in_page)};
}

// A chain is kChain threads': block (x, y, z) has the chains of sequences and kv heads 256 / kChain * x and on, part y of a row, every
// gridDim.z-th step of rows.  kRow: 16-byte pieces of a key or value, kOfPart: pieces of a part of both together; exponents and weights go with part 0.
// The rows of the next step are looked up while this one's are on their way.
// C: CTAs of a chain, a cluster, which take so many steps at once.
template <int kRow, int kOfPart, int kChain, int C>
__global__ void __launch_bounds__(kMoveThreads)
paged_move_kernel(const __grid_constant__ Move a, int chains) {
  constexpr int kTogether = kChain / kOfPart, kStep = kTogether * kMoveAtOnce, kBeside = (kStep + kChain - 1) / kChain;
  __shared__ Rows looked_up[kMoveThreads / kChain][2][kStep];
  const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int chain = blockIdx.x / C * (kMoveThreads / kChain) + threadIdx.x / kChain, tid = threadIdx.x % kChain, part = blockIdx.y;
  grid_launch_dependents();
  grid_dependency_wait();
  if (kChain < kMoveThreads && chain >= chains) return;  // (a warp leaves as one)
  const int b = chain / a.kv_heads, h = chain - b * a.kv_heads;
  const int n = min(max(a.counts[b], 0), a.most), first = a.first != nullptr ? a.first[b] : 0;
  const int* kept = a.kept + b * a.kept_seq + h * a.kept_head;
  auto meet = [] {
    if constexpr (C > 1) cluster_sync_all();
    else if constexpr (kChain == 32) __syncwarp();
    else __syncthreads();
  };
  const int *table = a.batch.table + static_cast<long long>(b) * a.batch.W, *into = a.into + static_cast<long long>(b) * a.into_W;
  auto look_up = [&](int i0, Rows* rows) {  // (all loads of a kind together: two trips to memory, however many rows a thread has)
    int k[kBeside], from[kBeside], to[kBeside];
#pragma unroll
    for (int e = 0; e < kBeside; ++e) {
      const int i = i0 + e * kChain + tid;
      k[e] = i < n && (kStep % kChain == 0 || e * kChain + tid < kStep) ? kept[i] : -1;
    }
#pragma unroll
    for (int e = 0; e < kBeside; ++e) {
      const bool fine = k[e] >= 0 && first >= 0;
      from[e] = fine ? page_there(table, a.batch.W, a.batch.page_shift, static_cast<long long>(first) + k[e]) : -1;
      to[e] = fine ? page_there(into, a.into_W, a.batch.page_shift, static_cast<long long>(first) + i0 + e * kChain + tid) : -1;
    }
#pragma unroll
    for (int e = 0; e < kBeside; ++e) {
      const int r = e * kChain + tid;
      if (kStep % kChain == 0 || r < kStep) rows[r] = i0 + r < n ? rows_of(a, h, first, k[e], i0 + r, from[e], to[e]) : Rows{-1, -1};
    }
  };
  const int r = tid / kOfPart, piece = part * kOfPart + tid % kOfPart;
  uint4* plane = reinterpret_cast<uint4*>(piece < kRow ? a.k : a.v) + (piece < kRow ? piece : piece - kRow);
  const bool beside = part == 0 && (a.k_exp != nullptr || a.weights != nullptr);
  const int by = C > 1 ? C * kStep : static_cast<int>(gridDim.z) * kStep;
  int i0 = (C > 1 ? rank : static_cast<int>(blockIdx.z)) * kStep, buffer = 0;
  look_up(i0, looked_up[threadIdx.x / kChain][0]);
  if constexpr (kChain == 32) __syncwarp();
  else __syncthreads();
  for (; i0 - rank * kStep < n; i0 += by, buffer ^= 1) {  // (the same steps for all of a cluster)
    const Rows* rows = looked_up[threadIdx.x / kChain][buffer];
    Rows mine[kMoveAtOnce], of_beside[kBeside];
    uint4 x[kMoveAtOnce];
    unsigned char ke[kBeside], ve[kBeside];
    float w[kBeside];
#pragma unroll
    for (int u = 0; u < kMoveAtOnce; ++u) {
      mine[u] = rows[u * kTogether + r];
      if (mine[u].from >= 0) x[u] = plane[static_cast<long long>(mine[u].from) * kRow];
    }
    if (beside) {
#pragma unroll
      for (int e = 0; e < kBeside; ++e) {
        const int at = e * kChain + tid;
        of_beside[e] = kStep % kChain == 0 || at < kStep ? rows[at] : Rows{-1, -1};
        if (of_beside[e].from < 0) continue;
        if (a.k_exp != nullptr) {
          ke[e] = a.k_exp[of_beside[e].from];
          ve[e] = a.v_exp[of_beside[e].from];
        }
        if (a.weights != nullptr) w[e] = a.weights[of_beside[e].from];
      }
    }
    if (i0 - rank * kStep + by < n) look_up(i0 + by, looked_up[threadIdx.x / kChain][buffer ^ 1]);
    meet();  // all of the step has been read, and the next one's rows are there
#pragma unroll
    for (int u = 0; u < kMoveAtOnce; ++u)
      if (mine[u].from >= 0) plane[static_cast<long long>(mine[u].to) * kRow] = x[u];
    if (beside) {
#pragma unroll
      for (int e = 0; e < kBeside; ++e) {
        if (of_beside[e].from < 0) continue;
        if (a.k_exp != nullptr) {
          a.k_exp[of_beside[e].to] = ke[e];
          a.v_exp[of_beside[e].to] = ve[e];
        }
        if (a.weights != nullptr) a.weights[of_beside[e].to] = w[e];
      }
    }
  }
}

int launched(cudaError_t err) {
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}

// Clusters of C along x.
template <typename... KArgs, typename... Args>
int launch_clusters(void (*kfn)(KArgs...), int C, dim3 grid, int threads, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  return launched(cudaLaunchKernelEx(&cfg, kfn, static_cast<KArgs>(args)...));
}

template <int C, int kThreads>
int launch_choose(const Choose& a, int B, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0};
  // room for a CTA's stretch of the longest sequence that the table allows, as far as there is some
  const long long longest = static_cast<long long>(a.batch.W) << a.batch.page_shift, stretch = (longest + C * kThreads - 1) / (C * kThreads) * kThreads;
  const int room = static_cast<int>(std::min(stretch, static_cast<long long>(kMostRoom)));
  if (C > 8 && cudaFuncSetAttribute(paged_choose_kernel<C, kThreads>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    cudaGetLastError();
    return FTB_ERR_LAUNCH;
  }
  if (!ensure_dynamic_smem(paged_choose_kernel<C, kThreads>, kMostRoom * 4, configured)) return FTB_ERR_LAUNCH;
  return launch_clusters(paged_choose_kernel<C, kThreads>, C, dim3(static_cast<unsigned>(B) * a.kv_heads * C), kThreads, static_cast<size_t>(room) * 4,
                         stream, a, room);
}
int launch_choose(const Choose& a, int B, cudaStream_t stream) {
  // One CTA, 8 or 16 of a cluster for each sequence and kv head, as the table has room for keys; us with the moves of 1032 rows, of (heads)
  // 4: 5000 keys 14.4 18.0 21.1, 8000 18.1 18.4 20.9, 30 000 38.5 18.2 21.4, 70 000 255 23.8 23.1, 200 001 728 34.4 28.6; 12: 200 001 keys 734 35.6
  // 50.4; 18: 12 000 keys 28.0 29.4, 30 000 39.0 30.1; 32: 30 000 39.4 42.0, 44 000 51.7 47.4, 70 000 267 58.3.  (One CTA keeps up to kMostRoom keys.)
  const long long longest = static_cast<long long>(a.batch.W) << a.batch.page_shift, heads = static_cast<long long>(B) * a.kv_heads, sms = current_sm_count();
  if (longest > 65536 && heads * 24 <= sms) return launch_choose<16, 1024>(a, B, stream);
  if ((longest > 8192 && heads * 8 <= sms) || (longest > kMostRoom && heads * 8 <= 2 * sms)) return launch_choose<8, 1024>(a, B, stream);
  return launch_choose<1, 512>(a, B, stream);
}

template <int kRow, int kOfPart, int kChain, int C>
int launch_move(const Move& a, int B, cudaStream_t stream) {
  constexpr int kStep = kChain / kOfPart * kMoveAtOnce, kChains = kMoveThreads / kChain;
  const int chains = B * a.kv_heads, blocks = (chains + kChains - 1) / kChains * C;
  // into other pages: enough blocks for every SM's room for them twice, so that one's end lies under others' work
  const int steps = (a.most + kStep - 1) / kStep;
  const int z = a.into == a.batch.table ? 1 : std::min(steps, std::max(1, 16 * current_sm_count() / blocks));
  return launch_clusters(paged_move_kernel<kRow, kOfPart, kChain, C>, C, dim3(blocks, 2 * kRow / kOfPart, z), kMoveThreads, 0, stream, a, chains);
}
template <int kRow>
int launch_move(const Move& a, int B, cudaStream_t stream) {
  // A few rows of a tree: a warp has them in one step or two.
  if (a.most <= 64) return launch_move<kRow, 2 * kRow, 32, 1>(a, B, stream);
  // In the same pages a part of a row is a chain, one step behind the other: clusters, which read hundreds of rows before they write them, as
  // long as their CTAs are on the device at a time, and parts of a row where they fill it with few heads.  2048 of 4096 rows of 16 bits, d 128, with
  // weights, us, of (heads) 4: parts 5.4, clusters of 8 9.2, of 4 15.8, one CTA 41.6; 32: 21.3, 15.1, 26.5, 44.6; 80: 56.7, 37.4, 36.4, 84.9; 160:
  // 120, 72, 71, 98; 384: 327, 157, 149, 144.5.  512 rows: 32 heads 18.1, 5.1, 7.7, 11.9; 384 200, 45, 41, 36.
  const long long heads = static_cast<long long>(B) * a.kv_heads, sms = current_sm_count();
  if (a.into == a.batch.table && heads * 64 <= 4 * sms) return launch_move<kRow, kRow / 4, kMoveThreads, 8>(a, B, stream);
  if (a.into == a.batch.table && heads * 8 <= 3 * sms) return launch_move<kRow, 2 * kRow, kMoveThreads, 8>(a, B, stream);
  if (a.into == a.batch.table && heads * 4 <= 6 * sms) return launch_move<kRow, 2 * kRow, kMoveThreads, 4>(a, B, stream);
  return launch_move<kRow, 2 * kRow, kMoveThreads, 1>(a, B, stream);
}
int move(const Move& a, int row_bytes, int B, cudaStream_t stream) {
  return row_bytes == 256 ? launch_move<16>(a, B, stream) : row_bytes == 128 ? launch_move<8>(a, B, stream) : launch_move<4>(a, B, stream);
}

// What both entry points ask of a cache: 0, or the reason for a refusal.
int check_cache(const void* k, const void* v, const void* k_exp, const void* v_exp, const int* table, const int* into, int B, int W, int into_W,
                int pages, int kv_heads, int page_size, int d) {
  if (!k || !v || !table || (k_exp == nullptr) != (v_exp == nullptr)) return FTB_ERR_ARG;
  if (B <= 0 || W <= 0 || (into != nullptr && into_W <= 0) || pages <= 0 || kv_heads <= 0 || kv_heads > 65536) return FTB_ERR_ARG;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return FTB_ERR_ARG;
  if ((d != 64 && d != 128) || static_cast<long long>(B) * kv_heads > INT_MAX / 8) return FTB_ERR_ARG;
  if (static_cast<long long>(pages) * kv_heads > INT_MAX / page_size) return FTB_ERR_ARG;  // rows are counted in 32 bits (so many would be 137 GB or more)
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_exp) | reinterpret_cast<uintptr_t>(v_exp)) & 15) != 0)
    return FTB_ERR_ALIGN;
  return FTB_OK;
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" int ftb_paged_cache_keep(void* k_cache, void* v_cache, unsigned char* k_exp, unsigned char* v_exp, float* weights,
                                    const int* kept, long long kept_seq, long long kept_head, const int* counts, const int* first,
                                    const int* table, const int* into, int B, int W, int into_W, int K, int pages, int kv_heads,
                                    int page_size, int d, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_cache(k_cache, v_cache, k_exp, v_exp, table, into, B, W, into_W, pages, kv_heads, page_size, d);
  if (rc) return rc;
  if (K < 0 || K > kMostKept || (K > 0 && !kept) || !counts) return FTB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(weights) & 3) != 0) return FTB_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  if (K == 0) return FTB_OK;
  if ((rc = check_device_sm100())) return rc;
  const PagedBatch batch{table, nullptr, nullptr, B, W, pages, 31 - __builtin_clz(static_cast<unsigned>(page_size))};
  const Move m{batch, into != nullptr ? into : table, into != nullptr ? into_W : W, kept, counts, first, kept_seq, kept_head, K, kv_heads,
               static_cast<unsigned char*>(k_cache), static_cast<unsigned char*>(v_cache), k_exp, v_exp, weights, static_cast<int*>(workspace)};
  return move(m, k_exp != nullptr ? d : 2 * d, B, static_cast<cudaStream_t>(stream));
}

extern "C" int ftb_paged_cache_evict(void* k_cache, void* v_cache, unsigned char* k_exp, unsigned char* v_exp, float* weights,
                                     const int* table, const int* lens, const int* into, int* lens_out, int* kept, int B, int W, int into_W,
                                     int keep, int recent, int pages, int kv_heads, int page_size, int d, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  int rc = check_cache(k_cache, v_cache, k_exp, v_exp, table, into, B, W, into_W, pages, kv_heads, page_size, d);
  if (rc) return rc;
  if (!weights || !lens || !lens_out || !kept || keep <= 0 || keep > kMostKept || recent < 0 || recent > keep) return FTB_ERR_ARG;
  if (static_cast<long long>(W) * page_size > kMostKept) return FTB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(weights) & 3) != 0) return FTB_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  const size_t rows = static_cast<size_t>(pages) * kv_heads * page_size, row = k_exp != nullptr ? d : 2 * d;
  const size_t kept_bytes = static_cast<size_t>(B) * kv_heads * keep * sizeof(int), lens_bytes = static_cast<size_t>(B) * sizeof(int);
  if (overlap(kept, kept_bytes, lens_out, lens_bytes)) return FTB_ERR_ARG;
  const void* out[2] = {kept, lens_out};
  const size_t out_bytes[2] = {kept_bytes, lens_bytes};
  for (int i = 0; i < 2; ++i)  // (the moves read what the choice has written; lens and table are read by all blocks)
    if (overlap(out[i], out_bytes[i], k_cache, rows * row) || overlap(out[i], out_bytes[i], v_cache, rows * row) ||
        (k_exp && (overlap(out[i], out_bytes[i], k_exp, rows) || overlap(out[i], out_bytes[i], v_exp, rows))) ||
        overlap(out[i], out_bytes[i], weights, rows * sizeof(float)) || overlap(out[i], out_bytes[i], lens, lens_bytes) ||
        overlap(out[i], out_bytes[i], table, lens_bytes * W) || (into && overlap(out[i], out_bytes[i], into, lens_bytes * into_W)))
      return FTB_ERR_ARG;
  if ((rc = check_device_sm100())) return rc;
  const PagedBatch batch{table, lens, nullptr, B, W, pages, 31 - __builtin_clz(static_cast<unsigned>(page_size))};
  int* status = static_cast<int*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Choose c{batch, weights, kept, lens_out, kv_heads, keep, recent, status};
  rc = launch_choose(c, B, s);
  if (rc) return rc;
  const Move m{batch, into != nullptr ? into : table, into != nullptr ? into_W : W, kept, lens_out, nullptr, static_cast<long long>(kv_heads) * keep,
               keep, keep, kv_heads, static_cast<unsigned char*>(k_cache), static_cast<unsigned char*>(v_cache), k_exp, v_exp, weights, status};
  return move(m, static_cast<int>(row), B, s);
}
