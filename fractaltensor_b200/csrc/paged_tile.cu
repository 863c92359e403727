// Attention over a paged cache for many rows: chunks of prompts, drafted tokens of large groups.  Tiles of query rows (token, head
// of a group) against blocks of 128 keys on the tensor cores (tcgen05), S = Q K^T and O += P V with accumulators in tensor
// memory, online softmax between them.
//
// 2048 tokens behind 14 336 keys, 32 heads of 128 over 8 kv heads, bf16: 558 us, 0.92 PFLOP/s; bound by the chain of a row's scores, 4300
// cycles a block of 256 rows beside 2048 of products, and by the joins (25 us).  96 sequences of 8500 keys on average in 8 bits, 5 tokens
// of 64 heads: 660 us, 0.2 PFLOP/s and 2.5 TB/s (847 where values are of 2^-40, with the sum apart for every block); bound by the instructions that make 8-bit keys operands (1.6 to 1.9 a cycle and SM).
// Trees of drafts (kTrees): a row's bits of the block's keys are laid out in shared memory when a block reaches into the new tokens, and taken with
// every look at the scores.  32 sequences of 33 tokens of 64 heads, up to 16 000 keys of 8 bits: 530 us for 256 of their 264 rows.
// Measured and not kept, the chunk: all 128 scores of a row in registers 616 us (spills; L1 is shared memory's), 32 scores loaded ahead of
// 32 in work 580, a warp for each slot's products 617, the slots' exponentials in turns 575, the second product in two halves 568 (of 566).
//
// One persistent CTA per SM walks its piece of the line of work (paged_work.cuh):
//   warp 0        the walk, announced to the others through a ring of stretches, and the loads of K and V, page by page: TMA boxes
//                 of a page's rows into the swizzled tiles that the products read; 8-bit pages and their exponents as they are
//   warp 1        issues the products
//   warps 2..9    softmax: two slots of 128 threads, a thread a row; they also fetch the queries and write the results
//   16-bit caches: one more warp zeroes values in front of and behind the keys that the tile sees (what lies there may be
//                 anything, and 0 * NaN is NaN), told by warp 0 which blocks need it
//   8-bit caches: four more warps turn codes into fp16 tiles, or, with 128 rows, eight, four of them one tile and the other four
//                 the next.  (They could load codes themselves, which would spare shared memory two passes; measured, they then
//                 wait for addresses to be translated, one load behind the other: 739 against 650 us for the drafts of 96 sequences.)
// A row's chain from scores to weights sits between two products, so that two slots keep the tensor cores busy.  Tiles of 256 rows:
// 128 to a slot, and a K or V block serves both.  Of 128: the slots take turns at the blocks; each has sums of its own for the same
// rows, which lie in the same lanes of tensor memory and are put together there.
//
// 8-bit caches: a block's codes become fp16 numbers code * 2^(7 + e - e_max), e_max the largest exponent of the block's keys (448 * 2^7 is
// below fp16's end): exact where exponents are within 22 of each other, off by 2^-39 of the block's largest number where within 31,
// and by 2^-31 of it behind that, where they are 0.  2^(e_max - 7) goes to the scores (keys) and into the weights (values, as in
// paged_short.cu, with a sum apart for blocks whose exponents are not ordinary), once a block.  Where exponents of a block lie further
// apart than 22 and a row does not see all of its keys, the largest may be of one that is hidden from it: that row is made a NaN, and
// gone through key by key as those are.  bf16 queries are scaled into fp16's range, row by row, by a power of two.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "../../include/ftb200.h"
#include "paged_forms.h"
#include "paged_work.cuh"
#include "tmap.h"

namespace ftb {
namespace {

constexpr int kKeys = 128, kAtLeast = 1, kStretches = 4, kRefs = 8, kFar = 256;
constexpr int kUp = 7, kExact = 15 + kUp;  // 8 bits: codes as fp16 are times 2^kUp; the smallest code is 2^-9, fp16's smallest number 2^-24
constexpr int kMostSlots = 14;
constexpr float kAbove = 8.f;  // as in flash_attn.cu: the maximum in use may lie 2^8 below the real one

struct Stretch {
  int b, h, flat0, rows, first, hi_all;
  PagedKeys keys;
  int block0, blocks;  // of 128 keys; blocks 0: nobody sees anything
  int whole, place;    // place: of the parts, where the tile is not whole
  long long pos0;
  int last;            // nothing behind this one
};

struct Edge {  // values in ring slot `slot`, with its next fill's parity: of the keys from key0 on only lo .. hi - 1 are seen
  int slot, key0, lo, hi;
  uint32_t phase;
};

template <bool k8, bool kTwo, int kWhat>
struct Control {
  PagedLineRoom line;
  Stretch ring[kStretches];
  uint64_t ring_full[kStretches], ring_empty[kStretches];
  uint64_t q_full[2], s_full[2], p_full[2], pv_done[2], o_free[2], begun, fin;
  uint64_t kv_full[kMostSlots], kv_empty[kMostSlots];    // tiles that the products read
  uint64_t raw_full[k8 ? kMostSlots : 1], raw_empty[k8 ? kMostSlots : 1];  // 8-bit blocks
  Edge edges[kStretches];
  uint64_t edge_full[kStretches], edge_empty[kStretches], v_fixed[kMostSlots];
  float top[2][128], sum[2][128];  // [slot][row]
  // 8 bits: what `sum` refers to, and a thread's own: the sum of blocks apart and what it refers to (in registers: 646 for 628 us of drafts)
  float sum_top[k8 ? 2 : 1][k8 ? 128 : 1], apart_l[k8 ? 2 : 1][k8 ? 128 : 1], apart_n[k8 ? 2 : 1][k8 ? 128 : 1];
  int see_lo[2][128], see_hi[2][128];
  uint32_t tree[kWhat == kTrees ? 2 : 1][4][kWhat == kTrees ? 128 : 1];  // [slot][word][row]: the bits of a block's keys, a thread's own
  int k_ref[kRefs], v_ref[kRefs];  // e_max of a block; + kFar: exponents more than kExact apart, in one that not every row sees all of
  uint32_t tmem_base;
  int abort, dead;
};

template <bool k8, int D, int R, int kWhat>
struct Plan {
  static constexpr bool kTwo = R == 256;
  static constexpr int kHalf = 128 * 128, kTile = D / 64 * kHalf;
  static constexpr int kQ = (kTwo ? 2 : 1) * kTile;
  static constexpr int kControl = (sizeof(Control<k8, kTwo, kWhat>) + 15) / 16 * 16, kRoom = 232448 - 1024 - kControl - kQ;
  static constexpr int kSlots = k8 ? (D == 128 ? 3 : 6) : kRoom / kTile < kMostSlots ? kRoom / kTile : kMostSlots;
  // 8-bit: a block's codes, and the exponents of its keys and values; as many on their way as there is room for
  static constexpr int kRaw = 128 * D + 256, kRawRoom = (kRoom - kSlots * kTile) / kRaw;
  static constexpr int kRawSlots = k8 ? (kRawRoom < kMostSlots ? kRawRoom : kMostSlots) : 0;
  static constexpr int kSmem = 1024 + kControl + kQ + kSlots * kTile + kRawSlots * kRaw;
  // Warps: a block of 256 rows keeps the softmax busy longer than four warps need for its tiles, and with fewer warps each has more
  // registers.
  static constexpr int kSoftmax = 8, kConvert = kTwo ? 4 : 8;
  static constexpr int kThreads = 32 * (2 + kSoftmax + (k8 ? kConvert : 1));
  static_assert(kSlots >= 3 && (!k8 || kRawSlots >= 3) && kSmem <= 232448, "shared memory budget");
};

// 16-byte piece `piece` of row `row` in a tile of 64-column halves of 128-byte swizzled rows.
__device__ __forceinline__ uint8_t* piece_ptr(uint8_t* tile, int row, int piece) {
  return tile + (piece >> 3) * (128 * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}

// Tile n of the stream of K and V blocks of a stretch.  kTwo: K0, V0, K1, V1, ..; else, the slots taking turns at the blocks,
// K0, K1, V0, K2, V1, .., the order in which the products come.
struct StreamTile {
  bool is_v;
  int j;
};
template <bool kTwo>
__device__ __forceinline__ StreamTile stream_tile(int n, int blocks) {
  if (kTwo) return {(n & 1) != 0, n >> 1};
  if (n == 0) return {false, 0};
  if (blocks == 1) return {true, 0};
  if (n == 1) return {false, 1};
  const int r = n - 2, turn = 2 * (blocks - 2);
  if (r >= turn) return {true, blocks - 2 + r - turn};
  return {(r & 1) == 0, (r & 1) == 0 ? r >> 1 : 2 + (r >> 1)};
}

// Blocks of a stretch that slot t takes part in: of kTwo j0 .. j1, else every second one; how many.
struct Mine {
  int j0, j1, n;
};
template <bool kTwo>
__device__ __forceinline__ Mine blocks_of_slot(const PagedAttn& a, const Stretch& x, int t) {
  if (!kTwo) return {t, x.blocks - 1, (x.blocks - t + 1) / 2};
  const int rows = min(128, x.rows - t * 128);
  if (rows <= 0 || x.blocks == 0) return {0, -1, 0};
  const PagedKeys k = keys_of_rows(a, x.pos0, x.first, x.hi_all, x.flat0 + t * 128, rows);
  if (k.hi <= k.lo) return {0, -1, 0};
  const int j0 = max(0, k.lo / kKeys - x.block0), j1 = min(x.blocks - 1, (k.hi - 1) / kKeys - x.block0);
  return {j0, j1, max(0, j1 - j0 + 1)};
}

template <typename T, bool k8, int D, int R, int kWhat>
__global__ void __launch_bounds__(Plan<k8, D, R, kWhat>::kThreads, 1)
paged_tile_kernel(const __grid_constant__ PagedAttn a, const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                  float* __restrict__ parts, PagedCut* __restrict__ cuts) {
  using P = Plan<k8, D, R, kWhat>;
  using C = typename std::conditional<k8, __half, T>::type;
  constexpr bool kTwo = P::kTwo;
  constexpr int kSlots = P::kSlots, kRawSlots = P::kRawSlots;
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = blockIdx.x;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + P::kQ;
  uint8_t* sRaw = sKV + kSlots * P::kTile;
  using Ctl = Control<k8, kTwo, kWhat>;
  Ctl& ctl = *reinterpret_cast<Ctl*>(sRaw + kRawSlots * P::kRaw);
  volatile int* s_abort = &ctl.abort;
  int* status = a.status;

  if (threadIdx.x == 0) {
    if constexpr (!k8) {
      prefetch_tmap(&mapK);
      prefetch_tmap(&mapV);
    }
    for (int i = 0; i < kStretches; ++i) {
      mbar_init(&ctl.ring_full[i], 1);
      mbar_init(&ctl.ring_empty[i], 1 + P::kSoftmax + (k8 ? P::kConvert : 0));
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.q_full[i], kTwo ? 4 : 8);
      mbar_init(&ctl.s_full[i], 1);
      mbar_init(&ctl.p_full[i], 4);
      mbar_init(&ctl.pv_done[i], 1);
      mbar_init(&ctl.o_free[i], kTwo ? 4 : 8);
    }
    mbar_init(&ctl.begun, 1);
    mbar_init(&ctl.fin, 8);
    for (int i = 0; i < kMostSlots; ++i) {
      mbar_init(&ctl.kv_full[i], k8 ? 4 : 1);
      mbar_init(&ctl.kv_empty[i], 1);
      mbar_init(&ctl.v_fixed[i], 1);
    }
    if constexpr (k8) {
      for (int i = 0; i < kMostSlots; ++i) {
        mbar_init(&ctl.raw_full[i], 1);
        mbar_init(&ctl.raw_empty[i], 4);
      }
    }
    for (int i = 0; i < kStretches; ++i) {
      mbar_init(&ctl.edge_full[i], 1);
      mbar_init(&ctl.edge_empty[i], 1);
    }
    ctl.abort = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  grid_dependency_wait();
  grid_launch_dependents();
  if (threadIdx.x == 0) {  // an earlier wait ran out: do nothing.  (An index out of its range was that call's error.)
    const int before = *reinterpret_cast<volatile int*>(status);
    ctl.dead = before != 0 && before != FTB_ERR_INDEX;
  }
  int seq0;
  long long at0;
  const PagedLine line = paged_line<R, kKeys, kWhat>(a, piece, gridDim.x, kAtLeast, ctl.line, &seq0, &at0);
  const bool idle = piece >= line.pieces || line.total == 0;
  if (idle || ctl.dead != 0) {
    if (threadIdx.x == 0) cuts[piece].last = -1;
    return;
  }
  if (warp == 1) {
    tmem_alloc(&ctl.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctl.tmem_base;
  // tensor memory: S0 [0, 128), S1 [128, 256), O0 [256, 256 + D), O1 [384, 384 + D); P_t (16-bit pairs)
  // over the first half of S_t's columns.

  // Stretch i of this CTA, as every role but the first warp gets it.
  auto await = [&](int i) -> bool {
    return mbar_wait_warp(&ctl.ring_full[i % kStretches], (i / kStretches) & 1, s_abort, status, FTB_ERR_TIMEOUT_TMA);
  };
  auto give_back = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.ring_empty[i % kStretches]);
  };

  if (warp == 0) {
    // --------------------------------------------------------- the walk, and the loads
    PagedWalk<R, kKeys, kWhat> walk;
    walk.begin(a, line, piece, seq0, at0);
    const int pages = kKeys >> a.batch.page_shift;  // of a block
    int slot = 0, edges = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto tell = [&](const Edge& e) -> bool {
      const int at = edges % kStretches;
      if (edges >= kStretches && !mbar_wait_warp(&ctl.edge_empty[at], (edges / kStretches - 1) & 1, s_abort, status, FTB_ERR_TIMEOUT_SLOT)) return false;
      if (lane == 0) {
        ctl.edges[at] = e;
        mbar_arrive(&ctl.edge_full[at]);
      }
      ++edges;
      return true;
    };
    for (int i = 0; ok && walk.more(); ++i) {
      const PagedTile w = walk.next(a);
      if (i >= kStretches && !mbar_wait_warp(&ctl.ring_empty[i % kStretches], (i / kStretches - 1) & 1, s_abort, status, FTB_ERR_TIMEOUT_SLOT)) break;
      const bool some = w.keys.hi > w.keys.lo;
      const int block0 = w.keys.lo / kKeys + w.r0, blocks = some ? w.r1 - w.r0 : 0;
      if (lane == 0) {
        Stretch& x = ctl.ring[i % kStretches];
        x.b = w.b;
        x.h = w.h;
        x.flat0 = w.flat0;
        x.rows = w.rows;
        x.first = walk.s.first;
        x.hi_all = walk.s.hi;
        x.keys = w.keys;
        x.block0 = block0;
        x.blocks = blocks;
        x.whole = w.r0 == 0 && w.r1 == w.units;
        x.place = 2 * piece + (w.r0 == 0 ? 1 : 0);
        x.pos0 = walk.s.pos0;
        x.last = !walk.more();
        mbar_arrive(&ctl.ring_full[i % kStretches]);
        if (i == 0) {
          const int last = last_piece_of(line, piece, w);
          cuts[piece].last = last;
          if (last >= 0) cuts[piece] = PagedCut{last, w.b, walk.s.first, w.flat0, w.rows, w.h, w.keys.lo, w.keys.hi, walk.s.pos0};
        }
      }
      const int* table = a.batch.table + static_cast<long long>(w.b) * a.batch.W;
      // this lane's page of tile n, or -1: one lane a page; those that nobody sees need not be there
      auto page_of_tile = [&](int n) -> int {
        const int key0 = (block0 + stream_tile<kTwo>(n, blocks).j) * kKeys, at = key0 + (lane << a.batch.page_shift);
        if (n >= 2 * blocks || lane >= pages || at >= w.keys.hi || at + (1 << a.batch.page_shift) <= w.keys.lo) return -1;
        return __ldg(table + (at >> a.batch.page_shift));
      };
      int page_next = page_of_tile(0);
      for (int n = 0; ok && n < 2 * blocks; ++n) {
        const StreamTile x = stream_tile<kTwo>(n, blocks);
        const int key0 = (block0 + x.j) * kKeys;
        const int p0 = w.keys.lo > key0 ? (w.keys.lo - key0) >> a.batch.page_shift : 0;
        const int p1 = min(pages, (w.keys.hi - key0 + (1 << a.batch.page_shift) - 1) >> a.batch.page_shift);
        const bool here = lane >= p0 && lane < p1;
        int page = page_next;
        page_next = page_of_tile(n + 1);  // on its way while this one waits for room
        uint64_t* full = k8 ? &ctl.raw_full[slot] : &ctl.kv_full[slot];
        ok = mbar_wait_warp(k8 ? &ctl.raw_empty[slot] : &ctl.kv_empty[slot], phase ^ 1u, s_abort, status, FTB_ERR_TIMEOUT_SLOT);
        if (!ok) break;
        if (here && (page < 0 || page >= a.batch.pages)) {
          atomicCAS(status, 0, FTB_ERR_INDEX);
          page = 0;
        }
        if (lane == 0) mbar_arrive_expect_tx(full, ((p1 - p0) << a.batch.page_shift) * (k8 ? D + (x.is_v ? 1 : 2) : 2 * D));
        __syncwarp();
        if (here) {
          if constexpr (k8) {
            const long long row = (static_cast<long long>(page) * a.kv_heads + w.h) << a.batch.page_shift;
            const uint32_t rows = 1u << a.batch.page_shift;
            uint8_t* dst = sRaw + slot * P::kRaw;
            bulk_load_1d(dst + lane * rows * D, (x.is_v ? a.v : a.k) + row * D, rows * D, full);
            bulk_load_1d(dst + 128 * D + 128 + lane * rows, a.v_exp + row, rows, full);
            if (!x.is_v) bulk_load_1d(dst + 128 * D + lane * rows, a.k_exp + row, rows, full);
          } else {
            const CUtensorMap* m = x.is_v ? &mapV : &mapK;
            uint8_t* dst = sKV + slot * P::kTile + (lane << a.batch.page_shift) * 128;
            const int y = (page * a.kv_heads + w.h) << a.batch.page_shift;
            tma_load_2d(dst, m, full, 0, y);
            if constexpr (D == 128) tma_load_2d(dst + P::kHalf, m, full, 64, y);
          }
        }
        if (!k8 && x.is_v && (key0 < w.keys.lo || key0 + kKeys > w.keys.hi)) ok = tell({slot, key0, w.keys.lo, w.keys.hi, phase});
        if (++slot == (k8 ? kRawSlots : kSlots)) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
    if (!k8 && ok) tell({-1, 0, 0, 0, 0u});
  } else if (warp == 1) {
    // ------------------------------------------------------------------- the products
    const bool leader = elect_one();
    constexpr uint32_t idesc_qk = make_idesc_f16(128, 128, Fmt<C>::kind, 0, 0);
    constexpr uint32_t idesc_pv = make_idesc_f16(128, D, Fmt<C>::kind, 0, 1);  // V is MN-major
    const uint64_t dQ = make_sdesc_sw128(smem_u32(sQ), 16, 1024);
    const uint64_t dK = make_sdesc_sw128(smem_u32(sKV), 16, 1024);
    const uint64_t dV = make_sdesc_sw128(smem_u32(sKV), P::kHalf, 1024);
    uint32_t full_bits = 0, fixed_bits = 0, p_phase[2] = {0, 0};
    int slot = 0;  // of the next tile of the stream
    bool ok = true;
    auto issue_s = [&](int t, int at) {
      const uint64_t dq = dQ + static_cast<uint64_t>(kTwo ? (t * P::kTile) >> 4 : 0), dk = dK + static_cast<uint64_t>((at * P::kTile) >> 4);
      if (leader) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k >> 2) * P::kHalf + (k & 3) * 32) >> 4;
          umma_ss(tmem_base + t * 128, dq + off, dk + off, idesc_qk, k != 0 ? 1u : 0u);
        }
        umma_commit(&ctl.s_full[t]);
      }
    };
    auto issue_pv = [&](int t, int at, bool first) {
      const uint64_t dv = dV + static_cast<uint64_t>((at * P::kTile) >> 4);
      if (leader) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_ts(tmem_base + 256 + t * 128, tmem_base + t * 128 + k * 8, dv + k * (2048 >> 4), idesc_pv, (!first || k != 0) ? 1u : 0u);
        umma_commit(&ctl.pv_done[t]);
      }
    };
    auto step = [&](int at) { return at + 1 == kSlots ? 0 : at + 1; };
    auto wait_tile = [&](int at) -> bool {
      if (!mbar_wait_warp(&ctl.kv_full[at], (full_bits >> at) & 1u, s_abort, status, FTB_ERR_TIMEOUT_TMA)) return false;
      full_bits ^= 1u << at;
      return true;
    };
    for (int i = 0; ok; ++i) {
      if (!await(i)) break;
      const Stretch x = ctl.ring[i % kStretches];
      give_back(i);
      const Mine m[2] = {blocks_of_slot<kTwo>(a, x, 0), blocks_of_slot<kTwo>(a, x, 1)};
      auto wait_v = [&](int at, int j) -> bool {  // values at the edges of what the tile sees have been zeroed
        if (!wait_tile(at)) return false;
        const int key0 = (x.block0 + j) * kKeys;
        if (k8 || (key0 >= x.keys.lo && key0 + kKeys <= x.keys.hi)) return true;
        const bool fine = mbar_wait_warp(&ctl.v_fixed[at], (fixed_bits >> at) & 1u, s_abort, status, FTB_ERR_TIMEOUT_TMA);
        fixed_bits ^= 1u << at;
        return fine;
      };
      auto wait_p = [&](int t) -> bool {
        if (!mbar_wait_warp(&ctl.p_full[t], p_phase[t], s_abort, status, FTB_ERR_TIMEOUT_EPI)) return false;
        p_phase[t] ^= 1u;
        tc_fence_after();
        return true;
      };
      // the queries are there, and the results of the stretch in front have been taken out of tensor memory
      for (int t = 0; t < (kTwo ? 2 : 1) && ok; ++t)
        ok = mbar_wait_warp(&ctl.q_full[t], i & 1, s_abort, status, FTB_ERR_TIMEOUT_EPI) &&
             (i == 0 || mbar_wait_warp(&ctl.o_free[t], (i - 1) & 1, s_abort, status, FTB_ERR_TIMEOUT_EPI));
      if (!ok) break;
      if (lane == 0) mbar_arrive(&ctl.begun);
      tc_fence_after();
      if constexpr (kTwo) {
        if (x.blocks > 0) {
          int k_at = slot;
          ok = wait_tile(k_at);
          if (ok) {
            for (int t = 0; t < 2; ++t)
              if (m[t].n > 0 && m[t].j0 == 0) issue_s(t, k_at);
            if (leader) umma_commit(&ctl.kv_empty[k_at]);
          }
          for (int j = 0; j < x.blocks && ok; ++j) {
            const bool more = j + 1 < x.blocks;
            const int v_at = step(k_at), next = step(v_at);
            ok = wait_v(v_at, j) && (!more || wait_tile(next));
            for (int t = 0; t < 2 && ok; ++t) {
              if (j >= m[t].j0 && j <= m[t].j1) {
                ok = wait_p(t);
                if (!ok) break;
                issue_pv(t, v_at, j == m[t].j0);
              }
              // (the tensor pipe runs in the order of issue: S_t(j + 1) overwrites P_t only after its product)
              if (more && j + 1 >= m[t].j0 && j + 1 <= m[t].j1) issue_s(t, next);
            }
            if (!ok) break;
            if (leader) {
              umma_commit(&ctl.kv_empty[v_at]);
              if (more) umma_commit(&ctl.kv_empty[next]);
            }
            k_at = next;
          }
          if (ok) slot = k_at;
        }
      } else {
        auto done = [&] {
          if (leader) umma_commit(&ctl.kv_empty[slot]);
          slot = step(slot);
        };
        for (int t = 0; t < 2 && t < x.blocks && ok; ++t) {
          ok = wait_tile(slot);
          if (!ok) break;
          issue_s(t, slot);
          done();
        }
        for (int j = 0; j < x.blocks && ok; ++j) {
          const int t = j & 1;
          ok = wait_v(slot, j) && wait_p(t);
          if (!ok) break;
          issue_pv(t, slot, j < 2);
          done();
          if (j + 2 < x.blocks) {
            ok = wait_tile(slot);
            if (!ok) break;
            issue_s(t, slot);
            done();
          }
        }
      }
      if (x.last) break;
    }
  } else if (warp < 2 + P::kSoftmax) {
    // ------------------------------------------------ softmax: slot t, row r of its 128
    const int t = (warp - 2) / 4, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t s_addr = lane_addr + t * 128, o_addr = lane_addr + 256 + t * 128;
    constexpr int kCols = kTwo ? D : D / 2;  // of the output, that this thread finishes
    const int c0 = kTwo ? 0 : t * kCols;
    // parities: bit 0 the next scores, 2 fin, 4 + t the next product P V of slot t in a stretch
    uint32_t par = 0;
    int blocks0 = 0;  // blocks of the stretches so far
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!await(i)) break;
      const Stretch& x = ctl.ring[i % kStretches];  // (read again where it is needed, and given back behind the results: registers)
      const int row0 = (kTwo ? t * 128 : 0) + quad * 32, row = row0 + lane;  // of the tile
      const bool busy = row0 < x.rows;  // this warp has rows
      const bool mine = row < x.rows;
      int tok, head;
      auto place = [&] {
        const int flat = x.flat0 + row, token = flat / a.group;
        tok = x.first + token;
        head = x.h * a.group + flat - token * a.group;
      };
      place();
      {  // (read back a block at a time, which saves registers)
        const long long pos = mine ? x.pos0 + tok : -1;
        ctl.see_hi[t][r] = static_cast<int>(max(-1ll, min(pos, static_cast<long long>(x.keys.hi) - 1)));
        ctl.see_lo[t][r] = a.window > 0 ? static_cast<int>(max(0ll, min(pos - a.window + 1, static_cast<long long>(INT_MAX)))) : 0;
      }
      float factor = a.scale_log2 * (k8 ? 1.f / (1 << kUp) : 1.f);

      // ---- queries: this thread's columns are those that it finishes
      if (busy) {
        uint8_t* tile = sQ + (kTwo ? t * P::kTile : 0);
        const T* src = static_cast<const T*>(a.q) + static_cast<long long>(tok) * a.q_row + static_cast<long long>(head) * a.q_head;
        constexpr int kPieces = kCols / 8;
        const int p0 = c0 / 8;
        if constexpr (k8 && !std::is_same<T, __half>::value) {
          uint32_t top = 0;
          if (mine) {
#pragma unroll
            for (int p = 0; p < D / 8; ++p) {
              const uint4 v = *reinterpret_cast<const uint4*>(src + p * 8);
              const uint32_t y = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
              top = max(top, max(y & 0xffffu, y >> 16));
            }
          }
          const int e = min(253, max(1, static_cast<int>(top >> 7)));
          const float by = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
          factor *= __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
          for (int p = 0; p < kPieces; ++p) {
            uint4 v = mine ? *reinterpret_cast<const uint4*>(src + (p0 + p) * 8) : make_uint4(0u, 0u, 0u, 0u);
            uint32_t* y = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = unpack2<T>(y[k]);
              y[k] = Fmt<__half>::pack2(f.x * by, f.y * by);
            }
            *reinterpret_cast<uint4*>(piece_ptr(tile, r, p0 + p)) = v;
          }
        } else {
          uint4 v[kPieces];
#pragma unroll
          for (int p = 0; p < kPieces; ++p) v[p] = mine ? *reinterpret_cast<const uint4*>(src + (p0 + p) * 8) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int p = 0; p < kPieces; ++p) *reinterpret_cast<uint4*>(piece_ptr(tile, r, p0 + p)) = v[p];
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.q_full[kTwo ? t : 0]);

      // ---- blocks
      const Mine m = blocks_of_slot<kTwo>(a, x, t);
      float top = 0.f, l = 0.f, near = kNear;  // 8 bits: l takes a block's weights where its values' largest exponent is below
      if constexpr (k8) {
        ctl.apart_l[t][r] = 0.f;
        ctl.apart_n[t][r] = -FLT_MAX;
      }
      for (int k = 0; k < m.n && ok; ++k) {
        const int j = kTwo ? m.j0 + k : 2 * k + t;
        ok = mbar_wait_warp(&ctl.s_full[t], par & 1u, s_abort, status, FTB_ERR_TIMEOUT_MMA);
        if (!ok) break;
        par ^= 1u;
        tc_fence_after();
        if (busy) {
          const int key0 = (x.block0 + j) * kKeys;
          const int lo_col = ctl.see_lo[t][r] - key0, hi_col = ctl.see_hi[t][r] - key0;
          const bool cut = __any_sync(0xffffffffu, mine && (lo_col > 0 || hi_col < kKeys - 1));
          const long long in_new = key0 - (x.pos0 + x.first);  // of the block's first key among the sequence's new tokens
          const bool masked = kWhat == kTrees && in_new > -kKeys;
          if (masked) {
            place();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const long long j = in_new + 32 * i;
              ctl.tree[t][i][r] = mine ? __funnelshift_r(tree_word(a, tok, j >> 5), tree_word(a, tok, (j >> 5) + 1), static_cast<uint32_t>(j & 31)) : 0u;
            }
          }
          float f = factor, add = 0.f, inv = 1.f;
          if constexpr (k8) {
            int kr = ctl.k_ref[(blocks0 + j) & (kRefs - 1)], vr = ctl.v_ref[(blocks0 + j) & (kRefs - 1)];
            if ((kr | vr) & kFar) {
              kr &= kFar - 1;
              vr &= kFar - 1;
              if (masked || lo_col > max(0, x.keys.lo - key0) || hi_col < min(kKeys, x.keys.hi - key0) - 1) factor = __uint_as_float(0x7fffffffu);
            }
            // (hidden scores are -inf already: times 0, as of a row of zeros and small keys, they would be NaN, as a score of 0 times
            // infinity.  No score moves: they are below 2^40 here.)
            f = fminf(fmaxf(factor * exponent_scale(kr), FLT_MIN), FLT_MAX);
            if (factor != factor) f = factor;
            add = static_cast<float>(vr - 127 - kUp);
            inv = exponent_scale(min(254, 254 + kUp - vr));  // (of use where `add` is ordinary)
          }
          // kChunk scores at a time, read again for the weights.  (A thread that spills goes to L2 for it: shared memory has taken
          // L1's room.  And loops instead of straight code: with several roles on an SM its instruction cache is what runs out.)
          constexpr int kChunk = k8 && !kTwo ? 32 : 64;
          uint32_t s[kChunk];
          auto scores = [&](int n) {
#pragma unroll
            for (int e = 0; e < kChunk; e += 32) tmem_ld32p(s_addr + n * kChunk + e, s + e);
            tmem_ld_wait();
            if (cut) {
              const int lo = lo_col - n * kChunk, hi = hi_col - n * kChunk;
              asm volatile("" ::: "memory");  // (a branch, not a select for every score)
#pragma unroll
              for (int e = 0; e < kChunk; ++e)
                if (e < lo || e > hi) s[e] = 0xff800000u;
            }
            if (masked) {
              asm volatile("" ::: "memory");
#pragma unroll
              for (int i = 0; i < kChunk / 32; ++i) {
                const uint32_t bits = ctl.tree[t][n * (kChunk / 32) + i][r];
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if ((bits >> e & 1u) == 0) s[32 * i + e] = 0xff800000u;
              }
            }
          };
          float mx = -INFINITY;
#pragma unroll 1
          for (int n = 0; n < kKeys / kChunk; ++n) {
            scores(n);
            float mx8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) mx8[e] = fmaxf(__uint_as_float(s[e]), __uint_as_float(s[8 + e]));
#pragma unroll
            for (int e = 16; e < kChunk; e += 16)
#pragma unroll
              for (int q = 0; q < 8; ++q) mx8[q] = fmax3(mx8[q], __uint_as_float(s[e + q]), __uint_as_float(s[e + 8 + q]));
            mx = fmax3(mx, fmax3(mx8[0], mx8[1], mx8[2]), fmaxf(fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
          }
          // (a row may see nothing of a block: the lowest finite number keeps its weights 0)
          const float m_new = fmaxf(fmaf(mx, f, add), -FLT_MAX);
          const bool apart = k8 && fabsf(add + kUp) > near;  // (the same in all lanes)
          if constexpr (k8) {
            if (apart) {
              const bool both = near > 0.f && k > 0;  // l holds something, and top is near the scores
              const float n = ctl.apart_n[t][r];
              float to = fmaxf(n, m_new - add);
              if (both) to = fmaxf(to, top);
              float more = ctl.apart_l[t][r] * exp2_fast(n - to) + (both ? l * exp2_fast(top - to) : 0.f);
#pragma unroll 1
              for (int n = 0; n < kKeys / kChunk; ++n) {
                scores(n);
#pragma unroll
                for (int e = 0; e < kChunk; ++e) more += exp2_fast(fmaf(__uint_as_float(s[e]), f, -to));
              }
              ctl.apart_l[t][r] = more;
              ctl.apart_n[t][r] = to;
              l = inv = 0.f;
            }
          }
          if (k == 0) {
            top = m_new;
          } else {
            const bool need = m_new - top > kAbove;
            if (__any_sync(0xffffffffu, need)) {
              // the product in front has to be done: O is at rest then
              ok = mbar_wait_warp(&ctl.pv_done[t], ((par >> (4 + t)) + k - 1) & 1u, s_abort, status, FTB_ERR_TIMEOUT_MMA);
              if (!ok) break;
              tc_fence_after();
              const float keep = need ? exp2_fast(top - m_new) : 1.f;
              if (need) top = m_new;
              l *= keep;
#pragma unroll 1
              for (int ch = 0; ch < D / 16; ++ch) {
                uint32_t o[16];
                tmem_ld16(o_addr + ch * 16, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tmem_st16(o_addr + ch * 16, o);
              }
              tmem_st_wait();
            }
          }
          if constexpr (k8) {
            if (apart) near = __any_sync(0xffffffffu, fabsf(top - ctl.apart_n[t][r]) > kNearTops) ? -1.f : kNear;
          }
          const float minus = add - top;
          const uint64_t f2 = dup_f32x2(f), minus2 = dup_f32x2(minus);
          uint64_t sum4[4] = {0, 0, 0, 0};
#pragma unroll 1
          for (int n = 0; n < kKeys / kChunk; ++n) {
            scores(n);
#pragma unroll
            for (int half = 0; half < kChunk / 32; ++half) {
              uint32_t pk[16];
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const int at = 32 * half + 2 * c;
                float p0, p1;
                unpair_f32x2(fma_to_f32x2(pair_f32x2(__uint_as_float(s[at]), __uint_as_float(s[at + 1])), f2, minus2), p0, p1);
                p0 = exp2_fast(p0);
                p1 = exp2_fast(p1);
                add_f32x2(sum4[c & 3], pair_f32x2(p0, p1));
                pk[c] = Fmt<C>::pack2(p0, p1);
              }
              tmem_st16(s_addr + n * (kChunk / 2) + half * 16, pk);  // over scores that this thread has read
            }
          }
          add_f32x2(sum4[0], sum4[1]);
          add_f32x2(sum4[2], sum4[3]);
          add_f32x2(sum4[0], sum4[2]);
          float l0, l1;
          unpair_f32x2(sum4[0], l0, l1);
          l = fmaf(l0 + l1, inv, l);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_full[t]);
      }
      // (a slot without blocks waits for no product: it must not hand over its next queries and results before the products have
      // taken notice of these)
      if (ok) ok = mbar_wait_warp(&ctl.begun, i & 1, s_abort, status, FTB_ERR_TIMEOUT_MMA);
      if (!ok) break;
      blocks0 += x.blocks;
      if (m.n == 0) top = -FLT_MAX;
      float l_top = top;  // what l refers to
      if constexpr (k8) {
        const float n = ctl.apart_n[t][r];
        l_top = near > 0.f ? fmaxf(n, top) : n;
        l = (near > 0.f ? l * exp2_fast(top - l_top) : 0.f) + ctl.apart_l[t][r] * exp2_fast(n - l_top);
      }

      // ---- results: of both slots, where they share the rows
      float other_m = -FLT_MAX, other_l = 0.f, other_top = -FLT_MAX;
      int n_other = 0;
      if (!kTwo && x.blocks > 0) {
        ctl.top[t][r] = top;
        ctl.sum[t][r] = l;
        if constexpr (k8) ctl.sum_top[t][r] = l_top;
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.fin);
        ok = mbar_wait_warp(&ctl.fin, par >> 2 & 1u, s_abort, status, FTB_ERR_TIMEOUT_EPI);
        if (!ok) break;
        par ^= 4u;
        n_other = blocks_of_slot<kTwo>(a, x, t ^ 1).n;
        other_m = ctl.top[t ^ 1][r];
        other_l = ctl.sum[t ^ 1][r];
        if constexpr (k8) other_top = ctl.sum_top[t ^ 1][r];
      }
      if (m.n > 0) ok = mbar_wait_warp(&ctl.pv_done[t], ((par >> (4 + t)) + m.n - 1) & 1u, s_abort, status, FTB_ERR_TIMEOUT_MMA);
      if (ok && n_other > 0) ok = mbar_wait_warp(&ctl.pv_done[t ^ 1], ((par >> (4 + (t ^ 1))) + n_other - 1) & 1u, s_abort, status, FTB_ERR_TIMEOUT_MMA);
      if (!ok) break;
      par ^= static_cast<uint32_t>(m.n & 1) << (4 + t) ^ static_cast<uint32_t>(n_other & 1) << (4 + (t ^ 1));
      tc_fence_after();
      const float all_m = fmaxf(top, other_m), keep = exp2_fast(top - all_m), take = exp2_fast(other_m - all_m);
      const float all_top = k8 ? fmaxf(l_top, other_top) : all_m;
      const float sum = k8 ? l * exp2_fast(l_top - all_top) + other_l * exp2_fast(other_top - all_top) : l * keep + other_l * take;
      // this thread's columns, 16 at a time
      auto columns = [&](int ch, float (&y)[16]) {
        uint32_t o[16], o2[16];
        if (m.n > 0) tmem_ld16(lane_addr + 256 + t * 128 + c0 + ch * 16, o);
        if (n_other > 0) tmem_ld16(lane_addr + 256 + (t ^ 1) * 128 + c0 + ch * 16, o2);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e)
          y[e] = (m.n > 0 ? __uint_as_float(o[e]) * keep : 0.f) + (n_other > 0 ? __uint_as_float(o2[e]) * take : 0.f);
      };
      float scale = x.whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f, scale2 = 1.f;
      if constexpr (k8) {  // to what the sum refers to (in two steps: it may be 2^135, where the numbers are small)
        scale2 = exp2_fast(0.5f * (all_m - all_top));
        scale *= scale2;
      }
      bool odd = false;
      if (busy) {
        place();
        T* out = static_cast<T*>(a.o) + (static_cast<long long>(tok) * a.kv_heads * a.group + head) * D + c0;
        float* place_of = parts + static_cast<size_t>(x.place) * part_floats<R, D>();
#pragma unroll 1
        for (int ch = 0; ch < kCols / 16; ++ch) {
          float y[16];
          columns(ch, y);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            y[e] *= scale;
            if constexpr (k8) y[e] *= scale2;
            odd |= y[e] != y[e];
          }
          if (mine) {
            if (x.whole) {
              uint4* dst = reinterpret_cast<uint4*>(out + ch * 16);
              dst[0] = make_uint4(Fmt<T>::pack2(y[0], y[1]), Fmt<T>::pack2(y[2], y[3]), Fmt<T>::pack2(y[4], y[5]), Fmt<T>::pack2(y[6], y[7]));
              dst[1] = make_uint4(Fmt<T>::pack2(y[8], y[9]), Fmt<T>::pack2(y[10], y[11]), Fmt<T>::pack2(y[12], y[13]), Fmt<T>::pack2(y[14], y[15]));
            } else {
              float4* dst = reinterpret_cast<float4*>(place_of + row * D + c0 + ch * 16);
#pragma unroll
              for (int e = 0; e < 4; ++e) dst[e] = make_float4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
            }
          }
        }
        // rows that something unseen may have made a NaN are left to the joining kernel, which goes through them key by key
        if (mine) {
          const bool again = odd && x.whole && hides<kWhat>(a, x.pos0 + tok, x.keys.lo, x.keys.hi);
          using Flag = typename std::conditional<kCols == D, uint32_t, uint16_t>::type;
          reinterpret_cast<Flag*>(a.odd + static_cast<long long>(tok) * a.kv_heads * a.group + head)[c0 / kCols] = again ? 1 : 0;
        }
        if (mine && !x.whole && c0 == 0) *reinterpret_cast<float2*>(place_of + R * D + 2 * row) = make_float2(all_top, sum);
        if (mine && x.whole && c0 == 0 && wants_lse<kWhat>(a)) put_lse(a, static_cast<long long>(tok) * a.kv_heads * a.group + head, all_top, sum);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.o_free[kTwo ? t : 0]);
      const bool last = x.last != 0;
      give_back(i);
      if (last) break;
    }
  } else if constexpr (!k8) {
    // ------------------------------------------------ values that nobody of the tile sees become zeros
    for (int i = 0;; ++i) {
      const int at = i % kStretches;
      if (!mbar_wait_warp(&ctl.edge_full[at], (i / kStretches) & 1, s_abort, status, FTB_ERR_TIMEOUT_TMA)) break;
      const Edge e = ctl.edges[at];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.edge_empty[at]);
      // (the products wait for this warp before they give the slot back: the fill is the one that was meant)
      if (e.slot < 0 || !mbar_wait_warp(&ctl.kv_full[e.slot], e.phase, s_abort, status, FTB_ERR_TIMEOUT_TMA)) break;
      uint8_t* tile = sKV + e.slot * P::kTile;
      for (int k = lane; k < kKeys * (D / 8); k += 32) {
        const int key = k / (D / 8), c = k - key * (D / 8);
        if (e.key0 + key < e.lo || e.key0 + key >= e.hi) *reinterpret_cast<uint4*>(piece_ptr(tile, key, c)) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.v_fixed[e.slot]);
    }
  } else {
    // ------------------------------------------------------------- codes to fp16
    // Groups of four warps take the tiles in turn; warp cw of a group converts keys 32 cw .. + 31.  Each warp finds the block's
    // largest exponents on its own: lane i holds the four bytes of keys 4 i .. + 3.
    const int cw = warp & 3, group = (warp - 2 - P::kSoftmax) >> 2;
    constexpr int kGroups = P::kConvert / 4;
    int count = 0, blocks0 = 0;  // tiles and blocks of the stretches so far
    bool ok = true;
    // a lane: piece c of keys first, first + 32 / kRow, ..
    constexpr int kRow = D / 16, kPieces = kRow;
    const int first = cw * 32 + lane / kRow, c = lane % kRow;
    // Where the two halves of a piece go in a tile, rows of `first` apart.  d 128: lanes of the upper half of a row begin with
    // the second one, so that eight lanes reach all banks.
    const bool swap = D == 128 && c >= 4;
    constexpr int kTurns = kRow / 4;  // after so many pieces the rows are 8 apart, and the swizzle is the same again
    uint32_t off[kTurns][2];
#pragma unroll
    for (int k = 0; k < kTurns; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = first + k * (32 / kRow), to = 2 * c + (swap ? 1 - e : e);
        off[k][e] = (to >> 3) * P::kHalf + first * 128 + (((to & 7) ^ (key & 7)) << 4);
      }
    for (int i = 0; ok; ++i) {
      if (!await(i)) break;
      const Stretch& x = ctl.ring[i % kStretches];
      const int tiles = 2 * x.blocks;
      // keys that every row sees: up to the first one's position, from the last one's window on
      const long long all_hi = x.pos0 + x.first + (kWhat == kTrees ? -1 : x.flat0 / a.group);
      const long long all_lo = a.window > 0 ? x.pos0 + x.first + (x.flat0 + x.rows - 1) / a.group - a.window + 1 : 0;
      for (int n = (group - count) & (kGroups - 1); n < tiles && ok; n += kGroups) {
        const StreamTile y = stream_tile<kTwo>(n, x.blocks);
        const int slot = (count + n) % kSlots, raw = (count + n) % kRawSlots;
        const int key0 = (x.block0 + y.j) * kKeys;
        const bool edge = key0 < x.keys.lo || key0 + kKeys > x.keys.hi;
        ok = mbar_wait_warp(&ctl.raw_full[raw], (count + n) / kRawSlots & 1, s_abort, status, FTB_ERR_TIMEOUT_TMA);
        if (!ok) break;
        const uint8_t* from = sRaw + raw * P::kRaw;
        const uint4* src = reinterpret_cast<const uint4*>(from) + first * kRow + c;
        uint4 v[kPieces];
#pragma unroll
        for (int k = 0; k < kPieces; ++k) v[k] = src[k * 32];
        uint32_t kw = reinterpret_cast<const uint32_t*>(from + 128 * D)[lane], vw = reinterpret_cast<const uint32_t*>(from + 128 * D + 128)[lane];
        if (edge) {  // keys that nobody sees: exponents 0
          uint32_t keep = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + 4 * lane + e >= x.keys.lo && key0 + 4 * lane + e < x.keys.hi) keep |= 0xffu << (8 * e);
          kw &= keep;
          vw &= keep;
        }
        // scales of this warp's rows, relative to the block's largest one (rows that are not finite apart)
        auto largest = [](uint32_t w) -> int {
          w &= ~__vcmpeq4(w, 0xffffffffu);
          w = __vmaxu4(w, w >> 16);
          return static_cast<int>(max(1u, max(w & 0xffu, w >> 8 & 0xffu)));
        };
        const uint32_t mine = y.is_v ? vw : kw;
        const int top = __reduce_max_sync(0xffffffffu, largest(mine));
        if (!y.is_v) {
          if (cw == 0) {
            const int ref = (blocks0 + y.j) & (kRefs - 1);
            int v_top = __reduce_max_sync(0xffffffffu, largest(vw)), far = 0;
            if (key0 + kKeys - 1 > all_hi || key0 < all_lo) {
              auto smallest = [](uint32_t w) -> uint32_t {  // (of those above 1: rows of zeros lose nothing, and others with 1, below 2^-117, count as zeros)
                w |= __vcmpleu4(w, 0x01010101u);
                w = __vminu4(w, w >> 16 | w << 16);
                return min(w & 0xffu, w >> 8 & 0xffu);
              };
              if (top - static_cast<int>(__reduce_min_sync(0xffffffffu, smallest(kw))) > kExact ||
                  v_top - static_cast<int>(__reduce_min_sync(0xffffffffu, smallest(vw))) > kExact)
                far = kFar;
            }
            if (lane == 0) {
              ctl.k_ref[ref] = top | far;
              ctl.v_ref[ref] = v_top;
            }
          }
        }
        const int e = __shfl_sync(0xffffffffu, mine, cw * 8 + (lane >> 2)) >> (8 * (lane & 3)) & 0xff;  // of key cw * 32 + lane
        const int below = max(0, top - e);
        // 2^(kUp - below) as fp16
        uint32_t by = below < kExact ? static_cast<uint32_t>(kExact - below) << 10 : below <= 24 + kUp ? 1u << (24 + kUp - below) : 0u;
        by |= by << 16;
        ok = mbar_wait_warp(&ctl.kv_empty[slot], ((count + n) / kSlots & 1) ^ 1u, s_abort, status, FTB_ERR_TIMEOUT_SLOT);
        if (!ok) break;
        uint8_t* tile = sKV + slot * P::kTile;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const int key = first + k * (32 / kRow);
          uint4 w = swap ? make_uint4(v[k].z, v[k].w, v[k].x, v[k].y) : v[k];
          if (edge && y.is_v && (key0 + key < x.keys.lo || key0 + key >= x.keys.hi)) w = make_uint4(0u, 0u, 0u, 0u);
          const uint32_t scale = __shfl_sync(0xffffffffu, by, key & 31);
          uint4 o;
          e4m3x4_to_f16x2(w.x, o.x, o.y);
          e4m3x4_to_f16x2(w.y, o.z, o.w);
          uint8_t* dst = tile + k * (32 / kRow) * 128;
          *reinterpret_cast<uint4*>(dst + off[k % kTurns][0]) = make_uint4(mul_f16x2(o.x, scale), mul_f16x2(o.y, scale), mul_f16x2(o.z, scale), mul_f16x2(o.w, scale));
          e4m3x4_to_f16x2(w.z, o.x, o.y);
          e4m3x4_to_f16x2(w.w, o.z, o.w);
          *reinterpret_cast<uint4*>(dst + off[k % kTurns][1]) = make_uint4(mul_f16x2(o.x, scale), mul_f16x2(o.y, scale), mul_f16x2(o.z, scale), mul_f16x2(o.w, scale));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ctl.raw_empty[raw]);
          mbar_arrive(&ctl.kv_full[slot]);
        }
      }
      const bool last = x.last != 0;
      blocks0 += x.blocks;
      give_back(i);
      count += tiles;
      if (last) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (ctl.abort) {
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <typename T, bool k8, int D, int R, int kWhat>
int launch(const PagedAttn& a, const CUtensorMap& mK, const CUtensorMap& mV, void* scratch, cudaStream_t stream) {
  using P = Plan<k8, D, R, kWhat>;
  static std::atomic<unsigned long long> configured{0};
  auto kfn = paged_tile_kernel<T, k8, D, R, kWhat>;
  if (!ensure_dynamic_smem(kfn, P::kSmem, configured)) return FTB_ERR_LAUNCH;
  const int pieces = paged_tile_pieces();
  float* parts = static_cast<float*>(scratch);
  const cudaError_t err = launch_dependent(kfn, dim3(pieces), dim3(P::kThreads), P::kSmem, stream, a, mK, mV, parts,
                                           reinterpret_cast<PagedCut*>(parts + 2 * pieces * part_floats<R, D>()));
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}
template <typename T, bool k8, int D, int R>
int launch(const PagedAttn& a, const CUtensorMap& mK, const CUtensorMap& mV, void* scratch, cudaStream_t stream) {
  return a.tree != nullptr  ? launch<T, k8, D, R, kTrees>(a, mK, mV, scratch, stream)
         : a.lse != nullptr ? launch<T, k8, D, R, kLse>(a, mK, mV, scratch, stream)
                            : launch<T, k8, D, R, kPlain>(a, mK, mV, scratch, stream);
}
template <typename T, int D, int R>
int launch(const PagedAttn& a, int dtype, void* scratch, cudaStream_t stream) {
  CUtensorMap mK = {}, mV = {};
  const uint64_t rows = (static_cast<uint64_t>(a.batch.pages) * a.kv_heads) << a.batch.page_shift;
  if (a.k_exp != nullptr) return launch<T, true, D, R>(a, mK, mV, scratch, stream);
  if (rows > 0x7fffffffull) return FTB_ERR_ARG;  // a copy's coordinates have 32 bits
  int rc;
  if ((rc = make_tmap_2d(&mK, a.k, dtype, rows, D, D, 1u << a.batch.page_shift, 64))) return rc;
  if ((rc = make_tmap_2d(&mV, a.v, dtype, rows, D, D, 1u << a.batch.page_shift, 64))) return rc;
  return launch<T, false, D, R>(a, mK, mV, scratch, stream);
}
template <typename T, int D>
int launch(const PagedAttn& a, int dtype, int rows, void* scratch, cudaStream_t stream) {
  return rows == 256 ? launch<T, D, 256>(a, dtype, scratch, stream) : launch<T, D, 128>(a, dtype, scratch, stream);
}

}  // namespace

int paged_tile_pieces() { return current_sm_count(); }

int paged_tile_launch(const PagedAttn& a, int d, int dtype, int rows, void* scratch, cudaStream_t stream) {
  if (dtype == FTB_F16) return d == 128 ? launch<__half, 128>(a, dtype, rows, scratch, stream) : launch<__half, 64>(a, dtype, rows, scratch, stream);
  return d == 128 ? launch<__nv_bfloat16, 128>(a, dtype, rows, scratch, stream) : launch<__nv_bfloat16, 64>(a, dtype, rows, scratch, stream);
}

}  // namespace ftb
