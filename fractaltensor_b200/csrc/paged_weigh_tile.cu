// Attention weight added up over a paged cache for many rows: chunks of prompts.  Blocks of 256 keys against tiles of 128 rows (token, head of a
// group) on the tensor cores (tcgen05), S^T = K Q^T with the keys on the M side, so that a key is a lane of tensor memory and its sum of
// exp(scale * q . k - lse) is one thread's, without a maximum to look for and without a second product.
//
// The rows are packed first, one kv head's behind another's, in the type of the products (over 8-bit caches fp16, bf16 rows
// divided by a power of two as in paged_short.cu), with what is taken from a score, lse in log2.  A row whose lse is not finite is packed
// as zeros and takes away infinity.
//
// One persistent CTA per SM takes an equal piece of the line of work, whose unit is a tile of rows against a block:
//   warp 0        the walk, announced through a ring of stretches, and the loads of the rows (TMA)
//   warp 1        issues the products, into one of two buffers of scores
//   warps 2..17   exponentials and sums, while the next tile's scores are made: a thread has a key of either half of the block and a quarter
//                 of the tile's rows
//   warps 18..21  load the keys of the next block, all of them on their way at once (8 at a time a warp: 332 for 142 us of 48 sequences of 4000 keys,
//                 64 rows), and make 8-bit codes fp16; a key's scale goes to its scores
// A block that a cut goes through leaves parts of its sums, which a second kernel adds up in their order.
//
// A score is one sum of the tensor core over all of d, which cuts off downwards: a chunk's weights are 3.4e-7 off (paged_weigh.cu has two sums for that reason).  Warps with a key
// that is not there, in a sequence's last block, go number by number.
//
// 2048 tokens of 32 heads of 128 over 8 kv heads, 16 384 keys of 8 bits: 331 us, 0.78 PFLOP/s.  Bound by no unit alone: without the
// exponentials (16 a cycle and SM, 245 us) it takes 285 us, without the products (122) 324, with neither 173, which is the rows' way from L2 for
// every block and the hand-overs between the warps.  Measured and not kept: a quarter to a half of the exponentials by a polynomial on the units that
// multiply and add (334 to 383 us), blocks of 512 keys (346), eight warps for the sums (352), each half of the warps with a buffer of its own (351).
// A few dozen rows behind a long sequence are bound by what comes before the first load: a thread of every CTA goes through the sequence's blocks, up to three times.  32 rows behind
// 131 072 keys, 8 kv heads: 178 us (42 by the keys' bytes), behind 524 288 keys of 8 bits of one kv head 449 (11).
#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "../../include/ftb200.h"
#include "paged_weigh.cuh"
#include "tmap.h"

namespace ftb {
namespace {

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kBlock = 256, kRows = 128, kSplit = 4, kPart = kRows / kSplit, kStretches = 4, kBeside = 4, kSums = 16, kLoaders = 4, kThreads = 32 * (2 + kSums + kLoaders), kPackThreads = 256;

// Rows as the products take them: [kv_heads][T * group][d], with [kv_heads][T * group] numbers each.
struct Packed {
  void* q;
  float* minus;
  float* factor;  // of a score, where it is not the same for all
};

template <typename T, bool k8, int D>
__global__ void __launch_bounds__(kPackThreads)
paged_weigh_pack_kernel(const __grid_constant__ Weigh x, Packed to, long long rows) {
  using C = typename std::conditional<k8, __half, T>::type;
  constexpr int kLanes = D / 8;  // of a row, 16 bytes each
  const PagedAttn& a = x.attn;
  const long long row = (static_cast<long long>(blockIdx.x) * kPackThreads + threadIdx.x) / kLanes;  // token, head
  const int lane = threadIdx.x % kLanes, heads = a.kv_heads * a.group;
  grid_launch_dependents();
  grid_dependency_wait();
  if (row >= rows) return;  // (the lanes of a row leave together)
  const int t = static_cast<int>(row / heads), head = static_cast<int>(row - static_cast<long long>(t) * heads);
  uint4 v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + t * a.q_row + head * a.q_head + lane * 8);
  const float lse = x.lse[row];
  const bool fine = fabsf(lse) < INFINITY;
  float factor = a.scale_log2;
  if constexpr (!std::is_same<T, C>::value) {
    uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    m = max(m & 0xffffu, m >> 16);
    const unsigned mask = D == 128 ? 0xffffu << (threadIdx.x & 16) : 0xffu << (threadIdx.x & 24);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(mask, m, o));
    const int e = min(253, max(1, static_cast<int>(m >> 7)));
    const float by = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
    factor *= __uint_as_float(static_cast<uint32_t>(e) << 23);
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(w[i]);
      w[i] = Fmt<C>::pack2(f.x * by, f.y * by);
    }
  }
  if (!fine) v = make_uint4(0u, 0u, 0u, 0u);
  const int h = head / a.group;
  const long long at = static_cast<long long>(h) * a.T * a.group + static_cast<long long>(t) * a.group + (head - h * a.group);
  reinterpret_cast<uint4*>(to.q)[at * kLanes + lane] = v;
  if (lane == 0) {
    to.minus[at] = fine ? -lse * kLog2E : -INFINITY;
    if (to.factor != nullptr) to.factor[at] = factor;
  }
}

// A stretch of a block that a piece works on: rows flat0 .. flat1 - 1 of kv head h, in tiles.
struct Stretch {
  int b, h, key0, flat0, flat1, first, tiles;
  PagedKeys keys;  // of the sequence
  long long base;  // position of its new tokens
  int whole, place, last;
};

// Rows that see some key of a block, and the tiles that they make.
struct BlockRows {
  int flat0, flat1, tiles;
};
__device__ __forceinline__ BlockRows rows_of_block(const PagedAttn& a, const PagedSeq& s, const PagedKeys& keys, int block) {
  const long long base = s.pos0 + s.first;
  const int k0 = max(block * kBlock, keys.lo), k1 = min((block + 1) * kBlock, keys.hi);  // block * kBlock < keys.hi
  BlockRows r;
  r.flat0 = static_cast<int>(min(static_cast<long long>(s.flats), max(0ll, k0 - base) * a.group));
  r.flat1 = a.window > 0 ? static_cast<int>(min(static_cast<long long>(s.flats), max(0ll, static_cast<long long>(a.window) + k1 - 1 - base) * a.group)) : s.flats;
  r.tiles = r.flat1 > r.flat0 ? (r.flat1 - r.flat0 + kRows - 1) / kRows : 0;
  return r;
}
__device__ __forceinline__ long long tiles_of_head(const PagedAttn& a, const PagedSeq& s) {
  const PagedKeys keys = all_keys(a, s);
  long long sum = 0;
  for (int block = keys.lo / kBlock, n = blocks_of<kBlock>(keys); n > 0; ++block, --n) sum += rows_of_block(a, s, keys, block).tiles;
  return sum;
}

// The tiles of a stretch with rows that see a key of the block's half h: first .. last - 1.
struct Tiles {
  int first, last;
};
__device__ __forceinline__ Tiles tiles_of_half(const PagedAttn& a, const Stretch& y, int h) {
  const int k0 = max(y.key0 + h * 128, y.keys.lo), k1 = min(y.key0 + (h + 1) * 128, y.keys.hi);
  if (k0 >= k1) return {0, 0};
  const long long f0 = max(0ll, k0 - y.base) * a.group - y.flat0;
  long long f1 = y.flat1 - y.flat0;
  if (a.window > 0) f1 = min(f1, max(0ll, static_cast<long long>(a.window) + k1 - 1 - y.base) * a.group - y.flat0);
  return {static_cast<int>(max(0ll, f0) / kRows), static_cast<int>((max(0ll, f1) + kRows - 1) / kRows)};
}

struct Cut {
  int last;  // the last piece with a part; -1: nothing to add up
  int b, h, key0;
  PagedKeys keys;
  long long base;
};

template <int D, bool kFactors>
struct Plan {
  static constexpr int kHalf = 128 * 128, kTile = D / 64 * kHalf;  // 128 rows of 64 and of d numbers
  static constexpr int kStages = D == 128 ? 2 : 4;
};

template <int D, bool kFactors>
struct Control {
  using P = Plan<D, kFactors>;
  // what goes with the rows of a tile, in a ring of its own: the rows' room is free again when the products are done
  alignas(16) float minus[kBeside][kRows], factor[kFactors ? kBeside : 1][kRows];
  int odd[kBeside];           // whether some row adds nothing
  float scale[2][kBlock];     // of a key's scores; of every second stretch, as the next one
  int row[2][kBlock];         // of the cache, -1: none
  PagedLineRoom line;
  Stretch ring[kStretches];
  uint64_t ring_full[kStretches], ring_empty[kStretches];
  uint64_t q_full[P::kStages], q_empty[P::kStages], beside_full[kBeside], beside_empty[kBeside], k_full[2], k_empty[2], s_full[2], s_empty[2], other_full[2];
  float other[2][kSplit - 1][kBlock];  // sums over the other quarters of the tiles
  uint32_t tmem_base;
  int abort, dead;
};

template <typename T, bool k8, int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_weigh_tile_kernel(const __grid_constant__ Weigh x, const __grid_constant__ CUtensorMap mapQ, Packed packed, float* __restrict__ parts, Cut* __restrict__ cuts) {
  using C = typename std::conditional<k8, __half, T>::type;
  constexpr bool kFactors = !std::is_same<T, C>::value;
  using P = Plan<D, kFactors>;
  constexpr int kStages = P::kStages;
  const PagedAttn& a = x.attn;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sK = smem, *sQ = sK + 4 * P::kTile;
  Control<D, kFactors>& ctl = *reinterpret_cast<Control<D, kFactors>*>(sQ + kStages * P::kTile);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = blockIdx.x;
  volatile int* s_abort = &ctl.abort;
  int* status = a.status;

  if (threadIdx.x == 0) {
    prefetch_tmap(&mapQ);
    for (int i = 0; i < kStretches; ++i) {
      mbar_init(&ctl.ring_full[i], 1);
      mbar_init(&ctl.ring_empty[i], 1 + kSums + kLoaders);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&ctl.q_full[i], 1);
      mbar_init(&ctl.q_empty[i], 1);
    }
    for (int i = 0; i < kBeside; ++i) {
      mbar_init(&ctl.beside_full[i], 1);
      mbar_init(&ctl.beside_empty[i], kSums);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.k_full[i], kLoaders);
      mbar_init(&ctl.k_empty[i], 1 + kSums);
      mbar_init(&ctl.s_full[i], 1);
      mbar_init(&ctl.s_empty[i], kSums);
      mbar_init(&ctl.other_full[i], kSums - kSums / kSplit);
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
  int seq;
  long long at;
  const PagedLine line = paged_line_of(a, piece, gridDim.x, 1, ctl.line, &seq, &at, [&](const PagedSeq& s) { return tiles_of_head(a, s); });
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
  const uint32_t tmem_base = ctl.tmem_base;  // scores: buffer p, half h of the keys: columns 256 p + 128 h .. + 127

  auto await = [&](int i) -> bool {
    return mbar_wait_warp(&ctl.ring_full[i % kStretches], (i / kStretches) & 1, s_abort, status, FTB_ERR_TIMEOUT_TMA);
  };
  auto give_back = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.ring_empty[i % kStretches]);
  };

  if (warp == 0) {
    // ------------------------------------------------------------- the walk, and the rows
    fence_proxy_async_all();  // (the rows have been packed by ordinary stores)
    long long u = piece_begin(line, piece);
    const long long u_end = piece_begin(line, piece + 1);
    PagedSeq s = paged_sequence(a, seq);
    PagedKeys keys = all_keys(a, s);
    int blocks = blocks_of<kBlock>(keys), h, n = 0;  // n: of the sequence's blocks
    {
      const long long per = tiles_of_head(a, s);
      h = static_cast<int>((u - at) / per);
      at += per * h;
    }
    int published = 0;
    // Finds the stretch that unit u is in, announces it and moves on.
    auto publish = [&](Stretch& y) -> bool {
      BlockRows r;
      for (;;) {
        r = n < blocks ? rows_of_block(a, s, keys, keys.lo / kBlock + n) : BlockRows{0, 0, 0};
        if (u < at + r.tiles) break;
        at += r.tiles;
        if (++n < blocks) continue;
        n = 0;
        if (blocks > 0 && ++h < a.kv_heads) continue;
        h = 0;
        do {
          s = paged_sequence(a, ++seq);
          keys = all_keys(a, s);
          blocks = blocks_of<kBlock>(keys);
        } while (blocks == 0);
      }
      const int r0 = static_cast<int>(u - at), r1 = static_cast<int>(min(static_cast<long long>(r.tiles), u_end - at));
      y.b = seq;
      y.h = h;
      y.key0 = (keys.lo / kBlock + n) * kBlock;
      y.flat0 = r.flat0 + r0 * kRows;
      y.flat1 = min(r.flat1, r.flat0 + r1 * kRows);
      y.first = s.first;
      y.tiles = r1 - r0;
      y.keys = keys;
      y.base = s.pos0 + s.first;
      y.whole = r0 == 0 && r1 == r.tiles;
      y.place = 2 * piece + (r0 == 0 ? 1 : 0);
      y.last = at + r1 >= u_end;
      const int i = published++;
      if (i >= kStretches && !mbar_wait_warp(&ctl.ring_empty[i % kStretches], (i / kStretches - 1) & 1, s_abort, status, FTB_ERR_TIMEOUT_SLOT)) return false;
      if (lane == 0) {
        ctl.ring[i % kStretches] = y;
        mbar_arrive(&ctl.ring_full[i % kStretches]);
        if (i == 0) {
          PagedTile t;
          t.begin = at;
          t.units = r.tiles;
          t.r0 = r0;
          const int last = last_piece_of(line, piece, t);
          cuts[piece].last = last;
          if (last >= 0) cuts[piece] = Cut{last, seq, h, y.key0, keys, y.base};
        }
      }
      u = at + r1;
      return true;
    };
    const long long all = static_cast<long long>(a.T) * a.group, numbers = all * a.kv_heads;
    Stretch now, next;
    bool ok = publish(next);
    int stage = 0, tile = 0;
    uint32_t phase = 0;
    for (bool more = true; ok && more;) {
      now = next;
      more = !now.last;
      if (more) ok = publish(next);  // (a block ahead, for the warps that load keys)
      const long long row0 = now.h * all + static_cast<long long>(now.first) * a.group;
      float4 minus, factor;
      auto fetch = [&](int flat) {  // four numbers of a tile a lane
        const long long i = row0 + flat + lane * 4;
        auto take = [&](const float* p, int k) { return i + k < numbers ? p[i + k] : 0.f; };
        minus = make_float4(take(packed.minus, 0), take(packed.minus, 1), take(packed.minus, 2), take(packed.minus, 3));
        if constexpr (kFactors) factor = make_float4(take(packed.factor, 0), take(packed.factor, 1), take(packed.factor, 2), take(packed.factor, 3));
      };
      fetch(now.flat0);
      for (int k = 0; ok && k < now.tiles; ++k, ++tile) {
        const int flat = now.flat0 + k * kRows, beside = tile % kBeside;
        ok = mbar_wait_warp(&ctl.beside_empty[beside], ((tile / kBeside) & 1) ^ 1u, s_abort, status, FTB_ERR_TIMEOUT_SLOT);
        if (!ok) break;
        reinterpret_cast<float4*>(ctl.minus[beside])[lane] = minus;
        if constexpr (kFactors) reinterpret_cast<float4*>(ctl.factor[beside])[lane] = factor;
        const bool odd = __any_sync(0xffffffffu, fminf(fminf(minus.x, minus.y), fminf(minus.z, minus.w)) == -INFINITY);
        if (lane == 0) ctl.odd[beside] = odd;
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.beside_full[beside]);
        ok = mbar_wait_warp(&ctl.q_empty[stage], phase ^ 1u, s_abort, status, FTB_ERR_TIMEOUT_SLOT);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&ctl.q_full[stage], P::kTile);
          const int y = static_cast<int>(row0 + flat);
          tma_load_2d(sQ + stage * P::kTile, &mapQ, &ctl.q_full[stage], 0, y);
          if constexpr (D == 128) tma_load_2d(sQ + stage * P::kTile + P::kHalf, &mapQ, &ctl.q_full[stage], 64, y);
        }
        if (k + 1 < now.tiles) fetch(flat + kRows);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------- the products
    const bool leader = elect_one();
    constexpr uint32_t idesc = make_idesc_f16(128, 128, Fmt<C>::kind, 0, 0);
    const uint64_t dK = make_sdesc_sw128(smem_u32(sK), 16, 1024), dQ = make_sdesc_sw128(smem_u32(sQ), 16, 1024);
    int stage = 0, tile = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!await(i)) break;
      const Stretch y = ctl.ring[i % kStretches];
      give_back(i);
      const int buffer = i & 1;
      const Tiles met[2] = {tiles_of_half(a, y, 0), tiles_of_half(a, y, 1)};
      ok = mbar_wait_warp(&ctl.k_full[buffer], (i >> 1) & 1, s_abort, status, FTB_ERR_TIMEOUT_TMA);
      for (int k = 0; ok && k < y.tiles; ++k, ++tile) {
        const int p = tile & 1;
        ok = mbar_wait_warp(&ctl.q_full[stage], phase, s_abort, status, FTB_ERR_TIMEOUT_TMA) &&
             mbar_wait_warp(&ctl.s_empty[p], ((tile >> 1) & 1) ^ 1u, s_abort, status, FTB_ERR_TIMEOUT_EPI);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (k < met[h].first || k >= met[h].last) continue;
            const uint64_t dk = dK + static_cast<uint64_t>(((buffer * 2 + h) * P::kTile) >> 4), dq = dQ + static_cast<uint64_t>((stage * P::kTile) >> 4);
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              const uint32_t off = ((j >> 2) * P::kHalf + (j & 3) * 32) >> 4;
              umma_ss(tmem_base + p * 256 + h * 128, dk + off, dq + off, idesc, j != 0 ? 1u : 0u);
            }
          }
          umma_commit(&ctl.s_full[p]);
          umma_commit(&ctl.q_empty[stage]);
          if (k + 1 == y.tiles) umma_commit(&ctl.k_empty[buffer]);
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (y.last) break;
    }
  } else if (warp < 2 + kSums) {
    // ------------------------------------------------ exponentials and sums: key `mine` of a block
    const int part = (warp - 2) >> 2, quad = warp & 3, lane_key = quad * 32 + lane;
    const uint32_t addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + part * kPart;
    int tile = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!await(i)) break;
      const Stretch& y = ctl.ring[i % kStretches];
      const int buffer = i & 1, tiles = y.tiles;
      ok = mbar_wait_warp(&ctl.k_full[buffer], (i >> 1) & 1, s_abort, status, FTB_ERR_TIMEOUT_TMA);
      if (!ok) break;
      // of this thread's keys: the rows that see one lie side by side, from .. to - 1 counted from the stretch's first one
      int from[2], to[2];
      float scale[2], sum[2] = {0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = y.key0 + h * 128 + lane_key;
        long long see0 = 0, see1 = 0;
        if (key >= y.keys.lo && key < y.keys.hi) {
          see0 = max(0ll, key - y.base) * a.group - y.flat0;
          see1 = y.flat1 - y.flat0;
          if (a.window > 0) see1 = min(see1, max(0ll, static_cast<long long>(a.window) + key - y.base) * a.group - y.flat0);
        }
        from[h] = static_cast<int>(max(0ll, see0)) - part * kPart;
        to[h] = static_cast<int>(max(0ll, see1)) - part * kPart;
        scale[h] = ctl.scale[buffer][h * 128 + lane_key];
      }
      // Tiles whose rows this warp's keys see all of.  (In the others a key sees none, or rows from .. to - 1.)
      const int plain0 = __reduce_max_sync(0xffffffffu, max(max(from[0], from[1]), 0) + kRows - 1) / kRows;
      const int plain1 = __reduce_min_sync(0xffffffffu, max(min(to[0], to[1]) + kRows - kPart, 0)) / kRows;
      for (int k = 0; k < tiles; ++k, ++tile) {
        const int p = tile & 1, beside = tile % kBeside;
        ok = mbar_wait_warp(&ctl.beside_full[beside], (tile / kBeside) & 1, s_abort, status, FTB_ERR_TIMEOUT_TMA) &&
             mbar_wait_warp(&ctl.s_full[p], (tile >> 1) & 1, s_abort, status, FTB_ERR_TIMEOUT_MMA);
        if (!ok) break;
        tc_fence_after();
        const uint32_t s_addr = addr + p * 256;
        const float *minus = ctl.minus[beside] + part * kPart, *factor = ctl.factor[kFactors ? beside : 0] + (kFactors ? part * kPart : 0);
        auto give_back_scores = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl.s_empty[p]);
        };
        if (k >= plain0 && k < plain1 && ctl.odd[beside] == 0) {
          // (both keys' scores beside one another: what goes with a row comes out of shared memory once for them.  And the scores' room is
          // given back as soon as they are in registers: what is to do with them does not hold up the products.)
          uint64_t sum2[2][2] = {};
#pragma unroll
          for (int n = 0; n < kPart / 16; ++n) {
            uint32_t s[2][16];
            tmem_ld16(s_addr + n * 16, s[0]);
            tmem_ld16(s_addr + 128 + n * 16, s[1]);
            tmem_ld_wait();
            if (n + 1 == kPart / 16) give_back_scores();
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
              const ulonglong2 m = *reinterpret_cast<const ulonglong2*>(minus + n * 16 + c);
              float4 f;
              if constexpr (kFactors) f = *reinterpret_cast<const float4*>(factor + n * 16 + c);
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint64_t s2 = pair_f32x2(__uint_as_float(s[h][c + 2 * e]), __uint_as_float(s[h][c + 2 * e + 1]));
                  uint64_t f2 = dup_f32x2(scale[h]);
                  if constexpr (kFactors)
                    f2 = pair_f32x2(fminf((e == 0 ? f.x : f.z) * scale[h], FLT_MAX), fminf((e == 0 ? f.y : f.w) * scale[h], FLT_MAX));
                  const uint64_t x2 = fma_to_f32x2(s2, f2, e == 0 ? m.x : m.y);
                  float p0, p1;
                  unpair_f32x2(x2, p0, p1);
                  add_f32x2(sum2[h][e], pair_f32x2(exp2_fast(p0), exp2_fast(p1)));
                }
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            add_f32x2(sum2[h][0], sum2[h][1]);
            float p0, p1;
            unpair_f32x2(sum2[h][0], p0, p1);
            sum[h] += p0 + p1;
          }
        } else {
          // at the edges, and where rows that add nothing may have met something that is not finite: number by number
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const float by = h == 0 ? scale[0] : scale[1];
            const int lo = max(0, (h == 0 ? from[0] : from[1]) - k * kRows), hi = min(kPart, (h == 0 ? to[0] : to[1]) - k * kRows);
            if (__all_sync(0xffffffffu, lo >= hi)) continue;  // (no scores have been made where nobody sees one)
            float all = 0.f;
#pragma unroll 1
            for (int c0 = 0; c0 < kPart; c0 += 16) {
              uint32_t s[16];
              tmem_ld16(s_addr + h * 128 + c0, s);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const float m = minus[c0 + c], f = kFactors ? fminf(factor[c0 + c] * by, FLT_MAX) : by;
                const bool counts = c0 + c >= lo && c0 + c < hi && m > -INFINITY;
                all += counts ? exp2_fast(fmaf(__uint_as_float(s[c]), f, m)) : 0.f;
              }
            }
            if (h == 0) sum[0] += all;
            else sum[1] += all;
          }
          give_back_scores();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.beside_empty[beside]);
      }
      if (!ok) break;
      if (part != 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) ctl.other[buffer][part - 1][h * 128 + lane_key] = sum[h];
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.other_full[buffer]);
      } else {
        ok = mbar_wait_warp(&ctl.other_full[buffer], (i >> 1) & 1, s_abort, status, FTB_ERR_TIMEOUT_EPI);
        if (!ok) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int mine = h * 128 + lane_key, key = y.key0 + mine, row = ctl.row[buffer][mine];
          float all = sum[h];
#pragma unroll
          for (int o = 0; o < kSplit - 1; ++o) all += ctl.other[buffer][o][mine];
          if (!y.whole) parts[static_cast<long long>(y.place) * kBlock + mine] = all;
          else if (row >= 0) x.weights[row] = key >= y.base ? all : x.weights[row] + all;
        }
      }
      const bool last = y.last != 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.k_empty[buffer]);
      give_back(i);
      if (last) break;
    }
  } else {
    // ------------------------------------------------------------- the keys: 64 of a block a warp
    const int of_block = (warp - 2 - kSums) * 64;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!await(i)) break;
      const Stretch& y = ctl.ring[i % kStretches];
      const int buffer = i & 1;
      const int* table = a.batch.table + static_cast<long long>(y.b) * a.batch.W;
      int rows[2];
      float scales[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // lane's keys
        const int key = y.key0 + of_block + e * 32 + lane;
        rows[e] = -1;
        if (key >= y.keys.lo && key < y.keys.hi) {
          const int page = table[key >> a.batch.page_shift];
          if (page >= 0 && page < a.batch.pages)
            rows[e] = ((page * a.kv_heads + y.h) << a.batch.page_shift) + (key & ((1 << a.batch.page_shift) - 1));
          else
            atomicCAS(status, 0, FTB_ERR_INDEX);
        }
        scales[e] = kFactors ? 1.f : a.scale_log2;
        if constexpr (k8) scales[e] = rows[e] >= 0 ? fminf(scales[e] * exponent_scale(a.k_exp[rows[e]]), FLT_MAX) : 1.f;
      }
      ok = mbar_wait_warp(&ctl.k_empty[buffer], ((i >> 1) & 1) ^ 1u, s_abort, status, FTB_ERR_TIMEOUT_SLOT);
      if (!ok) break;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ctl.row[buffer][of_block + e * 32 + lane] = rows[e];
        ctl.scale[buffer][of_block + e * 32 + lane] = scales[e];
      }
      uint8_t* tile = sK + (buffer * 2 + (of_block >> 7)) * P::kTile;
      // 16 bytes of a row of the cache a lane, as many on their way as there are: 16-bit rows straight into their places, codes by way of registers
      constexpr int kPieces = k8 ? D / 16 : D / 8, kTogether = 32 / kPieces, kTurns = 64 / kTogether;
      const int piece_of = lane % kPieces;
      auto put_at = [&](int q, int r) { return tile + (q >> 3) * P::kHalf + r * 128 + (((q & 7) ^ (r & 7)) << 4); };
      if constexpr (k8) {
        uint4 v[kTurns];
#pragma unroll
        for (int k = 0; k < kTurns; ++k) {
          const int row = __shfl_sync(0xffffffffu, rows[k * kTogether / 32], k * kTogether % 32 + lane / kPieces);
          v[k] = row >= 0 ? *reinterpret_cast<const uint4*>(a.k + static_cast<long long>(row) * D + piece_of * 16) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int k = 0; k < kTurns; ++k) {
          const int r = (of_block & 64) + k * kTogether + lane / kPieces;
          uint4 o;
          e4m3x4_to_f16x2(v[k].x, o.x, o.y);
          e4m3x4_to_f16x2(v[k].y, o.z, o.w);
          *reinterpret_cast<uint4*>(put_at(2 * piece_of, r)) = o;
          e4m3x4_to_f16x2(v[k].z, o.x, o.y);
          e4m3x4_to_f16x2(v[k].w, o.z, o.w);
          *reinterpret_cast<uint4*>(put_at(2 * piece_of + 1, r)) = o;
        }
      } else {
#pragma unroll
        for (int k = 0; k < kTurns; ++k) {
          const int row = __shfl_sync(0xffffffffu, rows[k * kTogether / 32], k * kTogether % 32 + lane / kPieces);
          copy16_async(reinterpret_cast<float*>(put_at(piece_of, (of_block & 64) + k * kTogether + lane / kPieces)),
                       reinterpret_cast<const float*>(a.k + static_cast<long long>(max(row, 0)) * (2 * D) + piece_of * 16), row >= 0);
        }
        copies_commit();
        copies_wait();
      }
      fence_proxy_async_smem();
      const bool last = y.last != 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.k_full[buffer]);
      give_back(i);
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

// The blocks that cuts go through: a key a thread.
__global__ void __launch_bounds__(kBlock)
paged_weigh_join_kernel(const __grid_constant__ Weigh x, const float* __restrict__ parts, const Cut* __restrict__ cuts) {
  const PagedAttn& a = x.attn;
  const int piece = blockIdx.x;
  grid_launch_dependents();
  grid_dependency_wait();
  const Cut c = cuts[piece];
  const int key = c.key0 + static_cast<int>(threadIdx.x);
  if (c.last < 0 || key < c.keys.lo || key >= c.keys.hi) return;
  const int page = a.batch.table[static_cast<long long>(c.b) * a.batch.W + (key >> a.batch.page_shift)];
  if (page < 0 || page >= a.batch.pages) return;  // (which has been said)
  // of piece - 1, which left the block's first rows in its second place, and of the others, in their first
  float sum = parts[(static_cast<long long>(piece - 1) * 2 + 1) * kBlock + threadIdx.x];
  for (int p = piece; p <= c.last; ++p) sum += parts[static_cast<long long>(p) * 2 * kBlock + threadIdx.x];
  float* w = x.weights + (((static_cast<long long>(page) * a.kv_heads + c.h) << a.batch.page_shift) + (key & ((1 << a.batch.page_shift) - 1)));
  *w = key >= c.base ? sum : *w + sum;
}

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
size_t packed_rows(int T, int kv_heads, int group) { return std::max(static_cast<size_t>(T) * kv_heads * group, static_cast<size_t>(kRows)); }

int launched(cudaError_t err) {
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}

template <typename T, bool k8, int D>
int launch(const Weigh& x, void* scratch, cudaStream_t stream) {
  using C = typename std::conditional<k8, __half, T>::type;
  constexpr bool kFactors = !std::is_same<T, C>::value;
  using P = Plan<D, kFactors>;
  constexpr int kSmem = 1024 + (4 + P::kStages) * P::kTile + static_cast<int>(sizeof(Control<D, kFactors>));
  static_assert(kSmem <= 232448, "shared memory budget");
  static std::atomic<unsigned long long> configured{0};
  auto kfn = paged_weigh_tile_kernel<T, k8, D>;
  if (!ensure_dynamic_smem(kfn, kSmem, configured)) return FTB_ERR_LAUNCH;
  const PagedAttn& a = x.attn;
  const size_t all = packed_rows(a.T, a.kv_heads, a.group);
  unsigned char* at = static_cast<unsigned char*>(scratch);
  auto take = [&](size_t n) {
    void* p = at;
    at += rounded(n);
    return p;
  };
  Packed packed;
  packed.q = take(all * D * 2);
  packed.minus = static_cast<float*>(take(all * sizeof(float)));
  packed.factor = static_cast<float*>(take(all * sizeof(float)));
  if (!kFactors) packed.factor = nullptr;
  const int pieces = current_sm_count();
  float* parts = static_cast<float*>(take(2 * static_cast<size_t>(pieces) * kBlock * sizeof(float)));
  Cut* cuts = static_cast<Cut*>(take(pieces * sizeof(Cut)));
  CUtensorMap map = {};
  int rc = make_tmap_2d(&map, packed.q, std::is_same<C, __half>::value ? FTB_F16 : FTB_BF16, all, D, D, kRows, 64);
  if (rc) return rc;
  const long long rows = static_cast<long long>(a.T) * a.kv_heads * a.group;
  constexpr int kRowsOfBlock = kPackThreads / (D / 8);
  rc = launched(launch_light(paged_weigh_pack_kernel<T, k8, D>, dim3(static_cast<unsigned>((rows + kRowsOfBlock - 1) / kRowsOfBlock)), dim3(kPackThreads), 0,
                             stream, x, packed, rows));
  if (rc) return rc;
  rc = launched(launch_dependent(kfn, dim3(pieces), dim3(kThreads), kSmem, stream, x, map, packed, parts, cuts));
  if (rc) return rc;
  return launched(launch_light(paged_weigh_join_kernel, dim3(pieces), dim3(kBlock), 0, stream, x, parts, cuts));
}
template <typename T, int D>
int launch(const Weigh& x, void* scratch, cudaStream_t stream) {
  return x.attn.k_exp != nullptr ? launch<T, true, D>(x, scratch, stream) : launch<T, false, D>(x, scratch, stream);
}
template <typename T>
int launch(const Weigh& x, int d, void* scratch, cudaStream_t stream) {
  return d == 128 ? launch<T, 128>(x, scratch, stream) : launch<T, 64>(x, scratch, stream);
}

}  // namespace

size_t paged_weigh_tile_scratch(int T, int kv_heads, int group, int d) {
  const size_t all = packed_rows(T, kv_heads, group);
  const size_t pieces = current_sm_count();
  return rounded(all * d * 2) + 2 * rounded(all * sizeof(float)) + rounded(2 * pieces * kBlock * sizeof(float)) + rounded(pieces * sizeof(Cut));
}

int paged_weigh_tile_launch(const Weigh& x, int d, int dtype, void* scratch, cudaStream_t stream) {
  return dtype == FTB_F16 ? launch<__half>(x, d, scratch, stream) : launch<__nv_bfloat16>(x, d, scratch, stream);
}

}  // namespace ftb
