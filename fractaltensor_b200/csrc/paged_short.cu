// Attention over a paged cache for few rows: a token or a few drafts of each sequence, up to 16 rows (token, head of a
// group) to a tile.
//
// 64 sequences of up to 8000 keys, 8 kv heads of 128, a token of 32 heads each: 182 us, 6.1 TB/s of keys and values; one of 100 001 keys
// of 4 kv heads 50 us with the join, 4.1 TB/s.  Bound by the bytes of the keys and values, which go from global memory into the registers that the products take them
// from, without a stop in shared memory: with the keys on the M side, S^T = K Q^T and O^T = V^T P^T
// (mma.m16n8k16), every lane's pieces of K and V are 16 contiguous bytes of a row, because the order of d under the sum, of
// the keys under the other, and of the output's rows is free:
//   S^T  lane (g, c) = (lane / 4, lane % 4) holds d = 32 j + 8 c .. + 7 of keys g and g + 8 (8-bit: 64 j + 16 c .. + 15), and
//        the same numbers of query g as the other operand
//   O^T  lane (g, c) holds d = 64 x + 8 g .. + 7 (8-bit, d 128: 16 g .. + 15) of keys 2c, 2c + 1, 2c + 8, 2c + 9: pairs of keys are put
//        together by byte permutes
// and P^T is the transpose of what the first product leaves, 8 x 8 numbers an instruction (movmatrix).
// A warp walks every fourth chunk of 16 keys of its CTA's piece on its own, with its own maximum and sum; the next
// chunk's keys are on their way while this one's weights are made, its values behind the second product.  Maxima are only looked
// for among lanes when some score is 2^8 above the one in use.
// 8-bit caches are taken as fp16, which holds every e4m3 number: a query row is scaled into fp16's range by a power of two
// (what it loses is below 2^-24 of the row's largest number), a key's scale 2^ke goes to its scores, and a value's 2^ve into its
// weight: 2^(x_j + ve_j - m) with m the largest x_j + ve_j, so that fp16 weights are as exact as the largest share in a row's result
// allows, whatever the keys' values are sized like.  The sum that divides takes the weights times 2^-ve_j where these exponents are
// ordinary.  A value of zeros, stored with the smallest exponent, or one tiny beside another has a weight below 2^-126, where they end, and
// 2^-ve_j ends at 2^127: chunks with such values go into a sum of their own, of 2^(x_j - n) with n the largest x_j.  Results refer to n
// then.  (That sum and n wait in shared memory.  64 sequences of up to 8000 keys of 8 bits, 8 kv heads: 128 us with 4 rows, 178 with 16, 4.4
// and 3.2 TB/s, as against 130 and 193 with exponentials of their own for every key, and 143 and 203 where values are of 2^-40.)
#include <climits>
#include <type_traits>

#include "../../include/ftb200.h"
#include "paged_query.cuh"
#include "paged_work.cuh"
#include "paged_forms.h"
#include "tmap.h"

namespace ftb {
namespace {

constexpr int kWarps = 4, kUnitKeys = 16 * kWarps, kAtLeast = 2;
static_assert(kWarps * 32 == kLineThreads, "the line is laid out by a block");
constexpr float kAbove = 8.f;  // weights up to 2^8 (fp16 ends at 2^16): scores may lie that far above the maximum in use

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <int D, int NT>
struct Merge {
  float o[kWarps][NT * 8][D + 4];  // (rows 16 bytes apart in the banks)
  float m[kWarps][NT * 8], l[kWarps][NT * 8], n[kWarps][NT * 8];
};

// Warps enough for 8 KB each on their way.  (16 rows a warp leave registers for two blocks; more rows for few tokens, as 24 and 48 in
// tiles of two groups of warps that share the keys through L1, were slower than the tiles of paged_tile.cu by 2 to 4 times.)
constexpr int blocks_per_sm(int nt) { return nt == 1 ? 3 : 2; }

template <typename T, bool k8, int D, int NT, int kWhat>
__global__ void __launch_bounds__(kWarps * 32, blocks_per_sm(NT))
paged_short_kernel(const __grid_constant__ PagedAttn a, float* __restrict__ parts, PagedCut* __restrict__ cuts) {
  using C = typename std::conditional<k8, __half, T>::type;
  constexpr int R = NT * 8, kSteps = D / 16, kKLoads = k8 ? D / 64 : D / 32;
  constexpr int kVWords = k8 ? D / 32 : D / 16;  // 32-bit words of one key's values a lane
  extern __shared__ __align__(16) unsigned char smem[];
  Merge<D, NT>& mg = *reinterpret_cast<Merge<D, NT>*>(smem);
  __shared__ int s_odd[R];
  __shared__ PagedLineRoom s_line;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int piece = blockIdx.x;
  grid_dependency_wait();
  grid_launch_dependents();
  PagedWalk<R, kUnitKeys, kWhat> walk;
  {
    int b;
    long long at;
    const PagedLine line = paged_line<R, kUnitKeys, kWhat>(a, piece, gridDim.x, kAtLeast, s_line, &b, &at);
    if (piece >= line.pieces || line.total == 0) {
      if (threadIdx.x == 0) cuts[piece].last = -1;
      return;
    }
    walk.begin(a, line, piece, b, at);
  }
  const int page_mask = (1 << a.batch.page_shift) - 1;

  for (bool first_tile = true; walk.more(); first_tile = false) {
    const PagedTile w = walk.next(a);
    const PagedSeq& s = walk.s;
    const int h = w.h, rows = w.rows, flat0 = w.flat0, lo = w.keys.lo, hi = w.keys.hi;
    const int* table = a.batch.table + static_cast<long long>(w.b) * a.batch.W;
    const long long first_pos = s.pos0 + s.first + flat0 / a.group, last_pos = s.pos0 + s.first + (flat0 + rows - 1) / a.group;
    if (first_tile && threadIdx.x == 0) {
      const int last = last_piece_of(walk.line, piece, w);
      cuts[piece].last = last;
      if (last >= 0) cuts[piece] = PagedCut{last, w.b, s.first, flat0, rows, h, lo, hi, s.pos0};
    }

    // ---- queries: lane (g, c) holds of row g what it holds of a key; limits and factors of rows 2c and 2c + 1
    uint32_t q[NT][kSteps][2];
    float factor[NT][2];
    int see_lo[NT][2], see_hi[NT][2];  // keys see_lo .. see_hi
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mine = load_query<T, k8, D>(a, s.first, h, flat0, nt * 8 + g, rows, c, q[nt]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        factor[nt][e] = __shfl_sync(0xffffffffu, mine, (2 * c + e) * 4);
        const int r = nt * 8 + 2 * c + e;
        const long long pos = r < rows ? s.pos0 + s.first + (flat0 + r) / a.group : -1ll;
        see_hi[nt][e] = static_cast<int>(max(-1ll, min(pos, static_cast<long long>(hi) - 1)));
        see_lo[nt][e] = a.window > 0 ? static_cast<int>(max(0ll, min(pos - a.window + 1, static_cast<long long>(INT_MAX)))) : 0;
      }
    }
    // chunks that every row sees whole need no mask: [all_lo, all_hi]
    int all_lo = 0, all_hi = static_cast<int>(max(-1ll, min(first_pos, static_cast<long long>(hi) - 1)));
    if (a.window > 0) all_lo = static_cast<int>(max(0ll, min(last_pos - a.window + 1, static_cast<long long>(INT_MAX))));
    const long long base = s.pos0 + s.first;  // of the sequence's new tokens
    if (kWhat == kTrees) all_hi = static_cast<int>(max(-1ll, min(base - 1, static_cast<long long>(all_hi))));

    float oacc[kSteps][NT][4], m[NT][2], l[NT][2];
    float near = kNear;  // 8 bits: l takes a chunk's weights where the values' exponents are below
    // the sum of the other chunks, and what it refers to: [row][lane] of this warp, where its part of the results will be
    float* apart_l = &mg.o[warp][0][0] + lane;
    float* apart_n = apart_l + NT * 2 * 32;
    static_assert(NT * 4 * 32 <= NT * 8 * (D + 4), "the room of a warp's results");
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -FLT_MAX;
      if constexpr (k8) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          apart_l[(nt * 2 + e) * 32] = 0.f;
          apart_n[(nt * 2 + e) * 32] = -FLT_MAX;
        }
      }
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) oacc[i][nt][0] = oacc[i][nt][1] = oacc[i][nt][2] = oacc[i][nt][3] = 0.f;
    }

    // ---- the walk
    int key0 = (lo / kUnitKeys + w.r0) * kUnitKeys + warp * 16;
    if (key0 + 15 < lo) key0 += kUnitKeys;  // (pages in front of the window need not be there)
    const int key_end = min(hi, (lo / kUnitKeys + w.r1) * kUnitKeys);
    auto row_of = [&](int page, int key) {  // the cache row of key: a page that the table does not have reads as page 0
      return ((static_cast<long long>(page) * a.kv_heads + h) << a.batch.page_shift) + (key & page_mask);
    };
    auto page_at = [&](int key) {
      const int page = key < key_end ? __ldg(table + (key >> a.batch.page_shift)) : 0;
      if (page >= 0 && page < a.batch.pages) return page;
      atomicCAS(a.status, 0, FTB_ERR_INDEX);
      return 0;
    };
    uint4 kf[2][kKLoads];
    uint32_t vf[4][kVWords];
    int ke[2] = {127, 127}, ve[2] = {127, 127};
    auto load_k = [&](long long row) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kKLoads; ++j)
          kf[i][j] = load_once(a.k + (row + g + 8 * i) * (k8 ? D : 2 * D) + j * 64 + c * 16);
      if constexpr (k8) {
        ke[0] = a.k_exp[row + g];
        ke[1] = a.k_exp[row + g + 8];
        ve[0] = a.v_exp[row + g];
        ve[1] = a.v_exp[row + g + 8];
      }
    };
    auto load_v = [&](long long row) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned char* src = a.v + (row + 2 * c + (i & 1) + (i >> 1) * 8) * (k8 ? D : 2 * D);
        if constexpr (kVWords == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(src + g * 8);
          vf[i][0] = x.x;
          vf[i][1] = x.y;
        } else {
#pragma unroll
          for (int j = 0; j < kVWords / 4; ++j) {
            const uint4 x = load_once(src + j * 128 + g * 16);
            vf[i][4 * j] = x.x;
            vf[i][4 * j + 1] = x.y;
            vf[i][4 * j + 2] = x.z;
            vf[i][4 * j + 3] = x.w;
          }
        }
      }
    };
    long long row = 0, row_next = 0;
    int page_next = 0;
    if (key0 < key_end) {
      row = row_of(page_at(key0), key0);
      page_next = page_at(key0 + kUnitKeys);
      load_k(row);
      load_v(row);
    }
    // (two chunks a turn: 128 for 130 us where 8 rows of 8 bits and d 128 are at their registers' end; 16 rows 191 for 178, d 64 151 for 146)
#pragma unroll (k8 && NT == 1 && D == 128 ? 2 : 1)
    for (; key0 < key_end; key0 += kUnitKeys) {
      const bool more = key0 + kUnitKeys < key_end;
      row_next = row_of(page_next, key0 + kUnitKeys);
      page_next = page_at(key0 + 2 * kUnitKeys);
      // scores, in log2: [key g | g + 8][row 2c | 2c + 1]
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
      for (int j = 0; j < kKLoads; ++j) {
        const uint32_t w0[4] = {kf[0][j].x, kf[0][j].y, kf[0][j].z, kf[0][j].w}, w1[4] = {kf[1][j].x, kf[1][j].y, kf[1][j].z, kf[1][j].w};
        if constexpr (k8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_f16x2(w0[i], a0, a2);
            e4m3x4_to_f16x2(w1[i], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<C>(sc[nt], a0, a1, a2, a3, q[nt][4 * j + i][0], q[nt][4 * j + i][1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<C>(sc[nt], w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1], q[nt][2 * j + i][0], q[nt][2 * j + i][1]);
        }
      }
      float inv0 = 1.f, inv1 = 1.f, add0 = 0.f, add1 = 0.f, s0 = 1.f, s1 = 1.f;
      if constexpr (k8) {
        s0 = exponent_scale(ke[0]);
        s1 = exponent_scale(ke[1]);
        add0 = static_cast<float>(ve[0] - 127);
        add1 = static_cast<float>(ve[1] - 127);
        inv0 = exponent_scale(max(0, 254 - ve[0]));
        inv1 = exponent_scale(max(0, 254 - ve[1]));
      }
      if (more) load_k(row_next);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // (the scales of query and key meet before the score: either alone may lead out of fp32's range.  A score of 0 stays one.)
          const float f = k8 ? fminf(factor[nt][i & 1] * (i < 2 ? s0 : s1), FLT_MAX) : factor[nt][i & 1];
          sc[nt][i] = fmaf(sc[nt][i], f, i < 2 ? add0 : add1);
        }
      const bool edge = key0 + 15 > all_hi || key0 < all_lo;
      if (edge) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + g + (i >> 1) * 8;
            if (key > see_hi[nt][i & 1] || key < see_lo[nt][i & 1]) sc[nt][i] = -INFINITY;
          }
        if (kWhat == kTrees) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = nt * 8 + 2 * c + (i & 1);
              const long long j = key0 + g + (i >> 1) * 8 - base;
              if (j >= 0 && r < rows && !in_tree(a, s.first + (flat0 + r) / a.group, j)) sc[nt][i] = -INFINITY;
            }
        }
      }
      if constexpr (k8) {
        if (__any_sync(0xffffffffu, fmaxf(fabsf(add0), fabsf(add1)) > near)) {
          auto largest = [](float x) {  // of the keys
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          };
          bool wide = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int at = (nt * 2 + e) * 32;
              const float x0 = sc[nt][e] - add0, x1 = sc[nt][2 + e] - add1, n = apart_n[at];
              float to = fmaxf(n, largest(fmaxf(x0, x1)));
              if (near > 0.f) to = fmaxf(to, m[nt][e]);  // (else l is 0, and m may be far from the scores)
              float sum = apart_l[at] * exp2_fast(n - to) + exp2_fast(x0 - to) + exp2_fast(x1 - to);
              if (near > 0.f) sum = fmaf(l[nt][e], exp2_fast(m[nt][e] - to), sum);
              apart_l[at] = sum;
              apart_n[at] = to;
              l[nt][e] = 0.f;
              // (m is going to be this, or up to 2^8 below)
              wide |= fabsf(fmaxf(m[nt][e], largest(fmaxf(sc[nt][e], sc[nt][2 + e]))) - to) > kNearTops;
            }
          near = __any_sync(0xffffffffu, wide) ? -1.f : kNear;
          inv0 = inv1 = 0.f;
        }
      }
      bool above = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) above |= sc[nt][i] > m[nt][i & 1] + kAbove;
      if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float keep[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(sc[nt][e], sc[nt][2 + e]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            x = fmaxf(x, m[nt][e]);
            keep[e] = exp2_fast(m[nt][e] - x);
            m[nt][e] = x;
            l[nt][e] *= keep[e];
          }
#pragma unroll
          for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) oacc[i][nt][e] *= keep[e & 1];
        }
      }
      uint32_t p[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = exp2_fast(sc[nt][i] - m[nt][i & 1]);
        l[nt][0] += fmaf(e[0], inv0, e[2] * inv1);
        l[nt][1] += fmaf(e[1], inv0, e[3] * inv1);
        p[nt][0] = transpose8x8(Fmt<C>::pack2(e[0], e[1]));
        p[nt][1] = transpose8x8(Fmt<C>::pack2(e[2], e[3]));
      }
      if (key0 < lo || key0 + 15 >= hi) {  // rows that nobody sees may hold anything: 0 * NaN is NaN
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 2 * c + (i & 1) + (i >> 1) * 8;
          if (key < lo || key >= hi) {
#pragma unroll
            for (int w = 0; w < kVWords; ++w) vf[i][w] = 0u;
          }
        }
      }
#pragma unroll
      for (int w = 0; w < kVWords; ++w) {
        if constexpr (k8) {
          const uint32_t x01 = __byte_perm(vf[0][w], vf[1][w], 0x5140), x23 = __byte_perm(vf[0][w], vf[1][w], 0x7362);
          const uint32_t y01 = __byte_perm(vf[2][w], vf[3][w], 0x5140), y23 = __byte_perm(vf[2][w], vf[3][w], 0x7362);
          uint32_t a0, a1, a2, a3, b0, b1, b2, b3;
          e4m3x4_to_f16x2(x01, a0, a1);
          e4m3x4_to_f16x2(y01, a2, a3);
          e4m3x4_to_f16x2(x23, b0, b1);
          e4m3x4_to_f16x2(y23, b2, b3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816<C>(oacc[2 * w][nt], a0, a1, a2, a3, p[nt][0], p[nt][1]);
            mma16816<C>(oacc[2 * w + 1][nt], b0, b1, b2, b3, p[nt][0], p[nt][1]);
          }
        } else {
          const uint32_t a0 = __byte_perm(vf[0][w], vf[1][w], 0x5410), a1 = __byte_perm(vf[0][w], vf[1][w], 0x7632);
          const uint32_t a2 = __byte_perm(vf[2][w], vf[3][w], 0x5410), a3 = __byte_perm(vf[2][w], vf[3][w], 0x7632);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<C>(oacc[w][nt], a0, a1, a2, a3, p[nt][0], p[nt][1]);
        }
      }
      if (more) load_v(row_next);
    }

    // ---- the four warps' results
    float n[NT][2];  // what l refers to
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        n[nt][e] = m[nt][e];
        if constexpr (k8) {
          const float sum = apart_l[(nt * 2 + e) * 32], from = apart_n[(nt * 2 + e) * 32];
          const float to = near > 0.f ? fmaxf(from, m[nt][e]) : from;
          l[nt][e] = (near > 0.f ? l[nt][e] * exp2_fast(m[nt][e] - to) : 0.f) + sum * exp2_fast(from - to);
          n[nt][e] = to;
        }
      }
    if constexpr (k8) __syncwarp();  // (results go over them)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[nt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int r = nt * 8 + 2 * c + e;
        if (g == 0) {
          mg.m[warp][r] = m[nt][e];
          mg.l[warp][r] = x;
          if constexpr (k8) mg.n[warp][r] = n[nt][e];
        }
        // rows g and g + 8 of product i are numbers d and d + 1 of the output
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int d = kVWords == 2 ? g * 8 + 2 * i : (i >> (k8 ? 3 : 2)) * (k8 ? 128 : 64) + g * (k8 ? 16 : 8) + (i & (k8 ? 7 : 3)) * 2;
          *reinterpret_cast<float2*>(&mg.o[warp][r][d]) = make_float2(oacc[i][nt][e], oacc[i][nt][2 + e]);
        }
      }
    if (threadIdx.x < R) s_odd[threadIdx.x] = 0;
    __syncthreads();
    const bool whole = w.r0 == 0 && w.r1 == w.units;
    float* part = parts + (static_cast<long long>(piece) * 2 + (w.r0 == 0 ? 1 : 0)) * part_floats<R, D>();
    for (int i = threadIdx.x; i < R * (D / 4); i += kWarps * 32) {
      const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
      if (r >= rows) break;
      float top = mg.m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, mg.m[w][r]);
      float top_n = top;
      if constexpr (k8) {
        top_n = mg.n[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top_n = fmaxf(top_n, mg.n[w][r]);
      }
      float sum = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float k = exp2_fast(mg.m[w][r] - top);
        const float4 y = *reinterpret_cast<const float4*>(&mg.o[w][r][d]);
        sum = fmaf(mg.l[w][r], k8 ? exp2_fast(mg.n[w][r] - top_n) : k, sum);
        x.x = fmaf(y.x, k, x.x);
        x.y = fmaf(y.y, k, x.y);
        x.z = fmaf(y.z, k, x.z);
        x.w = fmaf(y.w, k, x.w);
      }
      auto times = [&](float f) {
        x.x *= f;
        x.y *= f;
        x.z *= f;
        x.w *= f;
      };
      if (whole) times(sum == 0.f ? 0.f : 1.f / sum);
      if constexpr (k8) {  // to what the sum refers to (in two steps: it may be 2^135, where the numbers are small)
        const float half = exp2_fast(0.5f * (top - top_n));
        times(half);
        times(half);
      }
      if (whole) {
        const float all = x.x + x.y + x.z + x.w;
        if (all != all) s_odd[r] = 1;
        const int flat = flat0 + r, t = s.first + flat / a.group, head = h * a.group + flat % a.group;
        *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + (static_cast<long long>(t) * a.kv_heads * a.group + head) * D + d) =
            make_uint2(Fmt<T>::pack2(x.x, x.y), Fmt<T>::pack2(x.z, x.w));
        if (wants_lse<kWhat>(a) && d == 0) put_lse(a, static_cast<long long>(t) * a.kv_heads * a.group + head, top_n, sum);
      } else {
        *reinterpret_cast<float4*>(part + r * D + d) = x;
        if (d == 0) {
          part[R * D + 2 * r] = top_n;
          part[R * D + 2 * r + 1] = sum;
        }
      }
    }
    __syncthreads();
    // (rows that something unseen may have made a NaN are left to the joining kernel, which goes through them key by key)
    if (threadIdx.x < rows) {
      const int flat = flat0 + threadIdx.x, t = s.first + flat / a.group;
      a.odd[static_cast<long long>(t) * a.kv_heads * a.group + h * a.group + flat % a.group] =
          s_odd[threadIdx.x] != 0 && hides<kWhat>(a, s.pos0 + t, lo, hi) ? 1u : 0u;
    }
  }
}

template <typename T, bool k8, int D, int NT, int kWhat>
int launch(const PagedAttn& a, void* scratch, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0};
  auto kfn = paged_short_kernel<T, k8, D, NT, kWhat>;
  constexpr int kSmem = sizeof(Merge<D, NT>);
  if (!ensure_dynamic_smem(kfn, kSmem, configured)) return FTB_ERR_LAUNCH;
  // No more shared memory than the blocks need: what is on its way to registers passes L1, which has the rest.  (Left to itself
  // the division may stay as a kernel in front had it: 378 against 290 us for 96 sequences of 16 rows.)
  static std::atomic<unsigned long long> divided{0};
  static_assert(blocks_per_sm(NT) * (kSmem + 2048) <= kPagedCarveout, "the blocks of an SM");
  if (!set_smem_carveout(kfn, kPagedCarveout, divided)) return FTB_ERR_LAUNCH;
  const int pieces = paged_short_pieces(NT * 8);
  float* parts = static_cast<float*>(scratch);
  const cudaError_t err = launch_dependent(kfn, dim3(pieces), dim3(kWarps * 32), kSmem, stream, a, parts,
                                           reinterpret_cast<PagedCut*>(parts + 2 * pieces * part_floats<NT * 8, D>()));
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}
template <typename T, bool k8, int D, int NT>
int launch(const PagedAttn& a, void* scratch, cudaStream_t stream) {
  return a.tree != nullptr  ? launch<T, k8, D, NT, kTrees>(a, scratch, stream)
         : a.lse != nullptr ? launch<T, k8, D, NT, kLse>(a, scratch, stream)
                            : launch<T, k8, D, NT, kPlain>(a, scratch, stream);
}
template <typename T, int D, int NT>
int launch(const PagedAttn& a, void* scratch, cudaStream_t stream) {
  return a.k_exp != nullptr ? launch<T, true, D, NT>(a, scratch, stream) : launch<T, false, D, NT>(a, scratch, stream);
}
template <typename T, int D>
int launch(const PagedAttn& a, int rows, void* scratch, cudaStream_t stream) {
  return rows == 8 ? launch<T, D, 1>(a, scratch, stream) : launch<T, D, 2>(a, scratch, stream);
}

}  // namespace

int paged_short_pieces(int rows) { return current_sm_count() * blocks_per_sm(rows / 8); }

int paged_short_launch(const PagedAttn& a, int d, int dtype, int rows, void* scratch, cudaStream_t stream) {
  if (dtype == FTB_F16) return d == 128 ? launch<__half, 128>(a, rows, scratch, stream) : launch<__half, 64>(a, rows, scratch, stream);
  return d == 128 ? launch<__nv_bfloat16, 128>(a, rows, scratch, stream) : launch<__nv_bfloat16, 64>(a, rows, scratch, stream);
}

}  // namespace ftb
