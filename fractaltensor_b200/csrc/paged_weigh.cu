// What new tokens attend to, added up over a cache's keys: w_j += sum over tokens and heads of a kv head of exp(scale * q . k_j - lse), for
// the keys that a token sees; a new token's own key begins at 0.  lse is log(sum(exp(scale * q . k))) of each row, from the attention in front.
//
// With the keys on the M side of the products, S^T = K Q^T (mma.m16n8k16), a key's sum is over a row of the result: each key belongs to
// one warp, which goes through all rows (token, head of the group) that see it, in their order.  No two CTAs meet in a weight, and
// the sums are the same from call to call.  Keys go from global memory straight into the registers that the products take them from, as in
// paged_short.cu.  8-bit caches are taken as fp16, as there: a query row scaled into fp16's range by a power of two, a key's scale
// 2^e to its scores.
//
// The work: blocks of 64 keys of a sequence and kv head, in a line that is cut into as many pieces as there are CTAs, a block counting
// as often as there are tiles of rows.  A warp's next 16 keys are on their way while these are made weights of, the number of the page behind
// them one step longer.
//
// Bound by the bytes of the keys: 64 sequences of up to 8000 keys of 16 bits, 8 kv heads of 128, a token of 32 heads each 91 to 95 us (several GPUs), 6.1 TB/s (126 without
// keys on their way ahead); 4096 keys each 88 us, over 8 bits 75, 3.6 TB/s: there the trips of a warp's 16 keys, 2 KB, are what is short.  One
// sequence of 777 keys 6.2 us, a launch and four trips to memory one behind the other.
#include <cfloat>
#include <climits>
#include <type_traits>

#include "../../include/ftb200.h"
#include "paged_forms.h"
#include "paged_query.cuh"
#include "paged_weigh.cuh"
#include "tmap.h"

namespace ftb {
namespace {

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kWarps = 4, kBlockKeys = 16 * kWarps;
static_assert(kWarps * 32 == kLineThreads, "the line is laid out by a block");

// What a block of a sequence counts as.
template <int R>
__device__ __forceinline__ int cost_of(const PagedSeq& s) { return (s.flats + R - 1) / R; }

constexpr int blocks_per_sm(int nt) { return nt == 1 ? 4 : 3; }

template <typename T, bool k8, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, blocks_per_sm(NT))
paged_weigh_kernel(const __grid_constant__ Weigh x) {
  using C = typename std::conditional<k8, __half, T>::type;
  constexpr int R = NT * 8, kSteps = D / 16, kKLoads = k8 ? D / 64 : D / 32;
  // what the sequences of the units on their way are like (in registers it is the keys' room: 111 for 101 us of a decoding step)
  struct Of {
    long long base;  // position of the new tokens
    int first, flats, lo, hi;
  };
  __shared__ Of s_of[kWarps][4];
  __shared__ PagedLineRoom s_line;
  const PagedAttn& a = x.attn;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  grid_dependency_wait();
  grid_launch_dependents();
  int b;
  long long at;
  const PagedLine line = paged_line_of(a, blockIdx.x, gridDim.x, 1, s_line, &b, &at, [&](const PagedSeq& s) {
    return static_cast<long long>(blocks_of<kBlockKeys>(all_keys(a, s))) * cost_of<R>(s);
  });
  if (static_cast<int>(blockIdx.x) >= line.pieces || line.total == 0) return;
  // The units of this warp, one after the other: a sequence's are in the order kv head, block; a block is the piece's that its first unit is in.
  const int shift = a.batch.page_shift, heads = a.kv_heads * a.group;
  struct Unit {
    int h, key0, page, of;  // page -1: none; of: which sequence's, -1: none of its keys are this warp's
  };
  long long skip = piece_begin(line, blockIdx.x) - at, left = piece_begin(line, blockIdx.x + 1) - at;  // from the sequence's first unit
  int blocks, h, block, lo, hi, entered = 0;
  long long todo;  // blocks of the sequence that are left
  auto enter = [&] {
    const PagedSeq s = paged_sequence(a, b);
    const PagedKeys keys = all_keys(a, s);
    lo = keys.lo;
    hi = keys.hi;
    blocks = blocks_of<kBlockKeys>(keys);
    const int cost = max(1, cost_of<R>(s));
    const long long all = static_cast<long long>(blocks) * a.kv_heads, n0 = skip > 0 ? (skip + cost - 1) / cost : 0;
    todo = min(all, (left + cost - 1) / cost) - n0;
    skip -= all * cost;
    left -= all * cost;
    if (todo <= 0) return;
    h = static_cast<int>(n0 / blocks);
    block = static_cast<int>(n0 - static_cast<long long>(h) * blocks);
    // (of two units that are on their way and the next one; what a unit in work needs has been taken out)
    entered = (entered + 1) & 3;
    __syncwarp();
    if (lane == 0) s_of[warp][entered] = Of{s.pos0 + s.first, s.first, s.flats, lo, hi};
    __syncwarp();
  };
  enter();
  auto next = [&](Unit& u) -> bool {
    while (todo <= 0) {
      if (left <= 0 || ++b >= a.batch.B) return false;
      enter();
    }
    u.h = h;
    u.key0 = (lo / kBlockKeys + block) * kBlockKeys + warp * 16;
    u.of = u.key0 < hi && u.key0 + 16 > lo ? entered : -1;
    u.page = u.of >= 0 ? a.batch.table[static_cast<long long>(b) * a.batch.W + (u.key0 >> shift)] : -1;
    --todo;
    if (++block == blocks) {
      block = 0;
      ++h;
    }
    return true;
  };
  uint4 kf[2][kKLoads];
  float s0 = 1.f, s1 = 1.f, old = 0.f;
  long long row = 0;
  auto load = [&](Unit& u) {
    if (u.page < 0 || u.page >= a.batch.pages) {
      if (u.of >= 0) atomicCAS(a.status, 0, FTB_ERR_INDEX);
      u.page = -1;
      return;
    }
    row = ((static_cast<long long>(u.page) * a.kv_heads + u.h) << shift) + (u.key0 & ((1 << shift) - 1));
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < kKLoads; ++j) kf[i][j] = load_once(a.k + (row + g + 8 * i) * (k8 ? D : 2 * D) + j * 64 + c * 16);
    if constexpr (k8) {
      s0 = exponent_scale(a.k_exp[row + g]);
      s1 = exponent_scale(a.k_exp[row + g + 8]);
    }
    if (c < 2) old = x.weights[row + g + 8 * c];  // (lane (g, 0) has key g, lane (g, 1) key g + 8)
  };

  uint32_t q[NT][kSteps][2];
  float factor[NT][2], minus[NT][2];
  int see_lo[NT][2], see_hi[NT][2];
  int all_lo = 0, all_hi = -1;  // keys that all rows see, where all of their lse are finite
  int q_first = -1, q_h = -1;   // whose rows these are, where a tile has all of them
  // A unit's keys are on their way while the one's in front are made weights of, and its page's number one unit longer.
  Unit now, then, later;
  bool more = next(then), still = more && next(later);
  if (more) load(then);
  while (more) {
    now = then;
    const Of of = s_of[warp][max(0, now.of)];
    const float t0 = s0, t1 = s1, was = old;
    const long long at_row = row;
    more = still;
    then = later;
    auto go_on = [&] {
      if (more) load(then);
      still = more && next(later);
    };
    if (now.page < 0) {
      go_on();
      continue;
    }
    float sum0 = 0.f, sum1 = 0.f;
    bool gone_on = false;
    for (int flat0 = 0; flat0 < of.flats; flat0 += R) {
      const int rows = min(R, of.flats - flat0);
      const bool last = flat0 + R >= of.flats;
      if (of.base + (flat0 + rows - 1) / a.group < now.key0 ||                                  // in front of the keys
          (a.window > 0 && of.base + flat0 / a.group - a.window >= now.key0 + 15)) continue;    // they have left the window
      if (of.flats > R || q_first != of.first || q_h != now.h) {
        q_first = of.first;
        q_h = now.h;
        bool odd = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // (behind the last row that one again, which takes away infinity: zeros times an infinity of a key would be NaN)
          const float mine = load_query<T, k8, D>(a, of.first, now.h, flat0, min(nt * 8 + g, rows - 1), rows, c, q[nt]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            factor[nt][e] = __shfl_sync(0xffffffffu, mine, (2 * c + e) * 4);
            const int r = nt * 8 + 2 * c + e, flat = flat0 + r, token = flat / a.group;
            float lse = INFINITY;
            if (r < rows) lse = x.lse[static_cast<long long>(of.first + token) * heads + now.h * a.group + flat - token * a.group];
            const bool fine = fabsf(lse) < INFINITY;  // (not of a row that sees nothing, or something that is not finite)
            odd |= r < rows && !fine;
            minus[nt][e] = -lse * kLog2E;
            const long long pos = fine ? of.base + token : -1ll;
            see_hi[nt][e] = static_cast<int>(max(-1ll, min(pos, static_cast<long long>(of.hi) - 1)));
            see_lo[nt][e] = a.window > 0 ? static_cast<int>(max(0ll, min(pos - a.window + 1, static_cast<long long>(INT_MAX)))) : 0;
          }
        }
        const long long pos0 = of.base + flat0 / a.group, pos1 = of.base + (flat0 + rows - 1) / a.group;
        all_hi = __any_sync(0xffffffffu, odd) ? -1 : static_cast<int>(max(-1ll, min(pos0, static_cast<long long>(of.hi) - 1)));
        all_lo = max(of.lo, a.window > 0 ? static_cast<int>(max(0ll, min(pos1 - a.window + 1, static_cast<long long>(INT_MAX)))) : 0);
      }
      // (two sums, of half the products each: the unit cuts off what is below a sum's last bit, always downwards, and the fewer steps the
      // less.  9.9e-7 of the weights for a decoding step in one sum.)
      float sc[NT][4], sd[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[nt][i] = sd[nt][i] = 0.f;
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
            for (int nt = 0; nt < NT; ++nt) mma16816<C>(i & 1 ? sd[nt] : sc[nt], a0, a1, a2, a3, q[nt][4 * j + i][0], q[nt][4 * j + i][1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<C>(i & 1 ? sd[nt] : sc[nt], w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1], q[nt][2 * j + i][0], q[nt][2 * j + i][1]);
        }
      }
      if (last) {
        go_on();
        gone_on = true;
      }
      const bool plain = now.key0 + 15 <= all_hi && now.key0 >= all_lo;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = i & 1;
          // (the scales of query and key meet before the score: either alone may lead out of fp32's range)
          const float f = k8 ? fminf(factor[nt][e] * (i < 2 ? t0 : t1), FLT_MAX) : factor[nt][e];
          sc[nt][i] = exp2_fast(fmaf(sc[nt][i] + sd[nt][i], f, minus[nt][e]));
        }
      if (!plain) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = i & 1, key = now.key0 + g + (i >> 1) * 8;
            if (key > see_hi[nt][e] || key < see_lo[nt][e]) sc[nt][i] = 0.f;
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sum0 += sc[nt][0] + sc[nt][1];
        sum1 += sc[nt][2] + sc[nt][3];
      }
    }
    if (!gone_on) go_on();
    sum0 += __shfl_xor_sync(0xffffffffu, sum0, 1);
    sum1 += __shfl_xor_sync(0xffffffffu, sum1, 1);
    sum0 += __shfl_xor_sync(0xffffffffu, sum0, 2);
    sum1 += __shfl_xor_sync(0xffffffffu, sum1, 2);
    const int key = now.key0 + g + 8 * c;
    if (c < 2 && key >= of.lo && key < of.hi) {
      const float sum = c == 0 ? sum0 : sum1;
      x.weights[at_row + g + 8 * c] = key >= of.base ? sum : was + sum;
    }
  }
}

template <typename T, bool k8, int D, int NT>
int launch(const Weigh& x, cudaStream_t stream) {
  const cudaError_t err = launch_dependent(paged_weigh_kernel<T, k8, D, NT>, dim3(current_sm_count() * blocks_per_sm(NT)), dim3(kWarps * 32), 0, stream, x);
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}
template <typename T, int D>
int launch(const Weigh& x, int rows, cudaStream_t stream) {
  if (x.attn.k_exp != nullptr) return rows == 8 ? launch<T, true, D, 1>(x, stream) : launch<T, true, D, 2>(x, stream);
  return rows == 8 ? launch<T, false, D, 1>(x, stream) : launch<T, false, D, 2>(x, stream);
}
template <typename T>
int launch(const Weigh& x, int d, int rows, cudaStream_t stream) {
  return d == 128 ? launch<T, 128>(x, rows, stream) : launch<T, 64>(x, rows, stream);
}

// Which kernels run: few > 0: tiles of so many rows, for sequences of up to `most`; many: paged_weigh_tile.cu for the others.
struct Form {
  int few, most;
  bool many;
};
// `keys`: as many as the table has room for, the lengths being on the device (8 of 500 keys, 24 rows each: 12.1 us, with a table for 131 072 keys 17.5).
Form form_of(int T, int B, int group, int kv_heads, long long keys) {
  const long long rows = static_cast<long long>(T) * group;
  if (T <= B || rows <= 16) return {rows <= 8ll * B ? 8 : 16, INT_MAX, false};
  // Each tile of 16 rows goes through a block's keys, in registers, again, while paged_weigh_tile.cu takes as long for 20 rows as for 128, three
  // launches at least.  8 kv heads, 16 bits, here and there: one of 500 keys, 48 rows 9.6 and 12.6 us, 96 rows 14.1 and 13.0; of 16 000, 32 rows 23.5
  // and 30.7, 64 rows 38 and 31; 8 of 4000, 20 rows (8064 units) 39.7 and 37.3; 48 of 500, 32 rows (6144) 30.8 and 31.5; 48 of 4000, 20 rows 193 and 147.
  // 8 bits: one of 4000 keys, 48 rows 17.4 and 18.7, 64 rows 21 and 18.5; 8 of 4000, 20 rows 52 and 41.
  const long long tiles = (rows + 16ll * B - 1) / (16ll * B);
  if (tiles <= 3 && tiles * B * kv_heads * ((keys + 63) / 64) <= 4500) return {16, INT_MAX, false};
  if (B == 1) return {0, 0, true};
  return {16, 16, true};
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" size_t ftb_paged_attn_weights_scratch_bytes(int T, int B, int kv_heads, int group, int d) {
  if (T <= 0 || B <= 0 || kv_heads <= 0 || group <= 0 || d <= 0) return 0;
  if (T <= B || static_cast<long long>(T) * group <= 16) return 0;  // (never the other kernel; else it is the table's width that says)
  return paged_weigh_tile_scratch(T, kv_heads, group, d);
}

extern "C" int ftb_paged_attn_weights(const void* q, long long q_row, long long q_head, const void* k_cache, const unsigned char* k_exp,
                                      const float* lse, const int* table, const int* lens, const int* starts, float* weights, int T, int B,
                                      int W, int pages, int kv_heads, int group, int page_size, int d, int window, float scale, int dtype,
                                      void* scratch, size_t scratch_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  if ((T > 0 && (!q || !lse)) || !k_cache || !weights || !table || !lens || !starts) return FTB_ERR_ARG;
  if (T < 0 || B <= 0 || W <= 0 || pages <= 0 || kv_heads <= 0 || group <= 0 || window < 0) return FTB_ERR_ARG;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return FTB_ERR_ARG;
  if ((d != 64 && d != 128) || (dtype != FTB_F16 && dtype != FTB_BF16)) return FTB_ERR_ARG;
  if (!(scale > 0.f) || !(scale * kLog2E <= FLT_MAX)) return FTB_ERR_ARG;
  if (static_cast<long long>(kv_heads) * group > 65536 || static_cast<long long>(T) * group > INT_MAX) return FTB_ERR_ARG;
  if (((q_row | q_head) & 7) != 0) return FTB_ERR_ALIGN;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(k_exp)) & 15) != 0 ||
      ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(lse)) & 3) != 0)
    return FTB_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  if (T == 0) return FTB_OK;
  const int heads = kv_heads * group;
  const size_t rows = static_cast<size_t>(pages) * kv_heads * page_size, bytes = rows * sizeof(float);
  if (rows > INT_MAX) return FTB_ERR_ARG;
  if (overlap(weights, bytes, k_cache, rows * d * (k_exp != nullptr ? 1 : 2)) || (k_exp != nullptr && overlap(weights, bytes, k_exp, rows)) ||
      overlap(weights, bytes, lse, static_cast<size_t>(T) * heads * sizeof(float)) || over_rows(weights, static_cast<long long>(bytes / 2), q, T, q_row, heads, q_head, d))
    return FTB_ERR_ARG;
  const int rc = check_device_sm100();
  if (rc) return rc;
  Weigh x = {};
  PagedAttn& a = x.attn;
  a.batch = {table, lens, starts, B, W, pages, 31 - __builtin_clz(static_cast<unsigned>(page_size))};
  a.q = q;
  a.q_row = q_row;
  a.q_head = q_head;
  a.k = static_cast<const unsigned char*>(k_cache);
  a.k_exp = k_exp;
  a.T = T;
  a.kv_heads = kv_heads;
  a.group = group;
  a.window = window;
  a.scale_log2 = scale * kLog2E;
  a.status = static_cast<int*>(workspace);
  x.weights = weights;
  x.lse = lse;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Form f = form_of(T, B, group, kv_heads, static_cast<long long>(W) * page_size);
  if (f.many) {
    if (static_cast<long long>(T) * heads > INT_MAX) return FTB_ERR_ARG;  // a copy's coordinates have 32 bits
    if (scratch == nullptr || scratch_bytes < paged_weigh_tile_scratch(T, kv_heads, group, d)) return FTB_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(scratch) & 15) != 0) return FTB_ERR_ALIGN;
  }
  int err = FTB_OK;
  if (f.few > 0) {
    a.least_rows = 1;
    a.most_rows = f.most;
    err = dtype == FTB_F16 ? launch<__half>(x, d, f.few, s) : launch<__nv_bfloat16>(x, d, f.few, s);
  }
  if (f.many && err == FTB_OK) {
    a.least_rows = f.most + 1;
    a.most_rows = INT_MAX;
    err = paged_weigh_tile_launch(x, d, dtype, scratch, s);
  }
  return err;
}
