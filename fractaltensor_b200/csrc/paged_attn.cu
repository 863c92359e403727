// Attention of new tokens over a paged cache: o = sum_j softmax_j(scale * q . k_j) v_j over the keys j with
// pos - window < j <= pos, for a token at position pos, heads = group * kv_heads.
//
// Two kernels: paged_short.cu for sequences with few rows (token, head of a group), bound by the bytes of their keys and values, and
// paged_tile.cu for those with many, by matrix products on tiles of rows.  A call with both kinds runs both, each on its own; the
// lengths are on the device, so that it is there that a sequence is one or the other's.  Here: the choice, and what joins the tiles
// that the cuts between pieces of work went through.
//
// Scores, maxima, sums and results in the making have 32 bits.  Weights are rounded to the 16 bits that the second product takes (of the cache's
// type, fp16 over 8 bits): with bf16 results the error against 64 bits is 0.0019 of their size, 0.0017 where weights keep 32 bits.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cstdlib>
#include <type_traits>

#include "../../include/ftb200.h"
#include "paged_forms.h"
#include "paged_work.cuh"
#include "tmap.h"

namespace ftb {
namespace {

constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kJoinRows = 4, kMostCuts = 4 * kJoinThreads;

constexpr float kLog2E = 1.4426950408889634f;

struct Pieces {
  const float* parts;
  const PagedCut* cuts;
  int pieces, rows;  // rows of a tile
};

// Rows of whole tiles that have to be computed again: none, unless something in the cache is not finite, or dwarfs what is seen of its
// 8-bit block.  `warp` of `warps` in the grid.  Those of a tile lie side by side: a warp looks at four times eight (a sector of flags) far
// from each other.
template <typename T, bool k8, int D>
__device__ __forceinline__ void again_rows(const PagedAttn& a, long long warp, long long warps, int lane) {
  const int heads = a.kv_heads * a.group;
  const long long rows = static_cast<long long>(a.T) * heads;
  for (long long r0 = warp * 8; r0 < rows; r0 += warps * 32) {
    const long long mine = r0 + (lane >> 3) * warps * 8 + (lane & 7);
    unsigned again = __ballot_sync(0xffffffffu, mine < rows && a.odd[min(mine, rows - 1)] != 0);
    while (again != 0) {
      const int first = __ffs(again) - 1;
      const long long row = __shfl_sync(0xffffffffu, mine, first);
      again &= again - 1;
      const int t = static_cast<int>(row / heads);
      const RowPlace at = place_of_row(a.batch, t, lane);
      if (at.b < a.batch.B)  // (what no sequence has was not written either)
        attend_row<T, k8, D>(a, at.b, t, static_cast<int>(row - static_cast<long long>(t) * heads), at.pos, lane);
    }
  }
}

// Row r of a cut tile by one warp, its numbers x over the weights' sum l, to the output.
template <typename T, bool k8, int D>
__device__ __forceinline__ void finish_row(const PagedAttn& a, const PagedCut& c, int r, float l, float (&x)[D / 32], int lane) {
  const int heads = a.kv_heads * a.group;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float all = 0.f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) {
    x[e] *= inv;
    all += x[e];
  }
  const int flat = c.flat0 + r, t = c.first + flat / a.group, head = c.h * a.group + flat % a.group;
  uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(a.o) + (static_cast<long long>(t) * heads + head) * D) + lane * (D / 64);
#pragma unroll
  for (int e = 0; e < D / 64; ++e) out[e] = Fmt<T>::pack2(x[2 * e], x[2 * e + 1]);
  // (rows that something unseen may have made a NaN: key by key)
  if (__any_sync(0xffffffffu, all != all) && hides(a, c.pos0 + t, c.lo, c.hi)) attend_row<T, k8, D>(a, c.b, t, head, c.pos0 + t, lane);
}

// Parts first, first + by, .. of n of a row, added up: (m, l, x).
template <int D, typename Part>
__device__ __forceinline__ void add_parts(Part part, int R, int r, int first, int by, int n, int lane, float& m, float& l, float (&x)[D / 32]) {
  using Vec = typename std::conditional<D == 128, float4, float2>::type;
  m = -FLT_MAX;
  l = 0.f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) x[e] = 0.f;
  for (int i0 = first; i0 < n; i0 += 4 * by) {
    float2 ml[4];
    Vec v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * by;
      ml[k] = make_float2(-FLT_MAX, 0.f);
      v[k] = Vec{};
      if (i < n) {
        ml[k] = *reinterpret_cast<const float2*>(part(i) + R * D + 2 * r);
        v[k] = reinterpret_cast<const Vec*>(part(i) + r * D)[lane];
      }
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < 4; ++k) top = fmaxf(top, ml[k].x);
    const float keep = exp2_fast(m - top);
    m = top;
    l *= keep;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) x[e] *= keep;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float w = exp2_fast(ml[k].x - top);
      l = fmaf(ml[k].y, w, l);
#pragma unroll
      for (int e = 0; e < D / 32; ++e) x[e] = fmaf(reinterpret_cast<const float*>(&v[k])[e], w, x[e]);
    }
  }
}

// What the kernel for few rows leaves alone: block (x, y) takes row y of the tile with cut x, the parts spread over its warps: such
// tiles may have hundreds, and what they cost are trips to memory one behind the other.
constexpr int kFewWarps = 4;
template <typename T, bool k8, int D>
__global__ void __launch_bounds__(kFewWarps * 32)
paged_join_few_kernel(const __grid_constant__ PagedAttn a, Pieces few) {
  __shared__ float s_sum[kFewWarps][D];
  __shared__ float s_m[kFewWarps], s_l[kFewWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cut = blockIdx.x, r = blockIdx.y;
  grid_dependency_wait();
  grid_launch_dependents();
  const int last = few.cuts[cut].last;
  again_rows<T, k8, D>(a, (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * kFewWarps + warp,
                       static_cast<long long>(gridDim.x) * gridDim.y * kFewWarps, lane);
  if (last < 0) return;
  const PagedCut c = few.cuts[cut];
  if (r >= c.rows) return;
  const size_t floats = static_cast<size_t>(few.rows) * (D + 2);
  // part 0: of piece cut - 1, which left the tile's beginning in its second place; the others in their first
  auto part = [&](int i) { return few.parts + (static_cast<size_t>(cut - 1 + i) * 2 + (i == 0 ? 1 : 0)) * floats; };
  float m, l, x[D / 32];
  add_parts<D>(part, few.rows, r, warp, kFewWarps, last - cut + 2, lane, m, l, x);
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < D / 32; ++e) s_sum[warp][lane * (D / 32) + e] = x[e];
  __syncthreads();
  if (warp != 0) return;
  float top = s_m[0];
#pragma unroll
  for (int w = 1; w < kFewWarps; ++w) top = fmaxf(top, s_m[w]);
  l = 0.f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) x[e] = 0.f;
#pragma unroll
  for (int w = 0; w < kFewWarps; ++w) {
    const float k = exp2_fast(s_m[w] - top);
    l = fmaf(s_l[w], k, l);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) x[e] = fmaf(s_sum[w][lane * (D / 32) + e], k, x[e]);
  }
  finish_row<T, k8, D>(a, c, r, l, x, lane);
}

// What both kernels leave.  Every block finds the cuts that have something to join, and the warps take the rows of those tiles in turn,
// kJoinRows at a time, all on their way at once where there are two parts, as of most tiles of many rows.
template <typename T, bool k8, int D>
__global__ void __launch_bounds__(kJoinThreads, 3)
paged_join_kernel(const __grid_constant__ PagedAttn a, Pieces few, Pieces many) {
  constexpr int kPer = D / 32;  // numbers of a row a lane
  using Vec = typename std::conditional<kPer == 4, float4, float2>::type;
  __shared__ int s_before[kMostCuts + 1], s_warp[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  grid_launch_dependents();
  again_rows<T, k8, D>(a, static_cast<long long>(blockIdx.x) * kJoinWarps + warp, static_cast<long long>(gridDim.x) * kJoinWarps, lane);
  // turns of every cut, and how many lie in front of it
  const int cuts = few.pieces + many.pieces;
  {
    int turns[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = threadIdx.x * 4 + k;
      turns[k] = 0;
      if (i < cuts) {
        const PagedCut& c = i < few.pieces ? few.cuts[i] : many.cuts[i - few.pieces];
        turns[k] = c.last < 0 ? 0 : (c.rows + kJoinWarps * kJoinRows - 1) / (kJoinWarps * kJoinRows);
      }
      sum += turns[k];
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    int before = upto - sum;
    for (int w = 0; w < warp; ++w) before += s_warp[w];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s_before[threadIdx.x * 4 + k] = before;
      before += turns[k];
    }
    if (threadIdx.x == kJoinThreads - 1) s_before[kMostCuts] = before;
    __syncthreads();
  }
  const int all_turns = s_before[kMostCuts];
  for (int turn = blockIdx.x; turn < all_turns; turn += gridDim.x) {
    int at = 0;  // the cut with s_before[at] <= turn < s_before[at + 1]
#pragma unroll
    for (int step2 = kMostCuts / 2; step2 > 0; step2 >>= 1)
      if (s_before[at + step2] <= turn) at += step2;
    const bool is_few = at < few.pieces;
    const Pieces& p = is_few ? few : many;
    const int cut = at - (is_few ? 0 : few.pieces);
    const PagedCut c = p.cuts[cut];
    const int R = p.rows, n = c.last - cut + 2;  // parts: of piece cut - 1, which left the tile's beginning in its second place, and
                                                 // of the others to `last`, in their first
    const size_t floats = static_cast<size_t>(R) * (D + 2);
    auto part = [&](int i) { return p.parts + (static_cast<size_t>(cut - 1 + i) * 2 + (i == 0 ? 1 : 0)) * floats; };
    const int r0 = ((turn - s_before[at]) * kJoinWarps + warp) * kJoinRows;
    if (n == 2) {
      float2 ml[kJoinRows][2];
      Vec v[kJoinRows][2];
#pragma unroll
      for (int k = 0; k < kJoinRows; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = min(r0 + k, c.rows - 1);
          ml[k][i] = *reinterpret_cast<const float2*>(part(i) + R * D + 2 * r);
          v[k][i] = reinterpret_cast<const Vec*>(part(i) + r * D)[lane];
        }
#pragma unroll
      for (int k = 0; k < kJoinRows; ++k) {
        if (r0 + k >= c.rows) break;
        const float top = fmaxf(ml[k][0].x, ml[k][1].x), w0 = exp2_fast(ml[k][0].x - top), w1 = exp2_fast(ml[k][1].x - top);
        float x[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = reinterpret_cast<const float*>(&v[k][0])[e] * w0 + reinterpret_cast<const float*>(&v[k][1])[e] * w1;
        finish_row<T, k8, D>(a, c, r0 + k, ml[k][0].y * w0 + ml[k][1].y * w1, x, lane);
      }
      continue;
    }
    for (int r = r0; r < min(r0 + kJoinRows, c.rows); ++r) {
      float m, l, x[kPer];
      add_parts<D>(part, R, r, 0, 1, n, lane, m, l, x);
      finish_row<T, k8, D>(a, c, r, l, x, lane);
    }
  }
}

template <typename T, bool k8, int D>
int launch_join(const PagedAttn& a, const Pieces& few, const Pieces& many, cudaStream_t stream) {
  if (few.pieces + many.pieces > kMostCuts) return FTB_ERR_ARG;  // (a device of 256 SMs)
  static std::atomic<unsigned long long> divided{0}, divided_few{0};
  if (!set_smem_carveout(paged_join_kernel<T, k8, D>, kPagedCarveout, divided) ||
      !set_smem_carveout(paged_join_few_kernel<T, k8, D>, kPagedCarveout, divided_few))
    return FTB_ERR_LAUNCH;
  const cudaError_t err =
      many.pieces == 0 ? launch_dependent(paged_join_few_kernel<T, k8, D>, dim3(few.pieces, few.rows), dim3(kFewWarps * 32), 0, stream, a, few)
                       : launch_dependent(paged_join_kernel<T, k8, D>, dim3(3 * current_sm_count()), dim3(kJoinThreads), 0, stream, a, few, many);
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}
template <typename T>
int launch_join(const PagedAttn& a, int d, const Pieces& few, const Pieces& many, cudaStream_t stream) {
  if (a.k_exp != nullptr) return d == 128 ? launch_join<T, true, 128>(a, few, many, stream) : launch_join<T, true, 64>(a, few, many, stream);
  return d == 128 ? launch_join<T, false, 128>(a, few, many, stream) : launch_join<T, false, 64>(a, few, many, stream);
}

// What runs: few > 0: paged_short.cu with tiles of so many rows for sequences of up to `most` rows; many > 0: paged_tile.cu with tiles
// of so many for the others.
struct Form {
  int few, most, many;
};
Form form_of(int T, int B, int group) {
  const long long rows = static_cast<long long>(T) * group;
  // Not more tokens than sequences: a decoding step.  Where one of them has most of the tokens, its tiles read the keys once each, through
  // L2: 256 sequences, all but one without a token, 8 kv heads, 1000 keys, 24 tokens 23 us (with paged_tile.cu beside it 32), 100 tokens
  // 56 (39), 200 tokens 108 (41).  A step of a token each pays for that second launch: 8 sequences 15 us (23), 64 of up to 8000 keys 179
  // (186).  Which it is stands on the device alone.
  if (T <= B) return {rows <= 8ll * B ? 8 : 16, INT_MAX, 0};
  if (rows <= 16) return {rows <= 8 ? 8 : 16, INT_MAX, 0};
  const int many = rows > 128ll * B ? 256 : 128;
  if (B == 1) return {0, 0, many};
  // One tile of paged_short.cu: a second one would read the keys again.  96 sequences, 8 kv heads, 4500 keys of 16 bits: 8 rows
  // 273 us, 16 rows 302, as rows of paged_tile.cu 24 349, 64 367, 128 405; 8500 keys of 8 bits: 327, 400, then 650, 679, 728.
  const int few = group <= 8 && rows > 16ll * B ? 8 : 16;
  return {few, few, many};
}

// Whether n numbers at o (16 bits) meet the numbers of some of T rows of heads at q.
bool over_rows(const void* o, long long n, const void* q, int T, long long q_row, int heads, long long q_head, int d) {
  const long long span = (heads - 1) * q_head, lo = std::min(0ll, span), hi = std::max(0ll, span) + d;  // of a row
  const long long step = T > 1 ? std::abs(q_row) : 0, first = T > 1 && q_row < 0 ? (T - 1) * q_row : 0;
  // o's beginning, in numbers from where the lowest row is (both on 16-byte boundaries)
  const long long at = static_cast<long long>(reinterpret_cast<uintptr_t>(o) - reinterpret_cast<uintptr_t>(q)) / 2 - first;
  if (step == 0) return at < hi && at + n > lo;
  // rows r with r * step + hi > at and r * step + lo < at + n
  auto floor_div = [](long long x, long long y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
  const long long r0 = std::max(0ll, floor_div(at - hi, step) + 1), r1 = std::min(T - 1ll, floor_div(at + n - lo - 1, step));
  return r0 <= r1;
}

size_t places(int pieces, int rows, int d) { return 2 * static_cast<size_t>(pieces) * rows * (d + 2) * sizeof(float) + pieces * sizeof(PagedCut); }
size_t rounded(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" size_t ftb_paged_attn_scratch_bytes(int T, int B, int kv_heads, int group, int d) {
  if (T <= 0 || B <= 0 || kv_heads <= 0 || group <= 0 || d <= 0) return 0;
  const Form f = form_of(T, B, group);
  size_t n = rounded(static_cast<size_t>(T) * kv_heads * group * sizeof(uint32_t));
  if (f.few > 0) n += rounded(places(paged_short_pieces(f.few), f.few, d));
  if (f.many > 0) n += rounded(places(paged_tile_pieces(), f.many, d));
  return n;
}

extern "C" int ftb_paged_attn_fwd(const void* q, long long q_row, long long q_head, const void* k_cache, const void* v_cache,
                                  const unsigned char* k_exp, const unsigned char* v_exp, const int* table, const int* lens,
                                  const int* starts, void* o, int T, int B, int W, int pages, int kv_heads, int group,
                                  int page_size, int d, int window, float scale, int dtype, void* scratch, size_t scratch_bytes,
                                  void* workspace, size_t workspace_bytes, void* stream_) {
  if ((T > 0 && (!q || !o)) || !k_cache || !v_cache || !table || !lens || !starts || (k_exp == nullptr) != (v_exp == nullptr)) return FTB_ERR_ARG;
  if (T < 0 || B <= 0 || W <= 0 || pages <= 0 || kv_heads <= 0 || group <= 0 || window < 0) return FTB_ERR_ARG;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return FTB_ERR_ARG;
  if ((d != 64 && d != 128) || (dtype != FTB_F16 && dtype != FTB_BF16)) return FTB_ERR_ARG;
  if (!(scale > 0.f) || !(scale * kLog2E <= FLT_MAX)) return FTB_ERR_ARG;  // hidden scores are -inf behind the scale, those of 0 are not
  if (static_cast<long long>(kv_heads) * group > 65536 || static_cast<long long>(T) * group > INT_MAX) return FTB_ERR_ARG;
  if (((q_row | q_head) & 7) != 0) return FTB_ERR_ALIGN;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(k_cache) |
        reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(k_exp) | reinterpret_cast<uintptr_t>(v_exp)) & 15) != 0)
    return FTB_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  if (T == 0) return FTB_OK;
  // queries are read again by other blocks than those that write their rows, and so are pages
  const int heads = kv_heads * group;
  const size_t o_bytes = 2 * static_cast<size_t>(T) * heads * d, numbers = static_cast<size_t>(pages) * kv_heads * page_size * d;
  const size_t cache_bytes = k_exp != nullptr ? numbers : 2 * numbers, exp_bytes = k_exp != nullptr ? numbers / d : 0;
  if (over_rows(o, static_cast<long long>(o_bytes / 2), q, T, q_row, heads, q_head, d) || overlap(o, o_bytes, k_cache, cache_bytes) ||
      overlap(o, o_bytes, v_cache, cache_bytes) || overlap(o, o_bytes, k_exp, exp_bytes) || overlap(o, o_bytes, v_exp, exp_bytes))
    return FTB_ERR_ARG;
  const int rc = check_device_sm100();
  if (rc) return rc;
  PagedAttn a;
  a.batch = {table, lens, starts, B, W, pages, 31 - __builtin_clz(static_cast<unsigned>(page_size))};
  a.q = q;
  a.o = o;
  a.q_row = q_row;
  a.q_head = q_head;
  a.k = static_cast<const unsigned char*>(k_cache);
  a.v = static_cast<const unsigned char*>(v_cache);
  a.k_exp = k_exp;
  a.v_exp = v_exp;
  a.T = T;
  a.kv_heads = kv_heads;
  a.group = group;
  a.window = window;
  a.scale_log2 = scale * kLog2E;
  a.status = static_cast<int*>(workspace);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (scratch == nullptr || scratch_bytes < ftb_paged_attn_scratch_bytes(T, B, kv_heads, group, d)) return FTB_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(scratch) & 15) != 0) return FTB_ERR_ALIGN;
  const Form f = form_of(T, B, group);
  unsigned char* at = static_cast<unsigned char*>(scratch);
  a.odd = static_cast<uint32_t*>(scratch);
  at += rounded(static_cast<size_t>(T) * kv_heads * group * sizeof(uint32_t));
  auto pieces_at = [&](int pieces, int rows) {
    float* parts = reinterpret_cast<float*>(at);
    return Pieces{parts, reinterpret_cast<const PagedCut*>(parts + 2 * static_cast<size_t>(pieces) * rows * (d + 2)), pieces, rows};
  };
  Pieces few{nullptr, nullptr, 0, 0}, many{nullptr, nullptr, 0, 0};
  int err = FTB_OK;
  // (the kernel for few rows first: it lives on L1, of which the other one's shared memory leaves next to nothing until an SM is
  // empty: 378 against 294 us behind it for 96 sequences of 16 rows)
  if (f.few > 0) {
    a.least_rows = 1;
    a.most_rows = f.most;
    few = pieces_at(paged_short_pieces(f.few), f.few);
    err = paged_short_launch(a, d, dtype, f.few, at, stream);
    at += rounded(places(few.pieces, f.few, d));
  }
  if (f.many > 0 && err == FTB_OK) {
    a.least_rows = f.most + 1;
    a.most_rows = INT_MAX;
    many = pieces_at(paged_tile_pieces(), f.many);
    err = paged_tile_launch(a, d, dtype, f.many, at, stream);
  }
  if (err != FTB_OK) return err;
  return dtype == FTB_F16 ? launch_join<__half>(a, d, few, many, stream) : launch_join<__nv_bfloat16>(a, d, few, many, stream);
}
