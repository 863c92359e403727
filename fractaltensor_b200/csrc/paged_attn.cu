// Attention of new tokens over a paged cache: o = sum_j softmax_j(scale * q . k_j) v_j over the keys j with
// pos - window < j <= pos, for a token at position pos, heads = group * kv_heads.
//
// Two kernels: paged_short.cu for sequences with few rows (token, head of a group), bound by the bytes of their keys and values, and
// paged_tile.cu for those with many, by matrix products on tiles of rows.  A call with both kinds runs both, each on its own; the
// lengths are on the device, so that it is there that a sequence is one or the other's.  Here: the choice, and what joins the tiles
// that the cuts between pieces of work went through.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "../../include/ftb200.h"
#include "paged_forms.h"
#include "paged_work.cuh"
#include "tmap.h"

namespace ftb {
namespace {

constexpr int kJoinThreads = 128, kJoinBlocks = 8;

struct Pieces {
  const float* parts;
  const PagedCut* cuts;
  int pieces, rows;  // rows of a tile
};

// Block (x, y): the tile with cut x of the two kernels' cuts, every kJoinBlocks-th group of its rows.
template <typename T, bool k8, int D>
__global__ void __launch_bounds__(kJoinThreads)
paged_join_kernel(const __grid_constant__ PagedAttn a, Pieces few, Pieces many) {
  constexpr int kRows = kJoinThreads / (D / 4);
  __shared__ int s_odd[kRows];
  grid_dependency_wait();
  grid_launch_dependents();
  // rows of whole tiles that have to be computed again (none, unless something in the cache is not finite)
  {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = a.kv_heads * a.group;
    const long long rows = static_cast<long long>(a.T) * heads, step = static_cast<long long>(gridDim.x) * gridDim.y * kJoinThreads;
    for (long long r0 = (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * kJoinThreads + warp * 32; r0 < rows; r0 += step) {
      unsigned again = __ballot_sync(0xffffffffu, r0 + lane < rows && a.odd[min(r0 + lane, rows - 1)] != 0);
      while (again != 0) {
        const long long row = r0 + __ffs(again) - 1;
        again &= again - 1;
        const int t = static_cast<int>(row / heads), b = sequence_of_row(a.batch, t, lane);
        if (b < a.batch.B)  // (what no sequence has was not written either)
          attend_row<T, k8, D>(a, b, t, static_cast<int>(row - static_cast<long long>(t) * heads), position_of_row(a.batch, b, t), lane);
      }
    }
  }
  const bool is_few = static_cast<int>(blockIdx.x) < few.pieces;
  const Pieces& p = is_few ? few : many;
  const int cut = blockIdx.x - (is_few ? 0 : few.pieces);
  const PagedCut& c = p.cuts[cut];
  const int last = c.last;
  if (last < 0) return;
  const int R = p.rows, rows = c.rows;
  const size_t floats = static_cast<size_t>(R) * (D + 2);
  const int sub = threadIdx.x / (D / 4), d = (threadIdx.x - sub * (D / 4)) * 4, warp = threadIdx.x >> 5;
  for (int r0 = blockIdx.y * kRows; r0 < rows; r0 += kJoinBlocks * kRows) {
    if (threadIdx.x < kRows) s_odd[threadIdx.x] = 0;
    __syncthreads();
    const int r = r0 + sub, flat = c.flat0 + r, t = c.first + flat / a.group, head = c.h * a.group + flat % a.group;
    if (r < rows) {
      // piece cut - 1 left the tile's beginning (its second place), the others what follows (their first)
      auto part = [&](int i) { return p.parts + (static_cast<size_t>(i) * 2 + (i == cut - 1 ? 1 : 0)) * floats; };
      float top = -FLT_MAX;
#pragma unroll 8
      for (int i = cut - 1; i <= last; ++i) top = fmaxf(top, part(i)[R * D + 2 * r]);
      float sum = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int i = cut - 1; i <= last; ++i) {
        const float2 ml = *reinterpret_cast<const float2*>(part(i) + R * D + 2 * r);
        const float4 y = *reinterpret_cast<const float4*>(part(i) + r * D + d);
        const float k = exp2_fast(ml.x - top);
        sum = fmaf(ml.y, k, sum);
        x.x = fmaf(y.x, k, x.x);
        x.y = fmaf(y.y, k, x.y);
        x.z = fmaf(y.z, k, x.z);
        x.w = fmaf(y.w, k, x.w);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      x.x *= inv;
      x.y *= inv;
      x.z *= inv;
      x.w *= inv;
      const float all = x.x + x.y + x.z + x.w;
      if (all != all) s_odd[sub] = 1;
      *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + (static_cast<long long>(t) * a.kv_heads * a.group + head) * D + d) =
          make_uint2(Fmt<T>::pack2(x.x, x.y), Fmt<T>::pack2(x.z, x.w));
    }
    __syncthreads();
    for (int i = warp; i < kRows; i += kJoinThreads / 32) {
      const int flat_i = c.flat0 + r0 + i, ti = c.first + flat_i / a.group;
      if (r0 + i < rows && s_odd[i] != 0 && hides(a, c.pos0 + ti, c.lo, c.hi))
        attend_row<T, k8, D>(a, c.b, ti, c.h * a.group + flat_i % a.group, c.pos0 + ti, threadIdx.x & 31);
    }
    __syncthreads();
  }
}

template <typename T, bool k8, int D>
int launch_join(const PagedAttn& a, const Pieces& few, const Pieces& many, cudaStream_t stream) {
  const cudaError_t err = launch_dependent(paged_join_kernel<T, k8, D>, dim3(few.pieces + many.pieces, kJoinBlocks), dim3(kJoinThreads), 0,
                                           stream, a, few, many);
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
  // Not more tokens than sequences: a decoding step.  (Where one of them has them all the others are empty, and its tiles
  // are read through L2.)
  if (T <= B) return {rows <= 8ll * B ? 8 : 16, INT_MAX, 0};
  if (rows <= 16) return {rows <= 8 ? 8 : 16, INT_MAX, 0};
  const int many = rows > 128ll * B ? 256 : 128;
  if (B == 1) return {0, 0, many};
  // One tile of paged_short.cu: a second one would read the keys again.  16 rows of it take 1.4 to 1.9 times what 8 take, and
  // about what a tile of 128 does (96 sequences of 4500 keys of 16 bits, 8 kv heads: 8 rows 268 us, 16 378, 128 392; of 8500 of
  // 8 bits: 310, 509, 657).
  const int few = group <= 8 && rows > 16ll * B ? 8 : 16;
  return {few, few, many};
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
  if (!(scale > 0.f) || !(scale <= FLT_MAX)) return FTB_ERR_ARG;  // hidden scores are -inf behind the scale
  if (static_cast<long long>(kv_heads) * group > 65536 || static_cast<long long>(T) * group > INT_MAX) return FTB_ERR_ARG;
  if (((q_row | q_head) & 7) != 0) return FTB_ERR_ALIGN;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(k_cache) |
        reinterpret_cast<uintptr_t>(v_cache)) & 15) != 0)
    return FTB_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  if (T == 0) return FTB_OK;
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
  a.scale_log2 = scale * 1.4426950408889634f;
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
  if (f.many > 0) {
    a.least_rows = f.most + 1;
    a.most_rows = INT_MAX;
    many = pieces_at(paged_tile_pieces(), f.many);
    err = paged_tile_launch(a, d, dtype, f.many, at, stream);
    at += rounded(places(many.pieces, f.many, d));
  }
  if (f.few > 0 && err == FTB_OK) {
    a.least_rows = 1;
    a.most_rows = f.most;
    few = pieces_at(paged_short_pieces(f.few), f.few);
    err = paged_short_launch(a, d, dtype, f.few, at, stream);
  }
  if (err != FTB_OK) return err;
  return dtype == FTB_F16 ? launch_join<__half>(a, d, few, many, stream) : launch_join<__nv_bfloat16>(a, d, few, many, stream);
}
