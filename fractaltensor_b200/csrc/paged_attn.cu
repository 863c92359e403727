// Attention of new tokens over a paged cache: o = sum_j softmax_j(scale * q . k_j) v_j over the keys j with
// pos - window < j <= pos, for a token at position pos, heads = group * kv_heads.
#include <cfloat>
#include <climits>

#include "../../include/ftb200.h"
#include "paged_attn.cuh"
#include "tmap.h"

namespace ftb {
namespace {

constexpr int kRowWarps = 4;

// The simplest form: a warp a (token, head).
template <typename T, bool k8, int D>
__global__ void __launch_bounds__(kRowWarps * 32)
paged_rows_kernel(PagedAttn a) {
  __shared__ float s_q[kRowWarps][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * kRowWarps + warp;
  grid_launch_dependents();
  grid_dependency_wait();
  const int heads = a.kv_heads * a.group;
  if (row >= static_cast<long long>(a.T) * heads) return;
  const int t = static_cast<int>(row / heads), head = static_cast<int>(row - static_cast<long long>(t) * heads);
  const int b = sequence_of_row(a.batch, t, lane);
  if (b >= a.batch.B) return;
  attend_row<T, k8, D>(a, b, t, head, position_of_row(a.batch, b, t), s_q[warp], lane);
}

template <typename T, bool k8, int D>
int launch_rows(const PagedAttn& a, cudaStream_t stream) {
  const long long rows = static_cast<long long>(a.T) * a.kv_heads * a.group, grid = (rows + kRowWarps - 1) / kRowWarps;
  if (grid > INT_MAX) return FTB_ERR_ARG;
  const cudaError_t err = launch_light(paged_rows_kernel<T, k8, D>, dim3(static_cast<unsigned>(grid)), dim3(kRowWarps * 32), 0, stream, a);
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}
template <typename T>
int launch_rows(const PagedAttn& a, int d, cudaStream_t stream) {
  if (a.k_exp != nullptr) return d == 128 ? launch_rows<T, true, 128>(a, stream) : launch_rows<T, true, 64>(a, stream);
  return d == 128 ? launch_rows<T, false, 128>(a, stream) : launch_rows<T, false, 64>(a, stream);
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" size_t ftb_paged_attn_scratch_bytes(int T, int B, int kv_heads, int group, int d) { return 0; }

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
  if (static_cast<long long>(kv_heads) * group > 65536) return FTB_ERR_ARG;
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
  return dtype == FTB_F16 ? launch_rows<__half>(a, d, stream) : launch_rows<__nv_bfloat16>(a, d, stream);
}
