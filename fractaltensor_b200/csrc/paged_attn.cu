// Attention of new tokens over a paged cache: o = sum_j softmax_j(scale * q . k_j) v_j over the keys j with
// pos - window < j <= pos, for a token at position pos, heads = group * kv_heads.
#include <cfloat>
#include <climits>

#include "../../include/ftb200.h"
#include "paged_attn.cuh"
#include "paged_short.h"
#include "tmap.h"

namespace ftb {
namespace {

// Rows of a tile / 8, by the rows (token, head of a group) that a sequence has on average.
int short_form(int T, int B, int group) { return static_cast<long long>(T) * group <= 8ll * B ? 1 : 2; }

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" size_t ftb_paged_attn_scratch_bytes(int T, int B, int kv_heads, int group, int d) {
  if (T <= 0 || B <= 0 || kv_heads <= 0 || group <= 0 || d <= 0) return 0;
  return paged_short_scratch_bytes(short_form(T, B, group), d);
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
  if (scratch == nullptr || scratch_bytes < ftb_paged_attn_scratch_bytes(T, B, kv_heads, group, d)) return FTB_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(scratch) & 15) != 0) return FTB_ERR_ALIGN;
  return paged_short_launch(a, d, dtype, short_form(T, B, group), static_cast<float*>(scratch), stream);
}
