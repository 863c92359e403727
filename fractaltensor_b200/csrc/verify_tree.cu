// Trees of drafted tokens: what a token of a tree sees, and the verification of a tree against the target's probabilities.
//
// Tokens 0 .. N - 1 of a sequence, token 0 the last one that is certain, parents[i] < i; p_i are the target's probabilities behind token i.
// The path begins at token 0.  The drafted tokens x_c behind the token `at` that it has come to are asked in their order: with r the sum
// of p_at of those refused before it, c is taken if u_c * (1 - r) < p_at(x_c), which takes x with probability p_at(x) whatever
// else was drafted; the path goes on from there.  Where none is taken a token is drawn by u_0 from p_at without those refused.
//
// Whether a token is taken once its parent is on the path depends on its siblings alone, so that a thread a token finds that, all at once:
// the path is then a chain of first children taken.  (One warp that asked them one behind the other took 4 us for 25 tokens, of 10.)  Every
// token's number in its parent's row is loaded beforehand; then one row is read whole (draft_draw.cuh).
//
// 60 trees of 33 tokens over 130 001 words 20.7 us, 1.5 TB/s; one of 25 over 49 152 10 to 11.  Bound by steps one behind the other: parents and
// tokens, their numbers, the path, the row (14 us of 27 before eight numbers a thread were on their way beside those that are weighed), the
// others' sums, the stretch.
#include <climits>

#include "../../include/ftb200.h"
#include "draft_draw.cuh"
#include "paged_forms.h"
#include "tmap.h"

namespace ftb {
namespace {

// ----------------------------------------------------------------------------------------------- mask
constexpr int kMaskThreads = 128;

// A thread a token: the way up to its first ancestor, which meets the words of its bits from the last to the first.
__global__ void __launch_bounds__(kMaskThreads)
tree_mask_kernel(const int* __restrict__ parents, uint32_t* __restrict__ mask, long long rows, int N, int words) {
  const long long row = static_cast<long long>(blockIdx.x) * kMaskThreads + threadIdx.x;
  grid_launch_dependents();
  grid_dependency_wait();
  if (row >= rows) return;
  const int* of = parents + row / N * N;
  int i = static_cast<int>(row % N), w = words - 1;
  uint32_t* to = mask + row * words;
  uint32_t bits = 0;
  for (;;) {
    for (; w > i >> 5; --w) {
      to[w] = bits;
      bits = 0;
    }
    bits |= 1u << (i & 31);
    const int up = of[i];
    if (up < 0 || up >= i) break;  // (one that does not lie in front is none)
    i = up;
  }
  for (; w >= 0; --w) {
    to[w] = bits;
    bits = 0;
  }
}

// --------------------------------------------------------------------------------------- verification
constexpr int kMostTokens = 1024;

struct Tree {
  const float* p;
  const long long* tokens;
  const int* parents;
  const float* u;
  long long p_seq, p_row;
  int N, V;
};

// p without the refused tokens, which a warp looks for before it weighs some hundred numbers.  (Looked for at every number, a batch of 60 rows of
// 130 001 took 61 us.)
struct TreeRow {
  const float* pr;
  const int* refused;
  int n;
  bool some;

  __device__ __forceinline__ float p(int j) const { return pr[j]; }
  __device__ __forceinline__ float q(int) const { return 0.f; }
  __device__ __forceinline__ void look(int j, int count) {
    some = false;
    for (int i = threadIdx.x & 31; i < n; i += 32) some |= static_cast<unsigned>(refused[i] - j) < static_cast<unsigned>(count);
    some = __any_sync(0xffffffffu, some);
  }
  __device__ __forceinline__ double weight(float p, float, int j) const {
    double w = probability(p);
    if (some) {
      for (int i = 0; i < n; ++i)
        if (refused[i] == j) w = 0.0;
    }
    return w;
  }
  __device__ __forceinline__ void all() { n = 0; }
};

struct TreeRoom {  // in shared memory
  int token[kMostTokens], parent[kMostTokens], path[kMostTokens], refused[kMostTokens], next[kMostTokens];
  float u[kMostTokens], p[kMostTokens];
  int length, n_refused;
};

// All threads: the path, and the tokens that were refused behind its last one.
template <int kThreads>
__device__ __forceinline__ void find_path(TreeRoom& t, int N) {
  // a token that a sibling in front of it has too counts as 0
  for (int c = threadIdx.x; c < N; c += kThreads) {
    const int parent = t.parent[c], token = t.token[c];
    bool again = false;
    for (int j = max(parent, 0) + 1; j < c; ++j) again |= t.parent[j] == parent && t.token[j] == token;
    t.refused[c] = again;
    t.next[c] = INT_MAX;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < N; c += kThreads)
    if (t.refused[c] != 0) t.p[c] = 0.f;
  __syncthreads();
  for (int c = threadIdx.x; c < N; c += kThreads) {
    const int parent = t.parent[c];
    if (parent < 0) continue;
    double rest = 1.0;
    for (int j = parent + 1; j < c; ++j)
      if (t.parent[j] == parent) rest = fmax(rest - probability(t.p[j]), 0.0);
    if (static_cast<double>(t.u[c]) * rest < probability(t.p[c])) atomicMin(&t.next[parent], c);
  }
  if (threadIdx.x == 0) t.n_refused = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int at = 0; at < N; at = t.next[at]) t.path[n++] = at;  // (INT_MAX behind the last one)
    t.length = n;
  }
  __syncthreads();
  const int last = t.path[t.length - 1];
  for (int c = threadIdx.x; c < N; c += kThreads)
    if (t.parent[c] == last && t.token[c] >= 0) t.refused[atomicAdd(&t.n_refused, 1)] = t.token[c];
  __syncthreads();
}

// C: CTAs of a cluster, 1 or 8.
template <int C, int kThreads>
__global__ void __launch_bounds__(kThreads, C == 8 && kThreads == 512 ? 1 : 1024 / kThreads)
verify_tree_kernel(const __grid_constant__ Tree a, long long* __restrict__ tokens, int* __restrict__ path, int* __restrict__ counts_out, int* __restrict__ status) {
  __shared__ DrawRoom<C, kThreads> room;
  __shared__ TreeRoom t;
  const int b = blockIdx.x / C, rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  grid_dependency_wait();
  grid_launch_dependents();
  const int N = a.N, V = a.V;
  const long long seq = static_cast<long long>(b) * N;
  const float* p = a.p + b * a.p_seq;
  for (int i = threadIdx.x; i < N; i += kThreads) {
    const int parent = i > 0 ? a.parents[seq + i] : -1;
    const long long x = a.tokens[seq + i];
    const bool drafted = parent >= 0 && parent < i, known = x >= 0 && x < V;
    if (drafted && !known && rank == 0) atomicCAS(status, 0, FTB_ERR_INDEX);
    t.parent[i] = drafted ? parent : -1;
    t.token[i] = known ? static_cast<int>(x) : -1;
    t.u[i] = a.u[seq + i];
    t.p[i] = drafted && known ? p[parent * a.p_row + x] : 0.f;
  }
  __syncthreads();
  find_path<kThreads>(t, N);
  const int n = t.length;
  TreeRow row{p + t.path[n - 1] * a.p_row, t.refused, t.n_refused, false};
  const double total = draw_token<C, kThreads, true>(row, V, &t.u[0], rank, room, [&](int token) { tokens[seq + n - 1] = token; });
  if (rank == 0) {
    for (int i = threadIdx.x; i < N; i += kThreads) {
      if (i != n - 1 || !(total > 0.0)) tokens[seq + i] = i < n - 1 ? t.token[t.path[i + 1]] : -1;
      path[seq + i] = i < n ? t.path[i] : -1;
    }
    if (threadIdx.x == 0) {
      if (!(total > 0.0)) atomicCAS(status, 0, FTB_ERR_INDEX);
      counts_out[b] = n;
    }
  }
  if constexpr (C > 1) cluster_sync_all();  // nobody leaves while its sum may be read
}

template <int C, int kThreads>
cudaError_t launch(const Tree& a, int B, long long* tokens, int* path, int* counts_out, int* status, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B) * C);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, verify_tree_kernel<C, kThreads>, a, tokens, path, counts_out, status);
}

int launched(cudaError_t err) {
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" int ftb_tree_mask(const int* parents, int* mask, int B, int N, void* stream) {
  if (B < 0 || N < 0 || (B > 0 && N > 0 && (!parents || !mask))) return FTB_ERR_ARG;
  const long long rows = static_cast<long long>(B) * N;
  if (rows > INT_MAX) return FTB_ERR_ARG;
  if (rows == 0) return FTB_OK;
  const int words = (N + 31) / 32;
  if (overlap(parents, rows * sizeof(int), mask, static_cast<size_t>(rows) * words * sizeof(int))) return FTB_ERR_ARG;
  const int rc = check_device_sm100();
  if (rc) return rc;
  return launched(launch_light(tree_mask_kernel, dim3(static_cast<unsigned>((rows + kMaskThreads - 1) / kMaskThreads)), dim3(kMaskThreads), 0,
                               static_cast<cudaStream_t>(stream), parents, reinterpret_cast<uint32_t*>(mask), rows, N, words));
}

extern "C" int ftb_verify_tree(const float* probs, long long p_seq, long long p_row, const long long* tokens, const int* parents, const float* u,
                               long long* tokens_out, int* path, int* counts_out, int B, int N, int V, void* workspace, size_t workspace_bytes,
                               void* stream) {
  if (B < 0 || N <= 0 || N > kMostTokens || V <= 0 || V > 1 << 30 || B > INT_MAX / 8) return FTB_ERR_ARG;
  if (B > 0 && (!probs || !tokens || !parents || !u || !tokens_out || !path || !counts_out)) return FTB_ERR_ARG;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  if (B == 0) return FTB_OK;
  // (the CTAs of a sequence read its tokens and parents each for itself, while one of them may write results already)
  const size_t rows = static_cast<size_t>(B) * N;
  const void* in[3] = {tokens, parents, u};
  const size_t in_bytes[3] = {rows * 8, rows * 4, rows * 4};
  const void* out[3] = {tokens_out, path, counts_out};
  const size_t out_bytes[3] = {rows * 8, rows * 4, static_cast<size_t>(B) * 4};
  for (int o = 0; o < 3; ++o) {
    for (int i = 0; i < 3; ++i)
      if (overlap(out[o], out_bytes[o], in[i], in_bytes[i])) return FTB_ERR_ARG;
    if (over_rows(out[o], static_cast<long long>(out_bytes[o] / 2), probs, B, 2 * p_seq, N, 2 * p_row, 2ll * V)) return FTB_ERR_ARG;
    for (int i = 0; i < o; ++i)
      if (overlap(out[o], out_bytes[o], out[i], out_bytes[i])) return FTB_ERR_ARG;
  }
  const int rc = check_device_sm100();
  if (rc) return rc;
  const Tree a{probs, tokens, parents, u, p_seq, p_row, N, V};
  int* st = static_cast<int*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // As for drafts (verify_drafts.cu): clusters where a row has more than a few numbers a thread, small CTAs where there are many.
  return launched(V <= 4096                              ? launch<1, 512>(a, B, tokens_out, path, counts_out, st, s)
                  : B <= current_sm_count() / 8 ? launch<8, 512>(a, B, tokens_out, path, counts_out, st, s)
                                                                 : launch<8, 256>(a, B, tokens_out, path, counts_out, st, s));
}
