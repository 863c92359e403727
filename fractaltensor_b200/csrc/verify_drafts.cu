// Verification of drafted tokens against the target's probabilities, from random numbers that the caller gives.
//
// Sequence b has K drafted tokens x_0 .. x_{K-1}, drawn from the draft's probabilities q_i, and the target's
// probabilities p_0 .. p_K.  Draft i is taken if u_i * q_i(x_i) < p_i(x_i) (probability min(1, p / q)), the first that is
// not ends the run at n; token n is drawn from w = max(p_n - q_n, 0), or from p_K behind K taken drafts: the first j
// with w_0 + .. + w_j > u_K * sum(w).  Drafts without probabilities were certain: q_i is 1 at x_i.
//
// Only one row of p (and of q) a sequence is read whole.  Sums are kept in 64 bits: the chosen index follows from a
// comparison with a partial sum of up to V numbers, and in 32 bits the order of summation would decide it.
//
// Bound by the bytes of those rows: 100 sequences of 5 drafts over 130 001 words 29.9 us, 3.5 TB/s (one: 7.1 us, trips to memory one
// behind the other: the drafts' probabilities, the row, the stretch).  A cluster of CTAs takes a sequence, every warp a stretch of the row: one pass for the
// stretches' sums, which the CTAs hand each other through distributed shared memory, and a second look at the one stretch (a 64th of
// the row or less) in which the limit is passed.  Every CTA finds n on its own, which saves a step of waiting.
#include <climits>

#include "../../include/ftb200.h"
#include "draft_draw.cuh"
#include "tmap.h"

namespace ftb {
namespace {

struct Drafts {
  const float* p;
  const float* q;  // or nullptr
  const long long* drafts;
  const float* u;
  const int* counts;  // or nullptr: K each
  long long p_seq, p_row, q_seq, q_row;
  int K, V;
};

// What is left of p where q is taken from it, without one draft.
struct DraftRow {
  const float *pr, *qr;  // qr may be nullptr
  int without;           // or -1

  __device__ __forceinline__ float p(int j) const { return pr[j]; }
  __device__ __forceinline__ float q(int j) const { return qr != nullptr ? qr[j] : 0.f; }
  __device__ __forceinline__ void look(int, int) const {}
  __device__ __forceinline__ double weight(float p, float q, int j) const {
    const double w = static_cast<double>(p) - probability(q);  // (nothing is left of a p that is not positive)
    return w > 0.0 && p < __int_as_float(0x7f800000) && j != without ? w : 0.0;
  }
  __device__ __forceinline__ void all() {
    qr = nullptr;
    without = -1;
  }
};

// C: CTAs of a cluster, 1 or 8.  (512 threads and a cluster: for few sequences, a CTA an SM at most; the others have 40 registers, without spills.  With 28 and 16
// bytes of them, as when draw_token took the random number and the token's place as values, a batch took 31.4 us and one 7.9.)
template <int C, int kThreads>
__global__ void __launch_bounds__(kThreads, C == 8 && kThreads == 512 ? 1 : 1536 / kThreads)
verify_drafts_kernel(Drafts a, long long* __restrict__ tokens, int* __restrict__ counts_out, int* __restrict__ status) {
  __shared__ DrawRoom<C, kThreads> room;
  __shared__ int s_n;
  const int b = blockIdx.x / C, rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  if (threadIdx.x == 0) s_n = a.K;
  __syncthreads();
  grid_dependency_wait();
  grid_launch_dependents();
  const int K = a.K, V = a.V;
  const long long* x = a.drafts + static_cast<long long>(b) * K;
  const float* u = a.u + static_cast<long long>(b) * (K + 1);
  const float* p = a.p + b * a.p_seq;
  const float* q = a.q != nullptr ? a.q + b * a.q_seq : nullptr;
  long long id = threadIdx.x < K ? x[threadIdx.x] : 0;  // (on its way beside the count)
  const int mine = a.counts != nullptr ? min(max(a.counts[b], 0), K) : K;
  for (int i = threadIdx.x; i < mine; i += kThreads) {
    if (i >= kThreads) id = x[i];
    bool taken = false;
    if (id >= 0 && id < V) {
      const double qx = q != nullptr ? probability(q[i * a.q_row + id]) : 1.0;
      taken = static_cast<double>(u[i]) * qx < probability(p[i * a.p_row + id]);
    } else if (rank == 0) {
      atomicCAS(status, 0, FTB_ERR_INDEX);
    }
    if (!taken) atomicMin(&s_n, i);
  }
  __syncthreads();
  const int n = min(s_n, mine);
  DraftRow row{p + n * a.p_row, q != nullptr && n < mine ? q + n * a.q_row : nullptr,
               q == nullptr && n < mine && x[n] >= 0 && x[n] < V ? static_cast<int>(x[n]) : -1};
  const double total = draw_token<C, kThreads, false>(row, V, u + K, rank, room, [&](int token) { tokens[static_cast<long long>(b) * (K + 1) + n] = token; });
  if (rank == 0) {
    for (int i = threadIdx.x; i <= K; i += kThreads)
      if (i != n || !(total > 0.0)) tokens[static_cast<long long>(b) * (K + 1) + i] = i < n ? x[i] : -1;
    if (threadIdx.x == 0) {
      if (!(total > 0.0)) atomicCAS(status, 0, FTB_ERR_INDEX);
      counts_out[b] = n + 1;
    }
  }
  if constexpr (C > 1) cluster_sync_all();  // nobody leaves while its sum may be read
}

template <int C, int kThreads>
cudaError_t launch(const Drafts& a, int B, long long* tokens, int* counts_out, int* status, cudaStream_t stream) {
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
  return cudaLaunchKernelEx(&cfg, verify_drafts_kernel<C, kThreads>, a, tokens, counts_out, status);
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" int ftb_verify_drafts(const float* probs, long long p_seq, long long p_row, const float* draft_probs, long long q_seq,
                                 long long q_row, const long long* drafts, const float* u, const int* counts, long long* tokens,
                                 int* counts_out, int B, int K, int V, void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || K < 0 || V <= 0 || V > 1 << 30) return FTB_ERR_ARG;
  if (B > 0 && (!probs || (!drafts && K > 0) || !u || !tokens || !counts_out)) return FTB_ERR_ARG;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  if (B == 0) return FTB_OK;
  const int rc = check_device_sm100();
  if (rc) return rc;
  const Drafts a{probs, draft_probs, drafts, u, counts, p_seq, p_row, q_seq, q_row, K, V};
  if (B > 0x7fffffff / 8) return FTB_ERR_ARG;
  int* st = static_cast<int*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Clusters where a row has more than a few numbers a thread; small CTAs where there are so many that their beginnings, which
  // wait for single numbers, have to lie under the reading of others.
  const cudaError_t err = V <= 4096                              ? launch<1, 512>(a, B, tokens, counts_out, st, s)
                          : B <= current_sm_count() / 8 ? launch<8, 512>(a, B, tokens, counts_out, st, s)
                                                                 : launch<8, 256>(a, B, tokens, counts_out, st, s);
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}
