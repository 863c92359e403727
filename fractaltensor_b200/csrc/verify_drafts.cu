// Verification of drafted tokens against the target's probabilities, from random numbers that the caller gives.
//
// Sequence b has K drafted tokens x_0 .. x_{K-1}, drawn from the draft's probabilities q_i, and the target's
// probabilities p_0 .. p_K.  Draft i is taken if u_i * q_i(x_i) < p_i(x_i) (probability min(1, p / q)), the first that is
// not ends the run at n; token n is drawn from w = max(p_n - q_n, 0), or from p_K behind K taken drafts: the first j
// with w_0 + .. + w_j > u_K * sum(w).  Drafts without probabilities were certain: q_i is 1 at x_i.
//
// Only one row of p (and of q) a sequence is read whole.  Sums are kept in 64 bits: the chosen index follows from a
// comparison with a partial sum of up to V numbers, and in 32 bits the order of summation would decide it.
#include "../../include/ftb200.h"
#include "ptx.cuh"
#include "tmap.h"

namespace ftb {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;

struct Drafts {
  const float* p;
  const float* q;  // or nullptr
  const long long* drafts;
  const float* u;
  const int* counts;  // or nullptr: K each
  long long p_seq, p_row, q_seq, q_row;
  int K, V;
};

__device__ __forceinline__ double weight(const float* p, const float* q, int j, int without) {
  const float x = p[j];
  double w = x;
  if (q != nullptr) w -= static_cast<double>(q[j]);
  return w > 0.0 && x < __int_as_float(0x7f800000) && j != without ? w : 0.0;
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__global__ void __launch_bounds__(kThreads)
verify_drafts_kernel(Drafts a, long long* __restrict__ tokens, int* __restrict__ counts_out, int* __restrict__ status) {
  __shared__ double sums[kWarps];
  __shared__ int s_n, s_found;
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  const int K = a.K, V = a.V;
  const int mine = a.counts != nullptr ? min(max(a.counts[b], 0), K) : K;
  const long long* x = a.drafts + static_cast<long long>(b) * K;
  const float* u = a.u + static_cast<long long>(b) * (K + 1);
  const float* p = a.p + b * a.p_seq;
  const float* q = a.q != nullptr ? a.q + b * a.q_seq : nullptr;
  if (threadIdx.x == 0) {
    s_n = mine;
    s_found = V;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < mine; i += kThreads) {
    const long long id = x[i];
    bool taken = false;
    if (id >= 0 && id < V) {
      const double qx = q != nullptr ? static_cast<double>(q[i * a.q_row + id]) : 1.0;
      taken = static_cast<double>(u[i]) * qx < static_cast<double>(p[i * a.p_row + id]);
    } else {
      atomicCAS(status, 0, FTB_ERR_INDEX);
    }
    if (!taken) atomicMin(&s_n, i);
  }
  __syncthreads();
  const int n = s_n;
  const float* pr = p + n * a.p_row;
  const float* qr = q != nullptr && n < mine ? q + n * a.q_row : nullptr;
  int without = q == nullptr && n < mine && x[n] >= 0 && x[n] < V ? static_cast<int>(x[n]) : -1;
  // a warp's part of the row: whole groups of 32
  const int part = ((V + kThreads - 1) / kThreads) * 32, from = min(V, warp * part), to = min(V, from + part);
  double total = 0.0;
  for (int tries = 0; tries < 2; ++tries) {  // where p and q are the same, nothing is left of the difference: p itself
    double s = 0.0;
    for (int j = from + lane; j < to; j += 32) s += weight(pr, qr, j, without);
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) sums[warp] = s;
    __syncthreads();
    total = 0.0;
    for (int w = 0; w < kWarps; ++w) total += sums[w];
    if (total > 0.0) break;
    qr = nullptr;
    without = -1;
  }
  const double limit = static_cast<double>(u[K]) * total;
  double before = 0.0;
  int last = -1, first = kWarps;  // the last part that weighs anything, the first whose end is above the limit
  double at = 0.0;
  for (int w = 0; w < kWarps; ++w) {
    if (first == kWarps && at + sums[w] > limit) {
      first = w;
      before = at;
    }
    at += sums[w];
    if (sums[w] > 0.0) last = w;
  }
  if (first == kWarps && last >= 0) {  // u of 1 or above, or sums that round down: the last token that weighs anything
    first = last;
    before = -1e300;
  }
  if (warp == first) {
    int found = -1, heavy = -1;
    double run = before;
    for (int j0 = from; j0 < to && found < 0; j0 += 32) {
      const int j = j0 + lane;
      const double w = j < to ? weight(pr, qr, j, without) : 0.0;
      double s = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
      }
      const unsigned above = __ballot_sync(0xffffffffu, w > 0.0 && run + s > limit), some = __ballot_sync(0xffffffffu, w > 0.0);
      if (above != 0) found = j0 + __ffs(above) - 1;
      if (some != 0) heavy = j0 + 31 - __clz(some);
      run += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) s_found = found >= 0 ? found : heavy;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (!(total > 0.0)) atomicCAS(status, 0, FTB_ERR_INDEX);
    counts_out[b] = n + 1;
  }
  for (int i = threadIdx.x; i <= K; i += kThreads)
    tokens[static_cast<long long>(b) * (K + 1) + i] = i < n ? x[i] : i > n || !(total > 0.0) ? -1 : s_found;
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" int ftb_verify_drafts(const float* probs, long long p_seq, long long p_row, const float* draft_probs, long long q_seq,
                                 long long q_row, const long long* drafts, const float* u, const int* counts, long long* tokens,
                                 int* counts_out, int B, int K, int V, void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || K < 0 || V <= 0) return FTB_ERR_ARG;
  if (B > 0 && (!probs || (!drafts && K > 0) || !u || !tokens || !counts_out)) return FTB_ERR_ARG;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  if (B == 0) return FTB_OK;
  const int rc = check_device_sm100();
  if (rc) return rc;
  const Drafts a{probs, draft_probs, drafts, u, counts, p_seq, p_row, q_seq, q_row, K, V};
  const cudaError_t err = launch_light(verify_drafts_kernel, dim3(B), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), a,
                                       tokens, counts_out, static_cast<int*>(workspace));
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}
