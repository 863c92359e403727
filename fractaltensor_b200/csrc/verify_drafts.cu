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
// Bound by the bytes of those rows: 100 sequences of 5 drafts over 130 001 words 30.3 us, 3.4 TB/s (one: 7.5 us, trips to memory one
// behind the other: the drafts' probabilities, the row, the stretch).  A cluster of CTAs takes a sequence, every warp a stretch of the row: one pass for the
// stretches' sums, which the CTAs hand each other through distributed shared memory, and a second look at the one stretch (a 64th of
// the row or less) in which the limit is passed.  Every CTA finds n on its own, which saves a step of waiting.
#include <climits>

#include "../../include/ftb200.h"
#include "ptx.cuh"
#include "tmap.h"

namespace ftb {
namespace {

constexpr int kUnroll = 8;

struct Drafts {
  const float* p;
  const float* q;  // or nullptr
  const long long* drafts;
  const float* u;
  const int* counts;  // or nullptr: K each
  long long p_seq, p_row, q_seq, q_row;
  int K, V;
};

// What is not positive and finite counts as 0, in the target's rows and in the draft's.
__device__ __forceinline__ double probability(float x) {
  x = fmaxf(x, 0.f);  // (0 of a NaN)
  return static_cast<double>(x < __int_as_float(0x7f800000) ? x : 0.f);
}

__device__ __forceinline__ double weight_of(float p, float q, int j, int without) {
  const double w = static_cast<double>(p) - probability(q);  // (nothing is left of a p that is not positive)
  return w > 0.0 && p < __int_as_float(0x7f800000) && j != without ? w : 0.0;
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
  double x;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(x) : "r"(addr) : "memory");
  return x;
}

// C: CTAs of a cluster, 1 or 8.
template <int C, int kThreads>
__global__ void __launch_bounds__(kThreads, 1536 / kThreads)
verify_drafts_kernel(Drafts a, long long* __restrict__ tokens, int* __restrict__ counts_out, int* __restrict__ status) {
  constexpr int kWarps = kThreads / 32;
  __shared__ double sums[kWarps], totals[2];  // of the warps; of this CTA (in the two tries)
  __shared__ double s_total[C];
  __shared__ int s_n, s_found, s_heavy;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
  const double share = u[K];
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
  const float* pr = p + n * a.p_row;
  const float* qr = q != nullptr && n < mine ? q + n * a.q_row : nullptr;
  int without = q == nullptr && n < mine && x[n] >= 0 && x[n] < V ? static_cast<int>(x[n]) : -1;
  // a warp's stretch of the row: whole groups of 32
  const int stretch = ((V + C * kThreads - 1) / (C * kThreads)) * 32;
  const int from = static_cast<int>(min(static_cast<long long>(V), static_cast<long long>(rank * kWarps + warp) * stretch)), to = min(V, from + stretch);
  double total = 0.0, before = 0.0;  // of the row; of the CTAs in front of this one
  for (int tries = 0; tries < 2; ++tries) {  // where p and q are the same, nothing is left of the difference: p itself
    double s = 0.0;
    for (int j = from; j < to; j += 32 * kUnroll) {
      float pv[kUnroll], qv[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int at = j + k * 32 + lane;
        pv[k] = at < to ? pr[at] : 0.f;
        qv[k] = qr != nullptr && at < to ? qr[at] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) s += weight_of(pv[k], qv[k], j + k * 32 + lane, without);
    }
    s = warp_sum(s);
    if (lane == 0) sums[warp] = s;
    __syncthreads();
    double cta = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) cta += sums[w];
    if constexpr (C == 1) {
      total = cta;
      __syncthreads();
    } else {
      if (threadIdx.x == 0) totals[tries] = cta;
      cluster_sync_all();
      if (threadIdx.x < C) s_total[threadIdx.x] = ld_cluster_f64(map_to_cta(smem_u32(&totals[tries]), threadIdx.x));
      __syncthreads();
      total = before = 0.0;
#pragma unroll
      for (int r = 0; r < C; ++r) {
        if (r < rank) before += s_total[r];
        total += s_total[r];
      }
    }
    if (total > 0.0) break;
    qr = nullptr;
    without = -1;
  }
  // The stretch in which the limit is passed: sums[] are this CTA's still.  (u of 1 or above, or sums that round down: the last
  // stretch that weighs anything.)
  const double limit = share * total;
  // Which CTA has it follows from the CTAs' sums alone, the same in all of them.
  const bool passed = total > limit;
  bool past = false, own = C == 1;
  if constexpr (C > 1) {
    double at = 0.0;
    int weighs = -1;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      at += s_total[r];
      if (passed && !past && at > limit) {
        past = true;
        own = r == rank;
      }
      if (s_total[r] > 0.0) weighs = r;
    }
    if (!passed) own = weighs == rank;
  }
  int first = -1, last = -1;
  double in_front = before, begin = before;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (first < 0 && begin + sums[w] > limit) {
      first = w;
      in_front = begin;
    }
    begin += sums[w];
    if (sums[w] > 0.0) last = w;
  }
  const bool heaviest = !passed || first < 0;  // (sums that round differently: the last one too)
  if (heaviest) first = last;
  // That stretch again, by all warps of the CTA, kUnroll numbers side by side a lane: one scan over the warps' sums for
  // kThreads * kUnroll of them.
  if (own && total > 0.0) {  // of all CTAs, one
    const int begin_at = static_cast<int>(min(static_cast<long long>(V), static_cast<long long>(rank * kWarps + first) * stretch)), end_at = min(V, begin_at + stretch);
    int found = INT_MAX, heavy = -1;
    double run = in_front;
    for (int j0 = begin_at; j0 < end_at && found == INT_MAX; j0 += kThreads * kUnroll) {
      const int j = j0 + static_cast<int>(threadIdx.x) * kUnroll;
      double w[kUnroll], sum = 0.0;
      float pv[kUnroll], qv[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        pv[k] = j + k < end_at ? pr[j + k] : 0.f;
        qv[k] = qr != nullptr && j + k < end_at ? qr[j + k] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        w[k] = weight_of(pv[k], qv[k], j + k, without);
        sum += w[k];
      }
      double ends = sum;  // sum of the warp's lanes up to this one
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, ends, o);
        if (lane >= o) ends += y;
      }
      const double begins = __shfl_up_sync(0xffffffffu, ends, 1);
      __syncthreads();  // (sums, s_found and s_heavy have been read)
      if (lane == 31) sums[warp] = ends;
      if (threadIdx.x == 0) {
        s_found = INT_MAX;
        s_heavy = -1;
      }
      __syncthreads();
      double upto = run + (lane > 0 ? begins : 0.0);
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        if (v < warp) upto += sums[v];
        run += sums[v];
      }
      int here_found = INT_MAX, here_heavy = -1;
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        upto += w[k];
        if (w[k] > 0.0) {
          if (here_found == INT_MAX && !heaviest && upto > limit) here_found = j + k;
          here_heavy = j + k;
        }
      }
      here_found = __reduce_min_sync(0xffffffffu, here_found);
      here_heavy = __reduce_max_sync(0xffffffffu, here_heavy);
      if (lane == 0) {
        if (here_found != INT_MAX) atomicMin(&s_found, here_found);
        if (here_heavy >= 0) atomicMax(&s_heavy, here_heavy);
      }
      __syncthreads();
      found = s_found;
      if (s_heavy >= 0) heavy = s_heavy;
    }
    if (threadIdx.x == 0) tokens[static_cast<long long>(b) * (K + 1) + n] = found != INT_MAX ? found : heavy;
  }
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
