// Keys and values of new tokens into a paged cache, and back out of it.
//
// A warp takes one token: its kv_heads rows of keys and of values, 16 bytes of a 16-bit row a lane, several pieces in flight; into
// 8-bit rows 16 numbers a lane (whole sectors to write), out of them 8 (whole sectors again).  Rows that are written do not
// wait for their place: a token's sequence, position and page are found while they are on their way.
// 8-bit caches: a row's largest magnitude is found among the lanes that hold it, on the bit patterns; its exponent
// is the smallest e with max <= 448 * 2^(e - 127), taken from the bits of max as fp32: 448 = 1.75 * 2^8.
// Bound by memory: kv_heads * d * 2 * (2 + size in the cache) bytes a token.  8 kv heads of 128: 6 chunks of 500 to 2047 tokens into 8-bit
// pages of 32 and out again 17.7 us, 3.9 TB/s (what it can do without: 10.4); 37 sequences of up to 3000 tokens of 4 kv heads out of 8-bit
// pages 41.6 us, 4.8 TB/s (30.3); a token of each of 24 sequences 3.4 us, a launch.  Measured and not kept: two tokens a reading warp
// (48.6 us for the sequences), 16 numbers a reading lane (50).
#include <type_traits>

#include "../../include/ftb200.h"
#include "paged.cuh"
#include "tmap.h"

namespace ftb {
namespace {

constexpr int kThreads = 128;

struct Rows {
  const void* k;
  const void* v;
  long long k_row, k_head, v_row, v_head;  // distances in numbers
};
struct Cache {
  unsigned char *k, *v, *k_exp, *v_exp;
};

// 16 bytes of 16-bit numbers: the largest magnitude's bits in both halves' maxima.
__device__ __forceinline__ uint32_t largest(const uint4& x) {
  constexpr uint32_t kAbs = 0x7fff7fffu;
  const uint32_t m = __vmaxu2(__vmaxu2(x.x & kAbs, x.y & kAbs), __vmaxu2(x.z & kAbs, x.w & kAbs));
  return max(m & 0xffffu, m >> 16);
}

template <typename T>
__device__ __forceinline__ int row_exponent(uint32_t largest_bits) {
  const uint32_t bits = __float_as_uint(unpack2<T>(largest_bits).x);
  const int E = static_cast<int>(bits >> 23);
  if (E == 255) return 255;
  return max(1, E - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0));
}

// Eight numbers as codes.
template <typename T>
__device__ __forceinline__ uint2 to_codes(const uint4& x, int e) {
  if (e == 255) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
  const float inverse = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);  // 2^(127 - e); e <= 247
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = unpack2<T>(w[i]);
    f.x *= inverse;
    f.y *= inverse;
    c[i] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// A lane's piece of a row.
template <int kNumbers_, int D>
struct Pieces {
  static constexpr int kNumbers = kNumbers_, kOfRow = D / kNumbers, kAtOnce = 64 / kNumbers;
};

template <typename T, bool k8, int D>
__global__ void __launch_bounds__(kThreads)
paged_write_kernel(Rows in, Cache cache, PagedBatch batch, int T_rows, int kv_heads, int* __restrict__ status) {
  using P = Pieces<k8 ? 16 : 8, D>;
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  grid_launch_dependents();
  grid_dependency_wait();
  if (t >= T_rows) return;
  const int half = kv_heads * P::kOfRow, pieces = 2 * half;  // keys, then values
  long long row0 = -1;  // the row of head 0 in the cache
  for (int p0 = 0; p0 < pieces; p0 += 32 * P::kAtOnce) {
    uint4 x[P::kAtOnce][k8 ? 2 : 1];
#pragma unroll
    for (int i = 0; i < P::kAtOnce; ++i) {
      const int p = p0 + i * 32 + lane;
      const bool is_v = p >= half;
      const int q = is_v ? p - half : p, head = q / P::kOfRow, c = q % P::kOfRow;
      const T* src = is_v ? static_cast<const T*>(in.v) + t * in.v_row + head * in.v_head
                          : static_cast<const T*>(in.k) + t * in.k_row + head * in.k_head;
#pragma unroll
      for (int k = 0; k < (k8 ? 2 : 1); ++k) {
        x[i][k] = make_uint4(0u, 0u, 0u, 0u);
        if (p < pieces) x[i][k] = __ldcs(reinterpret_cast<const uint4*>(src + c * P::kNumbers) + k);
      }
    }
    if (p0 == 0) {
      const RowPlace at = place_of_row(batch, t, lane);
      if (at.b >= batch.B || at.pos < 0) return;
      const int page = page_of(batch, at.b, at.pos, status);
      if (page < 0) return;
      row0 = ((static_cast<long long>(page) * kv_heads) << batch.page_shift) + (at.pos & ((1 << batch.page_shift) - 1));
    }
#pragma unroll
    for (int i = 0; i < P::kAtOnce; ++i) {
      const int p = p0 + i * 32 + lane;
      const bool is_v = p >= half;
      const int q = is_v ? p - half : p, head = q / P::kOfRow, c = q % P::kOfRow;
      const long long row = row0 + (static_cast<long long>(head) << batch.page_shift);
      unsigned char* dst = is_v ? cache.v : cache.k;
      if constexpr (k8) {
        uint32_t m = max(largest(x[i][0]), largest(x[i][1]));
#pragma unroll
        for (int o = P::kOfRow / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int e = row_exponent<T>(m);
        if (p < pieces) {
          const uint2 lower = to_codes<T>(x[i][0], e), upper = to_codes<T>(x[i][1], e);
          *reinterpret_cast<uint4*>(dst + row * D + c * 16) = make_uint4(lower.x, lower.y, upper.x, upper.y);
          if (c == 0) (is_v ? cache.v_exp : cache.k_exp)[row] = static_cast<unsigned char>(e);
        }
      } else if (p < pieces) {
        *reinterpret_cast<uint4*>(dst + row * (2 * D) + c * 16) = x[i][0];
      }
    }
  }
}

// Piece `at` of the output: eight numbers.
template <typename T>
__device__ __forceinline__ void put8(T* out, long long at, const float* f) {
  __stcs(reinterpret_cast<uint4*>(out) + at, make_uint4(Fmt<T>::pack2(f[0], f[1]), Fmt<T>::pack2(f[2], f[3]),
                                                        Fmt<T>::pack2(f[4], f[5]), Fmt<T>::pack2(f[6], f[7])));
}
template <>
__device__ __forceinline__ void put8<float>(float* out, long long at, const float* f) {
  __stcs(reinterpret_cast<float4*>(out) + 2 * at, make_float4(f[0], f[1], f[2], f[3]));
  __stcs(reinterpret_cast<float4*>(out) + 2 * at + 1, make_float4(f[4], f[5], f[6], f[7]));
}

template <typename T, bool k8, int D>
__global__ void __launch_bounds__(kThreads)
paged_read_kernel(Cache cache, PagedBatch batch, T* __restrict__ k_out, T* __restrict__ v_out, int T_rows, int kv_heads,
                  int* __restrict__ status) {
  using P = Pieces<8, D>;
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  grid_launch_dependents();
  grid_dependency_wait();
  if (t >= T_rows) return;
  const RowPlace at = place_of_row(batch, t, lane);
  if (at.b >= batch.B) return;
  const int page = at.pos >= 0 ? page_of(batch, at.b, at.pos, status) : -1;
  const long long row0 = ((static_cast<long long>(page) * kv_heads) << batch.page_shift) + (at.pos & ((1 << batch.page_shift) - 1));
  const int half = kv_heads * P::kOfRow, pieces = 2 * half;
  for (int p0 = 0; p0 < pieces; p0 += 32 * P::kAtOnce) {
    using Piece = typename std::conditional<k8, uint2, uint4>::type;
    Piece x[P::kAtOnce];
    int e[P::kAtOnce];
#pragma unroll
    for (int i = 0; i < P::kAtOnce; ++i) {
      const int p = p0 + i * 32 + lane;
      x[i] = Piece{};
      e[i] = 0;
      if (p < pieces && page >= 0) {
        const bool is_v = p >= half;
        const int q = is_v ? p - half : p, head = q / P::kOfRow, c = q % P::kOfRow;
        const long long row = row0 + (static_cast<long long>(head) << batch.page_shift);
        x[i] = __ldcs(reinterpret_cast<const Piece*>((is_v ? cache.v : cache.k) + row * (k8 ? D : 2 * D)) + c);
        if constexpr (k8) e[i] = (is_v ? cache.v_exp : cache.k_exp)[row];
      }
    }
#pragma unroll
    for (int i = 0; i < P::kAtOnce; ++i) {
      const int p = p0 + i * 32 + lane;
      if (p < pieces) {
        const bool is_v = p >= half;
        const long long to = static_cast<long long>(t) * half + (is_v ? p - half : p);
        T* out = is_v ? v_out : k_out;
        if constexpr (k8) {
          const float scale = exponent_scale(e[i]);
          float f[8];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t lower, upper;
            e4m3x4_to_f16x2(j == 0 ? x[i].x : x[i].y, lower, upper);
            const float2 l = unpack2<__half>(lower), u = unpack2<__half>(upper);
            f[4 * j] = l.x * scale;
            f[4 * j + 1] = l.y * scale;
            f[4 * j + 2] = u.x * scale;
            f[4 * j + 3] = u.y * scale;
          }
          put8(out, to, f);
        } else {
          __stcs(reinterpret_cast<uint4*>(out) + to, x[i]);
        }
      }
    }
  }
}

// What the entry points over a cache share: 0, or the reason for a refusal.
struct Sizes {
  int T, B, W, pages, kv_heads, page_size, d;
};
int check_sizes(const Sizes& n, const void* k, const void* v, const void* k_exp, const void* v_exp, const int* table,
                const int* lens, const int* starts) {
  if (!k || !v || !table || !lens || !starts || (k_exp == nullptr) != (v_exp == nullptr)) return FTB_ERR_ARG;
  if (n.T < 0 || n.B <= 0 || n.W <= 0 || n.pages <= 0 || n.kv_heads <= 0 || n.kv_heads > 65536) return FTB_ERR_ARG;
  if (n.page_size != 16 && n.page_size != 32 && n.page_size != 64 && n.page_size != 128) return FTB_ERR_ARG;
  if (n.d != 64 && n.d != 128) return FTB_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_exp) | reinterpret_cast<uintptr_t>(v_exp)) & 15) != 0)
    return FTB_ERR_ALIGN;
  return FTB_OK;
}
PagedBatch batch_of(const Sizes& n, const int* table, const int* lens, const int* starts) {
  return {table, lens, starts, n.B, n.W, n.pages, 31 - __builtin_clz(static_cast<unsigned>(n.page_size))};
}

template <typename T, bool k8, int D>
cudaError_t launch_write(const Rows& in, const Cache& cache, const PagedBatch& batch, int T_rows, int kv_heads, int* status,
                         cudaStream_t stream) {
  return launch_light(paged_write_kernel<T, k8, D>, dim3((T_rows + kThreads / 32 - 1) / (kThreads / 32)), dim3(kThreads), 0, stream,
                      in, cache, batch, T_rows, kv_heads, status);
}
template <typename T>
cudaError_t launch_write(bool k8, int d, const Rows& in, const Cache& cache, const PagedBatch& batch, int T_rows, int kv_heads,
                         int* status, cudaStream_t stream) {
  if (d == 128)
    return k8 ? launch_write<T, true, 128>(in, cache, batch, T_rows, kv_heads, status, stream)
              : launch_write<T, false, 128>(in, cache, batch, T_rows, kv_heads, status, stream);
  return k8 ? launch_write<T, true, 64>(in, cache, batch, T_rows, kv_heads, status, stream)
            : launch_write<T, false, 64>(in, cache, batch, T_rows, kv_heads, status, stream);
}
template <typename T, bool k8>
cudaError_t launch_read(int d, const Cache& cache, const PagedBatch& batch, void* k_out, void* v_out, int T_rows, int kv_heads,
                        int* status, cudaStream_t stream) {
  return launch_light(d == 128 ? paged_read_kernel<T, k8, 128> : paged_read_kernel<T, k8, 64>,
                      dim3((T_rows + kThreads / 32 - 1) / (kThreads / 32)), dim3(kThreads), 0, stream, cache, batch,
                      static_cast<T*>(k_out), static_cast<T*>(v_out), T_rows, kv_heads, status);
}

int launched(cudaError_t err) {
  count_launch();
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? FTB_OK : FTB_ERR_LAUNCH;
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" int ftb_paged_cache_write(const void* k, const void* v, long long k_row, long long k_head, long long v_row,
                                     long long v_head, void* k_cache, void* v_cache, unsigned char* k_exp,
                                     unsigned char* v_exp, const int* table, const int* lens, const int* starts, int T, int B,
                                     int W, int pages, int kv_heads, int page_size, int d, int dtype, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const Sizes n{T, B, W, pages, kv_heads, page_size, d};
  int rc = check_sizes(n, k_cache, v_cache, k_exp, v_exp, table, lens, starts);
  if (rc) return rc;
  if ((T > 0 && (!k || !v)) || (dtype != FTB_F16 && dtype != FTB_BF16)) return FTB_ERR_ARG;
  if (((k_row | k_head | v_row | v_head) & 7) != 0 || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0)
    return FTB_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  if (T == 0) return FTB_OK;
  if ((rc = check_device_sm100())) return rc;
  const Rows in{k, v, k_row, k_head, v_row, v_head};
  const Cache cache{static_cast<unsigned char*>(k_cache), static_cast<unsigned char*>(v_cache), k_exp, v_exp};
  const PagedBatch batch = batch_of(n, table, lens, starts);
  int* status = static_cast<int*>(workspace);
  const bool k8 = k_exp != nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return launched(dtype == FTB_F16 ? launch_write<__half>(k8, d, in, cache, batch, T, kv_heads, status, s)
                                   : launch_write<__nv_bfloat16>(k8, d, in, cache, batch, T, kv_heads, status, s));
}

extern "C" int ftb_paged_cache_read(const void* k_cache, const void* v_cache, const unsigned char* k_exp,
                                    const unsigned char* v_exp, const int* table, const int* lens, const int* starts,
                                    void* k_out, void* v_out, int T, int B, int W, int pages, int kv_heads, int page_size,
                                    int d, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const Sizes n{T, B, W, pages, kv_heads, page_size, d};
  int rc = check_sizes(n, k_cache, v_cache, k_exp, v_exp, table, lens, starts);
  if (rc) return rc;
  const bool k8 = k_exp != nullptr;
  if ((T > 0 && (!k_out || !v_out)) || (dtype != FTB_F16 && dtype != FTB_BF16 && !(k8 && dtype == FTB_F32))) return FTB_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) != 0) return FTB_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < ftb_workspace_bytes()) return FTB_ERR_WORKSPACE;
  if (T == 0) return FTB_OK;
  const size_t numbers = static_cast<size_t>(pages) * kv_heads * page_size * d, cache_bytes = k8 ? numbers : 2 * numbers;
  const size_t out_bytes = static_cast<size_t>(T) * kv_heads * d * dtype_size(dtype), exp_bytes = k8 ? numbers / d : 0;
  if (overlap(k_out, out_bytes, v_out, out_bytes)) return FTB_ERR_ARG;
  for (const void* out : {k_out, v_out})
    if (overlap(out, out_bytes, k_cache, cache_bytes) || overlap(out, out_bytes, v_cache, cache_bytes) ||
        overlap(out, out_bytes, k_exp, exp_bytes) || overlap(out, out_bytes, v_exp, exp_bytes))
      return FTB_ERR_ARG;
  if ((rc = check_device_sm100())) return rc;
  const Cache cache{const_cast<unsigned char*>(static_cast<const unsigned char*>(k_cache)),
                    const_cast<unsigned char*>(static_cast<const unsigned char*>(v_cache)),
                    const_cast<unsigned char*>(k_exp), const_cast<unsigned char*>(v_exp)};
  const PagedBatch batch = batch_of(n, table, lens, starts);
  int* status = static_cast<int*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!k8)  // the rows as they are: one 16-bit type is as good as the other
    return launched(launch_read<__half, false>(d, cache, batch, k_out, v_out, T, kv_heads, status, s));
  return launched(dtype == FTB_F32   ? launch_read<float, true>(d, cache, batch, k_out, v_out, T, kv_heads, status, s)
                  : dtype == FTB_F16 ? launch_read<__half, true>(d, cache, batch, k_out, v_out, T, kv_heads, status, s)
                                     : launch_read<__nv_bfloat16, true>(d, cache, batch, k_out, v_out, T, kv_heads, status, s));
}
