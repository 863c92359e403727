// Attention over a paged cache: the arguments, and a row on its own.
#pragma once
#include <cfloat>

#include "paged.cuh"

namespace ftb {

struct PagedAttn {
  PagedBatch batch;
  const void* q;
  void* o;
  long long q_row, q_head;  // distances in numbers
  const unsigned char *k, *v, *k_exp, *v_exp;
  int T, kv_heads, group, window;  // window 0: none
  float scale_log2;
  int* status;
};

// Row `key` of kv head `h` of sequence b in the cache; a page that the table does not have reads as page 0.
__device__ __forceinline__ long long cache_row(const PagedAttn& a, int b, int h, long long key) {
  const int page = max(0, page_of(a.batch, b, key, a.status));
  return ((static_cast<long long>(page) * a.kv_heads + h) << a.batch.page_shift) + (key & ((1 << a.batch.page_shift) - 1));
}

// Whether a row at position pos of a tile that multiplies keys lo .. hi - 1 has some of them with weight 0 that it does not see: what
// they hold could have made its result a NaN.
__device__ __forceinline__ bool hides(const PagedAttn& a, long long pos, int lo, int hi) {
  return pos + 1 < hi || (a.window > 0 && pos + 1 - a.window > lo);
}

// The output of one (token, head) by one warp, key by key: nothing of a key that the token does not see is touched, not
// even with a weight of 0, which an infinity or a NaN there would make a NaN.  q: D floats of shared memory of the warp's.
template <typename T, bool k8, int D>
__device__ __noinline__ void attend_row(const PagedAttn& a, int b, int t, int head, long long pos, float* q, int lane) {
  constexpr int kPer = D / 32;  // numbers of the output a lane
  const int h = head / a.group;
  const T* src = static_cast<const T*>(a.q) + t * a.q_row + head * a.q_head;
  __syncwarp();
  for (int i = lane; i < D / 2; i += 32) {
    const float2 f = unpack2<T>(reinterpret_cast<const uint32_t*>(src)[i]);
    q[2 * i] = f.x * a.scale_log2;
    q[2 * i + 1] = f.y * a.scale_log2;
  }
  __syncwarp();
  const long long end = pos + 1, begin = a.window > 0 ? max(0ll, end - a.window) : 0;
  float m = -FLT_MAX, l = 0.f, acc[kPer] = {};
  for (long long j0 = begin; j0 < end; j0 += 32) {
    const long long j = j0 + lane;
    float s = -INFINITY;
    long long row = 0;
    if (j < end) {
      row = cache_row(a, b, h, j);
      s = 0.f;
      if constexpr (k8) {
        const uint4* k = reinterpret_cast<const uint4*>(a.k + row * D);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const uint4 x = k[c];
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 f = unpack2<__half>(e4m3x2_to_f16x2((w[i >> 1] >> ((i & 1) * 16)) & 0xffffu));
            s = fmaf(q[c * 16 + 2 * i], f.x, s);
            s = fmaf(q[c * 16 + 2 * i + 1], f.y, s);
          }
        }
        s *= exponent_scale(a.k_exp[row]);
      } else {
        const uint4* k = reinterpret_cast<const uint4*>(a.k + row * (2 * D));
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint4 x = k[c];
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            s = fmaf(q[c * 8 + 2 * i], f.x, s);
            s = fmaf(q[c * 8 + 2 * i + 1], f.y, s);
          }
        }
      }
    }
    float mx = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float m_new = fmaxf(m, mx), keep = exp2_fast(m - m_new);
    const float p = exp2_fast(s - m_new);
    float sum = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * keep + sum;
    m = m_new;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] *= keep;
    const int n = static_cast<int>(min(32ll, end - j0));
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(0xffffffffu, p, i);
      const long long r = __shfl_sync(0xffffffffu, row, i);
      float f[kPer];
      if constexpr (k8) {
        const unsigned char* v = a.v + r * D + lane * kPer;
        const float e = exponent_scale(a.v_exp[r]);
#pragma unroll
        for (int c = 0; c < kPer / 2; ++c) {
          const float2 g = unpack2<__half>(e4m3x2_to_f16x2(reinterpret_cast<const unsigned short*>(v)[c]));
          f[2 * c] = g.x * e;
          f[2 * c + 1] = g.y * e;
        }
      } else {
        const unsigned char* v = a.v + r * (2 * D) + lane * (2 * kPer);
#pragma unroll
        for (int c = 0; c < kPer / 2; ++c) {
          const float2 g = unpack2<T>(reinterpret_cast<const uint32_t*>(v)[c]);
          f[2 * c] = g.x;
          f[2 * c + 1] = g.y;
        }
      }
#pragma unroll
      for (int c = 0; c < kPer; ++c) acc[c] = fmaf(w, f[c], acc[c]);
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(a.o) + (static_cast<long long>(t) * a.kv_heads * a.group + head) * D) + lane * (kPer / 2);
#pragma unroll
  for (int c = 0; c < kPer / 2; ++c) out[c] = Fmt<T>::pack2(acc[2 * c] * inv, acc[2 * c + 1] * inv);
}

}  // namespace ftb
