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
  int least_rows, most_rows;       // sequences with so many rows (token, head of a group) of a kv head are this launch's
  float scale_log2;
  int* status;
  uint32_t* odd;                   // [T, heads]: not 0 where a row of the output has to be computed again, key by key
};

// 8 bits: values of 2^-30 to 2^30 times a code are ordinary, and maxima of scores with and without the values' exponents that are up to 2^40
// apart: weights, which end at 2^-126, then reach down to 2^-48 of the largest, and the terms of the sum that divides up to 2^38.
constexpr float kNear = 30.f;
constexpr float kNearTops = 40.f;

// Whether a row at position pos of a tile that multiplies keys lo .. hi - 1 has some of them with weight 0 that it does not see: what
// they hold could have made its result a NaN.
__device__ __forceinline__ bool hides(const PagedAttn& a, long long pos, int lo, int hi) {
  return pos + 1 < hi || (a.window > 0 && pos + 1 - a.window > lo);
}

// The output of one (token, head) by one warp, key by key: nothing of a key that the token does not see has a part
// in it, not even with a weight of 0, which an infinity or a NaN there would make a NaN.  A lane holds D / 32 numbers of a row; eight
// keys at a time, which are of one page and on their way together.  For rows that the kernels' products have made a NaN through such keys.
// It is for what should not happen: a row of 65 536 keys takes 9 ms (36 with a trip to memory for every key).  2048 tokens of 32 heads behind
// 14 336 keys, 0.5 ms, take 36 ms with a NaN at the last position, which the last 64 tokens do not see, and 86 with one in their middle.
template <typename T, bool k8, int D>
__device__ __noinline__ void attend_row(const PagedAttn& a, int b, int t, int head, long long pos, int lane) {
  constexpr int kPer = D / 32, kBatch = 8;
  const int h = head / a.group;
  const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + t * a.q_row + head * a.q_head) + lane * (kPer / 2);
  float q[kPer], acc[kPer] = {};
#pragma unroll
  for (int c = 0; c < kPer / 2; ++c) {
    const float2 f = unpack2<T>(src[c]);
    q[2 * c] = f.x;
    q[2 * c + 1] = f.y;
  }
  // this lane's numbers of a row of the cache; 8 bits: times 2^by
  auto numbers = [&](const unsigned char* cache, int by, long long row, float (&f)[kPer]) {
    if constexpr (k8) {
      const float e = exponent_scale(127 + by);
#pragma unroll
      for (int c = 0; c < kPer / 2; ++c) {
        const float2 g = unpack2<__half>(e4m3x2_to_f16x2(reinterpret_cast<const unsigned short*>(cache + row * D)[lane * (kPer / 2) + c]));
        f[2 * c] = g.x * e;
        f[2 * c + 1] = g.y * e;
      }
    } else {
#pragma unroll
      for (int c = 0; c < kPer / 2; ++c) {
        const float2 g = unpack2<T>(reinterpret_cast<const uint32_t*>(cache + row * (2 * D))[lane * (kPer / 2) + c]);
        f[2 * c] = g.x;
        f[2 * c + 1] = g.y;
      }
    }
  };
  const long long end = min(pos + 1, static_cast<long long>(a.batch.W) << a.batch.page_shift);
  const long long begin = a.window > 0 ? max(0ll, pos + 1 - a.window) : 0;
  float m = -FLT_MAX, l = 0.f;
  for (long long j0 = begin / kBatch * kBatch; j0 < end; j0 += kBatch) {
    const int page = max(0, page_of(a.batch, b, j0, a.status));
    const long long row0 = ((static_cast<long long>(page) * a.kv_heads + h) << a.batch.page_shift) + (j0 & ((1 << a.batch.page_shift) - 1));
    float s[kBatch], s_by[kBatch], v[kBatch][kPer];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      // (half of a key's scale before the product with the query and the rest behind it: either alone may lead out of fp32's range)
      const int ke = k8 ? a.k_exp[row0 + i] - 127 : 0, half = ke >> 1;
      s_by[i] = exponent_scale(127 + ke - half);
      float k[kPer];
      numbers(a.k, half, row0 + i, k);
      numbers(a.v, k8 ? a.v_exp[row0 + i] - 127 : 0, row0 + i, v[i]);
      s[i] = 0.f;
#pragma unroll
      for (int c = 0; c < kPer; ++c) s[i] = fmaf(q[c], k[c], s[i]);
    }
    float m_new = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
      // (the scale behind the product: a query's number times it may be too small to keep all its bits)
      s[i] = j0 + i >= begin && j0 + i < end ? s[i] * s_by[i] * a.scale_log2 : -INFINITY;
      m_new = fmaxf(m_new, s[i]);
    }
    const float keep = exp2_fast(m - m_new);
    m = m_new;
    l *= keep;
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[c] *= keep;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const bool seen = j0 + i >= begin && j0 + i < end;
      const float p = seen ? exp2_fast(s[i] - m) : 0.f;
      l += p;
#pragma unroll
      for (int c = 0; c < kPer; ++c) acc[c] = fmaf(p, seen ? v[i][c] : 0.f, acc[c]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(a.o) + (static_cast<long long>(t) * a.kv_heads * a.group + head) * D) + lane * (kPer / 2);
#pragma unroll
  for (int c = 0; c < kPer / 2; ++c) out[c] = Fmt<T>::pack2(acc[2 * c] * inv, acc[2 * c + 1] * inv);
}

}  // namespace ftb
