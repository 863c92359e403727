// Keys and query rows as operands of mma.m16n8k16 with the keys on the M side.
#pragma once
#include <type_traits>

#include "paged_attn.cuh"

namespace ftb {

// 16 bytes that nobody else asks for.
__device__ __forceinline__ uint4 load_once(const unsigned char* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Row `row` of a tile of `rows` that begins with flat0 (token, head of the group) of a sequence whose tokens begin with row `first`: lane (g, c) holds
// of it what it holds of a key, d = 32 j + 8 c .. + 7 (8-bit caches: 64 j + 16 c .. + 15); zeros behind the last row.  -> what the
// products with it are to be multiplied by: the scale in log2, for bf16 queries over an 8-bit cache times the power of two that the row
// was divided by to lie in fp16's range (what it loses is below 2^-24 of its largest number).
template <typename T, bool k8, int D>
__device__ __forceinline__ float load_query(const PagedAttn& a, int first, int h, int flat0, int row, int rows, int c, uint32_t (&q)[D / 16][2]) {
  const int flat = flat0 + row, token = flat / a.group;
  const T* src = static_cast<const T*>(a.q) + static_cast<long long>(first + token) * a.q_row +
                 static_cast<long long>(h * a.group + flat - token * a.group) * a.q_head;
  uint4 x[D / 32];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    x[j] = make_uint4(0u, 0u, 0u, 0u);
    const int d0 = k8 ? (j >> 1) * 64 + c * 16 + (j & 1) * 8 : j * 32 + c * 8;
    if (row < rows) x[j] = *reinterpret_cast<const uint4*>(src + d0);
  }
  float mine = a.scale_log2;
  if constexpr (k8 && !std::is_same<T, __half>::value) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t w = __vmaxu2(__vmaxu2(x[j].x & 0x7fff7fffu, x[j].y & 0x7fff7fffu), __vmaxu2(x[j].z & 0x7fff7fffu, x[j].w & 0x7fff7fffu));
      m = max(m, max(w & 0xffffu, w >> 16));
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // the row times 2^(127 - e), e its largest number's exponent: that one is in [1, 2).  (A row that is not finite stays so.)
    const int e = min(253, max(1, static_cast<int>(m >> 7)));
    const float by = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
    mine *= __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&x[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(w[i]);
        w[i] = Fmt<__half>::pack2(f.x * by, f.y * by);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    q[2 * j][0] = x[j].x;
    q[2 * j][1] = x[j].y;
    q[2 * j + 1][0] = x[j].z;
    q[2 * j + 1][1] = x[j].w;
  }
  return mine;
}

}  // namespace ftb
