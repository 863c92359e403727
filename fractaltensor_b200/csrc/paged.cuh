// What the kernels over a paged cache share: where a row of new tokens belongs, and reading 8-bit rows.
//
// A batch is described by starts [B + 1] (first row of each sequence's new tokens), lens [B] (keys of each
// sequence, the new ones included) and table [B, W] (its pages).  Token i of the n new ones of sequence b is at
// position lens[b] - n + i.  Pages are [kv_heads, page_size, d]: the rows of one head of a page lie side by side.
//
// 8-bit rows: d e4m3 codes and one exponent byte e, a row's numbers being code * 2^(e - 127).  A scale that is
// a power of two costs e4m3 nothing (the codes are floating-point numbers themselves, with the same relative step at
// every scale) and makes scaling exact in both directions; a byte of it is 1 / d of the row.
#pragma once
#include <cuda_fp8.h>

#include "ptx.cuh"

namespace ftb {

struct PagedBatch {
  const int* table;
  const int* lens;
  const int* starts;
  int B, W, pages, page_shift;
};

// Sequence b and position of row t (b = B: none has it; a negative position: in front of the sequence); the whole warp asks for the
// same t.  32 probes a round, the last one with all that the answer needs: one round trip to memory up to 32 sequences, two up to 1024.
struct RowPlace {
  int b;
  long long pos;
};
__device__ __forceinline__ RowPlace place_of_row(const PagedBatch& x, int t, int lane) {
  int lo = 0, hi = x.B;  // the smallest b with starts[b + 1] > t is in [lo, hi], where hi = B stands for none
  while (hi - lo > 32) {
    const int step = (hi - lo + 31) >> 5;
    const int at = lo + (lane + 1) * step - 1;
    const unsigned above = __ballot_sync(0xffffffffu, at < hi ? x.starts[at + 1] > t : true);
    if (above == 0) return {x.B, 0};
    lo += (__ffs(above) - 1) * step;
    hi = min(hi, lo + step - 1) + 1;  // (one more, so that it is among the probes)
    hi = min(hi, x.B);
  }
  const int at = lo + lane, b = min(at, x.B - 1);
  const int begin = x.starts[b], end = x.starts[b + 1], len = x.lens[b];
  const unsigned here = __ballot_sync(0xffffffffu, at < x.B && begin <= t && end > t);
  if (here == 0) return {x.B, 0};
  const int first = __ffs(here) - 1;
  return {lo + first, static_cast<long long>(__shfl_sync(0xffffffffu, len, first)) - __shfl_sync(0xffffffffu, end, first) + t};
}

// The page that holds position pos of sequence b, or -1 where the table has none (recorded in the status word).
__device__ __forceinline__ int page_of(const PagedBatch& x, int b, long long pos, int* status) {
  const long long i = pos >> x.page_shift;
  const int page = i < x.W ? x.table[static_cast<long long>(b) * x.W + i] : -1;
  if (page >= 0 && page < x.pages) return page;
  atomicCAS(status, 0, FTB_ERR_INDEX);
  return -1;
}

__device__ __forceinline__ float exponent_scale(int e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }

// Two e4m3 codes -> two fp16 numbers (exact; a NaN stays one).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}

// Four codes -> fp16 numbers of the lower and the upper two.
__device__ __forceinline__ void e4m3x4_to_f16x2(uint32_t codes, uint32_t& lower, uint32_t& upper) {
  asm("{\n.reg .b16 l, u;\nmov.b32 {l, u}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, u;\n}"
      : "=&r"(lower), "=r"(upper)
      : "r"(codes));
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

}  // namespace ftb
