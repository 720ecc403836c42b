// Warp-level 16x8x16 products with f32 accumulators, for operands that live in registers.
//
// Fragments (g = lane / 4, t = lane % 4): a0 = A[g][2t..], a1 = A[g + 8][2t..], a2 = A[g][2t + 8..],
// a3 = A[g + 8][2t + 8..]; b0 = B[2t..][g], b1 = B[2t + 8..][g]; d0, d1 = D[g][2t, 2t + 1],
// d2, d3 = D[g + 8][2t, 2t + 1].  The sum over k does not care which k a fragment position holds as
// long as A and B agree.
//
// These feed memory-bound kernels whose left operand is built in registers a few instructions before
// its use; the tcgen05 path would have to write it to shared memory first and read the result back
// from tensor memory, for contractions that are a few percent of the time.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace mira {

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if (BF16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from a zero accumulator.
template <bool BF16>
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
  if (BF16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t h2_bits(__half2 v) {
  uint32_t u;
  memcpy(&u, &v, 4);
  return u;
}
__device__ __forceinline__ __half2 bits_h2(uint32_t u) {
  __half2 v;
  memcpy(&v, &u, 4);
  return v;
}
__device__ __forceinline__ uint32_t b2_bits(__nv_bfloat162 v) {
  uint32_t u;
  memcpy(&u, &v, 4);
  return u;
}
__device__ __forceinline__ __nv_bfloat162 bits_b2(uint32_t u) {
  __nv_bfloat162 v;
  memcpy(&v, &u, 4);
  return v;
}

// x = hi + mid + lo with three bf16 values (as the upper halves of f32 words), by truncation: 24
// significant bits are three times eight, so the split is exact (below 2^-118 the last piece may lose
// bits under bf16's smallest value).  An infinity or NaN stays whole in the first piece.
__device__ __forceinline__ void split3_bf16(float x, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const uint32_t u = __float_as_uint(x);
  hi = u & 0xffff0000u;
  if ((u & 0x7f800000u) == 0x7f800000u) {
    if (u & 0x007fffffu) hi |= 0x00400000u;
    mid = lo = 0;
    return;
  }
  const float r = x - __uint_as_float(hi);
  mid = __float_as_uint(r) & 0xffff0000u;
  lo = __float_as_uint(r - __uint_as_float(mid));
}

}  // namespace mira
