// Keys and values in pages: addressing shared by the paged kernels, the element types of pages and
// rows, the kernel that appends new rows (with the conversion to the pages' type) and the kernel that
// duplicates pages.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "exact_math.cuh"
#include "memory_bound.cuh"
#include "qgemm_sm100.cuh"

namespace mira {

constexpr int PAGED_ERR = 4;   // error record: a page id, length or row range outside its bounds

struct PagedKv {
  void* k;
  void* v;
  float* ks;
  float* vs;
  int64_t kst[3], vst[3], kss[3], vss[3];   // element strides of (page, kv head, slot)
  const int32_t* table;
  int64_t table_ld;
  const int32_t* lengths;
  int batch, num_pages, max_pages, page_size, kv_heads, dh;
  QgDiv page_div;
  int* err;
};

// Tokens of sequence b, clamped to what its table row can hold (positions are below 2^31).
__device__ __forceinline__ int paged_length(const PagedKv& p, int b) {
  const int n = __ldg(p.lengths + b);
  const int cap = p.max_pages * p.page_size;
  if (n < 0 || n > cap) {
    atomicExch(p.err, PAGED_ERR);
    return n < 0 ? 0 : cap;
  }
  return n;
}

// Page and slot of a position; false (and an error record) when the table names no page of the pool.
__device__ __forceinline__ bool paged_slot(const PagedKv& p, const int32_t* row, int pos, int& page, int& slot) {
  const int i = qg_div(pos, p.page_div);
  slot = pos - i * p.page_size;
  page = __ldg(row + i);
  if (static_cast<uint32_t>(page) < static_cast<uint32_t>(p.num_pages)) return true;
  atomicExch(p.err, PAGED_ERR);
  return false;
}

// ---------------------------------------------------------------- element types

// One element of a MIRA_DT_* row as f32 (exact), and its store with one rounding.
__device__ __forceinline__ float dt_load(const void* p, int64_t i, int dtype) {
  if (dtype == MIRA_DT_F32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == MIRA_DT_F16) return __half2float(__ldg(static_cast<const __half*>(p) + i));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
}

// The same in two steps, for a load that is issued well before its value is used: converting at once
// would wait for it.
__device__ __forceinline__ uint32_t dt_load_raw(const void* p, int64_t i, int dtype) {
  return dtype == MIRA_DT_F32 ? __ldg(static_cast<const uint32_t*>(p) + i)
                              : uint32_t(__ldg(static_cast<const uint16_t*>(p) + i));
}
__device__ __forceinline__ float dt_from_raw(uint32_t raw, int dtype) {
  const float h = __half2float(__ushort_as_half(static_cast<uint16_t>(raw)));
  return __uint_as_float(dtype == MIRA_DT_F32 ? raw : dtype == MIRA_DT_F16 ? __float_as_uint(h) : raw << 16);
}

__device__ __forceinline__ void dt_store(void* p, int64_t i, int dtype, float v) {
  if (dtype == MIRA_DT_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == MIRA_DT_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------- append

struct AppendParams {
  PagedKv kv;
  const void* k_new;
  const void* v_new;
  int64_t kn[2], vn[2];       // element strides of (kv head, row)
  const int32_t* row_start;
  int64_t rows;
  int src_dtype, dtype;
};

// One warp per (row, kv head): the row's sequence by bisection of row_start, then the head's key and
// value converted lane by lane.
constexpr int APPEND_WARPS = 8;

__device__ __forceinline__ void append_row(const void* src, int64_t so, int src_dtype, void* dst, int64_t d0, int dtype,
                                           float* scale, int dh, int lane) {
  if (dtype != MIRA_DT_I8) {
    for (int i = lane; i < dh; i += 32) dt_store(dst, d0 + i, dtype, dt_load(src, so + i, src_dtype));
    return;
  }
  // scale = absmax / 127 and codes rint(x / scale), both IEEE divisions like the int8 weights
  float top = 0.0f;
  for (int i = lane; i < dh; i += 32) top = np_maximum(top, fabsf(dt_load(src, so + i, src_dtype)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = np_maximum(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = top > 0.0f ? __fdiv_rn(top, 127.0f) : 1.0f;
  if (lane == 0) *scale = s;
  for (int i = lane; i < dh; i += 32) {
    const float z = __fdiv_rn(dt_load(src, so + i, src_dtype), s);
    static_cast<int8_t*>(dst)[d0 + i] = static_cast<int8_t>(round_clip_i8(z) & 0xff);
  }
}

__global__ void __launch_bounds__(APPEND_WARPS * 32) kv_append_kernel(const __grid_constant__ AppendParams p) {
  const PagedKv& kv = p.kv;
  const int lane = threadIdx.x & 31;
  const int64_t tasks = p.rows * kv.kv_heads;
  const int64_t step = int64_t(gridDim.x) * APPEND_WARPS;
  for (int64_t t = blockIdx.x * int64_t(APPEND_WARPS) + (threadIdx.x >> 5); t < tasks; t += step) {
    const int64_t row = t / kv.kv_heads;
    const int h = int(t - row * kv.kv_heads);
    int b = int(row), from_end = 1;
    if (p.row_start != nullptr) {
      int lo = 0, hi = kv.batch;        // row_start[lo] <= row < row_start[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.row_start + mid) <= row) lo = mid;
        else hi = mid;
      }
      b = lo;
      from_end = int(__ldg(p.row_start + b + 1) - row);
    }
    const int n = paged_length(kv, b);
    if (n == 0 && p.row_start == nullptr) continue;
    const int pos = n - from_end;
    if (from_end <= 0 || pos < 0) {
      if (lane == 0) atomicExch(kv.err, PAGED_ERR);
      continue;
    }
    int page, slot;
    if (!paged_slot(kv, kv.table + b * kv.table_ld, pos, page, slot)) continue;
    append_row(p.k_new, h * p.kn[0] + row * p.kn[1], p.src_dtype, kv.k,
               page * kv.kst[0] + h * kv.kst[1] + slot * kv.kst[2], p.dtype,
               kv.ks + (page * kv.kss[0] + h * kv.kss[1] + slot * kv.kss[2]), kv.dh, lane);
    append_row(p.v_new, h * p.vn[0] + row * p.vn[1], p.src_dtype, kv.v,
               page * kv.vst[0] + h * kv.vst[1] + slot * kv.vst[2], p.dtype,
               kv.vs + (page * kv.vss[0] + h * kv.vss[1] + slot * kv.vss[2]), kv.dh, lane);
  }
}

// ---------------------------------------------------------------- page copies

constexpr int PAGE_COPY_PAIRS = 448;      // pairs per launch: the ids travel in the kernel's parameters
constexpr int PAGE_COPY_CHUNK = 16384;    // bytes of one block's share of a page
constexpr int PAGE_COPY_THREADS = 256;

struct PageCopyParams {
  struct Region {
    uint8_t* base;
    int64_t plane_stride, page_stride, page_bytes;
    int planes, chunks;      // chunks of a page
    int64_t first;           // first task of this region
    int vec;                 // 16-byte accesses
  } r[MIRA_PAGE_REGIONS];
  int n_regions, n;
  int64_t tasks;             // per pair
  int32_t src[PAGE_COPY_PAIRS], dst[PAGE_COPY_PAIRS];
};

// One block per (pair, plane, 16 KB of the page).
__global__ void __launch_bounds__(PAGE_COPY_THREADS) page_copy_kernel(const __grid_constant__ PageCopyParams p) {
  const int64_t total = p.tasks * p.n;
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int pair = int(t / p.tasks);
    int64_t in = t - pair * p.tasks;
    int ri = 0;
    while (ri + 1 < p.n_regions && in >= p.r[ri + 1].first) ++ri;
    const PageCopyParams::Region& r = p.r[ri];
    in -= r.first;
    const int64_t plane = in / r.chunks;
    const int64_t at = (in - plane * r.chunks) * PAGE_COPY_CHUNK;
    const int64_t bytes = min(int64_t(PAGE_COPY_CHUNK), r.page_bytes - at);
    const uint8_t* s = r.base + plane * r.plane_stride + p.src[pair] * r.page_stride + at;
    uint8_t* d = r.base + plane * r.plane_stride + p.dst[pair] * r.page_stride + at;
    if (r.vec) {
      const uint4* s4 = reinterpret_cast<const uint4*>(s);
      uint4* d4 = reinterpret_cast<uint4*>(d);
      const int n16 = int(bytes / 16);
#pragma unroll 4
      for (int i = threadIdx.x; i < n16; i += PAGE_COPY_THREADS) d4[i] = s4[i];
      for (int64_t i = int64_t(n16) * 16 + threadIdx.x; i < bytes; i += PAGE_COPY_THREADS) d[i] = s[i];
    } else {
      for (int64_t i = threadIdx.x; i < bytes; i += PAGE_COPY_THREADS) d[i] = s[i];
    }
  }
}

}  // namespace mira
