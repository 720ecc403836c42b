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

// A workspace begins with this many counters, whatever the operator and its sizes, and the sums of parts come
// after them: the counters, zero between calls, are then where no call of any size leaves a sum.
constexpr int64_t WORK_COUNTERS = 16384;
constexpr int64_t WORK_COUNTER_BYTES = WORK_COUNTERS * 4;

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

// Tokens of sequence b (positions are below 2^31), negative when its table row cannot hold them, which is recorded.
__device__ __forceinline__ int paged_count(const PagedKv& p, int b) {
  const int n = __ldg(p.lengths + b);
  if (n >= 0 && n <= p.max_pages * p.page_size) return n;
  atomicExch(p.err, PAGED_ERR);
  return -1;
}

// Tokens to be read of sequence b: those that its table row can hold.
__device__ __forceinline__ int paged_length(const PagedKv& p, int b) {
  const int n = paged_count(p, b);
  return n >= 0 ? n : __ldg(p.lengths + b) < 0 ? 0 : p.max_pages * p.page_size;
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
  QgDiv per_div;              // accesses of a head
};

// Bound: the new rows are read and written once (f32 into bf16: 6 bytes an element).  A warp takes one
// row, looks its sequence and its slot up once (the sequence by bisection of row_start, one probe per
// lane and turn) and copies all heads' keys and values: 16-byte reads where the rows allow, four in
// flight per lane, written in the width that they convert to.  24 prompts of up to 4096 tokens, 8 heads of
// 128, f32 into bf16 (518 MB): 86 us, 6.06 TB/s, 92% of the copy rate (one thread per element and look-up:
// 292 us).  64 rows of 12 heads of 64: 6.1 us, the time to launch it from the host.
constexpr int APPEND_WARPS = 8;

template <int DT> struct AppendElem;
template <> struct AppendElem<MIRA_DT_F32> { using type = float; };
template <> struct AppendElem<MIRA_DT_F16> { using type = __half; };
template <> struct AppendElem<MIRA_DT_BF16> { using type = __nv_bfloat16; };

template <int DT>
__device__ __forceinline__ float append_f32(typename AppendElem<DT>::type x) {
  if constexpr (DT == MIRA_DT_F32) return x;
  else if constexpr (DT == MIRA_DT_F16) return __half2float(x);
  else return __bfloat162float(x);
}
template <int DT>
__device__ __forceinline__ typename AppendElem<DT>::type append_to(float x) {
  if constexpr (DT == MIRA_DT_F32) return x;
  else if constexpr (DT == MIRA_DT_F16) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

// Four elements as one access.
template <class T> struct alignas(4 * sizeof(T)) Append4 { T v[4]; };

// W elements of a row from `at` on as f32 (0 past its end).
template <int SRC, int W>
__device__ __forceinline__ void append_get(const typename AppendElem<SRC>::type* row, int at, int dh, float (&x)[W]) {
  using S = typename AppendElem<SRC>::type;
  if constexpr (W == 4) {
    Append4<S> e{};
    if (at < dh) e = *reinterpret_cast<const Append4<S>*>(row + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = append_f32<SRC>(e.v[i]);
  } else {
    x[0] = at < dh ? append_f32<SRC>(row[at]) : 0.0f;
  }
}

// 8-bit codes of one row of keys or values, held by `lanes` lanes (lane `sub`), W elements each and turn:
// scale = absmax / 127 and codes rint(x / scale), both IEEE divisions like the int8 weights,
// whose instructions are the limit: 42156 rows of 8 heads of 128 from f32, 155 us (2.8 TB/s); reciprocals with
// the divisions left to the quotients near the middle of two codes were no faster.
template <int W, int TURNS>
__device__ __forceinline__ void append_codes(const float (&x)[TURNS][W], int8_t* dst, float* scale, int dh, int lanes, int sub, bool mine) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < TURNS; ++j)
#pragma unroll
    for (int i = 0; i < W; ++i) top = np_maximum(top, fabsf(x[j][i]));
  for (int o = lanes >> 1; o > 0; o >>= 1) top = np_maximum(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = top == 0.0f ? 1.0f : __fdiv_rn(top, 127.0f);      // NaN if the row has one, so that it shows
  if (!mine) return;
  if (sub == 0) *scale = s;
#pragma unroll
  for (int j = 0; j < TURNS; ++j) {
    const int at = (sub + 32 * j) * W;
    if (at >= dh) break;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) codes |= uint32_t(round_clip_i8(__fdiv_rn(x[j][i], s)) & 0xff) << (8 * i);
    if constexpr (W == 4) *reinterpret_cast<uint32_t*>(dst + at) = codes;
    else dst[at] = static_cast<int8_t>(codes);
  }
}

// The sequence of a row: the last b with row_start[b] <= row.  The whole warp asks.
__device__ __forceinline__ int append_sequence(const AppendParams& p, int64_t row, int lane) {
  int lo = 0, hi = p.kv.batch;        // row_start[lo] <= row < row_start[hi]
  while (hi - lo > 1) {
    const int width = (hi - lo + 31) / 32;
    const int at = lo + lane * width;
    const uint32_t le = __ballot_sync(0xffffffffu, at < hi && __ldg(p.row_start + at) <= row);
    const int last = 31 - __clz(le);  // -1: row_start[0] is above the row, which the caller refuses
    if (last < 0) return 0;
    lo += last * width;
    hi = min(hi, lo + width);
  }
  return lo;
}

// DST: MIRA_DT_I8, or the pages' type; VEC: rows and slots can be read and written four elements at a time.
template <int SRC, int DST, bool VEC>
__global__ void __launch_bounds__(APPEND_WARPS * 32) kv_append_kernel(const __grid_constant__ AppendParams p) {
  const PagedKv& kv = p.kv;
  const int lane = threadIdx.x & 31;
  for (int64_t row = blockIdx.x * int64_t(APPEND_WARPS) + (threadIdx.x >> 5); row < p.rows; row += int64_t(gridDim.x) * APPEND_WARPS) {
    int b = int(row), from_end = 1;
    if (p.row_start != nullptr) {
      b = append_sequence(p, row, lane);
      from_end = int(min(int64_t(__ldg(p.row_start + b + 1)) - row, int64_t(INT32_MAX)));
      if (__ldg(p.row_start + b) > row) from_end = 0;
    }
    const int n = paged_count(kv, b);
    if (n < 0 || (n == 0 && p.row_start == nullptr)) continue;      // where the rows belong is not known, or none is wanted
    const int pos = n - from_end;
    int page, slot;
    if (from_end <= 0 || pos < 0) {
      if (lane == 0) atomicExch(kv.err, PAGED_ERR);
      continue;
    }
    if (!paged_slot(kv, kv.table + b * kv.table_ld, pos, page, slot)) continue;
    const int64_t ko = page * kv.kst[0] + slot * kv.kst[2], vo = page * kv.vst[0] + slot * kv.vst[2];
    if constexpr (DST == MIRA_DT_I8) {
      // as many heads at once as the warp has room for
      using S = typename AppendElem<SRC>::type;
      constexpr int W = VEC ? 4 : 1, TURNS = MIRA_PAGED_DH_MAX / (32 * W);
      int lanes = 32;
      while (lanes > 1 && lanes / 2 * W >= kv.dh) lanes >>= 1;
      const int sub = lane & (lanes - 1);
      for (int h0 = 0; h0 < kv.kv_heads; h0 += 32 / lanes) {
        const int h = min(h0 + lane / lanes, kv.kv_heads - 1);
        const bool own = h0 + lane / lanes < kv.kv_heads;
        const S* kf = static_cast<const S*>(p.k_new) + h * p.kn[0] + row * p.kn[1];
        const S* vf = static_cast<const S*>(p.v_new) + h * p.vn[0] + row * p.vn[1];
        float k[TURNS][W], v[TURNS][W];
#pragma unroll
        for (int j = 0; j < TURNS; ++j) {
          append_get<SRC, W>(kf, (sub + 32 * j) * W, kv.dh, k[j]);
          append_get<SRC, W>(vf, (sub + 32 * j) * W, kv.dh, v[j]);
        }
        append_codes<W, TURNS>(k, static_cast<int8_t*>(kv.k) + ko + h * kv.kst[1],
                               kv.ks + page * kv.kss[0] + h * kv.kss[1] + slot * kv.kss[2], kv.dh, lanes, sub, own);
        append_codes<W, TURNS>(v, static_cast<int8_t*>(kv.v) + vo + h * kv.vst[1],
                               kv.vs + page * kv.vss[0] + h * kv.vss[1] + slot * kv.vss[2], kv.dh, lanes, sub, own);
      }
    } else {
      using S = typename AppendElem<SRC>::type;
      using D = typename AppendElem<DST>::type;
      const S* ks = static_cast<const S*>(p.k_new) + row * p.kn[1];
      const S* vs = static_cast<const S*>(p.v_new) + row * p.vn[1];
      D* kd = static_cast<D*>(kv.k) + ko;
      D* vd = static_cast<D*>(kv.v) + vo;
      constexpr int W = VEC ? 4 : 1, U = 4;
      const int per = kv.dh / W, total = kv.kv_heads * per;      // accesses of a head, of the row
      for (int e0 = lane; e0 < total; e0 += 32 * U) {
        Append4<S> k[U], v[U];
        int64_t kt[U], vt[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int e = e0 + 32 * u;
          if (e >= total) break;
          const int h = qg_div(e, p.per_div), d = (e - h * per) * W;
          kt[u] = h * kv.kst[1] + d;
          vt[u] = h * kv.vst[1] + d;
          const S* kf = ks + h * p.kn[0] + d;
          const S* vf = vs + h * p.vn[0] + d;
          if constexpr (VEC) {
            k[u] = *reinterpret_cast<const Append4<S>*>(kf);
            v[u] = *reinterpret_cast<const Append4<S>*>(vf);
          } else {
            k[u].v[0] = *kf;
            v[u].v[0] = *vf;
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (e0 + 32 * u >= total) break;
          if constexpr (VEC) {
            Append4<D> x, y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x.v[i] = append_to<DST>(append_f32<SRC>(k[u].v[i]));
              y.v[i] = append_to<DST>(append_f32<SRC>(v[u].v[i]));
            }
            *reinterpret_cast<Append4<D>*>(kd + kt[u]) = x;
            *reinterpret_cast<Append4<D>*>(vd + vt[u]) = y;
          } else {
            kd[kt[u]] = append_to<DST>(append_f32<SRC>(k[u].v[0]));
            vd[vt[u]] = append_to<DST>(append_f32<SRC>(v[u].v[0]));
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------- page copies

// Bound: the moved pages are read and written once.  The page ids travel in the kernel's parameters, so
// that nothing has to be copied to the device before it: few of them in a small parameter block (5 pages of
// 24 planes: 10.0 us a call; with 4 KB of parameters 12.5), up to 1000 in one launch.  700 pages of 16 KB in
// 32 planes (734 MB read and written): 120 us, 6.1 TB/s, 93% of the copy rate (in two launches 125.6).
constexpr int PAGE_COPY_FEW = 32, PAGE_COPY_SOME = 256, PAGE_COPY_MANY = 1000;     // pairs per launch
constexpr int PAGE_COPY_CHUNK = 16384;    // bytes of one block's share of a page
constexpr int PAGE_COPY_THREADS = 256;

struct PageCopyRegion {
  uint8_t* base;
  int64_t plane_stride, page_stride, page_bytes;
  int planes, chunks;      // chunks of a page
  int64_t first;           // first task of this region
  int vec;                 // 16-byte accesses
};

template <int PAIRS>
struct PageCopyParams {
  PageCopyRegion r[MIRA_PAGE_REGIONS];
  int n_regions, n;
  int64_t tasks;             // per pair
  int32_t src[PAIRS], dst[PAIRS];
};

// One block per (pair, plane, 16 KB of the page).
template <int PAIRS>
__global__ void __launch_bounds__(PAGE_COPY_THREADS) page_copy_kernel(const __grid_constant__ PageCopyParams<PAIRS> p) {
  const int64_t total = p.tasks * p.n;
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int pair = int(t / p.tasks);
    int64_t in = t - pair * p.tasks;
    int ri = 0;
    while (ri + 1 < p.n_regions && in >= p.r[ri + 1].first) ++ri;
    const PageCopyRegion& r = p.r[ri];
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
