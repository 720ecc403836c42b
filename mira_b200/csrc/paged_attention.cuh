// Attention of one new token per sequence over paged keys and values, split over the cache's length
// and joined inside one launch.
//
// Mathematics.  For a part S of the visible positions of one (sequence, head) let
//   m_S = max_{t in S} s_t,  l_S = sum_{t in S} 2^(s_t - m_S),  a_S = sum_{t in S} 2^(s_t - m_S) v_t
// with s_t = scale log2(e) q . k_t.  Parts join as m = max m_S, l = sum l_S 2^(m_S - m), a likewise,
// and o = a / l, lse = (m + log2 l) / log2(e).  Each lane group, warp and block keeps such a triple, so
// the keys and values are read once and no score is stored.
#pragma once
#include <cstdint>

#include "paged_kv.cuh"

namespace mira {

constexpr int PA_WARPS = 8;
constexpr int PA_THREADS = PA_WARPS * 32;

struct PagedAttnParams {
  PagedKv kv;
  const void* q;
  int64_t qs[3];            // element strides of (batch, head, element)
  int q_dtype;
  float scale_log2;         // scale * log2(e)
  int heads, group, head_blocks, units;   // units = kv_heads * head_blocks per sequence
  int window, sinks;        // window 0: none
  void* out;
  int64_t os[3];
  int8_t* out_i8;
  int64_t is[3];
  QuantScale q8;
  float* lse;
  float* part;              // partial triples, two slots per block
  int* counters;            // [batch * units], zero between calls
};

// ---------------------------------------------------------------- dealing out the work

// The visible positions of a sequence, numbered without the hole between the sinks and the window:
// visible i is position i for i < sinks and i + skip after them.
struct PaSeq {
  int n, sinks, skip, tiles;   // tiles: at least one, so that every output is written by someone
};

template <int TILE>
__device__ __forceinline__ PaSeq pa_seq(const PagedAttnParams& p, int b) {
  const int len = paged_length(p.kv, b);
  PaSeq s;
  const int start = (p.window > 0 && len > p.window) ? len - p.window : 0;
  s.sinks = p.sinks < start ? p.sinks : start;
  s.skip = start - s.sinks;
  s.n = len - s.skip;
  s.tiles = s.n > TILE ? (s.n - 1) / TILE + 1 : 1;
  return s;
}

// The tiles of all (sequence, unit) pairs form one line of `total` tiles, sequence by sequence and
// unit by unit; block c of g takes [total c / g, total (c + 1) / g).
__device__ __forceinline__ int64_t pa_lo(int64_t total, int64_t c, int64_t g) { return total * c / g; }
__device__ __forceinline__ int pa_block_of(int64_t total, int64_t x, int64_t g) {
  return static_cast<int>(((x + 1) * g - 1) / total);
}

// Sum of v over the block, and the sum over the lower-numbered threads (one barrier pair).
__device__ __forceinline__ int64_t pa_scan(int64_t v, int64_t& before, int64_t* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int64_t total = 0, base = 0;
#pragma unroll
  for (int w = 0; w < PA_WARPS; ++w) {
    if (w == warp) base = total;
    total += warp_sums[w];
  }
  before = base + x - v;
  return total;
}

// ---------------------------------------------------------------- rows of the pages

// VB bytes of a row as one access; elements of T as f32.
template <int VB> struct PaVec;
template <> struct PaVec<16> { using type = uint4; };
template <> struct PaVec<8> { using type = uint2; };
template <> struct PaVec<4> { using type = uint32_t; };
template <> struct PaVec<2> { using type = uint16_t; };
template <> struct PaVec<1> { using type = uint8_t; };

template <typename T, int VB>
__device__ __forceinline__ void pa_unpack(const typename PaVec<VB>::type& raw, float (&x)[VB / sizeof(T)]) {
  constexpr int VE = VB / int(sizeof(T));
  T e[VE];
  memcpy(e, &raw, VB);
#pragma unroll
  for (int i = 0; i < VE; ++i) x[i] = static_cast<float>(e[i]);
}

// ---------------------------------------------------------------- the end of a unit

// Writes the GP heads of (sequence b, unit) from their joined triples: acc(g, d) is a, m and l in smem.
template <int GP, class F>
__device__ __forceinline__ void pa_write(const PagedAttnParams& p, int b, int unit, const float* m, const float* l, F acc) {
  const int kvh = unit / p.head_blocks, g0 = (unit - kvh * p.head_blocks) * GP;
  const int live = min(GP, p.group - g0);
  const int h0 = kvh * p.group + g0;
  for (int i = threadIdx.x; i < live * p.kv.dh; i += PA_THREADS) {
    const int g = i / p.kv.dh, d = i - g * p.kv.dh;
    const float lg = l[g];
    const float o = lg == 0.0f ? 0.0f : __fdiv_rn(acc(g, d), lg);
    if (p.out != nullptr) dt_store(p.out, b * p.os[0] + (h0 + g) * p.os[1] + d * p.os[2], p.q_dtype, o);
    if (p.out_i8 != nullptr)
      p.out_i8[b * p.is[0] + (h0 + g) * p.is[1] + d * p.is[2]] = static_cast<int8_t>(quant_byte(o, p.q8) & 0xff);
  }
  if (p.lse != nullptr && int(threadIdx.x) < live) {
    const float lg = l[threadIdx.x];
    p.lse[int64_t(b) * p.heads + h0 + threadIdx.x] =
        lg == 0.0f ? -INFINITY : fmaf(m[threadIdx.x], 0.693147180559945309f, logf(lg));
  }
}

__device__ __forceinline__ float pa_weight(float m, float top) {
  return m == -INFINITY ? 0.0f : exp2f(m - top);   // a part without a finite score weighs nothing
}

// ---------------------------------------------------------------- the kernel on FMA units

// T: the pages' element; DHP: head dimension rounded up to 32, 64, 128 or 256; GP: query heads that
// share a pass over the rows; VB: bytes per access (16, or less where rows are not 16-byte aligned).
template <typename T, int DHP, int GP, int VB>
struct PaCfg {
  static constexpr int VE = VB / int(sizeof(T));            // elements of an access
  static constexpr int LPR = DHP / VE < 32 ? DHP / VE : 32; // lanes of a row
  static constexpr int NV = DHP / (VE * LPR);               // accesses of a lane per row
  static constexpr int EPL = VE * NV;                       // elements of a lane
  static constexpr int TPS = 32 / LPR;                      // rows of a warp access
  static constexpr int U = NV > 1 ? 2 : 4;                  // rows in flight per lane
  static constexpr int ROWS = TPS * U;                      // rows of a warp step
  static constexpr int TILE = PA_WARPS * ROWS;
  static constexpr int SMEM = (PA_WARPS * GP * (DHP + 2) + 2 * GP) * 4;
  static constexpr int SLOT = GP * (DHP + 2);               // floats of a partial triple
};

template <typename T, int DHP, int GP, int VB>
__global__ void __launch_bounds__(PA_THREADS) paged_attention_kernel(const __grid_constant__ PagedAttnParams p) {
  using C = PaCfg<T, DHP, GP, VB>;
  using V = typename PaVec<VB>::type;
  constexpr bool I8 = sizeof(T) == 1;
  extern __shared__ __align__(16) float sm[];
  float* s_acc = sm;                                  // [warp][GP][DHP]
  float* s_m = s_acc + PA_WARPS * GP * DHP;           // [warp][GP]
  float* s_l = s_m + PA_WARPS * GP;
  float* j_m = s_l + PA_WARPS * GP;                   // [GP] the block's
  float* j_l = j_m + GP;
  __shared__ int64_t s_scan[PA_WARPS];
  __shared__ int64_t s_found[2];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % C::LPR, slot_of_lane = lane / C::LPR;

  // this block's tiles
  int64_t total = 0;
  for (int b0 = 0; b0 < p.kv.batch; b0 += PA_THREADS) {
    const int b = b0 + threadIdx.x;
    int64_t before;
    total += pa_scan(b < p.kv.batch ? pa_seq<C::TILE>(p, b).tiles : 0, before, s_scan);
  }
  total *= p.units;
  const int64_t g = min(int64_t(gridDim.x), total);
  if (blockIdx.x >= g) return;
  const int64_t lo = pa_lo(total, blockIdx.x, g), hi = pa_lo(total, blockIdx.x + 1, g);
  {
    int64_t run = 0;
    for (int b0 = 0; b0 < p.kv.batch; b0 += PA_THREADS) {
      const int b = b0 + threadIdx.x;
      const int64_t mine = b < p.kv.batch ? int64_t(pa_seq<C::TILE>(p, b).tiles) * p.units : 0;
      int64_t before;
      const int64_t sum = pa_scan(mine, before, s_scan);
      before += run;
      if (mine > 0 && before <= lo && lo < before + mine) {
        s_found[0] = b;
        s_found[1] = before;
      }
      run += sum;
    }
    __syncthreads();
  }
  int b = int(s_found[0]);
  int64_t base = s_found[1];       // first tile of sequence b
  PaSeq seq = pa_seq<C::TILE>(p, b);

  for (int64_t cur = lo; cur < hi;) {
    while (cur >= base + int64_t(seq.tiles) * p.units) {
      base += int64_t(seq.tiles) * p.units;
      seq = pa_seq<C::TILE>(p, ++b);
    }
    const int unit = int((cur - base) / seq.tiles);
    const int64_t us = base + int64_t(unit) * seq.tiles, ue = us + seq.tiles;   // the unit's tiles
    const int64_t end = min(ue, hi);
    const int t0 = int(cur - us) * C::TILE, t1 = min(seq.n, int(end - us) * C::TILE);
    const int kvh = unit / p.head_blocks, g0 = (unit - kvh * p.head_blocks) * GP;

    // queries of the unit, scaled
    float q[GP][C::EPL];
#pragma unroll
    for (int gi = 0; gi < GP; ++gi)
#pragma unroll
      for (int j = 0; j < C::NV; ++j)
#pragma unroll
        for (int e = 0; e < C::VE; ++e) {
          const int d = (sub + j * C::LPR) * C::VE + e;
          q[gi][j * C::VE + e] = (g0 + gi < p.group && d < p.kv.dh)
              ? dt_load(p.q, b * p.qs[0] + (kvh * p.group + g0 + gi) * p.qs[1] + d * p.qs[2], p.q_dtype) * p.scale_log2
              : 0.0f;
        }
    float acc[GP][C::EPL], m[GP], l[GP];
#pragma unroll
    for (int gi = 0; gi < GP; ++gi) {
      m[gi] = -INFINITY;
      l[gi] = 0.0f;
#pragma unroll
      for (int e = 0; e < C::EPL; ++e) acc[gi][e] = 0.0f;
    }
    const int32_t* trow = p.kv.table + b * p.kv.table_ld;
    const T* kb = static_cast<const T*>(p.kv.k) + kvh * p.kv.kst[1];
    const T* vb = static_cast<const T*>(p.kv.v) + kvh * p.kv.vst[1];

    for (int w0 = t0 + warp * C::ROWS; w0 < t1; w0 += C::TILE) {
      V kr[C::U][C::NV], vr[C::U][C::NV];
      float ksc[C::U], vsc[C::U];
      bool ok[C::U];
#pragma unroll
      for (int u = 0; u < C::U; ++u) {
        const int i = w0 + u * C::TPS + slot_of_lane;
        int page = 0, slot = 0;
        ok[u] = i < t1 && paged_slot(p.kv, trow, i + (i < seq.sinks ? 0 : seq.skip), page, slot);
        const T* kp = kb + page * p.kv.kst[0] + slot * p.kv.kst[2];
        const T* vp = vb + page * p.kv.vst[0] + slot * p.kv.vst[2];
#pragma unroll
        for (int j = 0; j < C::NV; ++j) {
          const int d = (sub + j * C::LPR) * C::VE;
          const bool in = ok[u] && d < p.kv.dh;
          kr[u][j] = in ? __ldg(reinterpret_cast<const V*>(kp + d)) : V{};
          vr[u][j] = in ? __ldg(reinterpret_cast<const V*>(vp + d)) : V{};
        }
        if (I8) {
          ksc[u] = ok[u] ? __ldg(p.kv.ks + page * p.kv.kss[0] + kvh * p.kv.kss[1] + slot * p.kv.kss[2]) : 0.0f;
          vsc[u] = ok[u] ? __ldg(p.kv.vs + page * p.kv.vss[0] + kvh * p.kv.vss[1] + slot * p.kv.vss[2]) : 0.0f;
        }
      }
      float s[C::U][GP];
#pragma unroll
      for (int u = 0; u < C::U; ++u) {
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) s[u][gi] = 0.0f;
#pragma unroll
        for (int j = 0; j < C::NV; ++j) {
          float x[C::VE];
          pa_unpack<T, VB>(kr[u][j], x);
#pragma unroll
          for (int gi = 0; gi < GP; ++gi)
#pragma unroll
            for (int e = 0; e < C::VE; ++e) s[u][gi] = fmaf(q[gi][j * C::VE + e], x[e], s[u][gi]);
        }
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) {
#pragma unroll
          for (int o = 1; o < C::LPR; o <<= 1) s[u][gi] += __shfl_xor_sync(0xffffffffu, s[u][gi], o);
          if (I8) s[u][gi] *= ksc[u];
          if (!ok[u]) s[u][gi] = -INFINITY;
        }
      }
#pragma unroll
      for (int gi = 0; gi < GP; ++gi) {
        float top = m[gi];
#pragma unroll
        for (int u = 0; u < C::U; ++u) top = fmaxf(top, s[u][gi]);
        const float safe = top == -INFINITY ? 0.0f : top;
        const float fade = exp2f(m[gi] - safe);
        m[gi] = top;
        l[gi] *= fade;
#pragma unroll
        for (int e = 0; e < C::EPL; ++e) acc[gi][e] *= fade;
#pragma unroll
        for (int u = 0; u < C::U; ++u) {
          s[u][gi] = exp2f(s[u][gi] - safe);
          l[gi] += s[u][gi];
          if (I8) s[u][gi] *= vsc[u];
        }
      }
#pragma unroll
      for (int u = 0; u < C::U; ++u)
#pragma unroll
        for (int j = 0; j < C::NV; ++j) {
          float x[C::VE];
          pa_unpack<T, VB>(vr[u][j], x);
#pragma unroll
          for (int gi = 0; gi < GP; ++gi)
#pragma unroll
            for (int e = 0; e < C::VE; ++e)
              acc[gi][j * C::VE + e] = fmaf(s[u][gi], x[e], acc[gi][j * C::VE + e]);
        }
    }

    // join the warp's lane groups, then the warps
#pragma unroll
    for (int gi = 0; gi < GP; ++gi) {
#pragma unroll
      for (int o = C::LPR; o < 32; o <<= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m[gi], o), lo_ = __shfl_xor_sync(0xffffffffu, l[gi], o);
        const float top = fmaxf(m[gi], mo);
        const float wa = pa_weight(m[gi], top), wb = pa_weight(mo, top);
        l[gi] = l[gi] * wa + lo_ * wb;
        m[gi] = top;
#pragma unroll
        for (int e = 0; e < C::EPL; ++e)
          acc[gi][e] = acc[gi][e] * wa + __shfl_xor_sync(0xffffffffu, acc[gi][e], o) * wb;
      }
      if (slot_of_lane == 0) {
#pragma unroll
        for (int j = 0; j < C::NV; ++j)
#pragma unroll
          for (int e = 0; e < C::VE; ++e)
            s_acc[(warp * GP + gi) * DHP + (sub + j * C::LPR) * C::VE + e] = acc[gi][j * C::VE + e];
      }
      if (lane == 0) {
        s_m[warp * GP + gi] = m[gi];
        s_l[warp * GP + gi] = l[gi];
      }
    }
    __syncthreads();
    if (threadIdx.x < GP) {
      float top = -INFINITY, sum = 0.0f;
      for (int w = 0; w < PA_WARPS; ++w) top = fmaxf(top, s_m[w * GP + threadIdx.x]);
      for (int w = 0; w < PA_WARPS; ++w) {
        const float wt = pa_weight(s_m[w * GP + threadIdx.x], top);
        sum += s_l[w * GP + threadIdx.x] * wt;
        s_m[w * GP + threadIdx.x] = wt;      // from here on the warp's weight
      }
      j_m[threadIdx.x] = top;
      j_l[threadIdx.x] = sum;
    }
    __syncthreads();
    auto joined = [&](int gi, int d) {
      float a = 0.0f;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) a = fmaf(s_acc[(w * GP + gi) * DHP + d], s_m[w * GP + gi], a);
      return a;
    };
    const int first = pa_block_of(total, us, g), last = pa_block_of(total, ue - 1, g);
    if (first == last) {
      pa_write<GP>(p, b, unit, j_m, j_l, joined);
    } else {
      // a part of the unit: leave the triple in this block's slot; the last block to arrive joins all
      float* mine = p.part + (int64_t(blockIdx.x) * 2 + (lo >= us ? 0 : 1)) * C::SLOT;
      for (int i = threadIdx.x; i < GP * DHP; i += PA_THREADS) mine[2 * GP + i] = joined(i / DHP, i % DHP);
      if (threadIdx.x < GP) {
        mine[threadIdx.x] = j_m[threadIdx.x];
        mine[GP + threadIdx.x] = j_l[threadIdx.x];
      }
      __threadfence();
      __syncthreads();
      int* counter = p.counters + int64_t(b) * p.units + unit;
      if (threadIdx.x == 0) s_last = atomicAdd(counter, 1) == last - first;
      __syncthreads();
      if (s_last) {
        __threadfence();
        auto slot_of = [&](int c) {
          return p.part + (int64_t(c) * 2 + (pa_lo(total, c, g) >= us ? 0 : 1)) * C::SLOT;
        };
        if (threadIdx.x < GP) {
          float top = -INFINITY, sum = 0.0f;
          for (int c = first; c <= last; ++c) top = fmaxf(top, __ldcg(slot_of(c) + threadIdx.x));
          for (int c = first; c <= last; ++c)
            sum += __ldcg(slot_of(c) + GP + threadIdx.x) * pa_weight(__ldcg(slot_of(c) + threadIdx.x), top);
          j_m[threadIdx.x] = top;
          j_l[threadIdx.x] = sum;
        }
        __syncthreads();
        pa_write<GP>(p, b, unit, j_m, j_l, [&](int gi, int d) {
          float a = 0.0f;
          for (int c = first; c <= last; ++c) {
            const float* from = slot_of(c);
            a = fmaf(__ldcg(from + 2 * GP + gi * DHP + d), pa_weight(__ldcg(from + gi), j_m[gi]), a);
          }
          return a;
        });
        if (threadIdx.x == 0) *counter = 0;
      }
    }
    cur = end;
    __syncthreads();     // the shared triples are free again
  }
}

}  // namespace mira
