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

constexpr int PA_MAX_WARPS = 16;

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
  int* counters;            // [blocks], zero between calls
  int slots, feeders;       // steps in a warp's ring, copying warps of a block
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

// The tiles of all (sequence, unit) pairs form one line of length `total`, sequence by sequence and unit
// by unit; block c of g takes [total c / g, total (c + 1) / g).  Before its tiles each unit has an empty
// stretch of PA_PART_COST: a part's beginning and end take a block as long as about that many tiles, and
// without it the blocks that get many short sequences finish last (64 sequences of 16 to 1024 tokens: the
// last block at twice the median's time).  Of 10, 14, 20 and 28 tiles on 32 shapes, 20 is the best or within 4%
// of it on 28 (32 sequences of 32/8 heads up to 8192, bf16: 128 us, with 14 122; 80 x 96/12 heads, f32: 121 us, with
// 14 145; 48 x 20/4 heads of 80, bf16: 68 us, with 14 73); 4 loses up to 40%.
constexpr int PA_PART_COST = 20;
// Quotients of nonnegative numbers; nearly all fit 32 bits, where dividing takes a fraction of the time.
__device__ __forceinline__ int64_t pa_quot(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}
__device__ __forceinline__ int64_t pa_lo(int64_t total, int64_t c, int64_t g) { return pa_quot(total * c, g); }
__device__ __forceinline__ int pa_block_of(int64_t total, int64_t x, int64_t g) {
  return static_cast<int>(pa_quot((x + 1) * g - 1, total));
}

// Sum of v over the block, and the sum over the lower-numbered threads.
__device__ __forceinline__ int64_t pa_scan(int64_t v, int64_t& before, int64_t* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
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
  for (int w = 0; w < warps; ++w) {
    if (w == warp) base = total;
    total += warp_sums[w];
  }
  before = base + x - v;
  return total;
}

// A block's share of the line, and the part of a unit at its front.
struct PaWork {
  int64_t total, blocks;       // the line, and blocks that share it
  int64_t lo, hi;              // this block's share
  int64_t cur;                 // what is done of it
  int b;                       // the sequence there
  int64_t base;                // its first place
  PaSeq seq;
  // the part: unit and its tiles' places [ts, ue), of which this block does those up to `end`; visible
  // positions [t0, t1)
  int unit;
  int64_t ts, ue, end;
  int t0, t1;
};

// least: tiles that a block can do at once; no unit is cut into smaller parts, which would only add
// joining.
template <int TILE>
__device__ __forceinline__ bool pa_begin(const PagedAttnParams& p, int least, PaWork& w) {
  __shared__ int64_t s_scan[PA_MAX_WARPS];
  __shared__ int64_t s_found[2];
  auto length = [&](int b) { return b < p.kv.batch ? int64_t(pa_seq<TILE>(p, b).tiles + PA_PART_COST) * p.units : 0; };
  // where the sequence of this thread begins (of the last chunk of sequences, if there are many)
  int64_t mine = 0, before = 0, sum = 0;
  w.total = 0;
  for (int b0 = 0; b0 < p.kv.batch; b0 += blockDim.x) {
    mine = length(b0 + threadIdx.x);
    sum = pa_scan(mine, before, s_scan);
    w.total += sum;
  }
  const int64_t apart = max(int64_t(p.kv.batch) * p.units, pa_quot(w.total, least));
  w.blocks = min(min(int64_t(gridDim.x), w.total), apart);
  if (blockIdx.x >= w.blocks) return false;
  w.lo = w.cur = pa_lo(w.total, blockIdx.x, w.blocks);
  w.hi = pa_lo(w.total, blockIdx.x + 1, w.blocks);
  int64_t run = 0;
  for (int b0 = 0; b0 < p.kv.batch; b0 += blockDim.x) {
    if (p.kv.batch > int(blockDim.x)) {
      mine = length(b0 + threadIdx.x);
      sum = pa_scan(mine, before, s_scan);
    }
    if (run + before <= w.lo && w.lo < run + before + mine) {
      s_found[0] = b0 + threadIdx.x;
      s_found[1] = run + before;
    }
    run += sum;
  }
  __syncthreads();
  w.b = int(s_found[0]);
  w.base = s_found[1];
  w.seq = pa_seq<TILE>(p, w.b);
  return true;
}

template <int TILE>
__device__ __forceinline__ bool pa_part(const PagedAttnParams& p, PaWork& w) {
  while (w.cur < w.hi) {
    int64_t per = w.seq.tiles + PA_PART_COST;
    while (w.cur >= w.base + per * p.units) {
      w.base += per * p.units;
      w.seq = pa_seq<TILE>(p, ++w.b);
      per = w.seq.tiles + PA_PART_COST;
    }
    const int64_t in = w.cur - w.base;
    w.unit = int(pa_quot(in, per));
    const int64_t us = w.base + w.unit * per;
    w.ts = us + PA_PART_COST;
    w.ue = us + per;
    w.end = min(w.ue, w.hi);
    const int64_t from = max(w.cur, w.ts);
    if (from < w.end) {
      w.t0 = int(from - w.ts) * TILE;
      w.t1 = min(w.seq.n, int(w.end - w.ts) * TILE);
      return true;
    }
    w.cur = w.end;      // only the empty stretch was this block's
  }
  return false;
}

// ---------------------------------------------------------------- the end of a part

// Barrier among the first n threads of the block, those that compute and join.
__device__ __forceinline__ void pa_sync(int n) { asm volatile("bar.sync 1, %0;" ::"r"(n) : "memory"); }

__device__ __forceinline__ float pa_weight(float m, float top) {
  return m == -INFINITY ? 0.0f : exp2f(m - top);   // a part without a finite score weighs nothing
}

// Floats of a triple of `rows` heads: m [rows], l [rows], a [rows][dhp] from a multiple of four on.
__host__ __device__ constexpr int pa_head(int rows) { return (2 * rows + 3) & ~3; }
__host__ __device__ constexpr int pa_triple(int rows, int dhp) { return pa_head(rows) + rows * dhp; }
// Shared memory of pa_finish in floats: a triple per warp.
__host__ __device__ constexpr int pa_finish_floats(int warps, int rows, int dhp) { return warps * pa_triple(rows, dhp); }

// Writes four values d.. of head h of sequence b from its joined triple.  l is at least about 1 (the
// largest score's weight) or 0, so its reciprocal is as good as a division to the last place or two.
__device__ __forceinline__ void pa_write4(const PagedAttnParams& p, int b, int h, int d, const float4& a, float l) {
  const float inv = l == 0.0f ? 0.0f : __frcp_rn(l);
  const float v[4] = {a.x * inv, a.y * inv, a.z * inv, a.w * inv};
  if (p.out != nullptr) {
    const int64_t at = b * p.os[0] + h * p.os[1] + d * p.os[2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < p.kv.dh) dt_store(p.out, at + i * p.os[2], p.q_dtype, v[i]);
  }
  if (p.out_i8 != nullptr) {
    const int64_t at = b * p.is[0] + h * p.is[1] + d * p.is[2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < p.kv.dh) p.out_i8[at + i * p.is[2]] = static_cast<int8_t>(quant_byte(v[i], p.q8) & 0xff);
  }
}

__device__ __forceinline__ void pa_write_lse(const PagedAttnParams& p, int b, int h, float m, float l) {
  if (p.lse != nullptr)
    p.lse[int64_t(b) * p.heads + h] = l == 0.0f ? -INFINITY : fmaf(m, 0.693147180559945309f, logf(l));
}

__device__ __forceinline__ void pa_add4(float4& a, const float4& x, float w) {
  a.x = fmaf(x.x, w, a.x);
  a.y = fmaf(x.y, w, a.y);
  a.z = fmaf(x.z, w, a.z);
  a.w = fmaf(x.w, w, a.w);
}

// Where value 4 d4 of head h is in a triple in shared memory: groups of four are permuted so that the
// warps' stores fall on different banks.
template <int DHP>
__device__ __forceinline__ int pa_at(int rows, int h, int d4) { return pa_head(rows) + h * DHP + (d4 ^ (h >> 1 & 3)) * 4; }

// Joins the warps' triples of this part (sm: one triple per warp, `rows` of them used) and either
// writes the result, when the block had the whole unit, or leaves the joined triple in the block's
// slot; the last block of the unit to do so joins them all.  The block's first `warps` warps call it.
// h0: first of the unit's `live` heads.
template <int DHP>
__device__ __forceinline__ void pa_finish(const PagedAttnParams& p, const PaWork& w, float* sm, int warps, int rows, int h0, int live) {
  __shared__ int s_last;
  const int threads = warps * 32, triple = pa_triple(rows, DHP);
  pa_sync(threads);
  const bool whole = w.lo <= w.ts && w.ue <= w.hi;
  auto slot_of = [&](int64_t c) { return p.part + (c * 2 + (pa_lo(w.total, c, w.blocks) >= w.ts ? 0 : 1)) * triple; };
  float* mine = p.part + (int64_t(blockIdx.x) * 2 + (w.lo >= w.ts ? 0 : 1)) * triple;
  for (int e = threadIdx.x; e < live * (DHP / 4); e += threads) {
    const int g = e / (DHP / 4), d4 = e - g * (DHP / 4), d = d4 * 4;
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float top = -INFINITY, sum = 0.0f;
#pragma unroll 4
    for (int i = 0; i < warps; ++i) top = fmaxf(top, sm[i * triple + g]);
#pragma unroll 4
    for (int i = 0; i < warps; ++i) {
      const float* from = sm + i * triple;
      const float wt = pa_weight(from[g], top);
      sum += from[rows + g] * wt;
      pa_add4(a, *reinterpret_cast<const float4*>(from + pa_at<DHP>(rows, g, d4)), wt);
    }
    if (whole) {
      pa_write4(p, w.b, h0 + g, d, a, sum);
      if (d == 0) pa_write_lse(p, w.b, h0 + g, top, sum);
    } else {
      *reinterpret_cast<float4*>(mine + pa_head(rows) + g * DHP + d) = a;
      if (d == 0) {
        mine[g] = top;
        mine[rows + g] = sum;
      }
    }
  }
  if (whole) {
    pa_sync(threads);     // the triples are free again
    return;
  }
  const int first = pa_block_of(w.total, w.ts, w.blocks), last = pa_block_of(w.total, w.ue - 1, w.blocks);
  pa_sync(threads);
  int* counter = p.counters + first;      // of the units that a block begins only its last goes on in the next
  if (threadIdx.x == 0) {
    __threadfence();      // the whole block's slot, by the barrier before
    s_last = atomicAdd(counter, 1) == last - first;
  }
  pa_sync(threads);
  if (s_last) {
    __threadfence();
    // all but the first part start at their block's first tile, so they are in slot 0
    const float* from = slot_of(first);
    const float* next = p.part + (int64_t(first) + 1) * 2 * triple;
    const int n = last - first + 1;
    auto part = [&](int i) { return i == 0 ? from : next + int64_t(i - 1) * 2 * triple; };
    float* j_m = sm;
    float* j_l = sm + rows;
    float* wts = sm + pa_head(rows);                  // [n][live] weights, if they fit
    const bool fits = n * live <= warps * triple - pa_head(rows);
    // a warp per head: the largest m, then the sum
    for (int g = threadIdx.x >> 5; g < live; g += warps) {
      const int lane = threadIdx.x & 31;
      float top = -INFINITY, sum = 0.0f;
      // m and l of up to 64 parts at once, the rest (if any) one by one
      float m[2], l[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i = lane + 32 * u;
        m[u] = i < n ? __ldcg(part(i) + g) : -INFINITY;
        l[u] = i < n ? __ldcg(part(i) + rows + g) : 0.0f;
        top = fmaxf(top, m[u]);
      }
      for (int i = lane + 64; i < n; i += 32) top = fmaxf(top, __ldcg(part(i) + g));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i = lane + 32 * u;
        const float wt = pa_weight(m[u], top);
        if (fits && i < n) wts[i * live + g] = wt;
        sum += l[u] * wt;
      }
      for (int i = lane + 64; i < n; i += 32) {
        const float wt = pa_weight(__ldcg(part(i) + g), top);
        if (fits) wts[i * live + g] = wt;
        sum += __ldcg(part(i) + rows + g) * wt;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) {
        j_m[g] = top;
        j_l[g] = sum;
        pa_write_lse(p, w.b, h0 + g, top, sum);
      }
    }
    pa_sync(threads);
    constexpr int FLY = 16;      // loads in flight
    for (int e = threadIdx.x; e < live * (DHP / 4); e += threads) {
      const int g = e / (DHP / 4), d = (e - g * (DHP / 4)) * 4;
      float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const float top = j_m[g];
      for (int i = 0; i < n; i += FLY) {
        float4 x[FLY];
#pragma unroll
        for (int u = 0; u < FLY; ++u)
          x[u] = i + u < n ? __ldcg(reinterpret_cast<const float4*>(part(i + u) + pa_head(rows) + g * DHP + d))
                           : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int u = 0; u < FLY; ++u)
          if (i + u < n) pa_add4(a, x[u], fits ? wts[(i + u) * live + g] : pa_weight(__ldcg(part(i + u) + g), top));
      }
      pa_write4(p, w.b, h0 + g, d, a, j_l[g]);
    }
    if (threadIdx.x == 0) *counter = 0;
  }
  pa_sync(threads);     // the triples are free again
}

// ---------------------------------------------------------------- rows in flight

// What hides the memory's latency is bytes in flight, about 64 KB per SM at full bandwidth, at all times:
// also while a part is being joined and the next one begins.  A quarter to a half of a block's warps
// therefore only look rows up and copy them (cp.async, mostly 16 bytes a lane) to shared memory, through all of
// the block's parts.  Each computing warp has a ring of its own, filled by one copying warp, so that both
// sides of a ring take its slots in the same order and a barrier's parity always tells the round that is
// meant.  (With one ring for all, a warp could be two rounds from another: the parity of the wrong one then
// passes for the right one.)  The pieces lie in the order of the lanes that will use them (piece j of lane l
// at (32 j + l) * size), free of bank conflicts.
struct PaRing {
  uint8_t* steps;            // [computing warp][slot]
  uint64_t* full;            // per slot: its copies and `live` are there
  uint64_t* empty;           // per slot: its warp is done with it
  uint32_t* live;            // per slot: tokens of the step that count
  int slots;                 // of a warp
  int* abort;                // a wait gave up: nothing is right any more, but every barrier is still met
};

// Slots have a head of 32 bytes: full, empty, live.
__host__ __device__ constexpr int pa_ring_bytes(int slots, int step) { return slots * (step + 32); }

constexpr uint64_t PA_WAIT_NS = 2000000000ull;

// Every lane of the copying warp arrives on `full` when its copies have landed, and its lane 0 once more
// for `live`; the warp that used a step arrives on `empty`.
__device__ __forceinline__ PaRing pa_ring_at(uint8_t* at, int warps, int slots, int step, int* abort) {
  PaRing r;
  const int n = warps * slots;
  r.steps = at;
  r.full = reinterpret_cast<uint64_t*>(at + int64_t(n) * step);
  r.empty = r.full + n;
  r.live = reinterpret_cast<uint32_t*>(r.empty + n);
  r.slots = slots;
  r.abort = abort;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    mbar_init(r.full + i, 33);
    mbar_init(r.empty + i, 1);
  }
  if (threadIdx.x == 0) *abort = 0;
  fence_mbar_init();
  __syncthreads();
  return r;
}

__device__ __forceinline__ void pa_wait(const PaRing& r, uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity) || *reinterpret_cast<volatile int*>(r.abort)) return;
  mbar_wait(bar, parity, r.abort, PA_WAIT_NS);
}

// A place in a warp's ring: slot and the parity of its round.
struct PaPlace {
  int slot;
  uint32_t round;
  __device__ __forceinline__ void forward(int slots) {
    if (++slot == slots) {
      slot = 0;
      round ^= 1;
    }
  }
};

// One token of a step, held by one lane: its page and slot.  The page id is on its way while the step before is
// copied; nothing looks at it until then.
struct PaToken {
  int page, slot;
  bool in;            // a visible token
};

__device__ __forceinline__ PaToken pa_token(const PagedAttnParams& p, const PaWork& w, int i, bool mine) {
  PaToken t;
  t.in = mine && i < w.t1;
  const int pos = i + (i < w.seq.sinks ? 0 : w.seq.skip), at = qg_div(pos, p.kv.page_div);
  t.slot = pos - at * p.kv.page_size;
  t.page = 0;
  if (t.in) t.page = __ldg(p.kv.table + w.b * p.kv.table_ld + at);
  return t;
}

// Where its rows are, as byte offsets in the pages; not ok if it is none or the table names no page of the pool.
struct PaRows {
  int64_t k, v;
  bool ok;
};

template <typename T>
__device__ __forceinline__ PaRows pa_rows(const PagedAttnParams& p, PaToken& t) {
  PaRows r;
  r.ok = t.in && static_cast<uint32_t>(t.page) < static_cast<uint32_t>(p.kv.num_pages);
  if (t.in && !r.ok) atomicExch(p.kv.err, PAGED_ERR);
  if (!r.ok) t.page = t.slot = 0;
  r.k = (t.page * p.kv.kst[0] + t.slot * p.kv.kst[2]) * int(sizeof(T));
  r.v = (t.page * p.kv.vst[0] + t.slot * p.kv.vst[2]) * int(sizeof(T));
  return r;
}

// n: BYTES, or 0 for zeros, when nothing is read.
template <int BYTES>
__device__ __forceinline__ void pa_copy(uint32_t dst, const uint8_t* src, uint32_t n) {
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(BYTES) : "memory");
}

__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The steps of all of a block's parts are numbered through; step n is for computing warp n modulo their number.
// Copying warp `me` of `feeders`, which divide the computing warps, does steps me, me + feeders, .., i.e. fills
// the rings of computing warps me, me + feeders, ..  copy(w, tokens, step) issues the copies of the tokens into
// a slot and returns which of them count.  A step has to be copied in about 1000 clocks for the memory to stay
// busy (one copying warp of eight: twice the time), so that little may be worked out per step: the page ids
// come a step ahead, and full steps are copied without a look at each token (48 x 20/4 heads of 80 up to 8000,
// bf16: 72.2 -> 68.1 us).
__device__ __forceinline__ int pa_steps(const PaWork& w, int tile) { return w.t1 > w.t0 ? (w.t1 - w.t0 - 1) / tile + 1 : 0; }

template <int TILE, class Copy>
__device__ __forceinline__ void pa_feed(const PagedAttnParams& p, PaWork& w, const PaRing& ring, int step_bytes, int me, int feeders,
                                        int warps, Copy copy) {
  const int lane = threadIdx.x & 31;
  PaPlace place{0, 0};
  int to = me, mine = me;      // the next computing warp; this warp's next step, from the part's first
  while (pa_part<TILE>(p, w)) {
    const int steps = pa_steps(w, TILE);
    PaToken next = pa_token(p, w, w.t0 + mine * TILE + lane, lane < TILE);
    for (; mine < steps; mine += feeders) {
      const PaToken tokens = next;
      next = pa_token(p, w, w.t0 + (mine + feeders) * TILE + lane, lane < TILE);
      const int at = to * ring.slots + place.slot;
      pa_wait(ring, ring.empty + at, place.round ^ 1);       // the first round finds every slot empty
      __syncwarp();
      const uint32_t live = copy(w, tokens, ring.steps + int64_t(at) * step_bytes);
      cp_async_arrive_noinc(ring.full + at);
      if (lane == 0) {
        ring.live[at] = live;
        mbar_arrive(ring.full + at);
      }
      to += feeders;
      if (to >= warps) {
        to = me;
        place.forward(ring.slots);
      }
    }
    mine -= steps;
    w.cur = w.end;
  }
  cp_async_commit();
  cp_async_wait<0>();
}

// ---------------------------------------------------------------- f32 pages

// DHP: head dimension rounded up to 32, 64, 128 or 256; GP: query heads that share a pass over the rows.
// Bound: the visible rows are read once, 8 dh bytes a token and head; a score and its value row take 4 dh
// operations, which the FMA units do in the shadow of the loads for one query head per key head and
// no longer for four.  (Products on the tensor path need three bf16 values per element of k and v: six
// bytes for four, and six products for one.)
// A row is spread over LPR lanes, 16 bytes each, a warp takes TPS rows at a time and U times that in a
// step.  The LPR partial sums of the step's U GP scores are added crosswise, each exchange halving the
// number of scores a lane carries, so that a score's softmax is worked out in few lanes, not in all.
// 64 sequences of up to 1024 tokens, 12 heads of 64 (205 MB): 44.3 us, 4.6 TB/s; what is above the bytes' 31 us
// is mostly the launch, the dealing out, and the beginnings and ends of the 768 units' parts.
template <int DHP, int GP>
struct PaF32 {
  static constexpr int LPR = DHP / 4 < 32 ? DHP / 4 : 32;
  static constexpr int NV = DHP / (4 * LPR);
  static constexpr int EPL = 4 * NV;
  static constexpr int TPS = 32 / LPR;
  static constexpr int U = NV > 1 ? 4 : 8;
  static constexpr int TILE = TPS * U;                      // rows of a step
  static constexpr int STEP = 2 * U * NV * 512;
  static constexpr int N = U * GP;                          // scores of a lane group
  static constexpr int HALVINGS = N <= LPR ? (N == 4 ? 2 : N == 8 ? 3 : N == 16 ? 4 : 5) : (LPR == 8 ? 3 : LPR == 16 ? 4 : 5);
  static constexpr int LEFT = N >> HALVINGS;                // scores a lane ends up with
  static constexpr int WIDTH = LPR >> HALVINGS;             // lanes that end up with the same scores
  static constexpr int WARPS = GP * EPL <= 8 ? 16 : 12;     // of an SM
  // as many copying as computing warps: with one query head a step is copied about as fast as it is used (64 x 12
  // heads of 64 up to 1024 tokens: 44.3 us, with six computing and two copying warps 47.3)
  static constexpr bool EVEN = GP == 1;
};

template <int DHP, int GP>
__global__ void __launch_bounds__(PaF32<DHP, GP>::WARPS * 32, 1)
    paged_attention_f32_kernel(const __grid_constant__ PagedAttnParams p) {
  using C = PaF32<DHP, GP>;
  extern __shared__ __align__(128) uint8_t pa_smem[];       // ring, then the warps' triples
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, feeders = p.feeders, warps = (blockDim.x >> 5) - feeders;
  const int sub = lane % C::LPR, group0 = lane - sub, row0 = lane / C::LPR;
  float* sm = reinterpret_cast<float*>(pa_smem + pa_ring_bytes(warps * p.slots, C::STEP));
  PaWork w;
  if (!pa_begin<C::TILE>(p, warps, w)) return;
  const PaRing ring = pa_ring_at(pa_smem, warps, p.slots, C::STEP, &s_abort);

  if (warp >= warps) {
    uint32_t size[C::NV];        // of this lane's accesses of a row
#pragma unroll
    for (int j = 0; j < C::NV; ++j) size[j] = (sub + j * C::LPR) * 4 < p.kv.dh ? 16 : 0;
    auto copy = [&](const PaWork& w, PaToken tokens, uint8_t* step) {
      const PaRows tok = pa_rows<float>(p, tokens);
      const int kvh = w.unit / p.head_blocks;
      const uint8_t* kb = reinterpret_cast<const uint8_t*>(static_cast<const float*>(p.kv.k) + kvh * p.kv.kst[1] + sub * 4);
      const uint8_t* vb = reinterpret_cast<const uint8_t*>(static_cast<const float*>(p.kv.v) + kvh * p.kv.vst[1] + sub * 4);
      const uint32_t live = __ballot_sync(0xffffffffu, tok.ok);
      const uint32_t dst = smem_u32(step) + lane * 16;
      auto rows = [&](auto full) {
#pragma unroll
        for (int u = 0; u < C::U; ++u) {
          const int i = u * C::TPS + row0;
          const uint8_t* k = kb + __shfl_sync(0xffffffffu, tok.k, i);
          const uint8_t* v = vb + __shfl_sync(0xffffffffu, tok.v, i);
          const bool in = decltype(full)::value || (live >> i & 1);
#pragma unroll
          for (int j = 0; j < C::NV; ++j) {
            pa_copy<16>(dst + (u * C::NV + j) * 512, k + j * C::LPR * 16, in ? size[j] : 0);
            pa_copy<16>(dst + ((C::U + u) * C::NV + j) * 512, v + j * C::LPR * 16, in ? size[j] : 0);
          }
        }
      };
      if (live == uint32_t((uint64_t(1) << C::TILE) - 1)) rows(std::true_type{});
      else rows(std::false_type{});
      return live;
    };
    pa_feed<C::TILE>(p, w, ring, C::STEP, warp - warps, feeders, warps, copy);
    if (lane == 0 && s_abort) atomicExch(p.kv.err, 1);
    return;
  }

  PaPlace mine{0, 0};
  int next = warp;      // this warp's next step, from the part's first
  while (pa_part<C::TILE>(p, w)) {
    const int kvh = w.unit / p.head_blocks, g0 = (w.unit - kvh * p.head_blocks) * GP;
    const int steps = pa_steps(w, C::TILE);

    float q[GP][C::EPL], acc[GP][C::EPL], m[GP], l[C::LEFT];
#pragma unroll
    for (int gi = 0; gi < GP; ++gi) {
      m[gi] = -INFINITY;
#pragma unroll
      for (int e = 0; e < C::EPL; ++e) {
        const int d = (sub + (e / 4) * C::LPR) * 4 + e % 4;
        q[gi][e] = (g0 + gi < p.group && d < p.kv.dh)
            ? dt_load(p.q, w.b * p.qs[0] + (kvh * p.group + g0 + gi) * p.qs[1] + d * p.qs[2], p.q_dtype) * p.scale_log2
            : 0.0f;
        acc[gi][e] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < C::LEFT; ++i) l[i] = 0.0f;

    // this lane's scores are first .. first + LEFT - 1 of its group's rows, score u GP + gi
    const int first = sub / C::WIDTH * C::LEFT;
    for (; next < steps; next += warps) {
      const int slot = warp * ring.slots + mine.slot;
      pa_wait(ring, ring.full + slot, mine.round);
      const uint32_t now = ring.live[slot];
      const uint8_t* rows = ring.steps + int64_t(slot) * C::STEP + lane * 16;

      float s[C::N];
#pragma unroll
      for (int u = 0; u < C::U; ++u) {
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) s[u * GP + gi] = 0.0f;
#pragma unroll
        for (int j = 0; j < C::NV; ++j) {
          const float4 x = *reinterpret_cast<const float4*>(rows + (u * C::NV + j) * 512);
#pragma unroll
          for (int gi = 0; gi < GP; ++gi) {
            float& y = s[u * GP + gi];
            y = fmaf(q[gi][4 * j], x.x, y);
            y = fmaf(q[gi][4 * j + 1], x.y, y);
            y = fmaf(q[gi][4 * j + 2], x.z, y);
            y = fmaf(q[gi][4 * j + 3], x.w, y);
          }
        }
      }
      // exchange h: the lanes with bit LPR / 2^(h + 1) keep the upper half of the scores
#pragma unroll
      for (int h = 0; h < C::HALVINGS; ++h) {
        const int o = C::LPR >> (h + 1), half = C::N >> (h + 1);
        const bool upper = sub & o;
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const float give = upper ? s[i] : s[i + half], keep = upper ? s[i + half] : s[i];
          s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
#pragma unroll
      for (int o = C::WIDTH / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < C::LEFT; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
#pragma unroll
      for (int i = 0; i < C::LEFT; ++i) {
        const int u = (first + i) / GP;
        if (!(now >> (u * C::TPS + row0) & 1)) s[i] = -INFINITY;
      }
      // the largest of each head, in all lanes of the group
      float top[GP];
#pragma unroll
      for (int gi = 0; gi < GP; ++gi) top[gi] = m[gi];
      if (C::LEFT == 1) {
        float x = s[0];       // lanes whose score index agrees mod GP share a head
#pragma unroll
        for (int o = C::LPR / 2; o >= GP * C::WIDTH; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
#pragma unroll
        for (int gi = 0; gi < GP; ++gi)
          top[gi] = fmaxf(top[gi], GP == 1 ? x : __shfl_sync(0xffffffffu, x, group0 + gi * C::WIDTH));
      } else {
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) {
          float x = -INFINITY;
#pragma unroll
          for (int i = 0; i < C::LEFT; ++i)
            if ((first + i) % GP == gi) x = fmaxf(x, s[i]);
#pragma unroll
          for (int o = 1; o < C::LPR; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
          top[gi] = fmaxf(top[gi], x);
        }
      }
      bool moved = false;
#pragma unroll
      for (int gi = 0; gi < GP; ++gi) moved = moved || top[gi] > m[gi];
      if (__any_sync(0xffffffffu, moved)) {
        float fade[GP];
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) {
          fade[gi] = pa_exp2(m[gi] - (top[gi] == -INFINITY ? 0.0f : top[gi]));
          m[gi] = top[gi];
#pragma unroll
          for (int e = 0; e < C::EPL; ++e) acc[gi][e] *= fade[gi];
        }
#pragma unroll
        for (int i = 0; i < C::LEFT; ++i) {
          float f = fade[0];
#pragma unroll
          for (int gi = 1; gi < GP; ++gi) f = (first + i) % GP == gi ? fade[gi] : f;
          l[i] *= f;
        }
      }
#pragma unroll
      for (int i = 0; i < C::LEFT; ++i) {
        float z = m[0];
#pragma unroll
        for (int gi = 1; gi < GP; ++gi) z = (first + i) % GP == gi ? m[gi] : z;
        s[i] = pa_exp2(s[i] - (z == -INFINITY ? 0.0f : z));
        l[i] += s[i];
      }
#pragma unroll
      for (int u = 0; u < C::U; ++u) {
        float pr[GP];
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) {
          const int n = u * GP + gi;
          pr[gi] = __shfl_sync(0xffffffffu, s[n % C::LEFT], group0 + n / C::LEFT * C::WIDTH);
        }
#pragma unroll
        for (int j = 0; j < C::NV; ++j) {
          const float4 x = *reinterpret_cast<const float4*>(rows + ((C::U + u) * C::NV + j) * 512);
#pragma unroll
          for (int gi = 0; gi < GP; ++gi) {
            acc[gi][4 * j] = fmaf(pr[gi], x.x, acc[gi][4 * j]);
            acc[gi][4 * j + 1] = fmaf(pr[gi], x.y, acc[gi][4 * j + 1]);
            acc[gi][4 * j + 2] = fmaf(pr[gi], x.z, acc[gi][4 * j + 2]);
            acc[gi][4 * j + 3] = fmaf(pr[gi], x.w, acc[gi][4 * j + 3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(ring.empty + slot);
      mine.forward(ring.slots);
    }
    next -= steps;

    // l of each head: the lanes' sums of its scores
    float lsum[GP];
#pragma unroll
    for (int gi = 0; gi < GP; ++gi) {
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < C::LEFT; ++i)
        if ((first + i) % GP == gi) x += l[i];
#pragma unroll
      for (int o = C::WIDTH; o < C::LPR; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      lsum[gi] = x;
    }
    float* to = sm + warp * pa_triple(GP, DHP);
#pragma unroll
    for (int gi = 0; gi < GP; ++gi) {
#pragma unroll
      for (int o = C::LPR; o < 32; o <<= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m[gi], o), lo = __shfl_xor_sync(0xffffffffu, lsum[gi], o);
        const float top = fmaxf(m[gi], mo);
        const float wa = pa_weight(m[gi], top), wb = pa_weight(mo, top);
        lsum[gi] = lsum[gi] * wa + lo * wb;
        m[gi] = top;
#pragma unroll
        for (int e = 0; e < C::EPL; ++e)
          acc[gi][e] = acc[gi][e] * wa + __shfl_xor_sync(0xffffffffu, acc[gi][e], o) * wb;
      }
      if (row0 == 0) {
#pragma unroll
        for (int j = 0; j < C::NV; ++j)
          *reinterpret_cast<float4*>(to + pa_at<DHP>(GP, gi, sub + j * C::LPR)) =
              make_float4(acc[gi][4 * j], acc[gi][4 * j + 1], acc[gi][4 * j + 2], acc[gi][4 * j + 3]);
      }
      if (lane == 0) {
        to[gi] = m[gi];
        to[GP + gi] = lsum[gi];
      }
    }
    pa_finish<DHP>(p, w, sm, warps, GP, kvh * p.group + g0, min(GP, p.group - g0));
    w.cur = w.end;
  }
  if (threadIdx.x == 0 && s_abort) atomicExch(p.kv.err, 1);
}

// ---------------------------------------------------------------- rows that are not 16-byte aligned

// One element per access, eight a lane (the head dimension is taken as 256), two rows of a warp in flight;
// each query head reads the rows anew (the repeats come from the caches).  Right for every stride and
// size, and slow, bound by its narrow loads: 16-byte aligned rows go to the other kernels.
struct PaAny {
  static constexpr int WARPS = 8, EPL = 8, DHP = 32 * EPL, U = 2, TILE = WARPS * U;
  static constexpr int SMEM = pa_finish_floats(WARPS, 1, DHP) * 4;
};

template <typename T>
__global__ void __launch_bounds__(PaAny::WARPS * 32) paged_attention_any_kernel(const __grid_constant__ PagedAttnParams p) {
  using C = PaAny;
  constexpr bool I8 = sizeof(T) == 1;
  extern __shared__ __align__(16) float pa_floats[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  PaWork w;
  if (!pa_begin<C::TILE>(p, 1, w)) return;
  while (pa_part<C::TILE>(p, w)) {
    const int kvh = w.unit / p.head_blocks, h = kvh * p.group + (w.unit - kvh * p.head_blocks);
    float q[C::EPL], acc[C::EPL], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < C::EPL; ++e) {
      const int d = lane + 32 * e;
      q[e] = d < p.kv.dh ? dt_load(p.q, w.b * p.qs[0] + h * p.qs[1] + d * p.qs[2], p.q_dtype) * p.scale_log2 : 0.0f;
      acc[e] = 0.0f;
    }
    const int32_t* trow = p.kv.table + w.b * p.kv.table_ld;
    const T* kb = static_cast<const T*>(p.kv.k) + kvh * p.kv.kst[1];
    const T* vb = static_cast<const T*>(p.kv.v) + kvh * p.kv.vst[1];
    for (int i0 = w.t0 + warp * C::U; i0 < w.t1; i0 += C::TILE) {
      T k[C::U][C::EPL], v[C::U][C::EPL];
      float ks[C::U], vs[C::U];
      bool ok[C::U];
#pragma unroll
      for (int u = 0; u < C::U; ++u) {
        const int i = i0 + u;
        int page = 0, slot = 0;
        ok[u] = i < w.t1 && paged_slot(p.kv, trow, i + (i < w.seq.sinks ? 0 : w.seq.skip), page, slot);
        const T* kp = kb + page * p.kv.kst[0] + slot * p.kv.kst[2];
        const T* vp = vb + page * p.kv.vst[0] + slot * p.kv.vst[2];
#pragma unroll
        for (int e = 0; e < C::EPL; ++e) {
          const int d = lane + 32 * e;
          const bool in = ok[u] && d < p.kv.dh;
          k[u][e] = in ? kp[d] : T{};
          v[u][e] = in ? vp[d] : T{};
        }
        if (I8) {
          ks[u] = ok[u] ? p.kv.ks[page * p.kv.kss[0] + kvh * p.kv.kss[1] + slot * p.kv.kss[2]] : 0.0f;
          vs[u] = ok[u] ? p.kv.vs[page * p.kv.vss[0] + kvh * p.kv.vss[1] + slot * p.kv.vss[2]] : 0.0f;
        }
      }
      float s[C::U], top = m;
#pragma unroll
      for (int u = 0; u < C::U; ++u) {
        s[u] = 0.0f;
#pragma unroll
        for (int e = 0; e < C::EPL; ++e) s[u] = fmaf(q[e], static_cast<float>(k[u][e]), s[u]);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
        if (I8) s[u] *= ks[u];
        if (!ok[u]) s[u] = -INFINITY;
        top = fmaxf(top, s[u]);
      }
      const float safe = top == -INFINITY ? 0.0f : top, fade = exp2f(m - safe);
      m = top;
      l *= fade;
#pragma unroll
      for (int e = 0; e < C::EPL; ++e) acc[e] *= fade;
#pragma unroll
      for (int u = 0; u < C::U; ++u) {
        float x = exp2f(s[u] - safe);
        l += x;
        if (I8) x *= vs[u];
#pragma unroll
        for (int e = 0; e < C::EPL; ++e) acc[e] = fmaf(x, static_cast<float>(v[u][e]), acc[e]);
      }
    }
    float* mine = pa_floats + warp * pa_triple(1, C::DHP);
#pragma unroll
    for (int e = 0; e < C::EPL; ++e) mine[pa_head(1) + lane + 32 * e] = acc[e];
    if (lane == 0) {
      mine[0] = m;
      mine[1] = l;
    }
    pa_finish<C::DHP>(p, w, pa_floats, C::WARPS, 1, h, 1);
    w.cur = w.end;
  }
}

}  // namespace mira
