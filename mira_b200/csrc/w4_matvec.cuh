// Products of a few rows with 4-bit weights under group scales:
//   y[m, n] = steps(sum_g s[n, g] sum_{k in g} x[m, k] (w[n, k] - 8)).
//
// Bound: the weights are read once, n k / 2 bytes (+ scales); everything else has to hide behind that.
// An SM's share of the memory bandwidth is about 23 bytes a clock, i.e. 46 weights a clock that must
// be unpacked and multiplied by every row of x.  FMA units need two to three instructions per weight
// and row; the tensor path needs 1.1 (f16) or 1.4 (bf16) for the unpacking and next to nothing per row: a word of eight
// weights becomes four registers of exact bf16 (or f16) pairs, which ARE the left operand's fragment
// of two 16x8x16 products (16 weight rows x 16 k).  x is the right operand, its rows in the eight
// columns: bf16 and f16 rows as they are, an f32 row as three columns whose bf16 values add up to it
// exactly, so every product is exact and sums are f32.
//
// Layout.  A warp owns 16 weight rows and walks along k in stages of 256 (16 rows x 128 bytes), brought
// to its own ring in shared memory by cp.async (rows 144 bytes apart: the fragment reads of eight rows
// then fall on different banks without address arithmetic).  A slice of 32 k is 16 bytes of a row and
// lies in one group: the products of a group's slices of a stage are summed, then added scaled.  The
// eight warps of a block are wr row tiles times 8 / wr interleaved shares of k (a remainder idles), joined in shared
// memory; x is staged in a panel, whole where it fits, k in the fragments' order.  Blocks go through
// row groups with the ring running ahead over their ends.  Where the rows alone would leave SMs idle,
// or x is wide, k is also cut over blocks (blockIdx.z); the parts are joined in order by the block
// that finishes last.
// Measured: one f16 row through 32768 x 8192, groups of 64 (143 MB): 43 to 47 us, 3.3 TB/s; 374 warp instructions per
// 2 KB of weights keep 59% of the issue slots busy, and that, not the bytes, is the limit.  16 bf16 rows through
// 4096 x 4096, groups of 128, GELU: 14.4 to 16.6 us.  768 x 768: 6.1 us, the time to launch it from the host.  Three
// blocks per SM, stages of 512 k and any fixed wr were no faster.
#pragma once
#include <cstdint>

#include "mma_sm80.cuh"
#include "paged_kv.cuh"
#include "ptx_sm100.cuh"

namespace mira {

struct W4Params {
  const void* x;
  const uint8_t* w;
  const void* scales;
  void* out;
  int64_t ld_x, ld_w, ld_scales, ld_out;
  int m, n, k, groups;
  QgDiv slices_per_group;     // group / 32
  int wr;                     // row tiles of a block: 1, 2, 4 or 8
  int panel;                  // stages of x in shared memory, a multiple of 8 / wr
  int cuts, cut_stages;       // blocks along k and the stages of each
  float* part;                // [cut][m][n] sums of each cut
  int* counters;              // [pass over x][row group], zero between calls
  int x_vec;                  // rows of x can be read 16 bytes at a time
  int x_dtype, scale_dtype, out_dtype;
  int n_steps;
  mira_epi_step steps[MIRA_EPI_MAX_STEPS];
};

// The epilogue steps on one f32 result.
__device__ __forceinline__ float w4_steps(const W4Params& p, float y, int m, int n) {
  for (int s = 0; s < p.n_steps; ++s) {
    const mira_epi_step& st = p.steps[s];
    if (st.operand == MIRA_OPND_NONE) {
      y = apply_unary(st.op, y);
      continue;
    }
    float o = st.scalar;
    if (st.operand == MIRA_OPND_CHANNEL) o = __ldg(st.ptr + n);
    else if (st.operand == MIRA_OPND_ROW) o = __ldg(st.ptr + m);
    else if (st.operand == MIRA_OPND_FULL) o = st.ptr[int64_t(m) * st.ld + n];      // may be the output itself
    y = st.swapped ? apply_binary(st.op, o, y) : apply_binary(st.op, y, o);
  }
  return y;
}

constexpr int W4_WARPS = 8;
constexpr int W4_THREADS = W4_WARPS * 32;
constexpr int W4_STAGES = 3;
constexpr int W4_STAGE_K = 256;
constexpr int W4_SLICES = W4_STAGE_K / 32;
constexpr int W4_ROW_PITCH = W4_STAGE_K / 2 + 16;     // bytes of a row of a stage in shared memory
constexpr int W4_STAGE_BYTES = 16 * W4_ROW_PITCH;
constexpr int W4_RING = W4_WARPS * W4_STAGES * W4_STAGE_BYTES;
constexpr int W4_BLOCKS = 2;                         // per SM
constexpr int W4_SMEM = 112 << 10;

// Rows of x per pass over the weights, and the columns a row takes: an f32 row is three.  Up to two
// f32 rows their columns are adjacent in one block of eight; more rows have a block per piece.
__host__ __device__ constexpr int w4_rows(int x_dtype) { return x_dtype == MIRA_DT_F32 ? 8 : 16; }
__host__ __device__ constexpr int w4_pieces(int x_dtype) { return x_dtype == MIRA_DT_F32 ? 3 : 1; }
// Bytes of a column with `stages` stages: 64 more than a multiple of 128, so that the fragment reads of
// two columns cover all banks.
__host__ __device__ constexpr int w4_pitch(int stages) { return stages * W4_STAGE_K * 2 + 64; }
// Shared memory beside the panel: the ring, two buffers of joined sums, a stage's scales per warp.
__host__ __device__ constexpr int w4_fixed(int nb, int gs) {
  return W4_RING + 2 * W4_WARPS * (nb == 3 ? 1 : nb) * 8 * 16 * 4 + W4_WARPS * (W4_SLICES / gs) * 16 * 4;
}

// (w & mask) | base as one instruction: written in C it becomes two, each with its constant inside.
__device__ __forceinline__ uint32_t w4_or(uint32_t w, uint32_t mask, uint32_t base) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(base));
  return r;
}

// A word of eight weights as four registers of pairs (w0, w4), (w1, w5), (w2, w6), (w3, w7), each
// w - 8: the nibble is or-ed under the exponent of 1024 (f16) or 128 (bf16), whose last mantissa bit
// is worth 1, and the offset is subtracted exactly; f16 has room for a nibble shifted by four.  The
// constants are held in registers: the compiler would set them anew before every use.
template <bool BF16>
struct W4Unpack {
  uint32_t low, high, base, off, sixteenth, off16;
  __device__ __forceinline__ static uint32_t pin(uint32_t v) {
    uint32_t r;
    asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
    return r;
  }
  __device__ __forceinline__ W4Unpack()
      : low(pin(0x000f000fu)), high(pin(0x00f000f0u)), base(pin(BF16 ? 0x43004300u : 0x64006400u)),
        off(pin(BF16 ? 0x43084308u : 0x64086408u)),                  // 136 or 1032
        sixteenth(pin(0x2c002c00u)), off16(pin(0xd480d480u)) {}       // f16: 1 / 16, -72
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t (&a)[4]) const {
    if (BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = b2_bits(__hsub2(bits_b2(w4_or(w >> (4 * i), low, base)), bits_b2(off)));
    } else {
      const uint32_t v = w >> 8;
      a[0] = h2_bits(__hsub2(bits_h2(w4_or(w, low, base)), bits_h2(off)));
      a[1] = h2_bits(__hfma2(bits_h2(w4_or(w, high, base)), bits_h2(sixteenth), bits_h2(off16)));
      a[2] = h2_bits(__hsub2(bits_h2(w4_or(v, low, base)), bits_h2(off)));
      a[3] = h2_bits(__hfma2(bits_h2(w4_or(v, high, base)), bits_h2(sixteenth), bits_h2(off16)));
    }
  }
};

// Eight values of a row of x from element k on (0 past the end), as they are: f32 in eight words, 16-bit
// values in four.
template <int XT>
__device__ __forceinline__ void w4_load_x(const W4Params& p, int row, int k, uint32_t (&v)[XT == MIRA_DT_F32 ? 8 : 4]) {
  if constexpr (XT == MIRA_DT_F32) {
    const uint32_t* src = static_cast<const uint32_t*>(p.x) + row * p.ld_x + k;
    if (p.x_vec && k + 8 <= p.k) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(src)), b = __ldg(reinterpret_cast<const uint4*>(src) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = k + i < p.k ? __ldg(src + i) : 0u;
    }
  } else {
    const uint16_t* src = static_cast<const uint16_t*>(p.x) + row * p.ld_x + k;
    if (p.x_vec && k + 8 <= p.k) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(src));
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = (k + 2 * i < p.k ? uint32_t(__ldg(src + 2 * i)) : 0u) |
               (k + 2 * i + 1 < p.k ? uint32_t(__ldg(src + 2 * i + 1)) << 16 : 0u);
    }
  }
}

// The same in the order of the fragments, to a column of the panel (f32: to its three columns).
template <int XT>
__device__ __forceinline__ void w4_store_x(const uint32_t (&v)[XT == MIRA_DT_F32 ? 8 : 4], uint8_t* col, int piece_step) {
  if constexpr (XT == MIRA_DT_F32) {
    uint32_t c[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t h0, m0, l0, h1, m1, l1;
      split3_bf16(__uint_as_float(v[i]), h0, m0, l0);
      split3_bf16(__uint_as_float(v[i + 4]), h1, m1, l1);
      c[0][i] = __byte_perm(h0, h1, 0x7632);
      c[1][i] = __byte_perm(m0, m1, 0x7632);
      c[2][i] = __byte_perm(l0, l1, 0x7632);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
      *reinterpret_cast<uint4*>(col + j * piece_step) = make_uint4(c[j][0], c[j][1], c[j][2], c[j][3]);
  } else {
    *reinterpret_cast<uint4*>(col) = make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632),
                                                __byte_perm(v[1], v[3], 0x5410), __byte_perm(v[1], v[3], 0x7632));
  }
}

// XT: type of x; NB: blocks of eight columns (3: one per piece); GS: slices whose products are summed
// before the scale is applied, a divisor of the slices of a group (EXACT: all of them).
template <int XT, int NB, int GS, bool EXACT>
__global__ void __launch_bounds__(W4_THREADS, W4_BLOCKS) w4_matvec_kernel(const __grid_constant__ W4Params p) {
  constexpr bool BF16 = XT != MIRA_DT_F16;
  constexpr int PIECES = w4_pieces(XT), ROWS = w4_rows(XT);
  constexpr bool SPLIT = NB == 3;                // a block of columns per piece
  constexpr int OB = SPLIT ? 1 : NB;             // blocks of columns after the pieces are added
  constexpr int NS = W4_SLICES / GS;             // scales of a row per stage
  extern __shared__ __align__(128) uint8_t w4_smem[];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wk_n = W4_WARPS / p.wr, wr = warp % p.wr, wk = warp / p.wr;
  uint8_t* ring = w4_smem + warp * (W4_STAGES * W4_STAGE_BYTES);
  float* red0 = reinterpret_cast<float*>(w4_smem + W4_RING);        // two of [warp][column][16 rows]
  float* sc = red0 + 2 * W4_WARPS * OB * 8 * 16 + warp * (NS * 16);  // [scale][8][row g, row g + 8]
  uint8_t* panel = w4_smem + w4_fixed(NB, GS);
  const int pitch = w4_pitch(p.panel);
  const int m0 = blockIdx.y * ROWS, rows = min(ROWS, p.m - m0);
  const int first = blockIdx.z * p.cut_stages;                  // this block's stages along k
  const int stages = min(p.cut_stages, (p.k + W4_STAGE_K - 1) / W4_STAGE_K - first);
  const int mine = stages > wk ? (stages - wk - 1) / wk_n + 1 : 0;
  const int row_groups = (p.n + p.wr * 16 - 1) / (p.wr * 16);
  const int rounds = (row_groups - int(blockIdx.x) + int(gridDim.x) - 1) / int(gridDim.x);   // row groups of this block
  auto tile_row = [&](int round) { return ((int(blockIdx.x) + round * int(gridDim.x)) * p.wr + wr) * 16; };

  // this lane's chunks of a stage: rows lane / 8 + 4 j, chunk lane % 8; rows past the last one read the
  // last one and are not used.  The ring runs ahead over the row groups' ends.
  constexpr int CHUNKS = W4_STAGE_K / 32, TURNS = 16 * CHUNKS / 32;
  const int first_byte = (first + wk) * (W4_STAGE_K / 2) + (lane % CHUNKS) * 16;
  const uint32_t to = smem_u32(ring) + (lane / CHUNKS) * W4_ROW_PITCH + (lane % CHUNKS) * 16;
  int f_round = 0, f_stage = 0, f_slot = 0;
  const uint8_t* from[TURNS];
  int64_t left = 0;      // bytes of the rows from here on
  auto aim = [&]() {
    const int n0 = tile_row(f_round);
#pragma unroll
    for (int j = 0; j < TURNS; ++j)
      from[j] = p.w + int64_t(min(n0 + lane / CHUNKS + (32 / CHUNKS) * j, p.n - 1)) * p.ld_w + first_byte;
    left = p.ld_w - first_byte;
  };
  auto fetch = [&]() {
    if (f_round < rounds && mine > 0) {
      const uint32_t dst = to + f_slot * W4_STAGE_BYTES;
      const uint32_t bytes = left > 0 ? 16u : 0u;        // past a row's end: zeros, nothing is read
#pragma unroll
      for (int j = 0; j < TURNS; ++j) {
        cp_async_16(dst + j * (32 / CHUNKS) * W4_ROW_PITCH, from[j], bytes);
        from[j] += wk_n * (W4_STAGE_K / 2);
      }
      left -= wk_n * (W4_STAGE_K / 2);
      f_slot = f_slot + 1 == W4_STAGES ? 0 : f_slot + 1;
      if (++f_stage == mine) {
        f_stage = 0;
        if (++f_round < rounds) aim();
      }
    }
    cp_async_commit();
  };
  aim();
#pragma unroll
  for (int i = 0; i < W4_STAGES - 1; ++i) fetch();

  // scales of a stage: lane has row lane / 2, every second of the NS scales; read a stage ahead, they
  // pass through shared memory as f32.  Past the last group x is zero and so is the scale.
  constexpr int PER = (NS + 1) / 2;
  uint32_t next[PER];
  int64_t srow = 0;
  auto scales = [&](int kb) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int s = (lane & 1) + 2 * j;
      const int gi = EXACT ? kb * NS + s : qg_div(kb * W4_SLICES + s * GS, p.slices_per_group);
      next[j] = s < NS && gi < p.groups ? dt_load_raw(p.scales, srow + gi, p.scale_dtype) : 0u;
    }
  };
  auto aim_scales = [&](int round) { srow = int64_t(min(tile_row(round) + (lane >> 1), p.n - 1)) * p.ld_scales; };
  aim_scales(0);
  scales(first + wk);

  int col[NB];       // this lane's columns; those past the last row of x repeat it and are not used
#pragma unroll
  for (int b = 0; b < NB; ++b)
    col[b] = SPLIT ? (b * rows + min(g, rows - 1)) * pitch : min(b * 8 + g, rows * PIECES - 1) * pitch;
  const int row_step = SPLIT ? pitch : PIECES * pitch, piece_step = SPLIT ? rows * pitch : pitch;
  const W4Unpack<BF16> unpack;
  int slot = 0;

  for (int round = 0; round < rounds; ++round) {
    const int n0 = tile_row(round);
    float acc[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[b][i] = 0.0f;

    int i = 0;
    for (int p0 = 0; p0 < stages; p0 += p.panel) {
      const int in_panel = min(p.panel, stages - p0);
      if (round == 0 || p.panel < stages) {       // else all of x is there already
        __syncthreads();
        const int words = in_panel * (W4_STAGE_K / 8), total = rows * words;
        constexpr int FLY = XT == MIRA_DT_F32 ? 2 : 4;        // loads in flight
        for (int e0 = threadIdx.x; e0 < total; e0 += FLY * W4_THREADS) {
          uint32_t v[FLY][XT == MIRA_DT_F32 ? 8 : 4];
#pragma unroll
          for (int u = 0; u < FLY; ++u) {
            const int e = e0 + u * W4_THREADS, r = e / words;
            if (e < total) w4_load_x<XT>(p, m0 + r, (first + p0) * W4_STAGE_K + (e - r * words) * 8, v[u]);
          }
#pragma unroll
          for (int u = 0; u < FLY; ++u) {
            const int e = e0 + u * W4_THREADS, r = e / words;
            if (e < total) w4_store_x<XT>(v[u], panel + r * row_step + (e - r * words) * 16, piece_step);
          }
        }
        __syncthreads();
      }
      for (; i < mine && wk + i * wk_n < p0 + in_panel; ++i) {
        const int kb = wk + i * wk_n;
        cp_async_wait<W4_STAGES - 2>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int s = (lane & 1) + 2 * j;
          if (s < NS) sc[s * 16 + ((lane >> 1) & 7) * 2 + (lane >> 4)] = dt_from_raw(next[j], p.scale_dtype);
        }
        fetch();
        const bool ends = i + 1 == mine;
        if (ends) aim_scales(round + 1);
        scales(first + (ends ? wk : kb + wk_n));
        __syncwarp();
        const uint8_t* st = ring + slot * W4_STAGE_BYTES + g * W4_ROW_PITCH + t * 4;
        slot = slot + 1 == W4_STAGES ? 0 : slot + 1;
        const uint8_t* xs = panel + (kb - p0) * (W4_STAGE_K * 2) + t * 16;
        float d[NB][4];
#pragma unroll
        for (int s = 0; s < W4_SLICES; ++s) {
          uint32_t a[4], c[4];
          unpack(*reinterpret_cast<const uint32_t*>(st + s * 16), a);
          unpack(*reinterpret_cast<const uint32_t*>(st + 8 * W4_ROW_PITCH + s * 16), c);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint4 x = *reinterpret_cast<const uint4*>(xs + col[b] + s * 64);
            if (s % GS == 0) mma_16816_first<BF16>(d[b], a[0], c[0], a[1], c[1], x.x, x.y);
            else mma_16816<BF16>(d[b], a[0], c[0], a[1], c[1], x.x, x.y);
            mma_16816<BF16>(d[b], a[2], c[2], a[3], c[3], x.z, x.w);
          }
          if (s % GS == GS - 1) {
            const float2 u = *reinterpret_cast<const float2*>(sc + (s / GS) * 16 + g * 2);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              acc[b][0] = fmaf(u.x, d[b][0], acc[b][0]);
              acc[b][1] = fmaf(u.x, d[b][1], acc[b][1]);
              acc[b][2] = fmaf(u.y, d[b][2], acc[b][2]);
              acc[b][3] = fmaf(u.y, d[b][3], acc[b][3]);
            }
          }
        }
      }
    }

    // the shares of k and the pieces of x, joined through shared memory; a warp that owns all of k
    // waits for no other.  Two buffers take turns, so one barrier a round is enough.
    if (SPLIT) {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[0][j] = (acc[2 % NB][j] + acc[1 % NB][j]) + acc[0][j];
    }
    constexpr int JOIN = SPLIT ? 1 : PIECES;      // columns still to be added per row
    float* red = red0 + (round & 1) * (W4_WARPS * OB * 8 * 16);
#pragma unroll
    for (int b = 0; b < OB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) red[(warp * OB * 8 + b * 8 + 2 * t + (j & 1)) * 16 + g + (j >> 1) * 8] = acc[b][j];
    if (wk_n > 1) __syncthreads();
    else __syncwarp();
    const int tile_n = wk_n > 1 ? p.wr * 16 : 16, tile0 = wk_n > 1 ? n0 - wr * 16 : n0;
    for (int e = wk_n > 1 ? threadIdx.x : lane; e < rows * tile_n; e += wk_n > 1 ? W4_THREADS : 32) {
      const int r = e / tile_n, c = e - r * tile_n, n = tile0 + c;
      if (n >= p.n) continue;
      const int w0 = wk_n > 1 ? c >> 4 : warp;
      float y = 0.0f;
      for (int q = JOIN - 1; q >= 0; --q)
        for (int j = 0; j < wk_n; ++j) y += red[((j * p.wr + w0) * OB * 8 + r * JOIN + q) * 16 + (c & 15)];
      if (p.cuts == 1) dt_store(p.out, (m0 + r) * p.ld_out + n, p.out_dtype, w4_steps(p, y, m0 + r, n));
      else p.part[(int64_t(blockIdx.z) * p.m + m0 + r) * p.n + n] = y;
    }
    if (p.cuts > 1) {
      const int group = int(blockIdx.x) + round * int(gridDim.x);
      int* counter = p.counters + int64_t(blockIdx.y) * row_groups + group;
      __syncthreads();
      if (threadIdx.x == 0) {
        __threadfence();      // the whole block's sums, by the barrier before
        s_last = atomicAdd(counter, 1) == p.cuts - 1;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        const int width = p.wr * 16, at = group * width;
        constexpr int FLY = 4;       // results at a time, as many parts of each
        const int64_t step = int64_t(p.m) * p.n;
        for (int e0 = threadIdx.x; e0 < rows * width; e0 += FLY * W4_THREADS) {
          float y[FLY];
          const float* from[FLY];
#pragma unroll
          for (int u = 0; u < FLY; ++u) {
            const int e = e0 + u * W4_THREADS, r = e / width, n = at + e - r * width;
            from[u] = e < rows * width && n < p.n ? p.part + int64_t(m0 + r) * p.n + n : nullptr;
            y[u] = 0.0f;
          }
          for (int z0 = 0; z0 < p.cuts; z0 += 4) {      // added in order
            float x[FLY][4];
#pragma unroll
            for (int u = 0; u < FLY; ++u)
#pragma unroll
              for (int z = 0; z < 4; ++z) x[u][z] = from[u] != nullptr && z0 + z < p.cuts ? __ldcg(from[u] + (z0 + z) * step) : 0.0f;
#pragma unroll
            for (int u = 0; u < FLY; ++u)
#pragma unroll
              for (int z = 0; z < 4; ++z) y[u] += x[u][z];
          }
#pragma unroll
          for (int u = 0; u < FLY; ++u) {
            const int e = e0 + u * W4_THREADS, r = e / width, n = at + e - r * width;
            if (from[u] != nullptr) dt_store(p.out, (m0 + r) * p.ld_out + n, p.out_dtype, w4_steps(p, y[u], m0 + r, n));
          }
        }
        if (threadIdx.x == 0) *counter = 0;
      }
    }
  }
  cp_async_wait<0>();
}

}  // namespace mira
