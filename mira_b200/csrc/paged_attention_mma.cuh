// Paged attention of one token per sequence on the tensor path, for 16-bit and 8-bit pages.
//
// Bound: the visible keys and values are read once; an SM's share of the memory bandwidth is about 23
// bytes a clock.  The group's heads are the 16 rows of the products, so a key costs the same few
// instructions for one head as for sixteen, and what remains is unpacking, addresses and the softmax.
//
// No fragment crosses lanes: the sums over k of a product do not care in which order k comes, so a
// lane's 16-byte piece of a row, as it arrives from memory, is its share of a fragment.
//   S = Q K^T: lane (g, t) holds token g's elements VE t .. VE t + VE - 1 of each run of 4 VE: four of
//     them are the right operand of one 16x8x16 product; Q is laid out to match, once per unit.
//   O += P V: lane (g, t) holds elements VE g .. of each run of 8 VE of the tokens 2t, 2t + 1, 2t + 8 and
//     2t + 9; pairs of tokens of one element, one byte permutation each, are the right operand, column g
//     of tile i being element VE g + i; P's accumulators are already the left operand's layout.
// Exactness: q enters as one value of the pages' type where it has that type, else as three whose sum
// it is; 8-bit codes become exact f16 values.  p is f32 and enters as PP values that agree with it to 16
// bits or more (see PaMma), the row's sum l is of the f32 values.
#pragma once
#include <cstdint>

#include "mma_sm80.cuh"
#include "paged_attention.cuh"

namespace mira {

// T: the pages' element; DHP: head dimension rounded up to 64, 128 or 256; VB: bytes per access of a
// key row; QP: values per query element, 1 or 3.
template <typename T, int DHP, int VB, int QP>
struct PaMma {
  static constexpr bool I8 = sizeof(T) == 1;
  static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;      // else the products are f16
  static constexpr int KE = VB / int(sizeof(T));                           // elements of a key access
  static constexpr int KL = DHP / (4 * KE);                                // key accesses of a lane per token
  static constexpr int KS = DHP / 16;                                      // products along the head dimension
  static constexpr int VBV = VB < DHP * int(sizeof(T)) / 8 ? VB : DHP * int(sizeof(T)) / 8;
  static constexpr int VE = VBV / int(sizeof(T));
  static constexpr int VL = DHP / (8 * VE);                                // value accesses per token
  static constexpr int NT = DHP / 8;                                       // tiles of O
  static constexpr int TT = (DHP * int(sizeof(T)) <= 128) ? 2 : 1;         // runs of 16 tokens per step
  static constexpr int TILE = 16 * TT;                                     // tokens of a warp step
  // p: bf16 values have 8 bits, f16 ones 11.  16-bit results: 16 and 22 bits; f32 results (QP == 3): 24
  // and 22, whose error of 2^-22 of the largest weight is that of an f32 sum of a few terms.  In f16,
  // p is carried times 2^8: the smallest f16 is then 2^-32 of the largest weight.
  static constexpr int PP = BF16 && QP == 3 ? 3 : 2;
  static constexpr float SHIFT = BF16 ? 0.0f : 8.0f;
  static constexpr int K_BYTES = TT * 2 * KL * 32 * VB, V_BYTES = TT * 4 * VL * 32 * VBV;    // of a step
  static constexpr int STEP = K_BYTES + V_BYTES + (I8 ? 2 * 32 * 4 : 0);      // 8-bit pages: and the scales
  static constexpr int WARPS = DHP <= 128 ? 12 : 8;                           // of an SM, by registers
  static constexpr int Q_BYTES = QP * KS * 32 * 16;
};

// x = a + b (+ c) in 16-bit values, pairs packed.
template <bool BF16, int N>
__device__ __forceinline__ void pa_split2(float x, float y, uint32_t (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      out[i] = b2_bits(h);
      if (i + 1 < N) {
        x -= __uint_as_float(out[i] << 16);
        y -= __uint_as_float(out[i] & 0xffff0000u);
      }
    } else {
      const __half2 h = __floats2half2_rn(x, y);
      out[i] = h2_bits(h);
      if (i + 1 < N) {
        const float2 f = __half22float2(h);
        x -= f.x;
        y -= f.y;
      }
    }
  }
}

// Four 8-bit codes (as bytes + 128) -> two registers of f16 pairs (0, 1), (2, 3): the byte becomes the
// low mantissa bits of 1024, 1152 is subtracted exactly.
__device__ __forceinline__ uint32_t pa_codes(uint32_t biased, uint32_t sel) {
  return h2_bits(__hsub2(bits_h2(__byte_perm(biased, 0x64646464u, sel)), bits_h2(0x64806480u)));
}

template <int WORDS> struct PaWords { uint32_t w[WORDS]; };

template <int BYTES>
__device__ __forceinline__ PaWords<BYTES / 4> pa_held(const uint8_t* p) {
  PaWords<BYTES / 4> r;
  memcpy(&r, __builtin_assume_aligned(p, BYTES), BYTES);
  return r;
}

template <typename T, int DHP, int VB, int QP>
__global__ void __launch_bounds__(PaMma<T, DHP, VB, QP>::WARPS * 32, 1)
    paged_attention_mma_kernel(const __grid_constant__ PagedAttnParams p) {
  using C = PaMma<T, DHP, VB, QP>;
  extern __shared__ __align__(128) uint8_t pa_smem[];       // ring, queries, the warps' triples
  __shared__ float s_unit[16];        // per head: what turns a product into a scaled score
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, feeders = (blockDim.x >> 5) / 3, warps = (blockDim.x >> 5) - feeders;
  const int rows = min(16, p.group);
  uint4* s_q = reinterpret_cast<uint4*>(pa_smem + pa_ring_bytes(warps * p.slots, C::STEP));     // [piece][product][lane]
  float* s_join = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(s_q) + C::Q_BYTES);
  PaWork w;
  if (!pa_begin<C::TILE>(p, warps, w)) return;
  const PaRing ring = pa_ring_at(pa_smem, warps, p.slots, C::STEP, &s_abort);

  if (warp >= warps) {
    PaToken tok;
    int64_t ks_at = 0, vs_at = 0;
    auto look = [&](const PaWork& w, int at) {
      int page, slot;
      tok = pa_token<T>(p, w, p.kv.table + w.b * p.kv.table_ld, at + lane, lane < C::TILE, page, slot);
      if (C::I8) {
        const int kvh = w.unit / p.head_blocks;
        ks_at = page * p.kv.kss[0] + kvh * p.kv.kss[1] + slot * p.kv.kss[2];
        vs_at = page * p.kv.vss[0] + kvh * p.kv.vss[1] + slot * p.kv.vss[2];
      }
    };
    auto copy = [&](const PaWork& w, uint8_t* step) {
      const int kvh = w.unit / p.head_blocks;
      const uint8_t* kb = reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.kv.k) + kvh * p.kv.kst[1] + t * C::KE);
      const uint8_t* vb = reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.kv.v) + kvh * p.kv.vst[1] + g * C::VE);
      const uint32_t live = __ballot_sync(0xffffffffu, tok.ok);
      const uint32_t kd = smem_u32(step) + lane * VB, vd = smem_u32(step) + C::K_BYTES + lane * C::VBV;
      if (C::I8) {
        const uint32_t sd = smem_u32(step) + C::K_BYTES + C::V_BYTES + lane * 4;
        pa_copy<4>(sd, reinterpret_cast<const uint8_t*>(p.kv.ks + ks_at), tok.ok);
        pa_copy<4>(sd + 128, reinterpret_cast<const uint8_t*>(p.kv.vs + vs_at), tok.ok);
      }
#pragma unroll
      for (int r = 0; r < C::TT; ++r) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int i = r * 16 + n * 8 + g;
          const uint8_t* row = kb + __shfl_sync(0xffffffffu, tok.k, i);
          const bool in = live >> i & 1;
#pragma unroll
          for (int j = 0; j < C::KL; ++j)
            pa_copy<VB>(kd + ((r * 2 + n) * C::KL + j) * (32 * VB), row + j * 4 * VB, in && (j * 4 + t) * C::KE < p.kv.dh);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int i = r * 16 + (n >> 1) * 8 + 2 * t + (n & 1);
          const uint8_t* row = vb + __shfl_sync(0xffffffffu, tok.v, i);
          const bool in = live >> i & 1;
#pragma unroll
          for (int j = 0; j < C::VL; ++j)
            pa_copy<C::VBV>(vd + ((r * 4 + n) * C::VL + j) * (32 * C::VBV), row + j * 8 * C::VBV, in && (j * 8 + g) * C::VE < p.kv.dh);
        }
      }
      return live;
    };
    pa_feed<C::TILE>(p, w, ring, C::STEP, warp - warps, feeders, warps, look, copy);
    if (lane == 0 && s_abort) atomicExch(p.kv.err, 1);
    return;
  }

  PaPlace mine{0, 0};
  while (pa_part<C::TILE>(p, w)) {
    const int kvh = w.unit / p.head_blocks, g0 = (w.unit - kvh * p.head_blocks) * 16;
    const int h0 = kvh * p.group + g0, live_heads = min(16, p.group - g0);
    const int steps = w.t1 > w.t0 ? (w.t1 - w.t0 - 1) / C::TILE + 1 : 0;

    // queries of the unit in fragment order; a thread per (product, lane).  f16 values of a query that
    // is not f16 itself are taken after a power of two has brought its largest element to [128, 256).
    for (int h = warp; h < 16; h += warps) {
      float unit = p.scale_log2;
      if (QP == 3 && !C::BF16) {
        float top = 0.0f;
        if (h < live_heads)
          for (int d = lane; d < p.kv.dh; d += 32)
            top = fmaxf(top, fabsf(dt_load(p.q, w.b * p.qs[0] + (h0 + h) * p.qs[1] + d * p.qs[2], p.q_dtype)));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int e = int(__float_as_uint(top) >> 23);      // 2^(e - 127) <= top
        const int up = e == 0 || e == 255 ? 0 : min(max(134 - e, -126), 127);
        if (lane == 0) s_unit[h] = __int_as_float((127 + up) << 23);
      } else if (lane == 0) {
        s_unit[h] = unit;
      }
    }
    pa_sync(warps * 32);
    for (int i = threadIdx.x; i < C::KS * 32; i += warps * 32) {
      const int ks = i >> 5, l = i & 31, lg = l >> 2, lt = l & 3;
      const int d = (ks / (C::KE / 4)) * 4 * C::KE + lt * C::KE + (ks % (C::KE / 4)) * 4;
      float x[2][4];       // head g and g + 8, elements d .. d + 3
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = lg + 8 * hh;
          float v = h < live_heads && d + e < p.kv.dh
              ? dt_load(p.q, w.b * p.qs[0] + (h0 + h) * p.qs[1] + (d + e) * p.qs[2], p.q_dtype) : 0.0f;
          if (QP == 3 && !C::BF16) v *= s_unit[h];
          x[hh][e] = v;
        }
      uint32_t f[4][QP];
      if (C::BF16 && QP == 3) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a[3], b[3];
          split3_bf16(x[j & 1][(j >> 1) * 2], a[0], a[1], a[2]);
          split3_bf16(x[j & 1][(j >> 1) * 2 + 1], b[0], b[1], b[2]);
#pragma unroll
          for (int q = 0; q < QP; ++q) f[j][q] = __byte_perm(a[q], b[q], 0x7632);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) pa_split2<C::BF16, QP>(x[j & 1][(j >> 1) * 2], x[j & 1][(j >> 1) * 2 + 1], f[j]);
      }
#pragma unroll
      for (int q = 0; q < QP; ++q) s_q[(q * C::KS + ks) * 32 + l] = make_uint4(f[0][q], f[1][q], f[2][q], f[3][q]);
    }
    pa_sync(warps * 32);
    float unit0 = s_unit[g], unit1 = s_unit[g + 8];
    if (QP == 3 && !C::BF16) {      // powers of two: the division is exact
      unit0 = p.scale_log2 / unit0;
      unit1 = p.scale_log2 / unit1;
    }

    float acc[C::NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    uint32_t v_exp = 1;       // 8-bit pages: exponent of the largest value scale so far, which acc is divided by
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;

    for (int k = warp; k < steps; k += warps) {
      const int slot = warp * ring.slots + mine.slot;
      pa_wait(ring, ring.full + slot, mine.round);
      const uint32_t now = ring.live[slot];
      const uint8_t* step = ring.steps + int64_t(slot) * C::STEP;
      const uint8_t* kr = step + lane * VB;
      const uint8_t* vr = step + C::K_BYTES + lane * C::VBV;
      const float* sc = reinterpret_cast<const float*>(step + C::K_BYTES + C::V_BYTES);      // [k, v][token]

      // scores
      float s[C::TT][2][4], s2[C::TT][2][4];      // two sums each: half as many products wait for one another
#pragma unroll
      for (int r = 0; r < C::TT; ++r)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[r][n][i] = s2[r][n][i] = 0.0f;
#pragma unroll
      for (int j = 0; j < C::KL; ++j) {
        PaWords<VB / 4> kx[C::TT][2];
#pragma unroll
        for (int r = 0; r < C::TT; ++r)
#pragma unroll
          for (int n = 0; n < 2; ++n) kx[r][n] = pa_held<VB>(kr + ((r * 2 + n) * C::KL + j) * (32 * VB));
#pragma unroll
        for (int e = 0; e < C::KE / 4; ++e) {
          uint32_t b[C::TT][2][2];
#pragma unroll
          for (int r = 0; r < C::TT; ++r)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              if (C::I8) {
                const uint32_t x = kx[r][n].w[e] ^ 0x80808080u;
                b[r][n][0] = pa_codes(x, 0x4140);
                b[r][n][1] = pa_codes(x, 0x4342);
              } else {
                b[r][n][0] = kx[r][n].w[(2 * e) % (VB / 4)];
                b[r][n][1] = kx[r][n].w[(2 * e + 1) % (VB / 4)];
              }
            }
#pragma unroll
          for (int q = QP - 1; q >= 0; --q) {
            const uint4 a = s_q[(q * C::KS + j * (C::KE / 4) + e) * 32 + lane];
#pragma unroll
            for (int r = 0; r < C::TT; ++r)
#pragma unroll
              for (int n = 0; n < 2; ++n) mma_16816<C::BF16>(e & 1 ? s2[r][n] : s[r][n], a.x, a.y, a.z, a.w, b[r][n][0], b[r][n][1]);
          }
        }
      }
      float top0 = m0, top1 = m1;
#pragma unroll
      for (int r = 0; r < C::TT; ++r)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const bool in = now >> (r * 16 + n * 8 + 2 * t + i) & 1;
            const float ks = C::I8 ? sc[r * 16 + n * 8 + 2 * t + i] : 1.0f;
            s[r][n][i] = in ? (s[r][n][i] + s2[r][n][i]) * (C::I8 ? unit0 * ks : unit0) : -INFINITY;
            s[r][n][2 + i] = in ? (s[r][n][2 + i] + s2[r][n][2 + i]) * (C::I8 ? unit1 * ks : unit1) : -INFINITY;
            top0 = fmaxf(top0, s[r][n][i]);
            top1 = fmaxf(top1, s[r][n][2 + i]);
          }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, o));
        top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, o));
      }
      float grow = 1.0f, shrink = 1.0f;
      if (C::I8) {
        const float vscale = lane < C::TILE && (now >> lane & 1) ? sc[32 + lane] : 0.0f;
        const uint32_t e = min(max(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(vscale))) >> 23, v_exp), 253u);
        grow = __int_as_float((127 - min(int(e - v_exp), 126)) << 23);
        v_exp = e;
        shrink = __int_as_float((254 - e) << 23);
      }
      const float safe0 = top0 == -INFINITY ? 0.0f : top0, safe1 = top1 == -INFINITY ? 0.0f : top1;
      if (__any_sync(0xffffffffu, top0 > m0 || top1 > m1 || grow != 1.0f)) {
        const float f0 = pa_exp2(m0 - safe0), f1 = pa_exp2(m1 - safe1);
        m0 = top0;
        m1 = top1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int n = 0; n < C::NT; ++n) {
          acc[n][0] *= f0 * grow;
          acc[n][1] *= f0 * grow;
          acc[n][2] *= f1 * grow;
          acc[n][3] *= f1 * grow;
        }
      }
      const float z0 = safe0 - C::SHIFT, z1 = safe1 - C::SHIFT;
#pragma unroll
      for (int r = 0; r < C::TT; ++r) {
        uint32_t a[4][C::PP];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          float x0 = pa_exp2(s[r][n][0] - z0), x1 = pa_exp2(s[r][n][1] - z0);
          float y0 = pa_exp2(s[r][n][2] - z1), y1 = pa_exp2(s[r][n][3] - z1);
          l0 += x0 + x1;
          l1 += y0 + y1;
          if (C::I8) {
            const int i = r * 16 + n * 8 + 2 * t;       // a token that does not count has no scale either
            const float u0 = now >> i & 1 ? sc[32 + i] * shrink : 0.0f, u1 = now >> (i + 1) & 1 ? sc[33 + i] * shrink : 0.0f;
            x0 *= u0;
            x1 *= u1;
            y0 *= u0;
            y1 *= u1;
          }
          pa_split2<C::BF16, C::PP>(x0, x1, a[2 * n]);
          pa_split2<C::BF16, C::PP>(y0, y1, a[2 * n + 1]);
        }
#pragma unroll
        for (int j = 0; j < C::VL; ++j) {
          PaWords<C::VBV / 4> vx[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) vx[n] = pa_held<C::VBV>(vr + ((r * 4 + n) * C::VL + j) * (32 * C::VBV));
#pragma unroll
          for (int e = 0; e < C::VBV / 4; ++e) {
            constexpr int PER = 4 / int(sizeof(T));      // elements of a word
            uint32_t b[PER][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t x = vx[2 * h].w[e], y = vx[2 * h + 1].w[e];
              if (C::I8) {
                const uint32_t bx = x ^ 0x80808080u, by = y ^ 0x80808080u;
                const uint32_t low = __byte_perm(bx, by, 0x5140), high = __byte_perm(bx, by, 0x7362);
                b[0][h] = pa_codes(low, 0x4140);
                b[1][h] = pa_codes(low, 0x4342);
                b[2 % PER][h] = pa_codes(high, 0x4140);
                b[3 % PER][h] = pa_codes(high, 0x4342);
              } else {
                b[0][h] = __byte_perm(x, y, 0x5410);
                b[1][h] = __byte_perm(x, y, 0x7632);
              }
            }
#pragma unroll
            for (int i = 0; i < PER; ++i)
#pragma unroll
              for (int q = C::PP - 1; q >= 0; --q)
                mma_16816<C::BF16>(acc[j * C::VE + e * PER + i], a[0][q], a[1][q], a[2][q], a[3][q], b[i][0], b[i][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(ring.empty + slot);
      mine.forward(ring.slots);
    }
    // the warp's triple
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    const float back = C::BF16 ? 1.0f : 0x1p-8f;
    const float back_v = C::I8 ? back * __int_as_float(v_exp << 23) : back;
    float* to = s_join + warp * pa_triple(rows, DHP);
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int h = g + 8 * hh;
      if (h >= rows) continue;
      if (t == 0) {
        to[h] = hh ? m1 : m0;
        to[rows + h] = (hh ? l1 : l0) * back;
      }
      float* a = to + pa_head(rows) + h * DHP;
#pragma unroll
      for (int j = 0; j < C::VL; ++j)
#pragma unroll
        for (int i = 0; i < C::VE; ++i) {
          a[(j * 8 + 2 * t) * C::VE + i] = acc[j * C::VE + i][2 * hh] * back_v;
          a[(j * 8 + 2 * t + 1) * C::VE + i] = acc[j * C::VE + i][2 * hh + 1] * back_v;
        }
    }
    pa_finish<DHP>(p, w, s_join, warps, rows, h0, live_heads);
    w.cur = w.end;
  }
  if (threadIdx.x == 0 && s_abort) atomicExch(p.kv.err, 1);
}

}  // namespace mira
