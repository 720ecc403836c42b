// Paged attention of one token per sequence on the tensor path, for 16-bit and 8-bit pages.
//
// Bound: the visible keys and values are read once; an SM's share of the memory bandwidth is about 23
// bytes a clock, a step of 8 KB every 360 clocks.  The keys are the products' left operand, 16 tokens, and
// the heads that share them its eight columns (twice eight for groups of more than 8), so that the
// products, the softmax and the sums cost the same for one head as for eight, and little more than the
// unpacking, the addresses and the waiting.  (Products of 64 or 128 tokens at a time out of shared memory
// would leave the heads' columns as empty, and hand P back through memory; the operands here never leave
// the registers, and the bytes, not the products, set the pace.)
// Measured: 32 sequences of up to 8192 tokens, 32 heads over 8 of 128, bf16 (553 MB): 128 us, 4.3 TB/s, where
// the steps alone run at 91% of the copy rate and some 30 us go to the launch and the ends of the 256 units and their
// parts.  One sequence of 131071 tokens, 32 heads over 4, f16 (268 MB): 72 us; its steps take 47 us, joining
// the 37 parts of each unit 10.  48 sequences, window 4095, 20 heads over 4 of 80, codes under f32 queries
// (121 MB): 57.4 us; here the unpacking and products of the computing warps are the limit (issue slots 45%
// busy by eight to twelve warps of an SM).  Head sizes up to 96 have a class of their own: in that of 128 it took 62.7.
//   S^T = K Q^T: lane (g, t) holds elements VE t .. VE t + VE - 1 of each run of 4 VE of tokens g and g + 8,
//     16 bytes as they came from memory: four elements of each are a left fragment.  The sums over k do
//     not care in which order k comes; Q is laid out to match, once per unit.
//   O^T += V^T P^T: lane (g, t) holds elements VE g .. of each run of 8 VE of tokens 2t, 2t + 1, 2t + 8 and
//     2t + 9; pairs of tokens of one element, a byte permutation each, are left fragments with rows
//     (element i, g) and (element i + 1, g).  P^T is S^T's accumulators, packed and transposed in 8 x 8
//     blocks by movmatrix.
// Exactness: q enters as one value of the pages' type where it has that type, else as three bf16 values
// whose sum it is, or as two f16 values that agree with it to 2^-22 of the head's largest element; 8-bit
// codes become exact f16 (or bf16) values.  p is f32, with 8-bit pages times the value's scale, and enters as PP
// values that agree with it to 16 bits or more (see PaMma); the row's sum l is of the f32 values.
#pragma once
#include <cstdint>

#include "mma_sm80.cuh"
#include "paged_attention.cuh"

namespace mira {

// T: the pages' element; DHP: head dimension rounded up to 64, 96, 128 or 256; VB: bytes per access of a
// key row; QP: values per query element, 1, or 3 (bf16) or 2 (f16); NH: blocks of eight heads.
template <typename T, int DHP, int VB, int QP, int NH>
struct PaMma {
  static constexpr bool I8 = sizeof(T) == 1;
  static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;      // else the products are f16
  static constexpr int KE = VB / int(sizeof(T));                           // elements of a key access
  static constexpr int KL = DHP / (4 * KE);                                // key accesses of a lane per token
  static constexpr int KS = DHP / 16;                                      // products along the head dimension
  // bytes per access of a value row: eight lanes' accesses have to divide it
  static constexpr int VBV = DHP == 96 ? 4 * int(sizeof(T)) : VB < DHP * int(sizeof(T)) / 8 ? VB : DHP * int(sizeof(T)) / 8;
  static constexpr int VE = VBV / int(sizeof(T));
  static constexpr int VL = DHP / (8 * VE);                                // value accesses per token
  static constexpr int NT = DHP / 16;                                      // tiles of O
  static constexpr int TT = (DHP * int(sizeof(T)) <= 128) ? 2 : 1;         // runs of 16 tokens per step
  static constexpr int TILE = 16 * TT;                                     // tokens of a step
  // p: bf16 values have 8 bits, f16 ones 11.  16-bit results: 16 and 22 bits; f32 results (QP > 1): 24
  // and 22, whose error of 2^-22 of the largest weight is that of an f32 sum of a few terms; the same
  // goes for the two f16 values of a query element.  In f16, p is carried times 2^8: the smallest f16 is
  // then 2^-32 of the largest weight.
  // 8-bit pages: what enters is p times the value's scale, of sizes that nothing limits (an append gives a row
  // of zeros the scale 1, whatever its neighbours have).  It is taken relative to the largest scale so far and
  // times 2^V_SHIFT, as two f16 values as long as all scales so far are within 2^-V_NEAR of that one, so that an f16
  // rounds to 2^-31 of the largest weight times its own scale or less; then as three bf16 values, which have f32's
  // range (48 x 20/4 heads of 80, window: 57.4 us; with bf16 values for every step 66.1).
  static constexpr int PP = BF16 && QP > 1 ? 3 : 2;
  static constexpr float SHIFT = BF16 || I8 ? 0.0f : 8.0f;
  static constexpr int V_SHIFT = 14, V_NEAR = 8;
  static constexpr int K_BYTES = TT * 2 * KL * 32 * VB, V_BYTES = TT * 4 * VL * 32 * VBV;    // of a step
  static constexpr int STEP = K_BYTES + V_BYTES + (I8 ? 2 * 32 * 4 : 0);      // 8-bit pages: and the scales
  // warps of an SM, by the registers of the sums and by the ring: a computing warp wants two steps of it
  static constexpr int WARPS = STEP > 9000 || NH * DHP > 256 ? 6 : NH * DHP <= 128 ? 16 : 12;
  static constexpr int Q_BYTES = NH * QP * KS * 32 * 8;
};

// The 8 x 8 block of 16-bit values whose row g lane (g, t) holds columns 2t, 2t + 1 of, transposed.
__device__ __forceinline__ uint32_t pa_transpose(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

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

// The codes in the low bytes of both halves as a bf16 pair: the seven low bits under the exponent of 128, less 128,
// or 256 for the sign bit, which under the same exponent is the next one.
__device__ __forceinline__ uint32_t pa_codes_bf16(uint32_t x) {
  return b2_bits(__hsub2(bits_b2((x & 0x007f007fu) | 0x43004300u), bits_b2((x & 0x00800080u) | 0x43004300u)));
}

template <int WORDS> struct PaWords { uint32_t w[WORDS]; };

template <int BYTES>
__device__ __forceinline__ PaWords<BYTES / 4> pa_held(const uint8_t* p) {
  PaWords<BYTES / 4> r;
  memcpy(&r, __builtin_assume_aligned(p, BYTES), BYTES);
  return r;
}

template <typename T, int DHP, int VB, int QP, int NH>
__global__ void __launch_bounds__(PaMma<T, DHP, VB, QP, NH>::WARPS * 32, 1)
    paged_attention_mma_kernel(const __grid_constant__ PagedAttnParams p) {
  using C = PaMma<T, DHP, VB, QP, NH>;
  extern __shared__ __align__(128) uint8_t pa_smem[];       // ring, queries, the warps' triples
  __shared__ float s_unit[8 * NH];        // per head: what turns a product into a scaled score
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, feeders = p.feeders, warps = (blockDim.x >> 5) - feeders;
  const int rows = min(8 * NH, p.group);
  uint2* s_q = reinterpret_cast<uint2*>(pa_smem + pa_ring_bytes(warps * p.slots, C::STEP));     // [piece][heads][product][lane]
  float* s_join = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(s_q) + C::Q_BYTES);
  PaWork w;
  if (!pa_begin<C::TILE>(p, warps, w)) return;
  const PaRing ring = pa_ring_at(pa_smem, warps, p.slots, C::STEP, &s_abort);

  if (warp >= warps) {
    uint32_t ksize[C::KL], vsize[C::VL];       // of this lane's accesses of a row
#pragma unroll
    for (int j = 0; j < C::KL; ++j) ksize[j] = (j * 4 + t) * C::KE < p.kv.dh ? VB : 0;
#pragma unroll
    for (int j = 0; j < C::VL; ++j) vsize[j] = (j * 8 + g) * C::VE < p.kv.dh ? C::VBV : 0;
    auto copy = [&](const PaWork& w, PaToken tokens, uint8_t* step) {
      const PaRows tok = pa_rows<T>(p, tokens);
      const int kvh = w.unit / p.head_blocks;
      const uint8_t* kb = reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.kv.k) + kvh * p.kv.kst[1] + t * C::KE);
      const uint8_t* vb = reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.kv.v) + kvh * p.kv.vst[1] + g * C::VE);
      const uint32_t live = __ballot_sync(0xffffffffu, tok.ok);
      const uint32_t kd = smem_u32(step) + lane * VB, vd = smem_u32(step) + C::K_BYTES + lane * C::VBV;
      if (C::I8) {
        const uint32_t sd = smem_u32(step) + C::K_BYTES + C::V_BYTES + lane * 4;
        const float* ks = p.kv.ks + tokens.page * p.kv.kss[0] + kvh * p.kv.kss[1] + tokens.slot * p.kv.kss[2];
        const float* vs = p.kv.vs + tokens.page * p.kv.vss[0] + kvh * p.kv.vss[1] + tokens.slot * p.kv.vss[2];
        pa_copy<4>(sd, reinterpret_cast<const uint8_t*>(ks), tok.ok ? 4 : 0);
        pa_copy<4>(sd + 128, reinterpret_cast<const uint8_t*>(vs), tok.ok ? 4 : 0);
      }
      auto rows = [&](auto full) {
#pragma unroll
        for (int r = 0; r < C::TT; ++r) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int i = r * 16 + n * 8 + g;
            const uint8_t* row = kb + __shfl_sync(0xffffffffu, tok.k, i);
            const bool in = decltype(full)::value || (live >> i & 1);
#pragma unroll
            for (int j = 0; j < C::KL; ++j)
              pa_copy<VB>(kd + ((r * 2 + n) * C::KL + j) * (32 * VB), row + j * 4 * VB, in ? ksize[j] : 0);
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int i = r * 16 + (n >> 1) * 8 + 2 * t + (n & 1);
            const uint8_t* row = vb + __shfl_sync(0xffffffffu, tok.v, i);
            const bool in = decltype(full)::value || (live >> i & 1);
#pragma unroll
            for (int j = 0; j < C::VL; ++j)
              pa_copy<C::VBV>(vd + ((r * 4 + n) * C::VL + j) * (32 * C::VBV), row + j * 8 * C::VBV, in ? vsize[j] : 0);
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
    const int kvh = w.unit / p.head_blocks, g0 = (w.unit - kvh * p.head_blocks) * (8 * NH);
    const int h0 = kvh * p.group + g0, live_heads = min(8 * NH, p.group - g0);
    const int steps = pa_steps(w, C::TILE);

    // queries of the unit in fragment order, a warp per head, four elements of it per lane and turn.  f16
    // values of a query that is not f16 itself are taken after a power of two has brought its largest
    // element to [128, 256).
    for (int h = warp; h < 8 * NH; h += warps) {
      constexpr int TURNS = DHP / 128 > 1 ? DHP / 128 : 1;
      float x[TURNS][4], top = 0.0f;
#pragma unroll
      for (int i = 0; i < TURNS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = (i * 32 + lane) * 4 + e;
          x[i][e] = h < live_heads && d < p.kv.dh
              ? dt_load(p.q, w.b * p.qs[0] + (h0 + h) * p.qs[1] + d * p.qs[2], p.q_dtype) : 0.0f;
          top = fmaxf(top, fabsf(x[i][e]));
        }
      float up = 1.0f;
      if (QP > 1 && !C::BF16) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int e = int(__float_as_uint(top) >> 23);      // 2^(e - 127) <= top
        up = __int_as_float((127 + (e == 0 || e == 255 ? 0 : min(max(134 - e, -126), 127))) << 23);
      }
      if (lane == 0) s_unit[h] = p.scale_log2 / up;         // a power of two: exact
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int d = (i * 32 + lane) * 4;
        if (d >= DHP) break;
        const int lt = d % (4 * C::KE) / C::KE, ks = d / (4 * C::KE) * (C::KE / 4) + d % C::KE / 4;
        uint32_t f[2][QP];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (C::BF16 && QP == 3) {
            uint32_t a[3], b[3];
            split3_bf16(x[i][2 * j], a[0], a[1], a[2]);
            split3_bf16(x[i][2 * j + 1], b[0], b[1], b[2]);
#pragma unroll
            for (int q = 0; q < QP; ++q) f[j][q] = __byte_perm(a[q], b[q], 0x7632);
          } else {
            pa_split2<C::BF16, QP>(x[i][2 * j] * up, x[i][2 * j + 1] * up, f[j]);
          }
        }
#pragma unroll
        for (int q = 0; q < QP; ++q)
          s_q[((q * NH + h / 8) * C::KS + ks) * 32 + h % 8 * 4 + lt] = make_uint2(f[0][q], f[1][q]);
      }
    }
    pa_sync(warps * 32);
    // this lane's heads are 8 b + 2t + i
    float unit[NH][2], m[NH][2], l[NH][2], acc[C::NT][NH][4];
#pragma unroll
    for (int b = 0; b < NH; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        unit[b][i] = s_unit[8 * b + 2 * t + i];
        m[b][i] = -INFINITY;
        l[b][i] = 0.0f;
      }
    // 8-bit pages: exponents of the largest value scale so far, which acc is divided by, and of the smallest but 0
    uint32_t v_exp = C::V_SHIFT + 1, v_low = 255;
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
      for (int b = 0; b < NH; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][b][i] = 0.0f;

    for (; next < steps; next += warps) {
      const int slot = warp * ring.slots + mine.slot;
      pa_wait(ring, ring.full + slot, mine.round);
      const uint32_t now = ring.live[slot];
      const uint8_t* step = ring.steps + int64_t(slot) * C::STEP;
      const uint8_t* kr = step + lane * VB;
      const uint8_t* vr = step + C::K_BYTES + lane * C::VBV;
      const float* sc = reinterpret_cast<const float*>(step + C::K_BYTES + C::V_BYTES);      // [k, v][token]

      // scores of tokens 16 r + g (values 0, 1) and + 8 (2, 3); two sums each, so that half as many
      // products wait for one another
      float s[C::TT][NH][4], s2[C::TT][NH][4];
#pragma unroll
      for (int r = 0; r < C::TT; ++r)
#pragma unroll
        for (int b = 0; b < NH; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[r][b][i] = s2[r][b][i] = 0.0f;
#pragma unroll
      for (int j = 0; j < C::KL; ++j) {
        if (j * 4 * C::KE >= p.kv.dh) break;
        PaWords<VB / 4> kx[C::TT][2];
#pragma unroll
        for (int r = 0; r < C::TT; ++r)
#pragma unroll
          for (int n = 0; n < 2; ++n) kx[r][n] = pa_held<VB>(kr + ((r * 2 + n) * C::KL + j) * (32 * VB));
#pragma unroll
        for (int e = 0; e < C::KE / 4; ++e) {
          uint32_t a[C::TT][4];
#pragma unroll
          for (int r = 0; r < C::TT; ++r)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              if (C::I8) {
                const uint32_t x = kx[r][n].w[e] ^ 0x80808080u;
                a[r][n] = pa_codes(x, 0x4140);
                a[r][2 + n] = pa_codes(x, 0x4342);
              } else {
                a[r][n] = kx[r][n].w[(2 * e) % (VB / 4)];
                a[r][2 + n] = kx[r][n].w[(2 * e + 1) % (VB / 4)];
              }
            }
#pragma unroll
          for (int q = QP - 1; q >= 0; --q)
#pragma unroll
            for (int b = 0; b < NH; ++b) {
              const uint2 y = s_q[((q * NH + b) * C::KS + j * (C::KE / 4) + e) * 32 + lane];
#pragma unroll
              for (int r = 0; r < C::TT; ++r)
                mma_16816<C::BF16>(e & 1 ? s2[r][b] : s[r][b], a[r][0], a[r][1], a[r][2], a[r][3], y.x, y.y);
            }
        }
      }
      float top[NH][2];
#pragma unroll
      for (int b = 0; b < NH; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[b][i] = m[b][i];
#pragma unroll
          for (int r = 0; r < C::TT; ++r)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const int token = r * 16 + n * 8 + g;
              float& x = s[r][b][2 * n + i];
              x = now >> token & 1 ? (x + s2[r][b][2 * n + i]) * (C::I8 ? unit[b][i] * sc[token] : unit[b][i]) : -INFINITY;
              top[b][i] = fmaxf(top[b][i], x);
            }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) top[b][i] = fmaxf(top[b][i], __shfl_xor_sync(0xffffffffu, top[b][i], o));
        }
      float grow = 1.0f, shrink = 1.0f;
      bool spread = false;
      if (C::I8) {       // tokens that do not count have the scale 0
        const uint32_t bits = __float_as_uint(sc[32 + lane]) & 0x7fffffffu;
        const uint32_t e = min(max(__reduce_max_sync(0xffffffffu, bits) >> 23, v_exp), 254u);
        v_low = min(v_low, __reduce_min_sync(0xffffffffu, bits - 1) >> 23);      // 0 is left out as the largest
        spread = e > v_low + C::V_NEAR;
        grow = e - v_exp > 126 ? 0.0f : __int_as_float((127 - (e - v_exp)) << 23);
        v_exp = e;
        shrink = __int_as_float((254 + C::V_SHIFT - e) << 23);
      }
      bool moved = grow != 1.0f;
#pragma unroll
      for (int b = 0; b < NH; ++b) moved = moved || top[b][0] > m[b][0] || top[b][1] > m[b][1];
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int b = 0; b < NH; ++b)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float f = pa_exp2(m[b][i] - (top[b][i] == -INFINITY ? 0.0f : top[b][i]));
            m[b][i] = top[b][i];
            l[b][i] *= f;
#pragma unroll
            for (int n = 0; n < C::NT; ++n) {
              acc[n][b][i] *= f * grow;
              acc[n][b][2 + i] *= f * grow;
            }
          }
      }
      // the weights as PC values of bf16 (PBF16) or f16, times the values
      auto values = [&](int r, auto bf16, auto pieces) {
        constexpr bool PBF16 = decltype(bf16)::value;
        constexpr int PC = decltype(pieces)::value;
        uint32_t pt[NH][2][PC];          // P^T: tokens 2t, 2t + 1 (+ 8) of head g
#pragma unroll
        for (int b = 0; b < NH; ++b)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            float x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              x[i] = pa_exp2(s[r][b][2 * n + i] - ((m[b][i] == -INFINITY ? 0.0f : m[b][i]) - C::SHIFT));
              l[b][i] += x[i];
              if (C::I8) x[i] *= sc[32 + r * 16 + n * 8 + g] * shrink;
            }
            pa_split2<PBF16, PC>(x[0], x[1], pt[b][n]);
#pragma unroll
            for (int q = 0; q < PC; ++q) pt[b][n][q] = pa_transpose(pt[b][n][q]);
          }
#pragma unroll
        for (int j = 0; j < C::VL; ++j) {
          if (j * 8 * C::VE >= p.kv.dh) break;
          PaWords<C::VBV / 4> vx[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) vx[n] = pa_held<C::VBV>(vr + ((r * 4 + n) * C::VL + j) * (32 * C::VBV));
#pragma unroll
          for (int e = 0; e < C::VBV / 4; ++e) {
            constexpr int PER = 4 / int(sizeof(T));      // elements of a word
            uint32_t a[PER][2];                          // element, tokens 2t, 2t + 1 (+ 8)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t x = vx[2 * h].w[e], y = vx[2 * h + 1].w[e];
              if (C::I8 && PBF16) {
                const uint32_t low = __byte_perm(x, y, 0x5410), high = __byte_perm(x, y, 0x7632);
                a[0][h] = pa_codes_bf16(low);
                a[1][h] = pa_codes_bf16(low >> 8);
                a[2 % PER][h] = pa_codes_bf16(high);
                a[3 % PER][h] = pa_codes_bf16(high >> 8);
              } else if (C::I8) {
                const uint32_t bx = x ^ 0x80808080u, by = y ^ 0x80808080u;
                const uint32_t low = __byte_perm(bx, by, 0x5140), high = __byte_perm(bx, by, 0x7362);
                a[0][h] = pa_codes(low, 0x4140);
                a[1][h] = pa_codes(low, 0x4342);
                a[2 % PER][h] = pa_codes(high, 0x4140);
                a[3 % PER][h] = pa_codes(high, 0x4342);
              } else {
                a[0][h] = __byte_perm(x, y, 0x5410);
                a[1][h] = __byte_perm(x, y, 0x7632);
              }
            }
#pragma unroll
            for (int i = 0; i < PER / 2; ++i)
#pragma unroll
              for (int b = 0; b < NH; ++b)
#pragma unroll
                for (int q = PC - 1; q >= 0; --q)
                  mma_16816<PBF16>(acc[(j * C::VE + e * PER) / 2 + i][b], a[2 * i][0], a[2 * i + 1][0], a[2 * i][1], a[2 * i + 1][1],
                                   pt[b][0][q], pt[b][1][q]);
          }
        }
      };
#pragma unroll
      for (int r = 0; r < C::TT; ++r) {
        if (C::I8 && spread) values(r, std::true_type{}, std::integral_constant<int, 3>{});
        else values(r, std::integral_constant<bool, C::BF16>{}, std::integral_constant<int, C::PP>{});
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(ring.empty + slot);
      mine.forward(ring.slots);
    }
    next -= steps;

    // the warp's triple
    const float back = C::BF16 || C::I8 ? 1.0f : 0x1p-8f;
    const float back_v = C::I8 ? __int_as_float((v_exp - C::V_SHIFT) << 23) : back;
    float* to = s_join + warp * pa_triple(rows, DHP);
#pragma unroll
    for (int b = 0; b < NH; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[b][i] += __shfl_xor_sync(0xffffffffu, l[b][i], o);
        const int h = 8 * b + 2 * t + i;
        if (h >= rows) continue;
        if (g == 0) {
          to[h] = m[b][i];
          to[rows + h] = l[b][i] * back;
        }
        // tile n: elements 2 n and 2 n + 1 of the lane's runs
#pragma unroll
        for (int n = 0; n < C::NT; ++n) {
          const int d = ((2 * n) / C::VE * 8 + g) * C::VE + (2 * n) % C::VE;
          *reinterpret_cast<float2*>(to + pa_at<DHP>(rows, h, d / 4) + d % 4) = make_float2(acc[n][b][i] * back_v, acc[n][b][2 + i] * back_v);
        }
      }
    pa_finish<DHP>(p, w, s_join, warps, rows, h0, live_heads);
    w.cur = w.end;
  }
  if (threadIdx.x == 0 && s_abort) atomicExch(p.kv.err, 1);
}

}  // namespace mira
