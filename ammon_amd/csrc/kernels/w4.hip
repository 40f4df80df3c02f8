// w4.hip -- 4-bit weights and rows of 8-bit digits (w4_impl.h): matrices quantised and read
// back, rows quantised (after the residual's addition and RMSNorm, or as they are) and read back.
#include "w4_impl.h"

// A matrix [d, n] (fp32 or bf16) into W4: 16 lanes a group, a workgroup one panel's 16 rows of
// one group, blockIdx.x panels, blockIdx.y groups.  Matrices are stored once; what bounds it is that a
// lane reads its eight numbers one by one (14336 x 4096: 103 us of fp32, 2.6 TB/s, 78 of bf16, 1.9).
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_w4_store(ammon_k_w4 p) {
#pragma clang fp contract(off)
  const uint32_t row = threadIdx.x / 16, i = threadIdx.x & 15;
  const uint32_t groups = w4_groups(p.n);
  for (uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
    const uint32_t r = blockIdx.x * 16 + row;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t k = g * W4_GROUP + 8 * i + e;
      x[e] = r < p.d && k < p.n ? load_elem(p.w, p.dtype, (size_t)r * p.n + k) : 0.f;
    }
    const uint32_t top = abs_max16(x);
    float s = bf16_to_f32(f32_to_bf16(__uint_as_float(top) / 7.0f));
    s = s < 0x1p-126f ? 0.f : s;
    const bool bad = top >= W4_INF;
    const float inv = s > 0.f ? 1.0f / s : 0.f;
    uint32_t lo = 0, hi = 0;  // codes 0..3 and 4..7, a byte each
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = fminf(fmaxf(rintf(x[e] * inv), -7.f), 7.f);
      const float b = fminf(fmaxf(rintf(x[e + 4] * inv), -7.f), 7.f);
      lo |= ((uint32_t)(bad ? 0 : (int)a) & 15u) << (8 * e);
      hi |= ((uint32_t)(bad ? 0 : (int)b) & 15u) << (8 * e);
    }
    // lanes 4 j + 2 h + o have numbers 32 j + 16 h + 8 o .. + 7: those of half 1 go to the high
    // nibbles of the bytes of lane 4 j + o
    const uint32_t lo1 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)lo, AMMON_DPP_XOR2, 0xF, 0xF, false);
    const uint32_t hi1 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi, AMMON_DPP_XOR2, 0xF, 0xF, false);
    uint8_t *panel = (uint8_t *)p.w4 + (size_t)blockIdx.x * groups * W4_PANEL_BYTES;
    if ((i & 2) == 0) {
      uint2 word = make_uint2(lo | lo1 << 4, hi | hi1 << 4);
      *(uint2 *)(panel + (size_t)g * 1024 + (i / 4) * 256 + row * 16 + (i & 1) * 8) = word;
    }
    if (i == 0) {
      uint16_t *scales = (uint16_t *)(panel + (size_t)groups * 1024);
      scales[((row / 4) * groups + g) * 4 + row % 4] =
          bad ? (uint16_t)0x7fc0 : (uint16_t)(__float_as_uint(s) >> 16);
    }
  }
}

// W4 as [d, n] fp32 or bf16 (rounded to nearest even): a thread eight numbers of a row, written one
// by one (14336 x 4096: 152 us as fp32, 1.7 TB/s, 81 as bf16, 1.8).
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_w4_load(ammon_k_w4 p) {
  const uint32_t row = threadIdx.x / 16, i = threadIdx.x & 15;
  const uint32_t groups = w4_groups(p.n), r = blockIdx.x * 16 + row;
  if (r >= p.d) return;
  const uint8_t *panel = (const uint8_t *)p.w4 + (size_t)blockIdx.x * groups * W4_PANEL_BYTES;
  const uint16_t *scales = (const uint16_t *)(panel + (size_t)groups * 1024) + (row / 4) * groups * 4 + row % 4;
  for (uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
    uint2 word = *(const uint2 *)(panel + (size_t)g * 1024 + (i / 4) * 256 + row * 16 + (i & 1) * 8);
    if ((i & 2) == 0) word.x <<= 4, word.y <<= 4;
    const float s = bf16_to_f32(scales[4 * g]);
    const uint32_t k = g * W4_GROUP + 8 * i;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
      const uint32_t w = e < 4 ? word.x : word.y;
      const int c = (int)(w << (24 - 8 * (e & 3))) >> 28;
      if (k + e < p.n) store_elem(p.out, p.dtype, (size_t)r * p.n + k + e, s * (float)c);
    }
  }
}

// ---- rows of digits -------------------------------------------------------------------------

// Digits and scale of block g (lane i of 16: numbers 8 i .. + 7 of it) of token t.
template <int DIGITS>
AMMON_DEV void q8_put(void *rows, uint32_t blocks, uint32_t t, uint32_t g, uint32_t i,
                      const uint2 (&digits)[DIGITS], float s) {
  uint8_t *panel = (uint8_t *)rows + (size_t)(t / 16) * blocks * q8_block_bytes(DIGITS);
  uint8_t *at = panel + (size_t)g * 2048 * DIGITS + ((i >> 1) & 1) * 1024 + (i >> 2) * 256 + (t & 15) * 16 +
                (i & 1) * 8;
#pragma unroll
  for (int p = 0; p < DIGITS; ++p) *(uint2 *)(at + 2048 * p) = digits[p];
  if (i == 0) ((float *)(panel + (size_t)blocks * 2048 * DIGITS))[g * 16 + (t & 15)] = s;
}

AMMON_DEV double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// One workgroup a token.  h = x + residual, to sum; v = w (h / sqrt(mean(h^2) + eps)); the digits
// of v.  The mean is a sum in 64 bits, so that its order does not show in 32: the digits are the
// definition's to the last one.  Without w, the digits of x.  A row of up to 4096 R numbers is held
// in registers, everything it needs requested at once: R = 1, 2 or 4, by its length, since registers
// bound how many tokens a CU has in flight (2048 tokens of 4096: 32 us with R = 4).
//
// A panel's 16 tokens are 16 bytes each of a line, so the workgroups of a panel go to one XCD (they
// are dealt out to the eight in turn), whose L2 makes whole lines of their stores.
constexpr uint32_t Q8_WG = 512;
template <int DIGITS, int R> AMMON_DEV void q8_rows(const ammon_k_q8 &p) {
#pragma clang fp contract(off)
  __shared__ double red[Q8_WG / 64];
  const uint32_t tid = threadIdx.x, blocks = w4_groups(p.n), eights = blocks * 16;
  const uint32_t q = blockIdx.x >> 3, t = ((q >> 4) * 8 + (blockIdx.x & 7)) * 16 + (q & 15);
  if (t >= p.tokens) return;
  const size_t row = (size_t)t * p.n;
  const W4Row x(p.x + row, AMMON_K_F32, p.n), w(p.w, p.w_dtype, p.n);
  const W4Row res(p.residual ? p.residual + row : p.x, AMMON_K_F32, p.residual ? p.n : 0);
  const W4Row sum(p.residual ? p.sum + row : p.sum, AMMON_K_F32, p.residual ? p.n : 0);
  auto add = [&](u32x4 (&v)[2], const u32x4 (&r)[2]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e / 4][e % 4] = __float_as_uint(__uint_as_float(v[e / 4][e % 4]) + __uint_as_float(r[e / 4][e % 4]));
  };
  double ss = 0.0;
  auto square = [&](const u32x4 (&v)[2]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double h = (double)__uint_as_float(v[e / 4][e % 4]);
      ss = fma(h, h, ss);
    }
  };
  u32x4 v[R][2], u[R][2], f[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r * Q8_WG >= eights) break;  // (uniform)
    x.load(tid + r * Q8_WG, v[r]);
    if (p.residual) res.load(tid + r * Q8_WG, u[r]);
    if (p.w) w.load(tid + r * Q8_WG, f[r]);
  }
  float scale = 1.f;
  if (p.w) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r * Q8_WG >= eights) break;
      if (p.residual) {
        add(v[r], u[r]);
        sum.store(tid + r * Q8_WG, v[r]);
      }
      square(v[r]);
    }
    for (uint32_t c = tid + R * Q8_WG; c < eights; c += Q8_WG) {
      u32x4 h[2], g[2];
      x.load(c, h);
      if (p.residual) {
        res.load(c, g);
        add(h, g);
        sum.store(c, h);
      }
      square(h);
    }
    ss = wave_sum_f64(ss);
    if ((tid & 63) == 0) red[tid >> 6] = ss;
    __syncthreads();
    ss = red[0];
#pragma unroll
    for (uint32_t k = 1; k < Q8_WG / 64; ++k) ss += red[k];
    scale = (float)(1.0 / sqrt(ss / (double)p.n + (double)p.eps));
  }
  auto put = [&](uint32_t c, const u32x4 (&h)[2], const u32x4 (&g)[2]) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = __uint_as_float(h[e / 4][e % 4]);
      if (p.w) y[e] = w.number(g, e) * (scale * y[e]);
    }
    uint2 digits[DIGITS];
    const float s = q8_digits<DIGITS>(y, digits);
    if (c < eights) q8_put<DIGITS>(p.rows, blocks, t, c / 16, c & 15, digits, s);
  };
  // (a block's 16 lanes go together: eights and the stride are multiples of 16)
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r * Q8_WG >= eights) break;
    put(tid + r * Q8_WG, v[r], f[r]);
  }
  for (uint32_t c = tid + R * Q8_WG; c < eights; c += Q8_WG) {
    u32x4 h[2], g[2];
    // (with a sum, its own numbers, which this thread wrote: x may be where they went)
    if (p.residual)
      sum.load(c, h);
    else
      x.load(c, h);
    if (p.w) w.load(c, g);
    put(c, h, g);
  }
}
#define Q8_ROWS_KERNEL(DIGITS, R, OCC)                                                                   \
  extern "C" __global__ __launch_bounds__(Q8_WG, OCC) void ammon_q8_rows_##DIGITS##_r##R(ammon_k_q8 p) { \
    q8_rows<DIGITS, R>(p);                                                                               \
  }
Q8_ROWS_KERNEL(1, 1, 8)
Q8_ROWS_KERNEL(1, 2, 6)
Q8_ROWS_KERNEL(1, 4, 4)
Q8_ROWS_KERNEL(3, 1, 8)
Q8_ROWS_KERNEL(3, 2, 6)
Q8_ROWS_KERNEL(3, 4, 4)

// Rows back as fp32 [tokens, n]: a wave a block of a panel, a piece of eight tokens at a time: lane
// l has numbers 4 (l % 8) .. + 3 of the piece of token l / 8, so that a store is eight whole lines.
template <int DIGITS> AMMON_DEV void q8_load(const ammon_k_q8 &p) {
  const uint32_t blocks = w4_groups(p.n), lane = threadIdx.x & 63, f = lane & 7;
  const uint64_t total = (uint64_t)((p.tokens + 15) / 16) * blocks;
  for (uint64_t u = (uint64_t)blockIdx.x * AMMON_WAVES + threadIdx.x / 64; u < total;
       u += (uint64_t)gridDim.x * AMMON_WAVES) {
    const uint32_t panel = (uint32_t)(u / blocks), g = (uint32_t)(u % blocks);
    const uint8_t *base = (const uint8_t *)p.rows + (size_t)panel * blocks * q8_block_bytes(DIGITS);
    const uint8_t *at = base + (size_t)g * 2048 * DIGITS + (f >> 2) * 1024 + (f & 3) * 4;
    const float *scales = (const float *)(base + (size_t)blocks * 2048 * DIGITS) + g * 16;
    uint32_t d[8][DIGITS];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)  // piece i / 2, tokens 8 (i % 2) ..
#pragma unroll
      for (int k = 0; k < DIGITS; ++k)
        d[i][k] = *(const uint32_t *)(at + 2048 * k + (i / 2) * 256 + ((i & 1) * 8 + (lane >> 3)) * 16);
    const float s[2] = {scales[lane >> 3], scales[8 + (lane >> 3)]};
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t t = panel * 16 + (i & 1) * 8 + (lane >> 3), k0 = g * W4_GROUP + (i / 2) * 32 + 4 * f;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        int q = 0;
#pragma unroll
        for (int k = DIGITS - 1; k >= 0; --k) q = q * 256 + ((int)(d[i][k] << (24 - 8 * e)) >> 24);
        v[e] = (float)q * s[i & 1];
      }
      float *out = p.sum + (size_t)t * p.n + k0;
      if (t >= p.tokens) continue;
      if (p.vec && k0 < p.n) {
        *(f32x4a4 *)out = v;
      } else if (!p.vec) {
        for (uint32_t e = 0; e < 4; ++e)
          if (k0 + e < p.n) out[e] = v[e];
      }
    }
  }
}
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_q8_load_1(ammon_k_q8 p) { q8_load<1>(p); }
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_q8_load_3(ammon_k_q8 p) { q8_load<3>(p); }
