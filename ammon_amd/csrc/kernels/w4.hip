// w4.hip -- 4-bit weights and rows of 8-bit digits (w4_impl.h): matrices quantised and read
// back, rows quantised (after the residual's addition and RMSNorm, or as they are) and read back.
#include "w4_impl.h"

// A matrix [d, n] (fp32 or bf16) into W4: 16 lanes a group, a workgroup one panel's 16 rows of
// one group, blockIdx.x panels, blockIdx.y groups.
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_w4_store(ammon_k_w4 p) {
#pragma clang fp contract(off)
  const uint32_t row = threadIdx.x / 16, i = threadIdx.x & 15;
  const uint32_t groups = w4_groups(p.n);
  for (uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
    const uint32_t r = blockIdx.x * 16 + row;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (r < p.d) {
      const size_t at = (size_t)r * p.n;
      const void *src = p.dtype == AMMON_K_BF16 ? (const void *)((const uint16_t *)p.w + at)
                                                : (const void *)((const float *)p.w + at);
      w4_load8(src, p.dtype, g * 16 + i, p.n, p.vec != 0, x);
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

// W4 as [d, n] fp32 or bf16 (rounded to nearest even): a thread eight numbers of a row.
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
// definition's to the last one.  Without w, the digits of x.
template <int DIGITS> AMMON_DEV void q8_rows(const ammon_k_q8 &p) {
#pragma clang fp contract(off)
  constexpr int R = 4;  // eights of a row that a thread keeps in registers
  __shared__ double red[AMMON_WAVES];
  const uint32_t t = blockIdx.x, tid = threadIdx.x, blocks = w4_groups(p.n), eights = blocks * 16;
  const float *x = p.x + (size_t)t * p.n;
  const float *res = p.residual ? p.residual + (size_t)t * p.n : nullptr;
  float *sum = p.residual ? p.sum + (size_t)t * p.n : nullptr;
  const bool vec = p.vec != 0;
  auto load = [&](uint32_t c, float (&v)[8]) {
    w4_load8(x, c, p.n, vec, v);
    if (!res) return;
    float r[8];
    w4_load8(res, c, p.n, vec, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] + r[e];
  };
  auto keep = [&](uint32_t c, const float (&v)[8]) {
    if (!sum) return;
    const uint32_t k = 8 * c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (vec && k + 4 * h < p.n) {
        *(float4 *)(sum + k + 4 * h) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
      } else if (!vec) {
        for (int e = 4 * h; e < 4 * h + 4; ++e)
          if (k + e < p.n) sum[k + e] = v[e];
      }
    }
  };
  float v[R][8];
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (tid + r * AMMON_WG < eights) load(tid + r * AMMON_WG, v[r]);
  float scale = 1.f;
  if (p.w) {
    double ss = 0.0;
    auto add = [&](const float (&h)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fma((double)h[e], (double)h[e], ss);
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (tid + r * AMMON_WG < eights) {
        keep(tid + r * AMMON_WG, v[r]);
        add(v[r]);
      }
    for (uint32_t c = tid + R * AMMON_WG; c < eights; c += AMMON_WG) {
      float h[8];
      load(c, h);
      keep(c, h);
      add(h);
    }
    ss = wave_sum_f64(ss);
    if ((tid & 63) == 0) red[tid >> 6] = ss;
    __syncthreads();
    ss = red[0];
#pragma unroll
    for (int w = 1; w < AMMON_WAVES; ++w) ss += red[w];
    scale = (float)(1.0 / sqrt(ss / (double)p.n + (double)p.eps));
  }
  auto put = [&](uint32_t c, float (&h)[8]) {
    if (p.w) {
      float w[8];
      w4_load8(p.w, p.w_dtype, c, p.n, p.w_vec != 0, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = w[e] * (scale * h[e]);
    }
    uint2 digits[DIGITS];
    const float s = q8_digits<DIGITS>(h, digits);
    q8_put<DIGITS>(p.rows, blocks, t, c / 16, c & 15, digits, s);
  };
  // (a block's 16 lanes go together: eights and the stride are multiples of 16)
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (tid + r * AMMON_WG < eights) put(tid + r * AMMON_WG, v[r]);
  for (uint32_t c = tid + R * AMMON_WG; c < eights; c += AMMON_WG) {
    float h[8];
    // (with a sum, its own numbers, which this thread wrote: x may be where they went)
    if (sum)
      w4_load8(sum, c, p.n, vec, h);
    else
      load(c, h);
    put(c, h);
  }
}
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_q8_rows_1(ammon_k_q8 p) { q8_rows<1>(p); }
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_q8_rows_3(ammon_k_q8 p) { q8_rows<3>(p); }

// Rows back as fp32 [tokens, n]: a thread eight numbers of a row.
template <int DIGITS> AMMON_DEV void q8_load(const ammon_k_q8 &p) {
  const uint32_t blocks = w4_groups(p.n), eights = (p.n + 7) / 8;
  const uint64_t total = (uint64_t)p.tokens * eights;
  for (uint64_t u = (uint64_t)blockIdx.x * AMMON_WG + threadIdx.x; u < total;
       u += (uint64_t)gridDim.x * AMMON_WG) {
    const uint32_t t = (uint32_t)(u / eights), c = (uint32_t)(u % eights), g = c / 16, i = c & 15;
    const uint8_t *panel = (const uint8_t *)p.rows + (size_t)(t / 16) * blocks * q8_block_bytes(DIGITS);
    const uint8_t *at = panel + (size_t)g * 2048 * DIGITS + ((i >> 1) & 1) * 1024 + (i >> 2) * 256 +
                        (t & 15) * 16 + (i & 1) * 8;
    const float s = ((const float *)(panel + (size_t)blocks * 2048 * DIGITS))[g * 16 + (t & 15)];
    uint2 d[DIGITS];
#pragma unroll
    for (int k = 0; k < DIGITS; ++k) d[k] = *(const uint2 *)(at + 2048 * k);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int q = 0;
#pragma unroll
      for (int k = DIGITS - 1; k >= 0; --k)
        q = q * 256 + ((int)((e < 4 ? d[k].x : d[k].y) << (24 - 8 * (e & 3))) >> 24);
      v[e] = (float)q * s;
    }
    float *out = p.sum + (size_t)t * p.n + 8 * c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (p.vec && 8 * c + 4 * h < p.n) {
        *(float4 *)(out + 4 * h) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
      } else if (!p.vec) {
        for (int e = 4 * h; e < 4 * h + 4; ++e)
          if (8 * c + e < p.n) out[e] = v[e];
      }
    }
  }
}
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_q8_load_1(ammon_k_q8 p) { q8_load<1>(p); }
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_q8_load_3(ammon_k_q8 p) { q8_load<3>(p); }
