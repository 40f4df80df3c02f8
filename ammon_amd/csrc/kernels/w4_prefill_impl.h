// w4_prefill_impl.h -- products of rows of 8-bit digits with 4-bit weights (w4_impl.h) on
// integer matrix cores: Y[t] = W X[t] with the epilogues of the prefill GEMMs (prefill.hip).
//
// y[t, r] = sum_g s_w[r, g] s_x[t, g] sum_{k in g} c[r, k] q[t, k].  A tile is 16 rows x 16
// tokens; per group of 128 numbers and per digit two v_mfma_i32_16x16x64_i8 take 1 KiB of codes
// (operand A, an AND and a shift away from memory) and two halves of digits (operand B, as they
// lie in memory), exactly.  Lane l then has rows 4 (l / 16) .. + 3 of token l % 16, one sum per
// digit: joined (as whole numbers where they fit), converted, scaled and added to the fp32 total.
#pragma once

#include "qkv_store.h"
#include "w4_impl.h"

// RT panels of rows per wave x CT panels of tokens; KS = 1: the four waves have panels of their
// own, KS = 4: they split the groups of the same ones, and wave 0 adds the four sums in order.
template <int DIGITS, int MODE, uint32_t RT, uint32_t CT, uint32_t KS> struct W4Tile {
  static constexpr bool GATED = MODE == AMMON_GEMV_SWIGLU;
  static constexpr uint32_t RO = GATED ? RT / 2 : RT;          // panels of results per wave
  static constexpr uint32_t RW = RO * (AMMON_WAVES / KS);      // ... per workgroup
  static_assert(!GATED || RT % 2 == 0, "gate and up panels go together");

  ammon_k_gemm p;
  uint32_t lane, wave, groups, gbeg, gend, tok0;
  uint32_t panel[RT];           // virtual panel of results
  const uint8_t *w[RT];         // its codes, this lane's
  const uint8_t *ws[RT];        // its scales, this lane's
  const uint8_t *x[CT];         // digits, this lane's
  const float *xs[CT];          // scales, this lane's

  AMMON_DEV W4Tile(const ammon_k_gemm &p_, uint32_t rb, uint32_t tt, uint32_t ks) : p(p_) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    groups = w4_groups(p.n);
    gbeg = 0, gend = groups;
    if (p.ksplit > 1) {
      gbeg = min(ks * p.kchunks, groups);
      gend = min(gbeg + p.kchunks, groups);
    }
    const uint32_t first = rb * RW + (KS == 1 ? wave * RO : 0);
    if (KS > 1) {
      const uint32_t per = (gend - gbeg + KS - 1) / KS;
      gbeg = min(gbeg + wave * per, gend);
      gend = min(gbeg + per, gend);
    }
    const size_t bytes = (size_t)groups * W4_PANEL_BYTES;
    const uint32_t panels = ((GATED ? p.d : p.rows) + 15) / 16;
#pragma unroll
    for (uint32_t j = 0; j < RT; ++j) {
      panel[j] = first + (GATED ? j % RO : j);
      uint32_t at = min(panel[j], panels - 1);  // past the end: the last one, not stored
      const void *base = p.w0;
      if (GATED) base = j < RO ? p.w0 : p.w1;
      if (MODE == AMMON_GEMV_QKV) {
        const uint32_t q = p.d / 16, kv = p.kv_dim / 16;
        if (at >= q + kv)
          base = p.w2, at -= q + kv;
        else if (at >= q)
          base = p.w1, at -= q;
      }
      const uint8_t *b = (const uint8_t *)base + at * bytes;
      w[j] = b + lane * 16;
      ws[j] = b + (size_t)groups * 1024 + (size_t)(lane >> 4) * groups * 8;
    }
    tok0 = tt * 16 * CT;
    const uint32_t tpanels = (p.tokens + 15) / 16;
#pragma unroll
    for (uint32_t c = 0; c < CT; ++c) {
      const uint32_t at = min(tt * CT + c, tpanels - 1);
      const uint8_t *b = (const uint8_t *)p.x + (size_t)at * groups * q8_block_bytes(DIGITS);
      x[c] = b + lane * 16;
      xs[c] = (const float *)(b + (size_t)groups * 2048 * DIGITS) + (lane & 15);
    }
  }

  AMMON_DEV void run(f32x4 (&acc)[RT][CT]) const {
#pragma unroll
    for (uint32_t j = 0; j < RT; ++j)
#pragma unroll
      for (uint32_t c = 0; c < CT; ++c) acc[j][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t g = gbeg; g < gend; ++g) {
      u32x4 a[RT];
      u32x2 s[RT];
#pragma unroll
      for (uint32_t j = 0; j < RT; ++j) {
        a[j] = *(const u32x4 *)(w[j] + (size_t)g * 1024);
        s[j] = *(const u32x2 *)(ws[j] + (size_t)g * 8);
      }
#pragma unroll
      for (uint32_t c = 0; c < CT; ++c) {
        i32x4 b[DIGITS][2];
#pragma unroll
        for (int d = 0; d < DIGITS; ++d)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            b[d][h] = *(const i32x4 *)(x[c] + ((size_t)g * DIGITS + d) * 2048 + h * 1024);
        const float sx = xs[c][g * 16] * 0.0625f;  // (the codes are 16 c)
#pragma unroll
        for (uint32_t j = 0; j < RT; ++j) {
          i32x4 t[DIGITS];
#pragma unroll
          for (int d = 0; d < DIGITS; ++d) {
            t[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w4_half0(a[j]), b[d][0], i32x4{0, 0, 0, 0}, 0, 0, 0);
            t[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w4_half1(a[j]), b[d][1], t[d], 0, 0, 0);
          }
          const float sw[4] = {bf16_lo(s[j][0]), bf16_hi(s[j][0]), bf16_lo(s[j][1]), bf16_hi(s[j][1])};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // (a digit's sum is at most 2^21: two of them fit a word)
            const float f = DIGITS == 1
                                ? (float)t[0][r]
                                : fmaf((float)((t[DIGITS - 1][r] << 8) + t[DIGITS / 2][r]), 256.f, (float)t[0][r]);
            acc[j][c][r] = fmaf(f, sx * sw[r], acc[j][c][r]);
          }
        }
      }
    }
  }

  AMMON_DEV void store(const f32x4 (&acc)[RT][CT], uint32_t ks) const {
    const uint32_t rq = 4 * (lane >> 4);
    const bool split = p.ksplit > 1;
#pragma unroll
    for (uint32_t j = 0; j < RO; ++j)
#pragma unroll
      for (uint32_t c = 0; c < CT; ++c) {
        const uint32_t t = tok0 + 16 * c + (lane & 15), v = 16 * panel[j] + rq;
        if (t >= p.tokens) continue;
        if (MODE == AMMON_GEMV_QKV && !split) {
#pragma unroll
          for (int i = 0; i < 4; i += 2)
            if (v + i < p.rows) qkv_store_pair(p, t, v + i, acc[j][c][i], acc[j][c][i + 1]);
          continue;
        }
        const uint32_t width = split ? p.rows : p.d;
        float *y = (split ? p.ws + (size_t)ks * p.tokens * p.rows : p.y) + (size_t)t * width + v;
        const float *res = p.residual + (size_t)t * width + v;
        f32x4 out = acc[j][c];
        if (GATED) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float gate = acc[j][c][i], up = acc[j + RT - RO][c][i];
            float f = gate * (1.0f / (1.0f + expf(-gate)));
            out[i] = f * up;
          }
        }
        const bool add = MODE == AMMON_GEMV_RESIDUAL && !split;
        if ((width & 3u) == 0 && v < width) {
          if (add) out = *(const f32x4a4 *)res + out;
          *(f32x4a4 *)y = out;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (v + i < width) y[i] = add ? res[i] + out[i] : out[i];
        }
      }
  }
};

template <int DIGITS, int MODE, uint32_t RT, uint32_t CT, uint32_t KS>
AMMON_DEV void w4_gemm(const ammon_k_gemm &p) {
  using T = W4Tile<DIGITS, MODE, RT, CT, KS>;
  // id = ((row-block group, reduction range), token tile, XCD), as the prefill GEMMs' grid
  const uint32_t tiles = (p.tokens + 16 * CT - 1) / (16 * CT);
  const uint32_t ksplit = p.ksplit > 1 ? p.ksplit : 1;
  const uint32_t q = blockIdx.x >> 3;
  const uint32_t tt = q % tiles, ks = (q / tiles) % ksplit;
  const uint32_t rb = (q / tiles / ksplit) * 8 + (blockIdx.x & 7u);
  const uint32_t panels = ((T::GATED ? p.d : p.rows) + 15) / 16;
  if (rb * T::RW >= panels) return;  // padding of the last group (uniform)
  T tile(p, rb, tt, ks);
  f32x4 acc[RT][CT];
  tile.run(acc);
  if constexpr (KS > 1) {
    __shared__ f32x4 part[KS - 1][RT][CT][64];
    if (tile.wave) {
#pragma unroll
      for (uint32_t j = 0; j < RT; ++j)
#pragma unroll
        for (uint32_t c = 0; c < CT; ++c) part[tile.wave - 1][j][c][tile.lane] = acc[j][c];
    }
    __syncthreads();
    if (tile.wave) return;
#pragma unroll
    for (uint32_t j = 0; j < RT; ++j)
#pragma unroll
      for (uint32_t c = 0; c < CT; ++c)
#pragma unroll
        for (uint32_t w = 0; w + 1 < KS; ++w) acc[j][c] += part[w][j][c][tile.lane];
  }
  tile.store(acc, ks);
}
