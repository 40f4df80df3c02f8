// w4_gemv_impl.h -- products of one token's row with 4-bit weights (w4_impl.h): the modes of
// gemv_impl.h (plain, residual, SwiGLU, QKV, argmax candidates) over AMMON_W4 matrices.
//
// y_r = sum_k W[r, k] x_k.  x (RMS-normalised where a weight is given) becomes Q24 digits in LDS,
// once per workgroup; a wave multiplies 16 rows x 128 numbers, 1 KiB of codes, by two
// v_mfma_i32_16x16x64_i8: the codes are operand A as they lie in memory but for an AND and a
// shift, and the three digits are columns 0..2 of operand B (the other columns repeat the third
// and are scaled by 0).  A group's sums are exact; they are scaled by s_w s_x 256^digit, exact
// too, and added up over the groups in fp32 with one rounding each.
//
// A workgroup of 4 waves takes units of 16 virtual rows (a panel; SwiGLU: 8 gate and the same 8
// up rows) and splits the groups over its waves; each wave has the codes of U groups in two
// register buffers, the next ones requested before the current are multiplied.
#pragma once

#include "argmax_impl.h"
#include "w4_impl.h"

template <int MODE> struct W4Gemv {
  static constexpr uint32_t U = 8;  // groups a register buffer holds

  ammon_k_gemv p;
  uint32_t lane, wave, groups, per;  // per: groups of a wave
  uint8_t *digits;                   // LDS: [groups][2 halves][3 digits][64 bytes]
  float *scales;                     // LDS: [groups][4], s_x 256^digit / 16 (the codes are 16 c); 0
  // operands' addresses in the current unit
  struct Unit {
    const uint8_t *codes;
    const uint8_t *scales;
  };
  struct Buffer {
    u32x4 codes[U];
    u32x2 scales[U];
  };

  AMMON_DEV Unit unit(uint32_t u) const {
    const uint32_t j = lane >> 4;
    const void *const w0 = p.w0, *const w1 = p.w1, *const w2 = p.w2, *base = w0;
    uint32_t panel = u, row = lane & 15, quad = j;
    const size_t bytes = (size_t)groups * W4_PANEL_BYTES;
    if (MODE == AMMON_GEMV_SWIGLU) {
      // rows 0..7 gate, 8..15 up; results' quads 0, 1 gate, 2, 3 up
      const uint32_t half = (u & 1) * 8;
      panel = u >> 1;
      const uint8_t *codes = (const uint8_t *)(row < 8 ? w0 : w1) + panel * bytes;
      const uint8_t *sc = (const uint8_t *)(quad < 2 ? w0 : w1) + panel * bytes;
      row = half + (row & 7);
      quad = half / 4 + (quad & 1);
      return Unit{codes + j * 256 + row * 16, sc + (size_t)groups * 1024 + (size_t)quad * groups * 8};
    }
    if (MODE == AMMON_GEMV_QKV) {
      const uint32_t q = p.d / 16, kv = p.kv_dim / 16;
      base = u >= q + kv ? w2 : u >= q ? w1 : w0;
      panel -= u >= q + kv ? q + kv : u >= q ? q : 0;
    }
    const uint8_t *at = (const uint8_t *)base + panel * bytes;
    return Unit{at + j * 256 + row * 16, at + (size_t)groups * 1024 + (size_t)quad * groups * 8};
  }

  // Groups first .. + U - 1 of this wave's; past its last one, that one again (not multiplied).
  AMMON_DEV void load(const Unit &u, uint32_t first, uint32_t last, Buffer &b) const {
#pragma unroll
    for (uint32_t i = 0; i < U; ++i) {
      const uint32_t g = min(first + i, last);
      b.codes[i] = __builtin_nontemporal_load((const u32x4 *)(u.codes + (size_t)g * 1024));
      b.scales[i] = __builtin_nontemporal_load((const u32x2 *)(u.scales + (size_t)g * 8));
    }
  }

  AMMON_DEV void multiply(uint32_t first, uint32_t end, const Buffer &b, f32x4 &acc) const {
    const uint32_t col = min(lane & 15, 3u), digit = min(col, 2u), j = lane >> 4;
#pragma unroll
    for (uint32_t i = 0; i < U; ++i) {
      const uint32_t g = first + i;
      if (g >= end) break;
      const uint8_t *d = digits + ((size_t)g * 6 + digit) * 64 + j * 16;
      const i32x4 b0 = *(const i32x4 *)d, b1 = *(const i32x4 *)(d + 192);
      i32x4 c = i32x4{0, 0, 0, 0};
      c = __builtin_amdgcn_mfma_i32_16x16x64_i8(w4_half0(b.codes[i]), b0, c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_i32_16x16x64_i8(w4_half1(b.codes[i]), b1, c, 0, 0, 0);
      const float sx = scales[4 * g + col];
      const u32x2 s = b.scales[i];
      const float sw[4] = {bf16_lo(s[0]), bf16_hi(s[0]), bf16_lo(s[1]), bf16_hi(s[1])};
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = fmaf((float)c[r], sx * sw[r], acc[r]);
    }
  }

  // x as digits in LDS, normalised first where there is a weight.  red: AMMON_WAVES floats.
  AMMON_DEV void stage(float *red) {
    constexpr int R = 4;  // eights of x that a thread keeps in registers
    const uint32_t tid = threadIdx.x, eights = groups * 16, n = p.n;
    const bool vec = (n & 3u) == 0 && ((uintptr_t)p.x & 15u) == 0;
    const bool wvec = (n & 3u) == 0 && ((uintptr_t)p.norm_w & (p.norm_dtype == AMMON_K_BF16 ? 7u : 15u)) == 0;
    float v[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (tid + r * AMMON_WG < eights) w4_load8(p.x, tid + r * AMMON_WG, n, vec, v[r]);
    float scale = 1.f;
    if (p.norm_w) {
      float ss = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (tid + r * AMMON_WG < eights)
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(v[r][e], v[r][e], ss);
      for (uint32_t c = tid + R * AMMON_WG; c < eights; c += AMMON_WG) {
        float h[8];
        w4_load8(p.x, c, n, vec, h);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(h[e], h[e], ss);
      }
      ss = block_sum(ss, red);
      scale = 1.0f / sqrtf(ss / (float)n + p.eps);
    }
    auto put = [&](uint32_t c, float (&h)[8]) {
      if (p.norm_w) {
        float w[8];
        w4_load8(p.norm_w, p.norm_dtype, c, n, wvec, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = w[e] * (scale * h[e]);
      }
      uint2 d[3];
      const float s = q8_digits<3>(h, d);
      const uint32_t g = c / 16, i = c & 15;
      uint8_t *at = digits + ((size_t)g * 6 + ((i >> 1) & 1) * 3) * 64 + (i >> 2) * 16 + (i & 1) * 8;
#pragma unroll
      for (int k = 0; k < 3; ++k) *(uint2 *)(at + 64 * k) = d[k];
      if (i == 0) *(float4 *)(scales + 4 * g) = make_float4(s * 0.0625f, s * 16.f, s * 4096.f, 0.f);
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (tid + r * AMMON_WG < eights) put(tid + r * AMMON_WG, v[r]);
    for (uint32_t c = tid + R * AMMON_WG; c < eights; c += AMMON_WG) {
      float h[8];
      w4_load8(p.x, c, n, vec, h);
      put(c, h);
    }
  }

  // Rows' sums of unit u, red [waves][16]: added in wave order, then the mode's epilogue.
  AMMON_DEV float row_sum(const float *red, uint32_t r) const {
    float v = red[r];
#pragma unroll
    for (int w = 1; w < AMMON_WAVES; ++w) v += red[16 * w + r];
    return v;
  }
  AMMON_DEV void finish(uint32_t u, const float *red, uint32_t pos, float &cand_v, uint32_t &cand_i) const {
    const uint32_t e = threadIdx.x;
    if (MODE == AMMON_GEMV_SWIGLU) {
      if (e >= 8 || 8 * u + e >= p.d) return;
      const float gate = row_sum(red, e), up = row_sum(red, 8 + e);
      float v = gate * (1.0f / (1.0f + expf(-gate)));
      v = v * up;
      st_out(p.y + 8 * u + e, v);
    } else if (MODE == AMMON_GEMV_QKV) {
#pragma clang fp contract(off)
      const uint32_t vr = 16 * u + 2 * e;
      if (e >= 8 || vr >= p.rows) return;
      const float a0 = row_sum(red, 2 * e), a1 = row_sum(red, 2 * e + 1);
      const float nan = __uint_as_float(W4_NAN);
      if (pos >= p.seq) {  // out-of-range position: poison q (and rows), touch no cache
        if (vr < p.d) {
          st_out(p.y + vr, nan);
          st_out(p.y + vr + 1, nan);
        } else if (p.kv_rows) {
          const uint32_t rr = vr - p.d;
          store_pair_out(rr < p.kv_dim ? p.k_cache : p.v_cache, AMMON_K_F32, rr % p.kv_dim, nan, nan);
        }
        return;
      }
      if (vr < p.d + p.kv_dim) {
        const uint32_t rr = vr < p.d ? vr : vr - p.d, hd = rr % p.head;
        const float *cs = p.table + ((size_t)pos * (p.head / 2) + hd / 2) * 2;
        const float fcr = cs[0], fci = cs[1];
        const float o0 = a0 * fcr - a1 * fci;
        const float o1 = a0 * fci + a1 * fcr;
        if (vr < p.d) {
          st_out(p.y + vr, o0);
          st_out(p.y + vr + 1, o1);
        } else {
          const size_t dst = p.kv_rows ? rr : ((size_t)(rr / p.head) * p.seq + pos) * p.head + hd;
          store_pair_out(p.k_cache, p.kv_dtype, dst, o0, o1);
        }
      } else {
        const uint32_t rv = vr - p.d - p.kv_dim;
        const size_t dst = p.kv_rows ? rv : ((size_t)(rv / p.head) * p.seq + pos) * p.head + rv % p.head;
        store_pair_out(p.v_cache, p.kv_dtype, dst, a0, a1);
      }
    } else {
      const uint32_t vr = 16 * u + e;
      if (e >= 16 || vr >= p.rows) return;
      const float v = row_sum(red, e);
      st_out(p.y + vr, MODE == AMMON_GEMV_RESIDUAL ? ld_in(p.residual + vr) + v : v);
      if (MODE == AMMON_GEMV_PLAIN_ARGMAX && v == v) cand_merge(cand_v, cand_i, v, vr);
    }
  }

  AMMON_DEV void run(const ammon_k_gemv &params, uint32_t nwg, uint8_t *lds) {
    __shared__ float red[2][AMMON_WAVES][16];
    p = params;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    groups = w4_groups(p.n);
    per = (groups + AMMON_WAVES - 1) / AMMON_WAVES;
    scales = (float *)lds;
    digits = lds + (size_t)groups * 16;
    const uint32_t gbeg = min(wave * per, groups), gend = min(gbeg + per, groups);
    const uint32_t last = groups - 1;  // (a wave without groups requests the last one)
    const uint32_t chunks = (per + U - 1) / U, units = p.row_blocks;
    uint32_t pos = 0;
    if (MODE == AMMON_GEMV_QKV) pos = p.step->position;

    // steps (unit, chunk) of this workgroup, two buffers ahead
    const uint32_t total = blockIdx.x < units ? ((units - 1 - blockIdx.x) / nwg + 1) * chunks : 0;
    Buffer bufs[2];
    uint32_t lu = blockIdx.x, lc = 0;  // the next request's
    Unit at = unit(min(lu, units - 1));
    auto request = [&](Buffer &b) {
      if (lu >= units) return;
      load(at, gbeg + lc * U, gend ? min(gend - 1, last) : last, b);
      if (++lc == chunks) {
        lc = 0;
        lu += nwg;
        at = unit(min(lu, units - 1));
      }
    };
    request(bufs[0]);
    stage(&red[0][0][0]);
    __syncthreads();
    float cand_v = 0.f;
    uint32_t cand_i = ARGMAX_NONE;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t u = blockIdx.x, c = 0, flip = 0;
    auto step = [&](Buffer &now, Buffer &next) {
      request(next);
      multiply(gbeg + c * U, gend, now, acc);
      if (++c < chunks) return;
      // columns 0..2 of a row, then the waves
      float(&r)[AMMON_WAVES][16] = red[flip];
      f32x4 sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = group_sum16(acc[i], 4);
      if ((lane & 15) == 0) *(f32x4 *)&r[wave][4 * (lane >> 4)] = sum;
      __syncthreads();
      finish(u, &r[0][0], pos, cand_v, cand_i);
      acc = f32x4{0.f, 0.f, 0.f, 0.f};
      c = 0;
      u += nwg;
      flip ^= 1;
    };
    for (uint32_t i = 0; i < total; i += 2) {
      step(bufs[0], bufs[1]);
      if (i + 1 < total) step(bufs[1], bufs[0]);
    }
    if (MODE == AMMON_GEMV_PLAIN_ARGMAX) {
      __syncthreads();
      block_cand_reduce(cand_v, cand_i, &red[0][0][0], (uint32_t *)&red[1][0][0]);
      if (threadIdx.x == 0) {
        st_out(p.cand_v + blockIdx.x, cand_v);
        st_out(p.cand_i + blockIdx.x, cand_i);
      }
    }
  }
};
