// w4_gemv_impl.h -- products of one token's row with 4-bit weights (w4_impl.h): the modes of
// gemv_impl.h (plain, residual, SwiGLU, QKV, argmax candidates) over AMMON_W4 matrices.
//
// y_r = sum_k W[r, k] x_k.  x (RMS-normalised where a weight is given) becomes whole numbers in
// LDS, once per workgroup: as Q24's, but of four digits (2^-31 of a block's largest number: exact
// next to the fp32 sums), since a matrix instruction has 16 columns and takes them for nothing.  A
// wave multiplies 16 rows x 128 numbers, 1 KiB of codes, by two v_mfma_i32_16x16x64_i8: the codes
// are operand A as they lie in memory but for an AND and a shift, and the digits are columns 0..3
// of operand B (the other columns repeat them and are not used).  A group's sums are exact; they
// are scaled by s_w s_x 256^digit, exact too, and added up over the groups in fp32 with one
// rounding each.
//
// A workgroup of NW waves has sets of KS.  A set takes a unit of 16 virtual rows (a panel; SwiGLU:
// 8 gate and the same 8 up rows) at a time; its waves take the chunks of U groups in turn, and
// their sums meet in LDS.  Each wave has two chunks in registers: one is multiplied while the other
// is on its way, and is then requested anew.
//
// The norm's factor is one for the whole row: it is applied to the results, so that the digits
// (of w x) do not wait for the sum of squares.
#pragma once

#include "argmax_impl.h"
#include "w4_impl.h"

template <int MODE, uint32_t KS, uint32_t NW> struct W4Gemv {
  static constexpr uint32_t U = AMMON_W4_CHUNK;  // groups a register buffer holds
  static constexpr uint32_t US = NW / KS;        // sets
  static constexpr uint32_t THREADS = 64 * NW;
  static constexpr int D = 4;

  ammon_k_gemv p;
  uint32_t lane, wave, set, groups, chunks;  // chunks: a wave's of a unit
  float factor;                      // the norm's
  uint8_t *digits;                   // LDS: [groups][2 halves][4 digits][64 bytes]
  float *scales;                     // LDS: [groups][4], s_x 256^digit / 16 (the codes are 16 c)
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

  // The groups of this wave's chunk c of a unit; past the last group, that one (x is zeros there).
  // Codes are read once; scales are parts of lines that other chunks read too and stay in the
  // caches (as nontemporal loads they cost 4-10% of a long matrix's time; as two 16-byte loads of
  // two groups each, where groups are even, nothing was gained).
  AMMON_DEV void load(const Unit &u, uint32_t c, Buffer &b) const {
    const uint32_t first = (c * KS + wave) * U;
#pragma unroll
    for (uint32_t i = 0; i < U; ++i) {
      const uint32_t g = min(first + i, groups - 1);
      b.codes[i] = __builtin_nontemporal_load((const u32x4 *)(u.codes + (size_t)g * 1024));
      b.scales[i] = *(const u32x2 *)(u.scales + (size_t)g * 8);
    }
  }

  AMMON_DEV void multiply(uint32_t c, const Buffer &b, f32x4 &acc) const {
    const uint32_t first = (c * KS + wave) * U, col = lane & 3, j = lane >> 4;
#pragma unroll
    for (uint32_t i = 0; i < U; ++i) {
      const uint8_t *d = digits + (first + i) * (2 * D * 64) + col * 64 + j * 16;
      const i32x4 b0 = *(const i32x4 *)d, b1 = *(const i32x4 *)(d + D * 64);
      i32x4 t = i32x4{0, 0, 0, 0};
      t = __builtin_amdgcn_mfma_i32_16x16x64_i8(w4_half0(b.codes[i]), b0, t, 0, 0, 0);
      t = __builtin_amdgcn_mfma_i32_16x16x64_i8(w4_half1(b.codes[i]), b1, t, 0, 0, 0);
      const float sx = scales[4 * (first + i) + col];
      const u32x2 s = b.scales[i];
      const float sw[4] = {bf16_lo(s[0]), bf16_hi(s[0]), bf16_lo(s[1]), bf16_hi(s[1])};
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = fmaf((float)t[r], sx * sw[r], acc[r]);
    }
  }

  // x as digits in LDS, normalised first where there is a weight; zeros up to whole rounds of
  // chunks.  Eights of x: R of a thread's are requested by begin() and kept in registers, the
  // others read again by each pass of stage().
  static constexpr int R = 2;
  struct Staged {
    u32x4 x[R][2], w[R][2];
  };
  AMMON_DEV void begin(Staged &s) const {
    const W4Row x(p.x, AMMON_K_F32, p.n), w(p.norm_w, p.norm_dtype, p.n);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      x.load(threadIdx.x + r * THREADS, s.x[r]);
      if (p.norm_w) w.load(threadIdx.x + r * THREADS, s.w[r]);
    }
  }
  AMMON_DEV static void square(const u32x4 (&v)[2], float &ss) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = __uint_as_float(v[h][e]);
        ss = fmaf(f, f, ss);
      }
  }
  AMMON_DEV void put(uint32_t c, const u32x4 (&x)[2], const W4Row &wr, const u32x4 (&w)[2]) const {
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = __uint_as_float(x[e / 4][e % 4]);
    if (p.norm_w) {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = wr.number(w, e) * h[e];
    }
    uint2 d[D];
    const float s = q8_digits<D>(h, d);
    const uint32_t g = c / 16, i = c & 15;
    uint8_t *at = digits + g * (2 * D * 64) + ((i >> 1) & 1) * (D * 64) + (i >> 2) * 16 + (i & 1) * 8;
#pragma unroll
    for (int k = 0; k < D; ++k) *(uint2 *)(at + 64 * k) = d[k];
    if (i == 0) *(float4 *)(scales + 4 * g) = make_float4(s * 0.0625f, s * 16.f, s * 4096.f, s * 1048576.f);
  }
  // (and, for a norm, the waves' sums of squares to red [NW])
  AMMON_DEV void stage(const Staged &st, float *red) const {
    const uint32_t tid = threadIdx.x, eights = chunks * KS * U * 16;
    const W4Row xr(p.x, AMMON_K_F32, p.n), wr(p.norm_w, p.norm_dtype, p.n);
    float ss = 0.f;
    // (a block's 16 lanes go together: eights and the stride are multiples of 16)
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (tid + r * THREADS < eights) {
        if (p.norm_w) square(st.x[r], ss);
        put(tid + r * THREADS, st.x[r], wr, st.w[r]);
      }
    for (uint32_t c = tid + R * THREADS; c < eights; c += THREADS) {
      u32x4 v[2], w[2];
      xr.load(c, v);
      if (p.norm_w) {
        wr.load(c, w);
        square(v, ss);
      }
      put(c, v, wr, w);
    }
    if (p.norm_w) {
      ss = wave_sum(ss);
      if (lane == 0) red[threadIdx.x >> 6] = ss;
    }
  }

  // Rows' sums of unit u, red [waves][16]: added in wave order, then the mode's epilogue, by one
  // wave.
  AMMON_DEV float row_sum(const float *red, uint32_t r) const {
    float v = red[r];
#pragma unroll
    for (uint32_t w = 1; w < KS; ++w) v += red[16 * w + r];
    return v * factor;
  }
  AMMON_DEV void finish(uint32_t u, const float *red, uint32_t pos, float &cand_v, uint32_t &cand_i) const {
    const uint32_t e = lane;
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
    __shared__ float red[2][US][KS][16], squares[NW];
    p = params;
    lane = threadIdx.x & 63;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wave = w % KS, set = w / KS;
    groups = w4_groups(p.n);
    chunks = (groups + KS * U - 1) / (KS * U);
    scales = (float *)lds;
    digits = lds + (size_t)chunks * KS * U * 16;
    uint32_t pos = 0;
    if (MODE == AMMON_GEMV_QKV) pos = p.step->position;

    // The sets of a workgroup take units blockIdx.x, + nwg, .. in pairs of US; steps are (unit,
    // chunk), and a set without a unit in the last one multiplies the last unit again, unheard.
    const uint32_t units = p.row_blocks, rounds = (units + nwg * US - 1) / (nwg * US);
    const uint32_t total = rounds * chunks;
    auto unit_of = [&](uint32_t round) { return (round * nwg + blockIdx.x) * US + set; };
    uint32_t lr = 0, lc = 0;  // the next request's round and chunk
    Unit at = unit(min(unit_of(0), units - 1));
    auto request = [&](Buffer &b) {
      load(at, lc, b);
      if (++lc == chunks) {
        lc = 0;
        at = unit(min(unit_of(++lr), units - 1));
      }
    };
    Staged st;
    begin(st);
    Buffer b0, b1;
    request(b0);
    if (total > 1) request(b1);
    stage(st, squares);
    __syncthreads();
    factor = 1.f;
    if (p.norm_w) {
      float ss = squares[0];
#pragma unroll
      for (uint32_t k = 1; k < NW; ++k) ss += squares[k];
      factor = 1.0f / sqrtf(ss / (float)p.n + p.eps);
    }
    float cand_v = 0.f;
    uint32_t cand_i = ARGMAX_NONE;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t round = 0, c = 0;
    auto step = [&](const Buffer &now) {
      multiply(c, now, acc);
      if (++c < chunks) return;
      // the four columns of a row, then the set's waves
      float(&r)[KS][16] = red[round & 1][set];
      f32x4 sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = group_sum16(acc[i], 4);
      if ((lane & 15) == 0) *(f32x4 *)&r[wave][4 * (lane >> 4)] = sum;
      if (KS > 1)
        __syncthreads();
      else
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (the wave's own)
      const uint32_t u = unit_of(round);
      if (wave == round % KS && u < units) finish(u, &r[0][0], pos, cand_v, cand_i);
      acc = f32x4{0.f, 0.f, 0.f, 0.f};
      c = 0;
      ++round;
    };
    uint32_t i = 0;
    for (; i + 3 < total; i += 2) {
      step(b0);
      request(b0);
      step(b1);
      request(b1);
    }
    step(b0);
    if (i + 2 < total) request(b0);
    if (i + 1 < total) step(b1);
    if (i + 2 < total) step(b0);
    if (MODE == AMMON_GEMV_PLAIN_ARGMAX) {
      // the workgroup's candidate
      __syncthreads();
      float *sv = &red[0][0][0][0];
      uint32_t *si = (uint32_t *)&red[1][0][0][0];
#pragma unroll
      for (int off = 32; off > 0; off >>= 1)
        cand_merge(cand_v, cand_i, __shfl_xor(cand_v, off, 64), __shfl_xor(cand_i, off, 64));
      if (lane == 0) sv[w] = cand_v, si[w] = cand_i;
      __syncthreads();
      if (threadIdx.x == 0) {
        for (uint32_t k = 1; k < NW; ++k) cand_merge(cand_v, cand_i, sv[k], si[k]);
        st_out(p.cand_v + blockIdx.x, cand_v);
        st_out(p.cand_i + blockIdx.x, cand_i);
      }
    }
  }
};
