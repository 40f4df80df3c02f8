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
// A unit is 16 virtual rows (a panel; SwiGLU: 8 gate and the same 8 up rows).  Two ways share the
// units out:
//
// W4Sets, workgroups of NW waves in sets of KS.  A set takes a unit at a time; its waves take the
// chunks of U groups in turn, and their sums meet in LDS.  Each wave has two chunks in registers:
// one is multiplied while the other is on its way, and is then requested anew.
//
// W4Flat, one workgroup of 16 waves a CU, so that x is read and turned into digits once a CU.  Each
// wave takes a sixteenth of the groups of all the workgroup's units, one after the other: no CU has
// idle waves, and no wave waits for another before the end.  A wave's part of a unit is a piece in
// LDS; at the end every row adds up its pieces in the waves' order.
//
// The norm's factor is one for the whole row: it is applied to the results, so that the digits
// (of w x) do not wait for the sum of squares.
#pragma once

#include "argmax_impl.h"
#include "w4_impl.h"

// What a workgroup of NW waves has of either.
template <int MODE, uint32_t NW> struct W4Token {
  static constexpr uint32_t THREADS = 64 * NW;
  static constexpr int D = 4;

  ammon_k_gemv p;
  uint32_t lane, w, groups;  // w: the wave
  float factor;              // the norm's
  uint8_t *digits;  // LDS: [groups][2 halves][4 digits][64 bytes], half 1 from digit 3 on
  float *scales;    // LDS: [groups][4], s_x 256^digit / 16 (the codes are 16 c)

  // staged: groups that x is laid out for
  AMMON_DEV void start(const ammon_k_gemv &params, uint8_t *lds, uint32_t staged) {
    p = params;
    lane = threadIdx.x & 63;
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    groups = w4_groups(p.n);
    scales = (float *)lds;
    digits = lds + (size_t)staged * 16;
  }

  // Adds a group's products to a lane's four rows.
  AMMON_DEV void multiply(uint32_t g, const u32x4 &codes, const u32x2 &s, f32x4 &acc) const {
    const uint32_t col = lane & 3, j = lane >> 4;
    const uint8_t *d = digits + g * (2 * D * 64) + j * 16;
    const i32x4 b0 = *(const i32x4 *)(d + col * 64), b1 = *(const i32x4 *)(d + D * 64 + ((col + 1) & 3) * 64);
    i32x4 t = i32x4{0, 0, 0, 0};
    t = __builtin_amdgcn_mfma_i32_16x16x64_i8(w4_half0(codes), b0, t, 0, 0, 0);
    t = __builtin_amdgcn_mfma_i32_16x16x64_i8(w4_half1(codes), b1, t, 0, 0, 0);
    const float sx = scales[4 * g + col];
    const float sw[4] = {bf16_lo(s[0]), bf16_hi(s[0]), bf16_lo(s[1]), bf16_hi(s[1])};
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] = fmaf((float)t[r], sx * sw[r], acc[r]);
  }

  // x as digits in LDS, times the norm's weight where there is one; zeros past its end.  Eights of
  // x: R of a thread's are requested by begin(), before the matrix (whose loads are answered in
  // order), and kept in registers, if they can be read in whole pieces; others are read by stage().
  static constexpr int R = 2;
  struct Staged {
    u32x4 x[R][2], w[R][2];
  };
  AMMON_DEV bool normed() const { return MODE != AMMON_GEMV_RESIDUAL && p.norm_w; }
  AMMON_DEV bool whole() const {
    return W4Row(p.x, AMMON_K_F32, p.n).vec && (!normed() || W4Row(p.norm_w, p.norm_dtype, p.n).vec);
  }
  AMMON_DEV void begin(Staged &s) const {
    const bool v = whole(), bf = p.norm_dtype == AMMON_K_BF16;
    const __amdgpu_buffer_rsrc_t x = make_rsrc(p.x, v ? p.n * 4 : 0);
    const __amdgpu_buffer_rsrc_t nw = make_rsrc(p.norm_w, v ? p.n * (bf ? 2 : 4) : 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r > 0 && r * THREADS * 8 >= p.n) break;
      const uint32_t c = threadIdx.x + r * THREADS;
      s.x[r][0] = __builtin_amdgcn_raw_buffer_load_b128(x, 32 * c, 0, 0);
      s.x[r][1] = __builtin_amdgcn_raw_buffer_load_b128(x, 32 * c + 16, 0, 0);
      if (normed()) {
        s.w[r][0] = __builtin_amdgcn_raw_buffer_load_b128(nw, (bf ? 16 : 32) * c, 0, 0);
        if (!bf) s.w[r][1] = __builtin_amdgcn_raw_buffer_load_b128(nw, 32 * c + 16, 0, 0);
      }
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
    if (normed()) {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = wr.number(w, e) * h[e];
    }
    uint2 d[D];
    const float s = q8_digits<D>(h, d);
    const uint32_t g = c / 16, i = c & 15;
    // (half 1 is turned by a digit, so that a store's lanes meet all banks)
    const uint32_t half = (i >> 1) & 1;
    uint8_t *at = digits + g * (2 * D * 64) + half * (D * 64) + (i >> 2) * 16 + (i & 1) * 8;
#pragma unroll
    for (uint32_t k = 0; k < D; ++k) *(uint2 *)(at + 64 * ((k + half) & 3)) = d[k];
    if (i == 0) *(float4 *)(scales + 4 * g) = make_float4(s * 0.0625f, s * 16.f, s * 4096.f, s * 1048576.f);
  }
  // (of `staged` groups; and, for a norm, the waves' sums of squares to red [NW])
  AMMON_DEV void stage(const Staged &st, uint32_t staged, float *red) const {
    const uint32_t tid = threadIdx.x, eights = staged * 16;
    const W4Row xr(p.x, AMMON_K_F32, p.n), wr(p.norm_w, p.norm_dtype, p.n);
    float ss = 0.f;
    // (a block's 16 lanes go together: eights and the stride are multiples of 16)
    const bool v = whole();
    if (v) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (tid + r * THREADS < eights) {
          if (normed()) square(st.x[r], ss);
          put(tid + r * THREADS, st.x[r], wr, st.w[r]);
        }
    }
    for (uint32_t c = tid + (v ? R * THREADS : 0); c < eights; c += THREADS) {
      u32x4 x[2], nw[2] = {};
      xr.load(c, x);
      if (normed()) {
        wr.load(c, nw);
        square(x, ss);
      }
      put(c, x, wr, nw);
    }
    if (normed()) {
      ss = wave_sum(ss);
      if (lane == 0) red[w] = ss;
    }
  }

  // The norm's factor, from the waves' sums of squares.
  AMMON_DEV void scale(const float *red) {
    factor = 1.f;
    if (!normed()) return;
    float ss = red[0];
#pragma unroll
    for (uint32_t k = 1; k < NW; ++k) ss += red[k];
    factor = 1.0f / sqrtf(ss / (float)p.n + p.eps);
  }

  // The epilogue of unit u's row e, whose sum (and, SwiGLU, whose up row's) is given; QKV: of rows
  // 2 e and 2 e + 1.
  AMMON_DEV void finish(uint32_t u, uint32_t e, float a0, float a1, uint32_t pos, float &cand_v,
                        uint32_t &cand_i) const {
    if (MODE == AMMON_GEMV_SWIGLU) {
      if (8 * u + e >= p.d) return;
      const float gate = a0, up = a1;
      float v = gate * (1.0f / (1.0f + expf(-gate)));
      v = v * up;
      st_out(p.y + 8 * u + e, v);
    } else if (MODE == AMMON_GEMV_QKV) {
#pragma clang fp contract(off)
      const uint32_t vr = 16 * u + 2 * e;
      if (vr >= p.rows) return;
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
      if (vr >= p.rows) return;
      const float v = a0;
      st_out(p.y + vr, MODE == AMMON_GEMV_RESIDUAL ? ld_in(p.residual + vr) + v : v);
      if (MODE == AMMON_GEMV_PLAIN_ARGMAX && v == v) cand_merge(cand_v, cand_i, v, vr);
    }
  }

  // The workgroup's candidate of its threads'; sv, si: NW entries in LDS that nothing else uses now.
  AMMON_DEV void candidate(float cand_v, uint32_t cand_i, float *sv, uint32_t *si) const {
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
};

// ONE: a wave has one chunk of one unit (as a branch around the second request this costs the long
// matrices 2-4%: the wait for x then includes the first chunk).
template <int MODE, uint32_t KS, uint32_t NW, bool ONE> struct W4Sets : W4Token<MODE, NW> {
  using T = W4Token<MODE, NW>;
  using T::p, T::lane, T::w, T::groups;
  static constexpr uint32_t U = AMMON_W4_CHUNK;  // groups a register buffer holds
  static constexpr uint32_t US = NW / KS;        // sets
  static_assert(KS > 1 && NW % KS == 0, "sets of several waves");
  uint32_t wave, set, chunks;                    // of the set; chunks: a wave's of a unit

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
    const uint32_t first = (c * KS + wave) * U;
#pragma unroll
    for (uint32_t i = 0; i < U; ++i) T::multiply(first + i, b.codes[i], b.scales[i], acc);
  }

  // Unit u's rows, red [waves][16]: added in wave order, then the epilogue, by one wave.
  AMMON_DEV float row_sum(const float *red, uint32_t r) const {
    float v = red[r];
#pragma unroll
    for (uint32_t k = 1; k < KS; ++k) v += red[16 * k + r];
    return v * T::factor;
  }
  AMMON_DEV void rows(uint32_t u, const float *red, uint32_t pos, float &cand_v, uint32_t &cand_i) const {
    const uint32_t e = lane;
    if (MODE == AMMON_GEMV_SWIGLU) {
      if (e < 8) T::finish(u, e, row_sum(red, e), row_sum(red, 8 + e), pos, cand_v, cand_i);
    } else if (MODE == AMMON_GEMV_QKV) {
      if (e < 8) T::finish(u, e, row_sum(red, 2 * e), row_sum(red, 2 * e + 1), pos, cand_v, cand_i);
    } else {
      if (e < 16) T::finish(u, e, row_sum(red, e), 0.f, pos, cand_v, cand_i);
    }
  }

  AMMON_DEV void run(const ammon_k_gemv &params, uint32_t nwg, uint8_t *lds) {
    __shared__ float red[2][US][KS][16], squares[NW];
    chunks = (w4_groups(params.n) + KS * U - 1) / (KS * U);
    T::start(params, lds, chunks * KS * U);
    wave = w % KS, set = w / KS;
    typename T::Staged st;
    T::begin(st);
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
    Buffer b0, b1;
    request(b0);
    if (!ONE) request(b1);
    T::stage(st, chunks * KS * U, squares);
    __syncthreads();
    T::scale(squares);
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
      __syncthreads();
      const uint32_t u = unit_of(round);
      if (wave == round % KS && u < units) rows(u, &r[0][0], pos, cand_v, cand_i);
      acc = f32x4{0.f, 0.f, 0.f, 0.f};
      c = 0;
      ++round;
    };
    if (ONE) {
      step(b0);
    } else {
      uint32_t i = 0;
      for (; i + 3 < total; i += 2) {
        step(b0);
        request(b0);
        step(b1);
        request(b1);
      }
      step(b0);
      if (i + 2 < total) request(b0);
      step(b1);
      if (i + 2 < total) step(b0);
    }
    if (MODE == AMMON_GEMV_PLAIN_ARGMAX) {
      __syncthreads();
      T::candidate(cand_v, cand_i, &red[0][0][0][0], (uint32_t *)&red[1][0][0][0]);
    }
  }
};

template <int MODE> struct W4Flat : W4Token<MODE, 16> {
  static constexpr uint32_t NW = 16;
  using T = W4Token<MODE, NW>;
  using T::p, T::lane, T::w, T::groups;
  // groups a wave has in registers (4096 x 14336: 8.4 us, 6 8.6, 8 9.3; 10240 x 8192: 10.4, 11.1, 11.6)
  static constexpr uint32_t RING = 4;
  static constexpr uint32_t MOST = AMMON_W4_UNITS;  // units of a workgroup

  uint32_t nwg;

  struct Group {
    u32x4 codes;
    u32x2 scales;
  };
  // The groups of the workgroup's units, one after the other.  All of it is the wave's (scalar
  // registers); a lane adds its own offsets.
  struct Cursor {
    const uint8_t *codes, *scales;
    uint32_t unit, group, left;  // unit: of the workgroup's; left: groups still to be requested
  };
  ptrdiff_t lane_codes, lane_scales;  // SWIGLU's up rows: in the other matrix

  AMMON_DEV void lanes() {
    const uint32_t j = lane >> 4, row = lane & 15;
    if (MODE == AMMON_GEMV_SWIGLU) {
      // rows 0..7 gate, 8..15 up; results' quads 0, 1 gate, 2, 3 up
      const ptrdiff_t up = (const uint8_t *)p.w1 - (const uint8_t *)p.w0;
      lane_codes = j * 256 + (row & 7) * 16 + (row < 8 ? 0 : up);
      lane_scales = (j & 1) * groups * 8 + (j < 2 ? 0 : up);
    } else {
      lane_codes = j * 256 + row * 16;
      lane_scales = j * groups * 8;
    }
  }
  AMMON_DEV uint32_t unit_of(uint32_t u) const { return blockIdx.x + u * nwg; }
  AMMON_DEV void place(Cursor &c) const {
    const uint32_t u = unit_of(c.unit), half = MODE == AMMON_GEMV_SWIGLU ? u & 1 : 0;
    const void *const w0 = p.w0, *const w1 = p.w1, *const w2 = p.w2, *base = w0;
    uint32_t panel = MODE == AMMON_GEMV_SWIGLU ? u >> 1 : u;
    if (MODE == AMMON_GEMV_QKV) {
      const uint32_t q = p.d / 16, kv = p.kv_dim / 16;
      base = u >= q + kv ? w2 : u >= q ? w1 : w0;
      panel -= u >= q + kv ? q + kv : u >= q ? q : 0;
    }
    const uint8_t *at = (const uint8_t *)base + (size_t)panel * (groups * W4_PANEL_BYTES);
    c.codes = at + half * 128 + (size_t)c.group * 1024;
    c.scales = at + (size_t)groups * 1024 + half * groups * 16 + c.group * 8;
  }

  // The next group; after the last one, that one again.
  // Codes are read once; scales are parts of lines that other groups read too and stay in the
  // caches (as nontemporal loads they cost 4-10% of a long matrix's time).
  AMMON_DEV void request(Cursor &c, Group &g) const {
    g.codes = __builtin_nontemporal_load((const u32x4 *)(c.codes + lane_codes));
    g.scales = *(const u32x2 *)(c.scales + lane_scales);
    const uint32_t more = min(c.left - 1, 1u);
    c.left -= more;
    c.codes += 1024 * more;
    c.scales += 8 * more;
    c.group += more;
    if (c.group == groups) {
      c.group = 0;
      ++c.unit;
      place(c);
    }
  }

  AMMON_DEV void run(const ammon_k_gemv &params, uint32_t grid, uint8_t *lds) {
    // pieces of units: a wave's of the workgroup's unit u is w + u (both only grow along the groups)
    __shared__ float pieces[NW + MOST][2][16];  // [..][digits 0, 1 and 2, 3]
    __shared__ float squares[NW];
    T::start(params, lds, w4_groups(params.n));
    nwg = grid;
    typename T::Staged st;
    T::begin(st);
    lanes();
    // units (at most MOST, by the launch's rule) and groups; the wave's
    const uint32_t here = (p.row_blocks - blockIdx.x + nwg - 1) / nwg, total = here * groups;
    const uint32_t from = w * total / NW, count = (w + 1) * total / NW - from;
    const uint32_t unit = w * here / NW;  // from / groups
    Cursor c = {nullptr, nullptr, unit, from - unit * groups, max(count, 1u)};
    uint32_t at = w + unit, g = c.group;
    place(c);
    Group ring[RING];
#pragma unroll
    for (uint32_t i = 0; i < RING; ++i) request(c, ring[i]);
    uint32_t pos = 0;
    T::stage(st, groups, squares);
    if (MODE == AMMON_GEMV_QKV) pos = p.step->position;
    __syncthreads();
    T::scale(squares);
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    auto flush = [&] {
      f32x4 sum;  // (all lanes write, those of the same columns the same)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = group_sum16(acc[i], 2);
      *(f32x4 *)&pieces[at][(lane >> 1) & 1][4 * (lane >> 4)] = sum;
      acc = f32x4{0.f, 0.f, 0.f, 0.f};
      ++at;
      g = 0;
    };
    auto next = [&](const Group &now) {
      T::multiply(g, now.codes, now.scales, acc);
      // (sums that sink below the request keep its registers, and copies then wait for it)
      asm volatile("" : "+v"(acc));
      if (++g == groups) flush();
    };
    uint32_t k = 0;
    for (; k + 2 * RING <= count; k += RING) {
#pragma unroll
      for (uint32_t i = 0; i < RING; ++i) {
        next(ring[i]);
        request(c, ring[i]);
      }
    }
    // fewer than RING to be requested
#pragma unroll
    for (uint32_t i = 0; i < RING; ++i)
      if (k + i < count) {
        next(ring[i]);
        if (k + RING + i < count) request(c, ring[i]);
      }
    k += RING;
#pragma unroll
    for (uint32_t i = 0; i < RING; ++i)
      if (k + i < count) next(ring[i]);
    if (g != 0 || count == 0) flush();
    __syncthreads();

    // rows: 16 threads a unit; SwiGLU and QKV 8, each with two
    constexpr uint32_t ROWS = MODE == AMMON_GEMV_SWIGLU || MODE == AMMON_GEMV_QKV ? 8 : 16;
    const uint32_t u = threadIdx.x / ROWS, e = threadIdx.x % ROWS;
    float cand_v = 0.f;
    uint32_t cand_i = ARGMAX_NONE;
    if (u < here) {
      // the waves that have a unit's first and last group: the last w with w total / NW <= it, that
      // is (u NW + (NW - 1) / groups) / here and ((u + 1) NW - 1) / here (below 2^11: exact so)
      const float by = 1.f / (float)here;
      const uint32_t w0 = ((float)(u * NW + (groups >= NW ? 0 : (NW - 1) / groups)) + 0.5f) * by;
      const uint32_t w1 = ((float)(u * NW + NW - 1) + 0.5f) * by;
      const uint32_t r0 = MODE == AMMON_GEMV_QKV ? 2 * e : e, r1 = MODE == AMMON_GEMV_QKV ? 2 * e + 1 : 8 + e;
      float a0 = 0.f, a1 = 0.f;
      for (uint32_t v = w0; v <= w1; v += 4) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const float(&piece)[2][16] = pieces[min(v + i, w1) + u];
          const float v0 = piece[0][r0] + piece[1][r0], v1 = ROWS == 8 ? piece[0][r1] + piece[1][r1] : 0.f;
          a0 += v + i <= w1 ? v0 : 0.f;
          a1 += v + i <= w1 ? v1 : 0.f;
        }
      }
      T::finish(unit_of(u), e, a0 * T::factor, a1 * T::factor, pos, cand_v, cand_i);
    }
    if (MODE == AMMON_GEMV_PLAIN_ARGMAX) {
      __syncthreads();
      T::candidate(cand_v, cand_i, &pieces[0][0][0], (uint32_t *)&pieces[1][0][0]);
    }
  }
};
