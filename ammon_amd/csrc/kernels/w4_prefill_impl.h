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
  __amdgpu_buffer_rsrc_t w[RT]; // ... and its codes and scales
  __amdgpu_buffer_rsrc_t x;     // the tile's token panels
  uint32_t last;                // ... of which there are last + 1

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
      const void *const w0 = p.w0, *const w1 = p.w1, *const w2 = p.w2;
      const void *base = GATED && j >= RO ? w1 : w0;
      if (MODE == AMMON_GEMV_QKV) {
        const uint32_t q = p.d / 16, kv = p.kv_dim / 16;
        base = at >= q + kv ? w2 : at >= q ? w1 : w0;
        at -= at >= q + kv ? q + kv : at >= q ? q : 0;
      }
      w[j] = make_rsrc((const uint8_t *)base + at * bytes, (uint32_t)bytes);
    }
    tok0 = tt * 16 * CT;
    last = min(CT, (p.tokens + 15) / 16 - tt * CT) - 1;
    const size_t row = (size_t)groups * q8_block_bytes(DIGITS);
    x = make_rsrc((const uint8_t *)p.x + tt * CT * row, (uint32_t)((last + 1) * row));
  }

  // This lane's codes and scales of group g of its j-th panel of rows.
  AMMON_DEV u32x4 codes(uint32_t j, uint32_t g) const {
    return __builtin_amdgcn_raw_buffer_load_b128(w[j], lane * 16, g * 1024, 0);
  }
  AMMON_DEV u32x2 scales(uint32_t j, uint32_t g) const {
    return __builtin_amdgcn_raw_buffer_load_b64(w[j], (lane >> 4) * (groups * 8), groups * 1024 + g * 8, 0);
  }
  // Where half h of digit d of group g of token panel c is; past the last panel, that one's (not
  // stored).  And its scales.
  AMMON_DEV uint32_t digits_at(uint32_t c, uint32_t g, uint32_t half) const {
    return min(c, last) * (groups * q8_block_bytes(DIGITS)) + g * (2048 * DIGITS) + half * 1024;
  }
  AMMON_DEV uint32_t scales_at(uint32_t c) const {
    return min(c, last) * (groups * q8_block_bytes(DIGITS)) + groups * (2048 * DIGITS);
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
        a[j] = codes(j, g);
        s[j] = scales(j, g);
      }
#pragma unroll
      for (uint32_t c = 0; c < CT; ++c) {
        i32x4 b[DIGITS][2];
#pragma unroll
        for (int d = 0; d < DIGITS; ++d)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            b[d][h] = __builtin_bit_cast(
                i32x4, __builtin_amdgcn_raw_buffer_load_b128(x, lane * 16, digits_at(c, g, 2 * d + h), 0));
        const float sx = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(x, (lane & 15) * 4,
                                                                              scales_at(c) + g * 64, 0)) *
                         0.0625f;  // (the codes are 16 c)
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

// Long prompts: the same tiles with the tokens' digits staged in LDS, which the four waves share.
// Two buffers of a group's digits and scales, CT panels: the next group's are requested (straight
// into LDS; codes and weights' scales into registers) while the current one's are multiplied.
template <int DIGITS, int MODE, uint32_t RT, uint32_t CT> struct W4Big : W4Tile<DIGITS, MODE, RT, CT, 1> {
  using T = W4Tile<DIGITS, MODE, RT, CT, 1>;
  static constexpr uint32_t PIECES = CT * 2 * DIGITS;           // 1 KiB each
  static constexpr uint32_t BYTES = PIECES * 1024 + CT * 64;    // a buffer
  static_assert(PIECES % AMMON_WAVES == 0, "a wave's requests");
  static_assert(CT % 4 == 0, "scales' requests: four panels each");
  using T::T;

  struct A {
    u32x4 codes[RT];
    u32x2 scales[RT];
  };
  struct B {
    i32x4 half[DIGITS][2];
    float scale;
  };
  AMMON_DEV void load(uint32_t g, A &a) const {
#pragma unroll
    for (uint32_t j = 0; j < RT; ++j) {
      a.codes[j] = this->codes(j, g);
      a.scales[j] = this->scales(j, g);
    }
  }
#define W4_REQUEST(LANE, AT, TO, SIZE)                                                          \
  __builtin_amdgcn_raw_ptr_buffer_load_lds(                                                     \
      this->x, (__attribute__((address_space(3))) void *)(TO), SIZE, LANE, AT, 0, 0)
  AMMON_DEV void stage(uint32_t g, char *to) const {
    constexpr uint32_t PER = 2 * DIGITS;  // pieces of a panel
#pragma unroll
    for (uint32_t i = 0; i < PIECES / AMMON_WAVES; ++i) {
      const uint32_t at = i * AMMON_WAVES + this->wave;
      W4_REQUEST(this->lane * 16, this->digits_at(at / PER, g, at % PER), to + at * 1024, 16);
    }
    if (this->wave < CT / 4)
      W4_REQUEST(this->scales_at(this->wave * 4 + (this->lane >> 4)) + (this->lane & 15) * 4, g * 64,
                 to + PIECES * 1024 + this->wave * 256, 4);
  }
  AMMON_DEV void read(const char *buf, uint32_t c, B &b) const {
#pragma unroll
    for (int d = 0; d < DIGITS; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        b.half[d][h] = *(const i32x4 *)(buf + ((c * DIGITS + d) * 2 + h) * 1024 + this->lane * 16);
    b.scale = *(const float *)(buf + PIECES * 1024 + c * 64 + (this->lane & 15) * 4);
  }

  // Matrix and vector units side by side: while a step's two tiles are multiplied, the sums of the
  // step before are converted, scaled and added up.
  AMMON_DEV void multiply(const A &a, const char *buf, f32x4 (&acc)[RT][CT]) const {
    constexpr uint32_t S = RT / 2;  // steps of a token panel
    i32x4 lo[RT], hi[RT];
    float sw[RT][4];
    B b[2];
    read(buf, 0, b[0]);
#pragma unroll
    for (uint32_t j = 0; j < RT; ++j) {
      lo[j] = w4_half0(a.codes[j]);
      hi[j] = w4_half1(a.codes[j]);
      sw[j][0] = bf16_lo(a.scales[j][0]), sw[j][1] = bf16_hi(a.scales[j][0]);
      sw[j][2] = bf16_lo(a.scales[j][1]), sw[j][3] = bf16_hi(a.scales[j][1]);
    }
    i32x4 t[2][2][DIGITS];  // [step & 1][tile]
    float sx[2];            // [token panel & 1]
    auto add = [&](uint32_t step) {
      const uint32_t c = step / S;
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t j = step % S * 2 + i;
        const i32x4 *u = t[step & 1][i];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // (a digit's sum is at most 2^21: two of them fit a word)
          const float f = DIGITS == 1
                              ? (float)u[0][r]
                              : fmaf((float)((u[DIGITS - 1][r] << 8) + u[DIGITS / 2][r]), 256.f, (float)u[0][r]);
          acc[j][c][r] = fmaf(f, sx[c & 1] * sw[j][r], acc[j][c][r]);
        }
        // (added up here: the compiler moves it past the loop's branch else, and every tile's sums
        // wait in registers)
        asm volatile("" : "+v"(acc[j][c]));
      }
    };
#pragma unroll
    for (uint32_t step = 0; step < S * CT; ++step) {
      const uint32_t c = step / S;
      const B &now = b[c & 1];
      __builtin_amdgcn_sched_barrier(0);
      if (step % S == 0) {
        sx[c & 1] = now.scale * 0.0625f;  // (the codes are 16 c)
        if (c + 1 < CT) read(buf, c + 1, b[(c + 1) & 1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 0; d < DIGITS; ++d)
#pragma unroll
          for (uint32_t i = 0; i < 2; ++i) {
            const uint32_t j = step % S * 2 + i;
            i32x4 &u = t[step & 1][i][d];
            u = __builtin_amdgcn_mfma_i32_16x16x64_i8(h ? hi[j] : lo[j], now.half[d][h],
                                                      h ? u : i32x4{0, 0, 0, 0}, 0, 0, 0);
          }
      if (step) add(step - 1);
      if (step) {
#pragma unroll
        for (int m = 0; m < 4 * DIGITS; ++m) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);                     // a matrix instruction
          __builtin_amdgcn_sched_group_barrier(0x2, DIGITS == 1 ? 6 : 4, 0);  // vector ones beside it
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    add(S * CT - 1);
    __builtin_amdgcn_sched_barrier(0);
  }

  AMMON_DEV void run(f32x4 (&acc)[RT][CT], char *lds) const {
#pragma unroll
    for (uint32_t j = 0; j < RT; ++j)
#pragma unroll
      for (uint32_t c = 0; c < CT; ++c) acc[j][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (this->gbeg >= this->gend) return;
    A a0, a1;
    stage(this->gbeg, lds);
    load(this->gbeg, a0);
    const uint32_t last = this->gend - 1;
    auto turn = [&](uint32_t g, const A &now, A &next, uint32_t b) {
      wait_vmcnt<0>();
      __syncthreads();  // group g has landed; the other buffer is consumed
      // (after the last group, that one again: no branch)
      stage(min(g + 1, last), lds + (b ^ 1) * BYTES);
      load(min(g + 1, last), next);
      __builtin_amdgcn_sched_barrier(0);
      multiply(now, lds + b * BYTES, acc);
    };
    for (uint32_t g = this->gbeg; g < this->gend; g += 2) {
      turn(g, a0, a1, 0);
      if (g + 1 < this->gend) turn(g + 1, a1, a0, 1);
    }
    wait_vmcnt<0>();  // (requests into LDS end with the workgroup that made them)
  }
};

template <int DIGITS, int MODE, uint32_t RT, uint32_t CT> AMMON_DEV void w4_gemm_big(const ammon_k_gemm &p) {
  using T = W4Big<DIGITS, MODE, RT, CT>;
  __shared__ u32x4 lds[2 * T::BYTES / 16];
  const uint32_t tiles = (p.tokens + 16 * CT - 1) / (16 * CT);
  const uint32_t ksplit = p.ksplit > 1 ? p.ksplit : 1;
  const uint32_t q = blockIdx.x >> 3;
  const uint32_t tt = q % tiles, ks = (q / tiles) % ksplit;
  const uint32_t rb = (q / tiles / ksplit) * 8 + (blockIdx.x & 7u);
  const uint32_t panels = ((T::GATED ? p.d : p.rows) + 15) / 16;
  if (rb * T::RW >= panels) return;  // padding of the last group (uniform)
  T tile(p, rb, tt, ks);
  f32x4 acc[RT][CT];
  tile.run(acc, (char *)lds);
  tile.store(acc, ks);
}
