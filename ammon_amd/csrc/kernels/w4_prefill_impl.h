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

// RT panels of rows per wave x CT panels of tokens.  SPLIT 1: the workgroup's four waves have panels
// of their own; otherwise it has SPLIT waves, which split the groups of the same ones.
template <int DIGITS, int MODE, uint32_t RT, uint32_t CT, uint32_t SPLIT> struct W4Tile {
  static constexpr bool GATED = MODE == AMMON_GEMV_SWIGLU;
  static constexpr uint32_t RO = GATED ? RT / 2 : RT;                    // panels of results per wave
  static constexpr uint32_t RW = RO * (SPLIT == 1 ? AMMON_WAVES : 1);    // ... per workgroup
  static_assert(!GATED || RT % 2 == 0, "gate and up panels go together");

  ammon_k_gemm p;
  uint32_t lane, wave, groups, gbeg, gend, tok0;
  uint32_t panel[RT];           // virtual panel of results
  __amdgpu_buffer_rsrc_t w[RT]; // ... and its codes and scales
  __amdgpu_buffer_rsrc_t x;     // the tile's token panels
  uint32_t last;                // ... of which there are last + 1

  AMMON_DEV W4Tile(const ammon_k_gemm &p_, uint32_t rb, uint32_t tt, uint32_t ks) : p(p_) {
    begin();
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    groups = w4_groups(p.n);
    gbeg = 0, gend = groups;
    if (p.ksplit > 1) {
      gbeg = min(ks * p.kchunks, groups);
      gend = min(gbeg + p.kchunks, groups);
    }
    const uint32_t first = rb * RW + (SPLIT == 1 ? wave * RO : 0);
    if (SPLIT > 1) {  // as evenly as whole groups go
      const uint32_t n = gend - gbeg, per = n / SPLIT, more = n % SPLIT;
      gbeg += wave * per + min(wave, more);
      gend = gbeg + per + (wave < more ? 1 : 0);
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

  // This lane's place in a token panel's digits; past the last token, past the end (zeros, not read).
  AMMON_DEV uint32_t token_lane(uint32_t c) const {
    return tok0 + 16 * c + (lane & 15) < p.tokens ? lane * 16 : 0x80000000u;
  }

  // A group's operands straight from memory.
  struct Group {
    u32x4 a[RT];
    u32x2 s[RT];
    i32x4 b[CT][DIGITS][2];
    float sx[CT];
  };
  AMMON_DEV void load(uint32_t g, Group &o) const {
#pragma unroll
    for (uint32_t j = 0; j < RT; ++j) {
      o.a[j] = codes(j, g);
      o.s[j] = scales(j, g);
    }
#pragma unroll
    for (uint32_t c = 0; c < CT; ++c) {
#pragma unroll
      for (int d = 0; d < DIGITS; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          o.b[c][d][h] = __builtin_bit_cast(
              i32x4, __builtin_amdgcn_raw_buffer_load_b128(x, token_lane(c), digits_at(c, g, 2 * d + h), 0));
      o.sx[c] = __uint_as_float(
          __builtin_amdgcn_raw_buffer_load_b32(x, (lane & 15) * 4, scales_at(c) + g * 64, 0));
    }
  }
  AMMON_DEV void multiply(const Group &o, f32x4 (&acc)[RT][CT]) const {
#pragma unroll
    for (uint32_t j = 0; j < RT; ++j) {
      const i32x4 lo = w4_half0(o.a[j]), hi = w4_half1(o.a[j]);
      const float sw[4] = {bf16_lo(o.s[j][0]), bf16_hi(o.s[j][0]), bf16_lo(o.s[j][1]), bf16_hi(o.s[j][1])};
#pragma unroll
      for (uint32_t c = 0; c < CT; ++c) {
        i32x4 t[DIGITS];
#pragma unroll
        for (int d = 0; d < DIGITS; ++d)
          t[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo, o.b[c][d][0], start[d], 0, 0, 0);
#pragma unroll
        for (int d = 0; d < DIGITS; ++d)
          t[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi, o.b[c][d][1], t[d], 0, 0, 0);
        const float sx = o.sx[c] * 0.0625f;  // (the codes are 16 c)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[j][c][r] = fmaf(joined(t, r), sx * sw[r], acc[j][c][r]);
      }
    }
  }
  // Row r's sums of the digits as one number.  A digit's sum is at most 2^21: two of them fit a word,
  // and the lowest one of three starts at the bits of 1.5 2^23, so that it is that plus the sum
  // as a float already; the middle one starts at -1.5 2^23 / 256, which takes it off again: five
  // vector instructions for a sum in place of six (2048 tokens x 28672 x 4096 gated: 694 to 643 us).
  i32x4 start[DIGITS];
  AMMON_DEV void begin() {
#pragma unroll
    for (int d = 0; d < DIGITS; ++d) start[d] = i32x4{0, 0, 0, 0};
    if constexpr (DIGITS == 3) {
      start[0] = i32x4{0x4b400000, 0x4b400000, 0x4b400000, 0x4b400000};
      start[1] = i32x4{-49152, -49152, -49152, -49152};
      asm volatile("" : "+v"(start[0]), "+v"(start[1]));  // (kept in registers)
    }
  }
  AMMON_DEV static float joined(const i32x4 *t, int r) {
    if (DIGITS == 1) return (float)t[0][r];
    return fmaf((float)((t[DIGITS - 1][r] << 8) + t[DIGITS / 2][r]), 256.f, __int_as_float(t[0][r]));
  }

  AMMON_DEV void run(f32x4 (&acc)[RT][CT]) const {
#pragma unroll
    for (uint32_t j = 0; j < RT; ++j)
#pragma unroll
      for (uint32_t c = 0; c < CT; ++c) acc[j][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (gbeg >= gend) return;
    const uint32_t end = gend - 1;
    Group o0, o1;  // one multiplied, the next on its way
    load(gbeg, o0);
    for (uint32_t g = gbeg; g < gend; g += 2) {
      load(min(g + 1, end), o1);
      multiply(o0, acc);
      if (g + 1 >= gend) break;
      load(min(g + 2, end), o0);
      multiply(o1, acc);
    }
  }

  AMMON_DEV void store(const f32x4 (&acc)[RT][CT], uint32_t ks) const {
#pragma unroll
    for (uint32_t j = 0; j < RO; ++j)
#pragma unroll
      for (uint32_t c = 0; c < CT; ++c) put(panel[j], c, acc[j][c], acc[j + RT - RO][c], ks);
  }
  // A tile's results (gated: gate and up).
  AMMON_DEV void put(uint32_t pan, uint32_t c, const f32x4 &a, const f32x4 &up, uint32_t ks) const {
    const uint32_t t = tok0 + 16 * c + (lane & 15), v = 16 * pan + 4 * (lane >> 4);
    const bool split = p.ksplit > 1;
    if (t >= p.tokens) return;
    if (MODE == AMMON_GEMV_QKV && !split) {
#pragma unroll
      for (int i = 0; i < 4; i += 2)
        if (v + i < p.rows) qkv_store_pair(p, t, v + i, a[i], a[i + 1]);
      return;
    }
    const uint32_t width = split ? p.rows : p.d;
    float *y = (split ? p.ws + (size_t)ks * p.tokens * p.rows : p.y) + (size_t)t * width + v;
    const float *res = p.residual + (size_t)t * width + v;
    f32x4 out = a;
    if (GATED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = a[i] * (1.0f / (1.0f + expf(-a[i])));
        out[i] = f * up[i];
      }
    }
    const bool add = MODE == AMMON_GEMV_RESIDUAL && !split;
    if (v + 3 < width) {  // (at any float: the last rows of an odd matrix go one by one)
      if (add) out = *(const f32x4a4 *)res + out;
      *(f32x4a4 *)y = out;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i < width) y[i] = add ? res[i] + out[i] : out[i];
    }
  }
};

// Short prompts.  What bounds them is the digits' way from L2: a group's 1 KiB of codes meets 2 KiB
// of digits per digit and token panel, in every workgroup.  So workgroups have as many panels of
// rows as leave every CU one (16 tokens of three digits: 28672 x 4096 gated 22.9 us with one panel,
// 18.2 with two, 16.8 with four; 128256 x 4096 135, 94, 74; but 4096 x 4096 5.7, 7.9, 8.9), and
// tokens past the last one are not read (5 tokens: 24.0 to 20.1 us).  PANELS panels of results
// (gated: of each matrix) per workgroup, their groups split over SPLIT waves, whose sums meet in LDS
// and are added in wave order, a wave a panel and tokens'.
template <int DIGITS, int MODE, uint32_t PANELS, uint32_t CT, uint32_t SPLIT>
AMMON_DEV void w4_gemm_short(const ammon_k_gemm &p) {
  constexpr uint32_t RT = MODE == AMMON_GEMV_SWIGLU ? 2 * PANELS : PANELS;
  using T = W4Tile<DIGITS, MODE, RT, CT, SPLIT>;
  static_assert(PANELS * CT <= SPLIT, "a wave a panel and tokens'");
  __shared__ f32x4 part[SPLIT][RT][CT][64];
  // id = (eight blocks of rows, token tile, XCD): the token tiles of a block are adjacent on one XCD
  const uint32_t tiles = (p.tokens + 16 * CT - 1) / (16 * CT);
  const uint32_t q = blockIdx.x >> 3, tt = q % tiles, rb = (q / tiles) * 8 + (blockIdx.x & 7u);
  const uint32_t panels = ((T::GATED ? p.d : p.rows) + 15) / 16;
  if (rb * PANELS >= panels) return;  // padding of the last eight (uniform)
  T tile(p, rb, tt, 0);
  f32x4 acc[RT][CT];
  tile.run(acc);
#pragma unroll
  for (uint32_t j = 0; j < RT; ++j)
#pragma unroll
    for (uint32_t c = 0; c < CT; ++c) part[tile.wave][j][c][tile.lane] = acc[j][c];
  __syncthreads();
  if (tile.wave >= PANELS * CT) return;
  const uint32_t j = tile.wave % PANELS, c = tile.wave / PANELS;
  f32x4 sum[2];
#pragma unroll
  for (uint32_t m = 0; m < RT / PANELS; ++m) {
    sum[m] = part[0][j + m * PANELS][c][tile.lane];
#pragma unroll
    for (uint32_t w = 1; w < SPLIT; ++w) sum[m] += part[w][j + m * PANELS][c][tile.lane];
  }
  tile.put(rb * PANELS + j, c, sum[0], sum[RT / PANELS - 1], 0);
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

  // Groups that codes are requested ahead.  They come from farther away than the digits, and a
  // group of one digit is over sooner (28672 x 4096, 41 tokens: 26.8 us with 1, 22.9 with 2; of
  // three digits 8% slower with 2, for the registers).
  static constexpr uint32_t N = DIGITS == 1 ? 2 : 1;
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
        for (int r = 0; r < 4; ++r) acc[j][c][r] = fmaf(T::joined(u, r), sx[c & 1] * sw[j][r], acc[j][c][r]);
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
                                                      h ? u : this->start[d], 0, 0, 0);
          }
      if (step) add(step - 1);
      if (step) {
#pragma unroll
        for (int m = 0; m < 4 * DIGITS; ++m) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);                     // a matrix instruction
          __builtin_amdgcn_sched_group_barrier(0x2, DIGITS == 1 ? 6 : 3, 0);  // vector ones beside it
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
    const uint32_t end = this->gend - 1;
    A a[N + 1];
    load(this->gbeg, a[0]);
    stage(this->gbeg, lds);
    if (N == 2) load(min(this->gbeg + 1, end), a[1]);
    auto turn = [&](uint32_t g, const A &now, A &next, uint32_t b) {
      // group g's digits have landed (with N = 2, what was requested before the last codes)
      wait_vmcnt<N == 2 ? 2 * RT : 0>();
      __syncthreads();  // every wave's; the other buffer is consumed
      // (after the last group, that one again: no branch)
      stage(min(g + 1, end), lds + (b ^ 1) * BYTES);
      __builtin_amdgcn_sched_barrier(0);
      load(min(g + N, end), next);
      __builtin_amdgcn_sched_barrier(0);
      multiply(now, lds + b * BYTES, acc);
    };
    for (uint32_t g = this->gbeg, b = 0;; b ^= 1) {
      turn(g, a[0], a[N], b);
      if (++g >= this->gend) break;
      turn(g, a[1], a[0], b ^= 1);
      if (++g >= this->gend) break;
      if constexpr (N == 2) {
        turn(g, a[2], a[1], b ^= 1);
        if (++g >= this->gend) break;
      }
    }
    wait_vmcnt<0>();  // (requests into LDS end with the workgroup that made them)
  }
};

template <int DIGITS, int MODE, uint32_t RT, uint32_t CT> AMMON_DEV void w4_gemm_big(const ammon_k_gemm &p) {
  using T = W4Big<DIGITS, MODE, RT, CT>;
  __shared__ u32x4 lds[2 * T::BYTES / 16];
  // id = (eight (row block, reduction range), token tile, XCD): the token tiles of a row block's
  // range are adjacent on one XCD, whose L2 keeps its codes
  const uint32_t tiles = (p.tokens + 16 * CT - 1) / (16 * CT);
  const uint32_t ksplit = p.ksplit > 1 ? p.ksplit : 1;
  const uint32_t q = blockIdx.x >> 3, tt = q % tiles, rr = (q / tiles) * 8 + (blockIdx.x & 7u);
  const uint32_t blocks = (((T::GATED ? p.d : p.rows) + 15) / 16 + T::RW - 1) / T::RW;
  const uint32_t rb = rr % blocks, ks = rr / blocks;
  if (ks >= ksplit) return;  // padding of the last eight (uniform)
  T tile(p, rb, tt, ks);
  f32x4 acc[RT][CT];
  tile.run(acc, (char *)lds);
  tile.store(acc, ks);
}
