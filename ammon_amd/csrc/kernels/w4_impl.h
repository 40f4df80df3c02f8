// w4_impl.h -- 4-bit weights (AMMON_W4) and rows of 8-bit digits (AMMON_Q8, AMMON_Q24): their
// formats, read and written.  No counterpart in the reference, whose weights and rows are fp32.
//
// W4.  A matrix [d, n] in groups of 128 numbers of a row, the last one shorter: a scale s (bf16)
// and a code c in -8..7 per number, which stands for s c.  From numbers w, every step in fp32:
//     s = bf16(max |w| / 7), 0 where that is below 2^-126
//     c = clamp(rint(w (1 / s)), -7, 7), 0 where s = 0
// A group with a number that is not finite has s = NaN.
//
// Why so: codes are whole numbers and so are the digits of the rows they meet, so a group's
// products are summed by integer matrix instructions, exactly, and two nibbles become two signed
// bytes (16 c) by one AND, or a shift and an AND, for eight codes of a word at once -- the
// matrix instruction takes them as they are, where a floating-point form would take an
// instruction or more for each pair of codes.  bf16 scales have the weights' own range.
//
// Memory: panels of 16 rows, G = ceil(n / 128) groups; rows past d and numbers past n are zeros.
// A panel has its codes [G, 4 pieces, 16 rows, 16 bytes] -- byte b of piece j has number
// 32 j + b of the group in its low half and 32 j + 16 + b in its high half -- then its scales
// [4, G, 4], row 4 i + r of the panel at [i, g, r].  1056 G bytes a panel.  So the 16 rows x 128
// numbers of a group are 1 KiB in the order of a 16x16x64 matrix operand: lane l of a wave takes
// row l % 16 and piece l / 16, 16 bytes, one contiguous request a wave; and the scales that lane
// l needs beside its results (rows 4 (l / 16) .. + 3) are 8 bytes, one group after the other.
//
// Q8 and Q24.  Rows x [tokens, n] in blocks of 128 numbers, the last one shorter: a scale s
// (fp32) and a whole number q per number, which stands for s q:
//     Q8   s = max |x| / 127, 0 where that is below 2^-120; q = clamp(rint(x (1 / s)), -127, 127)
//     Q24  s the least power of two >= 2^-120 with max |x| < 127 2^16 s; q = rint(x / s)
// A block with a number that is not finite has s = NaN.  Q24 is off by at most 2^-22.9 of its
// block's largest number (or 2^-121): about the last bit of an fp32 that large.  q is one digit, or three,
// d0 + 256 d1 + 65536 d2, each in -128..127.
//
// Memory: panels of 16 tokens, B = ceil(n / 128) blocks: digits [B, digits, 2 halves, 4 pieces,
// 16 tokens, 16 bytes] -- byte b of half h and piece j is number 32 j + 16 h + b -- then scales
// [B, 16].  B (2048 digits + 64) bytes a panel.  A half is 1 KiB in the order of the other matrix
// operand: lane l token l % 16, piece l / 16.
#pragma once

#include "device_common.h"

#define W4_GROUP 128
#define W4_PANEL_BYTES 1056  // a panel's, per group
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

AMMON_DEV uint32_t w4_groups(uint32_t n) { return (n + W4_GROUP - 1) / W4_GROUP; }
// Bytes of a token panel per block.
AMMON_DEV constexpr uint32_t q8_block_bytes(uint32_t digits) { return 2048 * digits + 64; }

// A code word's (16 bytes of a lane) first and second half as signed bytes, 16 c.
AMMON_DEV i32x4 w4_half0(u32x4 w) {
  return __builtin_bit_cast(i32x4, (w << 4) & u32x4{0xf0f0f0f0u, 0xf0f0f0f0u, 0xf0f0f0f0u, 0xf0f0f0f0u});
}
AMMON_DEV i32x4 w4_half1(u32x4 w) {
  return __builtin_bit_cast(i32x4, w & u32x4{0xf0f0f0f0u, 0xf0f0f0f0u, 0xf0f0f0f0u, 0xf0f0f0f0u});
}

// The largest magnitude of 16 lanes' numbers x[0..7] as a bit pattern: the maximum of patterns,
// so that infinities and NaN (the largest patterns) win.
AMMON_DEV uint32_t abs_max16(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
#define ABS_MAX_STEP(CTRL) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, CTRL, 0xF, 0xF, false))
  ABS_MAX_STEP(AMMON_DPP_XOR1);
  ABS_MAX_STEP(AMMON_DPP_XOR2);
  ABS_MAX_STEP(AMMON_DPP_HALF_MIRROR);
  ABS_MAX_STEP(AMMON_DPP_MIRROR);
#undef ABS_MAX_STEP
  return m;
}

#define W4_NAN 0x7fc00000u
#define W4_INF 0x7f800000u

// A block of 128 numbers as 16 lanes make its digits: lane i has numbers 8 i .. + 7 (zeros past
// the end).  digits: eight bytes of each digit; returns the scale.
template <int DIGITS> AMMON_DEV float q8_digits(const float (&x)[8], uint2 (&digits)[DIGITS]) {
#pragma clang fp contract(off)
  const uint32_t top = abs_max16(x);
  const bool bad = top >= W4_INF;
  float s, inv;
  if (DIGITS == 1) {
    s = __uint_as_float(top) / 127.0f;
    s = s < 0x1p-120f ? 0.f : s;
    inv = s > 0.f ? 1.0f / s : 0.f;
  } else {
    // the exponent, one more where the fraction is at least 127 / 64
    const int k = max((int)((top + 0x20000u) >> 23) - 127 - (8 * DIGITS - 2), -120);
    s = __uint_as_float((uint32_t)(k + 127) << 23);
    inv = __uint_as_float((uint32_t)(127 - k) << 23);
  }
  // the digits of q as the bytes of a word: with 128 added to all but the highest they are what
  // carries leave, and flipping those top bits takes the 128 off again
  constexpr uint32_t BIAS = DIGITS == 4 ? 0x00808080u : DIGITS == 3 ? 0x00008080u : 0u;
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float f = rintf(x[e] * inv);
    if (DIGITS == 1) f = fminf(fmaxf(f, -127.f), 127.f);
    const uint32_t q = bad ? 0u : (uint32_t)(int)f;
    b[e] = (q + BIAS) ^ BIAS;
  }
  // four words' bytes, by digit
  auto four = [&](const uint32_t *w, uint32_t (&out)[4]) {
    // bytes of (y : x): x 0..3, y 4..7
    const uint32_t x01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);  // d0 d0' d1 d1'
    const uint32_t x23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    out[0] = __builtin_amdgcn_perm(x23, x01, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(x23, x01, 0x07060302u);
    const uint32_t y01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t y23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    out[2] = __builtin_amdgcn_perm(y23, y01, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(y23, y01, 0x07060302u);
  };
  uint32_t lo[4], hi[4];
  four(b, lo);
  four(b + 4, hi);
#pragma unroll
  for (int p = 0; p < DIGITS; ++p) digits[p] = make_uint2(lo[p], hi[p]);
  return bad ? __uint_as_float(W4_NAN) : s;
}

// A row of n numbers, read and written eight at a time through a buffer resource: past its end it
// reads as zeros and is not written, without a branch.  fp32, or bf16 as it lies (v[0]).
struct W4Row {
  __amdgpu_buffer_rsrc_t r;
  bool bf16, vec;  // vec: whole 16-byte pieces
  AMMON_DEV W4Row(const void *base, uint32_t dtype, uint32_t n) {
    bf16 = dtype == AMMON_K_BF16;
    r = make_rsrc(base, n * (bf16 ? 2 : 4));
    vec = bf16 ? (n & 7u) == 0 && ((uintptr_t)base & 3u) == 0 : (n & 3u) == 0;
  }
  AMMON_DEV void load(uint32_t c, u32x4 (&v)[2]) const {
    if (bf16) {
      if (vec) {
        v[0] = __builtin_amdgcn_raw_buffer_load_b128(r, 16 * c, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[0][e] = (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, 16 * c + 4 * e, 0, 0) |
                    (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, 16 * c + 4 * e + 2, 0, 0) << 16;
      }
      v[1] = u32x4{0, 0, 0, 0};
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (vec) {
          v[h] = __builtin_amdgcn_raw_buffer_load_b128(r, 32 * c + 16 * h, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[h][e] = __builtin_amdgcn_raw_buffer_load_b32(r, 32 * c + 16 * h + 4 * e, 0, 0);
        }
      }
    }
  }
  AMMON_DEV float number(const u32x4 (&v)[2], int e) const {
    if (!bf16) return __uint_as_float(v[e / 4][e % 4]);
    return e % 2 ? bf16_hi(v[0][e / 2]) : bf16_lo(v[0][e / 2]);
  }
  AMMON_DEV void store(uint32_t c, const u32x4 (&v)[2]) const {  // fp32
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (vec) {
        __builtin_amdgcn_raw_buffer_store_b128(v[h], r, 32 * c + 16 * h, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          __builtin_amdgcn_raw_buffer_store_b32(v[h][e], r, 32 * c + 16 * h + 4 * e, 0, 0);
      }
    }
  }
};
