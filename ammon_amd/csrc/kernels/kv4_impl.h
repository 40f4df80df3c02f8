// kv4_impl.h -- the 4-bit KV cache (AMMON_KV4): its format, read and written.  No
// counterpart in the reference, whose caches are fp32.
//
// Format.  A row (one kv head, one position) holds `head` numbers in groups of 32,
// the last one shorter where head is no multiple of 32.  Group j has a scale s and a
// bias b (fp16) and a code c in 0..15 per number, which stands for
// fp16(s (16 + c) + b), one rounding.  The offset 16 is what makes it cheap to
// read: the fp16 numbers 16..31 have one exponent and their four high mantissa bits
// are c, so code and constant are joined by one bitwise operation, and a packed fp16
// fused multiply-add gives two numbers.  From x, every step in fp32:
//     x = min(max(x, -16384), 16384)
//     s = fp16((max x - min x) / 15),  b = fp16(min x - 16 s)
//     c = clamp(rint((x - b) (1 / s) - 16), 0, 15), 0 where s = 0
// (|b| <= 16384 + 32 x 16384 / 15 is a finite fp16).  A group with a number that is
// not finite has s = b = NaN and so reads back as NaN.  What is lost: half a step of
// (max - min) / 15 per number, and 2^-11 each of the bias's and the number's size.
//
// Memory of one cache, NG = ceil(head / 32): the codes as 32-bit words [kv_heads,
// seq, 4, NG] -- word (p, j) has numbers 32 j + 8 p .. + 7 of the row, number + e in
// the bits 4 n.. with n = e / 2 (e even) or 4 + e / 2 (odd), so that one shift and
// mask gives two neighbours -- then s | b << 16 as [kv_heads, seq, NG].  20 NG bytes
// a row: 80 at head 128, where bf16 takes 256.
//
// Why the words are in the order (p, j): lane (position, p) of a score tile reads
// piece p of a row, 16 bytes at head 128, whose word j then has numbers of group j
// alone; lane i of a value tile reads word i of 8 positions, numbers of one group too.
#pragma once

#include "device_common.h"

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // at any float

#define KV4_LIMIT 16384.0f

AMMON_DEV uint32_t kv4_groups(uint32_t head) { return (head + 31) / 32; }

// Number + e of a word: its code's place.
constexpr int kv4_nibble(int e) { return e / 2 + 4 * (e & 1); }

// The mask of a code's bits in an fp16 mantissa and the fp16 number 16, twice, in
// registers of the two kinds that one v_and_or_b32 takes (as literals they were two
// instructions).
struct Kv4Bits {
  uint32_t mask = 0x03c003c0u, base = 0x4c004c00u;
  AMMON_DEV Kv4Bits() { asm("" : "+s"(mask), "+v"(base)); }
};

// Codes NIB nibbles up of a word's low and high half, as 16 + c.
template <int NIB> AMMON_DEV f16x2 kv4_pair(uint32_t w, const Kv4Bits &k) {
  const uint32_t at = NIB == 0 ? w << 6 : NIB == 1 ? w << 2 : NIB == 2 ? w >> 2 : w >> 6;
  return __builtin_bit_cast(f16x2, (at & k.mask) | k.base);
}

// The eight numbers of a word with scale | bias sb, in order.
AMMON_DEV f16x8 kv4_numbers(uint32_t w, uint32_t sb, const Kv4Bits &k) {
  const f16x2 p = __builtin_bit_cast(f16x2, sb);
  const f16x2 s = {p[0], p[0]}, b = {p[1], p[1]};
  const f16x2 v0 = __builtin_elementwise_fma(kv4_pair<0>(w, k), s, b);
  const f16x2 v1 = __builtin_elementwise_fma(kv4_pair<1>(w, k), s, b);
  const f16x2 v2 = __builtin_elementwise_fma(kv4_pair<2>(w, k), s, b);
  const f16x2 v3 = __builtin_elementwise_fma(kv4_pair<3>(w, k), s, b);
  return f16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

// Two floats as fp16 hi + lo, 22 bits: lo by one mixed-precision multiply-add each (the
// factor is hidden from the compiler, which would make a conversion and a subtraction).
AMMON_DEV void kv4_parts(float a, float b, float minus1, f16x2 &hi, f16x2 &lo) {
  hi = __builtin_convertvector(f32x2{a, b}, f16x2);
  lo = __builtin_convertvector(
      f32x2{__builtin_fmaf((float)hi[0], minus1, a), __builtin_fmaf((float)hi[1], minus1, b)}, f16x2);
}
AMMON_DEV float kv4_minus1() {
  float f = -1.f;
  asm("" : "+s"(f));
  return f;
}

// A weight's exponent is a score times a scale, less a reference maximum m.  As one fused
// multiply-add it differs from 0 at the maximum itself by as much as m was rounded, at
// |m| = 2^24 by 1: fp16 parts of the weights then overflow, or vanish.  Past KV4_FAR the
// product is rounded as the maximum was, and the difference is exact where it matters.
// (By a branch of its own ahead of the exponentials, which costs 0.4% of a decode step and
// nothing measurable of a prompt; with the exponentials in both arms 2% of a prompt.)
#define KV4_FAR 0x1p22f
AMMON_DEV float kv4_distance(float score, float scale, float m) {
#pragma clang fp contract(off)
  return score * scale - m;
}

// A row as 16 lanes quantise it: lane i (of aligned 16) has numbers 8 i .. + 7 in x
// (zeros past the head), its word and, in the four lanes of a group alike, scale | bias.
AMMON_DEV void kv4_quantise(const float (&x)[8], uint32_t i, uint32_t head, uint32_t &word,
                            uint32_t &sb) {
#pragma clang fp contract(off)
  float lo = INFINITY, hi = -INFINITY, z = 0.f, y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    z += x[e] * 0.f;  // NaN where a number is not finite
    y[e] = fminf(fmaxf(x[e], -KV4_LIMIT), KV4_LIMIT);
    if (8 * i + e < head) {
      lo = fminf(lo, y[e]);
      hi = fmaxf(hi, y[e]);
    }
  }
  lo = fminf(lo, dpp_get<AMMON_DPP_XOR1>(lo));
  hi = fmaxf(hi, dpp_get<AMMON_DPP_XOR1>(hi));
  z += dpp_get<AMMON_DPP_XOR1>(z);
  lo = fminf(lo, dpp_get<AMMON_DPP_XOR2>(lo));
  hi = fmaxf(hi, dpp_get<AMMON_DPP_XOR2>(hi));
  z += dpp_get<AMMON_DPP_XOR2>(z);
  const _Float16 s = (_Float16)((hi - lo) / 15.0f);
  const float sf = (float)s;
  const _Float16 b = (_Float16)(lo - 16.0f * sf);
  const float bf = (float)b, inv = sf > 0.f ? 1.0f / sf : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float c = fminf(fmaxf(rintf((y[e] - bf) * inv - 16.0f), 0.f), 15.f);
    w |= (8 * i + e < head ? (uint32_t)c : 0u) << (4 * kv4_nibble(e));
  }
  const bool ok = z == 0.f;
  word = ok ? w : 0u;
  sb = ok ? (uint32_t)__builtin_bit_cast(uint16_t, s) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16
          : 0x7e007e00u;
}

// Numbers 8 (i + 4 j) .. + 7 of an fp32 row, j < N, zeros past the head: every load is
// requested before any is used, and a lane past the head reads the last numbers (a branch
// or a select between the loads had them wait for each other: 1 us in a decode step).
template <int N>
AMMON_DEV void kv4_rows(const float *row, uint32_t i, uint32_t head, float (&x)[N][8]) {
  if (head % 8 == 0) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint32_t at = min(8 * (i + 4 * j), head - 8);
      const f32x4_any a = *(const f32x4_any *)(row + at), b = *(const f32x4_any *)(row + at + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] = e < 4 ? a[e] : b[e - 4];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) x[j][e] = ld_in(row + min(8 * (i + 4 * j) + e, head - 1));
    // (they are waited for here: left pending, they would be in the other path's waits too)
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(x[j][e]));
  }
}
// ... and the zeros, once they are to be used.
template <int N> AMMON_DEV void kv4_row_ends(uint32_t i, uint32_t head, float (&x)[N][8]) {
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) x[j][e] = 8 * (i + 4 * j) + e < head ? x[j][e] : 0.f;
}

// Where row (g, t) of a cache has its words and its scales | biases.
AMMON_DEV uint32_t *kv4_codes(const void *cache, uint32_t seq, uint32_t ng, uint32_t g, uint32_t t) {
  return (uint32_t *)cache + ((size_t)g * seq + t) * (4 * ng);
}
AMMON_DEV uint32_t *kv4_scales(const void *cache, uint32_t kv_heads, uint32_t seq, uint32_t ng,
                               uint32_t g, uint32_t t) {
  return (uint32_t *)cache + (size_t)kv_heads * seq * (4 * ng) + ((size_t)g * seq + t) * ng;
}

// Lane i's part (numbers 8 i .. + 7 in x) of row (g, t) written to the cache.
AMMON_DEV void kv4_put(void *cache, uint32_t kv_heads, uint32_t seq, uint32_t head, uint32_t g,
                       uint32_t t, uint32_t i, const float (&x)[8]) {
  uint32_t word, sb;
  kv4_quantise(x, i, head, word, sb);
  const uint32_t ng = kv4_groups(head), j = i >> 2, piece = i & 3;
  if (j >= ng) return;
  kv4_codes(cache, seq, ng, g, t)[piece * ng + j] = word;
  if (piece == 0) kv4_scales(cache, kv_heads, seq, ng, g, t)[j] = sb;
}
