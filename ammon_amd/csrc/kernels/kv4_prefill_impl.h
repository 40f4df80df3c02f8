// kv4_prefill_impl.h -- attention of many consecutive query tokens (prompt prefill)
// over a KV4 cache (kv4_impl.h), on matrix cores.
//
// As in attention_prefill_impl.h, the query rows (token, head of the group) of one kv
// head are tiled, 32 per wave, over a range of positions in chunks of 64; scores are
// computed as S^T, whose registers are the value product's B operand as they stand; the
// reference maximum moves by PF_SLACK or more.  What differs:
//
// K and V are expanded once per chunk and workgroup: codes and scales are loaded into
// registers one chunk ahead and written to LDS as fp16 numbers.  fp16 parts carry 11
// bits, so q and the weights take two each (bf16: two and three): 4 products per (row,
// position) pair and dimension, not 5.  q is scaled by a power of two per row, and the
// weights are up to 2^15, so that the low parts are no subnormals where they matter.
//
// Two groups of four waves, one wave of each per SIMD, take turns: while one multiplies
// (the value products of its chunk, then the scores of the next: 64 matrix instructions
// at head 128, 2050 cycles), the other does what is left to the vector unit (softmax, the
// weights' parts, and its share of expanding: the first group the keys, the second the
// values, some 290 instructions).  A barrier ends each turn.  Two workgroups of four waves
// per CU that run as they come took 4.2 us for a chunk of 2 x 128 rows, twice what one
// takes alone; taking turns, 256 rows take 2.3 us (alone; 3.1 with every CU at it).
//
//   turn     2 c              2 c + 1          2 c + 2
//   first    PV c-1, QK c     softmax c        PV c, QK c+1
//                             expand K c+1
//   second   softmax c-1      PV c-1, QK c     softmax c
//            expand V c                        expand V c+1
//
// So K c and V c each need two buffers (c's parity).
//
// What bounds it: alone, a turn is 2700 cycles, of which the matrix unit is busy 2050 and
// the issue of vector instructions (386 of both waves, and some 12 cycles for every matrix
// instruction) 2300.  With every CU at it a turn takes 3600 cycles, starts and ends
// included (301 tokens after 7001): the matrix unit is busy 58% of them, vector issue 54%.
// At head 128 the kernel has all 256 registers and spills 14 (60 bytes of scratch a lane),
// some of which come back in the chunk loop.  Measured, 32 q / 8 kv heads of 128: 301
// tokens after 7001 81 us (a bf16 cache 103), 300 after 3000 50 (67), 2048 tokens 97 (95:
// its tiles are balanced better; here a CU is busy 52% of the time): 354 TFLOP/s of
// products once each.
//
// Numbers that are not finite.  A stored group is finite or NaN (all of it); one with a
// scale or a bias that is not finite, however it came there, is taken as NaN.  NaN times
// the weight 0 of a masked position would reach the rows before it, so NaN groups are
// expanded as zeros and noted per position: a key's (any group) makes the scores of the
// rows that see the position NaN, a value's makes the group's outputs of those rows NaN.
#pragma once

#include "attention_prefill_impl.h"
#include "kv4_impl.h"

#define KV4_PF_BITS 7.0f  // weights are 2^(s - m + this); with PF_SLACK at most 2^15
#define KV4_PF_WG 512
#define KV4_PF_ROWS 256

template <int NG>
struct Kv4PrefillTile {
  typedef short i16x4 __attribute__((ext_vector_type(4)));
  typedef float f32x16 __attribute__((ext_vector_type(16)));
  typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));

  static constexpr uint32_t CH = 64;            // positions per chunk
  // LDS bytes per position: 256 and as much more as keeps the rows that are read at a
  // time on different banks (K: one 16-byte piece of 8 rows; V: 64 bytes of 4)
  static constexpr uint32_t KROW = 256 + 16, VROW = 256 + 64;
  static constexpr uint32_t VBUF = 2 * CH * KROW, NOTES = VBUF + 2 * CH * VROW;
  static constexpr uint32_t LDS_BYTES = NOTES + 4 * CH * 4;  // notes: K, V x 2 chunks
  static constexpr uint32_t OROW = 68;          // floats: 64 dims of a row of q or out
  static_assert(8 * 32 * OROW * 4 <= NOTES, "in the chunks' space");
  static constexpr int QF = 2 * NG;             // q fragments of 16 dims

  uint32_t lane, h, wave, second;  // second: the wave's group
  uint32_t g;                // kv head
  uint32_t t0, t1;           // this split's positions, up to the tile's last
  uint32_t row, qpos;        // this lane's query row and its position
  uint32_t wmin, wmax;       // positions of the wave's first and last row
  uint32_t head;
  bool live;                 // the wave has rows
  __amdgpu_buffer_rsrc_t codes, scales;  // of what the wave's group expands
  f16x8 qh[QF], ql[QF];
  float scale2;              // log2(e) / sqrt(head) times the row's q scale back
  uint32_t cw[NG], cp[NG];   // the next chunk to expand: a piece's words, its row's scales

  AMMON_DEV size_t row_at(const ammon_k_attention &p) const {
    const uint32_t G = p.q_heads / p.kv_heads, r = min(row, p.tokens * G - 1), token = r / G;
    return (size_t)token * p.q_heads + g * G + (r - token * G);
  }

  // NG words at byte `off` of a buffer (zeros past its end).
  AMMON_DEV static void words(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t (&w)[NG]) {
    if constexpr (NG == 4) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
      w[0] = v[0], w[1] = v[1], w[2] = v[2], w[3] = v[3];
    } else if constexpr (NG == 3) {
      const u32x3 v = __builtin_amdgcn_raw_buffer_load_b96(r, off, 0, 0);
      w[0] = v[0], w[1] = v[1], w[2] = v[2];
    } else if constexpr (NG == 2) {
      const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
      w[0] = v[0], w[1] = v[1];
    } else {
      w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
    }
  }

  // A thread's part of its group's K or V of a chunk: piece p of row r; 8 lanes have a
  // piece of 8 rows (their LDS writes use different banks), a wave 16 whole rows.
  AMMON_DEV static uint32_t part_row() { return (threadIdx.x & 7) | (threadIdx.x >> 5 & 7) << 3; }
  AMMON_DEV static uint32_t part_piece() { return threadIdx.x >> 3 & 3; }

  AMMON_DEV void load(uint32_t c) {
    const uint32_t t = c * CH + part_row();
    words(codes, t * (16 * NG) + part_piece() * (4 * NG), cw);
    words(scales, t * (4 * NG), cp);
  }

  // Expand the loaded K or V of chunk c; its NaN groups become zeros and are noted (bit
  // j: group j).
  AMMON_DEV void expand(char *lds, uint32_t c, const Kv4Bits &bits) {
    uint32_t found = 0;
    f16x2 any = __builtin_bit_cast(f16x2, cp[0]);
#pragma unroll
    for (int j = 1; j < NG; ++j) any += __builtin_bit_cast(f16x2, cp[j]);
    // (a sum of scales or of biases that is not finite: one is not, or they are large)
    any *= (_Float16)0;
    if (__any(any[0] + any[1] != (_Float16)0)) {
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const bool bad = (cp[j] & 0x7c00u) == 0x7c00u || (cp[j] & 0x7c000000u) == 0x7c000000u;
        found |= bad ? 1u << j : 0u;
        cp[j] = bad ? 0u : cp[j];
      }
    }
    const uint32_t r = part_row(), pc = part_piece(), b = c & 1;
    char *to = lds + (second ? VBUF + (b * CH + r) * VROW : (b * CH + r) * KROW) + pc * 16;
#pragma unroll
    for (int j = 0; j < NG; ++j) *(f16x8 *)(to + 64 * j) = kv4_numbers(cw[j], cp[j], bits);
    if (pc == 0) ((uint32_t *)(lds + NOTES))[(second * 2 + b) * CH + r] = found;
  }

  // A operand of the value product: 16 positions 16 kk.. in the order 4 h + i, 8 + 4 h +
  // i; lane = dim of 32 db...
  AMMON_DEV f16x8 v_frag(const char *vb, int kk, int db) const {
    const uint32_t s = lane & 15;
    const char *at = vb + (4 * h + (s >> 2)) * VROW + (lane >> 4 & 1) * 32 + (s & 3) * 8 + db * 64;
    typedef __attribute__((address_space(3))) i16x4 *tr;
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(at + kk * 16 * VROW));
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(at + (kk * 16 + 8) * VROW));
    return __builtin_bit_cast(f16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  AMMON_DEV static f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
  }

  // The lane's row's pointer, as lane r has it.
  template <typename T> AMMON_DEV static T *pointer_of(T *mine, int r) {
    const uint32_t lo = (uint32_t)(uintptr_t)mine, hi = (uint32_t)((uintptr_t)mine >> 32);
    return (T *)(uintptr_t)((uint64_t)(uint32_t)__shfl((int)hi, r) << 32 | (uint32_t)__shfl((int)lo, r));
  }
  typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

  // q of the lane's row as fp16 hi + lo of q 2^(14 - e), |q| < 2^e.  Through LDS, four
  // rows of 64 dims at a time, as finish() writes: a lane that reads its own row takes 16
  // bytes of a line at a time.
  AMMON_DEV void load_q(const ammon_k_attention &p, char *lds, float minus1) {
    const float *q = p.q + row_at(p) * head;
    float *mine = (float *)lds + wave * 32 * OROW;
    f32x4u v[(NG + 1) / 2][8];
    const uint32_t col = 4 * (lane & 15);
    const float *from[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) from[i] = pointer_of(q, 4 * i + (lane >> 4));
    if (head % 4 == 0) {
#pragma unroll
      for (int half = 0; half < (NG + 1) / 2; ++half)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[half][i] = *(const f32x4u *)(from[i] + min(64 * half + col, head - 4));
    } else {
#pragma unroll
      for (int half = 0; half < (NG + 1) / 2; ++half)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) v[half][i][e] = from[i][min(64 * half + col + e, head - 1)];
    }
#pragma unroll
    for (int half = 0; half < (NG + 1) / 2; ++half)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
          if (64 * half + col + e >= head) v[half][i][e] = 0.f;
    float x[QF][8], qmax = 0.f;
#pragma unroll
    for (int half = 0; half < (NG + 1) / 2; ++half) {
#pragma unroll
      for (int i = 0; i < 8; ++i) *(f32x4u *)(mine + (4 * i + (lane >> 4)) * OROW + col) = v[half][i];
      wave_lds_order();
#pragma unroll
      for (int kk = 4 * half; kk < QF && kk < 4 * half + 4; ++kk) {
        const float4 *r = (const float4 *)(mine + (lane & 31) * OROW + 16 * (kk & 3) + 8 * h);
        const float4 a = r[0], b = r[1];
        x[kk][0] = a.x, x[kk][1] = a.y, x[kk][2] = a.z, x[kk][3] = a.w;
        x[kk][4] = b.x, x[kk][5] = b.y, x[kk][6] = b.z, x[kk][7] = b.w;
#pragma unroll
        for (int e = 0; e < 8; ++e) qmax = fmaxf(qmax, fabsf(x[kk][e]));
      }
      wave_lds_order();
    }
    qmax = pair32_max(qmax);
    const int e2 = __builtin_amdgcn_frexp_expf(qmax);
#pragma unroll
    for (int kk = 0; kk < QF; ++kk)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        f16x2 hi, lo;
        kv4_parts(ldexpf(x[kk][e], 14 - e2), ldexpf(x[kk][e + 1], 14 - e2), minus1, hi, lo);
        qh[kk][e] = hi[0], qh[kk][e + 1] = hi[1];
        ql[kk][e] = lo[0], ql[kk][e + 1] = lo[1];
      }
    // (not 0: a masked score is -inf times this)
    scale2 = fmaxf(ldexpf(1.4426950408889634f / sqrtf((float)head), e2 - 14), 0x1p-126f);
  }

  // V fragments kk of dims 32 db.. of chunk c's, into their place.
  AMMON_DEV void read_v(const char *lds, uint32_t c, int db, int kk, f16x8 (&a)[4]) const {
    a[kk] = v_frag(lds + VBUF + (c & 1) * CH * VROW, kk, db);
  }
  // K fragments of step kk (16 dims) of chunk c, positions 32 b..
  AMMON_DEV void read_k(const char *lds, uint32_t c, int kk, f16x8 (&k)[2]) const {
    const char *ka = lds + (c & 1) * CH * KROW + (lane & 31) * KROW + h * 16;
#pragma unroll
    for (int b = 0; b < 2; ++b) k[b] = *(const f16x8 *)(ka + kk * 32 + b * 32 * KROW);
  }

  // A turn on the matrix unit: O += V P of chunk c (whose first fragments are in a), then
  // the scores of chunk c + 1.  Every operand is read three to six products before it is
  // used, and a block's sums are added to the output while the next block is multiplied.
  // (The chunk's value products are summed by themselves, small parts first, and added to
  // the output once: short chains of fp32 additions.)
  AMMON_DEV void multiply(const char *lds, uint32_t c, const f16x8 (&ph)[4], const f16x8 (&pl)[4],
                          f16x8 (&a)[4], f32x16 (&o)[NG], f32x16 (&s)[2]) const {
    f16x8 k[2][2];
    f32x16 t[2];
#pragma unroll
    for (int kk = 1; kk < 4; ++kk) read_v(lds, c, 0, kk, a);
#pragma unroll
    for (int db = 0; db < NG; ++db) {
      t[db & 1] = zero16();
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        t[db & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[kk], pl[kk], t[db & 1], 0, 0, 0);
        t[db & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[kk], ph[kk], t[db & 1], 0, 0, 0);
        if (db + 1 < NG) read_v(lds, c, db + 1, kk, a);
        if (db > 0) {
#pragma unroll
          for (int i = 4 * kk; i < 4 * kk + 4; ++i) o[db - 1][i] += t[(db - 1) & 1][i];
        }
        if (db + 1 == NG && kk == 3) read_k(lds, c + 1, 0, k[0]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    s[0] = zero16();
    s[1] = zero16();
#pragma unroll
    for (int kk = 0; kk < QF; ++kk) {
      if (kk + 1 < QF) read_k(lds, c + 1, kk + 1, k[(kk + 1) % 2]);
      score_step(k[kk % 2], kk, s);
      if (kk == 0) o[NG - 1] += t[(NG - 1) & 1];
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // The scores of chunk 0.
  AMMON_DEV void first_scores(const char *lds, f32x16 (&s)[2]) const {
    s[0] = zero16();
    s[1] = zero16();
#pragma unroll
    for (int kk = 0; kk < QF; ++kk) {
      f16x8 k[2];
      read_k(lds, 0, kk, k);
      score_step(k, kk, s);
    }
  }
  AMMON_DEV void score_step(const f16x8 (&k)[2], int kk, f32x16 (&s)[2]) const {
#pragma unroll
    for (int b = 0; b < 2; ++b) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[b], ql[kk], s[b], 0, 0, 0);
#pragma unroll
    for (int b = 0; b < 2; ++b) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[b], qh[kk], s[b], 0, 0, 0);
  }

  // One workgroup's part: unit u = (split, tile, kv head), kv head fastest, so that with 8
  // kv heads each XCD keeps one head's K and V in its L2; then the tiles from the last
  // (with causal masking the longest) to the first; the splits slowest, the first (which
  // every tile sees most of) first.  Workgroups are handed out in order to the shader
  // engines in turn, and one that finds its engine full holds up the rest: with the
  // splits faster than the tiles, every second engine had all the long ones (2048 tokens,
  // two splits: 106 us).
  AMMON_DEV void run(const ammon_k_attention &p, char *lds) {
    const uint32_t tiles = (p.tokens * (p.q_heads / p.kv_heads) + KV4_PF_ROWS - 1) / KV4_PF_ROWS;
    const uint32_t unit = blockIdx.x / p.kv_heads;
    if (unit >= tiles * p.splits) return;  // (the grid is a multiple of 8)
    g = blockIdx.x % p.kv_heads;
    const uint32_t tile = tiles - 1 - unit % tiles, split = unit / tiles;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    second = wave >> 2;
    lane = threadIdx.x & 63;
    h = lane >> 5;
    head = p.head;
    const uint32_t start = min(p.step->position, p.limit);  // (no sum with it wraps around)
    const uint32_t G = p.q_heads / p.kv_heads, rows = p.tokens * G;
    const uint32_t w0 = tile * KV4_PF_ROWS + 32 * wave;  // the wave's first row
    live = w0 < rows;
    wmin = start + (live ? w0 : rows - 1) / G;
    wmax = start + min(w0 + 31, rows - 1) / G;
    row = w0 + (lane & 31);
    qpos = start + min(row, rows - 1) / G;
    const uint32_t last = start + min(tile * KV4_PF_ROWS + KV4_PF_ROWS - 1, rows - 1) / G;
    t0 = split * p.split_len;
    t1 = min(min(last + 1, t0 + p.split_len), p.limit);
    if (t0 >= t1) return;  // no position of this range is live for any row (uniform)
    const void *cache = second ? p.v_cache : p.k_cache;
    codes = make_rsrc(kv4_codes(cache, p.seq, NG, g, t0), (t1 - t0) * (16 * NG));
    scales = make_rsrc(kv4_scales(cache, p.kv_heads, p.seq, NG, g, t0), (t1 - t0) * (4 * NG));
    const uint32_t nch = (t1 - t0 + CH - 1) / CH;
    const Kv4Bits bits;
    const float minus1 = kv4_minus1();
    load(0);
    load_q(p, lds, minus1);
    __syncthreads();  // (q's LDS is the chunks')

    f32x16 o[NG];
#pragma unroll
    for (int db = 0; db < NG; ++db) o[db] = zero16();
    float m = -INFINITY, l = 0.f;  // l: this lane's positions only, summed at the end
    bool far = false;              // uniform: a row's m past KV4_FAR
    uint32_t nan = 0;              // value groups of which the row sees one
    const uint32_t lim = min(qpos, t1 - 1);  // last position of this lane's row
    f32x16 s[2];
    f16x8 ph[4], pl[4];  // the weights' parts, of 16 positions each
    f16x8 a[4];          // the next V fragments
    // chunks of which the wave's rows see a position
    const uint32_t mine = !live || t0 > wmax ? 0 : min(nch, (wmax - t0) / CH + 1);

    // turn -1: K 0, and V 0 (which nobody needs before turn 2)
    expand(lds, 0, bits);
    load(1);  // (past the end: zeros)
    __syncthreads();
    if (second) __syncthreads();
    if (mine) first_scores(lds, s);
    __syncthreads();
    for (uint32_t c = 0; c < nch; ++c) {
      // (past the last chunk: zeros, whose scores nothing reads)
      expand(lds, c + 1, bits);
      load(c + 2);
      __builtin_amdgcn_sched_barrier(0);
      if (c < mine) {
        softmax(lds, c, lim, minus1, s, ph, pl, o, m, l, far, nan);
#pragma unroll
        for (int kk = 0; kk < 1; ++kk) read_v(lds, c, 0, kk, a);
      }
      __syncthreads();
      if (c < mine) multiply(lds, c, ph, pl, a, o, s);
      __syncthreads();
    }
    if (!second) __syncthreads();
#pragma unroll
    for (int db = 0; db < NG; ++db)
      if (nan >> db & 1)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = __uint_as_float(0x7fc00000u);
    finish(p, split, lds, o, m - KV4_PF_BITS, l);
  }

  // Scores s of chunk c to the parts of its weights.
  AMMON_DEV void softmax(const char *lds, uint32_t c, uint32_t lim, float minus1, f32x16 (&s)[2],
                         f16x8 (&ph)[4], f16x8 (&pl)[4], f32x16 (&o)[NG], float &m, float &l,
                         bool &far, uint32_t &nan) const {
    const uint32_t first = t0 + c * CH;
    const uint32_t *notes = (const uint32_t *)(lds + NOTES) + (c & 1) * CH + lane;
    const uint32_t kn = notes[0], vn = notes[2 * CH];
    const bool masked = first + CH - 1 > min(wmin, t1 - 1);  // uniform
    if (masked) {
      const int rest = (int)(lim - first) - 4 * (int)h;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + 8 * (i >> 2) + (i & 3) > rest) s[b][i] = -INFINITY;
    }
    if (__any((kn | vn) != 0)) {  // uniform
      // the positions of this chunk that the row sees
      const uint64_t seen = lim < first ? 0 : lim - first >= 63 ? ~0ull : (2ull << (lim - first)) - 1;
      const uint64_t bad = (__ballot(kn != 0) & seen) >> (4 * h);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((uint32_t)(bad >> 32 * b) & 1u << (8 * (i >> 2) + (i & 3)))
            s[b][i] = __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int j = 0; j < NG; ++j)
        if (__ballot(vn >> j & 1) & seen) nan |= 1u << j;
    }
    float mc = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mc = fmaxf(mc, s[b][i]);
    mc = pair32_max(mc) * scale2;
    if (__any(mc - m > PF_SLACK)) {
      const float mn = fmaxf(m, mc);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
      for (int db = 0; db < NG; ++db) o[db] *= f;
      l *= f;
      m = mn;
      far = __any(fabsf(m == -INFINITY ? 0.f : m) > KV4_FAR);
    }
    // (a row with no position yet keeps (m, l, o) = (-inf, 0, 0))
    const float mz = m == -INFINITY ? 0.f : m;
    float mu = mz - KV4_PF_BITS, by = scale2;
    if (far) {  // (scores become distances)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = kv4_distance(s[b][i], scale2, mz);
      mu = -KV4_PF_BITS;
      by = 1.f;
    }
    float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], by, -mu));
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        ls[i & 3] += s[b][i];
        ls[(i & 3) + 1] += s[b][i + 1];
        f16x2 hi, lo;
        kv4_parts(s[b][i], s[b][i + 1], minus1, hi, lo);
        const int at = 2 * b + i / 8, e = i % 8;
        ph[at][e] = hi[0], ph[at][e + 1] = hi[1];
        pl[at][e] = lo[0], pl[at][e + 1] = lo[1];
      }
    l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
  }

  // The result or partial of each row (m: what the weights are relative to), through LDS
  // (the chunks are done with): a lane has one row, and stores of 8 bytes of 64 rows each
  // cost more than the products (2048 tokens, two splits: 112 us).
  AMMON_DEV void finish(const ammon_k_attention &p, uint32_t split, char *lds, const f32x16 (&o)[NG],
                        float m, float l) const {
    l = pair32_sum(l);
    // the only split with a position of this row: the result (of a position out of range
    // NaN); else a partial, unless the split is dead for the row (the merge skips it)
    const bool in = qpos < p.limit;
    const bool direct = p.splits == 1 || (p.single_out && split == 0 && qpos < p.split_len && in);
    const bool write = live && row < p.tokens * (p.q_heads / p.kv_heads) &&
                       (direct || (in && t0 <= qpos));
    float *to = direct ? p.out + row_at(p) * head
                       : p.partial + (row_at(p) * p.splits + split) * (head + 2);
    if (!write) to = nullptr;
    if (write && !direct && h == 0) {
      to[head] = m * 0.6931471805599453f;  // natural-log units
      to[head + 1] = l;
    }
    const float f = !direct ? 1.f : in ? 1.f / l : __uint_as_float(0x7fc00000u);
    float *mine = (float *)lds + wave * 32 * OROW;
    float *dst[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = pointer_of(to, 4 * i + (lane >> 4));
#pragma unroll
    for (int half = 0; half < (NG + 1) / 2; ++half) {
#pragma unroll
      for (int db = 2 * half; db < NG && db < 2 * half + 2; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *(float4 *)(mine + (lane & 31) * OROW + 32 * (db & 1) + 2 * i + 4 * h) =
              make_float4(o[db][i] * f, o[db][i + 1] * f, o[db][i + 2] * f, o[db][i + 3] * f);
      wave_lds_order();
      const uint32_t d = 64 * half + 4 * (lane & 15);
      f32x4u v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = *(const f32x4u *)(mine + (4 * i + (lane >> 4)) * OROW + 4 * (lane & 15));
      if (head % 4 == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (dst[i] && d < head) *(f32x4u *)(dst[i] + d) = v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e)
            if (dst[i] && d + e < head) dst[i][d + e] = v[i][e];
      }
      wave_lds_order();
    }
  }
};
