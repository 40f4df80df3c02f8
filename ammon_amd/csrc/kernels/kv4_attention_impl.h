// kv4_attention_impl.h -- split-K decode attention over a KV4 cache (kv4_impl.h).
//
// Pass 1 of attention_impl.h's pair, any head up to 128 and up to 8 query heads per
// kv head: one workgroup per (split, kv head, eight query rows), on matrix cores; the
// partials have the other units' format, so pass 2 is theirs.  The query rows of a kv
// head are its query heads, token by token: a decode step has one set of rows, a short
// prompt fills the sets with several tokens' heads.  Chunks of 256 positions, 64 per
// wave; NCH chunks are requested ahead into a ring in LDS of which every wave reads
// back only its own rows, so the chunk loop has no barrier.
//
//   scores  S[t][h] = K[t] . q[h] on v_mfma_f32_16x16x32_f16, one per group of 32
//           numbers and 16 positions: A = K rows as kv4_numbers gives them, B = q as
//           fp16, hi in columns 0..7 and lo in 8..15: 22 bits (q is scaled by a power
//           of two to at most 2^13..2^14 first, so that lo is no subnormal where it
//           matters).  The halves' sum is a rotation by 8 columns; columns 0..7 then
//           go on with the first 32 positions' scores, 8..15 with the others'.
//   weights P = 2^(s log2e / sqrt(head) - m), fp32; m is a running maximum less
//           KV4_BITS, so that the fp16 parts of small weights are no subnormals
//           either, and moves only when a chunk exceeds that maximum by KV4_SLACK.
//   values  O^T[d][h] += V^T[d][t] P[t][h], 32 positions per v_mfma_f32_16x16x32_f16,
//           P as fp16 hi + lo (22 bits): lane i (of 16) of A has word i of 8
//           positions, joined half by half in pairs, and nibble n of the words is
//           value tile n.  Row 4 a + r of a score tile is position 4 r + a, so that
//           the four rows of V that a wave reads at a time are neighbours.
//           Above head 64 a product takes 32 positions, hi in one half of the columns
//           and lo in the other.  Up to head 64 a row has at most 8 words, and a
//           product takes 64 positions: lanes 0..7 of A and columns 0..7 are the first
//           32, the others the second, and the two blocks in which they meet are not
//           used.
//
// Tokens of one set see different numbers of positions.  Scores past a token's own are
// masked; a value that is not finite there, which a weight of 0 would not cancel, is
// taken as 0 and noted, and the outputs that it does belong to become NaN at the end.
//
// What bounds it.  Long contexts: HBM (8 kv heads of 64, 131072 positions: 84 MB in 23.8
// us with the merge, some 9 us of which any two dependent launches take).  Short ones: a
// wave's chain through its one chunk, in cycles 1800 for q and the position, 2900 until
// the chunk is there, 1700 for scores and weights, 1650 for values, 1900 for the merge of
// the waves and the partial (2600 with a barrier between maxima and rows); 525 vector and
// 32 matrix instructions a chunk, and a wave has its SIMD for itself (8192 positions of 8
// heads of 128, replayed in a graph: 9.5 us with the merge).  The wave that appends is
// some 1200 cycles behind the others.
// Measured and not kept: hi and lo in products of their own and 32 positions per wave
// (twice the matrix instructions, up to head 64 twice the vector ones: 34.0 us and 12.0
// where the above are 23.8 and 10.0 with the merge); units of eight waves (the same up to
// 32768 positions, 54 us against 41 at 131072 of head 128, where one fits on a CU in
// place of two).  A third chunk in the ring would leave room for two units per CU up to
// head 64, not four.
#pragma once

#include "attention_impl.h"
#include "kv4_impl.h"

#define KV4_BITS 10.0f
#define KV4_SLACK 4.0f
#define KV4_MAX_GROUP 8  // query heads per kv head
#define KV4_DPP_ROR8 0x128  // rows of 16 lanes by 8

// What one wave stages of a chunk: 64 positions' codes of K, their scales, then V's
// alike: whole requests of 64 lanes each, 16 bytes a lane for codes.
template <int NG> struct Kv4Stage {
  static constexpr uint32_t ROWS = 64;
  static constexpr uint32_t CODES = 16 * NG * ROWS, SCALES = 4 * NG * ROWS;  // bytes of K (or V)
  static constexpr uint32_t HALF = CODES + SCALES, WAVE = 2 * HALF;
  static constexpr uint32_t CHUNK = AMMON_WAVES * WAVE;
  static constexpr int SREQ = NG == 4 ? 1 : NG;  // a row's scales: 16 bytes, or NG words
  static constexpr int VREQ = NG + SREQ;         // V's requests, the last ones
  static constexpr int REQ = 2 * VREQ;
};

// A decode step, a decode step that appends its rows, several tokens of a prompt.
enum Kv4Mode { KV4_DECODE, KV4_APPEND, KV4_TOKENS };

template <int NG, Kv4Mode MODE>
struct Kv4Partial {
  using S = Kv4Stage<NG>;
  static constexpr int NCH = 2;
  static constexpr bool APPEND = MODE == KV4_APPEND, TOKENS = MODE == KV4_TOKENS;
  static constexpr uint32_t WROWS = S::ROWS, CROWS = AMMON_WAVES * WROWS;
  static constexpr bool PAIRED = NG <= 2;              // 64 positions a value product
  static constexpr uint32_t OROW = 32 * NG + 4;        // merge row: banks spread
  static constexpr uint32_t LDS_BYTES = S::CHUNK * NCH;
  // For the merge a wave leaves its output rows [half of the columns][8] in its part of
  // the first ring buffer, its maxima and sums in its part of the second.
  static_assert(NCH == 2 && 2 * KV4_MAX_GROUP * OROW * 4 <= S::WAVE, "merge rows");

  uint32_t split, g, G, lane, wave;
  uint32_t pos, t0, n;        // the first token's position; the split's first, and how many
                              // of them the last token sees
  uint32_t mine, fewest;      // ... this lane's column's token, the first token
  uint32_t row0, cols, rows;  // the set's first row, its rows, and all the rows
  const uint32_t *kc, *ks, *vc, *vs;  // codes and scales of the split's first row
  float qraw[NG][8];
  bool owner;         // APPEND: this wave has the new position
  float fresh[1][8];  // ... lanes 0..15: the new key, 16..31: the new value

  // The 16-byte piece of the wave's rows that LDS slot `at` of its codes holds.  At head
  // 128 a row's pieces are exchanged by its place, so that the 8 lanes of a score
  // operand's read phase (one piece of rows 0, 4, 8, 12, 1, ..) use different banks.
  AMMON_DEV static uint32_t piece(uint32_t at) { return NG == 4 ? at ^ (at >> 4 & 3) : at; }

  // Lane l's SIZE bytes at `from` into LDS at `to` + SIZE l.
#define KV4_REQUEST(FROM, TO, SIZE)                                                    \
  __builtin_amdgcn_global_load_lds(                                                    \
      (const __attribute__((address_space(1))) void *)(FROM),                          \
      (__attribute__((address_space(3))) void *)(TO), SIZE, 0, 0)

  // Rows r0.. of one cache.  Rows past the split take its last row: they are masked, and
  // what they hold is then no less finite than what the split holds (but for a new row's
  // place, see run).  A wave's rows are one piece of memory, so whole ones need no
  // lane's own row.
  AMMON_DEV void stage_half(char *to, const uint32_t *codes, const uint32_t *scales,
                            uint32_t r0) const {
    constexpr uint32_t per = NG == 4 ? 1 : NG;  // scale requests' units per row
    if (r0 + WROWS <= n) {
      const char *c = (const char *)(codes + (size_t)r0 * (4 * NG));
      const char *s = (const char *)(scales + (size_t)r0 * NG);
      const uint32_t at = piece(lane) * 16;  // (the exchange is the same in every request)
#pragma unroll
      for (int i = 0; i < NG; ++i) KV4_REQUEST(c + i * 1024 + (size_t)at, to + i * 1024, 16);
#pragma unroll
      for (int i = 0; i < S::SREQ; ++i) {
        if constexpr (NG == 4)
          KV4_REQUEST(s + (size_t)(lane * 16), to + S::CODES, 16);
        else
          KV4_REQUEST(s + i * 256 + (size_t)(lane * 4), to + S::CODES + i * 256, 4);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const uint32_t pc = piece(i * 64 + lane), r = pc / NG;
        const uint32_t *from = codes + (min(r0 + r, n - 1) * NG + (pc - r * NG)) * 4;
        KV4_REQUEST(from, to + i * 1024, 16);
      }
#pragma unroll
      for (int i = 0; i < S::SREQ; ++i) {
        const uint32_t u = i * 64 + lane, r = u / per;
        const uint32_t *from = scales + min(r0 + r, n - 1) * NG + (u - r * per);
        if constexpr (NG == 4)
          KV4_REQUEST(from, to + S::CODES, 16);
        else
          KV4_REQUEST(from, to + S::CODES + i * 256, 4);
      }
    }
  }
  // Chunk c of the split into ring buffer b.
  AMMON_DEV void stage(char *lds, uint32_t c, uint32_t b) const {
    char *to = lds + b * S::CHUNK + wave * S::WAVE;
    const uint32_t r0 = c * CROWS + wave * WROWS;
    stage_half(to, kc, ks, r0);
    stage_half(to + S::HALF, vc, vs, r0);
  }

  // False for a dead split or a position out of range, which write nothing.
  // Token `t` in range, and the split's first position seen by it.
  AMMON_DEV bool alive(const ammon_k_attention &p, uint32_t t) const {
    return pos + t < p.limit && t0 <= pos + t;
  }
  AMMON_DEV bool begin(const ammon_k_attention &p, uint32_t split_, uint32_t g_, uint32_t set,
                       char *lds) {
    split = split_;
    g = g_;
    G = p.group;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    rows = TOKENS ? p.tokens * G : G;
    row0 = TOKENS ? set * KV4_MAX_GROUP : 0;
    cols = min(rows - row0, (uint32_t)KV4_MAX_GROUP);
    // q and the new rows beside the position: none needs another.  (Columns past the rows take the
    // last one's; they are never used.)
    const uint32_t row = row0 + min(lane & 7, cols - 1);
    const uint32_t tok = TOKENS ? row / G : 0, first = TOKENS ? row0 / G : 0;
    const uint32_t last = TOKENS ? (row0 + cols - 1) / G : 0;
    const float *q = p.q + ((size_t)tok * p.q_heads + g * G + (row - tok * G)) * p.head;
    kv4_rows(q, lane >> 4, p.head, qraw);
    if constexpr (APPEND)
      kv4_rows((lane & 16 ? p.v_new : p.k_new) + (size_t)g * p.head, lane & 15, p.head, fresh);
    pos = min(p.step->position, p.limit);  // (no sum with it wraps around)
    t0 = split * p.split_len;
    if (pos + first >= p.limit) return false;
    const uint32_t end = min(pos + last, p.limit - 1);
    if (t0 > end) return false;
    n = min(p.split_len, end + 1 - t0);
    mine = !TOKENS ? n : alive(p, tok) ? min(p.split_len, pos + tok + 1 - t0) : 0;
    fewest = !TOKENS ? n : alive(p, first) ? min(p.split_len, pos + first + 1 - t0) : 0;
    kc = kv4_codes(p.k_cache, p.seq, NG, g, t0);
    vc = kv4_codes(p.v_cache, p.seq, NG, g, t0);
    ks = kv4_scales(p.k_cache, p.kv_heads, p.seq, NG, g, t0);
    vs = kv4_scales(p.v_cache, p.kv_heads, p.seq, NG, g, t0);
    // they have come with the position, or nearly: waiting for them here keeps the
    // compiler's wait, which would be for every request, out of the way of the requests
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int j = 0; j < NG; ++j) asm volatile("" : "+v"(qraw[j][e]));
      if constexpr (APPEND) asm volatile("" : "+v"(fresh[0][e]));
    }
    // the split's last position is the new one
    owner = APPEND && pos < t0 + p.split_len && (n - 1) % CROWS / WROWS == wave;
    stage(lds, 0, 0);
    if (n > CROWS) stage(lds, 1, 1);
    __builtin_amdgcn_sched_barrier(0);
    return true;
  }

  // Wait until at most EXTRA requests and k whole chunks (0 or 1) of this wave are
  // outstanding.
  template <int EXTRA> AMMON_DEV static void wait_chunks(uint32_t k) {
    if (k == 1) wait_vmcnt<EXTRA + S::REQ>();
    else wait_vmcnt<EXTRA>();
  }

  AMMON_DEV static float other_half(float v) { return dpp_get<KV4_DPP_ROR8>(v); }
  // fp16 numbers of v, but in the columns of BANKS (0x3: 0..7, 0xc: 8..15) the other
  // half's of w.
  template <int BANKS> AMMON_DEV static f16x8 halves(const f16x8 &v, const f16x8 &w) {
    const u32x4 a = __builtin_bit_cast(u32x4, v), b = __builtin_bit_cast(u32x4, w);
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r[e] = __builtin_amdgcn_update_dpp(a[e], b[e], KV4_DPP_ROR8, 0xf, BANKS, false);
    return __builtin_bit_cast(f16x8, r);
  }

  AMMON_DEV void run(const ammon_k_attention &p, char *lds) {
    const uint32_t h = lane & 15, grp = lane >> 4, head = p.head;
    const bool second = h >= 8;  // this lane's columns: the second half

    const Kv4Bits bits;
    const float minus1 = kv4_minus1();
    // q^T as the B operand, fp16 hi or lo of q 2^(14 - e), |q| < 2^e
    kv4_row_ends(grp, head, qraw);
    float qmax = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) qmax = fmaxf(qmax, fabsf(qraw[j][e]));
    qmax = pair32_max(pair16_max(qmax));
    const int qe = __builtin_amdgcn_frexp_expf(qmax);
    f16x8 qb[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        f16x2 hi, lo;
        kv4_parts(ldexpf(qraw[j][e], 14 - qe), ldexpf(qraw[j][e + 1], 14 - qe), minus1, hi, lo);
        qb[j][e] = second ? lo[0] : hi[0];
        qb[j][e + 1] = second ? lo[1] : hi[1];
      }
    // log2(e) / sqrt(head), and q's scale back (not 0: a masked score is -inf times this)
    const float scale2 = fmaxf(ldexpf(1.4426950408889634f / sqrtf((float)head), qe - 14), 0x1p-126f);

    uint32_t word = 0, sb = 0;
    if constexpr (APPEND) {
      if (owner) {
        kv4_row_ends(lane & 15, head, fresh);
        kv4_quantise(fresh[0], lane & 15, head, word, sb);
      }
    }
    const uint32_t fg = (lane & 15) >> 2, fp = lane & 3;  // its group and piece

    // This lane's places in the wave's part of a buffer, in bytes: of score tile T the
    // row 16 T + 4 (h % 4) + h / 4; of the values rows 4 r4 + grp and 16 more (and 32
    // more for the second half's lanes where the products are of 64 positions).
    const uint32_t krow = 4 * (h & 3) + (h >> 2);
    const uint32_t kword = krow * (16 * NG) + (NG == 4 ? grp ^ (h & 3) : grp) * (4 * NG);
    const uint32_t vrow = grp + (PAIRED && second ? 32 : 0);
    const uint32_t i = NG >= 3 ? h % (4 * NG) : h % (4 * NG) % 8;  // (more than the words: not used)
    const uint32_t vscale = S::HALF + S::CODES + (vrow * NG + i % NG) * 4;
    uint32_t vword[NG == 4 ? 4 : 1];  // ... for each r4 at head 128, whose pieces are exchanged
    if constexpr (NG == 4) {
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        vword[r4] = S::HALF + vrow * 64 + ((h >> 2) ^ r4) * 16 + (h & 3) * 4;
    } else {
      vword[0] = S::HALF + (vrow * (4 * NG) + i) * 4;
    }

    f32x4 o[8];  // tile n: lane has word rows 4 grp + r of its column
#pragma unroll
    for (int x = 0; x < 8; ++x) o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;  // m: the reference maximum; l: this lane's positions
    bool far = false;              // uniform: an m past KV4_FAR
    uint32_t bad = ~0u;            // first noted position of this lane's group of 32 numbers

    const uint32_t nch = (n + CROWS - 1) / CROWS;
    uint32_t b = 0;  // chunk c's ring buffer
    for (uint32_t c = 0; c < nch; ++c) {
      char *buf = lds + b * S::CHUNK + wave * S::WAVE;
      const uint32_t first = c * CROWS + wave * WROWS;  // the wave's first row
      if (first >= n) break;  // (uniform; this is the last chunk)
      const uint32_t later = min(c + NCH, nch) - 1 - c;  // chunks requested after this one
      if constexpr (APPEND) {
        if (owner && c == nch - 1) {  // the new row, into this wave's copy
          wait_chunks<0>(later);
          const uint32_t r = (n - 1) % WROWS, w = fp * NG + fg;
          const uint32_t at = NG == 4 ? (r * 4 + (fp ^ (r >> 2 & 3))) * 4 + fg : r * (4 * NG) + w;
          uint32_t *to = (uint32_t *)(buf + (lane & 16 ? S::HALF : 0));
          if (lane < 32 && fg < NG) {
            to[at] = word;
            if (fp == 0) to[S::CODES / 4 + r * NG + fg] = sb;
          }
          wave_lds_order();
        }
      }
      wait_chunks<S::VREQ>(later);
      // scores: of 16 positions each; sc[r] is position 16 (r / 4) + 4 (r % 4) + grp of
      // this lane's half, raw
      float sc[8];
      {
        f32x4 t[4];
#pragma unroll
        for (int T = 0; T < 4; ++T) {
          const char *kw = buf + kword + T * (256 * NG);
          const char *kp = buf + S::CODES + krow * (4 * NG) + T * (64 * NG);
          uint32_t w[NG], ps[NG];
          if constexpr (NG == 4) {
            const u32x4 a = *(const u32x4 *)kw, b4 = *(const u32x4 *)kp;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = a[j], ps[j] = b4[j];
          } else {
#pragma unroll
            for (int j = 0; j < NG; ++j)
              w[j] = ((const uint32_t *)kw)[j], ps[j] = ((const uint32_t *)kp)[j];
          }
          t[T] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < NG; ++j)
            t[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv4_numbers(w[j], ps[j], bits), qb[j], t[T], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float x = t[r >> 2][r & 3], y = t[2 + (r >> 2)][r & 3];
          sc[r] = (second ? y : x) + other_half(second ? x : y);
        }
      }
      if (first + WROWS > fewest) {
        const uint32_t at = first + (second ? 32 : 0) + grp;
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (at + 16 * (r >> 2) + 4 * (r & 3) >= mine) sc[r] = -INFINITY;
      }
      float mc = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])),
                       fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
      mc = fmaxf(mc, other_half(mc));
      mc = pair32_max(pair16_max(mc)) * scale2;
      if (__any(mc - m > KV4_SLACK)) {
        const float mn = fmaxf(m, mc);
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
        for (int x = 0; x < 8; ++x) o[x] *= f;
        l *= f;
        m = mn;
        far = __any(fabsf(m == -INFINITY ? 0.f : m) > KV4_FAR);
      }
      // (a wave with no position yet has m = -inf, and weights 0)
      const float mz = m == -INFINITY ? 0.f : m;
      float mu = KV4_BITS - mz, by = scale2;
      if (far) {  // (scores become distances)
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[e] = kv4_distance(sc[e], scale2, mz);
        mu = KV4_BITS;
        by = 1.f;
      }
      f16x8 ph, pl;
      float pw[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) pw[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], by, mu));
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        f16x2 hi, lo;
        kv4_parts(pw[e], pw[e + 1], minus1, hi, lo);
        ph[e] = hi[0], ph[e + 1] = hi[1];
        pl[e] = lo[0], pl[e + 1] = lo[1];
      }
      l += ((pw[0] + pw[1]) + (pw[2] + pw[3])) + ((pw[4] + pw[5]) + (pw[6] + pw[7]));
      // values: word i of positions e = 4 T + r, row 16 T + 4 r + grp
      wait_chunks<0>(later);
#pragma unroll
      for (int half = 0; half < (PAIRED ? 1 : 2); ++half) {
        uint32_t vraw[8], sraw[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t r = 32 * half + 16 * (e >> 2) + 4 * (e & 3);
          vraw[e] = *(const uint32_t *)(buf + vword[NG == 4 ? e & 3 : 0] + r * (16 * NG));
          sraw[e] = *(const uint32_t *)(buf + vscale + r * (4 * NG));
        }
        if constexpr (APPEND) {
          // Rows past the split hold what the new row's place held before: nothing that a
          // weight of 0 is sure to cancel.  As numbers they become 0.
          if (first + WROWS > n) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (first + vrow + 32 * half + 16 * (e >> 2) + 4 * (e & 3) >= n) sraw[e] = 0;
          }
        }
        if (TOKENS && fewest < n && first + WROWS > fewest) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t at = first + vrow + 32 * half + 16 * (e >> 2) + 4 * (e & 3), x = sraw[e];
            if (at >= fewest && ((x & 0x7c00u) == 0x7c00u || (x >> 16 & 0x7c00u) == 0x7c00u)) {
              bad = min(bad, min(at, n - 1));  // (rows past the split are copies of its last)
              sraw[e] = 0;
            }
          }
        }
        // hi in the columns whose positions these are, lo in the others
        f16x8 pb = ph;
        if constexpr (!PAIRED) pb = half ? halves<0x3>(ph, pl) : halves<0xc>(ph, pl);
        uint32_t wl[4], wh[4];
        f16x2 vs2[4], vb2[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t w0 = vraw[2 * u], w1 = vraw[2 * u + 1], s0 = sraw[2 * u], s1 = sraw[2 * u + 1];
          wl[u] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
          wh[u] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
          vs2[u] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(s1, s0, 0x05040100u));
          vb2[u] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(s1, s0, 0x07060302u));
        }
        auto values = [&](int at, const uint32_t (&x)[4], auto nib) {
          f16x8 a;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const f16x2 v = __builtin_elementwise_fma(kv4_pair<decltype(nib)::value>(x[u], bits), vs2[u], vb2[u]);
            a[2 * u] = v[0];
            a[2 * u + 1] = v[1];
          }
          if constexpr (PAIRED) o[at] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[at], 0, 0, 0);
          o[at] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pb, o[at], 0, 0, 0);
        };
        values(0, wl, Nib<0>{});
        values(1, wl, Nib<1>{});
        values(2, wl, Nib<2>{});
        values(3, wl, Nib<3>{});
        values(4, wh, Nib<0>{});
        values(5, wh, Nib<1>{});
        values(6, wh, Nib<2>{});
        values(7, wh, Nib<3>{});
      }
      // refill the buffer once this wave's reads of it have returned
      if (c + NCH < nch) {
        wave_lds_order();
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        stage(lds, c + NCH, b);
      }
      b = b + 1 == NCH ? 0 : b + 1;
    }

    // every request has landed before the ring is reused
    wait_vmcnt<0>();
    l = pair32_sum(pair16_sum(l));
    l += other_half(l);
    const float mr = m - KV4_BITS;  // the weights are relative to this
    auto rows_of = [&](uint32_t w) { return (float *)(lds + w * S::WAVE); };
    auto stats = [&](uint32_t w) { return (float *)(lds + S::CHUNK + w * S::WAVE); };  // maxima, sums
    if (lane < KV4_MAX_GROUP) {
      stats(wave)[lane] = mr;
      stats(wave)[KV4_MAX_GROUP + lane] = l;
    }
    if constexpr (TOKENS) {
      // the first position noted of each group of numbers, as a rule none
      if (fewest < n) {
        uint32_t *noted = (uint32_t *)stats(wave) + 4 * KV4_MAX_GROUP;
        if (lane < NG) noted[lane] = ~0u;
        if (__any(bad != ~0u)) {
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            uint32_t x = i % NG == j ? bad : ~0u;
            for (int s = 1; s < 64; s *= 2) x = min(x, (uint32_t)__shfl_xor((int)x, s));
            if (lane == 0) noted[j] = x;
          }
        }
      }
    }
    const bool block = !PAIRED || (grp >= 2) == second;  // its positions' words
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t w = PAIRED ? 4 * (grp & 1) + r : 4 * grp + r;  // word (w / NG, w % NG)
      if (block && (NG == 4 || w < 4 * NG)) {
        float4 *to = (float4 *)(rows_of(wave) + h * OROW + 32 * (w % NG) + 8 * (w / NG));
        to[0] = make_float4(o[0][r], o[4][r], o[1][r], o[5][r]);
        to[1] = make_float4(o[2][r], o[6][r], o[3][r], o[7][r]);
      }
    }
    __syncthreads();
    if constexpr (APPEND) {
      if (owner && lane < 32 && fg < NG) {
        const void *cache = lane & 16 ? p.v_cache : p.k_cache;
        kv4_codes(cache, p.seq, NG, g, pos)[fp * NG + fg] = word;
        if (fp == 0) kv4_scales(cache, p.kv_heads, p.seq, NG, g, pos)[fg] = sb;
      }
    }
    // a query row to a wave, two dimensions to a lane
    const uint32_t d = 2 * lane;
    for (uint32_t j = wave; j < cols; j += AMMON_WAVES) {
      uint32_t tok = 0, hh = j;
      if constexpr (TOKENS) {
        tok = (row0 + j) / G;
        hh = row0 + j - tok * G;
        if (!alive(p, tok)) {  // a merge writes the NaN of a position out of range
          if (direct_out(p)) write_nan(p, tok, hh);
          continue;
        }
      }
      // the waves' rows to their largest maximum, which is finite: the token sees the first
      // position, wave 0's
      float M = stats(0)[j];
#pragma unroll
      for (int w = 1; w < AMMON_WAVES; ++w) M = fmaxf(M, stats(w)[j]);
      float a = 0.f, b = 0.f, L = 0.f;
#pragma unroll
      for (int w = 0; w < AMMON_WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(stats(w)[j] - M);
        L += stats(w)[KV4_MAX_GROUP + j] * f;
        const float *row = rows_of(w) + j * OROW + (d < head ? d : 0);
        const float2 x = *(const float2 *)row, y = *(const float2 *)(row + KV4_MAX_GROUP * OROW);
        a += (x.x + y.x) * f;
        b += (x.y + y.y) * f;
      }
      if (TOKENS && fewest < n) {
        uint32_t x = ~0u;
        for (uint32_t w = 0; w < AMMON_WAVES; ++w)
          x = min(x, ((const uint32_t *)stats(w))[4 * KV4_MAX_GROUP + min(d / 32, NG - 1u)]);
        if (x <= pos + tok - t0) a = b = __uint_as_float(0x7fc00000u);
      }
      const size_t row = (size_t)tok * p.q_heads + g * G + hh;
      const bool direct = direct_out(p);
      float *to = direct ? p.out + row * head : p.partial + (row * p.splits + split) * (head + 2);
      if (d < head) st_out(to + d, direct ? a / L : a);
      if (d + 1 < head) st_out(to + d + 1, direct ? b / L : b);
      if (!direct && lane == 0) {
        st_out(to + head, M * 0.6931471805599453f);  // natural-log units
        st_out(to + head + 1, L);
      }
    }
  }

  AMMON_DEV void write_nan(const ammon_k_attention &p, uint32_t tok, uint32_t hh) const {
    float *to = p.out + ((size_t)tok * p.q_heads + g * G + hh) * p.head;
    for (uint32_t d = lane; d < p.head; d += 64) st_out(to + d, __uint_as_float(0x7fc00000u));
  }
  // A set that did not begin: with one split, all its tokens are out of range.
  AMMON_DEV void out_of_range(const ammon_k_attention &p) const {
    if (!direct_out(p)) return;
    for (uint32_t j = wave; j < cols; j += AMMON_WAVES) {
      const uint32_t tok = (row0 + j) / G;
      write_nan(p, tok, row0 + j - tok * G);
    }
  }

 private:
  template <int N> struct Nib { static constexpr int value = N; };
};
