// kv4_attention_impl.h -- split-K decode attention over a KV4 cache (kv4_impl.h).
//
// Pass 1 of attention_impl.h's pair, any head up to 128 and up to 8 query heads per
// kv head: one workgroup per (split, kv head), on matrix cores; the partials have
// the other units' format, so pass 2 is theirs.  Chunks of 128 positions, 32 per
// wave; NCH chunks are requested ahead into a ring in LDS of which every wave reads
// back only its own rows, so the chunk loop has no barrier.
//
//   scores  S[t][h] = K[t] . q[h] on v_mfma_f32_16x16x32_f16, one per group of 32
//           numbers: A = K rows as kv4_numbers gives them, B = q as fp16 hi + lo: 22
//           bits (q is scaled by a power of two to at most 2^13..2^14 first, so that
//           lo is no subnormal where it matters).
//   weights P = 2^(s log2e / sqrt(head) - m), fp32; m is a running maximum less
//           KV4_BITS, so that the fp16 parts of small weights are no subnormals
//           either, and moves only when a chunk exceeds that maximum by KV4_SLACK.
//   values  O^T[d][h] += V^T[d][t] P[t][h], 32 positions per v_mfma_f32_16x16x32_f16,
//           P as fp16 hi + lo (22 bits): lane i (of 16) of A has word i of 8
//           positions, joined half by half in pairs, and nibble n of the words is
//           value tile n.  Row 4 a + r of a score tile is position 4 r + a, so that
//           the four rows of V that a wave reads at a time are neighbours.
//
// What bounds it: HBM where the context is long.  Per 32 positions a wave issues some
// 270 VALU instructions and 32 MFMA (head 128) for 5 KiB, which take a CU's share of
// 5.5 TB/s as long as 570 VALU instructions on each SIMD.
#pragma once

#include "attention_impl.h"
#include "kv4_impl.h"

#define KV4_BITS 10.0f
#define KV4_SLACK 4.0f
#define KV4_MAX_GROUP 8  // query heads per kv head

// What one wave stages of a chunk: 32 positions' codes, K's then V's, in 16-byte
// pieces, and their scales, K's then V's: whole requests of 64 lanes each.
template <int NG> struct Kv4Stage {
  static constexpr uint32_t CODES = 512 * NG, SCALES = 128 * NG;  // bytes of K (or V)
  static constexpr uint32_t WAVE = 2 * (CODES + SCALES);
  static constexpr uint32_t CHUNK = AMMON_WAVES * WAVE;
  static constexpr int SREQ = NG == 4 ? 1 : NG;  // a row's scales: 16 bytes, or NG words
  static constexpr int VREQ = NG / 2;            // requests of V's codes alone, the last ones
  static constexpr int REQ = NG + SREQ;
};

template <int NG, int NCH, bool APPEND>
struct Kv4Partial {
  using S = Kv4Stage<NG>;
  static constexpr uint32_t WROWS = 32, CROWS = AMMON_WAVES * WROWS;
  static constexpr uint32_t MERGE = AMMON_WAVES * KV4_MAX_GROUP * ATT_STAGED_OROW * 4;
  static constexpr uint32_t RING = S::CHUNK * NCH > MERGE ? S::CHUNK * NCH : MERGE;
  static constexpr uint32_t LDS_BYTES = RING + (2 * AMMON_WAVES + 2) * KV4_MAX_GROUP * 4;
  static_assert(NCH >= 1 && NCH <= 4, "chunk buffers");

  uint32_t split, g, G, pos, t0, n, lane, wave;
  const uint32_t *kc, *ks, *vc, *vs;  // codes and scales of the split's first row
  float qraw[NG][8];
  bool owner;      // APPEND: this wave has the new position
  float fresh[8];  // ... lanes 0..15: the new key, 16..31: the new value

  // The 16-byte piece of the wave's rows that LDS slot `at` of its codes holds.  At head
  // 128 a row's pieces are exchanged by its place, so that the 8 lanes of a score
  // operand's read phase (one piece of rows 0, 4, 8, 12, 1, ..) use different banks.
  AMMON_DEV static uint32_t piece(uint32_t at) { return NG == 4 ? at ^ (at >> 4 & 3) : at; }

  // Lane l's SIZE bytes at `from` into LDS at `to` + SIZE l.
#define KV4_REQUEST(FROM, TO, SIZE)                                                    \
  __builtin_amdgcn_global_load_lds(                                                    \
      (const __attribute__((address_space(1))) void *)(FROM),                          \
      (__attribute__((address_space(3))) void *)(TO), SIZE, 0, 0)

  // Request i of the codes of rows r0.. (of K and V together: 64 NG pieces).  Rows past
  // the split take its last row: they are masked, and what they hold is then no less
  // finite than what the split holds (but for a new row's place, see run).
  AMMON_DEV void codes(char *to, uint32_t r0, int i) const {
    const uint32_t at = i * 64 + lane;
    const bool v = at >= 32 * NG;
    const uint32_t pc = piece(v ? at - 32 * NG : at), r = pc / NG;
    const uint32_t *from = (v ? vc : kc) + (min(r0 + r, n - 1) * NG + (pc - r * NG)) * 4;
    KV4_REQUEST(from, to + i * 1024, 16);
  }
  // Chunk c of the split into ring buffer b.
  AMMON_DEV void stage(char *lds, uint32_t c, uint32_t b) const {
    char *to = lds + b * S::CHUNK + wave * S::WAVE;
    const uint32_t r0 = c * CROWS + wave * WROWS;
#pragma unroll
    for (int i = 0; i < NG - S::VREQ; ++i) codes(to, r0, i);
#pragma unroll
    for (int i = 0; i < S::SREQ; ++i) {
      constexpr uint32_t per = NG == 4 ? 1 : NG;  // requests' units per row
      const uint32_t at = i * 64 + lane;
      const bool v = at >= 32 * per;
      const uint32_t u = v ? at - 32 * per : at, r = u / per;
      const uint32_t *from = (v ? vs : ks) + min(r0 + r, n - 1) * NG + (u - r * per);
      if constexpr (NG == 4)
        KV4_REQUEST(from, to + 2 * S::CODES, 16);
      else
        KV4_REQUEST(from, to + 2 * S::CODES + i * 256, 4);
    }
#pragma unroll
    for (int i = NG - S::VREQ; i < NG; ++i) codes(to, r0, i);
  }

  // False for a dead split or a position out of range, which write nothing.
  AMMON_DEV bool begin(const ammon_k_attention &p, uint32_t split_, uint32_t g_, char *lds) {
    split = split_;
    g = g_;
    G = p.q_heads / p.kv_heads;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // q beside the position: neither needs the other.  (Columns past the group take
    // head 0's; they are never used.)
    const uint32_t h = lane & 15;
    const float *q = p.q + (size_t)(g * G + (h < G ? h : 0)) * p.head;
#pragma unroll
    for (int j = 0; j < NG; ++j) kv4_row(q, 4 * j + (lane >> 4), p.head, qraw[j]);
    pos = p.step->position + p.pos_add;
    if (pos >= p.limit) return false;
    t0 = split * p.split_len;
    if (t0 > pos) return false;
    n = min(p.split_len, pos + 1 - t0);
    kc = kv4_codes(p.k_cache, p.seq, NG, g, t0);
    vc = kv4_codes(p.v_cache, p.seq, NG, g, t0);
    ks = kv4_scales(p.k_cache, p.kv_heads, p.seq, NG, g, t0);
    vs = kv4_scales(p.v_cache, p.kv_heads, p.seq, NG, g, t0);
    // q has come with the position, or nearly: waiting for it here keeps the compiler's
    // wait for it, which would be for every request, out of the way of the requests
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(qraw[j][e]));
    owner = false;
    if constexpr (APPEND) {
      // the split's last position is the new one
      owner = pos < t0 + p.split_len && (n - 1) % CROWS / WROWS == wave;
      if (owner) {
        const float *x = (lane & 16 ? p.v_new : p.k_new) + (size_t)g * p.head;
        kv4_row(x, lane & 15, p.head, fresh);
      }
    }
#pragma unroll
    for (int b = 0; b < NCH; ++b) stage(lds, b, b);
    __builtin_amdgcn_sched_barrier(0);
    return true;
  }

  // Wait until at most EXTRA requests and k whole chunks of this wave are outstanding.
  template <int EXTRA> AMMON_DEV static void wait_chunks(uint32_t k) {
    if (NCH > 3 && k >= 3) wait_vmcnt<EXTRA + 3 * S::REQ>();
    else if (NCH > 2 && k == 2) wait_vmcnt<EXTRA + 2 * S::REQ>();
    else if (NCH > 1 && k == 1) wait_vmcnt<EXTRA + S::REQ>();
    else wait_vmcnt<EXTRA>();
  }

  AMMON_DEV void run(const ammon_k_attention &p, char *lds) {
    float *s_m = (float *)(lds + RING);                  // [4][8] wave maxima
    float *s_l = s_m + AMMON_WAVES * KV4_MAX_GROUP;      // [4][8] wave sums
    float *s_M = s_l + AMMON_WAVES * KV4_MAX_GROUP;      // [8] workgroup maxima
    float *s_L = s_M + KV4_MAX_GROUP;                    // [8] workgroup sums
    const uint32_t h = lane & 15, grp = lane >> 4, head = p.head;

    const Kv4Bits bits;
    const float minus1 = kv4_minus1();
    // q^T as the B operand, fp16 hi + lo of q 2^(14 - e), |q| < 2^e
    float qmax = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) qmax = fmaxf(qmax, fabsf(qraw[j][e]));
    qmax = pair32_max(pair16_max(qmax));
    const int qe = __builtin_amdgcn_frexp_expf(qmax);
    f16x8 qhi[NG], qlo[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        f16x2 hi, lo;
        kv4_parts(ldexpf(qraw[j][e], 14 - qe), ldexpf(qraw[j][e + 1], 14 - qe), minus1, hi, lo);
        qhi[j][e] = hi[0], qhi[j][e + 1] = hi[1];
        qlo[j][e] = lo[0], qlo[j][e + 1] = lo[1];
      }
    // log2(e) / sqrt(head), and q's scale back
    const float scale2 = ldexpf(1.4426950408889634f / sqrtf((float)head), qe - 14);

    uint32_t word = 0, sb = 0;
    if constexpr (APPEND) {
      if (owner) kv4_quantise(fresh, lane & 15, head, word, sb);
    }
    const uint32_t fg = (lane & 15) >> 2, fp = lane & 3;  // its group and piece

    f32x4 o[8];  // tile n: lane has word rows 4 grp + r of head h
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;  // m: the reference maximum; l: this lane's positions

    const uint32_t nch = (n + CROWS - 1) / CROWS;
    uint32_t b = 0;  // chunk c's ring buffer
    for (uint32_t c = 0; c < nch; ++c) {
      char *buf = lds + b * S::CHUNK + wave * S::WAVE;
      uint32_t *kw = (uint32_t *)buf, *vw = (uint32_t *)(buf + S::CODES);
      uint32_t *kp = (uint32_t *)(buf + 2 * S::CODES), *vp = kp + S::SCALES / 4;
      // chunks requested after this one: the first NCH - 1, and then as the buffers
      // came free, up to the last
      const uint32_t later = min(c + NCH, max(nch, (uint32_t)NCH)) - 1 - c;
      if constexpr (APPEND) {
        if (owner && c == nch - 1) {  // the new row, into this wave's copy
          wait_chunks<0>(later);
          const uint32_t r = (n - 1) % WROWS, w = fp * NG + fg;
          const uint32_t at = NG == 4 ? (r * 4 + (fp ^ (r >> 2 & 3))) * 4 + fg : r * (4 * NG) + w;
          if (lane < 32 && fg < NG) {
            (lane & 16 ? vw : kw)[at] = word;
            if (fp == 0) (lane & 16 ? vp : kp)[r * NG + fg] = sb;
          }
          wave_lds_order();
        }
      }
      wait_chunks<S::VREQ>(later);
      // scores: A row `h` is position 16 T + 4 (h % 4) + h / 4
      f32x4 sc[2];
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        const uint32_t r = 16 * T + 4 * (h & 3) + (h >> 2);
        uint32_t w[NG], ps[NG];
        if constexpr (NG == 4) {
          const u32x4 a = ((const u32x4 *)kw)[r * 4 + (grp ^ (h & 3))], b = ((const u32x4 *)kp)[r];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = a[j], ps[j] = b[j];
        } else {
#pragma unroll
          for (int j = 0; j < NG; ++j) w[j] = kw[r * (4 * NG) + grp * NG + j], ps[j] = kp[r * NG + j];
        }
        f32x4 hi = {0.f, 0.f, 0.f, 0.f}, lo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          const f16x8 a = kv4_numbers(w[j], ps[j], bits);
          hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qhi[j], hi, 0, 0, 0);
          lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qlo[j], lo, 0, 0, 0);
        }
        // lane: row 4 grp + r, position 16 T + 4 r + grp, of head h
        const uint32_t first = c * CROWS + wave * WROWS + 16 * T + grp;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sc[T][i] = first + 4 * i < n ? (hi[i] + lo[i]) * scale2 : -INFINITY;
      }
      float mc = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                       fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
      mc = pair32_max(pair16_max(mc));
      if (__any(mc > m + KV4_SLACK)) {
        const float mn = fmaxf(m, mc);
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] *= f;
        l *= f;
        m = mn;
      }
      // (a wave with no position yet has m = -inf, and weights 0)
      const float mu = (m == -INFINITY ? 0.f : m) - KV4_BITS;
      f16x8 ph, pl;
      float pw[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) pw[e] = __builtin_amdgcn_exp2f(sc[e / 4][e % 4] - mu);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        f16x2 hi, lo;
        kv4_parts(pw[e], pw[e + 1], minus1, hi, lo);
        ph[e] = hi[0], ph[e + 1] = hi[1];
        pl[e] = lo[0], pl[e + 1] = lo[1];
      }
      l += ((pw[0] + pw[1]) + (pw[2] + pw[3])) + ((pw[4] + pw[5]) + (pw[6] + pw[7]));
      // values: words of positions e = 4 T + r, row 16 T + 4 r + grp
      wait_chunks<0>(later);
      const uint32_t i = NG == 4 ? h : h % (4 * NG);  // (rows past the words are not used)
      uint32_t vraw[8], sraw[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t r4 = e & 3, r = 16 * (e >> 2) + 4 * r4 + grp;
        vraw[e] = NG == 4 ? vw[r * 16 + ((h >> 2) ^ r4) * 4 + (h & 3)] : vw[r * (4 * NG) + i];
        sraw[e] = vp[r * NG + i % NG];
      }
      if constexpr (APPEND) {
        // Rows past the split hold what the new row's place held before: nothing that a
        // weight of 0 is sure to cancel.  As numbers they become 0.
        const uint32_t first = c * CROWS + wave * WROWS;
        if (first + WROWS > n) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (first + 16 * (e >> 2) + 4 * (e & 3) + grp >= n) sraw[e] = 0;
        }
      }
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
      auto tile = [&](const uint32_t (&x)[4], auto nib) {
        f16x8 a;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f16x2 v = __builtin_elementwise_fma(kv4_pair<decltype(nib)::value>(x[u], bits), vs2[u], vb2[u]);
          a[2 * u] = v[0];
          a[2 * u + 1] = v[1];
        }
        return a;
      };
      auto values = [&](int at, const f16x8 &a) {
        o[at] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[at], 0, 0, 0);
        o[at] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[at], 0, 0, 0);
      };
      values(0, tile(wl, Nib<0>{}));
      values(1, tile(wl, Nib<1>{}));
      values(2, tile(wl, Nib<2>{}));
      values(3, tile(wl, Nib<3>{}));
      values(4, tile(wh, Nib<0>{}));
      values(5, tile(wh, Nib<1>{}));
      values(6, tile(wh, Nib<2>{}));
      values(7, tile(wh, Nib<3>{}));
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
    const float mr = m - KV4_BITS;  // the weights are relative to this
    if (lane < KV4_MAX_GROUP) {
      s_m[wave * KV4_MAX_GROUP + lane] = mr;
      s_l[wave * KV4_MAX_GROUP + lane] = l;
    }
    if constexpr (APPEND) {
      if (owner && lane < 32 && fg < NG) {
        const void *cache = lane & 16 ? p.v_cache : p.k_cache;
        kv4_codes(cache, p.seq, NG, g, pos)[fp * NG + fg] = word;
        if (fp == 0) kv4_scales(cache, p.kv_heads, p.seq, NG, g, pos)[fg] = sb;
      }
    }
    __syncthreads();
    // this wave's tiles to the workgroup's maximum, rows [w][h][d]
    if (h < G) {
      float M = s_m[h];
#pragma unroll
      for (int w = 1; w < AMMON_WAVES; ++w) M = fmaxf(M, s_m[w * KV4_MAX_GROUP + h]);
      // M is finite: a live split's first position is wave 0's
      const float f = __builtin_amdgcn_exp2f(mr - M);
      float *row = (float *)lds + (wave * KV4_MAX_GROUP + h) * ATT_STAGED_OROW;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t w = 4 * grp + r;  // word (w / NG, w % NG)
        if (NG == 4 || w < 4 * NG) {
          float4 *to = (float4 *)(row + 32 * (w % NG) + 8 * (w / NG));
          to[0] = make_float4(o[0][r] * f, o[4][r] * f, o[1][r] * f, o[5][r] * f);
          to[1] = make_float4(o[2][r] * f, o[6][r] * f, o[3][r] * f, o[7][r] * f);
        }
      }
      if (wave == 0 && grp == 0) {
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < AMMON_WAVES; ++w)
          L += s_l[w * KV4_MAX_GROUP + h] * __builtin_amdgcn_exp2f(s_m[w * KV4_MAX_GROUP + h] - M);
        s_M[h] = M;
        s_L[h] = L;
      }
    }
    __syncthreads();
    const uint32_t slot_w = head + 2;
    for (uint32_t idx = threadIdx.x; idx < G * head; idx += AMMON_WG) {
      const uint32_t j = idx / head, d = idx - j * head;
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < AMMON_WAVES; ++w)
        total += ((const float *)lds)[(w * KV4_MAX_GROUP + j) * ATT_STAGED_OROW + d];
      const float M = s_M[j], L = s_L[j];
      if (direct_out(p)) {
        st_out(p.out + (size_t)(g * G + j) * head + d, total / L);
        continue;
      }
      float *to = p.partial + ((size_t)(g * G + j) * p.splits + split) * slot_w;
      st_out(to + d, total);
      if (d == 0) {
        st_out(to + head, M * 0.6931471805599453f);  // natural-log units
        st_out(to + head + 1, L);
      }
    }
  }

 private:
  template <int N> struct Nib { static constexpr int value = N; };
};
