// kv4.hip -- kernels of the 4-bit KV cache: rows stored and read back, split-K decode
// attention (units of kv4_attention_impl.h) and prefill attention (tiles of
// kv4_prefill_impl.h); the merges are attention.hip's.
#include "kv4_attention_impl.h"
#include "kv4_prefill_impl.h"

// Rows [tokens, kv_heads, head] (fp32) into the cache at position step->position + t:
// 16 lanes a row, 16 rows a workgroup, blockIdx.y 0 the keys, 1 the values.  One row in
// flight per 16 lanes bounds it: 2048 rows of 8 heads of 128 (19 MB, 4 head bytes read and
// 20 NG written per row) take 7.6 us traced, the load of as many bytes 5.1.
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_kv4_store(ammon_k_kv4 p) {
  const uint32_t r = blockIdx.x * (AMMON_WG / 16) + threadIdx.x / 16, i = threadIdx.x & 15;
  if (r >= p.tokens * p.kv_heads) return;  // (a row's 16 lanes go together)
  const uint32_t t = r / p.kv_heads, g = r - t * p.kv_heads;
  const uint64_t pos = (uint64_t)p.step->position + t;
  if (pos >= p.seq) return;  // out of range: the cache stays as it is
  const float *src = blockIdx.y ? p.v : p.k;
  void *cache = blockIdx.y ? p.v_cache : p.k_cache;
  float x[1][8];
  kv4_rows(src + (size_t)r * p.head, i, p.head, x);
  kv4_row_ends(i, p.head, x);
  kv4_put(cache, p.kv_heads, p.seq, p.head, g, (uint32_t)pos, i, x[0]);
}

// rope_store (rope.hip) into a KV4 cache: q rotated in place, a lane per pair, by the
// first ceil(q_numel / 2 / 256) workgroups; the rest rotate and store the rows of k
// [kv_heads, head], 16 lanes each.  The rotation's products round before the sum, as
// there.
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_kv4_rope_store(ammon_k_kv4 p) {
#pragma clang fp contract(off)
  const uint32_t pos = p.step->position;
  if (pos >= p.seq) return;
  const float *cs = p.table + (size_t)pos * p.head;
  const uint32_t qblocks = (p.q_numel / 2 + AMMON_WG - 1) / AMMON_WG;
  if (blockIdx.x < qblocks) {
    const uint32_t i = 2 * (blockIdx.x * AMMON_WG + threadIdx.x);
    if (i >= p.q_numel) return;
    const float fcr = cs[i % p.head], fci = cs[i % p.head + 1];
    const float q0 = p.q[i], q1 = p.q[i + 1];
    p.q[i] = q0 * fcr - q1 * fci;
    p.q[i + 1] = q0 * fci + q1 * fcr;
    return;
  }
  const uint32_t g = (blockIdx.x - qblocks) * (AMMON_WG / 16) + threadIdx.x / 16;
  if (g >= p.kv_heads) return;
  const uint32_t i = threadIdx.x & 15;
  float row[1][8];
  kv4_rows(p.k + (size_t)g * p.head, i, p.head, row);
  kv4_row_ends(i, p.head, row);
  float (&x)[8] = row[0];
#pragma unroll
  for (uint32_t e = 0; e < 8; e += 2) {
    const uint32_t d = 8 * i + e;
    const float fcr = d < p.head ? cs[d] : 0.f, fci = d < p.head ? cs[d + 1] : 0.f;
    const float a = x[e] * fcr - x[e + 1] * fci, b = x[e] * fci + x[e + 1] * fcr;
    x[e] = a;
    x[e + 1] = b;
  }
  kv4_put(p.k_cache, p.kv_heads, p.seq, p.head, g, pos, i, x);
}

// Positions first.. of the cache as numbers [kv_heads, tokens, head], fp32 or bf16: 16
// lanes a row, 8 numbers each, AMMON_KV4_LOAD_ROWS rows a lane, all requested before the
// first is written.  Bytes bound it: 32768 positions of 8 heads of 128, keys and values,
// to bf16 (176 MB) take 32.3 us, 5.4 TB/s, where one row a lane took 42.2 us and two
// 36.8; with stores that are not nontemporal four took 34.1.
extern "C" __global__ __launch_bounds__(AMMON_WG) void ammon_kv4_load(ammon_k_kv4 p) {
  const uint32_t i = threadIdx.x & 15, j = i >> 2, piece = i & 3, ng = kv4_groups(p.head);
  const uint32_t r0 = blockIdx.x * (AMMON_WG / 16 * AMMON_KV4_LOAD_ROWS) + threadIdx.x / 16;
  const uint32_t rows = p.tokens * p.kv_heads;
  if (r0 >= rows || 8 * i >= p.head) return;
  const void *cache = blockIdx.y ? p.v_cache : p.k_cache;
  void *out = blockIdx.y ? p.v_out : p.k_out;
  uint32_t w[AMMON_KV4_LOAD_ROWS], sb[AMMON_KV4_LOAD_ROWS];
#pragma unroll
  for (int x = 0; x < AMMON_KV4_LOAD_ROWS; ++x) {
    const uint32_t r = min(r0 + x * (AMMON_WG / 16), rows - 1);
    const uint32_t g = r / p.tokens, t = r - g * p.tokens + p.first;
    w[x] = kv4_codes(cache, p.seq, ng, g, t)[piece * ng + j];
    sb[x] = kv4_scales(cache, p.kv_heads, p.seq, ng, g, t)[j];
  }
#pragma unroll
  for (int x = 0; x < AMMON_KV4_LOAD_ROWS; ++x) {
    const uint32_t r = r0 + x * (AMMON_WG / 16);
    if (r >= rows) return;
    const f16x8 v = kv4_numbers(w[x], sb[x], Kv4Bits());
    const size_t at = (size_t)r * p.head + 8 * i;
    if (p.head % 8 == 0 && p.out_dtype == AMMON_K_F32) {
      f32x4 *to = (f32x4 *)((float *)out + at);
      const f32x4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
      __builtin_nontemporal_store(lo, to);
      __builtin_nontemporal_store(hi, to + 1);
    } else if (p.head % 8 == 0) {
      u32x4 b;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        b[e] = (uint32_t)f32_to_bf16(v[2 * e]) | (uint32_t)f32_to_bf16(v[2 * e + 1]) << 16;
      __builtin_nontemporal_store(b, (u32x4 *)((uint16_t *)out + at));
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e)
        if (8 * i + e < p.head) store_elem(out, p.out_dtype, at + e, v[e]);
    }
  }
}

// Pass 1 on a (splits, kv heads, sets of eight query rows) grid.
#define KV4_PARTIAL(NAME, NG, MODE)                                                   \
  extern "C" __global__ __launch_bounds__(AMMON_WG, 2) void NAME(const ammon_k_step *step, \
                                                                ammon_k_attention p_) { \
    using Unit = Kv4Partial<NG, MODE>;                                                 \
    __shared__ u32x4 lds[Unit::LDS_BYTES / 16];                                        \
    ammon_k_attention p = p_;                                                          \
    p.step = step;                                                                     \
    Unit unit;                                                                         \
    if (unit.begin(p, blockIdx.x, blockIdx.y, blockIdx.z, (char *)lds))                \
      unit.run(p, (char *)lds);                                                        \
    else                                                                               \
      unit.out_of_range(p);                                                            \
  }
#define KV4_PARTIAL_NG(NG)                                          \
  KV4_PARTIAL(ammon_kv4_partial_n##NG, NG, KV4_DECODE)              \
  KV4_PARTIAL(ammon_kv4_partial_append_n##NG, NG, KV4_APPEND)       \
  KV4_PARTIAL(ammon_kv4_partial_tokens_n##NG, NG, KV4_TOKENS)
KV4_PARTIAL_NG(1)
KV4_PARTIAL_NG(2)
KV4_PARTIAL_NG(3)
KV4_PARTIAL_NG(4)

// Prefill tiles: one workgroup of two groups of four waves per (256 query rows, split,
// kv head), one per CU.
#define KV4_PREFILL(NG)                                                                     \
  extern "C" __global__ __launch_bounds__(KV4_PF_WG, 2) void ammon_kv4_prefill_n##NG(       \
      const ammon_k_step *step, ammon_k_attention p_) {                                     \
    using Tile = Kv4PrefillTile<NG>;                                                        \
    __shared__ u32x4 lds[Tile::LDS_BYTES / 16];                                             \
    ammon_k_attention p = p_;                                                               \
    p.step = step;                                                                          \
    Tile unit;                                                                              \
    unit.run(p, (char *)lds);                                                               \
  }
KV4_PREFILL(1)
KV4_PREFILL(2)
KV4_PREFILL(3)
KV4_PREFILL(4)
