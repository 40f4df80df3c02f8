// qkv_store.h -- the QKV epilogue of the prefill GEMMs (prefill.hip, w4_prefill.hip).
#pragma once

#include "device_common.h"

// QKV epilogue of virtual rows (v, v + 1) of token t: rotate q and k pairs
// with the cos/sin table at position step->position + t; q to y, k and raw
// v rows to the head-major caches (src/kernels.rs:174-226), or with kv_rows to
// fp32 rows [tokens, kv_dim]; a position past the cache poisons q (and such
// rows) and touches no cache.  fcr, fci: the pair's cos and sin
// (unused for v rows and positions past the cache).
AMMON_DEV void qkv_store_pair(const ammon_k_gemm &p, uint32_t t, uint32_t v, float a0, float a1,
                              float fcr, float fci) {
#pragma clang fp contract(off)
  const uint32_t first = p.step->position, pos = first + t;
  const uint32_t kvd = p.kv_dim;
  if (first >= p.seq || t >= p.seq - first) {
    if (v < p.d) {
      p.y[(size_t)t * p.d + v] = __uint_as_float(0x7fc00000u);
      p.y[(size_t)t * p.d + v + 1] = __uint_as_float(0x7fc00000u);
    } else if (p.kv_rows) {
      const uint32_t rr = v - p.d;
      const float nan = __uint_as_float(0x7fc00000u);
      store_pair_out(rr < kvd ? p.k_cache : p.v_cache, AMMON_K_F32, (size_t)t * kvd + rr % kvd, nan, nan);
    }
    return;
  }
  if (v < p.d + kvd) {
    const uint32_t rr = v < p.d ? v : v - p.d;
    const float o0 = a0 * fcr - a1 * fci;
    const float o1 = a0 * fci + a1 * fcr;
    if (v < p.d) {
      p.y[(size_t)t * p.d + v] = o0;
      p.y[(size_t)t * p.d + v + 1] = o1;
    } else {
      store_pair_out(p.k_cache, p.kv_dtype,
                     p.kv_rows ? (size_t)t * kvd + rr
                               : ((size_t)(rr / p.head) * p.seq + pos) * p.head + rr % p.head,
                     o0, o1);
    }
  } else {
    const uint32_t rv = v - p.d - kvd;
    store_pair_out(p.v_cache, p.kv_dtype,
                   p.kv_rows ? (size_t)t * kvd + rv
                             : ((size_t)(rv / p.head) * p.seq + pos) * p.head + rv % p.head,
                   a0, a1);
  }
}

AMMON_DEV void qkv_store_pair(const ammon_k_gemm &p, uint32_t t, uint32_t v, float a0, float a1) {
  const uint32_t pos = p.step->position + t, rr = v < p.d ? v : v - p.d;
  float fcr = 0.f, fci = 0.f;
  if (pos < p.seq && v < p.d + p.kv_dim) {
    const float *cs = p.table + (size_t)pos * p.head + rr % p.head;
    fcr = cs[0], fci = cs[1];
  }
  qkv_store_pair(p, t, v, a0, a1, fcr, fci);
}
