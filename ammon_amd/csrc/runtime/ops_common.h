// ops_common.h -- what the C-ABI entry points (ops.cpp, w4.cpp) share: dtypes, overlap checks,
// launches, the GEMV family's arguments.
#pragma once

#include <algorithm>
#include <cmath>

#include "internal.h"

namespace ammon_rt {

using DeviceGuard = ammon_rt::DeviceScope;

inline uint32_t cdiv(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

inline bool valid_dtype(ammon_dtype d) { return d == AMMON_F32 || d == AMMON_BF16; }
inline bool valid_kv(ammon_dtype d) { return valid_dtype(d) || d == AMMON_KV4; }
inline size_t dsize(ammon_dtype d) { return d == AMMON_BF16 ? 2 : 4; }

inline bool overlaps(const void *a, size_t abytes, const void *b, size_t bbytes) {
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  return a0 < b0 + bbytes && b0 < a0 + abytes;
}

template <typename P>
ammon_status launch3(ammon_runtime *rt, ammon_stream s, hipFunction_t f, uint32_t gx, uint32_t gy,
                     uint32_t gz, uint32_t shmem, P &params, const char *what) {
  if (gx == 0 || gy == 0 || gz == 0) return AMMON_OK;
  DeviceGuard guard(rt->device);
  hipStream_t st = s ? (hipStream_t)s : rt->stream;
  void *args[] = {&params};
  hipError_t e = hipModuleLaunchKernel(f, gx, gy, gz, kWorkgroup, 1, 1, shmem, st, args, nullptr);
  if (e != hipSuccess) return hip_error(e, what);
  return AMMON_OK;
}

template <typename P>
ammon_status launch(ammon_runtime *rt, ammon_stream s, hipFunction_t f, uint32_t gx, uint32_t gy,
                    uint32_t shmem, P &params, const char *what) {
  return launch3(rt, s, f, gx, gy, 1, shmem, params, what);
}

#define REQUIRE_RT()                                              \
  do {                                                            \
    if (!rt) return set_error(AMMON_E_VALIDATION, "runtime is NULL"); \
  } while (0)

#define VALIDATE_ONLY()                                  \
  do {                                                   \
    if (stream == AMMON_STREAM_VALIDATE) return AMMON_OK; \
  } while (0)

struct GemvArgs {
  int mode;
  const void *w0, *w1, *w2;
  ammon_dtype w_dtype;
  uint32_t d, n, rows;
  const float *x;
  const void *norm_w;
  ammon_dtype norm_dtype;
  float eps;
  const float *residual;
  float *y;
  void *k_cache, *v_cache;
  const ammon_decode_step *step;
  const float *table;
  uint32_t kv_dim, head, seq;
  ammon_dtype kv_dtype;
  bool kv_rows;        // QKV: k and v as fp32 rows, not cache rows
  float *cand_v;       // PLAIN_ARGMAX: candidate arrays of cand_cap entries
  uint32_t *cand_i;
  uint32_t cand_cap;
};

// A GEMV over AMMON_W4 weights: validated and launched (w4.cpp).
ammon_status w4_gemv(ammon_runtime *rt, ammon_stream stream, const GemvArgs &a, const char *what,
                     uint32_t *grid_out);

}  // namespace ammon_rt
