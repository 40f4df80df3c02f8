// w4_gemv.hip -- one token's products with 4-bit weights (w4_gemv_impl.h): one launch = one pass
// with the workgroups of the grid, x's digits in dynamic LDS.
#include "w4_gemv_impl.h"

// (The fields that the first requests depend on come as leading scalar arguments, which are
// preloaded into SGPRs at wave launch; p0's own are ignored.)
#define W4_GEMV_KERNEL(NAME, NW, ...)                                                         \
  extern "C" __global__ __launch_bounds__(64 * NW, 4) void NAME(                              \
      const void *w0, const float *x, const void *norm_w, uint32_t n, uint32_t norm_dtype,    \
      uint32_t row_blocks, uint32_t nwg, const void *w1, const void *w2, ammon_k_gemv p0) {   \
    extern __shared__ u32x4 lds[];                                                            \
    ammon_k_gemv p = p0;                                                                      \
    p.w0 = w0;                                                                                \
    p.x = x;                                                                                  \
    p.norm_w = norm_w;                                                                        \
    p.n = n;                                                                                  \
    p.norm_dtype = norm_dtype;                                                                \
    p.row_blocks = row_blocks;                                                                \
    p.w1 = w1;                                                                                \
    p.w2 = w2;                                                                                \
    __VA_ARGS__ pass;                                                                         \
    pass.run(p, nwg, (uint8_t *)lds);                                                         \
  }
#define W4_GEMV_MODES(KERNEL)                                     \
  KERNEL(ammon_w4_gemv_plain, AMMON_GEMV_PLAIN)                   \
  KERNEL(ammon_w4_gemv_residual, AMMON_GEMV_RESIDUAL)             \
  KERNEL(ammon_w4_gemv_swiglu, AMMON_GEMV_SWIGLU)                 \
  KERNEL(ammon_w4_gemv_qkv, AMMON_GEMV_QKV)                       \
  KERNEL(ammon_w4_gemv_plain_argmax, AMMON_GEMV_PLAIN_ARGMAX)

#define K8_ONE(NAME, MODE) W4_GEMV_KERNEL(NAME##_k8_one, 8, W4Sets<MODE, 8, 8, true>)
#define K8(NAME, MODE) W4_GEMV_KERNEL(NAME##_k8, 8, W4Sets<MODE, 8, 8, false>)
#define K2(NAME, MODE) W4_GEMV_KERNEL(NAME##_k2, 8, W4Sets<MODE, 2, 8, false>)
#define K8_WIDE(NAME, MODE) W4_GEMV_KERNEL(NAME##_k8_wide, 16, W4Sets<MODE, 8, 16, false>)
#define FLAT(NAME, MODE) W4_GEMV_KERNEL(NAME##_flat, 16, W4Flat<MODE>)
W4_GEMV_MODES(K8_ONE)
W4_GEMV_MODES(K8)
W4_GEMV_MODES(K2)
W4_GEMV_MODES(K8_WIDE)
W4_GEMV_MODES(FLAT)
