// w4_gemv.hip -- one token's products with 4-bit weights (w4_gemv_impl.h): one launch = one pass
// with the workgroups of the grid, x's digits in dynamic LDS.
#include "w4_gemv_impl.h"

// KS waves of a set, NW of a workgroup
#define W4_GEMV_KERNEL(NAME, MODE, KS, NW)                                                     \
  extern "C" __global__ __launch_bounds__(64 * NW, 4) void NAME(ammon_k_gemv p, uint32_t nwg) { \
    extern __shared__ u32x4 lds[];                                                             \
    W4Gemv<MODE, KS, NW> pass;                                                                 \
    pass.run(p, nwg, (uint8_t *)lds);                                                          \
  }
#define W4_GEMV_MODES(SUFFIX, KS, NW)                                         \
  W4_GEMV_KERNEL(ammon_w4_gemv_plain##SUFFIX, AMMON_GEMV_PLAIN, KS, NW)       \
  W4_GEMV_KERNEL(ammon_w4_gemv_residual##SUFFIX, AMMON_GEMV_RESIDUAL, KS, NW) \
  W4_GEMV_KERNEL(ammon_w4_gemv_swiglu##SUFFIX, AMMON_GEMV_SWIGLU, KS, NW)     \
  W4_GEMV_KERNEL(ammon_w4_gemv_qkv##SUFFIX, AMMON_GEMV_QKV, KS, NW)           \
  W4_GEMV_KERNEL(ammon_w4_gemv_plain_argmax##SUFFIX, AMMON_GEMV_PLAIN_ARGMAX, KS, NW)

W4_GEMV_MODES(_k8, 8, 8)
W4_GEMV_MODES(_k2, 2, 8)
W4_GEMV_MODES(_k8_wide, 8, 16)
