// w4_gemv.hip -- one token's products with 4-bit weights (w4_gemv_impl.h): one launch = one pass
// with the workgroups of the grid, x's digits in dynamic LDS.
#include "w4_gemv_impl.h"

#define W4_GEMV_KERNEL(NAME, MODE, US)                                                          \
  extern "C" __global__ __launch_bounds__(64 * AMMON_W4_SET * US) void NAME(ammon_k_gemv p, uint32_t nwg) { \
    extern __shared__ u32x4 lds[];                                                              \
    W4Gemv<MODE, US> pass;                                                                      \
    pass.run(p, nwg, (uint8_t *)lds);                                                           \
  }
#define W4_GEMV_MODES(SUFFIX, US)                                        \
  W4_GEMV_KERNEL(ammon_w4_gemv_plain##SUFFIX, AMMON_GEMV_PLAIN, US)      \
  W4_GEMV_KERNEL(ammon_w4_gemv_residual##SUFFIX, AMMON_GEMV_RESIDUAL, US) \
  W4_GEMV_KERNEL(ammon_w4_gemv_swiglu##SUFFIX, AMMON_GEMV_SWIGLU, US)    \
  W4_GEMV_KERNEL(ammon_w4_gemv_qkv##SUFFIX, AMMON_GEMV_QKV, US)          \
  W4_GEMV_KERNEL(ammon_w4_gemv_plain_argmax##SUFFIX, AMMON_GEMV_PLAIN_ARGMAX, US)

W4_GEMV_MODES(_s1, 1)
W4_GEMV_MODES(_s2, 2)
