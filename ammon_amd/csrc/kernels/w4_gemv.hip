// w4_gemv.hip -- one token's products with 4-bit weights (w4_gemv_impl.h): one launch = one pass
// with the workgroups of the grid, x's digits in dynamic LDS.
#include "w4_gemv_impl.h"

#define W4_GEMV_KERNEL(NAME, MODE)                                                    \
  extern "C" __global__ __launch_bounds__(AMMON_WG) void NAME(ammon_k_gemv p, uint32_t nwg) { \
    extern __shared__ u32x4 lds[];                                                   \
    W4Gemv<MODE> pass;                                                               \
    pass.run(p, nwg, (uint8_t *)lds);                                                \
  }

W4_GEMV_KERNEL(ammon_w4_gemv_plain, AMMON_GEMV_PLAIN)
W4_GEMV_KERNEL(ammon_w4_gemv_residual, AMMON_GEMV_RESIDUAL)
W4_GEMV_KERNEL(ammon_w4_gemv_swiglu, AMMON_GEMV_SWIGLU)
W4_GEMV_KERNEL(ammon_w4_gemv_qkv, AMMON_GEMV_QKV)
W4_GEMV_KERNEL(ammon_w4_gemv_plain_argmax, AMMON_GEMV_PLAIN_ARGMAX)
