// w4_prefill.hip -- kernels of w4_prefill_impl.h's tiles.
#include "w4_prefill_impl.h"

#define W4_GEMM_KERNEL(NAME, DIGITS, MODE, RT, CT, KS)                           \
  extern "C" __global__ __launch_bounds__(AMMON_WG) void NAME(ammon_k_gemm p) { \
    w4_gemm<DIGITS, MODE, RT, CT, KS>(p);                                        \
  }
#define W4_GEMM_MODES(DIGITS, SUFFIX, RT, CT, KS)                                              \
  W4_GEMM_KERNEL(ammon_w4_gemm_plain_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_PLAIN, RT, CT, KS)       \
  W4_GEMM_KERNEL(ammon_w4_gemm_residual_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_RESIDUAL, RT, CT, KS) \
  W4_GEMM_KERNEL(ammon_w4_gemm_swiglu_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_SWIGLU, RT, CT, KS)     \
  W4_GEMM_KERNEL(ammon_w4_gemm_qkv_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_QKV, RT, CT, KS)

W4_GEMM_MODES(1, t16, 2, 1, 4)
W4_GEMM_MODES(3, t16, 2, 1, 4)
W4_GEMM_MODES(1, t64, 4, 4, 1)
W4_GEMM_MODES(3, t64, 4, 4, 1)
