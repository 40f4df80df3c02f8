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

#define W4_BIG_KERNEL(NAME, DIGITS, MODE, RT, CT)                                   \
  extern "C" __global__ __launch_bounds__(AMMON_WG, 2) void NAME(ammon_k_gemm p) { \
    w4_gemm_big<DIGITS, MODE, RT, CT>(p);                                          \
  }
#define W4_BIG_MODES(DIGITS, SUFFIX, RT, CT)                                               \
  W4_BIG_KERNEL(ammon_w4_gemm_plain_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_PLAIN, RT, CT)       \
  W4_BIG_KERNEL(ammon_w4_gemm_residual_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_RESIDUAL, RT, CT) \
  W4_BIG_KERNEL(ammon_w4_gemm_swiglu_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_SWIGLU, RT, CT)     \
  W4_BIG_KERNEL(ammon_w4_gemm_qkv_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_QKV, RT, CT)
W4_BIG_MODES(1, t64, 4, 4)
W4_BIG_MODES(3, t64, 4, 4)
