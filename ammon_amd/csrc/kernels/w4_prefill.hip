// w4_prefill.hip -- kernels of w4_prefill_impl.h's tiles.
#include "w4_prefill_impl.h"

#define W4_GEMM_UNGATED(KERNEL, DIGITS, SUFFIX, ...)                                             \
  KERNEL(ammon_w4_gemm_plain_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_PLAIN, __VA_ARGS__)       \
  KERNEL(ammon_w4_gemm_residual_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_RESIDUAL, __VA_ARGS__) \
  KERNEL(ammon_w4_gemm_qkv_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_QKV, __VA_ARGS__)
#define W4_GEMM_MODES(KERNEL, DIGITS, SUFFIX, ...)    \
  W4_GEMM_UNGATED(KERNEL, DIGITS, SUFFIX, __VA_ARGS__) \
  KERNEL(ammon_w4_gemm_swiglu_q##DIGITS##_##SUFFIX, DIGITS, AMMON_GEMV_SWIGLU, __VA_ARGS__)

// panels of results, token panels, waves
#define W4_SHORT_KERNEL(NAME, DIGITS, MODE, PANELS, CT, SPLIT)                    \
  extern "C" __global__ __launch_bounds__(64 * SPLIT) void NAME(ammon_k_gemm p) { \
    w4_gemm_short<DIGITS, MODE, PANELS, CT, SPLIT>(p);                            \
  }
W4_GEMM_MODES(W4_SHORT_KERNEL, 1, t16, 1, 1, 8)
W4_GEMM_UNGATED(W4_SHORT_KERNEL, 1, t16_deep, 1, 1, 16)
W4_GEMM_MODES(W4_SHORT_KERNEL, 1, t16_x4, 4, 1, 8)
W4_GEMM_MODES(W4_SHORT_KERNEL, 1, t32_x2, 2, 2, 8)
W4_GEMM_MODES(W4_SHORT_KERNEL, 3, t16, 1, 1, 8)
W4_GEMM_UNGATED(W4_SHORT_KERNEL, 3, t16_deep, 1, 1, 16)
W4_GEMM_MODES(W4_SHORT_KERNEL, 3, t16_x2, 2, 1, 8)
W4_GEMM_MODES(W4_SHORT_KERNEL, 3, t16_x4, 4, 1, 8)

// panels of rows per wave, token panels, workgroups per CU.  The long tile shares a wave's codes or the
// tokens' digits between more products: of one digit, whose sums' scaling keeps the vector units
// busy, the codes (2048 tokens x 28672 x 4096 gated: 313 us, 64-token tiles 375); of three the
// digits (660 us, 64-token tiles 778).
#define W4_BIG_KERNEL(NAME, DIGITS, MODE, RT, CT, OCC)                                \
  extern "C" __global__ __launch_bounds__(AMMON_WG, OCC) void NAME(ammon_k_gemm p) { \
    w4_gemm_big<DIGITS, MODE, RT, CT>(p);                                          \
  }
W4_GEMM_MODES(W4_BIG_KERNEL, 1, t64, 2, 4, 3)
W4_GEMM_MODES(W4_BIG_KERNEL, 1, long, 2, 8, 3)
W4_GEMM_MODES(W4_BIG_KERNEL, 3, t64, 2, 4, 3)
W4_GEMM_MODES(W4_BIG_KERNEL, 3, long, 4, 4, 2)
