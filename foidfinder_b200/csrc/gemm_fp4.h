// Internal interface of the block-scaled 4-bit operators (csrc/fp4_quant.cu, csrc/gemm_fp4.cu).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

#include "../../include/foidfinder_b200.h"

namespace ff {

constexpr int EPI_QKV_NORM_ROPE = FF_EPI_QKV_NORM_ROPE;  // beside the Epi values of gemm_args.h

struct Fp4Operand {
  const uint8_t *codes, *scales;
  const float* row_scale;  // FF_FP4_NV
};

// Plain data, passed by value as a kernel parameter.
struct Fp4GemmArgs {
  int M, N, K;
  int num_kb;  // 256-column steps
  int tiles_m, tiles_n;
  const float *row_scale, *col_scale;  // FF_FP4_NV
  const float* bias;                   // or NULL
  void* out;
  int64_t ldo;
  int out_cols, tma_cols;  // columns written, and how many of them through TMA stores (a multiple of 8)
  int norm, q_heads, k_heads;
  float qk_eps;
  const float *q_w, *q_b, *k_w, *k_b;
  const float *rope_cos, *rope_sin;
  int tokens;
  int w_const;  // 1: W and its scales are not written by a kernel that may still run
  int* err;
};

int quantize_fp4(const void* x, int dtype, int64_t ldx, const float* gamma, const float* beta, float eps, int rows,
                 int cols, int fmt, uint8_t* codes, uint8_t* scales, float* row_scale, cudaStream_t stream);
int gemm_fp4(const Fp4Operand& A, const Fp4Operand& W, int fmt, int M, int N, int K, const ff_fp4_epilogue* e, int tile,
             bool w_const, cudaStream_t stream);

}  // namespace ff
