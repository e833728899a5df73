// A product with 4-bit weights as both of its kernels take it: w4_linear.cu for few rows, w4_gemm.cu for more.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mvb {

struct W4LinearCall {
  __nv_bfloat16* y;
  int64_t ldy;
  const void* x;  // bf16, or 8 bits where there are row_scales; rows on 16 bytes
  int64_t ldx;
  const float* row_scales;
  const uint8_t* records;
  int rows, n, k, group;
};

int w4_gemm(const char* name, const W4LinearCall& call, cudaStream_t stream);

}  // namespace mvb
