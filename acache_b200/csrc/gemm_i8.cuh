// 8-bit projection for few rows (gemm_i8_few.cu), chosen by acache_linear_int8 (gemm_tc.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace acache {
namespace few {

// Measured on B200 against 256-row tiles with K slices (us): 16 rows: 4096 x 4096 5.5 against 9.5, 4096 x 12288 17.7
// against 19.1, 12288 x 4096 15.4 against 16.1, 3584 x 37888 42.7 against 35.6; 33 rows: 4096 x 4096 9.1 against 10.2,
// 4096 x 12288 29 against 18.5, 12288 x 4096 28 against 17; 64 rows: 4096 x 4096 9.9 against 11.6.
inline bool takes(int rows, int out_features, int in_features) {
  if (rows <= 16) return out_features <= 24576;
  return rows <= 64 && out_features <= 32 * 148 && in_features <= 6144;      // one CTA per SM
}

struct Params {
  const int8_t* x; int64_t x_stride; const float* x_scale; const int8_t* w; const float* w_scale; const void* bias; void* out;
  int64_t ldo; int M, N, K;
};

}  // namespace few

int linear_i8_few(const few::Params& p, int dtype, cudaStream_t st);

}  // namespace acache
