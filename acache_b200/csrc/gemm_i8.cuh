// 8-bit projection for few rows (gemm_i8_few.cu), chosen by acache_linear_int8 (gemm_tc.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace acache {
namespace few {

// Measured on B200 against 256-row tiles (us): 16 rows: 4096 x 4096 3.9 against 9.3, 4096 x 12288 13.5 against 17.5,
// 12288 x 4096 11.6 against 15.5, 3584 x 37888 about 35 either way; 32 rows: 4096 x 4096 5.3 against 9.1, 4096 x 12288 16.1
// against 15.1, 12288 x 4096 12.9 against 16.0, 3584 x 18944 21.4 against 20.3; 33 rows: 4096 x 4096 7.7 against 9.1, 64 rows
// 10.1 against 10.0; 33 rows 4096 x 12288 29 against 15.2, 12288 x 4096 28 against 16.0.
inline bool takes(int rows, int out_features, int in_features) {
  if (rows <= 32) return out_features <= 24576;
  return rows <= 64 && out_features <= 32 * 148 && in_features <= 6144;      // one CTA per SM
}

struct Params {
  const int8_t* x; int64_t x_stride; const float* x_scale; const int8_t* w; const float* w_scale; const void* bias; void* out;
  int64_t ldo; int M, N, K;
};

}  // namespace few

int linear_i8_few(const few::Params& p, int dtype, cudaStream_t st);

}  // namespace acache
