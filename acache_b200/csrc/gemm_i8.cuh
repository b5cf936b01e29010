// 8-bit projection for few rows (at most 48, gemm_i8_few.cu), chosen by acache_linear_int8 (gemm_tc.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace acache {
namespace few {

// Which launches it takes.  A CTA has 32 columns and the whole K range, a round of CTAs is one per SM, and a round costs in
// proportion to K and to the rows in steps of 16; the 256-row tiles cost nearly the same up to 256 rows and slice a long K range.
// Measured on B200, weights from HBM, us, this kernel / the tiles, in_features x out_features:
//   rows          16         24         32         33        48
//   512 x 4096     2.1 / 5.6  2.7 / 4.9  2.9 / 4.9  3.3 / 4.9  3.5 / 5.0
//   1024 x 12288   7.2 / 8.2  9.6 / 9.3  9.9 / 9.5 10.7 / 8.7 10.8 / 9.7
//   4096 x 4096    5.5 / 13.5 6.2 / 13.5 6.6 / 10.8 9.4 / 10.8 9.6 / 10.9
//   3584 x 4608    5.4 / 12.8 6.0 / 13.2 6.3 / 16.3 9.3 / 13.0 10.1 / 10.3
//   4096 x 12288  13.7 / 17.3 15.4 / 17.6 16.1 / 14.8 24.8 / 14.8
//   3584 x 18944  18.2 / 19.9 20.1 / 22.1 21.1 / 19.9 31.9 / 20.1
//   4096 x 24576  25.1 / 30.1 28.6 / 30.0 30.3 / 23.8
//   3584 x 37888  34.1 / 33.2 39.0 / 40.0 40.7 / 34.4
//   8192 x 8192   15.8 / 17.3 17.5 / 17.8 17.9 / 17.8 29.8 / 18.0
//   8192 x 512     5.3 / 9.5  7.1 / 9.7  7.3 / 9.7 11.3 / 9.7
//   12288 x 4096  11.5 / 15.2 12.4 / 15.8 12.8 / 15.9 22.0 / 16.0
//   18944 x 3584  15.5 / 18.8 17.7 / 19.4 18.3 / 19.8 32.2 / 20.0
//   28672 x 8192  43.6 / 44.2 50.5 / 44.8 52.6 / 45.1
//   16384 x 1024  11.1 / 12.4 13.6 / 12.6 13.9 / 12.7 26.3 / 12.7
//   32768 x 256   18.5 / 14.9 23.8 / 14.9 24.5 / 14.9 48.9 / 14.8
//   131056 x 64   71.2 / 30.9 87.9 / 31.2
inline bool takes(int rows, int out_features, int in_features) {
  const bool one_round = out_features <= 32 * 148;
  if (rows <= 16) return out_features <= 32768 && in_features <= 16ll * out_features;
  if (rows <= 32 && one_round) return in_features <= 8192 || in_features <= 8ll * out_features;
  if (rows <= 24) return out_features <= 24576 && in_features >= 2048 && in_features <= 8192;
  return rows <= 48 && one_round && in_features <= 6144;
}

struct Params {
  const int8_t* x; int64_t x_stride; const float* x_scale; const int8_t* w; const float* w_scale; const void* bias; void* out;
  int64_t ldo; int M, N, K;
};

}  // namespace few

int linear_i8_few(const few::Params& p, int dtype, cudaStream_t st);

}  // namespace acache
