// 8-bit projection for few rows (at most 48: the last running requests of a decode batch), bound by the bytes of
// the weight matrix:
//
//   out[i, j] = (sum_k x[i, k] w[j, k]) * x_scale[i] * w_scale[j] (+ bias[j]),   sums exact in 32-bit integers
//
// A CTA owns 32 columns and all rows; its 8 or 16 warps split the K range in steps of 64 and are added through shared
// memory at the end.  The operands go from global memory straight into the fragments of the m16n8k32 integer
// products: which k an element belongs to does not matter as long as both operands agree, so the four lanes that
// share a row each load 16 consecutive bytes of its 64 and feed them to two products as (bytes 0-7) and (bytes 8-15).
// No staging, no barrier before the end, and one launch (256-row tcgen05 tiles take 9 us for 33 x 4096 x 4096, since with so few
// tiles most of their time is the latency of a pair's 32 k blocks; this kernel 7.7 us, and 3.8 us for one row: 4.4 TB/s of
// weights).  gemm_i8.cuh has the rule.
#include "gemm_i8.cuh"
#include "common.cuh"
#include "tcgen05.cuh"

namespace acache {
namespace few {

constexpr int COLS = 32, NB = COLS / 8;
// warps of a CTA: 16 for up to 32 rows (16 x 12288 x 4096: 11.4 us against 13.7 with 8), 8 where the registers allow no
// more.  The kernel is compiled for one CTA per SM: left to itself the compiler keeps fewer loads in flight (24 us)
template <int MT> constexpr int kWarps = MT <= 2 ? 16 : 8;

__device__ __forceinline__ void mma_i8(int32_t* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int MT>
__global__ void __launch_bounds__(kWarps<MT> * 32, 1) linear_i8_few_kernel(const Params p) {
  constexpr int NW = kWarps<MT>, NT = NW * 32;
  chain_release();
  chain_wait();
  constexpr int LD = COLS + 8;                        // rows 8 banks apart: a half warp's 64-bit stores do not collide
  extern __shared__ __align__(16) int32_t red[];      // [NW][MT * 16][LD]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n0 = blockIdx.x * COLS;
  const int row = lane >> 2, kq = (lane & 3) * 16;
  const int8_t* xp[2 * MT];
  const int8_t* wp[NB];
  bool x_ok[2 * MT], w_ok[NB];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    x_ok[i] = row + 8 * i < p.M;
    xp[i] = p.x + (int64_t)(x_ok[i] ? row + 8 * i : 0) * p.x_stride;
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    w_ok[i] = n0 + row + 8 * i < p.N;
    wp[i] = p.w + (int64_t)(w_ok[i] ? n0 + row + 8 * i : 0) * p.K;
  }
  int32_t acc[MT][NB][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][n][e] = 0;

  constexpr int DEPTH = 2;                            // steps in flight per warp
  uint4 a[DEPTH][2 * MT], b[DEPTH][NB];
  auto load = [&](int buf, int k0) {
    const int k = k0 + kq;
    const bool in = k < p.K;                          // K is a multiple of 16
#pragma unroll
    for (int i = 0; i < NB; ++i) b[buf][i] = in && w_ok[i] ? ld_global_nc(wp[i] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i)
      a[buf][i] = in && x_ok[i] ? *reinterpret_cast<const uint4*>(xp[i] + k) : make_uint4(0, 0, 0, 0);
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const uint4 lo = a[buf][2 * m], hi = a[buf][2 * m + 1], w = b[buf][n];
        mma_i8(acc[m][n], lo.x, hi.x, lo.y, hi.y, w.x, w.y);
        mma_i8(acc[m][n], lo.z, hi.z, lo.w, hi.w, w.z, w.w);
      }
  };
  const int step = NW * 64;
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) load(d, warp * 64 + d * step);
  for (int k = warp * 64; k < p.K; k += DEPTH * step) {      // a step behind the end loads zeros and adds nothing
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      load((d + DEPTH - 1) % DEPTH, k + (d + DEPTH - 1) * step);
      multiply(d);
    }
  }

#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      int32_t* at = red + (warp * MT * 16 + m * 16 + row) * LD + n * 8 + (lane & 3) * 2;
      *reinterpret_cast<int2*>(at) = make_int2(acc[m][n][0], acc[m][n][1]);
      *reinterpret_cast<int2*>(at + 8 * LD) = make_int2(acc[m][n][2], acc[m][n][3]);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 16 * (COLS / 2); i += NT) {
    const int r = i / (COLS / 2), c = (i % (COLS / 2)) * 2, n = n0 + c;
    if (r >= p.M || n >= p.N) continue;               // N is a multiple of 16: columns n and n + 1 exist together
    int32_t s0 = 0, s1 = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int2 v = *reinterpret_cast<const int2*>(red + (w * MT * 16 + r) * LD + c);
      s0 += v.x;
      s1 += v.y;
    }
    const float xs = p.x_scale[r];
    float o0 = ((float)s0 * xs) * p.w_scale[n], o1 = ((float)s1 * xs) * p.w_scale[n + 1];
    if (p.bias) {
      o0 += to_f32<T>(((const T*)p.bias)[n]);
      o1 += to_f32<T>(((const T*)p.bias)[n + 1]);
    }
    *reinterpret_cast<uint32_t*>((T*)p.out + (int64_t)r * p.ldo + n) = tc::pack2<T>(o0, o1);
  }
}

template <typename T, int MT>
static int launch_mt(const Params& p, cudaStream_t st) {
  constexpr size_t smem = (size_t)kWarps<MT> * MT * 16 * (COLS + 8) * 4;
  auto kern = linear_i8_few_kernel<T, MT>;
  static std::atomic<uint64_t> allowed{0};
  ACACHE_CUDA_CHECK(allow_smem((const void*)kern, smem, allowed));
  ACACHE_CUDA_CHECK(launch_chained(kern, dim3((p.N + COLS - 1) / COLS), dim3(kWarps<MT> * 32), smem, st, p));
  ACACHE_LAUNCH_CHECK();
  return ACACHE_OK;
}

template <typename T>
static int launch(const Params& p, cudaStream_t st) {
  switch ((p.M + 15) / 16) {
    case 1: return launch_mt<T, 1>(p, st);
    case 2: return launch_mt<T, 2>(p, st);
    default: return launch_mt<T, 3>(p, st);            // the rule takes at most 48 rows
  }
}

}  // namespace few

int linear_i8_few(const few::Params& p, int dtype, cudaStream_t st) {
  return dtype == ACACHE_BF16 ? few::launch<__nv_bfloat16>(p, st) : few::launch<__half>(p, st);
}

}  // namespace acache
