// Rows quantised to 8-bit integers by the kernel that produces them (input side of the 8-bit
// projections in gemm_tc.cu and gemm_i8_few.cu):
//
//   a_i = max_k |y_ik|      q_ik = round(127 y_ik / a_i), ties to even      scale_i = a_i / 127
//
// where y is the row itself, its RMSNorm (with the residual add before it), or act(gate) * up of a
// row that holds both halves.  y stays in fp32 registers from the producer to the rounding: it is
// never rounded to the model type in between, which the unfused chain does.
//
// The quotient t = 127 y / a is formed as y * (127 / a), which is within 2 units of its last place, and
// for rows quantised as they are its 24 significant bits are rounded to 21.  For 16-bit y and a with
// significands Y, A < 2^11 the exact t lies on a tie k + 1/2 or at least t / (254 Y) > 2^-19 t from one
// (the difference is a whole number of units of y's last place over 2a), so rounding to 21 bits restores
// exact ties and moves nothing else across one: 16-bit rows are quantised as by exact division, at the
// price of a multiplication.  For fp32 rows such a rounding would move values that are no ties (2^-14 of them), so a quotient
// within its error of a tie is decided in 64 bits, where 127 y and (k + 1/2) a are exact.  Norms and gated values are fp32
// results without such ties.
//
// A norm's factor rsqrt(mean(x^2) + eps) cancels in q: q = round(127 x w / max|x w|), and only the scale
// gets it.  So the largest value and the sum of squares are reduced together, behind one barrier.  Where x w or
// the sum of squares leaves fp32 the row is done again, factor first.
//
// A row that holds an infinity or a NaN gets the scale NaN and zeros, so that everything computed
// from it is NaN; a row of zeros gets the scale 0.
//
// A CTA works on a row at a time, one pass over global memory (the row stays in registers), and while it reduces
// and rounds one row the next one it will take is on its way.  Bound by HBM at size and by a row's chain of reduction,
// barrier and division at 3-4 thousand columns: gate 2304 x 12288 27 us (5.2 TB/s), 512 x 12288 7.8 us; norm 4096 x 3584
// 12.5 us (14.6 with two barriers and the factor in every value), 2305 x 3584 7.9 us, 512 x 4096 3.3 us.
#include "common.cuh"
#include "tcgen05.cuh"

namespace acache {
namespace quant {

enum { SRC_ROWS = 0, SRC_NORM = 1, SRC_GATE = 2 };

struct Params {
  const void* x; int64_t x_stride; const void* delta; int64_t d_stride; const void* weight; float eps; int act;
  int8_t* q; float* scale; int n_rows, n_cols;
};

// silu(x) = x / (1 + e^-x) for two |x| <= 80 (e^-x leaves fp32 below, the exponent far above).  e^-x is a power of two whose exponent -x log2(e) is
// formed with what its rounding loses, since an error of d there is one of 0.7 d of the value: within 2^-20 of its value.  Fast
// powers and reciprocals, two values to an instruction: expf and exact divisions made the kernel bound by instructions
// (512 x 12288: 14 us against 8).  An infinity gives a NaN, as its row gets a NaN scale either way.
constexpr float kLog2e = 1.44269504f, kLog2eRest = 1.92596299e-8f;      // log2(e) is the two added
__device__ __forceinline__ uint64_t silu2(uint64_t x) {
  using namespace tc;
  float t0, t1, d0, d1;
  const uint64_t t = mul_f32x2(x, pack_f32x2(kLog2e, kLog2e));
  uint64_t rest = fma_f32x2(x, pack_f32x2(-kLog2e, -kLog2e), t);                 // what -t lacks of -x log2(e)
  rest = fma_f32x2(x, pack_f32x2(-kLog2eRest, -kLog2eRest), rest);
  unpack_f32x2(t, t0, t1);
  const uint64_t p = pack_f32x2(ex2(-t0), ex2(-t1));
  const uint64_t e = fma_f32x2(p, mul_f32x2(rest, pack_f32x2(0.69314718f, 0.69314718f)), p);
  unpack_f32x2(add_f32x2(e, pack_f32x2(1.f, 1.f)), d0, d1);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d1));
  return mul_f32x2(x, pack_f32x2(d0, d1));
}
__device__ __forceinline__ float relu(float x) { return x > 0.f ? x : (x == x ? 0.f : x); }      // a NaN stays
// gelu(x) = x (1 + erf(x / sqrt 2)) / 2 down to -3: two steps of erff over a sum that cancels, within 2^-14 of its value
__device__ __forceinline__ float gelu(float x) { return 0.5f * x * (1.f + erff(x * 0.70710678f)); }

// gates further from zero (silu) or below it (gelu) than this have forms of their own, which would cost the others a tenth (silu) to
// a third (gelu) more
__device__ __forceinline__ float far_limit(int act) { return act == 0 ? 80.f : (act == 1 ? INFINITY : 3.f); }
__device__ __forceinline__ float far_of(float x, int act) { return act == 0 ? fabsf(x) : -x; }
// silu as x e^x / (1 + e^x): within 2^-20 of its value, and 2^-149 |x| below -87, where e^x is subnormal; gelu as
// x erfc(-x / sqrt 2) / 2: the rounding of the argument counts x^2 times, within (x^2 + 8) 2^-23 of its value
__device__ __noinline__ float act_far(float x, int act) {
  if (act != 0) return 0.5f * x * erfcf(x * -0.70710678f);
  if (x > 0.f) return x;
  if (x < -128.f) return x * 0.f;                         // e^x is below all numbers, and its exponent might overflow
  const float t = x * kLog2e, rest = fmaf(x, kLog2eRest, fmaf(x, kLog2e, -t));
  float p;
  asm("ex2.approx.f32 %0, %1;" : "=f"(p) : "f"(t));       // with subnormal results
  const float z = fmaf(p, rest * 0.69314718f, p);
  return __fdividef(x * z, 1.f + z);
}

// y = act(gate) * up for N values; `far` grows to the largest far_of() of the gates
template <int N>
__device__ __forceinline__ void gated(const float (&g)[N], const float (&u)[N], int act, float (&y)[N], float& far) {
  using namespace tc;
  if (act == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 2) far = max3(far, fabsf(g[e]), fabsf(g[e + 1]));
#pragma unroll
    for (int e = 0; e < N; e += 2)
      unpack_f32x2(mul_f32x2(silu2(pack_f32x2(g[e], g[e + 1])), pack_f32x2(u[e], u[e + 1])), y[e], y[e + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) far = max3(far, -g[e], -g[e + 1]);
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = (act == 1 ? relu(g[e]) : gelu(g[e])) * u[e];
  }
}

// max(top, |a|, |b|), a NaN if one of them is
__device__ __forceinline__ float max_abs(float top, float a, float b) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(top), "f"(a), "f"(b));
  return m;
}
// |v| as bits that order like numbers: a NaN is larger than an infinity, which is larger than any number
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// what a row is shrunk by when its sum of squares leaves fp32: the largest values squared and added stay inside
constexpr float kShrink = 0x1p-75f;

struct RowScale { float pre, f, top; bool dead; };   // q = round((v * pre) * f), top the largest |v * pre|

// top_bits: the largest |v| of the row; the row itself is rs * v
__device__ __forceinline__ RowScale row_scale(uint32_t top_bits, float rs, float* scale_out) {
  RowScale r;
  const float top = __uint_as_float(top_bits), a = top * rs;
  const bool finite = abs_bits(a) < 0x7F800000u;
  r.pre = top < 0x1p-100f ? 0x1p100f : 1.f;     // keeps 127 / top inside the range of fp32
  r.dead = !finite || a == 0.f;
  r.top = top * r.pre;
  r.f = r.dead ? 0.f : 127.f / r.top;
  if (scale_out) *scale_out = finite ? a / 127.f : __uint_as_float(0x7FC00000u);
  return r;
}

// round(127 v / top) of a quotient t that lies near a tie
__device__ __noinline__ uint32_t round_near_tie(float v, float t, float top) {
  const int k = (int)floorf(fabsf(t) - 0.25f);          // between k and k + 1
  const double x = 127.0 * fabsf(v), tie = (k + 0.5) * top;
  const int q = k + (x > tie || (x == tie && (k & 1)));
  return (uint32_t)(v < 0.f ? -q : q);
}

// the quantised value of v * pre in the low byte (of a row that is not dead).  How a quotient next to a tie is rounded:
enum { AS_IT_IS = 0, TIES_16 = 1, TIES_32 = 2 };        // T a 16-bit type: 21 significant bits; fp32: exactly
template <typename T, int SRC> constexpr int kTies = SRC != SRC_ROWS ? AS_IT_IS : (sizeof(T) == 2 ? TIES_16 : TIES_32);
template <int TIES>
__device__ __forceinline__ uint32_t quantise(float v, const RowScale& r) {
  float t = v * r.f;
  if (TIES == TIES_16) t = __uint_as_float((__float_as_uint(t) + 4u) & ~7u);
  const float shifted = t + 0x1.8p23f;
  // t is within 2^-16 of the quotient
  if (TIES == TIES_32 && fabsf(t - (shifted - 0x1.8p23f)) > 0.5f - 0x1p-15f) return round_near_tie(v, t, r.top);
  return __float_as_uint(shifted);
}

template <int NT>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) m = max(m, red[i]);
  return m;
}

// the warp's sum into its place, to be read behind the next barrier
__device__ __forceinline__ void warp_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
}

template <int NT>
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) s += red[i];
  return s;
}

// CTAs per SM the kernel is compiled and launched for: 1024 threads (1280: norm 2305 x 3584 9.8 us against 8.3; 768: gate
// 512 x 12288 8.7 us against 7.7), 1536 for rows of one vector a thread
constexpr int resident(int nt, int vpt) { return vpt == 1 ? 1536 / nt : (vpt <= 4 ? 1024 / nt : 1); }

template <typename T, int SRC, int NT, int VPT>
__global__ void __launch_bounds__(NT, resident(NT, VPT)) quantise_kernel(const Params p) {
  constexpr int E = 16 / sizeof(T);
  constexpr bool TWO = SRC != SRC_ROWS;           // a second input row: up halves, or the residual update
  constexpr int TIES = kTies<T, SRC>;
  chain_release();
  chain_wait();
  // a thread's vectors of the next row, on their way while it works on the current one (they are its own: no barrier)
  extern __shared__ __align__(16) uint4 next_row[];      // [TWO ? 2 : 1][VPT][NT], and the weights of wide norms, [VPT][NT]
  __shared__ float red_sum[3][NT / 32];            // two buffers: a fast warp may be one row ahead of a slow one
  __shared__ uint32_t red_max[3][NT / 32];
  const int tid = threadIdx.x, nvec = p.n_cols / E;
  const bool two = SRC == SRC_GATE || (SRC == SRC_NORM && p.delta);
  auto fetch = [&](int64_t row) {
    const T* xr = (const T*)p.x + row * p.x_stride;
    const T* yr = SRC == SRC_GATE ? xr + p.n_cols : (const T*)p.delta + row * p.d_stride;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = tid + i * NT;
      if (c < nvec) {
        tc::cp_async16(tc::smem_u32(next_row + i * NT + tid), xr + (int64_t)c * E, true);
        if (TWO && two) tc::cp_async16(tc::smem_u32(next_row + (VPT + i) * NT + tid), yr + (int64_t)c * E, true);
      }
    }
    tc::cp_async_commit();
  };
  // the norm's weights, a thread's own vectors again: in registers, but in shared memory where they would spill
  constexpr bool W_SMEM = VPT > 2;
  [[maybe_unused]] uint4* weights = next_row + 2 * VPT * NT;
  [[maybe_unused]] uint4 held[W_SMEM ? 1 : VPT];
  int64_t row = blockIdx.x;
  if (SRC == SRC_NORM && W_SMEM) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = tid + i * NT;
      if (c < nvec) tc::cp_async16(tc::smem_u32(weights + c), (const T*)p.weight + (int64_t)c * E, true);
    }
  }
  fetch(row);
  if (SRC == SRC_NORM && !W_SMEM) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (tid + i * NT < nvec) held[i] = *reinterpret_cast<const uint4*>((const T*)p.weight + (int64_t)(tid + i * NT) * E);
  }
  const float inv_cols = 1.f / (float)p.n_cols;
  for (int parity = 0; row < p.n_rows; row += gridDim.x, parity ^= 1) {
    T* xr = (T*)p.x + row * p.x_stride;
    float y[VPT][E];                              // SRC_NORM: x * weight, without the row's factor
    float top = 0.f, ss = 0.f, rs = 1.f;
    [[maybe_unused]] float far = 0.f;
    tc::cp_async_wait<0>();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = tid + i * NT;
      if (c < nvec) {
        Vec16<T> a, b, w;
        a.u = next_row[i * NT + tid];
        if (SRC == SRC_NORM) w.u = W_SMEM ? weights[c] : held[W_SMEM ? 0 : i];
        if (TWO && two) b.u = next_row[(VPT + i) * NT + tid];
        if (SRC == SRC_NORM && two) {             // the residual add, rounded to T, written back
#pragma unroll
          for (int e = 0; e < E; ++e) a.e[e] = from_f32<T>(to_f32<T>(a.e[e]) + to_f32<T>(b.e[e]));
          *reinterpret_cast<uint4*>(xr + (int64_t)c * E) = a.u;
        }
        if constexpr (SRC == SRC_GATE) {
          float gate[E], up[E];
#pragma unroll
          for (int e = 0; e < E; ++e) {
            gate[e] = to_f32<T>(a.e[e]);
            up[e] = to_f32<T>(b.e[e]);
          }
          gated<E>(gate, up, p.act, y[i], far);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float v = to_f32<T>(a.e[e]);
            if (SRC == SRC_NORM) ss = fmaf(v, v, ss);
            y[i][e] = SRC == SRC_NORM ? v * to_f32<T>(w.e[e]) : v;
          }
        }
        if constexpr (SRC != SRC_GATE) {
#pragma unroll
          for (int e = 0; e < E; e += 2) top = max_abs(top, y[i][e], y[i][e + 1]);
        }
      }
    }
    if constexpr (SRC == SRC_GATE) {
      const float limit = far_limit(p.act);
      if (far > limit) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if (tid + i * NT < nvec) {
            Vec16<T> a, b;
            a.u = next_row[i * NT + tid];
            b.u = next_row[(VPT + i) * NT + tid];
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (far_of(to_f32<T>(a.e[e]), p.act) > limit) y[i][e] = act_far(to_f32<T>(a.e[e]), p.act) * to_f32<T>(b.e[e]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (tid + i * NT < nvec) {
#pragma unroll
          for (int e = 0; e < E; e += 2) top = max_abs(top, y[i][e], y[i][e + 1]);
        }
      }
    }
    if (row + gridDim.x < p.n_rows) fetch(row + gridDim.x);
    // one barrier for the row's largest value and, of a norm, its sum of squares
    if (SRC == SRC_NORM) warp_sum(ss, red_sum[parity]);
    uint32_t top_bits = block_max<NT>(abs_bits(top), red_max[parity]);
    if (SRC == SRC_NORM) {
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < NT / 32; ++i) ss += red_sum[parity][i];
      rs = rsqrtf(ss * inv_cols + p.eps);
    }
    RowScale r = row_scale(top_bits, rs, tid == 0 ? p.scale + row : nullptr);
    if (r.dead || r.pre != 1.f) {                 // rare, and the same for the whole CTA
      if (SRC == SRC_NORM && (top_bits >= 0x7F800000u || !(ss < INFINITY))) {
        // x * weight, or the sum of squares, may leave the range of fp32 where the norm does not: the factor first, from the
        // row in global memory, and the squares of smaller values
        float k = 1.f;
        if (!(ss < INFINITY)) {
          k = kShrink;
          ss = 0.f;
#pragma unroll
          for (int i = 0; i < VPT; ++i) {
            if (tid + i * NT < nvec) {
              Vec16<T> a;
              a.u = *reinterpret_cast<const uint4*>(xr + (int64_t)(tid + i * NT) * E);
#pragma unroll
              for (int e = 0; e < E; ++e) ss = fmaf(to_f32<T>(a.e[e]) * k, to_f32<T>(a.e[e]) * k, ss);
            }
          }
          rs = rsqrtf(block_sum<NT>(ss, red_sum[2]) * inv_cols + p.eps * k * k);
        }
        top = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if (tid + i * NT < nvec) {
            Vec16<T> a, w;
            a.u = *reinterpret_cast<const uint4*>(xr + (int64_t)(tid + i * NT) * E);
            w.u = W_SMEM ? weights[tid + i * NT] : held[W_SMEM ? 0 : i];
#pragma unroll
            for (int e = 0; e < E; ++e) y[i][e] = to_f32<T>(a.e[e]) * k * rs * to_f32<T>(w.e[e]);
#pragma unroll
            for (int e = 0; e < E; e += 2) top = max_abs(top, y[i][e], y[i][e + 1]);
          }
        }
        top_bits = block_max<NT>(abs_bits(top), red_max[2]);
        r = row_scale(top_bits, 1.f, tid == 0 ? p.scale + row : nullptr);
        __syncthreads();                          // the third buffers may be written again
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) y[i][e] *= r.pre;
    }
    int8_t* qr = p.q + row * p.n_cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = tid + i * NT;
      if (c < nvec) {
        uint32_t word[E / 4];
#pragma unroll
        for (int g = 0; g < E / 4; ++g) {
          const float* v = &y[i][4 * g];
          word[g] = __byte_perm(__byte_perm(quantise<TIES>(v[0], r), quantise<TIES>(v[1], r), 0x0040),
                                __byte_perm(quantise<TIES>(v[2], r), quantise<TIES>(v[3], r), 0x0040), 0x5410);
          if (r.dead) word[g] = 0;
        }
        if (E == 8) *reinterpret_cast<uint2*>(qr + (int64_t)c * E) = make_uint2(word[0], word[E / 4 - 1]);
        else *reinterpret_cast<uint32_t*>(qr + (int64_t)c * E) = word[0];
      }
    }
  }
}

// any width, alignment and stride: one element per thread and step, the row read again per phase
template <typename T, int SRC>
__global__ void __launch_bounds__(256) quantise_any_kernel(const Params p) {
  chain_release();
  chain_wait();
  __shared__ float red_sum[8];
  __shared__ uint32_t red_max[8];
  const int64_t row = blockIdx.x;
  T* xr = (T*)p.x + row * p.x_stride;
  float ss = 0.f, rs = 0.f, k = 1.f;
  if (SRC == SRC_NORM) {
    for (int c = threadIdx.x; c < p.n_cols; c += 256) {
      float v = to_f32<T>(xr[c]);
      if (p.delta) {
        const T s = from_f32<T>(v + to_f32<T>(((const T*)p.delta)[row * p.d_stride + c]));
        xr[c] = s;                                  // read back by this thread only
        v = to_f32<T>(s);
      }
      ss = fmaf(v, v, ss);
    }
    ss = block_sum<256>(ss, red_sum);
    if (!(ss < INFINITY)) {                           // the squares of smaller values
      k = kShrink;
      ss = 0.f;
      for (int c = threadIdx.x; c < p.n_cols; c += 256) ss = fmaf(to_f32<T>(xr[c]) * k, to_f32<T>(xr[c]) * k, ss);
      __syncthreads();
      ss = block_sum<256>(ss, red_sum);
    }
    rs = rsqrtf(ss / (float)p.n_cols + p.eps * k * k);
  }
  auto value = [&](int c) {
    const float v = to_f32<T>(xr[c]);
    if (SRC == SRC_NORM) return v * k * rs * to_f32<T>(((const T*)p.weight)[c]);
    if (SRC == SRC_GATE) {
      const float u[2] = {to_f32<T>(xr[p.n_cols + c]), 0.f}, g[2] = {v, 0.f};
      float y[2], far = 0.f;
      gated<2>(g, u, p.act, y, far);
      return far > far_limit(p.act) ? act_far(v, p.act) * u[0] : y[0];
    }
    return v;
  };
  uint32_t top = 0;
  for (int c = threadIdx.x; c < p.n_cols; c += 256) top = max(top, abs_bits(value(c)));
  top = block_max<256>(top, red_max);
  const RowScale r = row_scale(top, 1.f, threadIdx.x == 0 ? p.scale + row : nullptr);
  int8_t* qr = p.q + row * p.n_cols;
  for (int c = threadIdx.x; c < p.n_cols; c += 256) qr[c] = r.dead ? (int8_t)0 : (int8_t)(quantise<kTies<T, SRC>>(value(c) * r.pre, r) & 0xFFu);
}

template <typename T, int SRC, int NT, int VPT>
static int launch_row(const Params& p, cudaStream_t st) {
  constexpr size_t smem = (size_t)(SRC == SRC_ROWS ? 1 : (SRC == SRC_NORM && VPT > 2 ? 3 : 2)) * VPT * NT * 16;
  auto kern = quantise_kernel<T, SRC, NT, VPT>;
  static std::atomic<uint64_t> allowed{0};
  ACACHE_CUDA_CHECK(allow_smem((const void*)kern, smem, allowed));
  const int64_t most = (int64_t)kNumSMs * resident(NT, VPT);
  ACACHE_CUDA_CHECK(launch_chained(kern, dim3((unsigned)(p.n_rows < most ? p.n_rows : most)), dim3(NT), smem, st, p));
  ACACHE_LAUNCH_CHECK();
  return ACACHE_OK;
}

template <typename T, int SRC>
static int launch(const Params& p, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const bool vec = p.n_cols % E == 0 && p.x_stride % E == 0 && aligned16(p.x) && (!p.delta || (p.d_stride % E == 0 && aligned16(p.delta))) &&
                   (!p.weight || aligned16(p.weight)) && (reinterpret_cast<uintptr_t>(p.q) & 7) == 0;
  const int nvec = p.n_cols / E;
  // the row in registers: at most 8 vectors of 8 values a thread; wider rows are read again instead
  if (!vec || nvec > 4096) {
    ACACHE_CUDA_CHECK(launch_chained(quantise_any_kernel<T, SRC>, dim3(p.n_rows), dim3(256), 0, st, p));
    ACACHE_LAUNCH_CHECK();
    return ACACHE_OK;
  }
  if (nvec <= 128) return launch_row<T, SRC, 128, 1>(p, st);
  if (nvec <= 256) return launch_row<T, SRC, 256, 1>(p, st);
  if (nvec <= 512) return launch_row<T, SRC, 256, 2>(p, st);
  if (nvec <= 1024) return launch_row<T, SRC, 256, 4>(p, st);
  if (nvec <= 2048) return launch_row<T, SRC, 512, 4>(p, st);
  return launch_row<T, SRC, 512, 8>(p, st);
}

}  // namespace quant
}  // namespace acache

using namespace acache;

extern "C" int acache_quantize_rows(const void* x, int64_t x_stride, int n_rows, int n_cols, int dtype, int8_t* q,
                                    float* scale, void* stream) {
  if (!dtype_ok(dtype) || n_rows < 0 || n_cols <= 0) return ACACHE_EINVAL;
  if (n_rows == 0) return ACACHE_OK;
  if (!x || !q || !scale) return ACACHE_EINVAL;
  const quant::Params p{x, x_stride, nullptr, 0, nullptr, 0.f, 0, q, scale, n_rows, n_cols};
  ACACHE_DISPATCH_DTYPE(dtype, T, return (quant::launch<T, quant::SRC_ROWS>(p, (cudaStream_t)stream)));
  return ACACHE_EINVAL;
}

extern "C" int acache_rmsnorm_int8(void* x, int64_t x_stride, const void* delta, int64_t d_stride, const void* weight,
                                   int n_rows, int n_cols, float eps, int dtype, int8_t* q, float* scale, void* stream) {
  if (!dtype_ok(dtype) || n_rows < 0 || n_cols <= 0) return ACACHE_EINVAL;
  if (n_rows == 0) return ACACHE_OK;
  if (!x || !weight || !q || !scale) return ACACHE_EINVAL;
  const quant::Params p{x, x_stride, delta, d_stride, weight, eps, 0, q, scale, n_rows, n_cols};
  ACACHE_DISPATCH_DTYPE(dtype, T, return (quant::launch<T, quant::SRC_NORM>(p, (cudaStream_t)stream)));
  return ACACHE_EINVAL;
}

extern "C" int acache_act_mul_halves_int8(const void* x, int64_t x_stride, int n_rows, int ffn, int act, int dtype,
                                          int8_t* q, float* scale, void* stream) {
  if (!dtype_ok(dtype) || n_rows < 0 || ffn <= 0 || act < 0 || act > 2) return ACACHE_EINVAL;
  if (n_rows == 0) return ACACHE_OK;
  if (!x || !q || !scale) return ACACHE_EINVAL;
  const quant::Params p{x, x_stride, nullptr, 0, nullptr, 0.f, act, q, scale, n_rows, ffn};
  ACACHE_DISPATCH_DTYPE(dtype, T, return (quant::launch<T, quant::SRC_GATE>(p, (cudaStream_t)stream)));
  return ACACHE_EINVAL;
}
