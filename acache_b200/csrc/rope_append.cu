// Rotary positions computed from frequencies, and the rotated keys and the values appended to the
// paged cache:
//
//   angle_i = position * inv_freq_i,   (a, b) -> (a c - b s, b c + a s),   c, s = factor * (cos, sin)(angle_i)
//
// for the rotary / 2 pairs of every head: (x_i, x_{i + rotary/2}) in the half layout, (x_2i, x_2i+1) in the
// interleaved one.  The rest of the head is copied.  The angle is formed and reduced to [-pi, pi] in
// 64 bits (in 32 bits position 10^6 has an angle error of 0.03), sine and cosine of the reduced angle and
// the rotation are in 32 bits, the result is rounded to the tensors' type once.
//
// A CTA serves four tokens of a few rows (a row is one head of q, k or v): each lane loads its vectors of the four, the
// CTA fills a shared table of the tokens' sines and cosines (again in every CTA: cheaper than to share it more widely),
// and a lane gets the other halves of its pairs from a neighbour by shuffles, so every vector is loaded and stored
// once and a row's addresses are formed once.  Bound by HBM at size: 16411 rows of 28 + 2 x 4 heads of 128 (293 MB) in
// 52 us (5.7 TB/s), 2304 rows 11.4 us, 512 rows of 32 + 2 x 32 heads (25 MB) 7.7 us.  (A flat loop over vectors that finds
// the row by division took 78 and 9 us: as many integer instructions as the rest.)
#include "common.cuh"

namespace acache {
namespace rope {

struct Params {
  const void* q; int64_t q_stride; const void* k; int64_t k_stride; const void* v; int64_t v_stride;
  int n_tokens, n_heads, n_kv_heads, head_dim, rotary; const int64_t* positions; const double* inv_freq; float factor;
  void* out_q; int64_t oq_stride; void* out_k; void* out_v; const int32_t* slots; int64_t num_slots; int32_t* err_flag;
};

constexpr int NT = 128, kTokens = 4;      // threads and tokens of a CTA

__device__ __forceinline__ void sincos_of(double angle, float* s, float* c) {
  // 2 pi in two doubles: the reduced angle is right to 32 bits for every angle below 2^31 turns
  const double turns = rint(angle * 0.15915494309189535);
  double r = fma(turns, -6.283185307179586, angle);
  r = fma(turns, -2.4492935982947064e-16, r);
  sincosf((float)r, s, c);
}

// sines and cosines of tokens t0 .. t0 + nt - 1, and the slots their k and v go to (-1: nowhere).  P: pairs of a
// vector; a token's table is laid out by couples of pairs, [P / 2][vectors][2], so that neighbouring lanes read
// neighbouring 16 bytes (in pair order a vector's 64 bytes put eight lanes on the same banks in fours: a third
// more time); P = 1: in pair order.
template <int P>
__device__ __forceinline__ void fill_table(const Params& p, int t0, int nt, float2* table, int64_t* slot) {
  const int half = p.rotary / 2, vecs = half / P;
  for (int i = threadIdx.x; i < nt * half; i += NT) {
    const int t = i / half, pair = i - t * half;
    float s, c;
    sincos_of((double)p.positions[t0 + t] * p.inv_freq[pair], &s, &c);
    const int at = P == 1 ? pair : ((pair % P / 2) * vecs + pair / P) * 2 + (pair & 1);
    table[t * half + at] = make_float2(c * p.factor, s * p.factor);
  }
  if (threadIdx.x >= NT - kTokens && threadIdx.x - (NT - kTokens) < nt) {
    const int t = threadIdx.x - (NT - kTokens);
    int64_t v = p.slots ? (int64_t)p.slots[t0 + t] : t0 + t;
    if (p.slots && (v < -1 || v >= p.num_slots)) {
      if (p.err_flag) atomicExch(p.err_flag, 1);
      v = -1;
    }
    slot[t] = v;
  }
}

// row w of a token: q heads, then k heads, then v heads
template <typename T>
__device__ __forceinline__ const T* source_of(const Params& p, int64_t token, int w) {
  if (w < p.n_heads) return (const T*)p.q + token * p.q_stride + (int64_t)w * p.head_dim;
  w -= p.n_heads;
  if (w < p.n_kv_heads) return (const T*)p.k + token * p.k_stride + (int64_t)w * p.head_dim;
  return (const T*)p.v + token * p.v_stride + (int64_t)(w - p.n_kv_heads) * p.head_dim;
}
template <typename T>
__device__ __forceinline__ T* target_of(const Params& p, int64_t token, int w, int64_t slot) {
  if (w < p.n_heads) return (T*)p.out_q + token * p.oq_stride + (int64_t)w * p.head_dim;
  if (slot < 0) return nullptr;
  w -= p.n_heads;
  if (w < p.n_kv_heads) return (T*)p.out_k + (slot * p.n_kv_heads + w) * p.head_dim;
  return (T*)p.out_v + (slot * p.n_kv_heads + w - p.n_kv_heads) * p.head_dim;
}

// A CTA serves U tokens of NT / W rows; W lanes per row (the power of two that holds head_dim / E vectors), lane c
// holds elements c E .. c E + E - 1 of its row for each of the tokens.
template <typename T, bool INTERLEAVED, int W, int U>
__global__ void __launch_bounds__(NT, 8) rope_append_kernel(const Params p) {
  constexpr int E = 16 / (int)sizeof(T), GROUPS = NT / W, P = INTERLEAVED ? E / 2 : E;     // P: pairs of a vector
  extern __shared__ __align__(16) float2 table[];      // [U][rotary / 2] (cos, sin)
  __shared__ int64_t slot[kTokens];
  chain_release();
  chain_wait();
  const int half = p.rotary / 2, D = p.head_dim;
  const int t0 = blockIdx.x * U, nt = min(U, p.n_tokens - t0);
  const int c = threadIdx.x % W, row = blockIdx.y * GROUPS + threadIdx.x / W, lane = threadIdx.x & 31;
  const int rows = p.n_heads + p.n_kv_heads * (p.v ? 2 : 1);
  const bool live = row < rows && c * E < D, in_rot = c * E < p.rotary;
  const bool is_q = row < p.n_heads, is_v = row >= p.n_heads + p.n_kv_heads;
  // half layout: vector c of the first half pairs with vector c + half / E
  const bool first = INTERLEAVED || c * E < half;
  const int partner = INTERLEAVED || !in_rot ? lane : (first ? lane + half / E : lane - half / E);
  const int vecs = half / P, my_vec = INTERLEAVED || first ? c : c - half / E;      // table column of this lane
  const int h = is_q ? row : row - p.n_heads - (is_v ? p.n_kv_heads : 0);
  const int64_t stride = is_q ? p.q_stride : (is_v ? p.v_stride : p.k_stride);
  const T* src = (const T*)(is_q ? p.q : (is_v ? p.v : p.k)) + t0 * stride + (int64_t)h * D + c * E;
  uint4 x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) x[u] = live && u < nt ? ld_global_nc(src + u * stride) : make_uint4(0, 0, 0, 0);
  fill_table<P>(p, t0, nt, table, slot);
  __syncthreads();
  T* dst = is_q ? (T*)p.out_q + t0 * p.oq_stride + (int64_t)h * D + c * E : (T*)(is_v ? p.out_v : p.out_k) + (int64_t)h * D + c * E;
  const int64_t step = is_q ? p.oq_stride : (int64_t)p.n_kv_heads * D;       // per token, or per slot
  const bool rotate = !is_v && in_rot;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (u >= nt) break;                        // the same for the whole CTA
    Vec16<T> a, o;
    a.u = x[u];
    float2 cs[P];
    if (rotate) {
#pragma unroll
      for (int e = 0; e < P; e += 2) {
        const float4 v = *reinterpret_cast<const float4*>(table + u * half + ((e / 2) * vecs + my_vec) * 2);
        cs[e] = make_float2(v.x, v.y);
        cs[e + 1] = make_float2(v.z, v.w);
      }
    }
    if (INTERLEAVED) {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float lo = to_f32<T>(a.e[e]), hi = to_f32<T>(a.e[e + 1]);
        o.e[e] = from_f32<T>(lo * cs[e / 2].x - hi * cs[e / 2].y);
        o.e[e + 1] = from_f32<T>(hi * cs[e / 2].x + lo * cs[e / 2].y);
      }
    } else {
      Vec16<T> b;
      b.u.x = __shfl_sync(0xFFFFFFFFu, x[u].x, partner);
      b.u.y = __shfl_sync(0xFFFFFFFFu, x[u].y, partner);
      b.u.z = __shfl_sync(0xFFFFFFFFu, x[u].z, partner);
      b.u.w = __shfl_sync(0xFFFFFFFFu, x[u].w, partner);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float mine = to_f32<T>(a.e[e]), other = to_f32<T>(b.e[e]);
        o.e[e] = from_f32<T>(first ? mine * cs[e % P].x - other * cs[e % P].y : mine * cs[e % P].x + other * cs[e % P].y);
      }
    }
    const int64_t at = is_q ? u : slot[u];
    if (live && at >= 0) *reinterpret_cast<uint4*>(dst + at * step) = rotate ? o.u : a.u;
  }
}

// any head size, alignment and stride: one pair or one element per thread and step
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(NT) rope_append_any_kernel(const Params p) {
  extern __shared__ __align__(16) float2 table[];
  __shared__ int64_t slot[kTokens];
  chain_release();
  chain_wait();
  const int half = p.rotary / 2, D = p.head_dim, token = blockIdx.x;
  fill_table<1>(p, token, 1, table, slot);
  __syncthreads();
  const int rows = p.n_heads + p.n_kv_heads * (p.v ? 2 : 1), units = D - half;      // per row: pairs, then single elements
  for (int i = threadIdx.x; i < rows * units; i += NT) {
    const int w = i / units, u = i % units;
    const T* src = source_of<T>(p, token, w);
    T* dst = target_of<T>(p, token, w, slot[0]);
    if (!dst) continue;
    if (u >= half) {
      dst[u + half] = src[u + half];
      continue;
    }
    const int lo = INTERLEAVED ? 2 * u : u, hi = INTERLEAVED ? 2 * u + 1 : u + half;
    if (w < p.n_heads + p.n_kv_heads) {
      const float2 cs = table[u];
      const float x = to_f32<T>(src[lo]), y = to_f32<T>(src[hi]);
      dst[lo] = from_f32<T>(x * cs.x - y * cs.y);
      dst[hi] = from_f32<T>(y * cs.x + x * cs.y);
    } else {
      dst[lo] = src[lo];
      dst[hi] = src[hi];
    }
  }
}

template <typename T, bool INTERLEAVED>
static int launch(const Params& p, cudaStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool vec = p.head_dim % E == 0 && p.head_dim <= 32 * E && p.rotary % (2 * E) == 0 && 
                   p.q_stride % E == 0 && p.k_stride % E == 0 && p.oq_stride % E == 0 && aligned16(p.q) && aligned16(p.k) &&
                   aligned16(p.out_q) && aligned16(p.out_k) &&
                   (!p.v || (p.v_stride % E == 0 && aligned16(p.v) && aligned16(p.out_v)));
  const size_t entry = (size_t)(p.rotary / 2) * sizeof(float2);
  if (!vec) {
    ACACHE_CUDA_CHECK(launch_chained(rope_append_any_kernel<T, INTERLEAVED>, dim3(p.n_tokens), dim3(NT), entry, st, p));
    ACACHE_LAUNCH_CHECK();
    return ACACHE_OK;
  }
  int w = 1;           // rotary a multiple of two vectors: both halves are whole vectors, table entries come in twos
  while (w * E < p.head_dim) w *= 2;
  if (w < 8) w = 8;
  const int rows = p.n_heads + p.n_kv_heads * (p.v ? 2 : 1), groups = NT / w;
  const dim3 grid((p.n_tokens + kTokens - 1) / kTokens, (rows + groups - 1) / groups);
#define GO(W) ACACHE_CUDA_CHECK(launch_chained(rope_append_kernel<T, INTERLEAVED, W, kTokens>, grid, dim3(NT), kTokens * entry, st, p))
  if (w == 8) GO(8);
  else if (w == 16) GO(16);
  else GO(32);
#undef GO
  ACACHE_LAUNCH_CHECK();
  return ACACHE_OK;
}

}  // namespace rope
}  // namespace acache

using namespace acache;

extern "C" int acache_rope_append(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                  int64_t v_stride, int n_tokens, int n_heads, int n_kv_heads, int head_dim, int dtype,
                                  const int64_t* positions, const double* inv_freq, int rotary_dim, int interleaved,
                                  float attention_factor, void* out_q, int64_t out_q_stride, void* out_k, void* out_v,
                                  const int32_t* slot_mapping, int64_t num_slots, int32_t* err_flag, void* stream) {
  if (!dtype_ok(dtype) || n_tokens < 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || rotary_dim < 0 ||
      rotary_dim > head_dim || rotary_dim % 2 != 0 || num_slots < 0)
    return ACACHE_EINVAL;
  if (n_tokens == 0) return ACACHE_OK;
  if (!q || !k || !positions || !out_q || !out_k || (rotary_dim > 0 && !inv_freq) || (v && !out_v) || (slot_mapping && !v))
    return ACACHE_EINVAL;
  if (head_dim > 1024) return ACACHE_ELIMIT;     // the table of sines and cosines lies in shared memory
  const rope::Params p{q, q_stride, k, k_stride, v, v_stride, n_tokens, n_heads, n_kv_heads, head_dim, rotary_dim, positions,
                       inv_freq, attention_factor, out_q, out_q_stride, out_k, out_v, slot_mapping, num_slots, err_flag};
  ACACHE_DISPATCH_DTYPE(dtype, T, return interleaved ? (rope::launch<T, true>(p, (cudaStream_t)stream)) : (rope::launch<T, false>(p, (cudaStream_t)stream)));
  return ACACHE_EINVAL;
}
