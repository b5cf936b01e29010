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
// A CTA serves TOKENS tokens: it fills a shared table of their sines and cosines (one pair per thread and
// step, shared by all heads) and then streams the rows through 16-byte vectors.  Bound by HBM.
#include "common.cuh"

namespace acache {
namespace rope {

struct Params {
  const void* q; int64_t q_stride; const void* k; int64_t k_stride; const void* v; int64_t v_stride;
  int n_tokens, n_heads, n_kv_heads, head_dim, rotary; const int64_t* positions; const double* inv_freq; float factor;
  void* out_q; int64_t oq_stride; void* out_k; void* out_v; const int32_t* slots; int64_t num_slots; int32_t* err_flag;
};

constexpr int NT = 256;

__device__ __forceinline__ void sincos_of(double angle, float* s, float* c) {
  // 2 pi in two doubles: the reduced angle is right to 32 bits for every angle below 2^31 turns
  const double turns = rint(angle * 0.15915494309189535);
  double r = fma(turns, -6.283185307179586, angle);
  r = fma(turns, -2.4492935982947064e-16, r);
  sincosf((float)r, s, c);
}

// VEC: 16-byte vectors (aligned rows, rotary / 2 a multiple of the vector in the half layout); else single elements
template <typename T, bool INTERLEAVED, bool VEC>
__global__ void __launch_bounds__(NT) rope_append_kernel(const Params p, int tokens_per_cta) {
  constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;
  extern __shared__ float2 table[];            // [tokens_per_cta][rotary / 2] (cos, sin)
  chain_release();
  chain_wait();
  const int half = p.rotary / 2, D = p.head_dim;
  const int t0 = blockIdx.x * tokens_per_cta, nt = min(tokens_per_cta, p.n_tokens - t0);
  for (int i = threadIdx.x; i < nt * half; i += NT) {
    float s, c;
    sincos_of((double)p.positions[t0 + i / half] * p.inv_freq[i % half], &s, &c);
    table[i] = make_float2(c * p.factor, s * p.factor);
  }
  __syncthreads();
  // units of one vector (half layout inside the rotary part: the vector and its partner half a rotary part on)
  const int rot_units = INTERLEAVED ? p.rotary / (VEC ? E : 2) : half / E;
  const int tail_units = (D - p.rotary) / E;
  const int per_head = rot_units + tail_units;
  const int v_units = D / E;
  const int n_rot_heads = p.n_heads + p.n_kv_heads;
  const int per_token = n_rot_heads * per_head + (p.v ? p.n_kv_heads * v_units : 0);
  for (int u = threadIdx.x; u < nt * per_token; u += NT) {
    const int t = u / per_token;
    int w = u % per_token;
    const int64_t token = t0 + t;
    const T* src;
    T* dst;
    int64_t slot = token;
    const bool is_v = w >= n_rot_heads * per_head;
    int head, at;
    if (is_v) {
      w -= n_rot_heads * per_head;
      head = w / v_units;
      at = w % v_units;
    } else {
      head = w / per_head;
      at = w % per_head;
    }
    const bool is_q = !is_v && head < p.n_heads;
    if (!is_q && p.slots) {
      slot = p.slots[token];
      if (slot < 0 || slot >= p.num_slots) {
        if (slot != -1 && p.err_flag) atomicExch(p.err_flag, 1);
        continue;
      }
    }
    if (is_q) {
      src = (const T*)p.q + token * p.q_stride + (int64_t)head * D;
      dst = (T*)p.out_q + token * p.oq_stride + (int64_t)head * D;
    } else {
      const int h = is_v ? head : head - p.n_heads;
      src = (is_v ? (const T*)p.v + token * p.v_stride : (const T*)p.k + token * p.k_stride) + (int64_t)h * D;
      dst = (T*)(is_v ? p.out_v : p.out_k) + (slot * p.n_kv_heads + h) * D;
    }
    const float2* tab = table + t * half;
    if (is_v || at >= rot_units) {               // copied
      const int c = is_v ? at * E : p.rotary + (at - rot_units) * E;
      if (VEC) *reinterpret_cast<uint4*>(dst + c) = ld_global_nc(src + c);
      else dst[c] = src[c];
    } else if (!INTERLEAVED) {
      const int c = at * E;
      if (VEC) {
        Vec16<T> a, b, lo, hi;
        a.u = ld_global_nc(src + c);
        b.u = ld_global_nc(src + c + half);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 cs = tab[c + e];
          const float x = to_f32<T>(a.e[e]), y = to_f32<T>(b.e[e]);
          lo.e[e] = from_f32<T>(x * cs.x - y * cs.y);
          hi.e[e] = from_f32<T>(y * cs.x + x * cs.y);
        }
        *reinterpret_cast<uint4*>(dst + c) = lo.u;
        *reinterpret_cast<uint4*>(dst + c + half) = hi.u;
      } else {
        const float2 cs = tab[c];
        const float x = to_f32<T>(src[c]), y = to_f32<T>(src[c + half]);
        dst[c] = from_f32<T>(x * cs.x - y * cs.y);
        dst[c + half] = from_f32<T>(y * cs.x + x * cs.y);
      }
    } else if (VEC) {
      const int c = at * E;
      Vec16<T> a, o;
      a.u = ld_global_nc(src + c);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 cs = tab[(c + e) / 2];
        const float x = to_f32<T>(a.e[e]), y = to_f32<T>(a.e[(e + 1) % E]);
        o.e[e] = from_f32<T>(x * cs.x - y * cs.y);
        o.e[(e + 1) % E] = from_f32<T>(y * cs.x + x * cs.y);
      }
      *reinterpret_cast<uint4*>(dst + c) = o.u;
    } else {
      const float2 cs = tab[at];
      const float x = to_f32<T>(src[2 * at]), y = to_f32<T>(src[2 * at + 1]);
      dst[2 * at] = from_f32<T>(x * cs.x - y * cs.y);
      dst[2 * at + 1] = from_f32<T>(y * cs.x + x * cs.y);
    }
  }
}

template <typename T>
static int launch(const Params& p, bool interleaved, cudaStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool vec = p.head_dim % E == 0 && p.rotary % E == 0 && (interleaved || (p.rotary / 2) % E == 0) &&
                   p.q_stride % E == 0 && p.k_stride % E == 0 && p.oq_stride % E == 0 && aligned16(p.q) && aligned16(p.k) &&
                   aligned16(p.out_q) && aligned16(p.out_k) &&
                   (!p.v || (p.v_stride % E == 0 && aligned16(p.v) && aligned16(p.out_v)));
  const int tokens = 1;
  const dim3 grid((p.n_tokens + tokens - 1) / tokens);
  const size_t smem = (size_t)tokens * (p.rotary / 2) * sizeof(float2);
#define GO(I, V) ACACHE_CUDA_CHECK(launch_chained(rope_append_kernel<T, I, V>, grid, dim3(NT), smem, st, p, tokens))
  if (interleaved) {
    if (vec) GO(true, true);
    else GO(true, false);
  } else {
    if (vec) GO(false, true);
    else GO(false, false);
  }
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
  ACACHE_DISPATCH_DTYPE(dtype, T, return (rope::launch<T>(p, interleaved != 0, (cudaStream_t)stream)));
  return ACACHE_EINVAL;
}
