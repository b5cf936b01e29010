// Shared-prefix attention is computed in parts (a range of keys for a set of rows) that are merged at the
// end: the description of a segment (the shared prefix, or the requests' own keys) that the kernels of
// attention_shared.cu and attention_shared_wide.cu have in common.
#pragma once
#include "common.cuh"

namespace acache {
namespace parts {

// Keys of a segment and where its partial results go.  A partial result of row (query, head) is O / l
// (fp32) and lse = log2(sum of 2^score) over the part's keys, -inf (and O not written) when it has none.
struct Seg {
  const int32_t* cu_q;      // NULL: one request over all total_q query rows
  const int32_t* cu_k;      // NULL: one request over all n_slots entries
  const int32_t* slots; int n_slots; int total_q;
  int splits;               // key ranges per request
  const int32_t* keep; int64_t keep_stride;   // bits of request r: keep[r * keep_stride ...] (NULL: every key)
  const int32_t* req_cu; int n_req;           // which request a query row belongs to, for keep
  float* o; float* lse; int64_t n_rows; int first_part;   // [part][n_rows = total_q * n_heads][head_dim]
  // 256-row tiles only: ctas > 0 shares units x unit_tiles key tiles out evenly over that many CTAs (units: KV heads x 256-row
  // blocks of the one request); `splits` is then the number of parts that a unit may be in
  int ctas, units, unit_tiles;
};

struct Args {
  const void* q; int64_t q_stride; const void* k_cache; const void* v_cache; int64_t num_slots; int n_heads, n_kv_heads,
      head_dim, dtype; float scale_log2; int32_t* err_flag; cudaStream_t st;
};

#ifdef __CUDACC__
// Softmax weights are rounded to the tensors' type T before their product with V, as the tensor cores take them (their sum is not
// rounded): half a step of every weight, 1.4 (bf16) to 1.3 (fp16) times the error that the rounding of the result alone makes.
// They are 2^(score - reference), and the reference follows the row's largest score once that is kLag above it.  fp16 numbers
// are subnormal below 2^-14, so there the reference is kept kHead below the largest score when it is set: weights reach up to
// 2^15 and have full precision down to 2^-21 of the largest (2^-32 of it, absolutely, below).
template <typename T> constexpr float kHead = 0.f;
template <> inline constexpr float kHead<__half> = 7.f;
template <typename T> constexpr float kLag = 8.f + kHead<T>;

struct Range { int q0, n_q, k0, n_k; };

// rows and keys of request b, kept inside the arrays whatever the offsets say
__device__ __forceinline__ Range request_range(const Seg& s, int b) {
  Range r;
  r.q0 = s.cu_q ? min(max(s.cu_q[b], 0), s.total_q) : 0;
  r.n_q = (s.cu_q ? min(max(s.cu_q[b + 1], r.q0), s.total_q) : s.total_q) - r.q0;
  r.k0 = s.cu_k ? min(max(s.cu_k[b], 0), s.n_slots) : 0;
  r.n_k = (s.cu_k ? min(max(s.cu_k[b + 1], r.k0), s.n_slots) : s.n_slots) - r.k0;
  return r;
}
// narrows r to key range `split` (whole tiles of `tile` keys) and returns its first key's index in the request
__device__ __forceinline__ int split_range(const Seg& s, int split, int tile, Range& r) {
  const int tiles = (r.n_k + tile - 1) / tile, per = (tiles + s.splits - 1) / s.splits;
  const int begin = min(split * per * tile, r.n_k), end = min((split + 1) * per * tile, r.n_k);
  r.k0 += begin;
  r.n_k = end - begin;
  return begin;
}
// the request that query row `q` belongs to
__device__ __forceinline__ int request_of(const int32_t* cu, int n_req, int q) {
  int lo = 0, hi = n_req;            // cu[lo] <= q < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= q) lo = mid;
    else hi = mid;
  }
  return lo;
}
#endif

}  // namespace parts

int attention_wide_parts(const parts::Args& a, const parts::Seg& seg, int n_requests, int max_q);

}  // namespace acache
