// Attention of a batch whose requests share one long prefix of the paged cache, the prefix read once for
// all of them:
//
//   o_r = sum_{j in prefix, kept by r's request} w_rj v_j + sum_{j in the request's own keys} w_rj v_j
//   w_rj = exp(scale q_r k_j) / (sum of the same over both key sets)
//
// The softmax sum splits over any partition of the keys, so the work is cut into parts (prefix parts over the
// rows of ALL requests, own parts over each request's rows), each part yields (O / l, log2 of its sum), and a
// row's parts are merged at the end:  o = sum_p 2^(lse_p - top) O_p / sum_p 2^(lse_p - top).
//
// A part whose rows fill the tensor cores' 128-row tiles goes to attention_shared_wide.cu
// (tcgen05, 256 rows share a staged K/V tile).  A part with few rows (single tokens, short blocks: bound by
// the bytes of K and V) goes to rows_kernel below.
//
// rows_kernel: a CTA = (KV head, key range, request, 16 or 32 virtual rows), a virtual row being a (query,
// head-of-the-GQA-group) pair; a warp = (16 rows, one of four key groups).  The groups split the keys in runs of 32
// and share nothing until the end: each gathers its own blocks of 16 keys through the slot map (16-byte cp.async into a
// ring of its own, two blocks ahead, the map looked up further ahead still), multiplies with m16n8k16 tensor-core
// instructions (fp32 accumulators), keeps its own running maximum, sum and O in registers, and the four are merged
// through shared memory.  128-row tcgen05 tiles would leave 3/4 or more of every product empty here.
//
// A key that a request drops still runs through the products with weight 0, and 0 times an infinity or a NaN in
// its V row is a NaN: the merge looks for NaN in prefix parts under a keep mask and, when it meets one,
// recomputes that row's prefix part key by key without the dropped keys.
#include "attention_parts.cuh"
#include "common.cuh"
#include "tcgen05.cuh"

namespace acache {
namespace shared_prefix {

using tc::cp_async16;
using tc::cp_async_commit;
using tc::cp_async_wait;
using tc::ex2;
using tc::pack2;
using tc::smem_u32;

constexpr int KB = 16;                // keys of a block
constexpr int NS = 3;                 // stages of a group's ring

// how the final result is formed from the prefix parts
struct Merge {
  void* out; int64_t o_stride; int n_parts;      // parts [0, n_parts) of the workspace belong to the prefix
  const int32_t* prefix_slots; int prefix_len;   // for the recomputation under a keep mask
};

template <typename T> __device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// byte offset of 16-byte chunk c of row r: rows of D elements, chunks xor-ed with the row so that eight rows'
// chunks at one position lie in different banks
template <int D> __device__ __forceinline__ uint32_t at(int r, int c) { return (uint32_t)(r * D * 2 + ((c ^ (r & 7)) << 4)); }

template <typename T, int N> __device__ __forceinline__ void load_vec(const T* p, float* o) {
  if constexpr (N == 4) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = to_f32<T>(e[i]);
  } else {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
    o[0] = to_f32<T>(e[0]);
    o[1] = to_f32<T>(e[1]);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

// a row's prefix result key by key, without the keys its request drops; lse: log2 of the row's prefix sum
template <typename T, int D>
__device__ __noinline__ void recompute_prefix(const parts::Args& a, const parts::Seg& s, const Merge& mg, int q_row, int head,
                                              float lse, float* o) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int kvh = head / (a.n_heads / a.n_kv_heads);
  const uint32_t* bits = reinterpret_cast<const uint32_t*>(s.keep) + (int64_t)parts::request_of(s.req_cu, s.n_req, q_row) * s.keep_stride;
  float q[E];
  load_vec<T, E>((const T*)a.q + (int64_t)q_row * a.q_stride + (int64_t)head * D + lane * E, q);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int j = 0; j < mg.prefix_len; ++j) {
    const int32_t slot = mg.prefix_slots[j];
    if (slot < 0 || slot >= a.num_slots || !((bits[j >> 5] >> (j & 31)) & 1u)) continue;
    const int64_t off = ((int64_t)slot * a.n_kv_heads + kvh) * D + lane * E;
    float k[E], v[E], dot = 0.f;
    load_vec<T, E>((const T*)a.k_cache + off, k);
    load_vec<T, E>((const T*)a.v_cache + off, v);
#pragma unroll
    for (int e = 0; e < E; ++e) dot = fmaf(q[e], k[e], dot);
    const float w = ex2(warp_sum(dot) * a.scale_log2 - lse);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(w, v[e], o[e]);
  }
}

// one warp: parts [begin, end) of N rows added to (acc, m, l), acc = the sum of weights 2^(score - m) times V.
// The loads of the N rows, and of several parts, are in flight together.
template <int D, int N, int U>
__device__ __forceinline__ void merge_parts(const parts::Seg& s, int begin, int end, const int64_t (&row)[N], const bool (&live)[N],
                                            float (&acc)[N][D / 32], float (&m)[N], float (&l)[N]) {
  constexpr int E = D / 32;                          // U: parts whose loads are in flight together
  const int lane = threadIdx.x & 31;
  for (int base = begin; base < end; base += 32) {
    const int cnt = min(32, end - base);
    float w[N], v[U][N][E];
    // O of a part without keys was never written: it is loaded with the others and not used
    auto load = [&](int i) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const float* o = s.o + ((int64_t)(base + min(i + u, cnt - 1)) * s.n_rows + row[n]) * D + lane * E;
          if constexpr (E == 4) {
            const float4 x = *reinterpret_cast<const float4*>(o);
            v[u][n][0] = x.x; v[u][n][1] = x.y; v[u][n][2] = x.z; v[u][n][3] = x.w;
          } else {
            const float2 x = *reinterpret_cast<const float2*>(o);
            v[u][n][0] = x.x; v[u][n][1] = x.y;
          }
        }
    };
#pragma unroll
    for (int n = 0; n < N; ++n) w[n] = live[n] && lane < cnt ? s.lse[(int64_t)(base + lane) * s.n_rows + row[n]] : -INFINITY;
    load(0);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float top = fmaxf(m[n], warp_max(w[n]));
      // a side without keys has the sum 0; one with nothing but NaN scores has a NaN sum, which reaches the result
      const float f = m[n] == -INFINITY && l[n] == 0.f ? 0.f : ex2(m[n] - top);
      w[n] = w[n] == -INFINITY ? 0.f : ex2(w[n] - top);
      l[n] = l[n] * f + warp_sum(w[n]);
      m[n] = top;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[n][e] = f == 0.f ? 0.f : acc[n][e] * f;
    }
    for (int i = 0; i < cnt; i += U) {
      if (i > 0) load(i);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < N; ++n) {
          float wi = __shfl_sync(0xFFFFFFFFu, w[n], (i + u) & 31);
          if (i + u >= cnt) wi = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[n][e] = wi == 0.f ? acc[n][e] : fmaf(wi, v[u][n][e], acc[n][e]);
        }
    }
  }
}

// the rare way of a row whose merged value holds a NaN under a keep mask: the prefix side again, key by key
// where it is NaN
template <typename T, int D>
__device__ __noinline__ void finish_again(const parts::Args& a, const parts::Seg& s, const parts::Seg& prefix, const Merge& mg,
                                          int own_begin, int own_end, int q_row, int head, const float* own_acc, float own_m,
                                          float own_l, float* v) {
  constexpr int E = D / 32;
  const int64_t row[1] = {(int64_t)q_row * a.n_heads + head};
  const bool live[1] = {true};
  float own[1][E], m[1] = {own_m}, l[1] = {own_l}, pre[1][E], pm[1] = {-INFINITY}, pl[1] = {0.f};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    own[0][e] = own_acc[e];
    pre[0][e] = 0.f;
  }
  merge_parts<D, 1, 4>(s, own_begin, own_end, row, live, own, m, l);
  merge_parts<D, 1, 4>(s, 0, mg.n_parts, row, live, pre, pm, pl);
  if (pl[0] > 0.f) {
    float again[E];
    recompute_prefix<T, D>(a, prefix, mg, q_row, head, pm[0] + log2f(pl[0]), again);
#pragma unroll
    for (int e = 0; e < E; ++e) pre[0][e] = isnan(pre[0][e]) ? again[e] * pl[0] : pre[0][e];
  }
  const float top = fmaxf(m[0], pm[0]);
  const float fo = m[0] == -INFINITY && l[0] == 0.f ? 0.f : ex2(m[0] - top);
  const float fp = pm[0] == -INFINITY && pl[0] == 0.f ? 0.f : ex2(pm[0] - top);
  const float inv = 1.f / (l[0] * fo + pl[0] * fp);
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = ((fo == 0.f ? 0.f : own[0][e] * fo) + (fp == 0.f ? 0.f : pre[0][e] * fp)) * inv;
}

// one warp: the final values of N rows from (acc, m, l) of the keys that have no part in the workspace, the prefix
// parts and own parts [own_begin, own_end)
template <typename T, int D, int N, int U>
__device__ __forceinline__ void finish_rows(const parts::Args& a, const parts::Seg& s, const parts::Seg& prefix, const Merge& mg,
                                            int own_begin, int own_end, const int (&q_row)[N], const int (&head)[N],
                                            const bool (&live)[N], float (&acc)[N][D / 32], float (&m)[N], float (&l)[N]) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  int64_t row[N];
  float acc0[N][E], m0[N], l0[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    row[n] = (int64_t)q_row[n] * a.n_heads + head[n];
    m0[n] = m[n];
    l0[n] = l[n];
#pragma unroll
    for (int e = 0; e < E; ++e) acc0[n][e] = acc[n][e];
  }
  // the prefix's parts and the own ones follow each other in the workspace
  merge_parts<D, N, U>(s, mg.n_parts > 0 ? 0 : own_begin, mg.n_parts > 0 && own_end == own_begin ? mg.n_parts : own_end, row, live, acc, m, l);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!live[n]) continue;
    const float inv = l[n] == 0.f ? 0.f : 1.f / l[n];          // no key at all: zeros
    float v[E];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = acc[n][e] * inv;
      bad |= isnan(v[e]);
    }
    if (prefix.keep && mg.n_parts > 0 && __any_sync(0xFFFFFFFFu, bad))
      finish_again<T, D>(a, s, prefix, mg, own_begin, own_end, q_row[n], head[n], acc0[n], m0[n], l0[n], v);
    T* dst = (T*)mg.out + (int64_t)q_row[n] * mg.o_stride + (int64_t)head[n] * D + lane * E;
    if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    else *reinterpret_cast<uint32_t*>(dst) = pack2<T>(v[0], v[1]);
  }
}

// final: the segment is the requests' own keys in one range each and the CTA also merges the prefix parts (written by
// the kernel before it in the stream) and writes the output; else it leaves a part.  The wait for that kernel comes before
// the first read, although only the merge needs its parts: what older kernels of the stream wrote (q, slots, K, V) is only
// promised to a thread that has waited itself.  Waiting before the merge alone took 65 us instead of 69.6 for 16 x 32 rows, and
// 9.9 instead of 13.1 for four tokens over 600 keys, without that promise.
// NG: key groups of a CTA, 4 or 2; both keep 16 warps (two row tiles) on an SM, two groups make more and longer CTAs.
template <typename T, int D, int RT, int NG>
__global__ void __launch_bounds__(RT * NG * 32, 8 / NG) rows_kernel(const __grid_constant__ parts::Args a, const __grid_constant__ parts::Seg s,
                                                               const __grid_constant__ parts::Seg prefix,
                                                               const __grid_constant__ Merge mg, int final) {
  constexpr int NT = RT * NG * 32, ROWS = RT * 16, CH = D / 8, KS = D / 16, E = D / 32;
  constexpr int BLOCK = KB * D * 2;             // bytes of K (or V) of a block
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* sQ = smem;                           // [ROWS][D]
  uint8_t* ring = smem + ROWS * D * 2;          // [NG][NS][K | V]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grp = warp % NG, rt = warp / NG;    // key group and row tile of the warp

  chain_release();
  chain_wait();
  const int g = a.n_heads / a.n_kv_heads, kvh = blockIdx.x, b = blockIdx.z;
  const int split = blockIdx.y % s.splits, m0 = blockIdx.y / s.splits * ROWS;
  parts::Range r = parts::request_range(s, b);
  const int first_key = parts::split_range(s, split, 2 * KB * NG, r);
  const int vrows = r.n_q * g;
  if (m0 >= vrows) return;
  const int64_t kv_row = (int64_t)a.n_kv_heads * D;

  // ---- the keys of this group: runs of 32 (two blocks) grp, grp + NG, ...; one load looks a run's slots up,
  // three runs ahead of their use
  const int n_runs = (r.n_k + 2 * KB - 1) / (2 * KB), my_runs = n_runs > grp ? (n_runs - grp + NG - 1) / NG : 0;
  const int mine = 2 * my_runs;                 // blocks; the last may lie behind the end
  const uint32_t my_ring = smem_u32(ring) + grp * (NS * 2 * BLOCK);
  const T* kc = (const T*)a.k_cache + (int64_t)kvh * D;
  const T* vc = (const T*)a.v_cache + (int64_t)kvh * D;
  // lane l holds the slot of key l of a run; -1 = takes no part
  auto slots_of = [&](int u) -> int32_t {
    const int j = (grp + u * NG) * 2 * KB + lane;
    return u < my_runs && j < r.n_k ? s.slots[r.k0 + j] : -1;
  };
  int32_t run_now = slots_of(0), run_a = slots_of(1), run_b = slots_of(2);

  // ---- queries
  for (int i = tid; i < ROWS * CH; i += NT) {
    const int row = i / CH, c = i % CH, vr = m0 + row;
    const bool ok = vr < vrows;
    const T* src = (const T*)a.q + (int64_t)(r.q0 + (ok ? vr / g : 0)) * a.q_stride + (int64_t)(kvh * g + (ok ? vr % g : 0)) * D + c * 8;
    cp_async16(smem_u32(sQ) + at<D>(row, c), src, ok);
  }
  cp_async_commit();

  auto gather = [&](int i) -> uint32_t {        // block i into its stage (each row tile's warp a part of it); its dead keys
    const uint32_t kb = my_ring + (i % NS) * (2 * BLOCK), vb = kb + BLOCK;
    constexpr int RPI = 32 / CH, STEPS = KB / RPI / RT;     // rows per step of the warp
    const int c = lane % CH, half = (i & 1) * KB;
    int32_t slot = run_now;
    if (slot < -1 || slot >= a.num_slots) {
      if (a.err_flag) atomicExch(a.err_flag, 3);
      slot = -1;
    }
    const uint32_t dead = __ballot_sync(0xFFFFFFFFu, slot < 0) >> half;
    if (i < mine) {
#pragma unroll
      for (int it = 0; it < STEPS; ++it) {
        const int row = (rt * STEPS + it) * RPI + lane / CH;
        const int32_t sl = __shfl_sync(0xFFFFFFFFu, slot, half + row);
        const int64_t off = (int64_t)(sl < 0 ? 0 : sl) * kv_row + c * 8;
        cp_async16(kb + at<D>(row, c), kc + off, sl >= 0);
        cp_async16(vb + at<D>(row, c), vc + off, sl >= 0);
      }
    }
    cp_async_commit();
    if (i & 1) {
      run_now = run_a;
      run_a = run_b;
      run_b = slots_of(i / 2 + 3);
    }
    return dead;
  };
  // the warps that share a group's blocks
  auto group_sync = [&]() {
    if constexpr (RT == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "n"(RT * 32) : "memory");
  };
  // dead keys of the blocks in flight, oldest first
  uint32_t dead_q[NS];
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) dead_q[i] = gather(i);

  // which keys the rows of this thread keep: rows lane / 4 + 8 h of the tile
  const uint16_t* keep[2];
  if (s.keep) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int vr = min(m0 + rt * 16 + lane / 4 + 8 * h, vrows - 1);
      keep[h] = reinterpret_cast<const uint16_t*>(s.keep + (int64_t)parts::request_of(s.req_cu, s.n_req, r.q0 + vr / g) * s.keep_stride) + first_key / KB;
    }
  }
  cp_async_wait<NS - 1>();
  __syncthreads();                              // the queries have landed
  const uint32_t q_addr = smem_u32(sQ);

  float o[D / 8][4], m_ref[2] = {-INFINITY, -INFINITY}, l_sum[2] = {0.f, 0.f};
#pragma unroll
  for (int d = 0; d < D / 8; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[d][e] = 0.f;

  for (int i = 0; i < mine; ++i) {
    uint32_t kept[2];
    if (s.keep) {
#pragma unroll
      for (int h = 0; h < 2; ++h) kept[h] = keep[h][2 * (grp + (i / 2) * NG) + (i & 1)];
    }
    cp_async_wait<NS - 2>();
    group_sync();                               // block i is there, block i - 1 has been read by all
    dead_q[NS - 1] = gather(i + NS - 1);
    const uint32_t kb = my_ring + (i % NS) * (2 * BLOCK), vb = kb + BLOCK;

    // ---- scores: keys 0-7 and 8-15 of the block against the row tile
    float sc[2][4];
#pragma unroll
    for (int e = 0; e < 8; ++e) sc[e / 4][e % 4] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t kf[4], qf[4];
      ldsm4(kb + at<D>((lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1)), kf);
      ldsm4(q_addr + at<D>(rt * 16 + (lane & 15), 2 * ks + (lane >> 4)), qf);
      mma16816<T>(sc[0], qf, kf[0], kf[1]);
      mma16816<T>(sc[1], qf, kf[2], kf[3]);
    }
    // ---- keys that take no part, per row under a keep mask
    const uint32_t dead = dead_q[0] & 0xFFFFu;
    if (dead != 0u || s.keep) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t gone = (s.keep ? dead | ~kept[h] : dead) >> (2 * (lane & 3));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((gone >> ((e & 1) + 8 * (e >> 1))) & 1u) sc[e >> 1][2 * h + (e & 1)] = -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < NS - 1; ++k) dead_q[k] = dead_q[k + 1];
    // ---- online softmax; O is rescaled only when a row's maximum grows by more than 2^8 (attention_parts.cuh)
    constexpr float kHead = parts::kHead<T>, kLag = parts::kLag<T>;
    float mx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
      mx[h] = v * a.scale_log2;
    }
    if (__any_sync(0xFFFFFFFFu, mx[0] > m_ref[0] + kLag || mx[1] > m_ref[1] + kLag)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool grow = mx[h] > m_ref[h] + kLag;
        const float f = grow ? ex2(m_ref[h] - (mx[h] - kHead)) : 1.f;
        if (grow) m_ref[h] = mx[h] - kHead;
        l_sum[h] *= f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][2 * h] *= f;
          o[d][2 * h + 1] *= f;
        }
      }
    }
    uint32_t pa[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float mu = m_ref[h] == -INFINITY ? 0.f : m_ref[h];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float p0 = ex2(fmaf(sc[n][2 * h], a.scale_log2, -mu)), p1 = ex2(fmaf(sc[n][2 * h + 1], a.scale_log2, -mu));
        l_sum[h] += p0 + p1;
        pa[2 * n + h] = pack2<T>(p0, p1);
      }
    }
    // ---- O += P V
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      uint32_t vf[4];
      ldsm4t(vb + at<D>(lane & 15, 2 * d + (lane >> 4)), vf);
      mma16816<T>(o[2 * d], pa, vf[0], vf[1]);
      mma16816<T>(o[2 * d + 1], pa, vf[2], vf[3]);
    }
  }
  cp_async_wait<0>();

  // ---- the groups' results through shared memory (over the ring)
  __syncthreads();
  constexpr int LD = D + 8;                     // rows 8 banks apart: the float2 stores of a half warp do not collide
  float* sO = reinterpret_cast<float*>(ring);   // [NG][ROWS][LD], then the groups' maxima and sums [NG][ROWS]
  static_assert(NG * ROWS * (LD + 2) * 4 <= NG * NS * 2 * BLOCK, "the exchange lies over the ring");
  float* s_m = sO + NG * ROWS * LD;
  float* s_l = s_m + NG * ROWS;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = rt * 16 + lane / 4 + 8 * h;
    float l = l_sum[h];
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
    if ((lane & 3) == 0) {
      s_m[grp * ROWS + row] = m_ref[h];
      s_l[grp * ROWS + row] = l;
    }
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
      *reinterpret_cast<float2*>(sO + (grp * ROWS + row) * LD + d * 8 + 2 * (lane & 3)) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
  }
  __syncthreads();
  constexpr int N = 4;                          // rows that a warp finishes together
#pragma unroll 1
  for (int row0 = warp; row0 < ROWS; row0 += N * RT * NG) {
    float acc[N][E], m[N], l[N];
    int q_row[N], head[N];
    bool live[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int row = row0 + n * (RT * NG), vr = m0 + row;
      live[n] = row < ROWS && vr < vrows;
      q_row[n] = r.q0 + (live[n] ? vr / g : 0);
      head[n] = kvh * g + (live[n] ? vr % g : 0);
      m[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int w = 0; w < NG; ++w) m[n] = fmaxf(m[n], s_m[w * ROWS + (row & (ROWS - 1))]);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[n][e] = 0.f;
#pragma unroll
      for (int w = 0; w < NG; ++w) {
        const float mw = s_m[w * ROWS + (row & (ROWS - 1))], lw = s_l[w * ROWS + (row & (ROWS - 1))];
        const bool none = mw == -INFINITY && lw == 0.f;        // no key (only NaN scores leave a NaN sum)
        const float f = none ? 0.f : ex2(mw - m[n]);
        l[n] = fmaf(f, lw, l[n]);
        float x[E];
        const float* src = sO + (w * ROWS + (row & (ROWS - 1))) * LD + lane * E;
        if constexpr (E == 4) {
          const float4 t = *reinterpret_cast<const float4*>(src);
          x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
        } else {
          const float2 t = *reinterpret_cast<const float2*>(src);
          x[0] = t.x; x[1] = t.y;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) acc[n][e] = none ? acc[n][e] : fmaf(f, x[e], acc[n][e]);
      }
    }
    if (final) {
      finish_rows<T, D, N, RT == 1 ? 6 : 2>(a, s, prefix, mg, s.first_part, s.first_part, q_row, head, live, acc, m, l);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!live[n]) continue;
        const int64_t at_row = (int64_t)(s.first_part + split) * s.n_rows + (int64_t)q_row[n] * a.n_heads + head[n];
        const bool any_key = m[n] != -INFINITY || l[n] != 0.f;
        if (any_key) {
          const float inv = 1.f / l[n];
          float* dst = s.o + at_row * D + lane * E;
          if constexpr (E == 4) *reinterpret_cast<float4*>(dst) = make_float4(acc[n][0] * inv, acc[n][1] * inv, acc[n][2] * inv, acc[n][3] * inv);
          else *reinterpret_cast<float2*>(dst) = make_float2(acc[n][0] * inv, acc[n][1] * inv);
        }
        if (lane == 0) s.lse[at_row] = any_key ? m[n] + log2f(l[n]) : -INFINITY;
      }
    }
  }
}

// prefix parts and own parts into the output, one warp for four rows (28672 rows of two parts: 12 us, one row per warp 16)
template <typename T, int D>
__global__ void __launch_bounds__(128) merge_kernel(const __grid_constant__ parts::Args a, const __grid_constant__ parts::Seg own,
                                                    const __grid_constant__ parts::Seg prefix, const __grid_constant__ Merge mg, int n_req) {
  constexpr int N = 4;
  chain_release();
  chain_wait();
  const int64_t row0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * N;
  // rows behind the last sequence (or before the first) have no result
  const int first = own.cu_q[0], last = min(own.cu_q[n_req], own.total_q);
  int q_row[N], head[N];
  bool live[N];
  float acc[N][D / 32], m[N], l[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int64_t row = min(row0 + n, own.n_rows - 1);
    q_row[n] = (int)(row / a.n_heads);
    head[n] = (int)(row - (int64_t)q_row[n] * a.n_heads);
    live[n] = row0 + n < own.n_rows && q_row[n] >= first && q_row[n] < last;
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[n][e] = 0.f;
  }
  finish_rows<T, D, N, 2>(a, own, prefix, mg, own.first_part, own.first_part + own.splits, q_row, head, live, acc, m, l);
}

// 32 truth values to a word: bit j of word w of a row is key 32 w + j
__global__ void __launch_bounds__(256) pack_keep_kernel(const uint8_t* __restrict__ keep, int64_t stride, int n_keys, int words,
                                                        uint32_t* __restrict__ out, int64_t total) {
  chain_release();
  chain_wait();
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < total; w += (int64_t)gridDim.x * 8) {
    const int64_t row = w / words, key = (w % words) * 32 + (threadIdx.x & 31);
    const uint32_t bits = __ballot_sync(0xFFFFFFFFu, key < n_keys && keep[row * stride + key] != 0);
    if ((threadIdx.x & 31) == 0) out[w] = bits;
  }
}

// ------------------------------------------------------------------------------------------------ host
// How a segment runs.
struct Segment {
  bool wide;                          // 256-row tcgen05 tiles, else rows_kernel
  int groups;                         // NG of rows_kernel
  int64_t units;                      // CTAs in one key range each
};
static Segment segment(int64_t requests, int64_t rows_per_request, int n_kv_heads) {
  Segment c;
  // 256-row tiles from more than 96 rows (measured: 224 rows of 32 requests 190 us in all against 227 with 32-row CTAs, a
  // prefix part of 128 rows and 32 heads 25.5 us against 36.6, of 84 rows and 2 heads 12.1 us against 10.6)
  c.wide = rows_per_request > 96;
  const int64_t tile_rows = c.wide ? 256 : (rows_per_request <= 16 ? 16 : 32);
  c.units = n_kv_heads * requests * ((rows_per_request + tile_rows - 1) / tile_rows);
  // few CTAs: four key groups each, two CTAs per SM; many: two groups, four per SM, so that they run in fewer rounds
  c.groups = c.units <= 2 * kNumSMs ? 4 : 2;
  return c;
}

struct Plan {
  Segment pre, own;
  int prefix_splits, own_splits;
  int prefix_ctas;                    // > 0: the prefix's key tiles are shared out evenly over this many CTAs
  bool final;                         // the own segment's CTAs merge, no merge kernel
};

// Key ranges per request.  The prefix is cut so that its CTAs fill the SMs once, into ranges of at least two tiles.  The
// requests' own keys stay in one range, whose CTA also merges the prefix parts, unless few long ones leave most SMs idle:
// 64 keys take a four-group CTA about 0.65 us and the merge kernel 5 us.  Fitted while the own part still ran beside the prefix
// part (us; both came out 3-5 longer since, the choice was not fitted again): 16 requests x 32 rows x 32 heads over 800 keys, own
// keys merged in place 66 with two prefix ranges and 69 with one, with a merge kernel 73-81; 64 tokens over 32768 keys 67 with
// 18 ranges (72 when a merge kernel took 79 and 14 ranges 83).
static Plan make_plan(int total_q, int batch, int max_q, int max_k, int prefix_len, int n_heads, int n_kv_heads) {
  const int64_t g = n_heads / n_kv_heads;
  if (max_q > total_q) max_q = total_q;
  Plan p;
  p.pre = segment(1, total_q * g, n_kv_heads);
  p.own = segment(batch, max_q * g, n_kv_heads);
  auto splits = [](int64_t slots, int64_t units, int64_t keys, int64_t least) {
    if (units <= 0) return 1;
    int64_t s = slots / units;
    if (s > keys / least) s = keys / least;
    return (int)(s > 32 ? 32 : (s < 1 ? 1 : s));
  };
  p.prefix_splits = p.pre.wide ? splits(kNumSMs, p.pre.units, prefix_len, 256) : splits(kNumSMs, p.pre.units, prefix_len, 120);
  p.prefix_ctas = 0;
  if (p.pre.wide && prefix_len > 0) {
    // rounds of whole ranges against even shares (whose CTAs start and end a range twice): 2.4 us a 128-key tile, 8 us a range,
    // 0.3 us for every part that a row's merge reads
    const int64_t tiles = (prefix_len + 127) / 128, per = (tiles + p.prefix_splits - 1) / p.prefix_splits;
    const double ranges = (double)((p.pre.units * p.prefix_splits + kNumSMs - 1) / kNumSMs) * (per * 2.4 + 8.0) + 0.3 * p.prefix_splits;
    const int64_t ctas = p.pre.units * tiles < kNumSMs ? p.pre.units * tiles : kNumSMs;
    const double shares = (double)(p.pre.units * tiles) / ctas * 2.4 + 8.0 * (p.pre.units > ctas ? 1 + (p.pre.units + ctas - 1) / ctas : 2) +
                          0.3 * ((ctas + p.pre.units - 1) / p.pre.units + 1);
    if (shares < 0.95 * ranges) {
      p.prefix_ctas = (int)ctas;
      p.prefix_splits = (int)((ctas + p.pre.units - 1) / p.pre.units) + 1;
    }
  }
  p.own_splits = splits(p.own.wide ? kNumSMs : 2 * kNumSMs, p.own.units, max_k, 256);
  if (!p.own.wide && max_k / 64 * 0.65 * (p.own_splits - 1) < 5.0 * p.own_splits) p.own_splits = 1;
  p.final = !p.own.wide && p.own_splits == 1;
  return p;
}

template <typename T, int D, int RT, int NG>
static int launch_rows(const parts::Args& a, const parts::Seg& s, const parts::Seg& prefix, const Merge& mg, int n_requests,
                       int max_q, int final) {
  // with four groups two CTAs fit an SM, with two four (to the byte: 4 x (56 KB + 1 KB), head_dim 128)
  constexpr size_t smem = (size_t)RT * 16 * D * 2 + (size_t)NG * NS * 2 * KB * D * 2;
  auto kern = rows_kernel<T, D, RT, NG>;
  static std::atomic<uint64_t> allowed{0};
  ACACHE_CUDA_CHECK(allow_smem((const void*)kern, smem, allowed));
  const int g = a.n_heads / a.n_kv_heads;
  const int64_t tiles = ((int64_t)max_q * g + RT * 16 - 1) / (RT * 16);
  if (tiles * s.splits > 65535) return ACACHE_ELIMIT;
  ACACHE_CUDA_CHECK(launch_chained(kern, dim3(a.n_kv_heads, (unsigned)(tiles * s.splits), n_requests), dim3(RT * NG * 32), smem, a.st,
                                   a, s, prefix, mg, final));
  ACACHE_LAUNCH_CHECK();
  return ACACHE_OK;
}

template <typename T, int D, int RT>
static int launch_rows_ng(const parts::Args& a, const parts::Seg& s, const parts::Seg& prefix, const Merge& mg, int n_requests,
                          int max_q, int groups, int final) {
  if (groups == 4) return launch_rows<T, D, RT, 4>(a, s, prefix, mg, n_requests, max_q, final);
  return launch_rows<T, D, RT, 2>(a, s, prefix, mg, n_requests, max_q, final);
}

// one segment: its parts (or, final, the output)
template <typename T, int D>
static int launch_segment(const parts::Args& a, const parts::Seg& s, const Segment& how, const parts::Seg& prefix, const Merge& mg,
                          int n_requests, int max_q, int final) {
  if (how.wide) return attention_wide_parts(a, s, n_requests, max_q);
  if ((int64_t)max_q * (a.n_heads / a.n_kv_heads) <= 16)
    return launch_rows_ng<T, D, 1>(a, s, prefix, mg, n_requests, max_q, how.groups, final);
  return launch_rows_ng<T, D, 2>(a, s, prefix, mg, n_requests, max_q, how.groups, final);
}

template <typename T, int D>
static int run(const parts::Args& a, const parts::Seg& prefix, const parts::Seg& own, const Merge& mg, const Plan& plan, int batch,
               int max_q) {
  if (mg.n_parts > 0) {
    const int rc = launch_segment<T, D>(a, prefix, plan.pre, prefix, mg, 1, prefix.total_q, 0);
    if (rc != ACACHE_OK) return rc;
  }
  const int rc = launch_segment<T, D>(a, own, plan.own, prefix, mg, batch, max_q, plan.final);
  if (rc != ACACHE_OK || plan.final) return rc;
  ACACHE_CUDA_CHECK(launch_chained(merge_kernel<T, D>, dim3((unsigned)((own.n_rows + 15) / 16)), dim3(128), 0, a.st, a, own, prefix, mg, batch));
  ACACHE_LAUNCH_CHECK();
  return ACACHE_OK;
}

}  // namespace shared_prefix
}  // namespace acache

using namespace acache;

extern "C" int64_t acache_shared_prefix_attention_plan(int total_q, int n_heads, int n_kv_heads, int head_dim, int batch,
                                                       int max_seqlen_q, int max_seqlen_k, int prefix_len, int32_t* launches) {
  if (launches) *launches = 0;
  if (total_q <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || head_dim <= 0 || batch <= 0 || max_seqlen_q <= 0 ||
      max_seqlen_k < 0 || prefix_len < 0)
    return 0;                          // nothing to compute, or a call that is refused
  const shared_prefix::Plan p = shared_prefix::make_plan(total_q, batch, max_seqlen_q, max_seqlen_k, prefix_len, n_heads, n_kv_heads);
  const int64_t parts = p.prefix_splits + p.own_splits;
  if (launches) *launches = (prefix_len > 0) + 1 + !p.final;
  return parts * total_q * n_heads * (int64_t)(head_dim + 1) * 4;
}

extern "C" int64_t acache_shared_prefix_attention_scratch_bytes(int total_q, int n_heads, int n_kv_heads, int head_dim, int batch,
                                                                int max_seqlen_q, int max_seqlen_k, int prefix_len) {
  return acache_shared_prefix_attention_plan(total_q, n_heads, n_kv_heads, head_dim, batch, max_seqlen_q, max_seqlen_k, prefix_len, nullptr);
}

extern "C" int acache_shared_prefix_attention(const void* q, int64_t q_stride, void* out, int64_t o_stride, const void* k_cache,
                                              const void* v_cache, int64_t num_slots, int total_q, int n_heads, int n_kv_heads,
                                              int head_dim, int dtype, const int32_t* prefix_slots, int prefix_len,
                                              const int32_t* prefix_keep, int64_t keep_stride, const int32_t* cu_seqlens_q,
                                              const int32_t* cu_seqlens_k, int batch, int max_seqlen_q, int max_seqlen_k,
                                              const int32_t* read_slot_mapping, int n_slots, float softmax_scale, void* scratch,
                                              int64_t scratch_bytes, int32_t* err_flag, void* stream) {
  if (!dtype_ok(dtype) || total_q < 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || head_dim <= 0 || batch < 0 ||
      prefix_len < 0 || max_seqlen_q < 0 || max_seqlen_k < 0 || n_slots < 0 || num_slots < 0)
    return ACACHE_EINVAL;
  if (total_q == 0 || batch == 0 || max_seqlen_q == 0) return ACACHE_OK;
  if (!q || !out || !k_cache || !v_cache || !cu_seqlens_q || !cu_seqlens_k || !scratch || (prefix_len > 0 && !prefix_slots) ||
      (n_slots > 0 && !read_slot_mapping))
    return ACACHE_EINVAL;
  const float scale_log2 = softmax_scale * 1.4426950408889634f;
  if (!(scale_log2 > 0.f) || scale_log2 > 3.0e38f) return ACACHE_EINVAL;      // maxima are taken before the scale, dead keys are -inf
  if (dtype == ACACHE_F32 || (head_dim != 64 && head_dim != 128) || q_stride % 8 != 0 || o_stride % 8 != 0 || !aligned16(q) ||
      !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(scratch))
    return ACACHE_EUNSUPPORTED;
  if (prefix_keep && (keep_stride % 2 != 0 || keep_stride * 32 < prefix_len || (reinterpret_cast<uintptr_t>(prefix_keep) & 7) != 0))
    return ACACHE_EINVAL;
  if (num_slots > 0x7FFFFFFFll || batch > 65535 / 32 || prefix_len > (1 << 30) || n_slots > (1 << 30) ||
      (int64_t)total_q * (n_heads / n_kv_heads) > (1 << 23) || n_kv_heads > 65535)
    return ACACHE_ELIMIT;
  if (max_seqlen_q > total_q) max_seqlen_q = total_q;     // as the plan takes it
  const shared_prefix::Plan plan =
      shared_prefix::make_plan(total_q, batch, max_seqlen_q, max_seqlen_k, prefix_len, n_heads, n_kv_heads);
  const int64_t n_rows = (int64_t)total_q * n_heads, n_parts = plan.prefix_splits + plan.own_splits;
  if (scratch_bytes < n_parts * n_rows * (head_dim + 1) * 4) return ACACHE_EINVAL;
  float* o = (float*)scratch;
  float* lse = o + n_parts * n_rows * head_dim;
  const parts::Args a{q, q_stride, k_cache, v_cache, num_slots, n_heads, n_kv_heads, head_dim, dtype,
                      scale_log2, err_flag, (cudaStream_t)stream};
  const parts::Seg prefix{nullptr, nullptr, prefix_slots, prefix_len, total_q, plan.prefix_splits, prefix_keep, keep_stride, cu_seqlens_q,
                          batch, o, lse, n_rows, 0, plan.prefix_ctas, (int)plan.pre.units, (prefix_len + 127) / 128};
  const parts::Seg own{cu_seqlens_q, cu_seqlens_k, read_slot_mapping, n_slots, total_q, plan.own_splits, nullptr, 0, nullptr, 0, o, lse,
                       n_rows, plan.prefix_splits, 0, 0, 0};
  const shared_prefix::Merge mg{out, o_stride, prefix_len > 0 ? plan.prefix_splits : 0, prefix_slots, prefix_len};
  if (dtype == ACACHE_BF16)
    return head_dim == 128 ? shared_prefix::run<__nv_bfloat16, 128>(a, prefix, own, mg, plan, batch, max_seqlen_q)
                           : shared_prefix::run<__nv_bfloat16, 64>(a, prefix, own, mg, plan, batch, max_seqlen_q);
  return head_dim == 128 ? shared_prefix::run<__half, 128>(a, prefix, own, mg, plan, batch, max_seqlen_q)
                         : shared_prefix::run<__half, 64>(a, prefix, own, mg, plan, batch, max_seqlen_q);
}

extern "C" int acache_pack_keep_mask(const uint8_t* keep, int64_t stride, int batch, int prefix_len, int32_t* words, int64_t words_stride,
                                     void* stream) {
  if (batch < 0 || prefix_len < 0 || words_stride < (prefix_len + 31) / 32 || words_stride > (1 << 26)) return ACACHE_EINVAL;
  if (batch == 0 || words_stride == 0) return ACACHE_OK;
  if (!keep || !words) return ACACHE_EINVAL;
  const int64_t total = (int64_t)batch * words_stride;
  int64_t blocks = (total + 7) / 8;
  if (blocks > kNumSMs * 8) blocks = kNumSMs * 8;
  ACACHE_CUDA_CHECK(launch_chained(shared_prefix::pack_keep_kernel, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, keep, stride,
                                   prefix_len, (int)words_stride, (uint32_t*)words, total));
  ACACHE_LAUNCH_CHECK();
  return ACACHE_OK;
}
