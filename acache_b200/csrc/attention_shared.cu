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
// A part whose rows fill the tensor cores' 128-row tiles goes to the split form of attention_tc256.cu
// (tcgen05, 256 rows share a staged K/V tile).  A part with few rows (single tokens, short blocks: bound by
// the bytes of K and V) goes to rows_kernel below.
//
// rows_kernel: a CTA = (KV head, key range, request, 16 or 32 virtual rows), a virtual row being a (query,
// head-of-the-GQA-group) pair.  Its four warps split the keys in blocks of 16 and share nothing until the end:
// each gathers its own blocks through the slot map (16-byte cp.async into a ring of its own, three blocks
// ahead), multiplies with m16n8k16 tensor-core instructions (fp32 accumulators), keeps its own running
// maximum, sum and O in registers, and the four are merged through shared memory.  No barrier in the loop.
// 128-row tcgen05 tiles would leave 3/4 of every product empty here and need the whole CTA in step.
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

constexpr int NW = 4, NT = NW * 32;   // warps of a CTA
constexpr int KB = 16;                // keys of a block
constexpr int NS = 3;                 // blocks in flight per warp
constexpr int kMaxParts = 64;

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

// one warp: parts [begin, end) of a row added to (acc, m, l), acc = the sum of weights 2^(score - m) times V
template <int D>
__device__ __forceinline__ void merge_parts(const parts::Seg& s, int begin, int end, int64_t row, float* acc, float& m, float& l) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  for (int base = begin; base < end; base += 32) {
    const int n = min(32, end - base);
    const float lse = lane < n ? s.lse[(int64_t)(base + lane) * s.n_rows + row] : -INFINITY;
    const float top = fmaxf(m, warp_max(lse));
    const float f = m == -INFINITY && l == 0.f ? 0.f : ex2(m - top);
    const float w = lse == -INFINITY ? 0.f : ex2(lse - top);
    l = l * f + warp_sum(w);
    m = top;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = f == 0.f ? 0.f : acc[e] * f;
    for (int i = 0; i < n; ++i) {
      const float wi = __shfl_sync(0xFFFFFFFFu, w, i);
      if (wi == 0.f) continue;                  // a part without keys wrote no O
      const float* o = s.o + ((int64_t)(base + i) * s.n_rows + row) * D + lane * E;
      if constexpr (E == 4) {
        const float4 v = *reinterpret_cast<const float4*>(o);
        acc[0] = fmaf(wi, v.x, acc[0]);
        acc[1] = fmaf(wi, v.y, acc[1]);
        acc[2] = fmaf(wi, v.z, acc[2]);
        acc[3] = fmaf(wi, v.w, acc[3]);
      } else {
        const float2 v = *reinterpret_cast<const float2*>(o);
        acc[0] = fmaf(wi, v.x, acc[0]);
        acc[1] = fmaf(wi, v.y, acc[1]);
      }
    }
  }
}

// one warp: the row's final value from (acc, m, l) of its own keys and the prefix parts
template <typename T, int D>
__device__ __forceinline__ void finish_row(const parts::Args& a, const parts::Seg& prefix, const Merge& mg, int q_row, int head,
                                           float* acc, float m, float l) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)q_row * a.n_heads + head;
  float pre[E], pm = -INFINITY, pl = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) pre[e] = 0.f;
  merge_parts<D>(prefix, 0, mg.n_parts, row, pre, pm, pl);
  if (prefix.keep) {
    bool bad = false;
#pragma unroll
    for (int e = 0; e < E; ++e) bad |= isnan(pre[e]);
    if (__any_sync(0xFFFFFFFFu, bad) && pl > 0.f) {
      float again[E];
      recompute_prefix<T, D>(a, prefix, mg, q_row, head, pm + log2f(pl), again);
#pragma unroll
      for (int e = 0; e < E; ++e) pre[e] = isnan(pre[e]) ? again[e] * pl : pre[e];
    }
  }
  const float top = fmaxf(m, pm);
  // a side without keys has the sum 0; one with NaN scores has a NaN sum, which reaches the result
  const float fo = m == -INFINITY && l == 0.f ? 0.f : ex2(m - top), fp = pm == -INFINITY && pl == 0.f ? 0.f : ex2(pm - top);
  const float total = l * fo + pl * fp;
  const float inv = total == 0.f ? 0.f : 1.f / total;         // no key at all: zeros
  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = ((fo == 0.f ? 0.f : acc[e] * fo) + (fp == 0.f ? 0.f : pre[e] * fp)) * inv;
  T* dst = (T*)mg.out + (int64_t)q_row * mg.o_stride + (int64_t)head * D + lane * E;
  if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  else *reinterpret_cast<uint32_t*>(dst) = pack2<T>(v[0], v[1]);
}

// FINAL: the segment is the requests' own keys in one range each: the CTA also merges the prefix parts (written by
// the kernel before it in the stream, beside which it may run) and writes the output.  Else it leaves a part.
template <typename T, int D, int MT, bool FINAL>
__global__ void __launch_bounds__(NT, 2) rows_kernel(const __grid_constant__ parts::Args a, const __grid_constant__ parts::Seg s,
                                                     const __grid_constant__ parts::Seg prefix, const __grid_constant__ Merge mg,
                                                     int beside) {
  constexpr int ROWS = MT * 16, CH = D / 8, KS = D / 16, E = D / 32;
  constexpr int BLOCK = KB * D * 2;             // bytes of K (or V) of a block
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* sQ = smem;                           // [ROWS][D]
  uint8_t* ring = smem + ROWS * D * 2;          // [NW][NS][K | V]
  __shared__ float s_m[NW][ROWS], s_l[NW][ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // beside: the kernel before this one in the stream belongs to the same call and this one reads nothing
  // of it before the merge; the kernels before that one have completed
  if (!beside) chain_wait();
  chain_release();
  const int g = a.n_heads / a.n_kv_heads, kvh = blockIdx.x, b = blockIdx.z;
  const int split = blockIdx.y % s.splits, m0 = blockIdx.y / s.splits * ROWS;
  parts::Range r = parts::request_range(s, b);
  const int first_key = parts::split_range(s, split, KB * NW, r);
  const int vrows = r.n_q * g;
  if (m0 >= vrows) {
    if (beside) chain_wait();                   // this grid may not end before the one it runs beside
    return;
  }
  const int64_t kv_row = (int64_t)a.n_kv_heads * D;

  // ---- queries
  for (int i = tid; i < ROWS * CH; i += NT) {
    const int row = i / CH, c = i % CH, vr = m0 + row;
    const bool ok = vr < vrows;
    const T* src = (const T*)a.q + (int64_t)(r.q0 + (ok ? vr / g : 0)) * a.q_stride + (int64_t)(kvh * g + (ok ? vr % g : 0)) * D + c * 8;
    cp_async16(smem_u32(sQ) + at<D>(row, c), src, ok);
  }
  cp_async_commit();

  // ---- the keys of this warp: blocks warp, warp + NW, ...
  const int n_blocks = (r.n_k + KB - 1) / KB;
  const int mine = n_blocks > warp ? (n_blocks - warp + NW - 1) / NW : 0;
  const uint32_t my_ring = smem_u32(ring) + warp * (NS * 2 * BLOCK);
  const T* kc = (const T*)a.k_cache + (int64_t)kvh * D;
  const T* vc = (const T*)a.v_cache + (int64_t)kvh * D;
  // lane l (and l + 16) holds the slot of key l of a block; -1 = takes no part
  auto slot_of = [&](int i) -> int32_t {
    const int j = (warp + i * NW) * KB + (lane & 15);
    return i < mine && j < r.n_k ? s.slots[r.k0 + j] : -1;
  };
  auto check_slot = [&](int32_t v) -> int32_t {
    if (v < -1 || v >= a.num_slots) {
      if (a.err_flag) atomicExch(a.err_flag, 3);
      return -1;
    }
    return v;
  };
  auto gather = [&](int i, int32_t slot) {      // block i into its stage
    const uint32_t kb = my_ring + (i % NS) * (2 * BLOCK), vb = kb + BLOCK;
    constexpr int RPI = 32 / CH;                // rows per step of the warp
    const int c = lane % CH;
#pragma unroll
    for (int it = 0; it < KB / RPI; ++it) {
      const int row = it * RPI + lane / CH;
      const int32_t sl = __shfl_sync(0xFFFFFFFFu, slot, row);
      const int64_t off = (int64_t)(sl < 0 ? 0 : sl) * kv_row + c * 8;
      cp_async16(kb + at<D>(row, c), kc + off, sl >= 0);
      cp_async16(vb + at<D>(row, c), vc + off, sl >= 0);
    }
  };
  // dead keys of the blocks in flight, oldest first
  uint32_t dead_q[NS];
  int32_t next_slot = slot_of(0);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    const int32_t slot = check_slot(next_slot);
    next_slot = slot_of(i + 1);
    dead_q[i] = __ballot_sync(0xFFFFFFFFu, slot < 0);
    if (i < mine) gather(i, slot);
    cp_async_commit();
  }

  // which keys the rows of this thread keep: rows lane / 4 + 8 h
  const uint16_t* keep[2 * MT];
  if (s.keep) {
#pragma unroll
    for (int h = 0; h < 2 * MT; ++h) {
      const int vr = min(m0 + lane / 4 + 8 * h, vrows - 1);
      keep[h] = reinterpret_cast<const uint16_t*>(s.keep + (int64_t)parts::request_of(s.req_cu, s.n_req, r.q0 + vr / g) * s.keep_stride) + first_key / KB;
    }
  }

  cp_async_wait<NS - 1>();
  __syncthreads();                              // the queries have landed
  uint32_t qa[MT == 1 ? KS : 1][4];
  const uint32_t q_addr = smem_u32(sQ);
  if constexpr (MT == 1) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ldsm4(q_addr + at<D>(lane & 15, 2 * ks + (lane >> 4)), qa[ks]);
  }

  float o[MT][D / 8][4], m_ref[2 * MT], l_sum[2 * MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][d][e] = 0.f;
#pragma unroll
  for (int h = 0; h < 2 * MT; ++h) {
    m_ref[h] = -INFINITY;
    l_sum[h] = 0.f;
  }

  for (int i = 0; i < mine; ++i) {
    {
      const int32_t slot = check_slot(next_slot);
      next_slot = slot_of(i + NS);
      dead_q[NS - 1] = __ballot_sync(0xFFFFFFFFu, slot < 0);
      if (i + NS - 1 < mine) gather(i + NS - 1, slot);
      cp_async_commit();
    }
    uint32_t kept[2 * MT];
    if (s.keep) {
#pragma unroll
      for (int h = 0; h < 2 * MT; ++h) kept[h] = keep[h][warp + i * NW];
    }
    cp_async_wait<NS - 1>();
    __syncwarp();
    const uint32_t kb = my_ring + (i % NS) * (2 * BLOCK), vb = kb + BLOCK;

    // ---- scores: keys 0-7 and 8-15 of the block against every row tile
    float sc[MT][2][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) sc[t][e / 4][e % 4] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t kf[4];
      ldsm4(kb + at<D>((lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1)), kf);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if constexpr (MT == 1) {
          mma16816<T>(sc[t][0], qa[ks], kf[0], kf[1]);
          mma16816<T>(sc[t][1], qa[ks], kf[2], kf[3]);
        } else {
          uint32_t qf[4];
          ldsm4(q_addr + at<D>(t * 16 + (lane & 15), 2 * ks + (lane >> 4)), qf);
          mma16816<T>(sc[t][0], qf, kf[0], kf[1]);
          mma16816<T>(sc[t][1], qf, kf[2], kf[3]);
        }
      }
    }
    // ---- keys that take no part, per row under a keep mask
    const uint32_t dead = dead_q[0] & 0xFFFFu;
    if (dead != 0u || s.keep) {
#pragma unroll
      for (int h = 0; h < 2 * MT; ++h) {
        const uint32_t gone = (s.keep ? dead | ~kept[h] : dead) >> (2 * (lane & 3));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((gone >> ((e & 1) + 8 * (e >> 1))) & 1u) sc[h / 2][e >> 1][2 * (h & 1) + (e & 1)] = -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < NS - 1; ++k) dead_q[k] = dead_q[k + 1];
    // ---- online softmax; O is rescaled only when a row's maximum grows by more than 2^8
    float mx[2 * MT];
    bool grows = false;
#pragma unroll
    for (int h = 0; h < 2 * MT; ++h) {
      const float* c0 = &sc[h / 2][0][2 * (h & 1)];
      const float* c1 = &sc[h / 2][1][2 * (h & 1)];
      float v = fmaxf(fmaxf(c0[0], c0[1]), fmaxf(c1[0], c1[1]));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
      mx[h] = v * a.scale_log2;
      grows |= mx[h] > m_ref[h] + 8.f;
    }
    if (__any_sync(0xFFFFFFFFu, grows)) {
#pragma unroll
      for (int h = 0; h < 2 * MT; ++h) {
        const bool grow = mx[h] > m_ref[h] + 8.f;
        const float f = grow ? ex2(m_ref[h] - mx[h]) : 1.f;
        if (grow) m_ref[h] = mx[h];
        l_sum[h] *= f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[h / 2][d][2 * (h & 1)] *= f;
          o[h / 2][d][2 * (h & 1) + 1] *= f;
        }
      }
    }
    uint32_t pa[MT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float mu = m_ref[2 * t + h] == -INFINITY ? 0.f : m_ref[2 * t + h];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = ex2(fmaf(sc[t][n][2 * h], a.scale_log2, -mu)), p1 = ex2(fmaf(sc[t][n][2 * h + 1], a.scale_log2, -mu));
          l_sum[2 * t + h] += p0 + p1;
          pa[t][2 * n + h] = pack2<T>(p0, p1);
        }
      }
    }
    // ---- O += P V
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      uint32_t vf[4];
      ldsm4t(vb + at<D>(lane & 15, 2 * d + (lane >> 4)), vf);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        mma16816<T>(o[t][2 * d], pa[t], vf[0], vf[1]);
        mma16816<T>(o[t][2 * d + 1], pa[t], vf[2], vf[3]);
      }
    }
    __syncwarp();                               // the stage may be written again
  }
  cp_async_wait<0>();

  // ---- the four warps' results through shared memory (over the ring)
  __syncthreads();
  constexpr int LD = D + 4;
  float* sO = reinterpret_cast<float*>(ring);   // [NW][ROWS][LD]
#pragma unroll
  for (int h = 0; h < 2 * MT; ++h) {
    const int row = lane / 4 + 8 * h;
    float l = l_sum[h];
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
    if ((lane & 3) == 0) {
      s_m[warp][row] = m_ref[h];
      s_l[warp][row] = l;
    }
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
      *reinterpret_cast<float2*>(sO + (warp * ROWS + row) * LD + d * 8 + 2 * (lane & 3)) =
          make_float2(o[h / 2][d][2 * (h & 1)], o[h / 2][d][2 * (h & 1) + 1]);
  }
  __syncthreads();
  if (beside) chain_wait();                     // the prefix parts are there
  for (int row = warp; row < ROWS && m0 + row < vrows; row += NW) {
    float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, s_m[w][row]);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = s_m[w][row];
      if (mw == -INFINITY && s_l[w][row] == 0.f) continue;   // no key (only NaN scores leave a NaN sum)
      const float f = ex2(mw - m);
      l = fmaf(f, s_l[w][row], l);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(f, sO[(w * ROWS + row) * LD + lane * E + e], acc[e]);
    }
    const int vr = m0 + row, q_row = r.q0 + vr / g, head = kvh * g + vr % g;
    if constexpr (FINAL) {
      finish_row<T, D>(a, prefix, mg, q_row, head, acc, m, l);
    } else {
      const int64_t at_row = (int64_t)(s.first_part + split) * s.n_rows + (int64_t)q_row * a.n_heads + head;
      const bool any_key = m != -INFINITY || l != 0.f;
      if (any_key) {
        const float inv = 1.f / l;
#pragma unroll
        for (int e = 0; e < E; ++e) s.o[at_row * D + lane * E + e] = acc[e] * inv;
      }
      if (lane == 0) s.lse[at_row] = any_key ? m + log2f(l) : -INFINITY;
    }
  }
}

// one warp per row: own parts and prefix parts into the output
template <typename T, int D>
__global__ void __launch_bounds__(128) merge_kernel(const __grid_constant__ parts::Args a, const __grid_constant__ parts::Seg own,
                                                    const __grid_constant__ parts::Seg prefix, const __grid_constant__ Merge mg, int n_req) {
  chain_release();
  chain_wait();
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int q_row = (int)(row / a.n_heads), head = (int)(row % a.n_heads);
  // rows behind the last sequence (or before the first) have no result
  if (q_row >= own.total_q || q_row < own.cu_q[0] || q_row >= own.cu_q[n_req]) return;
  float acc[D / 32], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
  merge_parts<D>(own, own.first_part, own.first_part + own.splits, row, acc, m, l);
  finish_row<T, D>(a, prefix, mg, q_row, head, acc, m, l);
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
struct Plan {
  bool prefix_wide, own_wide;         // 256-row tcgen05 tiles instead of rows_kernel
  int prefix_splits, own_splits;
};

static int clamp_splits(int64_t want, int64_t keys, int min_keys) {
  const int64_t most = keys / min_keys;
  if (want > most) want = most;
  if (want > 32) want = 32;
  return want < 1 ? 1 : (int)want;
}

static Plan make_plan(int total_q, int batch, int max_q, int max_k, int prefix_len, int n_heads, int n_kv_heads) {
  const int64_t g = n_heads / n_kv_heads, all = total_q * g, per_request = max_q * g;
  Plan p;
  p.prefix_wide = all > 32;
  p.own_wide = per_request > 128;
  if (p.prefix_wide) p.prefix_splits = clamp_splits(kNumSMs / (n_kv_heads * ((all + 255) / 256)), prefix_len, 256);
  else p.prefix_splits = clamp_splits(2 * kNumSMs / (n_kv_heads * ((all + 31) / 32)), prefix_len, 128);
  if (p.own_wide) p.own_splits = clamp_splits(kNumSMs / (n_kv_heads * batch * ((per_request + 255) / 256)), max_k, 256);
  else p.own_splits = clamp_splits(2 * kNumSMs / (n_kv_heads * (int64_t)batch * ((per_request + 31) / 32)), max_k, 256);
  return p;
}

template <typename T, int D, int MT, bool FINAL>
static int launch_rows(const parts::Args& a, const parts::Seg& s, const parts::Seg& prefix, const Merge& mg, int n_requests,
                       int max_q, int beside) {
  constexpr size_t ring = (size_t)NW * NS * 2 * KB * D * 2, merge = (size_t)NW * MT * 16 * (D + 4) * 4;
  constexpr size_t smem = MT * 16 * D * 2 + (ring > merge ? ring : merge);
  auto kern = rows_kernel<T, D, MT, FINAL>;
  ACACHE_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int g = a.n_heads / a.n_kv_heads;
  const int64_t tiles = ((int64_t)max_q * g + MT * 16 - 1) / (MT * 16);
  if (tiles * s.splits > 65535) return ACACHE_ELIMIT;
  ACACHE_CUDA_CHECK(launch_chained(kern, dim3(a.n_kv_heads, (unsigned)(tiles * s.splits), n_requests), dim3(NT), smem, a.st, a, s,
                                   prefix, mg, beside));
  ACACHE_LAUNCH_CHECK();
  return ACACHE_OK;
}

template <typename T, int D, bool FINAL>
static int launch_rows_mt(const parts::Args& a, const parts::Seg& s, const parts::Seg& prefix, const Merge& mg, int n_requests,
                          int max_q, int beside) {
  if ((int64_t)max_q * (a.n_heads / a.n_kv_heads) <= 16) return launch_rows<T, D, 1, FINAL>(a, s, prefix, mg, n_requests, max_q, beside);
  return launch_rows<T, D, 2, FINAL>(a, s, prefix, mg, n_requests, max_q, beside);
}

template <typename T, int D>
static int run(const parts::Args& a, parts::Seg prefix, parts::Seg own, Merge mg, const Plan& plan, int batch, int max_q) {
  int rc;
  if (mg.n_parts > 0) {
    rc = plan.prefix_wide ? attention_tc256_parts(a, prefix, 1, prefix.total_q)
                          : launch_rows_mt<T, D, false>(a, prefix, prefix, mg, 1, prefix.total_q, 0);
    if (rc != ACACHE_OK) return rc;
  }
  const int beside = mg.n_parts > 0 ? 1 : 0;
  if (!plan.own_wide && plan.own_splits == 1) return launch_rows_mt<T, D, true>(a, own, prefix, mg, batch, max_q, beside);
  rc = plan.own_wide ? attention_tc256_parts(a, own, batch, max_q) : launch_rows_mt<T, D, false>(a, own, prefix, mg, batch, max_q, beside);
  if (rc != ACACHE_OK) return rc;
  ACACHE_CUDA_CHECK(launch_chained(merge_kernel<T, D>, dim3((unsigned)((own.n_rows + 3) / 4)), dim3(128), 0, a.st, a, own, prefix, mg, batch));
  ACACHE_LAUNCH_CHECK();
  return ACACHE_OK;
}

}  // namespace shared_prefix
}  // namespace acache

using namespace acache;

extern "C" int64_t acache_shared_prefix_attention_scratch_bytes(int total_q, int n_heads, int n_kv_heads, int head_dim, int batch,
                                                                int max_seqlen_q, int max_seqlen_k, int prefix_len) {
  if (total_q <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || head_dim <= 0 || batch <= 0 || max_seqlen_q < 0 ||
      max_seqlen_k < 0 || prefix_len < 0)
    return 0;
  const shared_prefix::Plan p = shared_prefix::make_plan(total_q, batch, max_seqlen_q, max_seqlen_k, prefix_len, n_heads, n_kv_heads);
  const int64_t parts = p.prefix_splits + p.own_splits;
  return parts * total_q * n_heads * (int64_t)(head_dim + 1) * 4;
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
  if (dtype == ACACHE_F32 || (head_dim != 64 && head_dim != 128) || q_stride % 8 != 0 || o_stride % 8 != 0 || !aligned16(q) ||
      !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(scratch))
    return ACACHE_EUNSUPPORTED;
  if (prefix_keep && (keep_stride % 2 != 0 || keep_stride * 32 < prefix_len || (reinterpret_cast<uintptr_t>(prefix_keep) & 7) != 0))
    return ACACHE_EINVAL;
  if (num_slots > 0x7FFFFFFFll || batch > 65535 / 32 || prefix_len > (1 << 30) || n_slots > (1 << 30) ||
      (int64_t)total_q * (n_heads / n_kv_heads) > (1 << 23) || n_kv_heads > 65535)
    return ACACHE_ELIMIT;
  if (max_seqlen_q > total_q) max_seqlen_q = total_q;
  const shared_prefix::Plan plan =
      shared_prefix::make_plan(total_q, batch, max_seqlen_q, max_seqlen_k, prefix_len, n_heads, n_kv_heads);
  const int64_t n_rows = (int64_t)total_q * n_heads, n_parts = plan.prefix_splits + plan.own_splits;
  if (scratch_bytes < n_parts * n_rows * (head_dim + 1) * 4) return ACACHE_EINVAL;
  float* o = (float*)scratch;
  float* lse = o + n_parts * n_rows * head_dim;
  const parts::Args a{q, q_stride, k_cache, v_cache, num_slots, n_heads, n_kv_heads, head_dim, dtype,
                      softmax_scale * 1.4426950408889634f, err_flag, (cudaStream_t)stream};
  const parts::Seg prefix{nullptr, nullptr, prefix_slots, prefix_len, total_q, plan.prefix_splits, prefix_keep, keep_stride, cu_seqlens_q,
                          batch, o, lse, n_rows, 0};
  const parts::Seg own{cu_seqlens_q, cu_seqlens_k, read_slot_mapping, n_slots, total_q, plan.own_splits, nullptr, 0, nullptr, 0, o, lse,
                       n_rows, plan.prefix_splits};
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
