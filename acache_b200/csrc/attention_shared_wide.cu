// Parts of shared-prefix attention (attention_shared.cu) whose rows fill the tensor cores' tiles: tcgen05 + TMEM,
// bf16 / fp16, head_dim 64 / 128.
//
// A CTA works on (KV head, request and key range, 256 virtual rows), one of them or a share of several; a virtual row is a
// (query, head-of-the-GQA-group) pair.  The rows are two blocks of 128 that share every staged tile of 128 keys and take turns: while the tensor cores
// work on one block's products, the other block's threads are in their softmax.  Roles hand over through mbarriers:
//   warps 0-15   softmax: two threads per row, one for each half of a tile's keys;
//   warp 16      issues the products: for one row block after the other O += P(i) V(i), then S(i+1) = Q K(i+1)^T; the warp
//                waits as a whole and one elected lane issues.  One stream of products in this order keeps the blocks
//                half a period apart; with an issuing warp per block the products interleave one by one, both blocks get
//                their scores at the same time, and the tensor cores and the exponentials take turns (5600 cycles a
//                tile against 4400);
//   warps 17,18  gather the K and the V tiles through the slot map (16-byte cp.async into the 128-byte-swizzled operand
//                layout, two stages each); the K warp publishes which keys of a tile take no part.
// TMEM (512 columns): row block r holds S at 256 r and O at 256 r + 128.  P(i) lies over S(i): the first key half's
// weights in columns 0-31, the second's in 64-95, so each thread overwrites scores that it has read itself.
//
// Every thread keeps its row's reference maximum, the same in both threads of a row, and forms a tile's weights against
// it while it looks for the tile's maximum.  When neither thread sees a score beyond 2^8 times it (one barrier with a vote
// per tile and pair of warps says so) the weights stand; otherwise the two exchange their maxima, each rescales its half
// of O (after P V(i-1)), and both form the weights again with the new one.  The final division by the row sum makes it
// exact.  Weights are rounded to the tensors' type before P V, their sum is not (attention_parts.cuh).
//
// The result of a row is (O / l, log2 of its sum), fp32, turned through shared memory so that warps write whole 128-byte
// lines.  The S and O barriers of tile i are number i & 1 of two: a waiter is never a full round of them behind, since
// the tile two on needs the stage or the P that the waiter still holds.  All waits are bounded; when one runs out the
// kernel raises error code 5, frees its TMEM and returns.
//
// Bound, per 128 keys and 256 rows, by the exponentials (16 a cycle and SM: 2048 cycles) and the products (M = 128, K = 16
// products take 64 cycles at N = 128 and 48 at N = 64: 2048 cycles); what a tile costs besides is a fixed chain of TMEM
// loads, maxima, votes and barriers (a block's softmax about 2600 cycles, 1300 of them exponentials, its products 1100,
// the hand-overs 700), which is why a tile has 128 keys: with 64 (and two S buffers) 128 keys took 4800 cycles, with one
// thread per row as with two.  Measured: 7168 rows x 8192 keys, 4 heads (120 GFLOP) in 144 us on all 148 SMs, 0.83 PFLOP/s.
#include "attention_parts.cuh"
#include "common.cuh"
#include "tcgen05.cuh"

namespace acache {
namespace wide_parts {

using namespace tc;

constexpr int BM = 128, RB = 2, BN = 128, HN = BN / 2;       // rows of a block, blocks, keys of a tile and of a thread
constexpr int W_ROWS = 16, W_ISSUE = W_ROWS, W_LOADK = W_ISSUE + 1, W_LOADV = W_LOADK + 1, NT = (W_LOADV + 1) * 32;
constexpr int NS = 2;                 // stages of K and of V, barriers per event that alternate with the tile
constexpr int RING = 4;               // tiles whose dead-key masks are kept
constexpr uint32_t kTmemCols = 512;

// barriers, in units of 8 bytes
enum { BAR_K = 0, BAR_V = BAR_K + NS, BAR_S = BAR_V + NS, BAR_O = BAR_S + RB * NS, BAR_P = BAR_O + RB * NS, BAR_Q = BAR_P + RB,
       N_BARS = BAR_Q + RB };

// SHARES: the CTA takes a share of all tiles (s.ctas), else one part.  A template, since what a loop over pieces keeps in
// registers costs the one-part form 3 %.
template <typename T, int D, bool SHARES>
__global__ void __launch_bounds__(NT, 1)
wide_parts_kernel(const __grid_constant__ parts::Args a, const __grid_constant__ parts::Seg s) {
  constexpr int CH = D * 2 / 16;                      // 16-byte chunks per row
  constexpr int Q_BYTES = BM * D * 2, KV_BYTES = BN * D * 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {                // the swizzled operand layout needs 1024-byte aligned atoms
    if (threadIdx.x == 0 && a.err_flag) atomicExch(a.err_flag, 6);
    chain_wait();
    return;
  }
  uint8_t* sQ = smem;                                 // RB blocks
  uint8_t* sK = sQ + RB * Q_BYTES;
  uint8_t* sV = sK + NS * KV_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + NS * KV_BYTES);
  uint32_t* ring_words = reinterpret_cast<uint32_t*>(bars + ((N_BARS + 1) & ~1));
  uint32_t* tmem_slot = ring_words + RING * 8;
  volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_max = reinterpret_cast<float*>(tmem_slot + 4);      // [2 halves][256 rows]
  const uint32_t dead_ring = smem_u32(ring_words), bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + (uint32_t)i * 8u; };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = a.n_heads / a.n_kv_heads;
  // row warps: row block, TMEM lane quadrant and key half
  const bool is_row = warp < W_ROWS;
  const int quad = warp & 3, rb = (warp >> 2) & 1, half = warp >> 3;
  const int row = rb * BM + quad * 32 + lane;

  chain_release();
  chain_wait();

  auto wait_bar = [&](uint32_t at, uint32_t parity) -> bool {      // bounded; ends too when another role has given up
    const long long t0 = clock64();
    for (uint32_t it = 0;; ++it) {
      uint32_t done;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done) : "r"(at), "r"(parity) : "memory");
      if (done) return true;
      if ((it & 63) == 63) {
        if (*give_up) return false;
        if (clock64() - t0 > kWaitCycles) {
          *give_up = 1;
          return false;
        }
        __nanosleep(32);
      }
    }
  };
  auto wait_tile = [&](int first, int t) { return wait_bar(bar(first + (t & 1)), (uint32_t)((t >> 1) & 1)); };
  auto arrive = [&](uint32_t at) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(at) : "memory"); };
  auto warp_arrive = [&](uint32_t at) {
    __syncwarp();
    if (lane == 0) arrive(at);
  };

  // One part per CTA, or (SHARES) its share of all tiles of all units, a unit being a KV head and 256 rows over the whole
  // prefix: the share may end in the middle of a unit and go on in the next, each piece is a part.
  [[maybe_unused]] int64_t at = 0, end = 1;
  if constexpr (SHARES) {
    const int64_t all = (int64_t)s.units * s.unit_tiles;
    at = blockIdx.x * all / s.ctas;
    end = (blockIdx.x + 1) * all / s.ctas;
  }
  bool first_piece = true;
  do {
  int kvh = blockIdx.x, m0 = blockIdx.z * (RB * BM), part, first_tile, spare = 0;
  parts::Range r = parts::request_range(s, SHARES ? 0 : blockIdx.y / s.splits);
  const int vrows = r.n_q * g;
  if constexpr (SHARES) {
    const int64_t all = (int64_t)s.units * s.unit_tiles;
    const int unit = (int)(at / s.unit_tiles);
    const int64_t unit0 = (int64_t)unit * s.unit_tiles;
    first_tile = (int)(at - unit0);
    const int last_tile = (int)min((int64_t)s.unit_tiles, end - unit0);
    kvh = unit % a.n_kv_heads;
    m0 = unit / a.n_kv_heads * (RB * BM);
    part = (int)(blockIdx.x - ((unit0 + 1) * s.ctas - 1) / all);        // CTAs since the one that holds the unit's first tile
    if (last_tile == s.unit_tiles) spare = s.splits - 1 - part;         // parts of the unit that no CTA has
    r.k0 += first_tile * BN;
    r.n_k = min(r.n_k, last_tile * BN) - first_tile * BN;
    at = unit0 + last_tile;
  } else {
    part = blockIdx.y % s.splits;
    if (m0 >= vrows) return;
    first_tile = parts::split_range(s, part, BN, r) / BN;
  }
  const int n_tiles = (r.n_k + BN - 1) / BN;
  const int vr = m0 + row;
  const bool row_ok = is_row && vr < vrows;
  const int qi = row_ok ? vr / g : 0, head = kvh * g + (row_ok ? vr - qi * g : 0);
  const int64_t part_row = (int64_t)(s.first_part + part) * s.n_rows + (int64_t)(r.q0 + qi) * a.n_heads + head;
  if (n_tiles == 0) {                                  // not with shares: a share has a tile of every unit it touches
    if (row_ok && half == 0) s.lse[part_row] = -INFINITY;
    return;
  }

  if (tid == 0) {
    if (!first_piece)
      for (int i = 0; i < N_BARS; ++i) asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bar(i)) : "memory");
    for (int i = 0; i < 2 * NS; ++i) mbar_init(bar(BAR_K + i), 1);                    // a loader warp
    for (int i = 0; i < 2 * RB * NS; ++i) mbar_init(bar(BAR_S + i), 1);               // product commits
    for (int i = 0; i < 2 * RB; ++i) mbar_init(bar(BAR_P + i), 8);                    // row warps of a block
    if (first_piece) *give_up = 0;
    for (int t = 0; t < RING * 2; ++t) ring_words[t * 4 + 2] = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (first_piece && warp == W_ISSUE) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // ---- the queries, while TMEM is being allocated
  if (is_row) {
    constexpr int RPI = 256 / CH;                      // rows per step of a block's 256 threads
    const int t = half * 128 + quad * 32 + lane, c = t % CH;
    int v = m0 + rb * BM + t / CH, q_at = v / g, h_at = v - q_at * g;
    const int q_step = RPI / g, h_step = RPI - q_step * g;
    const T* base = (const T*)a.q + (int64_t)r.q0 * a.q_stride + (int64_t)kvh * g * D + c * 8;
#pragma unroll
    for (int it = 0; it < BM / RPI; ++it) {
      const bool ok = v < vrows;
      cp_async16(smem_u32(sQ) + rb * Q_BYTES + swz<D>(BM, t / CH + it * RPI, c),
                 base + (ok ? (int64_t)q_at * a.q_stride + (int64_t)h_at * D : 0), ok);
      v += RPI;
      q_at += q_step;
      h_at += h_step;
      if (h_at >= g) {
        h_at -= g;
        ++q_at;
      }
    }
    cp_async_commit();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == W_ISSUE) {
    // ---------------------------------------------------------------- products
    const uint32_t idesc_s = make_idesc(Fmt<T>::id, 0, BN, BM), idesc_o = make_idesc(Fmt<T>::id, 1, D, BM);
    auto done_on = [&](int blk, uint32_t at) {
      if (m0 + blk * BM < vrows) mma_commit(at);
      else arrive(at);                                 // a block of padding: no products, the hand-over stays
    };
    auto issue_s = [&](int blk, int i) {               // by one lane
      if (m0 + blk * BM < vrows) {
        const uint32_t qb = smem_u32(sQ) + blk * Q_BYTES, kb = smem_u32(sK) + (i & 1) * KV_BYTES;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          mma_ss(tmem + blk * 256, make_desc(qb + (ks / 4) * (BM * 128) + (ks % 4) * 32, 16, 1024),
                 make_desc(kb + (ks / 4) * (BN * 128) + (ks % 4) * 32, 16, 1024), idesc_s, ks > 0 ? 1u : 0u);
      }
      done_on(blk, bar(BAR_S + blk * NS + (i & 1)));
    };
    bool ok = wait_bar(bar(BAR_Q), 0);
    ok = ok && wait_bar(bar(BAR_Q + 1), 0) && wait_tile(BAR_K, 0);
    ok = __all_sync(0xFFFFFFFFu, ok);
    tc_fence_after();
    if (ok && elect_one()) {
      issue_s(0, 0);
      issue_s(1, 0);
    }
    __syncwarp();
    for (int i = 0; i < n_tiles && ok; ++i) {
      ok = wait_tile(BAR_V, i);
      if (i + 1 < n_tiles) ok = ok && wait_tile(BAR_K, i + 1);
#pragma unroll
      for (int blk = 0; blk < RB; ++blk) {
        ok = ok && wait_bar(bar(BAR_P + blk), (uint32_t)(i & 1));
        ok = __all_sync(0xFFFFFFFFu, ok);
        tc_fence_after();
        if (ok && elect_one()) {
          if (m0 + blk * BM < vrows) {
            const uint32_t vb = smem_u32(sV) + (i & 1) * KV_BYTES;
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks)       // 16 keys: 8 columns of a half's weights
              mma_ts(tmem + blk * 256 + 128, tmem + blk * 256 + (ks / 4) * HN + (ks % 4) * 8, make_desc(vb + ks * 2048, BN * 128, 1024),
                     idesc_o, (i > 0 || ks > 0) ? 1u : 0u);
          }
          done_on(blk, bar(BAR_O + blk * NS + (i & 1)));
          if (i + 1 < n_tiles) issue_s(blk, i + 1);    // after P V(i), which reads P(i) where S(i + 1) goes
        }
        __syncwarp();
      }
    }
  } else if (!is_row) {
    // ---------------------------------------------------------------- loaders
    const bool for_k = warp < W_LOADV;
    constexpr int RPI = 32 / CH;                       // rows per step
    const int c = lane % CH, r0 = lane / CH;
    const T* cache = (const T*)(for_k ? a.k_cache : a.v_cache) + (int64_t)kvh * D + c * 8;
    const int64_t kv_row = (int64_t)a.n_kv_heads * D;
    const uint32_t stage0 = smem_u32(for_k ? sK : sV);
    const int bar_land = for_k ? BAR_K : BAR_V, bar_read = for_k ? BAR_S : BAR_O;
    // lane l looks up keys l, l + 32, ... of a tile, two tiles ahead; behind the end: -1
    auto fetch = [&](int i, int32_t (&raw)[4]) {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int j = i * BN + h * 32 + lane;
        raw[h] = i < n_tiles && j < r.n_k ? s.slots[r.k0 + j] : -1;
      }
    };
    int32_t now[4], nxt[4];
    fetch(0, now);
    fetch(1, nxt);
    bool ok = true;
    for (int i = 0; i < n_tiles; ++i) {
      if (i >= NS) {                                   // the stage held tile i - 2, read by both blocks' products
        ok = wait_tile(bar_read, i - NS) && wait_tile(bar_read + NS, i - NS);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
      }
      uint32_t dead[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (now[h] < -1 || now[h] >= a.num_slots) {
          if (warp == W_LOADK && a.err_flag) atomicExch(a.err_flag, 3);
          now[h] = -1;
        }
        dead[h] = __ballot_sync(0xFFFFFFFFu, now[h] < 0);
      }
      if (warp == W_LOADK && lane < 2)                           // the ring's slot held tile i - 4, whose softmax ended long ago
        asm volatile("st.volatile.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dead_ring + (i % RING) * 32 + lane * 16),
                     "r"(lane ? dead[2] : dead[0]), "r"(lane ? dead[3] : dead[1]), "r"((uint32_t)i + 1u), "r"(0u) : "memory");
      const uint32_t stage = stage0 + (i & 1) * KV_BYTES;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
#pragma unroll
        for (int it = 0; it < 32 / RPI; ++it) {
          const int key = r0 + it * RPI;
          const int32_t sl = __shfl_sync(0xFFFFFFFFu, now[h], key);
          cp_async16(stage + swz<D>(BN, h * 32 + key, c), cache + (int64_t)(sl < 0 ? 0 : sl) * kv_row, sl >= 0);
        }
      }
      cp_async_commit();
#pragma unroll
      for (int h = 0; h < 4; ++h) now[h] = nxt[h];
      fetch(i + 2, nxt);
      cp_async_wait<0>();
      fence_proxy_async();
      warp_arrive(bar(bar_land + (i & 1)));
    }
    if (!ok) *give_up = 1;
  } else {
    // ---------------------------------------------------------------- softmax
    cp_async_wait<0>();
    fence_proxy_async();
    warp_arrive(bar(BAR_Q + rb));
    const uint32_t t_lane = tmem + ((uint32_t)(quad * 32) << 16), col_o = t_lane + rb * 256 + 128;
    const uint2* keep = nullptr;
    if (s.keep && row_ok)
      keep = reinterpret_cast<const uint2*>(s.keep + (int64_t)parts::request_of(s.req_cu, s.n_req, r.q0 + qi) * s.keep_stride) +
             first_tile * 2 + half;
    const bool warp_live = m0 + rb * BM + quad * 32 < vrows;
    const int pair_bar = 1 + rb * 4 + quad;            // the two warps that share 32 rows
    auto vote = [&](bool mine) -> bool {               // a barrier of the two warps that says whether any thread's is true
      int any = mine;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %0, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
          : "+r"(any) : "r"(pair_bar) : "memory");
      return any != 0;
    };
    constexpr float kHead = parts::kHead<T>, kLag = parts::kLag<T>;
    float m_ref = -INFINITY, l_sum = 0.f;
    bool ok = true;
    for (int i = 0; i < n_tiles; ++i) {
      uint2 kept = make_uint2(0xFFFFFFFFu, 0xFFFFFFFFu);
      if (keep && i * BN + half * HN < r.n_k) kept = keep[2 * i];      // the words end with the last 64 keys
      ok = wait_tile(BAR_S + rb * NS, i) && ok;
      tc_fence_after();
      if (warp_live) {
        const uint32_t col_s = t_lane + rb * 256 + half * HN;
        // the tile's dead keys, published by the K loader long before the product that was awaited
        uint32_t xa[32], xb[32];
        tmem_ld32(col_s, xa);
        uint32_t dl, dh, tag, pad;
        auto read_ring = [&]() {
          asm volatile("ld.volatile.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(dl), "=r"(dh), "=r"(tag), "=r"(pad)
                       : "r"(dead_ring + (i % RING) * 32 + half * 16) : "memory");
        };
        read_ring();
        if (tag != (uint32_t)i + 1u) {
          const long long t0 = clock64();
          while (tag != (uint32_t)i + 1u && clock64() - t0 < kWaitCycles && !*give_up) {
            __nanosleep(32);
            read_ring();
          }
          if (tag != (uint32_t)i + 1u) ok = false;
        }
        const bool bad = !ok || *give_up != 0;
        dl |= ~kept.x;
        dh |= ~kept.y;
        const bool any_dead = __any_sync(0xFFFFFFFFu, (dl | dh) != 0u);
        const uint64_t sc2 = pack_f32x2(a.scale_log2, a.scale_log2);
        uint64_t rs2;
        float mx;
        uint32_t w[32];
        // 32 scores: dead ones to -inf, the maximum into mx, weights against the row's reference, two to a word, and their sum
        auto weigh = [&](uint32_t (&x)[32], uint32_t dead, uint32_t* out, uint64_t nm2) {
          if (any_dead) {
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = (dead >> c) & 1u ? 0xFF800000u : x[c];
          }
          float m4[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) m4[k] = fmaxf(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1]));
#pragma unroll
          for (int c = 8; c < 32; c += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) m4[k] = max3(m4[k], __uint_as_float(x[c + 2 * k]), __uint_as_float(x[c + 2 * k + 1]));
          mx = max3(mx, max3(m4[0], m4[1], m4[2]), m4[3]);
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float x0, x1;
            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), sc2, nm2), x0, x1);
            const float p0 = ex2(x0), p1 = ex2(x1);
            rs2 = add_f32x2(rs2, pack_f32x2(p0, p1));
            out[c / 2] = pack2<T>(p0, p1);
          }
        };
        bool leave = false;
        for (;;) {                                     // xa is on its way
          const float m_use = m_ref == -INFINITY ? 0.f : m_ref;    // no live key so far: every weight is 0 (or not used)
          const uint64_t nm2 = pack_f32x2(-m_use, -m_use);
          rs2 = pack_f32x2(0.f, 0.f);
          mx = -INFINITY;
          tmem_wait_ld();
          tmem_ld32(col_s + 32, xb);
          weigh(xa, dl, w, nm2);
          tmem_wait_ld();
          weigh(xb, dh, w + 16, nm2);
          mx *= a.scale_log2;
          // does any of the 64 threads see a score beyond its row's reference (or know of a wait that ran out)?
          if (!vote(mx > m_ref + kLag || bad)) break;
          s_max[half * 256 + row] = mx;
          if (vote(bad)) {             // both warps leave together: neither may meet the other's barrier alone
            leave = true;
            break;
          }
          mx = fmaxf(mx, s_max[(half ^ 1) * 256 + row]);
          const bool grow = mx > m_ref + kLag;
          const float f = grow ? ex2(m_ref - (mx - kHead)) : 1.0f;
          l_sum *= f;
          if (grow) m_ref = mx - kHead;
          if (i > 0) {
            // O may only be touched between two products: P V(i-1) is done, P V(i) needs this thread's P(i)
            ok = wait_tile(BAR_O + rb * NS, i - 1) && ok;
            tc_fence_after();
#pragma unroll 1
            for (int c0 = half * (D / 2); c0 < (half + 1) * (D / 2); c0 += 32) {
              tmem_ld32(col_o + c0, xa);
              tmem_wait_ld();
#pragma unroll
              for (int c = 0; c < 32; ++c) xa[c] = __float_as_uint(__uint_as_float(xa[c]) * f);
              tmem_st32(col_o + c0, xa);
            }
            tmem_wait_st();
          }
          asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");      // s_max may be written again
          tmem_ld32(col_s, xa);                        // the weights again, against the new reference
        }
        if (leave) {
          ok = false;
          break;
        }
        tmem_st32(col_s, w);
        tmem_wait_st();
        float r0, r1;
        unpack_f32x2(rs2, r0, r1);
        l_sum += r0 + r1;
      }
      tc_fence_before();
      warp_arrive(bar(BAR_P + rb));
      if (!warp_live && !ok) break;
    }
    if (ok) ok = wait_tile(BAR_O + rb * NS, n_tiles - 1);
    tc_fence_after();
    if (!ok) *give_up = 1;
    s_max[half * 256 + row] = l_sum;
    asm volatile("bar.sync 15, %0;" ::"n"(W_ROWS * 32) : "memory");      // also: both blocks' products have read Q, K and V
    if (*give_up) {
      if (tid == 0 && a.err_flag) atomicExch(a.err_flag, 5);
    } else if (warp_live) {
      l_sum += s_max[(half ^ 1) * 256 + row];
      const bool any_key = m_ref != -INFINITY || l_sum != 0.f;   // nothing but NaN scores: a NaN sum
      const float inv = any_key ? 1.0f / l_sum : 0.f;
      const uint32_t writes = __ballot_sync(0xFFFFFFFFu, row_ok && any_key);
      uint8_t* turn = smem + warp * 4096;              // 32 rows x 32 columns of fp32, 16-byte chunks xor-ed with the row
      uint32_t o[32];
#pragma unroll 1
      for (int c0 = half * (D / 2); c0 < (half + 1) * (D / 2); c0 += 32) {
        tmem_ld32(col_o + c0, o);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          *reinterpret_cast<float4*>(turn + lane * 128 + ((k ^ (lane & 7)) << 4)) =
              make_float4(__uint_as_float(o[4 * k]) * inv, __uint_as_float(o[4 * k + 1]) * inv, __uint_as_float(o[4 * k + 2]) * inv,
                          __uint_as_float(o[4 * k + 3]) * inv);
        __syncwarp();
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int rr = it * 4 + (lane >> 3), k = lane & 7;
          const int64_t dst = __shfl_sync(0xFFFFFFFFu, part_row, rr);
          if ((writes >> rr) & 1u)
            *reinterpret_cast<float4*>(s.o + dst * D + c0 + k * 4) = *reinterpret_cast<const float4*>(turn + rr * 128 + ((k ^ (rr & 7)) << 4));
        }
        __syncwarp();
      }
      if (row_ok && half == 0) {
        s.lse[part_row] = any_key ? m_ref + log2f(l_sum) : -INFINITY;
        for (int i = 1; i <= spare; ++i) s.lse[part_row + i * s.n_rows] = -INFINITY;
      }
    }
  }
  cp_async_wait<0>();
  tc_fence_before();
  if (__syncthreads_or(*give_up)) break;
  tc_fence_after();
  first_piece = false;
  } while (SHARES && at < end);
  if (warp == W_ISSUE)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(kTmemCols) : "memory");
}

template <typename T, int D, bool SHARES>
static int launch(const parts::Args& a, const parts::Seg& seg, int n_requests, int max_q) {
  constexpr size_t smem = (size_t)RB * BM * D * 2 + (size_t)2 * NS * BN * D * 2 + N_BARS * 8 + 16 + RING * 32 + 16 + 2 * 256 * 4;
  const int g = a.n_heads / a.n_kv_heads;
  const int tiles = (max_q * g + RB * BM - 1) / (RB * BM);
  auto kern = wide_parts_kernel<T, D, SHARES>;
  static std::atomic<uint64_t> allowed{0};
  ACACHE_CUDA_CHECK(allow_smem((const void*)kern, smem, allowed));
  const dim3 grid = SHARES ? dim3(seg.ctas) : dim3(a.n_kv_heads, n_requests * seg.splits, tiles);
  ACACHE_CUDA_CHECK(launch_chained(kern, grid, dim3(NT), smem, a.st, a, seg));
  ACACHE_LAUNCH_CHECK();
  return ACACHE_OK;
}

template <typename T, int D>
static int launch_form(const parts::Args& a, const parts::Seg& seg, int n_requests, int max_q) {
  return seg.ctas > 0 ? launch<T, D, true>(a, seg, n_requests, max_q) : launch<T, D, false>(a, seg, n_requests, max_q);
}

}  // namespace wide_parts

int attention_wide_parts(const parts::Args& a, const parts::Seg& seg, int n_requests, int max_q) {
  using namespace wide_parts;
  if (a.dtype == ACACHE_BF16)
    return a.head_dim == 128 ? launch_form<__nv_bfloat16, 128>(a, seg, n_requests, max_q) : launch_form<__nv_bfloat16, 64>(a, seg, n_requests, max_q);
  return a.head_dim == 128 ? launch_form<__half, 128>(a, seg, n_requests, max_q) : launch_form<__half, 64>(a, seg, n_requests, max_q);
}

}  // namespace acache
