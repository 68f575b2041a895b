// Attention over packed sequences on tcgen05: o = softmax(scale q k^T + mask) v with fp32 scores, statistics and sums.
//
// One pass over the keys with a running maximum m and sum l for each query row: for each 128-key tile
//   s = q k^T,  m' = max(m, max s),  p = exp2(c (s - m')),  l = l exp2(c (m - m')) + sum p,  o = o exp2(c (m - m')) + p v
// with c = scale log2(e), and o / l at the end.  The scores never leave the SM.
//
// A CTA owns two 128-row query tiles (a work item) and streams its key and value tiles once for both: while the tensor
// cores multiply for one tile, the softmax of the other runs.  TMEM (512 columns): S0, S1 (128 fp32 columns each; the
// 16-bit p of a tile overwrites its scores and is the A operand of the second product straight from TMEM) and O0, O1.
// Warps 0-3 and 4-7: softmax of tile 0 and 1, one thread per row (no shuffles).  Warp 8: MMA issue.  Warp 9: TMA.
// Warp 10: clears the value rows behind a sequence's end.
//
// Rows of a query tile are (position, head of the group) pairs: the query heads that share a key head sit in the same
// tile, so grouped heads read each key tile once and a single token fills `group` rows.
//
// m is lowered lazily: o and l are rescaled only where the maximum grew by more than 2^kRescaleLog2 in p's units; until
// then p may exceed 1 by up to that factor, which fp32 sums, bf16 p and fp16 p all hold.  The result is the same
// quotient; the O read-modify-write disappears from nearly every tile.
//
// p is rounded to the inputs' 16-bit type (a tcgen05 product takes both operands in one type; error 2^-9 or 2^-12
// relative per weight, the same as the output's own rounding); l sums the unrounded p.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <type_traits>

#include "ptx.cuh"
#include "qk_rope.cuh"

namespace convrot {

constexpr int kAtTile = 128;
constexpr int kAtThreads = 384;
constexpr int kAtPanelBytes = 128 * 128;  // 128 rows x 64 channels of 16 bits, 128-byte swizzled rows
constexpr float kRescaleLog2 = 8.0f;

template <int NP>
struct AttnCfg {  // NP: 64-channel panels of a head (1: D <= 64, 2: D <= 128)
  static constexpr int kTileBytes = NP * kAtPanelBytes;
  static constexpr int kStages = NP == 2 ? 5 : 8;
  static constexpr int kNumBars = 2 * kStages + 2 + 2 + 2 + 4 + 2 + 3;
  static constexpr int kSmemBytes = (2 + kStages) * kTileBytes + 8 * kNumBars + 16 + 1024;
  static constexpr int kO = 256;  // first TMEM column of O0; O1 follows NP * 64 columns later
};

struct AttnParams {
  const int32_t* cu_q;  // [batch + 1] or null (one sequence)
  const int32_t* cu_k;
  int batch, Tq, Tk;
  int heads_kv, group, D;
  int positions;  // query positions in a 128-row tile: 128 / group
  float scale_log2;
  int causal;
  void* out;
  int64_t out_t, out_h;
  float* lse;  // [Tq, heads] or null
  // Split keys: sequence b's tiles are divided into ceil(tiles / chunk_tiles) parts, at most max_splits; each part
  // writes its normalised rows and their log2-sum-exp, joined by attention_combine_kernel.
  int max_splits, chunk_tiles;
  float* part_o;    // [max_splits, Tq, heads, D]
  float* part_lse;  // [max_splits, Tq, heads]
  uint64_t wait_limit_ns;
  int* error_word;
};

// ------------------------------------------------------------------------------------------------ work items

struct AttnItem {
  int q0, lq, k0, lk;  // the sequence's rows
  int head;            // key head
  int pos;             // first query position of the item (two tiles of `positions`)
  int split, t_lo, t_hi;  // key tiles [t_lo, t_hi) of this split
};

__device__ __forceinline__ void attn_bounds(const int32_t* cu, int b, int total, int& begin, int& len) {
  if (!cu) {
    begin = 0;
    len = total;
    return;
  }
  // clamped, so that no content of the array can lead outside the tensors
  const int lo = min(max(__ldg(cu + b), 0), total);
  begin = lo;
  len = min(max(__ldg(cu + b + 1), lo), total) - lo;
}

__device__ __forceinline__ int attn_splits(const AttnParams& p, int lk) {
  if (p.max_splits <= 1) return 1;
  const int tiles = (lk + kAtTile - 1) / kAtTile;
  return min(p.max_splits, max(1, (tiles + p.chunk_tiles - 1) / p.chunk_tiles));
}

// Finds items in increasing order; the whole warp calls next().  (base, b) is the first item and the index of the block
// of 32 sequences last looked at.
struct AttnWalk {
  int64_t base = 0;
  int block = 0;

  __device__ __forceinline__ bool find(const AttnParams& p, int64_t item, int lane, AttnItem& it) {
    const int span = 2 * p.positions;
    while (block < p.batch) {
      const int b = block + lane;
      int q0 = 0, lq = 0, k0 = 0, lk = 0;
      int64_t mine = 0;
      if (b < p.batch) {
        attn_bounds(p.cu_q, b, p.Tq, q0, lq);
        attn_bounds(p.cu_k, b, p.Tk, k0, lk);
        mine = static_cast<int64_t>((lq + span - 1) / span) * attn_splits(p, lk) * p.heads_kv;
      }
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const int64_t rel = item - base;
      const uint32_t after = __ballot_sync(0xffffffffu, rel < upto);
      if (!after) {
        base += __shfl_sync(0xffffffffu, upto, 31);
        block += 32;
        continue;
      }
      const int src = __ffs(after) - 1;
      it.q0 = __shfl_sync(0xffffffffu, q0, src);
      it.lq = __shfl_sync(0xffffffffu, lq, src);
      it.k0 = __shfl_sync(0xffffffffu, k0, src);
      it.lk = __shfl_sync(0xffffffffu, lk, src);
      const int local = static_cast<int>(rel - __shfl_sync(0xffffffffu, upto - mine, src));
      const int ns = attn_splits(p, it.lk);
      const int nq = (it.lq + span - 1) / span;
      const int per_head = ns * nq;
      it.head = local / per_head;
      const int in_head = local - it.head * per_head;
      int qt = in_head / ns;
      it.split = in_head - qt * ns;
      if (p.causal) qt = nq - 1 - qt;  // the longest first
      it.pos = qt * span;
      const int tiles = (it.lk + kAtTile - 1) / kAtTile;
      const int per = (tiles + ns - 1) / ns;
      it.t_lo = min(it.split * per, tiles);
      it.t_hi = min(it.t_lo + per, tiles);
      return true;
    }
    return false;
  }
};

// Keys that the last position of query tile i sees, and the key tiles of this split that it needs.
__device__ __forceinline__ int attn_tiles(const AttnParams& p, const AttnItem& it, int i) {
  const int first = it.pos + i * p.positions;
  if (first >= it.lq) return 0;
  const int last = min(first + p.positions, it.lq) - 1;
  const int limit = p.causal ? min(it.lk, last + it.lk - it.lq + 1) : it.lk;
  const int tiles = limit <= 0 ? 0 : (limit + kAtTile - 1) / kAtTile;
  return max(0, min(tiles, it.t_hi) - it.t_lo);
}

// ------------------------------------------------------------------------------------------------ small wrappers

template <int N>
__device__ __forceinline__ void setmaxnreg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void setmaxnreg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// D[tmem] (+)= A[tmem] . B[smem desc]: A's rows are TMEM lanes, two 16-bit elements to a column.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Descriptor of an operand whose N (or M) dimension is contiguous: 64-element 128-byte swizzled rows, one row per K
// index; eight K rows are 1024 bytes (stride byte offset), the next 64 elements of N are `panel_bytes` further (leading
// byte offset).
__device__ __forceinline__ uint64_t make_nmajor_desc(uint32_t smem_addr, uint32_t panel_bytes) {
  return (static_cast<uint64_t>(smem_addr >> 4) & 0x3fffull) | (static_cast<uint64_t>(panel_bytes >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor of kind::f16 with an fp32 accumulator; both operands bf16 or both fp16.
__device__ __forceinline__ uint32_t make_idesc_f16(bool bf16, int M, int N, bool b_nmajor) {
  const uint32_t t = bf16 ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | (b_nmajor ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------------------------------------ the kernel

template <class T, int NP>
__global__ void __launch_bounds__(kAtThreads, 1)
    attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                     const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ AttnParams p) {
  using Cfg = AttnCfg<NP>;
  constexpr int S = Cfg::kStages;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t attn_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(attn_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;                         // two query tiles
  uint8_t* ring = smem + 2 * Cfg::kTileBytes;     // key and value tiles in turn
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(ring + S * Cfg::kTileBytes);
  uint64_t* kv_empty = kv_full + S;
  uint64_t* q_full = kv_empty + S;   // [2]
  uint64_t* q_empty = q_full + 2;    // [2]
  uint64_t* s_full = q_empty + 2;    // [2] scores of tile i are in TMEM (and every earlier product is done)
  uint64_t* p_full = s_full + 2;     // [2][2] halves of p of tile i are in TMEM
  uint64_t* o_full = p_full + 4;     // [2] tile i's last product of the item is done
  uint64_t* v_need = o_full + 2;     // a value tile with rows behind the sequence has arrived
  uint64_t* v_fixed = v_need + 1;    // and those rows are cleared
  uint64_t* drain = v_fixed + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(kv_full + Cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(v_need, 1);
    mbar_init(v_fixed, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 8) {
    tmem_alloc<512>(tmem_holder);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const uint64_t limit = p.wait_limit_ns;
  auto fail = [&]() {
    *abort_flag = 1;
    if (p.error_word) atomicCAS(p.error_word, 0, 6 /* CONVROT_ERR_TIMEOUT */);
  };
  AttnWalk walk;
  AttnItem it;

  if (warp >= 8) {
    setmaxnreg_dec<56>();
    if (warp == 9) {
      // -------------------------------------------------------------- TMA producer
      uint32_t stage = 0, phase = 0, issued_mask = 0, issued_parity = 0;
      uint32_t q_count[2] = {0, 0};
      bool ok = true;
      for (int64_t item = blockIdx.x; ok && walk.find(p, item, lane, it); item += gridDim.x) {
        const int n0 = attn_tiles(p, it, 0), n1 = attn_tiles(p, it, 1);
        const int n = max(n0, n1);
        if (lane == 0) {
          auto load_q = [&](int i) {
            if (!mbar_wait_bounded(&q_empty[i], (q_count[i] & 1) ^ 1, limit, abort_flag)) return false;
            mbar_arrive_expect_tx(&q_full[i], NP * 128 * p.positions * p.group);
            for (int c = 0; c < NP; ++c)
              tma_load_3d(q_smem + i * Cfg::kTileBytes + c * kAtPanelBytes, &tmap_q, &q_full[i], c * 64,
                          it.head * p.group, it.q0 + it.pos + i * p.positions);
            ++q_count[i];
            return true;
          };
          auto load_kv = [&](const CUtensorMap* map, int tile) {
            if (!mbar_wait_bounded(&kv_empty[stage], phase ^ 1, limit, abort_flag)) return false;
            mbar_arrive_expect_tx(&kv_full[stage], Cfg::kTileBytes);
            for (int c = 0; c < NP; ++c)
              tma_load_3d(ring + stage * Cfg::kTileBytes + c * kAtPanelBytes, map, &kv_full[stage], c * 64, it.head,
                          it.k0 + tile * kAtTile);
            issued_mask |= 1u << stage;
            issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
            if (++stage == S) {
              stage = 0;
              phase ^= 1;
            }
            return true;
          };
          if (n0 > 0) ok = load_q(0);
          for (int j = 0; ok && j < n; ++j) {
            ok = load_kv(&tmap_k, it.t_lo + j);
            if (ok && j == 0 && n1 > 0) ok = load_q(1);
            if (ok) ok = load_kv(&tmap_v, it.t_lo + j);
          }
          if (!ok) fail();
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      }
      if (!ok && lane == 0) {  // let every load this thread issued land before the CTA leaves
        volatile int never = 0;
        for (int s = 0; s < S; ++s)
          if (issued_mask >> s & 1) mbar_wait_bounded(&kv_full[s], issued_parity >> s & 1, limit, &never);
        for (int i = 0; i < 2; ++i)
          if (q_count[i]) mbar_wait_bounded(&q_full[i], (q_count[i] - 1) & 1, limit, &never);
      }
    } else if (warp == 8) {
      // -------------------------------------------------------------- MMA issuer
      const uint32_t idesc_qk = make_idesc_f16(kBf16, 128, 128, false);
      const int n_pv = (p.D + 15) / 16 * 16;
      const uint32_t idesc_pv = make_idesc_f16(kBf16, 128, n_pv, true);
      const int ksteps = (p.D + 15) / 16;
      const uint32_t q_base = smem_u32(q_smem), ring_base = smem_u32(ring);
      uint32_t slot = 0, slot_phase = 0;  // next ring slot to be consumed
      uint32_t q_count[2] = {0, 0}, p_count[2] = {0, 0}, fixes = 0;
      bool ok = true;
      for (int64_t item = blockIdx.x; ok && walk.find(p, item, lane, it); item += gridDim.x) {
        const int nt[2] = {attn_tiles(p, it, 0), attn_tiles(p, it, 1)};
        const int n = max(nt[0], nt[1]);
        if (lane == 0 && n > 0) {
          auto take = [&](uint32_t& s, uint32_t& ph) {  // the next ring slot, in load order
            s = slot;
            ph = slot_phase;
            if (++slot == S) {
              slot = 0;
              slot_phase ^= 1;
            }
          };
          auto qk = [&](int i, uint32_t s) {  // S_i = Q_i K^T
            const uint64_t a0 = make_kmajor_desc(q_base + i * Cfg::kTileBytes, 128);
            const uint64_t b0 = make_kmajor_desc(ring_base + s * Cfg::kTileBytes, 128);
            for (int k = 0; k < ksteps; ++k) {
              const uint32_t off = ((k >> 2) * kAtPanelBytes + (k & 3) * 32) >> 4;
              mma_f16(tmem + i * 128, a0 + off, b0 + off, idesc_qk, k > 0);
            }
            mma_commit(&s_full[i]);
          };
          uint32_t ks, kph, vs, vph;
          take(ks, kph);
          ok = mbar_wait_bounded(&kv_full[ks], kph, limit, abort_flag);
          for (int i = 0; ok && i < 2; ++i) {
            if (nt[i] == 0) continue;
            if (!(ok = mbar_wait_bounded(&q_full[i], q_count[i] & 1, limit, abort_flag))) break;
            ++q_count[i];
            tc_fence_after();
            qk(i, ks);
            if (nt[i] == 1) mma_commit(&q_empty[i]);
          }
          if (ok) mma_commit(&kv_empty[ks]);
          for (int j = 0; ok && j < n; ++j) {
            take(vs, vph);
            if (!(ok = mbar_wait_bounded(&kv_full[vs], vph, limit, abort_flag))) break;
            // cleared by warp 10 while the softmax still works on this tile
            bool fixing = (it.t_lo + j + 1) * kAtTile > it.lk && it.k0 + it.lk < p.Tk;
            if (fixing) mbar_arrive(v_need);
            bool have_k = false;
            if (j + 1 < n) take(ks, kph);
            for (int i = 0; ok && i < 2; ++i) {
              if (j >= nt[i]) continue;
              const uint64_t b0 = make_nmajor_desc(ring_base + vs * Cfg::kTileBytes, kAtPanelBytes);
              const uint32_t d = tmem + Cfg::kO + i * (NP * 64);
              for (int h = 0; ok && h < 2; ++h) {
                if (!(ok = mbar_wait_bounded(&p_full[2 * i + h], p_count[i] & 1, limit, abort_flag))) break;
                if (fixing) {
                  if (!(ok = mbar_wait_bounded(v_fixed, fixes & 1, limit, abort_flag))) break;
                  fixing = false;
                  ++fixes;
                }
                tc_fence_after();
#pragma unroll
                for (int k = 4 * h; k < 4 * h + 4; ++k)
                  mma_f16_ts(d, tmem + i * 128 + k * 8, b0 + ((k * 16 * 128) >> 4), idesc_pv, j > 0 || k > 0);
              }
              if (!ok) break;
              ++p_count[i];
              if (j + 1 == nt[i]) {
                mma_commit(&o_full[i]);
              } else {
                if (!have_k) {
                  if (!(ok = mbar_wait_bounded(&kv_full[ks], kph, limit, abort_flag))) break;
                  have_k = true;
                  tc_fence_after();
                }
                qk(i, ks);
                if (j + 2 == nt[i]) mma_commit(&q_empty[i]);
              }
            }
            if (!ok) break;
            mma_commit(&kv_empty[vs]);
            if (j + 1 < n) mma_commit(&kv_empty[ks]);
          }
          if (!ok) fail();
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      }
      if (!ok && lane == 0) {  // the products still in flight read shared memory and TMEM
        volatile int never = 0;
        mma_commit(drain);
        mbar_wait_bounded(drain, 0, limit, &never);
      }
    } else if (warp == 10) {
      // -------------------------------------------------------------- value rows behind a sequence's end
      // Their weights are exactly zero, but 0 * NaN is not: another request's rows must not reach this one.  (Rows
      // behind the tensor's end are zeros that TMA filled in.)
      uint32_t slot = 0, fixes = 0;
      bool ok = true;
      for (int64_t item = blockIdx.x; ok && walk.find(p, item, lane, it); item += gridDim.x) {
        const int n = max(attn_tiles(p, it, 0), attn_tiles(p, it, 1));
        if (n == 0) continue;
        const int rows = it.lk - (it.t_lo + n - 1) * kAtTile;
        const uint32_t at = (slot + 2 * n - 1) % S;  // the item's last value tile
        slot = (slot + 2 * n) % S;
        if (rows >= kAtTile || it.k0 + it.lk >= p.Tk) continue;
        ok = mbar_wait_bounded(v_need, fixes & 1, limit, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++fixes;
        for (int c = 0; c < NP; ++c)
          for (int r = rows * 8 + lane; r < kAtTile * 8; r += 32)
            *reinterpret_cast<uint4*>(ring + at * Cfg::kTileBytes + c * kAtPanelBytes + r * 16) =
                make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_fixed);
      }
      if (!ok && lane == 0) fail();
    }
  } else {
    // ---------------------------------------------------------------- softmax and output of tile i
    setmaxnreg_inc<224>();
    const int i = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + i * 128;
    const uint32_t o_addr = tmem + lanes + Cfg::kO + i * (NP * 64);
    const int row_pos = row / p.group, row_head = row - row_pos * p.group;
    const float c2 = p.scale_log2;
    uint32_t count = 0, items = 0;
    bool ok = true;
    for (int64_t item = blockIdx.x; ok && walk.find(p, item, lane, it); item += gridDim.x) {
      const int n = attn_tiles(p, it, i);
      const int pos = it.pos + i * p.positions + row_pos;
      const bool valid = row_pos < p.positions && pos < it.lq;
      const int keys = !valid ? 0 : (p.causal ? min(it.lk, pos + it.lk - it.lq + 1) : it.lk);
      const bool warp_valid = __any_sync(0xffffffffu, valid);
      // tiles before this one need no mask in any row of the warp
      const int full = __reduce_min_sync(0xffffffffu, valid ? max(keys, 0) : 0x7fffffff) / kAtTile;
      float m = -CUDART_INF_F, l = 0.0f;
      for (int j = 0; j < n; ++j, ++count) {
        ok = mbar_wait_bounded(&s_full[i], count & 1, limit, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (!warp_valid) {
          if (lane == 0) {
            mbar_arrive(&p_full[2 * i]);
            mbar_arrive(&p_full[2 * i + 1]);
          }
          continue;
        }
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_addr + c * 32, s[c]);
        tmem_ld_wait();
        if (it.t_lo + j >= full) {
          const int seen = keys - (it.t_lo + j) * kAtTile;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e >= seen) s[c][e] = 0xff800000u;
        }
        float mx[4] = {m, m, m, m};
#pragma unroll
        for (int e = 0; e < 32; ++e)
#pragma unroll
          for (int c = 0; c < 4; ++c) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][e]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool grow = m == -CUDART_INF_F ? top != m : (top - m) * c2 > kRescaleLog2;
        if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? (m == -CUDART_INF_F ? 0.0f : exp2_approx((m - top) * c2)) : 1.0f;
          if (grow) m = top;
          l *= f;
          if (j > 0) {  // s_full also says that the products into O so far are done
#pragma unroll 1
            for (int c = 0; c < 2 * NP; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(o_addr + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st_32x32b_x32(o_addr + c * 32, o);
            }
          }
        }
        const float neg = m == -CUDART_INF_F ? 0.0f : -m * c2;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float a = exp2_approx(fmaf(__uint_as_float(s[2 * h + e / 16][(2 * e) % 32]), c2, neg));
            const float b = exp2_approx(fmaf(__uint_as_float(s[2 * h + e / 16][(2 * e) % 32 + 1]), c2, neg));
            sum[(e & 1) * 2] += a;
            sum[(e & 1) * 2 + 1] += b;
            pk[e] = Pack16<T>::pack(a, b);
          }
          tmem_st_32x32b_x32(s_addr + h * 32, pk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * i + h]);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
      if (!ok) break;
      // ------------------------------------------------------------ the item's rows
      if (n > 0) {
        ok = mbar_wait_bounded(&o_full[i], items & 1, limit, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++items;
        tc_fence_after();
      }
      if (!warp_valid) continue;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a row that sees no key gives zeros
      const int64_t t = it.q0 + pos;
      const int head = it.head * p.group + row_head;
      const int heads = p.heads_kv * p.group;
      const bool parts = p.max_splits > 1;
      const int64_t part = ((static_cast<int64_t>(it.split) * p.Tq + t) * heads + head);
#pragma unroll
      for (int c = 0; c < 2 * NP; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(o_addr + c * 32, o);
          tmem_ld_wait();
        }
        if (valid) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            const int col = c * 32 + e;
            if (col < p.D) {
              float f[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) f[k] = n > 0 && inv != 0.0f ? __uint_as_float(o[e + k]) * inv : 0.0f;
              if (parts) {
                float4* dst = reinterpret_cast<float4*>(p.part_o + part * p.D + col);
                dst[0] = make_float4(f[0], f[1], f[2], f[3]);
                dst[1] = make_float4(f[4], f[5], f[6], f[7]);
              } else {
                uint4 u;
                u.x = Pack16<T>::pack(f[0], f[1]);
                u.y = Pack16<T>::pack(f[2], f[3]);
                u.z = Pack16<T>::pack(f[4], f[5]);
                u.w = Pack16<T>::pack(f[6], f[7]);
                *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + t * p.out_t + head * p.out_h + col) = u;
              }
            }
          }
        }
      }
      if (valid) {
        const float lse2 = l == 0.0f ? -CUDART_INF_F : fmaf(m, c2, log2f(l));
        if (parts)
          p.part_lse[part] = lse2;
        else if (p.lse)
          p.lse[t * heads + head] = lse2 * 0.69314718055994530942f;
      }
    }
    if (!ok && lane == 0) fail();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc<512>(tmem);
  }
}

// Joins the key splits: o = sum_s w_s o_s with w_s = 2^(lse_s - m) / sum 2^(lse_s - m), in split order.  One warp for
// each row of out; the partial rows were just written and mostly come from L2.
template <class T>
__global__ void __launch_bounds__(256) attention_combine_kernel(const __grid_constant__ AttnParams p) {
  const int heads = p.heads_kv * p.group;
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(p.Tq) * heads;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (r >= rows) return;
  const int t = static_cast<int>(r / heads);
  const int head = static_cast<int>(r - static_cast<int64_t>(t) * heads);
  int q0 = 0, lq = p.Tq, k0 = 0, lk = p.Tk;
  if (p.cu_q) {  // the last sequence that starts at or before t (offsets do not decrease)
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.cu_q + mid) <= t)
        lo = mid;
      else
        hi = mid;
    }
    attn_bounds(p.cu_q, lo, p.Tq, q0, lq);
    attn_bounds(p.cu_k, lo, p.Tk, k0, lk);
    if (t < q0 || t >= q0 + lq) return;  // a row of no sequence stays as it was
  }
  const int ns = attn_splits(p, lk);
  float m = -CUDART_INF_F;
  for (int s = lane; s < ns; s += 32) m = fmaxf(m, p.part_lse[s * rows + r]);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const int c = lane * 4;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float total = 0.0f;
  for (int s = 0; s < ns; ++s) {
    const float z = p.part_lse[s * rows + r];
    if (z == -CUDART_INF_F) continue;
    const float w = exp2f(z - m);
    total += w;
    if (c < p.D) {
      const float4 f = *reinterpret_cast<const float4*>(p.part_o + (s * rows + r) * p.D + c);
      acc.x = fmaf(w, f.x, acc.x), acc.y = fmaf(w, f.y, acc.y), acc.z = fmaf(w, f.z, acc.z), acc.w = fmaf(w, f.w, acc.w);
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if (c < p.D)
    *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + t * p.out_t + head * p.out_h + c) =
        make_uint2(Pack16<T>::pack(acc.x * inv, acc.y * inv), Pack16<T>::pack(acc.z * inv, acc.w * inv));
  if (p.lse && lane == 0) p.lse[r] = total == 0.0f ? -CUDART_INF_F : (m + log2f(total)) * 0.69314718055994530942f;
}

}  // namespace convrot
