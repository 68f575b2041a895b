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
constexpr int kFirstSteps = 6;  // 16-key steps of a tile's weights that are handed over before the rest
constexpr int kPolyEvery = 1000;  // one of so many pairs of weights takes exp2_poly instead of the special-function unit

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
  int base = 0;
  int block = 0;

  __device__ __forceinline__ bool find(const AttnParams& p, int item, int lane, AttnItem& it) {
    const int span = 2 * p.positions;
    while (block < p.batch) {
      const int b = block + lane;
      int q0 = 0, lq = 0, k0 = 0, lk = 0;
      int mine = 0;
      if (b < p.batch) {
        attn_bounds(p.cu_q, b, p.Tq, q0, lq);
        attn_bounds(p.cu_k, b, p.Tk, k0, lk);
        mine = (lq + span - 1) / span * attn_splits(p, lk) * p.heads_kv;
      }
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const int rel = item - base;
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
      const int local = rel - __shfl_sync(0xffffffffu, upto - mine, src);
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

// A value that is the same in every lane, as one the compiler may keep in a uniform register and branch on without
// divergence.  The tcgen05 descriptors and addresses have to be in uniform registers: from ordinary ones, each 64-cycle
// product took about 140 cycles to issue.
template <class V>
__device__ __forceinline__ V uniform(V v) {
  return __shfl_sync(0xffffffffu, v, 0);
}

// Waits for a phase of the mbarrier at a shared address, without a result: past the time limit it raises the abort flag
// (and the device error word) and returns, and later waits return soon after, so that every loop below runs to its end on
// whatever data there is and only the TMA producer, which must not pile up loads, looks at the flag.  A result would
// have to be voted on by the issuing warp at every step; that vote and a first look at %globaltimer cost the MMA warp
// more than the wait itself.
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {  // without suspending the thread
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

struct AttnGuard {
  volatile int* abort;
  uint64_t limit_ns;
  int* error_word;

  __device__ __forceinline__ void wait(uint32_t bar, uint32_t parity) const {
    if (bar_try(bar, parity)) return;
    slow(bar, parity);
  }
  // Polls for a while before it lets the hardware suspend the thread, which takes longer to wake (1.3 % of the time of
  // 8192 x 40 heads).
  __device__ __forceinline__ void poll(uint32_t bar, uint32_t parity) const {
    for (int i = 0; i < 64; ++i)
      if (bar_test(bar, parity)) return;
    wait(bar, parity);
  }
  // Two barriers that are usually ready: their latencies overlap.
  __device__ __forceinline__ void both(uint32_t a, uint32_t a_parity, uint32_t b, uint32_t b_parity) const {
    const bool x = bar_test(a, a_parity), y = bar_test(b, b_parity);
    if (x && y) return;
    wait(a, a_parity);
    wait(b, b_parity);
  }
  __device__ __forceinline__ void slow(uint32_t bar, uint32_t parity) const {
    uint64_t since = 0;
    for (uint32_t spin = 1; !bar_try(bar, parity); ++spin) {
      if (spin & 127) continue;
      if (*abort) return;
      const uint64_t now = globaltimer_ns();
      if (since == 0) since = now;
      if (now - since > limit_ns) {
        *abort = 1;
        if (error_word) atomicCAS(error_word, 0, 6 /* CONVROT_ERR_TIMEOUT */);
        return;
      }
    }
  }
};

__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void bar_commit(uint32_t bar) {  // mma_commit by shared address
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one of them is
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Two fp32 lanes in a 64-bit register (one issue slot for both).
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 2^x of two lanes on the FMA pipe: x = n + f with n = rint(x) (by adding and subtracting 1.5 * 2^23, which leaves n in
// the low bits of the sum) and |f| <= 1/2, 2^f = 1 + f q(f) with a cubic q fitted to the smallest largest relative error
// (2.9e-6, far below the 16-bit rounding of the weights), and n added to the exponent.  x is below 2^7 and not NaN (a
// row with a NaN score has a NaN maximum, and the special-function lanes carry it); at -127 and below, -infinity
// included, the result is exactly 0.
__device__ __forceinline__ float2 exp2_poly(uint64_t x) {
  const float2 v = unpack2(x);
  const uint64_t xc = pack2(fmaxf(v.x, -127.0f), fmaxf(v.y, -127.0f));
  const uint64_t t = add2(xc, pack2(12582912.0f, 12582912.0f));
  const uint64_t n = add2(t, pack2(-12582912.0f, -12582912.0f));
  const uint64_t f = fma2(n, pack2(-1.0f, -1.0f), xc);
  uint64_t q = fma2(f, pack2(0.0095828531f, 0.0095828531f), pack2(0.055906427f, 0.055906427f));
  q = fma2(q, f, pack2(0.24024099f, 0.24024099f));
  q = fma2(q, f, pack2(0.69312419f, 0.69312419f));
  q = fma2(q, f, pack2(1.0f, 1.0f));
  const float2 y = unpack2(q), k = unpack2(t);
  return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(k.x) << 23)),
                     __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(k.y) << 23)));
}

// Weights 2^(c2 s + neg) of 32 scores, their sums (two lanes of two), and the weights in 16 bits.
template <class T>
__device__ __forceinline__ void weights(const uint32_t (&s)[32], float c2, float neg, uint64_t (&sum)[2],
                                        uint32_t (&pk)[16]) {
  const uint64_t scale2 = pack2(c2, c2), neg2 = pack2(neg, neg);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint64_t x = fma2(pack2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), scale2, neg2);
    float2 y;
    if (e % kPolyEvery == kPolyEvery - 1) {
      y = exp2_poly(x);
    } else {
      const float2 v = unpack2(x);
      y = make_float2(exp2_approx(v.x), exp2_approx(v.y));
    }
    sum[e & 1] = add2(sum[e & 1], pack2(y.x, y.y));
    pk[e] = Pack16<T>::pack(y.x, y.y);
  }
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
  uint8_t* q_smem = smem;                      // two query tiles
  uint8_t* ring = smem + 2 * Cfg::kTileBytes;  // key and value tiles in turn
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + S * Cfg::kTileBytes);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + Cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const uint32_t bar0 = smem_u32(bars);
  auto kv_full = [&](int s) { return bar0 + 8 * s; };
  auto kv_empty = [&](int s) { return bar0 + 8 * (S + s); };
  auto q_full = [&](int i) { return bar0 + 8 * (2 * S + i); };
  auto q_empty = [&](int i) { return bar0 + 8 * (2 * S + 2 + i); };
  auto s_full = [&](int i) { return bar0 + 8 * (2 * S + 4 + i); };  // scores of tile i (and all products before) done
  auto o_full = [&](int i) { return bar0 + 8 * (2 * S + 6 + i); };  // tile i's last product of the item done
  auto p_full = [&](int i, int part) { return bar0 + 8 * (2 * S + 8 + 2 * i + part); };  // weights of tile i in TMEM
  const uint32_t v_need = bar0 + 8 * (2 * S + 12);   // a value tile with rows behind the sequence has arrived
  const uint32_t v_fixed = bar0 + 8 * (2 * S + 13);  // and those rows are cleared
  const uint32_t drain = bar0 + 8 * (2 * S + 14);

  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int b = 0; b < Cfg::kNumBars; ++b) mbar_init(&bars[b], b >= 2 * S + 8 && b < 2 * S + 12 ? 4 : 1);
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
  const uint32_t tmem = uniform(*tmem_holder);
  const AttnGuard guard{abort_flag, p.wait_limit_ns, p.error_word};
  AttnWalk walk;
  AttnItem it;

  if (warp >= 8) {
    setmaxnreg_dec<72>();
    if (warp == 9) {
      // -------------------------------------------------------------- TMA producer
      uint32_t stage = 0, phase = 0, issued_mask = 0, issued_parity = 0;
      uint32_t q_count[2] = {0, 0};
      bool stop = false;
      for (int item = blockIdx.x; !stop && walk.find(p, item, lane, it); item += gridDim.x) {
        const int n0 = attn_tiles(p, it, 0), n1 = attn_tiles(p, it, 1);
        const int n = max(n0, n1);
        if (lane == 0) {
          auto load_q = [&](int i) {
            guard.wait(q_empty(i), (q_count[i] & 1) ^ 1);
            if ((stop = *abort_flag != 0)) return;
            uint64_t* full = bars + 2 * S + i;
            mbar_arrive_expect_tx(full, NP * 128 * p.positions * p.group);
            for (int c = 0; c < NP; ++c)
              tma_load_3d(q_smem + i * Cfg::kTileBytes + c * kAtPanelBytes, &tmap_q, full, c * 64, it.head * p.group,
                          it.q0 + it.pos + i * p.positions);
            ++q_count[i];
          };
          auto load_kv = [&](const CUtensorMap* map, int tile) {
            guard.wait(kv_empty(stage), phase ^ 1);
            if ((stop = *abort_flag != 0)) return;
            uint64_t* full = bars + stage;
            mbar_arrive_expect_tx(full, Cfg::kTileBytes);
            for (int c = 0; c < NP; ++c)
              tma_load_3d(ring + stage * Cfg::kTileBytes + c * kAtPanelBytes, map, full, c * 64, it.head,
                          it.k0 + tile * kAtTile);
            issued_mask |= 1u << stage;
            issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
            if (++stage == S) {
              stage = 0;
              phase ^= 1;
            }
          };
          if (n0 > 0) load_q(0);
          for (int j = 0; !stop && j < n; ++j) {
            load_kv(&tmap_k, it.t_lo + j);
            if (!stop && j == 0 && n1 > 0) load_q(1);
            if (!stop) load_kv(&tmap_v, it.t_lo + j);
          }
        }
        stop = uniform(stop ? 1 : 0) != 0;
      }
      if (stop && lane == 0) {  // let every load this thread issued land before the CTA leaves
        volatile int never = 0;
        for (int s = 0; s < S; ++s)
          if (issued_mask >> s & 1) mbar_wait_bounded(bars + s, issued_parity >> s & 1, p.wait_limit_ns, &never);
        for (int i = 0; i < 2; ++i)
          if (q_count[i]) mbar_wait_bounded(bars + 2 * S + i, (q_count[i] - 1) & 1, p.wait_limit_ns, &never);
      }
    } else if (warp == 8) {
      // -------------------------------------------------------------- MMA issuer
      // The whole warp walks the loop and one elected lane issues, in fully unrolled runs that end with their commits:
      // under a branch on the lane number the descriptors cannot live in uniform registers, and each of the 64-cycle
      // products then took over 100 cycles to issue.
      const uint32_t idesc_qk = make_idesc_f16(kBf16, 128, 128, false);
      const uint32_t idesc_pv = make_idesc_f16(kBf16, 128, (p.D + 15) / 16 * 16, true);
      const int ksteps = (p.D + 15) / 16;
      const uint64_t q_desc = make_kmajor_desc(smem_u32(q_smem), 128);
      const uint64_t k_desc = make_kmajor_desc(smem_u32(ring), 128);
      const uint64_t v_desc = make_nmajor_desc(smem_u32(ring), kAtPanelBytes);
      constexpr uint32_t kTileStep = Cfg::kTileBytes >> 4;
      uint32_t slot = 0, slot_phase = 0;  // next ring slot to be consumed
      uint32_t q_count[2] = {0, 0}, p_count[2] = {0, 0}, fixes = 0;
      auto take = [&](uint32_t& s, uint32_t& phase) {  // the next ring slot, in load order
        s = slot;
        phase = slot_phase;
        if (++slot == S) {
          slot = 0;
          slot_phase ^= 1;
        }
      };
      auto qk = [&](int i, uint32_t s) {  // S_i = Q_i K^T, by the elected lane
        const uint64_t a0 = q_desc + i * kTileStep, b0 = k_desc + s * kTileStep;
#pragma unroll
        for (int k = 0; k < 4 * NP; ++k) {
          const uint32_t off = ((k >> 2) * kAtPanelBytes + (k & 3) * 32) >> 4;
          if (k < ksteps) mma_f16(tmem + i * 128, a0 + off, b0 + off, idesc_qk, k > 0);
        }
        bar_commit(s_full(i));
      };
      for (int item = blockIdx.x; walk.find(p, item, lane, it); item += gridDim.x) {
        const int nt[2] = {uniform(attn_tiles(p, it, 0)), uniform(attn_tiles(p, it, 1))};
        const int n = max(nt[0], nt[1]);
        if (n == 0) continue;
        uint32_t ks = 0, kph = 0, vs = 0, vph = 0;
        take(ks, kph);
        guard.wait(kv_full(ks), kph);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (nt[i] > 0) {
            guard.wait(q_full(i), q_count[i] & 1);
            ++q_count[i];
          }
          tc_fence_after();
          if (elect_one()) {
            if (nt[i] > 0) qk(i, ks);
            if (nt[i] == 1) bar_commit(q_empty(i));
            if (i == 1) bar_commit(kv_empty(ks));
          }
          __syncwarp();
        }
        for (int j = 0; j < n; ++j) {
          take(vs, vph);
          if (j + 1 < n) {  // (the loads run ahead: neither wait lasts)
            take(ks, kph);
            guard.both(kv_full(vs), vph, kv_full(ks), kph);
          } else {
            guard.wait(kv_full(vs), vph);
          }
          // cleared by warp 10 while the softmax still works on this tile
          bool fixing = uniform((it.t_lo + j + 1) * kAtTile > it.lk && it.k0 + it.lk < p.Tk);
          if (fixing && lane == 0) bar_arrive(v_need);
          const uint64_t b0 = v_desc + vs * kTileStep;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t d = tmem + Cfg::kO + i * (NP * 64), a0 = tmem + i * 128;
            const bool works = j < nt[i], ends = j + 1 == nt[i];
            if (works) {
              guard.wait(p_full(i, 0), p_count[i] & 1);
              if (fixing) {
                guard.wait(v_fixed, fixes & 1);
                fixing = false;
                ++fixes;
              }
              tc_fence_after();
              if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kFirstSteps; ++k)
                  mma_f16_ts(d, a0 + k * 8, b0 + ((k * 16 * 128) >> 4), idesc_pv, k > 0 ? 1 : j > 0);
              }
              __syncwarp();
              guard.wait(p_full(i, 1), p_count[i] & 1);
              ++p_count[i];
              tc_fence_after();
            }
            if (elect_one()) {
              if (works) {
#pragma unroll
                for (int k = kFirstSteps; k < 8; ++k)
                  mma_f16_ts(d, a0 + k * 8, b0 + ((k * 16 * 128) >> 4), idesc_pv, 1);
                if (ends) {
                  bar_commit(o_full(i));
                } else {
                  qk(i, ks);
                  if (j + 2 == nt[i]) bar_commit(q_empty(i));
                }
              }
              if (i == 1) {  // both tiles are served
                bar_commit(kv_empty(vs));
                if (j + 1 < n) bar_commit(kv_empty(ks));
              }
            }
            __syncwarp();
          }
        }
      }
      if (*abort_flag) {  // the products still in flight read shared memory and TMEM
        volatile int never = 0;
        if (elect_one()) bar_commit(drain);
        __syncwarp();
        mbar_wait_bounded(bars + 2 * S + 14, 0, p.wait_limit_ns, &never);
      }
    } else if (warp == 10) {
      // -------------------------------------------------------------- value rows behind a sequence's end
      // Their weights are exactly zero, but 0 * NaN is not: another request's rows must not reach this one.  (Rows
      // behind the tensor's end are zeros that TMA filled in.)
      uint32_t slot = 0, fixes = 0;
      for (int item = blockIdx.x; walk.find(p, item, lane, it); item += gridDim.x) {
        const int n = max(attn_tiles(p, it, 0), attn_tiles(p, it, 1));
        if (n == 0) continue;
        const int rows = it.lk - (it.t_lo + n - 1) * kAtTile;
        const uint32_t at = (slot + 2 * n - 1) % S;  // the item's last value tile
        slot = (slot + 2 * n) % S;
        if (rows >= kAtTile || it.k0 + it.lk >= p.Tk) continue;
        guard.wait(v_need, fixes & 1);
        ++fixes;
        __syncwarp();
        for (int c = 0; c < NP; ++c)
          for (int r = rows * 8 + lane; r < kAtTile * 8; r += 32)
            *reinterpret_cast<uint4*>(ring + at * Cfg::kTileBytes + c * kAtPanelBytes + r * 16) =
                make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) bar_arrive(v_fixed);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax and output of tile i
    setmaxnreg_inc<216>();
    const int i = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + i * 128;
    const uint32_t o_addr = tmem + lanes + Cfg::kO + i * (NP * 64);
    const int row_pos = row / p.group, row_head = row - row_pos * p.group;
    const float c2 = p.scale_log2;
    uint32_t count = 0, items = 0;
    for (int item = blockIdx.x; walk.find(p, item, lane, it); item += gridDim.x) {
      const int n = uniform(attn_tiles(p, it, i));
      const int pos = it.pos + i * p.positions + row_pos;
      const bool valid = row_pos < p.positions && pos < it.lq;
      const int keys = !valid ? 0 : (p.causal ? min(it.lk, pos + it.lk - it.lq + 1) : it.lk);
      const bool warp_valid = __any_sync(0xffffffffu, valid);
      // tiles before this one need no mask in any row of the warp
      const int full = __reduce_min_sync(0xffffffffu, valid ? max(keys, 0) : 0x7fffffff) / kAtTile;
      float m = -CUDART_INF_F, l = 0.0f;
      for (int j = 0; j < n; ++j, ++count) {
        guard.poll(s_full(i), count & 1);
        __syncwarp();
        auto hand_over = [&](int part) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(p_full(i, part));
        };
        if (!warp_valid) {
          hand_over(0);
          hand_over(1);
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
        // The first half of the weights is taken with the maximum so far, while the tile's own maximum is still being
        // found: it seldom grows enough to matter, and then the half is taken again.  Finding the maximum first would
        // leave the special-function unit idle meanwhile.
        uint64_t sum[2];
        float neg;
#pragma unroll 1
        for (bool again = false;; again = true) {
          neg = m == -CUDART_INF_F ? 0.0f : -m * c2;
          sum[0] = sum[1] = 0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
            weights<T>(s[c], c2, neg, sum, pk);
            tmem_st_32x32b_x16(s_addr + c * 16, pk);
          }
          if (again) break;
          float mx[4] = {m, m, m, m};
#pragma unroll
          for (int e = 0; e < 32; e += 2)
#pragma unroll
            for (int c = 0; c < 4; ++c) mx[c] = max3(mx[c], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
          const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
          const bool grow = m == -CUDART_INF_F ? top != m : !((top - m) * c2 <= kRescaleLog2);
          if (!__any_sync(0xffffffffu, grow)) break;
          const float f = grow ? (m == -CUDART_INF_F ? 0.0f : exp2_approx((m - top) * c2)) : 1.0f;
          if (grow) m = fmaf(top, 0.0f, top);  // top, and NaN for +infinity: its weight is exp(inf - inf)
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
        if (kFirstSteps == 4) hand_over(0);
#pragma unroll
        for (int c = 2; c < 4; ++c) {
          uint32_t pk[16];
          weights<T>(s[c], c2, neg, sum, pk);
          tmem_st_32x32b_x16(s_addr + c * 16, pk);
          if (c == 2 && kFirstSteps == 6) hand_over(0);
        }
        hand_over(1);
        const float2 a = unpack2(add2(sum[0], sum[1]));
        l += a.x + a.y;
      }
      // ------------------------------------------------------------ the item's rows
      if (n > 0) {
        guard.wait(o_full(i), items & 1);
        ++items;
        __syncwarp();
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
