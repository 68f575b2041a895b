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
// Warp 10: looks over value tiles that a row sees in part.  Warp 11: finds the work.
//
// Rows of a query tile are (position, head of the group) pairs: the query heads that share a key head sit in the same
// tile, so grouped heads read each key tile once and a single token fills `group` rows.
//
// m is raised lazily: o and l are rescaled only where the maximum grew by more than 2^kRescaleLog2 in p's units; until
// then p may exceed 1 by up to that factor, which fp32 sums, bf16 p and fp16 p all hold.  The result is the same
// quotient; the O read-modify-write disappears from nearly every tile.
//
// p is rounded to the inputs' 16-bit type (a tcgen05 product takes both operands in one type; half a step relative per
// weight, the same as the output's own rounding); l sums the unrounded p.
//
// What bounds it.  A step of two 128 x 128 tiles at 128 channels needs 2048 cycles of the tensor pipe and as many of
// the special-function unit (2^15 exponentials at 16 a cycle); it takes about 3100, since the weights of a tile depend
// on its scores and the next scores go where the weights were: the two tiles cover each other's latency only in part.
// ncu on 8192 tokens x 18 heads: tensor pipe 67 % of active cycles, special-function unit 67 %.  32760 tokens x 5
// heads: 1.95 ms, 1410 TFLOP/s (causal 1.04 ms, 1320) in a burst; 1220 over seconds, where the 1000 W limit brings the
// clock to 1.5 GHz.  Single tokens over long caches: 5.7 TB/s of keys and values.  Short keys (333) pay 6000 to 8000
// cycles an item for its first tile, its output and the cold code of both, beside 9500 of steps: 283 us for 32760 x 40
// heads.  At 64 channels the exponentials alone are the floor: 8192 tokens x 40 heads 0.93 ms of 0.58.
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
constexpr uint64_t kDrainNs = 1000000000ull;  // for work of its own that a CTA that gave up has still in flight
constexpr float kRescaleLog2 = 8.0f;
constexpr int kFirstSteps = 6;  // 16-key steps of a tile's weights (three of four pieces) handed over before the rest

constexpr int kItems = 4;        // items on their way through the CTA
constexpr int kBadWords = 13;     // of an item: any, and a bit for each key of the (at most 3) tiles seen in part
constexpr int kMaxShares = 192;  // most CTAs that share the last items evenly

template <int NP>
struct AttnCfg {  // NP: 64-channel panels of a head (1: D <= 64, 2: D <= 128)
  static constexpr int kTileBytes = NP * kAtPanelBytes;
  static constexpr int kStages = NP == 2 ? 4 : 8;
  static constexpr int kStageOut = 4096;  // output staging of a warp: 32 rows of 128 bytes
  static constexpr int kNumBars = 2 * kStages + 19 + 3 * kItems;
  static constexpr int kSmallBytes =
      8 * kNumBars + kItems * 48 + 2 * 16 + 5 * kMaxShares + 4 + 16 + 4 * kItems * kBadWords;
  static constexpr int kSmemBytes = (2 + kStages) * kTileBytes + 8 * kStageOut + kSmallBytes + 1024;
  static constexpr int kO = 256;  // TMEM columns from S_i to O_i
};

struct AttnParams {
  const int32_t* cu_q;  // [batch + 1] or null (one sequence)
  const int32_t* cu_k;
  int batch, Tq, Tk;
  int heads_kv, group, D;
  int positions;      // query positions in a 128-row tile: 128 / group
  int group_inverse;  // 65536 / group, rounded up: exact for the quotient of a row below 128
  float scale_log2;
  int causal;
  int head_block;  // key heads whose items follow each other by query tile
  const void* v;  // (the kernel's loads go through the tensor maps)
  int64_t v_t, v_h;
  void* out;
  int64_t out_t, out_h;
  float* lse;  // [Tq, heads] or null
  // shares > 0: the items that do not fill a whole wave of `shares` CTAs are divided evenly by key tiles, and what is
  // not a whole item goes to part_o / part_lse, joined by attention_combine_kernel.
  int shares;
  int* meta;        // [kMaxShares + 4]: shares in use, items, first item, all work, prefix of the items' work
  float* part_o;    // [2 shares, 256, D] normalised rows
  float* part_lse;  // [2 shares, 256] log2-sum-exp
  uint64_t wait_limit_ns;
  int* error_word;
};

// ------------------------------------------------------------------------------------------------ work items
//
// An item is two neighbouring query tiles of one key head of one sequence, with all of its key tiles.  The grid has one
// CTA for each; a resident CTA's scheduler warp (11) finds its item in the offset arrays, hands it to the other warps
// through shared memory, and then takes over the next CTA that has not been launched (cluster launch control): dynamic
// balance without a counter in memory, no start-up between items, and the loads of the next item begin while the last
// tiles of this one are multiplied.  Causal items come longest first within a head.
//
// Where the last wave of items would leave SMs idle, its items are divided evenly (AttnParams::shares): share s of G
// gets the s-th G-th of their key tiles, whichever items these lie in.  32760 tokens x 5 heads are 640 items on 148
// SMs, 5 waves for 4.3 waves of work.
//
// An item of a single query tile (a sequence's last one, or a few new tokens over a long cache) uses both softmax
// groups all the same: tile 0 takes the even key tiles and tile 1 the odd ones, each with its own m, l and o, joined at
// the end ("twin").

struct AttnItem {
  int q_row, left;  // first row of q and out; query positions from there to the sequence's end
  int k_row, keys;  // first row of k and v; keys from there to the sequence's end
  int head;         // key head
  int see;          // keys from k_row that the first position sees (position r: r more, if causal)
  int nt[2];        // key tiles of each query tile
  int twin;         // tile 1 is tile 0 again
  int check;        // first key tile whose values have to be looked at (see warp 10)
  int part;         // slot of the partial result, or -1
  int valid;        // 0: no more work
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

// A sequence and an item's place in it.
struct AttnPlace {
  int q0, lq, k0, lk, head, pos;
};

// Key tiles that the query tile beginning at position `first` needs.
__device__ __forceinline__ int attn_tiles(const AttnParams& p, const AttnPlace& a, int first) {
  if (first >= a.lq) return 0;
  const int last = min(first + p.positions, a.lq) - 1;
  const int limit = p.causal ? min(a.lk, last + a.lk - a.lq + 1) : a.lk;
  return limit <= 0 ? 0 : (limit + kAtTile - 1) / kAtTile;
}

// An item's place from its number within its sequence.
__device__ __forceinline__ void attn_place(const AttnParams& p, int local, AttnPlace& a) {
  const int span = 2 * p.positions;
  const int nq = (a.lq + span - 1) / span;
  // blocks of `head_block` heads; in a block by query tile, and for each by head
  const int block = local / (nq * p.head_block), in_block = local - block * nq * p.head_block;
  const int heads = min(p.head_block, p.heads_kv - block * p.head_block);
  const int qt = heads == 1 ? in_block : in_block / heads;
  a.head = block * p.head_block + in_block - qt * heads;
  a.pos = (p.causal ? nq - 1 - qt : qt) * span;
}

// Work of an item in units of one 128 x 128 tile: a step of a pair of tiles counts two.  An item has at least 7: its first
// tile and its output take as long, and items that cannot be divided (AttnShares::snap) get a share each.
__device__ __forceinline__ int attn_unit(const AttnParams& p, const AttnPlace& a) {
  return a.lq - a.pos > p.positions ? 2 : 1;
}
__device__ __forceinline__ int attn_work(const AttnParams& p, const AttnPlace& a) {
  const int n = max(attn_tiles(p, a, a.pos), attn_tiles(p, a, a.pos + p.positions));
  return max(n * attn_unit(p, a), 7);
}

// Sum of v over the lanes up to this one.
__device__ __forceinline__ int attn_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Finds items by number; the whole warp calls find().  (base, block) is the number of the first item of the 32 sequences
// last looked at.
struct AttnWalk {
  int base = 0;
  int block = 0;

  __device__ __forceinline__ bool find(const AttnParams& p, int item, int lane, AttnPlace& a) {
    if (item < 0) return false;
    const int span = 2 * p.positions;
    if (!p.cu_q) {
      a.q0 = a.k0 = 0;
      a.lq = p.Tq;
      a.lk = p.Tk;
      if (item >= (p.Tq + span - 1) / span * p.heads_kv) return false;
      attn_place(p, item, a);
      return true;
    }
    if (item < base) base = block = 0;
    while (block < p.batch) {
      const int b = block + lane;
      int q0 = 0, lq = 0, k0 = 0, lk = 0;
      if (b < p.batch) {
        attn_bounds(p.cu_q, b, p.Tq, q0, lq);
        attn_bounds(p.cu_k, b, p.Tk, k0, lk);
      }
      const int mine = (lq + span - 1) / span * p.heads_kv, upto = attn_scan(mine, lane);
      const int rel = item - base;
      const uint32_t after = __ballot_sync(0xffffffffu, rel < upto);
      if (!after) {
        base += __shfl_sync(0xffffffffu, upto, 31);
        block += 32;
        continue;
      }
      const int src = __ffs(after) - 1;
      a.q0 = __shfl_sync(0xffffffffu, q0, src);
      a.lq = __shfl_sync(0xffffffffu, lq, src);
      a.k0 = __shfl_sync(0xffffffffu, k0, src);
      a.lk = __shfl_sync(0xffffffffu, lk, src);
      attn_place(p, rel - __shfl_sync(0xffffffffu, upto - mine, src), a);
      // (the items of sequences that overlap, which the arrays must not hold, can pass 32 bits)
      return a.pos >= 0 && a.pos < a.lq && a.head >= 0 && a.head < p.heads_kv;
    }
    return false;
  }
};

// All items of the call.
__device__ __forceinline__ int attn_count(const AttnParams& p, int lane) {
  const int span = 2 * p.positions;
  int n = 0;
  for (int b = lane; b < p.batch; b += 32) {
    int q0, lq;
    attn_bounds(p.cu_q, b, p.Tq, q0, lq);
    n += (lq + span - 1) / span;
  }
  return __reduce_add_sync(0xffffffffu, n) * p.heads_kv;
}

// Even division of the last items.  pre[x] is the work before item x of them (`items` of them, `total` in all) and
// units[x] the work of one of its steps; share s of `shares` begins at edge(s): at a whole step of the item that it falls
// into, or at that item's edge if little would be cut off.
struct AttnShares {
  int* pre;
  uint8_t* units;
  int items, total, shares;

  // Fills pre and units for the items from number `first` on (the whole warp).
  __device__ __forceinline__ void divide(const AttnParams& p, const AttnWalk& walk, int first, int lane) {
    const int span = 2 * p.positions;
    total = 0;
    if (lane == 0) pre[0] = 0;
#pragma unroll 1
    for (int k = 0; k < items; k += 32) {
      // a lane for each of 32 items, which looks its sequence up among 32 sequences at a time, held by a lane each
      const int number = first + k + lane;
      int base = walk.base, work = 0, unit = 1;
#pragma unroll 1
      for (int block = walk.block; block < p.batch && base < first + k + 32; block += 32) {
        AttnPlace mine = {};
        if (block + lane < p.batch) {
          attn_bounds(p.cu_q, block + lane, p.Tq, mine.q0, mine.lq);
          attn_bounds(p.cu_k, block + lane, p.Tk, mine.k0, mine.lk);
        }
        const int upto = attn_scan((mine.lq + span - 1) / span * p.heads_kv, lane);
        const int rel = number - base;
        int at = 0;  // sequences that end at or before the item
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const int v = __shfl_sync(0xffffffffu, upto, at + o - 1);
          if (v <= rel) at += o;
        }
        AttnPlace a;
        a.lq = __shfl_sync(0xffffffffu, mine.lq, at);
        a.lk = __shfl_sync(0xffffffffu, mine.lk, at);
        const int before = __shfl_sync(0xffffffffu, upto, max(at - 1, 0)), all = __shfl_sync(0xffffffffu, upto, 31);
        if (rel >= 0 && rel < all) {
          attn_place(p, rel - (at ? before : 0), a);
          work = attn_work(p, a);
          unit = attn_unit(p, a);
        }
        base += all;
      }
      work = k + lane < items ? work : 0;
      work = attn_scan(work, lane);
      if (k + lane < items) {
        pre[k + lane + 1] = total + work;
        units[k + lane] = static_cast<uint8_t>(unit);
      }
      total += __shfl_sync(0xffffffffu, work, 31);
    }
    __syncwarp();
    // A share of less than 8 units costs more than it saves, unless it is an item of its own.  (No two edges can fall on
    // one step: they are at least 7 units apart.)
    shares = max(1, min(p.shares, max(total / 8, items)));
  }
  __device__ __forceinline__ int item_at(int x, int lane) const {  // the item that work unit x < total lies in
    int n = 0;
#pragma unroll 1
    for (int i = 0; i < items; i += 32)
      n += __popc(__ballot_sync(0xffffffffu, i + lane < items && pre[i + lane + 1] <= x));
    return n;
  }
  __device__ __forceinline__ int snap(int x, int from, int upto, int unit) const {
    if (x - from < 4 || upto - x < 4) return x - from < upto - x ? from : upto;
    return from + (x - from + unit - 1) / unit * unit;
  }
  __device__ __forceinline__ int place(int s) const {  // before it is moved to a step
    const int q = total / shares;  // total * s / shares, without its 64-bit product
    return q * s + (total - q * shares) * s / shares;
  }
  __device__ __forceinline__ int edge(int s, int lane) const {
    if (s >= shares) return total;
    const int x = place(s), i = item_at(x, lane);
    return snap(x, pre[i], pre[i + 1], units[i]);
  }
};

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

// Waits for a phase of the mbarrier at a shared address, without a result: when no key or value tile was asked for within
// the time limit (an item may well take longer, and warps 10 and 11 wait for its last tiles) it raises the abort flag
// (and the device error word) and returns, and so does every later wait after two failed tries (about 2 us), so that every
// loop below runs to its end on whatever data there is, at a few microseconds a key tile, and only the TMA producer, which
// must not pile up loads, looks at the flag.  A result would have to be voted on by the issuing warp at every step; that
// vote and a first look at %globaltimer cost the MMA warp more than the wait itself, and a look at the flag at every 64th
// tile alone made 32760 tokens x 5 heads 1.6 % slower.
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
  uint32_t abort;  // shared address of the flag; behind it, the number of tiles asked for so far
  const AttnParams& p;

  __device__ __forceinline__ bool aborted() const {
    int v;
    asm volatile("ld.volatile.shared.s32 %0, [%1];" : "=r"(v) : "r"(abort) : "memory");
    return v != 0;
  }

  __device__ __forceinline__ void progress(uint32_t loads) const {
    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort + 4), "r"(loads) : "memory");
  }

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
    uint32_t seen = 0;
    while (!bar_try(bar, parity)) {
      if (aborted()) return;
      const uint64_t now = globaltimer_ns();
      uint32_t loads;
      asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(loads) : "r"(abort + 4) : "memory");
      if (since == 0 || loads != seen) {
        since = now;
        seen = loads;
      }
      if (now - since > p.wait_limit_ns) {
        asm volatile("st.volatile.shared.s32 [%0], 1;" ::"r"(abort) : "memory");
        if (p.error_word) atomicCAS(p.error_word, 0, 6 /* CONVROT_ERR_TIMEOUT */);
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

// Asks for the next CTA of the grid that has not been launched; the 16-byte answer arrives on `bar`.
__device__ __forceinline__ void launch_cancel(uint32_t answer, uint32_t bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer),
      "r"(bar)
      : "memory");
}

// blockIdx.x of the CTA that was taken over, or -1 if none is left.
__device__ __forceinline__ int launch_cancelled(uint32_t answer) {
  int got, x = -1;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.s32 %0, 1, 0, p;\n\t"
      "mov.s32 %1, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(answer)
      : "memory");
  return got ? x : -1;
}

// Weights 2^(c2 s + neg) of 32 scores, their sums (two lanes of two), and the weights in 16 bits.  All of them on the
// special-function unit: one in 2, 3, 4, 8 or 16 of them by a quartic on the FMA pipe shortened this step, but the
// kernel took 3 to 13 % longer at 128 channels (more issue slots beside the MMA warp, and a lower clock under the power
// limit) and gained nothing at 64.
template <class T>
__device__ __forceinline__ void weights(const uint32_t (&s)[32], float c2, float neg, uint64_t (&sum)[2],
                                        uint32_t (&pk)[16]) {
  const uint64_t scale2 = pack2(c2, c2), neg2 = pack2(neg, neg);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint64_t x = fma2(pack2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), scale2, neg2);
    const float2 v = unpack2(x);
    const float2 y = make_float2(exp2_approx(v.x), exp2_approx(v.y));
    sum[e & 1] = add2(sum[e & 1], pack2(y.x, y.y));
    pk[e] = Pack16<T>::pack(y.x, y.y);
  }
}

// ------------------------------------------------------------------------------------------------ the kernel

template <class T, int NP, bool CAUSAL>
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
  uint8_t* staging = ring + S * Cfg::kTileBytes;
  uint8_t* small = staging + 8 * Cfg::kStageOut;
  AttnItem* item_smem = reinterpret_cast<AttnItem*>(small);              // [kItems]
  const uint32_t answers = smem_u32(small + kItems * sizeof(AttnItem));       // [2] of launch control
  uint64_t* bars = reinterpret_cast<uint64_t*>(small + kItems * sizeof(AttnItem) + 32);
  int* pre = reinterpret_cast<int*>(bars + Cfg::kNumBars);
  uint8_t* units = reinterpret_cast<uint8_t*>(pre + kMaxShares + 1);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(units + kMaxShares);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  uint32_t* bad = tmem_holder + 4;
  const uint32_t bar0 = smem_u32(bars);
  auto kv_full = [&](int s) { return bar0 + 8 * s; };
  auto kv_empty = [&](int s) { return bar0 + 8 * (S + s); };
  auto q_full = [&](int i) { return bar0 + 8 * (2 * S + i); };
  auto q_empty = [&](int i) { return bar0 + 8 * (2 * S + 2 + i); };
  auto s_full = [&](int i) { return bar0 + 8 * (2 * S + 4 + i); };  // scores of tile i (and all products before) done
  auto o_full = [&](int i) { return bar0 + 8 * (2 * S + 6 + i); };  // tile i's last product of the item done
  auto p_full = [&](int i, int part) { return bar0 + 8 * (2 * S + 8 + 2 * i + part); };  // weights of tile i in TMEM
  const uint32_t v_need = bar0 + 8 * (2 * S + 12);      // a value tile with rows behind the sequence has arrived
  const uint32_t v_fixed = bar0 + 8 * (2 * S + 13);     // and those rows are cleared
  const uint32_t drain = bar0 + 8 * (2 * S + 14);
  const uint32_t twin_ready = bar0 + 8 * (2 * S + 15);  // tile 1's o is in TMEM, its m and l in shared memory
  const uint32_t twin_done = bar0 + 8 * (2 * S + 16);   // and was read
  auto answer_full = [&](int i) { return bar0 + 8 * (2 * S + 17 + i); };
  auto item_full = [&](int i) { return bar0 + 8 * (2 * S + 19 + i); };
  auto item_empty = [&](int i) { return bar0 + 8 * (2 * S + 19 + kItems + i); };
  auto want = [&](int i) { return bar0 + 8 * (2 * S + 19 + 2 * kItems + i); };  // the item's loads are all issued
  constexpr int kReaders = 11;                          // warps that read an item: all but the scheduler

  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int b = 0; b < Cfg::kNumBars; ++b) {
      const int c = b - 2 * S;
      const bool by_warps = (c >= 8 && c < 12) || c == 15 || c == 16, by_readers = c >= 19 + kItems && c < 19 + 2 * kItems;
      mbar_init(&bars[b], by_warps ? 4 : by_readers ? kReaders : 1);
    }
    abort_flag[0] = abort_flag[1] = 0;  // and the progress behind it
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
  grid_wait();  // what is above may run beside the end of the kernel before; nothing below may
  // (not before the kernel that joins the parts: its blocks would gather on the first SMs that are free)
  if (p.shares == 0) grid_release();
  const AttnGuard guard{smem_u32(const_cast<int*>(abort_flag)), p};

  // The next item, in every reading warp; false at the end of the work (or after a failed wait).  The warp is done with
  // the item's place in shared memory once it calls release().
  uint32_t item_count = 0;
  AttnItem* item = nullptr;
  auto next_item = [&]() {
    const int at = item_count % kItems;
    guard.wait(item_full(at), (item_count / kItems) & 1);
    item = item_smem + at;
    return uniform(item->valid) != 0 && !guard.aborted();
  };
  auto release = [&]() {
    __syncwarp();
    if (lane == 0) bar_arrive(item_empty(item_count % kItems));
    ++item_count;
  };
  AttnItem it;
  auto copy_item = [&]() {  // for the warps that need most of it
    const int4* src = reinterpret_cast<const int4*>(item);
    const int4 x = src[0], y = src[1], z = src[2];
    it.q_row = uniform(x.x), it.left = uniform(x.y), it.k_row = uniform(x.z), it.keys = uniform(x.w);
    it.head = uniform(y.x), it.see = uniform(y.y), it.nt[0] = uniform(y.z), it.nt[1] = uniform(y.w);
    it.twin = uniform(z.x), it.check = uniform(z.y), it.part = uniform(z.z), it.valid = uniform(z.w);
    release();
  };

  if (warp >= 8) {
    setmaxnreg_dec<56>();
    if (warp == 11) {
      // -------------------------------------------------------------- scheduler
      // (One call site for each piece of work: unrolled and called from several places this warp's code was 66 of the
      // kernel's 157 KB.)
      AttnWalk walk;
      AttnPlace a;
      const int items = attn_count(p, lane);
      const int whole = p.shares > 0 ? items / p.shares * p.shares : items;
      AttnShares sh{pre, units, items - whole, 0, 0};
      uint32_t sent = 0, asked = 0;
      bool brief = false;
      auto send = [&](const AttnItem& x) {
        const int at = sent % kItems;
        guard.wait(item_empty(at), ((sent / kItems) & 1) ^ 1);
        if (uniform(guard.aborted())) return;  // the place may still be read: rows of one item, limits of another
        if (lane == 0) {
          int4* dst = reinterpret_cast<int4*>(item_smem + at);
          dst[0] = make_int4(x.q_row, x.left, x.k_row, x.keys);
          dst[1] = make_int4(x.head, x.see, x.nt[0], x.nt[1]);
          dst[2] = make_int4(x.twin, x.check, x.part, x.valid);
          bar_arrive(item_full(at));  // releases the stores above
        }
        __syncwarp();
        ++sent;
      };
      int v = blockIdx.x;
#pragma unroll 1
      while (v >= 0) {
        const int s = v - whole;
        int x = 0, end = 1;  // a whole item, or the share [x, end) of the last ones
        if (s >= 0) {
          end = 0;
          if (s < p.shares) {
            if (sh.shares == 0) sh.divide(p, walk, whole, lane);
            if (s == 0) {  // for the kernel that joins the parts
              for (int i = lane; i <= sh.items; i += 32) p.meta[4 + i] = sh.items ? pre[i] : 0;
              if (lane == 0) p.meta[0] = sh.shares, p.meta[1] = sh.items, p.meta[2] = whole, p.meta[3] = sh.total;
            }
            if (sh.total > 0 && s < sh.shares) {  // (without items, pre and units hold nothing)
#pragma unroll 1
              for (int k = 0; k < 2; ++k) {
                x = end;
                end = sh.edge(s + k, lane);
              }
            }
          }
        }
#pragma unroll 1
        while (x < end) {
          int index = v, lo = 0, hi = 0x7fffffff, part = -1, next = end;
          if (s >= 0) {
            const int i = sh.item_at(x, lane), from = pre[i], upto = pre[i + 1], shift = units[i] - 1;
            next = min(upto, end);
            index = whole + i;
            lo = (x - from) >> shift;
            hi = (next - from) >> shift;
            if (x > from || next < upto) part = 2 * s + (x > from ? 0 : 1);
          }
          x = next;
          if (!walk.find(p, index, lane, a)) continue;
          AttnItem it;
          const int n0 = attn_tiles(p, a, a.pos), n1 = attn_tiles(p, a, a.pos + p.positions);
          const int first = lo * kAtTile;
          it.q_row = a.q0 + a.pos;
          it.left = a.lq - a.pos;
          it.k_row = a.k0 + first;
          it.keys = a.lk - first;
          it.head = a.head;
          it.see = (p.causal ? a.pos + a.lk - a.lq + 1 : a.lk) - first;
          it.nt[0] = max(min(n0, hi) - lo, 0);
          it.nt[1] = max(min(n1, hi) - lo, 0);
          it.twin = it.left <= p.positions && it.nt[0] > 1;
          const int n = max(it.nt[0], it.nt[1]);
          // the last tile if rows behind it are another's, and the tiles that the first position does not see whole
          it.check = n > 0 && n * kAtTile > it.keys && a.k0 + a.lk < p.Tk ? n - 1 : n;
          if (p.causal) it.check = min(it.check, max(it.see, 0) / kAtTile);
          if (it.twin) {
            it.nt[1] = n / 2;
            it.nt[0] = n - it.nt[1];
          }
          it.part = part;
          it.valid = 1;
          brief = n <= 8;
          send(it);
        }
        // The next one, once this one's loads are all under way (two steps before its end): asked for earlier, it would
        // be taken from CTAs that are free sooner.  Short items are asked for one ahead, since finding one takes as long
        // as three steps.
        const uint32_t behind = brief ? 2 : 1;
        if (sent >= behind) guard.wait(want((sent - behind) % kItems), ((sent - behind) / kItems) & 1);
        const int slot = asked & 1;
        if (lane == 0) {
          mbar_arrive_expect_tx(bars + 2 * S + 17 + slot, 16);
          launch_cancel(answers + 16 * slot, answer_full(slot));
        }
        __syncwarp();
        guard.wait(answer_full(slot), (asked >> 1) & 1);
        if (guard.aborted()) {  // (an answer still on its way writes to shared memory)
          volatile int never = 0;
          mbar_wait_bounded(bars + 2 * S + 17 + slot, (asked >> 1) & 1, kDrainNs, &never);
        }
        v = uniform(launch_cancelled(answers + 16 * slot));
        fence_proxy_async_smem();  // the answer was read before it is overwritten
        __syncwarp();
        ++asked;
        if (guard.aborted()) v = -1;
      }
      AttnItem over = {};
      send(over);
    } else if (warp == 9) {
      // -------------------------------------------------------------- TMA producer
      uint32_t stage = 0, phase = 0, issued_mask = 0, issued_parity = 0, loads = 0;
      uint32_t q_count[2] = {0, 0};
      bool stop = false;
      while (next_item()) {
        copy_item();
        if (lane == 0) {
          auto load_q = [&](int i) {
            guard.wait(q_empty(i), (q_count[i] & 1) ^ 1);
            if ((stop = guard.aborted())) return;
            uint64_t* full = bars + 2 * S + i;
            mbar_arrive_expect_tx(full, NP * 128 * p.positions * p.group);
            for (int c = 0; c < NP; ++c)
              tma_load_3d(q_smem + i * Cfg::kTileBytes + c * kAtPanelBytes, &tmap_q, full, c * 64, it.head * p.group,
                          it.q_row + i * p.positions);
            ++q_count[i];
          };
          const bool twin = it.twin != 0;
          const int n = twin ? it.nt[0] + it.nt[1] : max(it.nt[0], it.nt[1]);
          // K0 V0 K1 V1 ..., or K0 K1 V0 K2 V1 K3 ... V(n-2) V(n-1) for a twin; Q0 before K0, Q1 behind it
#pragma unroll 1
          for (int x = 0; !stop && x < 2 * n; ++x) {
            if (x < 2) {
              if ((x == 0 ? it.nt[0] : it.nt[1]) > 0 && !(twin && x == 1)) load_q(x);
              if (stop) break;
            }
            const int y = x - 2;
            const bool value = twin ? y >= 0 && ((y & 1) == 0 || (y >> 1) + 2 >= n) : (x & 1) != 0;
            const int tile = !twin ? x >> 1 : y < 0 ? x : (y & 1) == 0 ? y >> 1 : min((y >> 1) + 2, n - 1);
            guard.wait(kv_empty(stage), phase ^ 1);
            if ((stop = guard.aborted())) break;
            uint64_t* full = bars + stage;
            mbar_arrive_expect_tx(full, Cfg::kTileBytes);
            for (int c = 0; c < NP; ++c)
              tma_load_3d(ring + stage * Cfg::kTileBytes + c * kAtPanelBytes, value ? &tmap_v : &tmap_k, full, c * 64,
                          it.head, it.k_row + tile * kAtTile);
            guard.progress(++loads);
            issued_mask |= 1u << stage;
            issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
            if (++stage == S) {
              stage = 0;
              phase ^= 1;
            }
          }
          bar_arrive(want((item_count - 1) % kItems));
        }
        __syncwarp();
      }
      if (guard.aborted() && lane == 0) {  // let every load this thread issued land before the CTA leaves
        volatile int never = 0;
        for (int s = 0; s < S; ++s)
          if (issued_mask >> s & 1) mbar_wait_bounded(bars + s, issued_parity >> s & 1, kDrainNs, &never);
        for (int i = 0; i < 2; ++i)
          if (q_count[i]) mbar_wait_bounded(bars + 2 * S + i, (q_count[i] - 1) & 1, kDrainNs, &never);
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
      uint32_t q_phase = 0, p_phase = 0, fixes = 0;  // a bit for each tile
      auto take = [&](uint32_t& s, uint32_t& phase) {  // the next ring slot, in load order
        s = slot;
        phase = slot_phase;
        if (++slot == S) {
          slot = 0;
          slot_phase ^= 1;
        }
      };
      auto qk = [&](int i, uint32_t q, uint32_t s) {  // S_i = Q K^T, by the elected lane
        const uint64_t a0 = q_desc + q * kTileStep, b0 = k_desc + s * kTileStep;
#pragma unroll
        for (int k = 0; k < 4 * NP; ++k) {
          const uint32_t off = ((k >> 2) * kAtPanelBytes + (k & 3) * 32) >> 4;
          if (k < ksteps) mma_f16(tmem + i * 128, a0 + off, b0 + off, idesc_qk, k > 0);
        }
        bar_commit(s_full(i));
      };
      while (next_item()) {
        copy_item();
        const bool twin = it.twin != 0;
        const int n = max(it.nt[0], it.nt[1]), all = it.nt[0] + it.nt[1];
        if (n == 0) continue;
        uint32_t ks = 0, kph = 0, vs = 0, vph = 0;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int mine = i == 0 ? it.nt[0] : it.nt[1], q = twin ? 0 : i;
          if (i == 0 || twin) {
            take(ks, kph);
            guard.wait(kv_full(ks), kph);
          }
          if (mine > 0 && q == i) {
            guard.wait(q_full(i), q_phase >> i & 1);
            q_phase ^= 1u << i;
          }
          tc_fence_after();
          if (elect_one()) {
            if (mine > 0) qk(i, q, ks);
            if (twin ? all == 2 && i == 1 : mine == 1) bar_commit(q_empty(q));
            if (i == 1 || twin) bar_commit(kv_empty(ks));
          }
          __syncwarp();
        }
        // Warp 10 looks at the values of the tiles from `check` on, one tile ahead of their use (they are the next load).
        auto look = [&](int tile) {
          if (tile < it.check || tile >= (twin ? all : n)) return;
          guard.wait(kv_full(slot), slot_phase);
          if (lane == 0) bar_arrive(v_need);
        };
        look(0);
#pragma unroll 1
        for (int step = 0; step < 2 * n; ++step) {
          const int i = step & 1, j = step >> 1, mine = i == 0 ? it.nt[0] : it.nt[1], q = twin ? 0 : i;
          const bool works = j < mine, ends = j + 1 >= mine;
          if (twin && !works) continue;
          const int tile = twin ? step : j;  // key tile whose weights are multiplied
          const bool has_k = twin ? tile + 2 < all : j + 1 < n;
          if (i == 0 || twin) {
            take(vs, vph);
            if (has_k) {  // (the loads run ahead: neither wait lasts)
              take(ks, kph);
              guard.both(kv_full(vs), vph, kv_full(ks), kph);
            } else {
              guard.wait(kv_full(vs), vph);
            }
            if (tile >= it.check) {
              guard.wait(v_fixed, fixes & 1);
              ++fixes;
            }
          }
          const uint64_t b0 = v_desc + vs * kTileStep;
          const uint32_t d = tmem + Cfg::kO + i * 128, a0 = tmem + i * 128;
          if (works) {
            guard.wait(p_full(i, 0), p_phase >> i & 1);
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kFirstSteps; ++k)
                mma_f16_ts(d, a0 + k * 8, b0 + ((k * 16 * 128) >> 4), idesc_pv, k > 0 ? 1 : j > 0);
            }
            __syncwarp();
            guard.wait(p_full(i, 1), p_phase >> i & 1);
            p_phase ^= 1u << i;
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
                qk(i, q, ks);
                if (twin ? tile + 3 == all : j + 2 == mine) bar_commit(q_empty(q));
              }
            }
            if (i == 1 || twin) {  // all that read the slots are issued
              bar_commit(kv_empty(vs));
              if (has_k) bar_commit(kv_empty(ks));
            }
          }
          __syncwarp();
          if (i == 1 || twin) look(tile + 1);
        }
      }
      if (guard.aborted()) {  // the products still in flight read shared memory and TMEM
        volatile int never = 0;
        if (elect_one()) bar_commit(drain);
        __syncwarp();
        mbar_wait_bounded(bars + 2 * S + 14, 0, kDrainNs, &never);
      }
    } else if (warp == 10) {
      // -------------------------------------------------------------- values that a row of the tile must not meet
      // A weight of zero does not keep a NaN or an infinity out of a product.  Rows behind a sequence's end (another
      // request's) are cleared.  In the tiles that causal rows see in part, values that are not finite are cleared and
      // their keys noted: the rows that do see them get those values with the output.  (Rows behind the tensor's end
      // are zeros that TMA filled in.)
      uint32_t slot = 0, fixes = 0;
      while (next_item()) {
        uint32_t* noted = bad + (item_count % kItems) * kBadWords;
        copy_item();
        const int n = it.twin ? it.nt[0] + it.nt[1] : max(it.nt[0], it.nt[1]);
        if (it.check < n && lane < kBadWords) noted[lane] = 0;
        __syncwarp();
#pragma unroll 1
        for (int t = it.check; t < n; ++t) {
          const uint32_t load = it.twin ? min(2 * t + 2, 2 * n - 1) : 2 * t + 1;  // its number among the item's loads
          uint8_t* tile = ring + (slot + load) % S * Cfg::kTileBytes;
          guard.wait(v_need, fixes & 1);
          ++fixes;
          __syncwarp();
          const int rows = min(it.keys - t * kAtTile, kAtTile);
          if (rows < kAtTile)
            for (int c = 0; c < NP; ++c)
              for (int r = rows * 8 + lane; r < kAtTile * 8; r += 32)
                *reinterpret_cast<uint4*>(tile + c * kAtPanelBytes + r * 16) = make_uint4(0, 0, 0, 0);
          if (CAUSAL) {
            // 0 * x is NaN for what is not finite; two values to an instruction, several loads in flight
            using T2 = typename Pack16<T>::Two;
            const T2 zero = Pack16<T>::both(0.0f);
            T2 sum[2] = {zero, zero};
#pragma unroll 1
            for (int c = 0; c < NP; ++c) {
#pragma unroll 8
              for (int r = 0; r < kAtTile; r += 4) {  // 8 lanes for each of 4 rows (zeros behind the end by now)
                const uint4 v = *reinterpret_cast<const uint4*>(tile + c * kAtPanelBytes + r * 128 + lane * 16);
                sum[0] = __hfma2(*reinterpret_cast<const T2*>(&v.x), zero, sum[0]);
                sum[1] = __hfma2(*reinterpret_cast<const T2*>(&v.y), zero, sum[1]);
                sum[0] = __hfma2(*reinterpret_cast<const T2*>(&v.z), zero, sum[0]);
                sum[1] = __hfma2(*reinterpret_cast<const T2*>(&v.w), zero, sum[1]);
              }
            }
            const T2 all = __hadd2(sum[0], sum[1]);
            if (__any_sync(0xffffffffu, !__hbeq2(all, zero))) {
              constexpr uint32_t kExp = kBf16 ? 0x7f807f80u : 0x7c007c00u;
#pragma unroll 1
              for (int r = 0; r < rows; r += 4) {
                uint32_t hit = 0;
#pragma unroll 1
                for (int c = 0; c < NP; ++c) {
                  uint32_t* at = reinterpret_cast<uint32_t*>(tile + c * kAtPanelBytes + r * 128 + lane * 16);
#pragma unroll 1
                  for (int k = 0; k < 4; ++k) {
                    const uint32_t m = __vcmpeq2(at[k] & kExp, kExp);
                    at[k] &= ~m;
                    hit |= m;
                  }
                }
                const uint32_t which = __ballot_sync(0xffffffffu, hit != 0);
                if (which && lane == 0) {
                  uint32_t rows4 = 0;
                  for (int k = 0; k < 4; ++k) rows4 |= (which >> 8 * k & 0xff) ? 1u << k : 0u;
                  noted[1 + (t - it.check) * 4 + r / 32] |= rows4 << (r & 31);
                  noted[0] = 1;
                }
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) bar_arrive(v_fixed);
        }
        slot = (slot + 2 * n) % S;
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax and output of tile i
    setmaxnreg_inc<224>();
    const int i = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t s_addr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + i * 128;
    const float c2 = p.scale_log2;
    // fp16 weights are taken times 2^7 (at most 2^15 with the lazy maximum): more of the small ones stay normal numbers
    constexpr float kShift = kBf16 ? 0.0f : 7.0f;
    uint32_t s_phase = 0, o_phase = 0, twin_phase = 0;
    while (next_item()) {
      const bool twin = uniform(item->twin) != 0;
      const int n = uniform(item->nt[i]);
      // (registers are short below: what only the output needs is worked out again there)
      auto position = [&](bool& valid) {
        const int in_tile = row * p.group_inverse >> 16;  // row / group
        const int pos = (twin ? 0 : i * p.positions) + in_tile;
        valid = in_tile < p.positions && pos < item->left;
        return pos;
      };
      bool valid;
      const int pos = position(valid);
      const int keys = !valid ? 0 : (CAUSAL ? min(item->keys, item->see + pos) : item->keys);
      const bool warp_valid = __any_sync(0xffffffffu, valid);
      // tiles before this one need no mask in any row of the warp
      const int full = __reduce_min_sync(0xffffffffu, valid ? max(keys, 0) : 0x7fffffff) / kAtTile;
      float m = -CUDART_INF_F, l = 0.0f;
      for (int j = 0; j < n; ++j) {
        guard.poll(s_full(i), s_phase);
        s_phase ^= 1;
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
        const int tile = twin ? 2 * j + i : j;
        if (tile >= full) {
          // Scores that a row does not see become -infinity in place, 32 columns at a time (a loop, not 128 selects in a
          // row: seldom run, straight code costs ten cycles and more an instruction to fetch).
          const int seen = keys - tile * kAtTile;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const int left = seen - c * 32;
            if (!__any_sync(0xffffffffu, left < 32)) continue;
            const uint32_t sees = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
            uint32_t x[32];
            tmem_ld_32x32b_x32(s_addr + c * 32, x);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = sees >> e & 1u ? x[e] : 0xff800000u;
            tmem_st_32x32b_x32(s_addr + c * 32, x);
          }
          tmem_st_wait();
        }
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_addr + c * 32, s[c]);
        tmem_ld_wait();
        // The first half of the weights is taken with the maximum so far, while the tile's own maximum is still being
        // found: it seldom grows enough to matter, and then the half is taken again.  Finding the maximum first would
        // leave the special-function unit idle meanwhile.
        if (j == 0) {  // the first tile goes by the maximum of its first 32 scores
          float mx[2] = {m, m};
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            mx[0] = max3(mx[0], __uint_as_float(s[0][e]), __uint_as_float(s[0][e + 1]));
            mx[1] = max3(mx[1], __uint_as_float(s[0][e + 2]), __uint_as_float(s[0][e + 3]));
          }
          m = max3(mx[0], mx[1], mx[1]);
          m = m == -CUDART_INF_F ? m : fmaf(m, 0.0f, m);
        }
        uint64_t sum[2];
        float neg;
#pragma unroll 1
        for (bool again = false;; again = true) {
          neg = m == -CUDART_INF_F ? 0.0f : fmaf(-m, c2, kShift);
          sum[0] = sum[1] = 0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
            weights<T>(s[c], c2, neg, sum, pk);
            tmem_st_32x32b_x16(s_addr + c * 16, pk);
          }
          if (again) break;
          float mx[2] = {m, m};
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              mx[0] = max3(mx[0], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
              mx[1] = max3(mx[1], __uint_as_float(s[c][e + 2]), __uint_as_float(s[c][e + 3]));
            }
          const float top = max3(mx[0], mx[1], mx[1]);
          // (rows without a query hold what was in shared memory: they must not ask for a rescaling at every tile)
          const bool grow = keys > 0 && (m == -CUDART_INF_F ? top != m : !((top - m) * c2 <= kRescaleLog2));
          if (!__any_sync(0xffffffffu, grow)) break;
          const float f = grow ? (m == -CUDART_INF_F ? 0.0f : exp2_approx((m - top) * c2)) : 1.0f;
          if (grow) m = fmaf(top, 0.0f, top);  // top, and NaN for +infinity: its weight is exp(inf - inf)
          l *= f;
          if (j > 0) {  // s_full also says that the products into O so far are done
#pragma unroll 1
            for (int c = 0; c < 2 * NP; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(s_addr + Cfg::kO + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st_32x32b_x32(s_addr + Cfg::kO + c * 32, o);
            }
          }
        }
#pragma unroll
        for (int c = 2; c < 4; ++c) {
          uint32_t pk[16];
          weights<T>(s[c], c2, neg, sum, pk);
          tmem_st_32x32b_x16(s_addr + c * 16, pk);
          if (c == 2) hand_over(0);
        }
        hand_over(1);
        const float2 a = unpack2(add2(sum[0], sum[1]));
        l += a.x + a.y;
      }
      // ------------------------------------------------------------ the item's rows
      if (n > 0) {
        guard.wait(o_full(i), o_phase);
        o_phase ^= 1;
        __syncwarp();
        tc_fence_after();
      }
      float w0 = 1.0f, w1 = 0.0f;  // of this tile's o, and of tile 1's in a twin item
      if (twin) {
        // m and l go through the staging of tile 1's warp, which has no rows to write (not through TMEM: the next item's
        // scores may already go where this one's were)
        const uint32_t pass = smem_u32(staging + (4 + (warp & 3)) * Cfg::kStageOut) + lane * 8;
        if (i == 1) {
          asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(pass), "f"(m), "f"(l) : "memory");
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(twin_ready);
          guard.wait(twin_done, twin_phase);
          twin_phase ^= 1;
          release();
          continue;
        }
        guard.wait(twin_ready, twin_phase);
        twin_phase ^= 1;
        __syncwarp();
        tc_fence_after();
        float m1, l1;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(m1), "=f"(l1) : "r"(pass) : "memory");
        const float top = max3(m, m1, m1);  // NaN if one is
        if (top != -CUDART_INF_F) {
          w0 = m == -CUDART_INF_F ? 0.0f : exp2_approx((m - top) * c2);
          w1 = m1 == -CUDART_INF_F ? 0.0f : exp2_approx((m1 - top) * c2);
          l = l * w0 + l1 * w1;
          m = top;
        }
      }
      if (warp_valid) {
        const float inv = l == 0.0f ? 0.0f : __frcp_rn(l);  // a row that sees no key gives zeros
        w0 *= inv;
        w1 *= inv;
        const bool parts = uniform(item->part) >= 0, any = n > 0 && inv != 0.0f;
        int r = row;
        asm volatile("" : "+r"(r));  // not kept from before
        const int in_tile = r * p.group_inverse >> 16;
        const int64_t t = item->q_row + (twin ? 0 : i * p.positions) + in_tile;
        const int head = item->head * p.group + r - in_tile * p.group;
        const int64_t part = static_cast<int64_t>(item->part) * 256 + i * 128 + row;
        if (valid && (parts || p.lse)) {
          const float lse2 = l == 0.0f ? -CUDART_INF_F : fmaf(m, c2, log2f(l) - kShift);
          if (parts)
            p.part_lse[part] = lse2;
          else
            p.lse[t * (p.heads_kv * p.group) + head] = lse2 * 0.69314718055994530942f;
        }
        // Rows go out through the warp's staging buffer, 128 bytes of 32 rows at a time, so that eight lanes write 128
        // bytes of a row together (16 bytes of each lane's own row per store took 8000 cycles for a tile, and held up
        // every other access of the SM meanwhile).
        uint64_t base = parts ? reinterpret_cast<uint64_t>(p.part_o + part * p.D)
                              : reinterpret_cast<uint64_t>(static_cast<T*>(p.out) + t * p.out_t + head * p.out_h);
        if (!valid) base = 0;
        const int row_bytes = p.D * (parts ? 4 : 2);
        const uint32_t stage = smem_u32(staging + warp * Cfg::kStageOut);
        auto put = [&](int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {  // 16 bytes of this lane's row
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 +
                                                                        ((piece ^ (lane & 7)) << 4)),
                       "r"(a), "r"(b), "r"(c), "r"(d)
                       : "memory");
        };
        auto write_out = [&](int from) {  // bytes [from, from + 128) of the rows
          __syncwarp();
          const int at = from + (lane & 7) * 16;
          uint32_t v[8][4];
          uint64_t to[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int src = 4 * k + (lane >> 3);
            to[k] = __shfl_sync(0xffffffffu, base, src);
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v[k][0]), "=r"(v[k][1]), "=r"(v[k][2]), "=r"(v[k][3])
                         : "r"(stage + src * 128 + (((lane & 7) ^ (src & 7)) << 4))
                         : "memory");
          }
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (to[k] && at < row_bytes)
              asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(to[k] + at), "r"(v[k][0]), "r"(v[k][1]),
                           "r"(v[k][2]), "r"(v[k][3])
                           : "memory");
          __syncwarp();
        };
#pragma unroll 1
        for (int c = 0; c < 2 * NP; ++c) {
          uint32_t o[32];
          if (n > 0) {
            tmem_ld_32x32b_x32(s_addr + Cfg::kO + c * 32, o);
            tmem_ld_wait();
          }
          if (twin) {
            uint32_t o1[32];
            tmem_ld_32x32b_x32(s_addr + Cfg::kO + 128 + c * 32, o1);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = __float_as_uint(fmaf(__uint_as_float(o1[e]), w1, __uint_as_float(o[e]) * w0));
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * w0);
          }
          if (!__all_sync(0xffffffffu, any)) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = any ? o[e] : 0;
          }
          if (parts) {
#pragma unroll
            for (int e = 0; e < 8; ++e) put(e, o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          } else {
            auto two = [&](int e) { return Pack16<T>::pack(__uint_as_float(o[e]), __uint_as_float(o[e + 1])); };
#pragma unroll
            for (int e = 0; e < 4; ++e)
              put((c & 1) * 4 + e, two(8 * e), two(8 * e + 2), two(8 * e + 4), two(8 * e + 6));
            if (!(c & 1)) continue;
          }
          write_out((parts ? c : c >> 1) * 128);
        }
        if (CAUSAL) {  // values that are not finite, in tiles that rows see in part: seldom more than this look
          const volatile uint32_t* noted = bad + (item_count % kItems) * kBadWords;
          if (item->check < (item->twin ? item->nt[0] + item->nt[1] : max(item->nt[0], item->nt[1])) && noted[0]) {
            // (everything worked out again: nothing is kept in registers for this)
            int r = row;
            asm volatile("" : "+r"(r));
            const int in_tile = r * p.group_inverse >> 16, pos = (item->twin ? 0 : i * p.positions) + in_tile;
            const int limit = in_tile < p.positions && pos < item->left ? min(item->keys, item->see + pos) : 0;
            const int slot = item->part;
            T* to = static_cast<T*>(p.out) + static_cast<int64_t>(item->q_row + pos) * p.out_t +
                    (item->head * p.group + r - in_tile * p.group) * p.out_h;
            float* part_to = p.part_o + (static_cast<int64_t>(slot) * 256 + i * 128 + r) * p.D;
#pragma unroll 1
            for (int k = 0; k < 32 * (kBadWords - 1); ++k) {
              const int key = item->check * kAtTile + k;
              if (!(noted[1 + k / 32] >> (k & 31) & 1) || key >= limit) continue;
              const T* v = static_cast<const T*>(p.v) + (item->k_row + key) * p.v_t + item->head * p.v_h;
#pragma unroll 1
              for (int d = 0; d < p.D; ++d) {
                const float x = static_cast<float>(v[d]);
                if (isfinite(x)) continue;
                if (slot >= 0)
                  part_to[d] += x;
                else
                  to[d] = static_cast<T>(static_cast<float>(to[d]) + x);
              }
            }
          }
        }
      }
      if (twin) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(twin_done);
      }
      release();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc<512>(tmem);
  }
}

// Joins the parts of the items that were divided: o = sum_s w_s o_s with w_s = 2^(lse_s - m) / sum 2^(lse_s - m), in
// the order of the shares.  Block (x, y): rows y, y + gridDim.y, ... (by eights) of the x-th divided item; one warp a
// row.  The partial rows were just written and mostly come from L2; what bounds it is the launch and three loads behind
// each other (9 us of the 127 for 1560 queries x 5 heads over 32760 keys; with a walk over the shares for each item, and
// the rows loaded behind their weights, 14).
template <class T>
__global__ void __launch_bounds__(256) attention_combine_kernel(const __grid_constant__ AttnParams p) {
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31;
  const int x = blockIdx.x;
  const int shares = p.meta[0], items = p.meta[1], whole = p.meta[2], all = p.meta[3];
  const int from = p.meta[4 + x], upto = p.meta[5 + x];
  // Where the first kernel gave up, or offsets of sequences that overlap made more items than the grid has CTAs, no plan
  // was written and the workspace holds anything.  With these limits every such content leads either nowhere or to rows
  // of a sequence: find() takes no item but the call's own, and parts beyond the workspace's are not read.
  if (x >= items || items >= kMaxShares || shares < 1 || shares > p.shares || all < 1) return;
  if (whole < 0 || whole % p.shares != 0 || from < 0 || upto <= from || upto > all) return;
  // The edges inside this item: place(s) = all s / shares in [from + 4, upto - 4] (AttnShares::snap).  Looked at before the
  // item's sequence is searched for, which takes several loads: most items of many short requests are not divided.
  const int64_t low = (int64_t{from} + 4) * shares, high = (int64_t{upto} - 3) * shares;
  const int s0 = max(1, static_cast<int>((low + all - 1) / all));
  const int last = min(shares - 1, static_cast<int>((high + all - 1) / all) - 1);
  if (last < s0) return;  // one share has it all
  AttnWalk walk;
  AttnPlace a;
  if (!walk.find(p, whole + x, lane, a)) return;
  const int first = s0 - 1;
  const int heads = p.heads_kv * p.group;
  const int rows = min(a.lq - a.pos, 2 * p.positions) * p.group;
  const int c = lane * 4;
  for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.y * 8) {
    const int position = r / p.group, head = r - position * p.group;
    const int tile = position >= p.positions ? 1 : 0;
    const int at = tile * 128 + (position - tile * p.positions) * p.group + head;
    auto slot = [&](int s) {  // the first part of an item is its share's last
      return (2 * static_cast<int64_t>(s) + (s == first ? 1 : 0)) * 256 + at;
    };
    auto part = [&](int s) {  // (a part without keys holds zeros)
      return s <= last && c < p.D ? *reinterpret_cast<const float4*>(p.part_o + slot(s) * p.D + c)
                                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    };
    float4 f[4];  // on their way while the weights are found
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = part(first + k);
    float z = first + lane <= last ? p.part_lse[slot(first + lane)] : -CUDART_INF_F;
    float m = z;
    for (int s = first + 32 + lane; s <= last; s += 32) m = max3(m, p.part_lse[slot(s)], p.part_lse[slot(s)]);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, m, o);
      m = max3(m, other, other);
    }
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float total = 0.0f;
    for (int b = first; b <= last; b += 32) {  // a lane for each part's weight
      if (b > first) z = b + lane <= last ? p.part_lse[slot(b + lane)] : -CUDART_INF_F;
      const float mine = z == -CUDART_INF_F ? 0.0f : exp2f(z - m);
      for (int k = 0; k < 32 && b + k <= last; k += 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w = __shfl_sync(0xffffffffu, mine, k + e);
          total += w;
          acc.x = fmaf(w, f[e].x, acc.x), acc.y = fmaf(w, f[e].y, acc.y);
          acc.z = fmaf(w, f[e].z, acc.z), acc.w = fmaf(w, f[e].w, acc.w);
          f[e] = part(b + k + 4 + e);
        }
      }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int64_t t = a.q0 + a.pos + position;
    const int h = a.head * p.group + head;
    if (c < p.D)
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + t * p.out_t + h * p.out_h + c) =
          make_uint2(Pack16<T>::pack(acc.x * inv, acc.y * inv), Pack16<T>::pack(acc.z * inv, acc.w * inv));
    if (p.lse && lane == 0)
      p.lse[t * heads + h] = total == 0.0f ? -CUDART_INF_F : (m + log2f(total)) * 0.69314718055994530942f;
  }
}

}  // namespace convrot
