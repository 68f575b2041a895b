// Rotary positions with several axes, and the per-head RMS norm of queries and keys with the rotation in one pass.
//
// rotary_table_kernel: pair j of a head belongs to one position axis a (time, height, width, ...) and turns by
//   angle[t, j] = pos[t, a] * theta_a^(-2 i / d_a),   out[t, j] = (cos, sin) in fp32.
// The angle of a far position has to be known modulo 2 pi: pos * frequency is formed and reduced in fp64 (in units of
// pi, where the reduction x - 2 rint(x / 2) is exact), split into a float and its remainder, and the remainder enters
// through sin(h + l) = sin h + l cos h.  Each frequency / pi is a host-computed kernel argument, so no thread
// evaluates a power.  Bound by its 8 bytes of output per pair (and, at a few hundred rows, by its launch).
//
// qk_norm_rope_kernel: for each head row x of q and k
//   y = x * rsqrt(mean(x^2) + eps) * w,   (a, b) -> (a c - b s, b c + a s) for each pair of the first R channels,
// all in fp32, rounded once to the output type.  Bound by HBM (each row read once, written once): 32760 tokens of 2 x 40
// heads of 128 take 220 us, 6.2 TB/s (231 with pairs half the rotated width apart; a plain copy of the same bytes 205),
// ncu sees the issue slots as the next bound.  A lane holds 8 neighbouring channels (one 16-byte load) or two such
// pieces, so that both channels of a pair are always its own; a row lies in a power-of-two group of lanes, so the sum of
// squares is a few shuffles and the statistics never touch memory.  A warp takes several rows of one token at once:
// kRopeRows independent loads in flight per lane, and one read of the token's table row for all of them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace convrot {

// A kernel launched with programmatic stream serialisation may begin while the one before it in the stream ends:
// grid_wait() holds until that one is complete and its writes are visible, and has to come before the first access to
// memory; grid_release() lets the next such kernel begin as soon as this one's last blocks are placed.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

constexpr int kRopeMaxPairs = 128;
constexpr int kRopeMaxAxes = 8;

struct RotaryTableParams {
  double freq_over_pi[kRopeMaxPairs];
  uint8_t axis[kRopeMaxPairs];
  const void* pos;
  int64_t ld_pos;
  int64_t rows;
  int pairs;
  float2* out;
};

template <class Pos>
__global__ void __launch_bounds__(256) rotary_table_kernel(const __grid_constant__ RotaryTableParams p) {
  // (read from the arguments directly, 32 frequencies of a warp are 32 accesses one after the other: 33 us instead of
  // 5 for 32760 x 64 pairs)
  __shared__ double freq[kRopeMaxPairs];
  __shared__ int axis[kRopeMaxPairs];
  if (threadIdx.x < p.pairs) {
    freq[threadIdx.x] = p.freq_over_pi[threadIdx.x];
    axis[threadIdx.x] = p.axis[threadIdx.x];
  }
  __syncthreads();
  grid_wait();
  grid_release();
  const int64_t n = p.rows * p.pairs;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += step) {
    // 32-bit division wherever it fits (a 64-bit one costs several times as much)
    const int64_t t = n <= 0x7fffffff ? static_cast<uint32_t>(i) / static_cast<uint32_t>(p.pairs) : i / p.pairs;
    const int j = static_cast<int>(i - t * p.pairs);
    const double pos = static_cast<double>(static_cast<const Pos*>(p.pos)[t * p.ld_pos + axis[j]]);
    double x = pos * freq[j];
    x = fma(-2.0, rint(0.5 * x), x);
    const float h = static_cast<float>(x);
    const float l = static_cast<float>((x - static_cast<double>(h)) * 3.14159265358979323846);
    float s, c;
    sincospif(h, &s, &c);
    p.out[i] = make_float2(fmaf(-l, s, c), fmaf(l, c, s));
  }
}

struct QkRopeParams {
  const void* in[2];  // q, k: [T, H, D]
  void* out[2];
  int64_t in_t[2], in_h[2], out_t[2], out_h[2];  // strides in elements
  const void* weight[2];                         // [D] or null
  int heads[2];
  const float2* table;  // [T, R / 2] (cos, sin) or null
  int64_t ld_table;     // pairs
  int64_t rows;         // T
  int D, R;
  int lanes_log2;  // lanes of one head row: a power of two
  int items, items_q;  // warp items of one token, and of its q
  int norm, weight_f32;
  float eps, inv_D;
};

constexpr int kRopeRows = 4;  // 16-byte loads of a lane in flight (2: 339 us instead of 220, 8: 262)
constexpr int kRopeWarps = 2;

template <class T>
struct Pack16;
template <>
struct Pack16<__nv_bfloat16> {
  using Two = __nv_bfloat162;
  static __device__ __forceinline__ Two both(float a) { return __float2bfloat162_rn(a); }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Pack16<__half> {
  using Two = __half2;
  static __device__ __forceinline__ Two both(float a) { return __float2half2_rn(a); }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Eight channels of a norm weight at element c; ones where there is none.
template <class T>
__device__ __forceinline__ void load_weight8(const void* w, int f32, int c, float (&o)[8]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 1.0f;
  } else if (f32) {
    const float4* w4 = reinterpret_cast<const float4*>(static_cast<const float*>(w) + c);
    const float4 a = __ldg(w4), b = __ldg(w4 + 1);
    o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
  } else {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(w) + c));
    const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Pack16<T>::unpack(v[i]);
      o[2 * i] = f.x, o[2 * i + 1] = f.y;
    }
  }
}

// A warp item is a few steps of rows of q or of k of one token.  Weights and rotation are joined once for all of an item's
// rows: with (a, b) a pair and a' = inv a, b' = inv b, out = (a' (wa c) - b' (wb s), b' (wb c) + a' (wa s)), so a row
// costs two operations an element beside its sum of squares and the scale, and two channels go through each as one
// paired instruction.  (For 32760 tokens x 2 x 40 heads of 128: every row with its own weight and rotation 350 us, bound
// by issue slots; unpaired 223, and 238 with pairs R / 2 apart.)  With pairs of neighbours a lane holds 8 channels; with
// pairs R / 2 apart it holds the 8 channels and their partners, R / 2 further (fetched by shuffles from the partners'
// lane they cost 306 us), and lanes behind the rotated part hold 16 channels in a row.
template <class T, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_kernel(const __grid_constant__ QkRopeParams p) {
  constexpr int CH = INTERLEAVED ? 1 : 2;  // 8-channel pieces of a lane
  constexpr int kSteps = kRopeRows / CH;
  constexpr int kPartner = INTERLEAVED ? 1 : 4;  // registers of two channels
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kRopeWarps + (threadIdx.x >> 5);
  if (item >= p.rows * p.items) return;  // whole warps
  const int64_t t = p.rows * p.items <= 0x7fffffff
                        ? static_cast<uint32_t>(item) / static_cast<uint32_t>(p.items)
                        : item / p.items;
  const int lanes = 1 << p.lanes_log2;
  const int at = lane & (lanes - 1);
  const int half = p.R >> 1;
  const bool turns = INTERLEAVED ? at * 8 < p.R : at * 8 < half;
  const int c = INTERLEAVED || turns ? at * 8 : p.R + (at * 8 - half) * 2;  // this lane's first channel
  const int apart = turns ? half : 8;                                       // and its second piece (CH == 2)
  const int per = 32 >> p.lanes_log2;                                       // rows of one step of the warp
  int group = static_cast<int>(item - t * p.items);
  const bool is_k = group >= p.items_q;
  if (is_k) group -= p.items_q;
  const int heads = is_k ? p.heads[1] : p.heads[0];
  const int row0 = group * (kSteps * per) + (lane >> p.lanes_log2);
  const int64_t in_h = is_k ? p.in_h[1] : p.in_h[0], out_h = is_k ? p.out_h[1] : p.out_h[0];
  const T* in = static_cast<const T*>(is_k ? p.in[1] : p.in[0]) + t * (is_k ? p.in_t[1] : p.in_t[0]) + row0 * in_h + c;
  T* out = static_cast<T*>(is_k ? p.out[1] : p.out[0]) + t * (is_k ? p.out_t[1] : p.out_t[0]) + row0 * out_h + c;
  bool here[CH];
#pragma unroll
  for (int h = 0; h < CH; ++h) here[h] = c + h * apart < p.D;

  uint4 raw[kSteps][CH];
#pragma unroll
  for (int r = 0; r < kSteps; ++r)
#pragma unroll
    for (int h = 0; h < CH; ++h) {
      raw[r][h] = make_uint4(0, 0, 0, 0);
      if (here[h] && row0 + r * per < heads)
        raw[r][h] = __ldcs(reinterpret_cast<const uint4*>(in + r * per * in_h + h * apart));
    }

  // Two channels to a register, so that an instruction works on both: with pairs of neighbours channels (0, 2), (1, 3),
  // (4, 6), (5, 7), else neighbours; element i's partner is i ^ kPartner either way, with kPartner = 1 or 4 registers.
  // out[i] = mine[i] x[i] + other[i] x[i ^ kPartner]
  constexpr int kRegs = 4 * CH;
  uint64_t mine[kRegs], other[kRegs];
  {
    float m[8 * CH], o[8 * CH];
#pragma unroll
    for (int h = 0; h < CH; ++h) {
      float w[8] = {};
      if (here[h]) load_weight8<T>(is_k ? p.weight[1] : p.weight[0], p.weight_f32, c + h * apart, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) m[8 * h + i] = w[i], o[8 * h + i] = 0.0f;
    }
    if (p.table && turns) {
      constexpr int kApart = INTERLEAVED ? 1 : 8;
      const float4* src = reinterpret_cast<const float4*>(p.table + t * p.ld_table + (INTERLEAVED ? c >> 1 : c));
#pragma unroll
      for (int i = 0; i < 2 * CH; ++i) {
        const float4 f = __ldg(src + i);
        const float cs[2] = {f.x, f.z}, sn[2] = {f.y, f.w};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int a = INTERLEAVED ? 4 * i + 2 * k : 2 * i + k, b = a + kApart;
          const float wa = m[a], wb = m[b];
          m[a] = wa * cs[k], o[a] = -wb * sn[k];
          m[b] = wb * cs[k], o[b] = wa * sn[k];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int a = INTERLEAVED ? (i >> 1) * 4 + (i & 1) : 2 * i, b = INTERLEAVED ? a + 2 : a + 1;
      mine[i] = pack2(m[a], m[b]);
      other[i] = pack2(o[a], o[b]);
    }
  }

  // (two rows of 16 channels a lane at once take 93 registers, and 245 us instead of 231)
  constexpr int kBatch = INTERLEAVED ? kSteps : 1;  // rows whose shuffles overlap
#pragma unroll
  for (int r0 = 0; r0 < kSteps; r0 += kBatch) {
    uint64_t x[kBatch][kRegs];
#pragma unroll
    for (int r = 0; r < kBatch; ++r)
#pragma unroll
      for (int h = 0; h < CH; ++h) {
        const uint4 u = raw[r0 + r][h];
        const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float2 f = Pack16<T>::unpack(v[i]), g = Pack16<T>::unpack(v[i + 1]);
          x[r][4 * h + i] = INTERLEAVED ? pack2(f.x, g.x) : pack2(f.x, f.y);
          x[r][4 * h + i + 1] = INTERLEAVED ? pack2(f.y, g.y) : pack2(g.x, g.y);
        }
      }
    if (p.norm) {
      float sum[kBatch];
#pragma unroll
      for (int r = 0; r < kBatch; ++r) {
        uint64_t s2 = 0;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) s2 = fma2(x[r][i], x[r][i], s2);
        const float2 s = unpack2(s2);
        sum[r] = s.x + s.y;
      }
      for (int o = lanes >> 1; o; o >>= 1)
#pragma unroll
        for (int r = 0; r < kBatch; ++r) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], o);
#pragma unroll
      for (int r = 0; r < kBatch; ++r) {
        const float inv = rsqrtf(fmaf(sum[r], p.inv_D, p.eps));
#pragma unroll
        for (int i = 0; i < kRegs; ++i) x[r][i] = mul2(x[r][i], pack2(inv, inv));
      }
    }
#pragma unroll
    for (int r = 0; r < kBatch; ++r) {
      float2 y[kRegs];
      if (p.table && turns) {
#pragma unroll
        for (int i = 0; i < kRegs; ++i) y[i] = unpack2(fma2(x[r][i], mine[i], mul2(x[r][i ^ kPartner], other[i])));
      } else {
#pragma unroll
        for (int i = 0; i < kRegs; ++i) y[i] = unpack2(mul2(x[r][i], mine[i]));
      }
#pragma unroll
      for (int h = 0; h < CH; ++h)
        if (here[h] && row0 + (r0 + r) * per < heads) {
          uint32_t u[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = 4 * h + i;
            if (INTERLEAVED)
              u[i] = (i & 1) ? Pack16<T>::pack(y[k - 1].y, y[k].y) : Pack16<T>::pack(y[k].x, y[k + 1].x);
            else
              u[i] = Pack16<T>::pack(y[k].x, y[k].y);
          }
          __stcs(reinterpret_cast<uint4*>(out + (r0 + r) * per * out_h + h * apart),
                 make_uint4(u[0], u[1], u[2], u[3]));
        }
    }
  }
}

}  // namespace convrot
