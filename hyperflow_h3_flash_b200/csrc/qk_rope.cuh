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
// all in fp32, rounded once to the output type.  Bound by HBM (each row read once, written once; 8 fp32 operations per
// element).  A lane holds 8 neighbouring channels (one 16-byte load), a row lies in a power-of-two group of lanes, so
// the sum of squares is a few shuffles and the statistics never touch memory; pairs half a rotated width apart reach
// each other by shuffles as well.  A warp takes kRopeRows row groups of one token at once: that many independent loads
// in flight per lane, and one read of the token's table row for all of them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace convrot {

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
  const int64_t n = p.rows * p.pairs;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += step) {
    // 32-bit division wherever it fits (a 64-bit one costs several times as much)
    const int64_t t = n <= 0x7fffffff ? static_cast<uint32_t>(i) / static_cast<uint32_t>(p.pairs) : i / p.pairs;
    const int j = static_cast<int>(i - t * p.pairs);
    const double pos = static_cast<double>(static_cast<const Pos*>(p.pos)[t * p.ld_pos + p.axis[j]]);
    double x = pos * p.freq_over_pi[j];
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
  int lanes_log2;  // lanes of one head row: the power of two that holds D / 8
  int items;       // warp items of one token
  int norm, weight_f32;
  float eps;
};

constexpr int kRopeRows = 4;
constexpr int kRopeWarps = 8;

template <class T>
struct Pack16;
template <>
struct Pack16<__nv_bfloat16> {
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

template <class T, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_kernel(const __grid_constant__ QkRopeParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kRopeWarps + (threadIdx.x >> 5);
  if (item >= p.rows * p.items) return;  // whole warps
  const int64_t t = item / p.items;
  const int lanes = 1 << p.lanes_log2;
  const int at = lane & (lanes - 1);
  const int c = at * 8;  // this lane's first channel
  const bool here = c < p.D;
  const int per = 32 >> p.lanes_log2;  // rows of one step of the warp
  const int row0 = static_cast<int>(item - t * p.items) * (kRopeRows * per) + (lane >> p.lanes_log2);
  const int total = p.heads[0] + p.heads[1];

  uint4 raw[kRopeRows];
  int which[kRopeRows], head[kRopeRows];
#pragma unroll
  for (int r = 0; r < kRopeRows; ++r) {
    const int row = row0 + r * per;
    which[r] = row >= total ? -1 : (row >= p.heads[0] ? 1 : 0);
    head[r] = which[r] == 1 ? row - p.heads[0] : row;
    raw[r] = make_uint4(0, 0, 0, 0);
    if (here && which[r] >= 0) {
      const int w = which[r];
      raw[r] = *reinterpret_cast<const uint4*>(static_cast<const T*>(w ? p.in[1] : p.in[0]) +
                                               t * (w ? p.in_t[1] : p.in_t[0]) +
                                               head[r] * (w ? p.in_h[1] : p.in_h[0]) + c);
    }
  }

  // (cos, sin) of this lane's channels: 4 pairs of neighbours, or 8 pairs half the rotated width apart
  constexpr int kPairs = INTERLEAVED ? 4 : 8;
  float2 cs[kPairs];
  const int half = p.R >> 1;
  const bool turns = p.table && c < p.R;
  const bool second = !INTERLEAVED && c >= half;
  if (turns) {
    const float4* src = reinterpret_cast<const float4*>(p.table + t * p.ld_table +
                                                        (INTERLEAVED ? c >> 1 : (second ? c - half : c)));
#pragma unroll
    for (int i = 0; i < kPairs / 2; ++i) {
      const float4 f = __ldg(src + i);
      cs[2 * i] = make_float2(f.x, f.y);
      cs[2 * i + 1] = make_float2(f.z, f.w);
    }
  }
  float wq[8], wk[8];
  if (here) {
    load_weight8<T>(p.weight[0], p.weight_f32, c, wq);
    load_weight8<T>(p.weight[1], p.weight_f32, c, wk);
  }

#pragma unroll
  for (int r = 0; r < kRopeRows; ++r) {
    const uint32_t v[4] = {raw[r].x, raw[r].y, raw[r].z, raw[r].w};
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Pack16<T>::unpack(v[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
    if (p.norm) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
      for (int o = lanes >> 1; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float inv = rsqrtf(sum / static_cast<float>(p.D) + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * (which[r] == 1 ? wk[i] : wq[i]);
    }
    if (p.table) {  // uniform
      if (INTERLEAVED) {
        if (turns) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = a * cs[i % kPairs].x - b * cs[i % kPairs].y;
            x[2 * i + 1] = b * cs[i % kPairs].x + a * cs[i % kPairs].y;
          }
        }
      } else {
        const int partner = (lane & ~(lanes - 1)) | (turns ? (second ? at - (half >> 3) : at + (half >> 3)) : at);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float o = __shfl_sync(0xffffffffu, x[i], partner);
          if (turns) x[i] = x[i] * cs[i % kPairs].x + (second ? o : -o) * cs[i % kPairs].y;
        }
      }
    }
    if (here && which[r] >= 0) {
      const int w = which[r];
      uint4 u;
      u.x = Pack16<T>::pack(x[0], x[1]);
      u.y = Pack16<T>::pack(x[2], x[3]);
      u.z = Pack16<T>::pack(x[4], x[5]);
      u.w = Pack16<T>::pack(x[6], x[7]);
      *reinterpret_cast<uint4*>(static_cast<T*>(w ? p.out[1] : p.out[0]) + t * (w ? p.out_t[1] : p.out_t[0]) +
                                head[r] * (w ? p.out_h[1] : p.out_h[0]) + c) = u;
    }
  }
}

}  // namespace convrot
