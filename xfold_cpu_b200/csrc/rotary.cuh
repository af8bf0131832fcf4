// Rotary positions on queries and keys (HBM-bound: every value is read and written once).
//
// The first `rotated` dims of a head hold rotated / 2 pairs (a, b): neighbours
// (2 i, 2 i + 1), or the halves' (i, i + rotated / 2).  Pair i of the token at
// position p turns by the angle p f_i and grows by `magnitude`:
//   a' = m (a cos - b sin),  b' = m (b cos + a sin)
// The backward pass is the transposed map: the same with -sin.  Dims past
// `rotated` are copied.
//
// A thread owns VEC neighbouring dims (and, in the halves' layout, their
// partners) of one token and walks over a share of the heads of q and k, so the sines
// and cosines are computed once for the heads it serves.  The angle is taken in whole turns,
// in f64, and its fraction goes to f32: an f32 product would be off by p 2^-25, 2e-3 rad at
// position 65536.
// Measured on 2 x 8191 tokens of 24 heads of 128 in bf16: 43 us all turned (4.7 TB/s), 48 us with 32
// dims turned, where part of a warp computes and the rest copies.
#pragma once

#include "common.cuh"
#include "layer_norm_train.cuh"  // LnVec, ln_float, ln_round

namespace xfb {

struct RotaryTensor {
  const void* x;
  int64_t sb, sh, sn;  // strides in elements; the head dim is contiguous
  void* y;
  int64_t yb, yh, yn;
};

struct RotaryArgs {
  RotaryTensor q, k;
  int H, G;                  // heads of q, heads of k
  int64_t B, n;
  int d, rotated;
  const float* freq;         // [rotated / 2]
  const void* positions;     // positions[b * pos_sb + i], or null: offset + i
  int positions_64;          // they are int64 (else int32)
  int64_t pos_sb;
  int64_t offset;
  float magnitude;
  int inverse;
  int head_step;             // head shares: blockIdx.y takes heads y, y + head_step, ...
};

__device__ __forceinline__ void rotary_sincos(double position, float freq, float magnitude,
                                              int inverse, float& s, float& c) {
  const double turns = position * (static_cast<double>(freq) * 0.15915494309189535);  // 1 / (2 pi)
  sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
  c *= magnitude;
  s *= inverse ? -magnitude : magnitude;
}

template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  using Vec = LnVec<T, VEC>;
  // Threads of a token: the rotated dims (both halves by one thread), then the copied ones.
  // With INTERLEAVED and VEC = 1 a "vector" is one pair.
  constexpr bool kPair = INTERLEAVED && VEC == 1;
  constexpr int W = kPair ? 2 : VEC;  // dims of a thread's load
  const int half = a.rotated / 2;
  const int turning = INTERLEAVED ? a.rotated / W : half / VEC;
  const int copied = (a.d - a.rotated + VEC - 1) / VEC;
  const int per_token = turning + copied;
  const int64_t total = a.B * a.n * per_token;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; at < total;
       at += step) {
    const int64_t token = at / per_token;
    const int part = static_cast<int>(at - token * per_token);
    const int64_t b = token / a.n, i = token - b * a.n;
    const bool turns = part < turning;
    const int dim = turns ? part * W : a.rotated + (part - turning) * VEC;
    constexpr int PAIRS = INTERLEAVED ? (kPair ? 1 : VEC / 2) : VEC;
    float sn[PAIRS], cs[PAIRS];
    if (turns) {
      const int64_t place = b * a.pos_sb + i;
      const double position = static_cast<double>(
          a.positions == nullptr ? a.offset + i
          : a.positions_64       ? static_cast<const int64_t*>(a.positions)[place]
                                 : static_cast<const int32_t*>(a.positions)[place]);
#pragma unroll
      for (int p = 0; p < PAIRS; ++p)
        rotary_sincos(position, a.freq[(INTERLEAVED ? dim / 2 : dim) + p], a.magnitude, a.inverse,
                      sn[p], cs[p]);
    }
    for (int h = blockIdx.y; h < a.H + a.G; h += a.head_step) {
      const bool is_q = h < a.H;
      const RotaryTensor& r = is_q ? a.q : a.k;
      const int hh = is_q ? h : h - a.H;
      const T* x = static_cast<const T*>(r.x) + b * r.sb + hh * r.sh + i * r.sn + dim;
      T* y = static_cast<T*>(r.y) + b * r.yb + hh * r.yh + i * r.yn + dim;
      if (!turns) {
        *reinterpret_cast<Vec*>(y) = *reinterpret_cast<const Vec*>(x);
      } else if constexpr (kPair) {
        const float u = ln_float(x[0]), v = ln_float(x[1]);
        y[0] = ln_round<T>(u * cs[0] - v * sn[0]);
        y[1] = ln_round<T>(v * cs[0] + u * sn[0]);
      } else if constexpr (INTERLEAVED) {
        const Vec in = *reinterpret_cast<const Vec*>(x);
        Vec o;
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
          const float u = ln_float(in.v[2 * p]), v = ln_float(in.v[2 * p + 1]);
          o.v[2 * p] = ln_round<T>(u * cs[p] - v * sn[p]);
          o.v[2 * p + 1] = ln_round<T>(v * cs[p] + u * sn[p]);
        }
        *reinterpret_cast<Vec*>(y) = o;
      } else {
        const Vec lo = *reinterpret_cast<const Vec*>(x);
        const Vec hi = *reinterpret_cast<const Vec*>(x + half);
        Vec ol, oh;
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
          const float u = ln_float(lo.v[p]), v = ln_float(hi.v[p]);
          ol.v[p] = ln_round<T>(u * cs[p] - v * sn[p]);
          oh.v[p] = ln_round<T>(v * cs[p] + u * sn[p]);
        }
        *reinterpret_cast<Vec*>(y) = ol;
        *reinterpret_cast<Vec*>(y + half) = oh;
      }
    }
  }
}

}  // namespace xfb
