// Queries and keys of new tokens: each head's norm, if there is one, and the
// rotation by positions of several axes, in one pass (ocrvl_op_rotate).
//
//   y = x / sqrt(mean x^2 + eps) * w
//   pair p (dims p and p + pairs, or 2 p and 2 p + 1): angle = pos[axis p] freq[p]
//   (u, v) -> (u cos - v sin, v cos + u sin);  dims behind 2 pairs stay y
// A warp a token (or a share of a token's heads): it works out the token's cosines and
// sines once, two lanes' worth in shared memory, then goes through the heads with a lane
// for 2 V dims.  The angle is a 64-bit product of turns, whose whole part is dropped before
// it becomes 32 bits, so far positions keep their last bits.
#pragma once
#include "packed.cuh"

namespace ocrvl {
namespace paged {

constexpr int kRotateWarps = 8;
constexpr int kRotateMost = 128;  // pairs

struct RotateArgs {
  const char *q, *k;
  char *q_out, *k_out;
  const void *q_weight, *k_weight;
  const int *pos;
  long long q_stride, k_stride, q_out_stride, k_out_stride, pos_stride;  // bytes; entries
  int n_tokens, heads, kv_heads, dim, pairs, neighbours;
  int lanes, at_once, lane_factor;  // lanes of a row, rows at once, 2^16 / lanes rounded up
  float eps, one_dim;               // 1 / dim
  double turns[kRotateMost];  // freq / 2 pi
  unsigned char axis[kRotateMost];
};

// V values as they lie in memory, and as 32-bit floats.
template <typename T, int V>
struct Run {
  uint32_t w[V * sizeof(T) / 4];

  __device__ __forceinline__ void load(const T *p) {
    if constexpr (V * sizeof(T) == 16)
      *(uint4 *)w = *(const uint4 *)p;
    else
      *(uint2 *)w = *(const uint2 *)p;
  }
  __device__ __forceinline__ void floats(float (&x)[V]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; i++) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; i++) {
        const float2 f = unpack2<T>(w[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    }
  }
};
template <typename T, int V>
__device__ __forceinline__ void store_v(T *p, const float (&x)[V]) {
  if constexpr (sizeof(T) == 4) {
    *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]);
  } else if constexpr (V == 8) {
    *(uint4 *)p = make_uint4(pack2(x[0], x[1], T()), pack2(x[2], x[3], T()), pack2(x[4], x[5], T()), pack2(x[6], x[7], T()));
  } else {
    *(uint2 *)p = make_uint2(pack2(x[0], x[1], T()), pack2(x[2], x[3], T()));
  }
}

constexpr int kRotateSteps = 4;  // of rows whose loads go out together

// NORM: 0 none, 1 weights of T, 2 weights of f32.  LANES: of a row, 0: any number.
template <typename T, int V, int NORM, int LANES>
__global__ void __launch_bounds__(kRotateWarps * 32, 2) k_rotate(const __grid_constant__ RotateArgs a) {
  __shared__ __align__(16) float trig[kRotateWarps][2][kRotateMost];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.x * kRotateWarps + warp;
  if (token >= a.n_tokens) return;  // the whole warp
  const int lanes = LANES ? LANES : a.lanes, at_once = LANES ? 32 / (LANES ? LANES : 1) : a.at_once;
  const int sub = LANES ? lane / (LANES ? LANES : 1) : lane * a.lane_factor >> 16, v = lane - sub * lanes, rotated = a.pairs / V;
  // the lane's two runs of V dims
  const int d0 = v >= rotated ? 2 * a.pairs + 2 * V * (v - rotated) : a.neighbours ? 2 * V * v : V * v;
  const int d1 = v >= rotated || a.neighbours ? d0 + V : a.pairs + d0;
  const int start = blockIdx.y * at_once + sub, step = gridDim.y * at_once;
  using Rows = Run<T, V>[kRotateSteps][2];
  auto load = [&](Rows &x, int r0, int n, const char *in) {
#pragma unroll
    for (int i = 0; i < kRotateSteps; i++) {
      const int r = r0 + i * step;
      const T *from = (const T *)in + r * a.dim;
      if (r < n && sub < at_once) x[i][0].load(from + d0), x[i][1].load(from + d1);
    }
  };
  const char *q = a.q + token * a.q_stride, *k = a.k + token * a.k_stride;
  Rows xq;
  load(xq, start, a.heads, q);  // on their way during what follows

  float *cs = trig[warp][0], *sn = trig[warp][1];
  for (int p = lane; p < a.pairs; p += 32) {
    const double x = (double)a.pos[token * a.pos_stride + a.axis[p]] * a.turns[p];
    sincospif(2.f * (float)(x - rint(x)), &sn[p], &cs[p]);
  }
  __syncwarp();
  float c[V] = {}, s[V] = {};
  if (v < rotated) {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      *(float4 *)(c + e) = *(const float4 *)(cs + V * v + e);
      *(float4 *)(s + e) = *(const float4 *)(sn + V * v + e);
    }
  }
  auto turn = [&](const Rows &raw, int r0, int n, char *out, const float (&w0)[V], const float (&w1)[V]) {
#pragma unroll
    for (int i = 0; i < kRotateSteps; i++) {
      const int r = r0 + i * step;
      if (!__any_sync(~0u, r < n)) break;
      const bool there = r < n && sub < at_once;
      float x[V], y[V];
      raw[i][0].floats(x), raw[i][1].floats(y);
      if constexpr (NORM > 0) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < V; e++) sum = fmaf(x[e], x[e], fmaf(y[e], y[e], sum));
        if constexpr (LANES > 0) {
#pragma unroll
          for (int d = LANES / 2; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
        } else {  // the row's first lane collects, all ask it
#pragma unroll
          for (int d = 16; d; d >>= 1) {
            const float other = __shfl_down_sync(~0u, sum, d);
            if (v < d && v + d < lanes) sum += other;
          }
          sum = __shfl_sync(~0u, sum, lane - v);
        }
        const float inv = rsqrtf(sum * a.one_dim + a.eps);
#pragma unroll
        for (int e = 0; e < V; e++) x[e] *= inv * w0[e], y[e] *= inv * w1[e];
      }
      float z0[V], z1[V];
      if (v >= rotated) {
#pragma unroll
        for (int e = 0; e < V; e++) z0[e] = x[e], z1[e] = y[e];
      } else if (!a.neighbours) {
#pragma unroll
        for (int e = 0; e < V; e++) z0[e] = x[e] * c[e] - y[e] * s[e], z1[e] = y[e] * c[e] + x[e] * s[e];
      } else {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          z0[e] = x[e] * c[e / 2] - x[e + 1] * s[e / 2], z0[e + 1] = x[e + 1] * c[e / 2] + x[e] * s[e / 2];
          z1[e] = y[e] * c[V / 2 + e / 2] - y[e + 1] * s[V / 2 + e / 2], z1[e + 1] = y[e + 1] * c[V / 2 + e / 2] + y[e] * s[V / 2 + e / 2];
        }
      }
      T *to = (T *)out + r * a.dim;
      if (there) store_v<T, V>(to + d0, z0), store_v<T, V>(to + d1, z1);
    }
  };
  auto weights = [&](float (&w0)[V], float (&w1)[V], const void *weight) {
    if constexpr (NORM == 1) {
      Run<T, V> x;
      x.load((const T *)weight + d0), x.floats(w0);
      x.load((const T *)weight + d1), x.floats(w1);
    }
    if constexpr (NORM == 2) {
#pragma unroll
      for (int e = 0; e < V; e += 4)
        *(float4 *)(w0 + e) = *(const float4 *)((const float *)weight + d0 + e), *(float4 *)(w1 + e) = *(const float4 *)((const float *)weight + d1 + e);
    }
  };
  const int all = step * kRotateSteps;
  float w0[V], w1[V];
  weights(w0, w1, a.q_weight);
  Rows xk;
  if (a.kv_heads) load(xk, start, a.kv_heads, k);
  turn(xq, start, a.heads, a.q_out + token * a.q_out_stride, w0, w1);
  for (int r0 = start + all; __any_sync(~0u, r0 < a.heads); r0 += all) {
    load(xq, r0, a.heads, q);
    turn(xq, r0, a.heads, a.q_out + token * a.q_out_stride, w0, w1);
  }
  if (!a.kv_heads) return;
  weights(w0, w1, a.k_weight);
  turn(xk, start, a.kv_heads, a.k_out + token * a.k_out_stride, w0, w1);
  for (int r0 = start + all; __any_sync(~0u, r0 < a.kv_heads); r0 += all) {
    load(xk, r0, a.kv_heads, k);
    turn(xk, r0, a.kv_heads, a.k_out + token * a.k_out_stride, w0, w1);
  }
}

}  // namespace paged
}  // namespace ocrvl
