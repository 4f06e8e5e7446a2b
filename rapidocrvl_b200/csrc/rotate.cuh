// Queries and keys of new tokens: each head's norm, if there is one, and the
// rotation by positions of several axes, in one pass (ocrvl_op_rotate).
//
//   y = x / sqrt(mean x^2 + eps) * w
//   pair p (dims p and p + pairs, or 2 p and 2 p + 1): angle = pos[axis p] freq[p]
//   (u, v) -> (u cos - v sin, v cos + u sin);  dims behind 2 pairs stay y
// A token's heads lie side by side, so a warp streams them as they are through a ring of its own in shared
// memory (cp.async: what is on its way costs no registers), a batch of rows at a time, and goes on
// with the tokens that follow it.  It works out a token's cosines and sines once, two a lane, then takes a row with a lane
// for 2 V dims, two numbers an instruction.  The angle is a 64-bit product of turns, whose whole part is dropped before
// it becomes 32 bits, so far positions keep their last bits.
//
// 9,928 bf16 tokens of 16 + 2 heads of 128, normed: 23.9 us, 3.8 TB/s, where a plain copy of them takes 17.5; 1,200 warp
// instructions a token.  Rows loaded into registers, one number an instruction: 30.5; the ring and pairs of numbers made it 25.1.  4,900 f16 patches of 16 + 16 heads of 72: 13.5 us.  One token: 5.8 us, a launch and two loads.
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
  int steps, q_batches, batches;    // of a batch; of the queries; of a token
  float eps, one_dim;               // 1 / dim
  double turns[kRotateMost];  // freq / 2 pi
  unsigned char axis[kRotateMost];
};

// Two 32-bit numbers in a register pair.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ float2 both(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
  Pair p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
  return p;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(a), "l"(b), "l"(c));
  return p;
}

// V values: from memory (shared or not), and to it.
template <typename T, int V, bool SHARED>
__device__ __forceinline__ void load_run(Pair (&x)[V / 2], const T *p) {
  uint32_t w[V * sizeof(T) / 4];
  if constexpr (V * sizeof(T) == 16) {
    if constexpr (SHARED)
      lds4u(reinterpret_cast<uint32_t(&)[4]>(w), smem_addr(p));
    else
      *(uint4 *)w = *(const uint4 *)p;
  } else {
    if constexpr (SHARED)
      asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(smem_addr(p)));
    else
      *(uint2 *)w = *(const uint2 *)p;
  }
#pragma unroll
  for (int i = 0; i < V / 2; i++) {
    if constexpr (sizeof(T) == 4) {
      x[i] = pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else {
      const float2 f = unpack2<T>(w[i]);
      x[i] = pair(f.x, f.y);
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_run(T *p, const Pair (&x)[V / 2]) {
  float2 f[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; i++) f[i] = both(x[i]);
  if constexpr (sizeof(T) == 4)
    *(float4 *)p = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
  else if constexpr (V == 8)
    *(uint4 *)p = make_uint4(pack2(f[0].x, f[0].y, T()), pack2(f[1].x, f[1].y, T()), pack2(f[2].x, f[2].y, T()), pack2(f[3].x, f[3].y, T()));
  else
    *(uint2 *)p = make_uint2(pack2(f[0].x, f[0].y, T()), pack2(f[1].x, f[1].y, T()));
}

constexpr int kRotateSteps = 4;  // of a batch at most: rows at once
constexpr int kRotateStages = 3;
template <typename T, int V>
constexpr int kRotateStage = 64 * kRotateSteps * V * (int)sizeof(T);  // bytes: 32 lanes of 2 V values a step
template <typename T, int V>
constexpr int kRotateSmem = kRotateWarps * (kRotateStages * kRotateStage<T, V> + 2 * kRotateMost * 4);
constexpr int kRotateBlocks = 2;  // an SM

// NORM: 0 none, 1 weights of T, 2 weights of f32.  LANES: of a row, 0: any number.
template <typename T, int V, int NORM, int LANES>
__global__ void __launch_bounds__(kRotateWarps * 32, kRotateBlocks) k_rotate(const __grid_constant__ RotateArgs a) {
  extern __shared__ __align__(16) char sm[];
  constexpr int STAGE = kRotateStage<T, V>, NS = kRotateStages;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  char *ring = sm + warp * (NS * STAGE);
  float *cs = (float *)(sm + kRotateWarps * NS * STAGE) + warp * (2 * kRotateMost), *sn = cs + kRotateMost;
  // this warp's tokens, and of each its batches
  long long token = warp * gridDim.x + blockIdx.x;
  const int next = kRotateWarps * gridDim.x;
  if (token >= a.n_tokens || blockIdx.y >= a.batches) {  // the whole warp
    pdl_wait();  // on every path: this grid's end is to mean that of the one before it too
    return;
  }
  const int lanes = LANES ? LANES : a.lanes, at_once = LANES ? 32 / (LANES ? LANES : 1) : a.at_once;
  const int sub = LANES ? lane / (LANES ? LANES : 1) : lane * a.lane_factor >> 16, v = lane - sub * lanes, rotated = a.pairs / V;
  const int d0 = v >= rotated ? 2 * a.pairs + 2 * V * (v - rotated) : a.neighbours ? 2 * V * v : V * v;  // the lane's two runs of V dims
  const int d1 = v >= rotated || a.neighbours ? d0 + V : a.pairs + d0;
  const int batch_rows = at_once * a.steps, row_bytes = a.dim * (int)sizeof(T);
  // Copies the batch that is next in line: (to_token, to_batch), to_stage.
  long long to_token = token;
  int to_batch = blockIdx.y, to_stage = 0;
  const uint32_t ring_at = smem_addr(ring) + lane * 16;
  auto fetch = [&] {
    if (to_token < a.n_tokens) {
      const bool is_q = to_batch < a.q_batches;
      const int r0 = (is_q ? to_batch : to_batch - a.q_batches) * batch_rows, n = min(batch_rows, (is_q ? a.heads : a.kv_heads) - r0);
      const char *from = (is_q ? a.q + to_token * a.q_stride : a.k + to_token * a.k_stride) + (long long)r0 * row_bytes + lane * 16;
      const int bytes = n * row_bytes - lane * 16;
      const uint32_t to = ring_at + to_stage * STAGE;
#pragma unroll
      for (int i = 0; i < STAGE / 512; i++)
        if (i * 512 < bytes) copy16(to + i * 512, from + i * 512);
      if ((to_batch += gridDim.y) >= a.batches) to_batch = blockIdx.y, to_token += next;
    }
    to_stage = to_stage + 1 == NS ? 0 : to_stage + 1;
    copy_commit();
  };
  pdl_wait();
  pdl_launch();
#pragma unroll
  for (int i = 0; i < NS - 1; i++) fetch();
  // The tables through their addresses: as constants, which a warp reads one address at a time, they took 4 us of 31.
  const double *turns = a.turns;
  const unsigned char *axis = a.axis;
  asm("" : "+l"(turns));
  asm("" : "+l"(axis));
  constexpr int MINE = kRotateMost / 32;
  double my_turns[MINE];
  int my_axis[MINE], my_pos[MINE];
#pragma unroll
  for (int i = 0; i < MINE; i++)
    if (i * 32 + lane < a.pairs) {
      my_turns[i] = turns[i * 32 + lane], my_axis[i] = axis[i * 32 + lane];
      my_pos[i] = __ldg(a.pos + token * a.pos_stride + my_axis[i]);
    }

  Pair c[V / 2] = {}, s[V / 2] = {}, w0[V / 2], w1[V / 2];
  auto weights = [&](const void *weight) {
    if constexpr (NORM == 1) load_run<T, V, false>(w0, (const T *)weight + d0), load_run<T, V, false>(w1, (const T *)weight + d1);
    if constexpr (NORM == 2) {
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        load_run<float, 4, false>(reinterpret_cast<Pair(&)[2]>(w0[e / 2]), (const float *)weight + d0 + e);
        load_run<float, 4, false>(reinterpret_cast<Pair(&)[2]>(w1[e / 2]), (const float *)weight + d1 + e);
      }
    }
  };
  int stage = 0, weights_of = -1;
  for (; token < a.n_tokens; token += next) {
#pragma unroll
    for (int i = 0; i < MINE; i++)
      if (i * 32 + lane < a.pairs) {
        const double x = (double)my_pos[i] * my_turns[i];
        sincospif(2.f * (float)(x - rint(x)), &sn[i * 32 + lane], &cs[i * 32 + lane]);
        if (next < a.n_tokens - token) my_pos[i] = __ldg(a.pos + (token + next) * a.pos_stride + my_axis[i]);
      }
    __syncwarp();
    if (v < rotated) {
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        load_run<float, 4, true>(reinterpret_cast<Pair(&)[2]>(c[e / 2]), cs + V * v + e);
        load_run<float, 4, true>(reinterpret_cast<Pair(&)[2]>(s[e / 2]), sn + V * v + e);
      }
    }
    for (int batch = blockIdx.y; batch < a.batches; batch += gridDim.y) {
      const bool is_q = batch < a.q_batches;
      if (NORM > 0 && weights_of != is_q) weights(is_q ? a.q_weight : a.k_weight), weights_of = is_q;
      copy_wait<NS - 2>();
      __syncwarp();  // the stage before this one is read by all lanes, the cosines too
      fetch();
      const int r0 = (is_q ? batch : batch - a.q_batches) * batch_rows, n = min(batch_rows, (is_q ? a.heads : a.kv_heads) - r0);
      T *to = (T *)(is_q ? a.q_out + token * a.q_out_stride : a.k_out + token * a.k_out_stride) + ((long long)r0 + sub) * a.dim;
      const T *from = (const T *)(ring + stage * STAGE) + sub * a.dim;
      stage = stage + 1 == NS ? 0 : stage + 1;
#pragma unroll
      for (int i = 0; i < kRotateSteps; i++) {
        if (i * at_once >= n) break;
        const bool there = sub < at_once && i * at_once + sub < n;
        const int at = i * at_once * a.dim;
        Pair x[V / 2], y[V / 2];
        load_run<T, V, true>(x, from + at + d0), load_run<T, V, true>(y, from + at + d1);
        Pair c1[V / 2], s1[V / 2], m1[V / 2];  // cosines, sines and the sines' negatives, by the norm
        if constexpr (NORM > 0) {
          Pair sq[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < V / 2; e++) sq[0] = fma(x[e], x[e], sq[0]), sq[1] = fma(y[e], y[e], sq[1]);
          const float2 p = both(sq[0]), q = both(sq[1]);
          float sum = (p.x + p.y) + (q.x + q.y);
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
          const Pair i2 = pair(inv, inv), n2 = pair(-inv, -inv);
#pragma unroll
          for (int e = 0; e < V / 2; e++) {
            x[e] = mul(x[e], w0[e]), y[e] = mul(y[e], w1[e]);
            c1[e] = mul(c[e], i2), s1[e] = mul(s[e], i2), m1[e] = mul(s[e], n2);
          }
          if (v >= rotated) {
#pragma unroll
            for (int e = 0; e < V / 2; e++) x[e] = mul(x[e], i2), y[e] = mul(y[e], i2);
          }
        } else {
          const Pair n2 = pair(-1.f, -1.f);
#pragma unroll
          for (int e = 0; e < V / 2; e++) c1[e] = c[e], s1[e] = s[e], m1[e] = mul(s[e], n2);
        }
        if (v < rotated) {
          if (!a.neighbours) {
#pragma unroll
            for (int e = 0; e < V / 2; e++) {
              const Pair u = x[e];
              x[e] = fma(y[e], m1[e], mul(u, c1[e])), y[e] = fma(u, s1[e], mul(y[e], c1[e]));
            }
          } else {
#pragma unroll
            for (int e = 0; e < V; e++) {  // pair e of the lane: in x, then in y
              Pair &p = e < V / 2 ? x[e] : y[e - V / 2];
              const float2 u = both(p), cc = both(c1[e / 2]), ss = both(s1[e / 2]);
              const float co = e & 1 ? cc.y : cc.x, si = e & 1 ? ss.y : ss.x;
              p = pair(u.x * co - u.y * si, u.y * co + u.x * si);
            }
          }
        }
        if (there) store_run<T, V>(to + at + d0, x), store_run<T, V>(to + at + d1, y);
      }
    }
    __syncwarp();  // the cosines are read
  }
  copy_wait<0>();
}

}  // namespace paged
}  // namespace ocrvl
