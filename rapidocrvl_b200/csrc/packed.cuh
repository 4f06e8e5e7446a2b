// The packed cache: K and V in 4 bits, quantised as they are written
// (ocrvl_op_packed_append) and read back (ocrvl_op_packed_read).
//
// 32 consecutive dims x of a position's row share a scale s, and each is c s:
//   s = max |x| / 7 rounded to five significant bits, c = x / s rounded to a whole number, -7 .. 7
// Five bits times three are eight, so every c s is a bf16 number: the products that
// read a cache take it without a further rounding.  Codes c + 8 are stored as halfwords
// of four dims, those of the groups side by side: halfword (d / 4 % 8) G + d / 32 holds
// dims d .. d + 3 (G = D / 32 groups), so that what a lane of the matrix instructions needs
// of all groups lies together.
#pragma once
#include "paged.cuh"

namespace ocrvl {
namespace paged {

// One layer of a packed cache, or all of them: bytes but for the table's stride.
struct Packed {
  char *k, *v, *k_scale, *v_scale;
  const int *table;
  long long page, layer, head, scale_page, scale_layer, scale_head, table_stride;
  int shift, num_pages, max_pages;

  // the page of a position, or -1
  __device__ __forceinline__ int page_of(int b, int pos) const {
    const int e = pos >> shift;
    if (pos < 0 || e >= max_pages) return -1;
    const int pg = table[b * table_stride + e];
    return pg >= 0 && pg < num_pages ? pg : -1;
  }
};

struct PackArgs {
  Packed c;
  char *k, *v;  // [layer][token][head][dim]
  const int *lens, *indptr, *path, *n_path;
  int *new_lens;
  long long token, layer;  // bytes, of k and v
  int capacity, layers, batch, kv_heads, n_tokens, max_path;
};

constexpr int kPackLayers = 3;     // layers a warp takes of a token at once
constexpr int kPackThreads = 256;

// 8 values as 32-bit floats, and back.
__device__ __forceinline__ void load8(float (&x)[8], const float *p) {
  const float4 a = __ldg((const float4 *)p), b = __ldg((const float4 *)p + 1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t two);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t two) { return __half22float2(*reinterpret_cast<__half2 *>(&two)); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t two) {
  return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T *p) {
  const uint4 a = __ldg((const uint4 *)p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = unpack2<T>(w[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
  *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]);
  *((float4 *)p + 1) = make_float4(x[4], x[5], x[6], x[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
  *(uint4 *)p = make_uint4(pack2(x[0], x[1], T()), pack2(x[2], x[3], T()), pack2(x[4], x[5], T()), pack2(x[6], x[7], T()));
}

// The scale of a group by its largest magnitude: max / 7 rounded to five significant bits, to the even
// one of two.  (A 32-bit quotient is never rounded onto a border between two such numbers that it does not
// lie on: those are six-bit m, 7 m is a float, and the next float is 4/7 of a rounding further at least.)
__device__ __forceinline__ float group_scale(float most) {
  const uint32_t u = __float_as_uint(__fdiv_rn(most, 7.f));
  const uint32_t r = (u + 0x3ffffu + (u >> 19 & 1u)) & 0xfff80000u;
  return r < 0x00800000u ? 0.f : __uint_as_float(r);
}

// Lane i of a row's D / 8 has dims 8 i .. 8 i + 7: of group j = i / 4, halfwords 2 t and 2 t + 1 of it
// (t = i % 4).  Packs them; returns the four bytes at `at` of the row's codes, and the scale.
template <int D>
__device__ __forceinline__ uint32_t pack8(const float (&x)[8], int i, int *at, float *scale) {
  constexpr int G = D / 32;
  // The magnitudes' bits have the order of the numbers, infinities and NaN above all others.
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
  most = max(most, __shfl_xor_sync(~0u, most, 1));
  most = max(most, __shfl_xor_sync(~0u, most, 2));
  const bool finite = most < 0x7f800000u;
  const float s = finite ? group_scale(__uint_as_float(most)) : 0.f;
  uint32_t lo = 0x8888u, hi = 0x8888u;
  if (s > 0.f) {
    lo = hi = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      // The quotient is not rounded onto a border k + 1/2 either ((k + 1/2) s has nine bits), so its nearest
      // whole number is the exact quotient's.
      const uint32_t c = (uint32_t)((int)rintf(__fdiv_rn(x[e], s)) + 8) << e % 4 * 4;
      if (e < 4)
        lo |= c;
      else
        hi |= c;
    }
  }
  *scale = finite ? s : __uint_as_float(0x7fc00000u);
  // two groups' halfwords side by side: the even group's lane takes halfwords 2 t, the odd one's 2 t + 1
  const int j = i / 4, t = i % 4;
  const uint32_t other = __shfl_xor_sync(~0u, j & 1 ? lo : hi, 4);
  *at = (2 * t + (j & 1)) * (2 * G) + (j & ~1) * 2;
  return j & 1 ? other | hi << 16 : lo | other << 16;
}

// The 8 numbers of lane i (as above) of a row whose codes' four bytes at its place are `word`.
template <int D>
__device__ __forceinline__ void unpack8(float (&x)[8], uint32_t word, float scale, int i) {
  const int j = i / 4;
  const uint32_t other = __shfl_xor_sync(~0u, j & 1 ? word & 0xffffu : word >> 16, 4);
  const uint32_t lo = j & 1 ? other : word & 0xffffu, hi = j & 1 ? word >> 16 : other;
#pragma unroll
  for (int e = 0; e < 8; e++) x[e] = (float)((int)((e < 4 ? lo : hi) >> e % 4 * 4 & 15u) - 8) * scale;
}

// A warp an item: K and V of one token in up to kPackLayers layers, all heads; D / 8 lanes a row.
template <typename T, int D>
__global__ void __launch_bounds__(kPackThreads) k_packed_append(const PackArgs a) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES;  // of a row; rows at once
  const int b = blockIdx.y, lane = threadIdx.x & 31, i8 = lane % LANES, sub = lane / LANES;
  const int first = min(max(a.indptr[b], 0), a.n_tokens), count = min(max(a.indptr[b + 1], first), a.n_tokens) - first;
  const int len = min(max(a.lens[b], 0), a.capacity);
  const int n = a.path ? min(max(a.n_path[b], 0), a.max_path) : count;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.new_lens[b] = min(len + n, a.capacity);
  const int groups = (a.layers + kPackLayers - 1) / kPackLayers;
  const long long items = (long long)n * groups;
  for (long long it = blockIdx.x * (kPackThreads / 32) + (threadIdx.x >> 5); it < items; it += gridDim.x * (kPackThreads / 32)) {
    const int i = (int)(it / groups), layer0 = (int)(it % groups) * kPackLayers;
    if (i >= a.capacity - len) break;
    const int pos = len + i;
    const int node = a.path ? a.path[(long long)b * a.max_path + i] : i;
    if (node < 0 || node >= count) continue;
    const int pg = a.c.page_of(b, pos);
    if (pg < 0) continue;
    const int in_page = pos & ((1 << a.c.shift) - 1);
    for (int h0 = 0; h0 < a.kv_heads; h0 += ROWS) {
      const int h = h0 + sub;
      const bool there = h < a.kv_heads;
      const long long from = layer0 * a.layer + (first + node) * a.token + ((long long)(there ? h : 0) * D + i8 * 8) * (int)sizeof(T);
      const long long to = pg * a.c.page + layer0 * a.c.layer + h * a.c.head + (long long)in_page * (D / 2);
      const long long to_s = pg * a.c.scale_page + layer0 * a.c.scale_layer + h * a.c.scale_head + (long long)in_page * (D / 16) + i8 / 4 * 2;
      float x[2 * kPackLayers][8];
#pragma unroll
      for (int r = 0; r < 2 * kPackLayers; r++)
        if (layer0 + r / 2 < a.layers) load8(x[r], (const T *)((r & 1 ? a.v : a.k) + from + r / 2 * a.layer));
#pragma unroll
      for (int r = 0; r < 2 * kPackLayers; r++) {
        if (layer0 + r / 2 >= a.layers) break;
        int at;
        float s;
        const uint32_t word = pack8<D>(x[r], i8, &at, &s);
        if (!there) continue;
        *(uint32_t *)((r & 1 ? a.c.v : a.c.k) + to + r / 2 * a.c.layer + at) = word;
        if (i8 % 4 == 0)
          *(uint16_t *)((r & 1 ? a.c.v_scale : a.c.k_scale) + to_s + r / 2 * a.c.scale_layer) = (uint16_t)(__float_as_uint(s) >> 16);
      }
    }
  }
}

// The other way, items as above; a token without a page reads as 0.
template <typename T, int D>
__global__ void __launch_bounds__(kPackThreads) k_packed_read(const PackArgs a) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES, G = D / 32;
  const int b = blockIdx.y, lane = threadIdx.x & 31, i8 = lane % LANES, sub = lane / LANES;
  const int first = min(max(a.indptr[b], 0), a.n_tokens), count = min(max(a.indptr[b + 1], first), a.n_tokens) - first;
  const int len = min(max(a.lens[b], 0), a.capacity);
  const int groups = (a.layers + kPackLayers - 1) / kPackLayers;
  const int at = (2 * (i8 % 4) + (i8 / 4 & 1)) * (2 * G) + (i8 / 4 & ~1) * 2;
  const long long items = (long long)count * groups;
  for (long long it = blockIdx.x * (kPackThreads / 32) + (threadIdx.x >> 5); it < items; it += gridDim.x * (kPackThreads / 32)) {
    const int i = (int)(it / groups), layer0 = (int)(it % groups) * kPackLayers;
    const int pos = i < a.capacity - len ? len + i : -1;
    const int pg = a.c.page_of(b, pos), in_page = pos & ((1 << a.c.shift) - 1);  // without a page nothing of it is used
    for (int h0 = 0; h0 < a.kv_heads; h0 += ROWS) {
      const int h = h0 + sub;
      const bool there = h < a.kv_heads, mapped = there && pg >= 0;
      const long long to = layer0 * a.layer + (first + i) * a.token + ((long long)h * D + i8 * 8) * (int)sizeof(T);
      const long long from = (mapped ? pg : 0) * a.c.page + layer0 * a.c.layer + h * a.c.head + (long long)in_page * (D / 2) + at;
      const long long from_s = (mapped ? pg : 0) * a.c.scale_page + layer0 * a.c.scale_layer + h * a.c.scale_head + (long long)in_page * (D / 16) + i8 / 4 * 2;
      uint32_t word[2 * kPackLayers], s[2 * kPackLayers];
#pragma unroll
      for (int r = 0; r < 2 * kPackLayers; r++) {
        word[r] = 0x88888888u, s[r] = 0;
        if (mapped && layer0 + r / 2 < a.layers) {
          word[r] = __ldg((const uint32_t *)((r & 1 ? a.c.v : a.c.k) + from + r / 2 * a.c.layer));
          s[r] = __ldg((const uint16_t *)((r & 1 ? a.c.v_scale : a.c.k_scale) + from_s + r / 2 * a.c.scale_layer));
        }
      }
#pragma unroll
      for (int r = 0; r < 2 * kPackLayers; r++) {
        if (layer0 + r / 2 >= a.layers) break;
        float x[8];
        unpack8<D>(x, word[r], __uint_as_float(s[r] << 16), i8);
        if (there) store8((T *)((r & 1 ? a.v : a.k) + to + r / 2 * a.layer), x);
      }
    }
  }
}

}  // namespace paged
}  // namespace ocrvl
