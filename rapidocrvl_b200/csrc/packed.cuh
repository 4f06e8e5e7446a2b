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
//
// A warp takes 16 positions of one (layer, K or V, head), so that a page is looked up and addresses are worked out once for 16
// rows (a warp for single rows: the bf16 read below took 45.6 us, this split 26.8 at once).  Read: 23,600 bf16 positions of 4 layers 23.4 us, 5.3
// TB/s; 1,497 f32 positions of 18 layers 12.4 us, 5.1 TB/s, bound by memory.  Append and
// read of 1,241 bf16 tokens of 18 layers 19.4 us, bound by the append's instructions (a quotient exact to its rounding, the
// group's largest); of the accepted paths of 64 sequences 11.0 us, two launches with three loads behind one another each.
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

constexpr int kPackWarps = 4, kPackThreads = kPackWarps * 32;
template <typename T>
constexpr int kPackRows = sizeof(T) == 4 ? 2 : 4;  // steps whose loads go out together

// 8 values of a row: as they lie in memory, and as 32-bit floats.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t two);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t two) { return __half22float2(*reinterpret_cast<__half2 *>(&two)); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t two) {
  return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];

  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = __ldg((const uint4 *)p + i);
  }
  __device__ __forceinline__ void floats(float (&x)[8]) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = __uint_as_float(u[i]);
    } else {
      const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 f = unpack2<T>(u[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    }
  }
};

// Lifted nibbles: nibble i of both halfwords as 16 + nibble, two numbers of B (at the top of the mantissa of 16).  The base may
// come from a register: as a constant it costs another instruction in loops that have no register left.
template <typename B>
__device__ __forceinline__ constexpr uint32_t lifted_base() {
  return std::is_same<B, __half>::value ? 0x64006400u : 0x41804180u;  // f16's, 1024 twice, is for whole numbers of loops
}
template <typename B>
__device__ __forceinline__ uint32_t lifted(uint32_t x, int i, uint32_t base = std::is_same<B, __half>::value ? 0x4c004c00u : 0x41804180u) {
  if constexpr (std::is_same<B, __half>::value)
    return ((i < 2 ? x << (6 - 4 * i) : x >> (4 * i - 6)) & 0x03c003c0u) | base;
  else
    return ((i < 1 ? x << 3 : x >> (4 * i - 3)) & 0x00780078u) | base;
}
template <typename B>
struct Two;
template <>
struct Two<__half> {
  using V = __half2;
};
template <>
struct Two<__nv_bfloat16> {
  using V = __nv_bfloat162;
};
template <typename B>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  using V = typename Two<B>::V;
  V r = __hfma2(*reinterpret_cast<V *>(&a), *reinterpret_cast<V *>(&b), *reinterpret_cast<V *>(&c));
  return *reinterpret_cast<uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t add2(uint32_t a, uint32_t b) {  // of f16
  __half2 r = __hadd2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
  return *reinterpret_cast<uint32_t *>(&r);
}
template <typename B>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  using V = typename Two<B>::V;
  V r = __hsub2(*reinterpret_cast<V *>(&a), *reinterpret_cast<V *>(&b));
  return *reinterpret_cast<uint32_t *>(&r);
}
template <typename B>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  using V = typename Two<B>::V;
  V r = __hmul2(*reinterpret_cast<V *>(&a), *reinterpret_cast<V *>(&b));
  return *reinterpret_cast<uint32_t *>(&r);
}
// Nibble i of both halfwords of codes as c times their scales: exact.  In one fused step where there is room for 24 s;
// f16 has none for the largest scales of f16 numbers (nor bf16 from 2^-5 of its largest on), so that the 24 is taken off before.
template <typename B, bool ROOM = !std::is_same<B, __half>::value>
struct Scaled {
  uint32_t s, minus;
  __device__ __forceinline__ explicit Scaled(uint32_t s_) : s(s_), minus(0) {
    static_assert(!ROOM || !std::is_same<B, __half>::value, "");
    if constexpr (ROOM) minus = mul2<B>(s, 0xc1c0c1c0u);  // -24
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t codes, int i, uint32_t base) const {  // with room
    return fma2<B>(lifted<B>(codes, i, base), s, minus);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t codes, int i) const {
    if constexpr (ROOM)
      return fma2<B>(lifted<B>(codes, i), s, minus);
    else
      return mul2<B>(sub2<B>(lifted<B>(codes, i), std::is_same<B, __half>::value ? 0x4e004e00u : 0x41c041c0u), s);
  }
};
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
__device__ __forceinline__ uint32_t halves(uint32_t a, uint32_t b, int high) { return high ? high_halves(a, b) : low_halves(a, b); }

// x / y correctly rounded but for its last 2^-45, for y's reciprocal to 2^-22 and a quotient of ordinary size: the first
// quotient's rest is exact in one fused step, and what the second adds is off by 2^-22 of itself.
__device__ __forceinline__ float quotient(float x, float y, float reciprocal) {
  const float q = x * reciprocal;
  return fmaf(fmaf(-q, y, x), reciprocal, q);
}

// The scale of a group by its largest magnitude: max / 7 rounded to five significant bits, to the even
// one of two.  (A 32-bit quotient is never rounded onto a border between two such numbers that it does not
// lie on: those are six-bit m, 7 m is a float, and the next float is 4/7 of a rounding further at least.)
// Below 63/64 of 2^-126 that is no normal number.
__device__ __forceinline__ float group_scale(float most) {
  const float y = quotient(most, 7.f, 1.f / 7.f);
  const uint32_t u = __float_as_uint(y), r = (u + 0x3ffffu + (u >> 19 & 1u)) & 0xfff80000u;
  return y < 0x1.f8p-127f ? 0.f : __uint_as_float(r);
}

// Lane i of a row's D / 8 has dims 8 i .. 8 i + 7: of group j = i / 4, halfwords 2 t and 2 t + 1 of it
// (t = i % 4).  Packs them; returns the four bytes at place(i) of the row's codes, and the scale.
template <int D>
__device__ __forceinline__ int place(int i) {
  const int j = i / 4, t = i % 4;
  return (2 * t + (j & 1)) * (D / 16) + (j & ~1) * 2;
}
template <int D, typename T>
__device__ __forceinline__ uint32_t pack8(const Eight<T> &e8, int i, float *scale) {
  // The magnitudes' bits have the order of the numbers, infinities and NaN above all others.
  uint32_t most;
  bool finite;
  float x[8];
  e8.floats(x);
  if constexpr (sizeof(T) == 4) {
    most = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
    most = max(most, __shfl_xor_sync(~0u, most, 1));
    most = max(most, __shfl_xor_sync(~0u, most, 2));
    finite = most < 0x7f800000u;
  } else {
    const uint32_t m = 0x7fff7fffu;
    uint32_t two = __vmaxu2(__vmaxu2(e8.w[0].x & m, e8.w[0].y & m), __vmaxu2(e8.w[0].z & m, e8.w[0].w & m));
    two = __vmaxu2(two, __shfl_xor_sync(~0u, two, 1));
    two = __vmaxu2(two, __shfl_xor_sync(~0u, two, 2));
    const uint32_t one = max(two & 0xffffu, two >> 16);
    finite = one < (std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u);
    most = __float_as_uint(unpack2<T>(one).x);
  }
  const float s = finite ? group_scale(__uint_as_float(most)) : 0.f;
  // s is 2^-126 to 2^126, or 0: its reciprocal is an ordinary number
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  inv = s > 0.f ? inv : 0.f;
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    // The quotient is not rounded onto a border k + 1/2 either ((k + 1/2) s has nine bits), so its nearest
    // whole number is the exact quotient's.  In 1.5 2^23 + 8 + q the sum's rounding makes it whole (of two the even), and its
    // last bits are c + 8.
    c[e] = __float_as_uint(quotient(x[e], s, inv) + 12582920.f);
  }
  uint32_t lo = c[0] + (c[1] << 4) + (c[2] << 8) + (c[3] << 12), hi = c[4] + (c[5] << 4) + (c[6] << 8) + (c[7] << 12);
  if (!finite) lo = hi = 0x8888u;
  *scale = finite ? s : __uint_as_float(0x7fc00000u);
  // two groups' halfwords side by side: the even group's lane takes halfwords 2 t, the odd one's 2 t + 1
  const bool odd = i / 4 & 1;
  const uint32_t other = __shfl_xor_sync(~0u, odd ? lo : hi, 4);
  return odd ? low_halves(other, hi) : low_halves(lo, other);
}

// Stores the 8 numbers of lane i (as above) of a row whose codes' four bytes at its place are `word`, scale twice.  sectors: `to` is
// 32-byte aligned, so that f32 goes out as whole sectors of memory, not as halves of them (1,497 tokens of 18 layers 18.3 us, 12.5 so).
template <int D, typename T>
__device__ __forceinline__ void unpack8(T *to, uint32_t word, uint32_t scale, int i, bool there, bool sectors) {
  using B = __nv_bfloat16;
  const bool odd = i / 4 & 1;
  const uint32_t other = __shfl_xor_sync(~0u, odd ? word : word >> 16, 4);
  const uint32_t codes = odd ? __byte_perm(other, word, 0x7610) : low_halves(word, other);
  const Scaled<B, false> by(scale);
  uint32_t x[4], y[4];  // dims (k, 4 + k), then in order
#pragma unroll
  for (int k = 0; k < 4; k++) x[k] = by(codes, k);
  y[0] = low_halves(x[0], x[1]), y[1] = low_halves(x[2], x[3]), y[2] = high_halves(x[0], x[1]), y[3] = high_halves(x[2], x[3]);
  if constexpr (std::is_same<T, B>::value) {
    if (there) *(uint4 *)to = make_uint4(y[0], y[1], y[2], y[3]);
  } else {
    float f[8];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float2 z = unpack2<B>(y[k]);
      f[2 * k] = z.x, f[2 * k + 1] = z.y;
    }
    if (!there) return;
    if constexpr (sizeof(T) == 4) {
      if (sectors) {
        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]),
                     "f"(f[5]), "f"(f[6]), "f"(f[7])
                     : "memory");
      } else {
        *(float4 *)to = make_float4(f[0], f[1], f[2], f[3]);
        *((float4 *)to + 1) = make_float4(f[4], f[5], f[6], f[7]);
      }
    } else {
      *(uint4 *)to = make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()), pack2(f[4], f[5], T()), pack2(f[6], f[7], T()));
    }
  }
}

// What a warp takes: chunks of 16 positions of one (layer, K or V, head), blockIdx.x and further on of the
// sequence blockIdx.y's, so that a page is looked up, and addresses are worked out, once for 16 rows.  D / 8 lanes a row,
// kPackRows rows on their way at once.
template <int D>
struct PackItem {
  static constexpr int LANES = D / 8, ROWS = 32 / LANES, STEPS = kChunk / ROWS;  // of a row; rows at once; steps a chunk
  int first, count, len;   // of the sequence: tokens, cached positions
  int layer, v, head;

  __device__ __forceinline__ PackItem(const PackArgs &a, int b) {
    first = min(max(a.indptr[b], 0), a.n_tokens), count = min(max(a.indptr[b + 1], first), a.n_tokens) - first;
    len = min(max(a.lens[b], 0), a.capacity);
  }
  __device__ __forceinline__ bool at(const PackArgs &a, int c) {
    if (c >= a.layers * 2 * a.kv_heads) return false;
    const int lv = c / a.kv_heads;
    head = c - lv * a.kv_heads, v = lv & 1, layer = lv >> 1;
    return true;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kPackThreads) k_packed_append(const PackArgs a) {
  using I = PackItem<D>;
  const int b = blockIdx.y, lane = threadIdx.x & 31, i8 = lane % I::LANES, sub = lane / I::LANES;
  pdl_wait();
  pdl_launch();
  I x(a, b);
  const int n = min(a.path ? min(max(a.n_path[b], 0), a.max_path) : x.count, a.capacity - x.len);
  if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) a.new_lens[b] = x.len + n;
  if (n == 0) return;
  const int end = x.len + n, codes_at = sub * (D / 2) + place<D>(i8), scales_at = sub * (D / 16) + i8 / 4 * 2;
  for (int c = blockIdx.z * kPackWarps + (threadIdx.x >> 5); x.at(a, c); c += gridDim.z * kPackWarps) {
    const char *from = (x.v ? a.v : a.k) + x.layer * a.layer + x.first * a.token + (x.head * D + i8 * 8) * (long long)sizeof(T);
    for (int p0 = (x.len / kChunk + blockIdx.x) * kChunk; p0 < end; p0 += gridDim.x * kChunk) {
      const int pg = a.c.page_of(b, p0);
      const long long in_page = p0 & ((1 << a.c.shift) - 1);
      char *codes = (x.v ? a.c.v : a.c.k) + pg * a.c.page + x.layer * a.c.layer + x.head * a.c.head + in_page * (D / 2) + codes_at;
      char *scales = (x.v ? a.c.v_scale : a.c.k_scale) + pg * a.c.scale_page + x.layer * a.c.scale_layer + x.head * a.c.scale_head +
                     in_page * (D / 16) + scales_at;
      const int first = max(0, x.len - p0) / I::ROWS, last = min(I::STEPS, (end - p0 + I::ROWS - 1) / I::ROWS);  // steps with tokens
#pragma unroll 1
      for (int s0 = first; s0 < last; s0 += kPackRows<T>) {
        Eight<T> y[kPackRows<T>];
        bool there[kPackRows<T>];
#pragma unroll
        for (int r = 0; r < kPackRows<T>; r++) {
          const int i = p0 - x.len + (s0 + r) * I::ROWS + sub;
          there[r] = i >= 0 && i < n && s0 + r < last;
          const int node = there[r] && a.path ? a.path[(long long)b * a.max_path + i] : i;
          there[r] = there[r] && node >= 0 && node < x.count;
          if (there[r]) y[r].load((const T *)(from + node * a.token));  // not waiting for the page
        }
#pragma unroll
        for (int r = 0; r < kPackRows<T>; r++) {
          if (!__any_sync(~0u, there[r])) continue;
          float s;
          const uint32_t word = pack8<D>(y[r], i8, &s);
          if (!there[r] || pg < 0) continue;
          *(uint32_t *)(codes + (s0 + r) * (I::ROWS * D / 2)) = word;
          if (i8 % 4 == 0) *(uint16_t *)(scales + (s0 + r) * (I::ROWS * D / 16)) = (uint16_t)(__float_as_uint(s) >> 16);
        }
      }
    }
  }
}

// A token without a page reads as 0.
template <typename T, int D>
__global__ void __launch_bounds__(kPackThreads) k_packed_read(const PackArgs a) {
  using I = PackItem<D>;
  const int b = blockIdx.y, lane = threadIdx.x & 31, i8 = lane % I::LANES, sub = lane / I::LANES;
  pdl_wait();
  pdl_launch();
  I x(a, b);
  if (x.count == 0) return;
  const bool sectors = (((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.token | (uintptr_t)a.layer) & 31) == 0;
  const int codes_at = sub * (D / 2) + place<D>(i8), scales_at = sub * (D / 16) + i8 / 4 * 2;
  for (int c = blockIdx.z * kPackWarps + (threadIdx.x >> 5); x.at(a, c); c += gridDim.z * kPackWarps) {
    char *to = (x.v ? a.v : a.k) + x.layer * a.layer + x.first * a.token + (x.head * D + i8 * 8) * (long long)sizeof(T);
    const int skip = x.len % kChunk, chunks = (int)(((long long)skip + x.count + kChunk - 1) / kChunk);
    const char *codes0 = (x.v ? a.c.v : a.c.k) + x.layer * a.c.layer + x.head * a.c.head + codes_at;
    const char *scales0 = (x.v ? a.c.v_scale : a.c.k_scale) + x.layer * a.c.scale_layer + x.head * a.c.scale_head + scales_at;
    uint32_t word_next[I::STEPS], s_next[I::STEPS];  // of the chunk after the one that is stored
    auto fetch = [&](int ch) {
      const long long p0 = (x.len / kChunk + (long long)ch) * kChunk;
      const int pg = p0 < a.capacity ? a.c.page_of(b, (int)p0) : -1;
      const long long in_page = p0 & ((1 << a.c.shift) - 1);
      const char *codes = codes0 + pg * a.c.page + in_page * (D / 2), *scales = scales0 + pg * a.c.scale_page + in_page * (D / 16);
#pragma unroll
      for (int r = 0; r < I::STEPS; r++) {
        word_next[r] = 0x88888888u, s_next[r] = 0;
        if (pg >= 0) {  // the page holds the whole chunk
          word_next[r] = __ldg((const uint32_t *)(codes + r * (I::ROWS * D / 2)));
          s_next[r] = __ldg((const uint16_t *)(scales + r * (I::ROWS * D / 16)));
        }
      }
    };
    if ((int)blockIdx.x < chunks) fetch(blockIdx.x);
    for (int ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
      uint32_t word[I::STEPS], s[I::STEPS];
#pragma unroll
      for (int r = 0; r < I::STEPS; r++) word[r] = word_next[r], s[r] = s_next[r];
      if (ch + gridDim.x < chunks) fetch(ch + gridDim.x);
      const int i0 = (int)((long long)ch * kChunk - skip);
#pragma unroll
      for (int r = 0; r < I::STEPS; r++) {
        const int i = i0 + r * I::ROWS + sub;
        unpack8<D>((T *)(to + i * a.token), word[r], __byte_perm(s[r], 0, 0x1010), i8, i >= 0 && i < x.count, sectors);
      }
    }
  }
}

}  // namespace paged
}  // namespace ocrvl
