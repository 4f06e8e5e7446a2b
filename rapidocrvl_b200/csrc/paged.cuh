// Device helpers of the paged-cache operators: the cache's addressing, warp
// fragments of the 32-bit (tf32, three products) and 16-bit matrix
// instructions, asynchronous copies.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace ocrvl {
namespace paged {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kChunk = 16;  // positions a warp takes at a time: never more than one page

// One layer of a cache.
struct Cache {
  const char *k, *v;  // at the layer
  const int *table;
  long long page_bytes, head_bytes, table_stride;
  int token_bytes, max_pages, num_pages, page_shift;
};

// The sequences' cached lengths and drafted tokens, with every value from
// device memory brought into its range.
struct Seqs {
  const int *lens, *indptr;
  int batch, n_tokens, max_draft, capacity;  // capacity: positions the table has room for

  __device__ int len(int b) const { return min(max(lens[b], 0), capacity); }
  // first token and count
  __device__ int tokens(int b, int *first) const {
    const int lo = min(max(indptr[b], 0), n_tokens), hi = min(max(indptr[b + 1], lo), n_tokens);
    *first = lo;
    return min(hi - lo, max_draft);
  }
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes, or 16 zero bytes where !there (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float exp2_(float x) {  // 0 at -inf; relative error below 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// sum + low += x, without the roundings of sum: over 100,000 positions, each far below the sum so far, those
// would add up to 1e-4 of it.
__device__ __forceinline__ void add_exactly(float &sum, float &low, float x) {
  const float s = sum + x, y = s - sum;
  low += (sum - (s - y)) + (x - y);
  sum = s;
}

// ---- fragments ----------------------------------------------------------
// x = hi + lo with hi the nearest tf32 (11 significant bits); lo keeps the
// rest, of which the instruction takes 11 bits: 22 bits of x in all.  Past the
// largest tf32 hi is that one, so that it is never infinite: an infinity or NaN is lo's alone.
__device__ __forceinline__ void split(float x, uint32_t &hi, uint32_t &lo) {
  float y;  // |x| up to what rounds to the largest tf32, with x's sign
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(__uint_as_float(0x7f7fefffu)));
  hi = (__float_as_uint(y) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ float4 lds4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void lds4u(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void sts4u(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t *>(&h);
}

// 8 x 8 16-bit values, a row g and two columns 2 t, 2 t + 1 a lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// The same for 32-bit values: a, b in columns 2 t, 2 t + 1 become those of rows 2 t, 2 t + 1.
__device__ __forceinline__ void transpose8(float a, float b, float &x, float &y) {
  const uint32_t u = __float_as_uint(a), v = __float_as_uint(b);
  const uint32_t lo = transpose8(__byte_perm(u, v, 0x5410)), hi = transpose8(__byte_perm(u, v, 0x7632));
  x = __uint_as_float(__byte_perm(lo, hi, 0x5410));
  y = __uint_as_float(__byte_perm(lo, hi, 0x7632));
}

// What a type's chunk of 16 positions x D looks like in shared memory and how
// the matrix instructions read it.  The positions are the 16 rows of the
// instruction and the query rows its 8 columns, so 8 rows (one token of eight
// heads) fill it: s' = K q' and o' = V' p'.  Rows of K and V are stored
// whole; the 16-byte pieces of a row are exchanged by a rule on the row so that the
// fragment loads of a warp hit 32 different banks.
template <typename T, int D>
struct Tile {
  static constexpr bool f32 = sizeof(T) == 4;
  static constexpr int kRowBytes = D * (int)sizeof(T);
  static constexpr int kBytes = kChunk * kRowBytes;
  static constexpr int kPieces = kRowBytes / 16;
  static constexpr int kQBytes = f32 ? 8 * D * 8 : 8 * D * 2;  // fragments of 8 query rows
  static constexpr int kQRegs = f32 ? 8 : 2;                   // of them, a lane's registers for 16 dims
  static constexpr int kTiles = D / 16;                        // output tiles of 16 dims

  static __device__ __forceinline__ int k_piece(int row, int piece) {
    return f32 ? piece ^ ((row & 1) << 2) : piece ^ (row & 7);
  }
  static __device__ __forceinline__ int v_piece(int row, int piece) {
    return f32 ? piece ^ (((row >> 1) & 3) << 1) : piece ^ (row & 7);
  }

  // A warp's copies of 16 rows, `valid` of them there.
  template <bool V>
  static __device__ __forceinline__ void load(uint32_t dst, const char *src, long long row_bytes, int valid, int lane) {
    constexpr int kLanes = kPieces < 32 ? kPieces : 32;  // lanes a row
    constexpr int kRows = 32 / kLanes;                   // rows at a time
    const int piece = lane % kLanes, r0 = lane / kLanes;
    const char *from = src + r0 * row_bytes + piece * 16;
    const long long step = kRows * row_bytes;
    if (valid == kChunk) {
#pragma unroll
      for (int i = 0; i < kChunk / kRows; i++, from += step) {
        const int row = i * kRows + r0;
        copy16(dst + row * kRowBytes + (V ? v_piece(row, piece) : k_piece(row, piece)) * 16, from);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kChunk / kRows; i++, from += step) {
        const int row = i * kRows + r0;
        copy16(dst + row * kRowBytes + (V ? v_piece(row, piece) : k_piece(row, piece)) * 16, row < valid ? from : src, row < valid);
      }
    }
  }

  // Writes the fragments of `tiles` x 8 query rows; row(r) gives row r's address
  // or NULL (a zero row).  Called by a whole block of `threads`.
  //   f32: per 16 dims, two float4 a lane, the high and the low parts of row
  //   g's dims 4t .. 4t+3 (the contraction takes the dims in the order that
  //   lets K be read 16 bytes at a time).
  //   16 bits: per 16 dims, two registers a lane: row g's dims 2t, 2t+1 and 2t+8, 2t+9.
  static constexpr int kQItems = (f32 ? D / 16 : D / 32) * 32;  // 16-byte items of 8 rows
  // An item's value, and where it goes.
  template <typename Row>
  static __device__ __forceinline__ uint4 q_fetch(int i, Row row) {
    const int blk = i / 32 % (kQItems / 32), g = (i & 31) >> 2, t = i & 3;
    const T *a = row(i / kQItems * 8 + g);
    if constexpr (f32) {
      return a ? *reinterpret_cast<const uint4 *>(a + blk * 16 + t * 4) : make_uint4(0u, 0u, 0u, 0u);
    } else {
      const uint32_t *p = reinterpret_cast<const uint32_t *>(a) + blk * 16 + t;  // pairs of dims
      return a ? make_uint4(p[0], p[4], p[8], p[12]) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  static __device__ __forceinline__ void q_put(uint32_t dst, int i, uint4 x) {
    const int blk = i / 32 % (kQItems / 32);
    const uint32_t to = dst + i / kQItems * kQBytes + (i & 31) * 16;
    if constexpr (f32) {
      uint32_t h[4], l[4];
      split(__uint_as_float(x.x), h[0], l[0]), split(__uint_as_float(x.y), h[1], l[1]);
      split(__uint_as_float(x.z), h[2], l[2]), split(__uint_as_float(x.w), h[3], l[3]);
      sts4u(to + blk * 1024, h[0], h[1], h[2], h[3]);
      sts4u(to + blk * 1024 + 512, l[0], l[1], l[2], l[3]);
    } else {
      sts4u(to + blk * 512, x.x, x.y, x.z, x.w);
    }
  }
  template <typename Row>
  static __device__ __forceinline__ void query(uint32_t dst, int tiles, int tid, int threads, Row row) {
#pragma unroll 4
    for (int i = tid; i < tiles * kQItems; i += threads) q_put(dst, i, q_fetch(i, row));
  }
  // A lane's registers of the fragments for dims 16 blk .. + 15.
  static __device__ __forceinline__ void q_load(uint32_t (&r)[kQRegs], uint32_t q, int blk, int lane) {
    if constexpr (f32) {
      uint32_t h[4], l[4];
      lds4u(h, q + blk * 1024 + lane * 16);
      lds4u(l, q + blk * 1024 + 512 + lane * 16);
#pragma unroll
      for (int i = 0; i < 4; i++) r[i] = h[i], r[4 + i] = l[i];
    } else {
      asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(q + (blk >> 1) * 512 + lane * 16 + (blk & 1) * 8));
    }
  }

  // K's fragments for dims 16 blk .. + 15.
  //   f32: [step of 8 dims][register], hi and lo.
  struct KFrag {
    uint32_t hi[f32 ? 2 : 1][4], lo[f32 ? 2 : 1][4];
  };
  static __device__ __forceinline__ void k_load(KFrag &f, int blk, uint32_t k, int lane) {
    if constexpr (f32) {
      const int g = lane >> 2, t = lane & 3;
      const float4 x = lds4(k + g * kRowBytes + k_piece(g, blk * 4 + t) * 16);
      const float4 y = lds4(k + (g + 8) * kRowBytes + k_piece(g + 8, blk * 4 + t) * 16);
      split(x.x, f.hi[0][0], f.lo[0][0]), split(y.x, f.hi[0][1], f.lo[0][1]);
      split(x.y, f.hi[0][2], f.lo[0][2]), split(y.y, f.hi[0][3], f.lo[0][3]);
      split(x.z, f.hi[1][0], f.lo[1][0]), split(y.z, f.hi[1][1], f.lo[1][1]);
      split(x.w, f.hi[1][2], f.lo[1][2]), split(y.w, f.hi[1][3], f.lo[1][3]);
    } else {
      const int row = lane & 15;
      ldmatrix4(f.hi[0], k + row * kRowBytes + k_piece(row, blk * 2 + (lane >> 4)) * 16);
    }
  }

  // s (with c for f32) += the chunk's 16 positions' dims 16 blk .. + 15 times
  // 8 rows': elements 0, 1 are position g and rows 2 t, 2 t + 1; elements 2, 3
  // position g + 8.  f32 is three tf32 products, hi hi + hi lo + lo hi, the
  // small ones summed apart in c.
  static __device__ __forceinline__ void k_product(float (&s)[4], float (&c)[2][4], const uint32_t (&q)[kQRegs], const KFrag &f) {
    if constexpr (f32) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        mma_tf32(c[0], f.lo[i], q[2 * i], q[2 * i + 1]);
        mma_tf32(c[1], f.hi[i], q[4 + 2 * i], q[5 + 2 * i]);
        mma_tf32(s, f.hi[i], q[2 * i], q[2 * i + 1]);
      }
    } else {
      mma_16<T>(s, f.hi[0], q[0], q[1]);
    }
  }

  // s[n] of NT x 8 rows.  The fragments of the rows come from registers
  // (qr, NT = 1) or from shared memory.
  template <int NT, bool REGS>
  static __device__ __forceinline__ void scores(float (&s)[NT][4], const uint32_t (&qr)[REGS ? kTiles : 1][kQRegs], uint32_t q, uint32_t k,
                                                int lane) {
    static_assert(!REGS || NT == 1, "");
    float c[NT][2][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) s[n][e] = c[n][0][e] = c[n][1][e] = 0.f;
#pragma unroll
    for (int blk = 0; blk < kTiles; blk++) {
      KFrag f;
      k_load(f, blk, k, lane);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        if constexpr (REGS) {
          k_product(s[n], c[n], qr[blk], f);
        } else {
          uint32_t x[kQRegs];
          q_load(x, q + n * kQBytes, blk, lane);
          k_product(s[n], c[n], x, f);
        }
      }
    }
    if constexpr (f32) {
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[n][e] += c[n][0][e] + c[n][1][e];
    }
  }

  // The dim that element e of output tile i holds (elements 0, 2 are of row
  // 2 t, elements 1, 3 of row 2 t + 1).
  static __device__ __forceinline__ int out_dim(int i, int e, int g) {
    return f32 ? (i >> 1) * 32 + 4 * g + (i & 1) * 2 + (e >> 1) : i * 16 + g + (e >> 1) * 8;
  }

  // o += v' p' over the chunk's 16 positions; p in the layout of scores().
  // f32: the chunk's product is summed apart and added in one rounded
  // addition, since the matrix instruction's own sums are cut, not rounded,
  // which over thousands of chunks would add up.
  template <int NT>
  static __device__ __forceinline__ void values(float (&o)[kTiles][NT][4], const float (&p)[NT][4], uint32_t v, int lane) {
    const int g = lane >> 2, t = lane & 3;
    if constexpr (f32) {
      uint32_t ph[NT][2][2], pl[NT][2][2];  // [positions 8 j ..][2t, 2t+1] of row g
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          float x, y;
          transpose8(p[n][2 * j], p[n][2 * j + 1], x, y);
          split(x, ph[n][j][0], pl[n][j][0]), split(y, ph[n][j][1], pl[n][j][1]);
        }
#pragma unroll
      for (int blk = 0; blk < D / 32; blk++) {
        uint32_t vh[2][2][4], vl[2][2][4];  // [tile][positions 8 j ..]
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int row = j * 8 + 2 * t;
          const float4 x = lds4(v + row * kRowBytes + v_piece(row, blk * 8 + g) * 16);
          const float4 y = lds4(v + (row + 1) * kRowBytes + v_piece(row + 1, blk * 8 + g) * 16);
          split(x.x, vh[0][j][0], vl[0][j][0]), split(x.y, vh[0][j][1], vl[0][j][1]);
          split(y.x, vh[0][j][2], vl[0][j][2]), split(y.y, vh[0][j][3], vl[0][j][3]);
          split(x.z, vh[1][j][0], vl[1][j][0]), split(x.w, vh[1][j][1], vl[1][j][1]);
          split(y.z, vh[1][j][2], vl[1][j][2]), split(y.w, vh[1][j][3], vl[1][j][3]);
        }
        float a[NT][2][4] = {};
#pragma unroll
        for (int j = 0; j < 2; j++) {
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) mma_tf32(a[n][i], vl[i][j], ph[n][j][0], ph[n][j][1]);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) mma_tf32(a[n][i], vh[i][j], pl[n][j][0], pl[n][j][1]);
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) mma_tf32(a[n][i], vh[i][j], ph[n][j][0], ph[n][j][1]);
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[2 * blk + i][n][e] += a[n][i][e];
      }
    } else {
      uint32_t b[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) b[n][j] = transpose8(pack2(p[n][2 * j], p[n][2 * j + 1], T()));
      const int row = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
      for (int i = 0; i < kTiles; i++) {
        uint32_t a[4];
        ldmatrix4_t(a, v + row * kRowBytes + v_piece(row, i * 2 + ((lane >> 3) & 1)) * 16);
#pragma unroll
        for (int n = 0; n < NT; n++) mma_16<T>(o[i][n], a, b[n][0], b[n][1]);
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ void store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
template <typename T>
__device__ __forceinline__ void store4(T *p, float4 v) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(pack2(v.x, v.y, T()), pack2(v.z, v.w, T()));
}

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace paged
}  // namespace ocrvl
