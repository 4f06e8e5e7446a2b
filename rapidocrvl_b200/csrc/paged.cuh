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

// ---- fragments ----------------------------------------------------------
// x = hi + lo with hi the nearest tf32 (11 significant bits); lo keeps the
// rest, of which the instruction takes 11 bits: 22 bits of x in all.
__device__ __forceinline__ void split(float x, uint32_t &hi, uint32_t &lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
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

// What a type's chunk of 16 rows x D looks like in shared memory and how the
// matrix instructions read it.  Rows are stored whole; the 16-byte pieces of a
// row are exchanged by a rule on the row so that the fragment loads of a warp
// hit 32 different banks.
template <typename T, int D>
struct Tile {
  static constexpr bool f32 = sizeof(T) == 4;
  static constexpr int kRowBytes = D * (int)sizeof(T);
  static constexpr int kBytes = kChunk * kRowBytes;
  static constexpr int kPieces = kRowBytes / 16;
  static constexpr int kQBytes = f32 ? 16 * D * 8 : 16 * D * 2;  // query fragments of 16 rows

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
#pragma unroll
    for (int i = 0; i < kChunk / kRows; i++) {
      const int row = i * kRows + r0;
      const bool there = row < valid;
      copy16(dst + row * kRowBytes + (V ? v_piece(row, piece) : k_piece(row, piece)) * 16,
             src + (there ? row * row_bytes + piece * 16 : 0), there);
    }
  }

  // Writes the query fragments of 16 rows; row(r) gives row r's address or
  // NULL (a zero row).  Called by a whole block of `threads`.
  //   f32: per 16 dims, four float4 a lane: high parts of rows g and g + 8,
  //   then the low parts, dims 4t .. 4t+3 (the contraction takes the dims in
  //   the order that lets K be read 16 bytes at a time).
  //   16 bits: per 16 dims, the four registers of the m16k16 fragment.
  template <typename Row>
  static __device__ __forceinline__ void query(uint32_t dst, int tid, int threads, Row row) {
    constexpr int kItems = (D / 16) * 32;
    for (int i = tid; i < kItems; i += threads) {
      const int lane = i & 31, blk = i >> 5, g = lane >> 2, t = lane & 3;
      const T *a = row(g), *b = row(g + 8);
      if constexpr (f32) {
        const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 x = a ? *reinterpret_cast<const float4 *>(a + blk * 16 + t * 4) : z;
        const float4 y = b ? *reinterpret_cast<const float4 *>(b + blk * 16 + t * 4) : z;
        uint32_t h[8], l[8];
        split(x.x, h[0], l[0]), split(x.y, h[1], l[1]), split(x.z, h[2], l[2]), split(x.w, h[3], l[3]);
        split(y.x, h[4], l[4]), split(y.y, h[5], l[5]), split(y.z, h[6], l[6]), split(y.w, h[7], l[7]);
        const uint32_t to = dst + blk * 2048 + lane * 16;
        // the fragment's order: (g, k), (g+8, k), (g, k+4), (g+8, k+4)
        sts4u(to, h[0], h[4], h[1], h[5]);
        sts4u(to + 512, h[2], h[6], h[3], h[7]);
        sts4u(to + 1024, l[0], l[4], l[1], l[5]);
        sts4u(to + 1536, l[2], l[6], l[3], l[7]);
      } else {
        const uint32_t *p = reinterpret_cast<const uint32_t *>(a), *q = reinterpret_cast<const uint32_t *>(b);
        const int c = blk * 8 + t;  // pairs of dims
        sts4u(dst + blk * 512 + lane * 16, p ? p[c] : 0u, q ? q[c] : 0u, p ? p[c + 4] : 0u, q ? q[c + 4] : 0u);
      }
    }
  }

  // The chunk's K as matrix operands.
  struct KFrag {
    uint32_t hi[D / 16][f32 ? 8 : 4], lo[f32 ? D / 16 : 1][f32 ? 8 : 1];
  };
  static __device__ __forceinline__ void k_load(KFrag &f, int blk, uint32_t k, int lane) {
    if constexpr (f32) {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int n = 0; n < 2; n++) {
        const int row = n * 8 + g;
        const float4 x = lds4(k + row * kRowBytes + k_piece(row, blk * 4 + t) * 16);
        uint32_t *h = f.hi[blk] + n * 4, *l = f.lo[blk] + n * 4;
        split(x.x, h[0], l[0]), split(x.y, h[1], l[1]), split(x.z, h[2], l[2]), split(x.w, h[3], l[3]);
      }
    } else {
      const int row = (lane >> 4) * 8 + (lane & 7);
      ldmatrix4(f.hi[blk], k + row * kRowBytes + k_piece(row, blk * 2 + ((lane >> 3) & 1)) * 16);
    }
  }

  // s[n][.] (with c[n][.] for f32) += 16 rows' dims 16 blk .. + 15 times the
  // chunk's 16 positions: the accumulator layout of m16n8 (rows g and g + 8,
  // positions 8 n + 2 t and + 1).  f32 is three tf32 products,
  // hi hi + hi lo + lo hi, the small ones summed apart in c.
  static __device__ __forceinline__ void k_product(float (&s)[2][4], float (&c)[2][4], uint32_t q, const KFrag &f, int blk,
                                                   int lane) {
    if constexpr (f32) {
      const uint32_t at = q + blk * 2048 + lane * 16;
#pragma unroll
      for (int step = 0; step < 2; step++) {
        uint32_t h[4], l[4];
        lds4u(h, at + step * 512);
        lds4u(l, at + 1024 + step * 512);
        // neighbours use different accumulators: a chain of its own takes 11.5 ns a link
        const uint32_t *kh = f.hi[blk] + 2 * step, *kl = f.lo[blk] + 2 * step;
        mma_tf32(c[0], h, kl[0], kl[1]);
        mma_tf32(c[1], h, kl[4], kl[5]);
        mma_tf32(s[0], h, kh[0], kh[1]);
        mma_tf32(s[1], h, kh[4], kh[5]);
        mma_tf32(c[0], l, kh[0], kh[1]);
        mma_tf32(c[1], l, kh[4], kh[5]);
      }
    } else {
      uint32_t x[4];
      lds4u(x, q + blk * 512 + lane * 16);
      mma_16<T>(s[0], x, f.hi[blk][0], f.hi[blk][1]);
      mma_16<T>(s[1], x, f.hi[blk][2], f.hi[blk][3]);
    }
  }

  // s[mt] = q . k of MT x 16 rows.
  template <int MT>
  static __device__ __forceinline__ void scores(float (&s)[MT][2][4], uint32_t q, uint32_t k, int lane) {
    float c[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int i = 0; i < 8; i++) s[m][i >> 2][i & 3] = c[m][i >> 2][i & 3] = 0.f;
    KFrag f;
#pragma unroll
    for (int blk = 0; blk < D / 16; blk++) {
      k_load(f, blk, k, lane);
#pragma unroll
      for (int m = 0; m < MT; m++) k_product(s[m], c[m], q + m * kQBytes, f, blk, lane);
    }
    if constexpr (f32) {
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 8; i++) s[m][i >> 2][i & 3] += c[m][i >> 2][i & 3];
    }
  }

  // The dim that accumulator element e (0, 1 of row g; 2, 3 of row g + 8) of
  // output tile nt holds.
  static __device__ __forceinline__ int out_dim(int nt, int e, int t) {
    return f32 ? (nt >> 2) * 32 + 8 * t + (e & 1) * 4 + (nt & 3) : nt * 8 + 2 * t + (e & 1);
  }

  // o = o * alpha + p v over the chunk's 16 positions; p in the layout of
  // scores().  alpha[mt][0], [1]: of rows g and g + 8; rescale: whether any
  // alpha of the warp is not 1.
  // f32: the chunk's product is summed apart and added in one rounded
  // multiply-add, since the matrix instruction's own sums are cut, not
  // rounded, which over thousands of chunks would add up.
  template <int MT>
  static __device__ __forceinline__ void values(float (&o)[MT][D / 8][4], const float (&p)[MT][2][4],
                                                const float (&alpha)[MT][2], bool rescale, uint32_t v, int lane) {
    const int g = lane >> 2, t = lane & 3;
    if constexpr (f32) {
      uint32_t ph[MT][2][4], pl[MT][2][4];
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < 2; n++) {
          split(p[m][n][0], ph[m][n][0], pl[m][n][0]);  // (g, position 2t)
          split(p[m][n][2], ph[m][n][1], pl[m][n][1]);  // (g+8, 2t)
          split(p[m][n][1], ph[m][n][2], pl[m][n][2]);  // (g, 2t+1)
          split(p[m][n][3], ph[m][n][3], pl[m][n][3]);  // (g+8, 2t+1)
        }
#pragma unroll
      for (int blk = 0; blk < D / 32; blk++) {
        uint32_t vh[2][2][4], vl[2][2][4];  // [positions 8n ..][2t, 2t+1][dim 4g + i]
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const int row = n * 8 + 2 * t + j;
            const float4 x = lds4(v + row * kRowBytes + v_piece(row, blk * 8 + g) * 16);
            split(x.x, vh[n][j][0], vl[n][j][0]), split(x.y, vh[n][j][1], vl[n][j][1]);
            split(x.z, vh[n][j][2], vl[n][j][2]), split(x.w, vh[n][j][3], vl[n][j][3]);
          }
#pragma unroll
        for (int m = 0; m < MT; m++) {
          float a[4][4] = {};
#pragma unroll
          for (int n = 0; n < 2; n++) {
#pragma unroll
            for (int i = 0; i < 4; i++) mma_tf32(a[i], ph[m][n], vl[n][0][i], vl[n][1][i]);
#pragma unroll
            for (int i = 0; i < 4; i++) mma_tf32(a[i], pl[m][n], vh[n][0][i], vh[n][1][i]);
          }
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) mma_tf32(a[i], ph[m][n], vh[n][0][i], vh[n][1][i]);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float(&to)[4] = o[m][blk * 4 + i];
            to[0] = fmaf(to[0], alpha[m][0], a[i][0]);
            to[1] = fmaf(to[1], alpha[m][0], a[i][1]);
            to[2] = fmaf(to[2], alpha[m][1], a[i][2]);
            to[3] = fmaf(to[3], alpha[m][1], a[i][3]);
          }
        }
      }
    } else {
      if (rescale) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int nt = 0; nt < D / 8; nt++) {
            o[m][nt][0] *= alpha[m][0];
            o[m][nt][1] *= alpha[m][0];
            o[m][nt][2] *= alpha[m][1];
            o[m][nt][3] *= alpha[m][1];
          }
      }
      uint32_t a[MT][4];
#pragma unroll
      for (int m = 0; m < MT; m++) {
        a[m][0] = pack2(p[m][0][0], p[m][0][1], T());
        a[m][1] = pack2(p[m][0][2], p[m][0][3], T());
        a[m][2] = pack2(p[m][1][0], p[m][1][1], T());
        a[m][3] = pack2(p[m][1][2], p[m][1][3], T());
      }
      const int row = lane & 15;
#pragma unroll
      for (int c = 0; c < D / 16; c++) {
        uint32_t b[4];
        ldmatrix4_t(b, v + row * kRowBytes + v_piece(row, c * 2 + (lane >> 4)) * 16);
#pragma unroll
        for (int m = 0; m < MT; m++) {
          mma_16<T>(o[m][2 * c], a[m], b[0], b[1]);
          mma_16<T>(o[m][2 * c + 1], a[m], b[2], b[3]);
        }
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
