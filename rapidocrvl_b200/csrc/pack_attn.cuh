// Attention of drafted tokens over a packed cache and over one another
// (ocrvl_op_packed_attn where a kv head has few rows, and for f32 with any number).
//
// The mathematics, segments and runs are tree_attn.cuh's; only the cache is read in another way.
// The 16 positions of a chunk are the rows of the matrix instruction, 8 query rows its
// columns.  Codes become 16-bit numbers in registers:
//   K   c + 8 as f16, against f16 queries: a row's power of two brings its largest value below 2^14; a group of 32 dims is
//       summed from -8 sum q on, then times its scale in 32 bits.  f32: c itself, so that nothing cancels, against two f16
//       parts of a query (22 bits)
//   V   c s in T (f32: in bf16, which holds it exactly, against weights of three bf16 parts)
// so products are exact and only sums are rounded.  A lane finds all that it needs of a row in one piece: of K, dims
// 32 j + 8 t .. + 7 of each group j, of V, dims 32 j + 4 g .. + 3 (g = lane / 4, t = lane % 4).  The chunk's
// positions are the instruction's rows in the order 0 1 4 5 8 9 12 13, 2 3 6 7 10 11 14 15, so that a
// lane's four positions of V, and their scales, are neighbours.
//
// 64 sequences of up to 4,096 positions, one token: bf16 27.7 us, f32 34.8, against 6.3 us of bytes.  A chunk costs a warp some
// 445 instructions, many on the integer pipe (half rate): masks, shifts and byte permutations that make operands of codes, for
// eight rows only.  With launch, start and join, and the longest sequence's chunks behind one another, that is the time.
// Tried in bf16: clusters of four 33.2 us, one block a segment 37.4; runs 34.8 and three blocks an SM (spills) 35.4, both before the
// longest sequences came first; shifts as products 34.8 where 33.2 without.  One sequence of 700,
// f32: 6.8 us, a launch and three loads behind one another.
#pragma once
#include "packed.cuh"
#include "tree_attn.cuh"

namespace ocrvl {
namespace paged {

template <typename T>
using Product = std::conditional_t<std::is_same<T, __half>::value, __half, __nv_bfloat16>;  // the type of V's products

// The four pairs of nibbles u = c + 8 of two halfwords as f16: a nibble's bits as they lie there, or four places up, are
// 2^-24 u and 2^-20 u, numbers below the smallest normal one, which the matrix instruction takes like any other.  So a pair
// costs one mask, and four one shift; the queries of odd dims are a 16th, and 8 of each sum is taken off as the accumulator's
// first value.
__device__ __forceinline__ void nibbles4(uint32_t (&u)[4], uint32_t x) {
  const uint32_t y = x >> 8;
  u[0] = x & 0x000f000fu, u[1] = x & 0x00f000f0u, u[2] = y & 0x000f000fu, u[3] = y & 0x00f000f0u;
}
// As whole numbers c: (1024 + u) - 1032 and (1024 + 16 u) / 16 - 72, all exact.  base: 1024 twice, from a register (as
// a constant it costs an instruction a pair).
__device__ __forceinline__ void whole4(uint32_t (&c)[4], uint32_t x, uint32_t base) {
  const uint32_t minus = 0xe408e408u, low = 0x2c002c00u, minus72 = 0xd480d480u;
  nibbles4(c, x);
  c[0] = add2(c[0] | base, minus), c[1] = fma2<__half>(c[1] | base, low, minus72);
  c[2] = add2(c[2] | base, minus), c[3] = fma2<__half>(c[3] | base, low, minus72);
}

// x as three bf16 numbers, in the upper halves: exact (8 bits each, cut, so that none is rounded up to
// infinity); what is not finite is the last one's alone, so that it meets nothing but another's first part.
__device__ __forceinline__ void split3(float x, uint32_t (&p)[3]) {
  const uint32_t hi = __float_as_uint(x) & 0xffff0000u;
  const float r = x - __uint_as_float(hi);
  const uint32_t mid = __float_as_uint(r) & 0xffff0000u;
  const bool finite = (hi & 0x7f800000u) != 0x7f800000u;
  p[0] = finite ? hi : 0u, p[1] = finite ? mid : 0u;
  p[2] = finite ? __float_as_uint(r - __uint_as_float(mid)) : __float_as_uint(x) | ((__float_as_uint(x) & 0x7fffffu) ? 0x400000u : 0u);
}

// Four values as they lie in memory.
template <typename T>
struct Four {
  uint32_t w[sizeof(T)];

  __device__ __forceinline__ void load(const T *p) {
    if constexpr (sizeof(T) == 4) {
      const uint4 x = *(const uint4 *)p;
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
      const uint2 x = *(const uint2 *)p;
      w[0] = x.x, w[1] = x.y;
    }
  }
  __device__ __forceinline__ float4 floats() const {
    if constexpr (sizeof(T) == 4) {
      return make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
      const float2 a = unpack2<T>(w[0]), b = unpack2<T>(w[1]);
      return make_float4(a.x, a.y, b.x, b.y);
    }
  }
};

template <typename T, int D>
struct PackTile {
  using B = Product<T>;
  static constexpr bool f32 = sizeof(T) == 4;
  static constexpr int G = D / 32;                     // groups of a row
  static constexpr int kParts = f32 ? 3 : 1;           // of a weight
  static constexpr int kQParts = f32 ? 2 : 1;          // of a query
  static constexpr float kOdd = f32 ? 1.f : 16.f;      // how much smaller a query's odd dims are: their codes are that much larger
  static constexpr float kUnit = f32 ? 1.f : 0x1p24f;  // one over what a code is
  static constexpr int kCodes = kChunk * D / 2;        // bytes of a chunk's K or V
  static constexpr int kScales = kChunk * G * 2;
  static constexpr int kStage = 2 * (kCodes + kScales);  // K, V, their scales
  static constexpr int kQBytes = kQParts * G * 512;     // fragments of 8 query rows: [part][group][lane] of 16 bytes
  static constexpr int kTiles = D / 16;

  // Where 16-byte piece x of a position's row lies: exchanged so that the fragment loads of a warp (K: rows 0 1 4 5
  // .., V: a row of every four) hit different banks.
  static __device__ __forceinline__ int k_at(int row, int x) {
    return D == 128 ? row * 64 + x * 16 : (row ^ (row >> 2 & 1) << 1) * 32 + x * 16;
  }
  static __device__ __forceinline__ int v_at(int row, int x) {
    return D == 128 ? (row ^ (row >> 2 & 1)) * 64 + (x ^ (row >> 3 & 1) << 1) * 16 : (row ^ (row >> 2 & 3)) * 32 + x * 16;
  }
  // A warp's copies of a chunk: k, v, s are the lane's own.
  static __device__ __forceinline__ void load(uint32_t to, const char *k, const char *v, const char *s, int lane) {
#pragma unroll
    for (int i = 0; i < kCodes / 512; i++) {
      const int p = i * 32 + lane, row = p / (D / 32), x = p % (D / 32);
      copy16(to + k_at(row, x), k + i * 512);
      copy16(to + kCodes + v_at(row, x), v + i * 512);
    }
    if (lane < 2 * (kScales / 16)) copy16(to + 2 * kCodes + lane * 16, s);
  }

  // The position of row g of the matrix instruction; row g + 8 has that plus 2.
  static __device__ __forceinline__ int position(int g) { return 4 * (g >> 1) + (g & 1); }

  // ---- fragments of a query row's 8 consecutive dims: pairs (i, 4 + i) of f16 parts of up times the row (odd ones a 16th)
  static __device__ __forceinline__ void pairs8(uint32_t (&f)[kQParts][4], const float (&x)[8], float up) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float z = i & 1 ? up / kOdd : up, a = x[i] * z, b = x[4 + i] * z;
      f[0][i] = pack2(a, b, __half());
      if constexpr (f32) {
        const float2 hi = unpack2<__half>(f[0][i]);
        f[kQParts - 1][i] = pack2(a - hi.x, b - hi.y, __half());
      }
    }
  }
  // Dims 32 j + 4 g .. + 3 of row r of 8, from the fragments: up times them.
  static __device__ __forceinline__ float4 four(uint32_t q, int r, int j, int g) {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kQParts; w++) {
      uint32_t f[4];
      lds4u(f, q + (w * G + j) * 512 + (r * 4 + (g >> 1)) * 16);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 y = unpack2<__half>(f[i]);
        x[i] += g & 1 ? y.y : y.x;
      }
    }
    return make_float4(x[0], kOdd * x[1], x[2], kOdd * x[3]);
  }

  // ---- cached keys: s of NT x 8 rows (times 2^-24 their up).  q: the fragments' address; qr: they themselves (NT = 1, 16
  // bits); first: -8 times the sums of q, [row][group], and fr a lane's own.
  template <int NT, bool REGS>
  static __device__ __forceinline__ void scores(float (&s)[NT][4], const uint32_t (&qr)[REGS ? G : 1][4], const float (&fr)[REGS ? G : 1][2],
                                                uint32_t q, const float *first, uint32_t st, int lane) {
    const int g = lane >> 2, t = lane & 3, p0 = position(g);
    uint32_t k[2][4], ks[2][2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const int pos = p0 + 2 * r;
      const uint32_t at = st + 2 * kCodes + pos * (G * 2);
      if constexpr (D == 128) {
        lds4u(k[r], st + k_at(pos, t));
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(ks[r][0]), "=r"(ks[r][1]) : "r"(at));
      } else {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(k[r][0]), "=r"(k[r][2]) : "r"(st + k_at(pos, t >> 1) + (t & 1) * 8));
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(ks[r][0]) : "r"(at));
      }
    }
#pragma unroll
    for (int j = 0; j < G; j++) {
      uint32_t c0[4], c1[4];
      const uint32_t x0 = halves(k[0][j >> 1], k[0][2 + (j >> 1)], j & 1), x1 = halves(k[1][j >> 1], k[1][2 + (j >> 1)], j & 1);
      if constexpr (f32)
        whole4(c0, x0, 0x64006400u), whole4(c1, x1, 0x64006400u);
      else
        nibbles4(c0, x0), nibbles4(c1, x1);
      const uint32_t a0[4] = {c0[0], c1[0], c0[1], c1[1]}, a1[4] = {c0[2], c1[2], c0[3], c1[3]};
      const float s0 = __uint_as_float(j & 1 ? ks[0][j >> 1] & 0xffff0000u : ks[0][j >> 1] << 16);
      const float s1 = __uint_as_float(j & 1 ? ks[1][j >> 1] & 0xffff0000u : ks[1][j >> 1] << 16);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float p[4];
        if constexpr (f32)
          p[0] = p[1] = p[2] = p[3] = 0.f;
        else if constexpr (REGS)
          p[0] = p[2] = fr[j][0], p[1] = p[3] = fr[j][1];
        else
          p[0] = p[2] = first[(n * 8 + 2 * t) * G + j], p[1] = p[3] = first[(n * 8 + 2 * t + 1) * G + j];
#pragma unroll
        for (int w = kQParts - 1; w >= 0; w--) {  // the small part first
          uint32_t b[4];
          if constexpr (REGS) {
#pragma unroll
            for (int i = 0; i < 4; i++) b[i] = qr[j][i];
          } else {
            lds4u(b, q + n * kQBytes + (w * G + j) * 512 + lane * 16);
          }
          mma_16<__half>(p, a0, b[0], b[1]);
          mma_16<__half>(p, a1, b[2], b[3]);
        }
        s[n][0] = j ? fmaf(s0, p[0], s[n][0]) : s0 * p[0], s[n][1] = j ? fmaf(s0, p[1], s[n][1]) : s0 * p[1];
        s[n][2] = j ? fmaf(s1, p[2], s[n][2]) : s1 * p[2], s[n][3] = j ? fmaf(s1, p[3], s[n][3]) : s1 * p[3];
      }
    }
  }

  // The weights of a chunk (as scores leaves them) as the products' second operand.
  template <int NT>
  static __device__ __forceinline__ void weights(uint32_t (&b)[kParts][NT][2], const float (&p)[NT][4]) {
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int r = 0; r < 2; r++) {
        if constexpr (f32) {
          uint32_t u[3], v[3];
          split3(p[n][2 * r], u), split3(p[n][2 * r + 1], v);
#pragma unroll
          for (int w = 0; w < 3; w++) b[w][n][r] = transpose8(high_halves(u[w], v[w]));
        } else {
          b[0][n][r] = transpose8(pack2(p[n][2 * r], p[n][2 * r + 1], T()));
        }
      }
  }

  // o += v' p over the chunk; tile 2 j + h of o has dims 32 j + 4 g + 2 h (elements 0, 1) and the next (2, 3).
  template <int NT>
  static __device__ __forceinline__ void values(float (&o)[kTiles][NT][4], const uint32_t (&b)[kParts][NT][2], uint32_t st, int valid, int lane,
                                                uint32_t base) {
    const int g = lane >> 2, t = lane & 3;
    uint32_t v[4][2], vs[4][2];  // of positions 4 t + i
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (D == 128)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[i][0]), "=r"(v[i][1]) : "r"(st + kCodes + v_at(4 * t + i, g >> 1) + (g & 1) * 8));
      else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[i][0]) : "r"(st + kCodes + v_at(4 * t + i, g >> 2) + (g & 3) * 4));
    }
    const uint32_t at = st + 2 * kCodes + kScales + t * (8 * G);
    uint32_t x[4];
    lds4u(x, at);
    if constexpr (D == 128) {
      vs[0][0] = x[0], vs[0][1] = x[1], vs[1][0] = x[2], vs[1][1] = x[3];
      lds4u(x, at + 16);
      vs[2][0] = x[0], vs[2][1] = x[1], vs[3][0] = x[2], vs[3][1] = x[3];
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) vs[i][0] = x[i];
    }
    if (valid < kChunk) {  // what lies behind the end may hold anything
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int w = 0; w < (G + 1) / 2; w++) vs[i][w] = 4 * t + i < valid ? vs[i][w] : 0u;
    }
#pragma unroll
    for (int j = 0; j < G; j++) {
      uint32_t s01 = halves(vs[0][j >> 1], vs[1][j >> 1], j & 1), s23 = halves(vs[2][j >> 1], vs[3][j >> 1], j & 1);
      if constexpr (std::is_same<B, __half>::value) {
        s01 = pack2(__uint_as_float(s01 << 16), __uint_as_float(s01 & 0xffff0000u), B());
        s23 = pack2(__uint_as_float(s23 << 16), __uint_as_float(s23 & 0xffff0000u), B());
      }
      const uint32_t x01 = halves(v[0][j >> 1], v[1][j >> 1], j & 1), x23 = halves(v[2][j >> 1], v[3][j >> 1], j & 1);
      uint32_t y01[4], y23[4];
      if constexpr (std::is_same<B, __half>::value) {
        whole4(y01, x01, base), whole4(y23, x23, base);
#pragma unroll
        for (int i = 0; i < 4; i++) y01[i] = mul2<B>(y01[i], s01), y23[i] = mul2<B>(y23[i], s23);
      } else {
        const Scaled<B> by01(s01), by23(s23);
#pragma unroll
        for (int i = 0; i < 4; i++) y01[i] = by01(x01, i, base), y23[i] = by23(x23, i, base);
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t a[4] = {y01[2 * h], y01[2 * h + 1], y23[2 * h], y23[2 * h + 1]};
        product<NT>(o[2 * j + h], a, b);
      }
    }
  }

  // o of a tile += a times the weights.  f32: summed apart and added in one rounded addition, since
  // the matrix instruction's own sums are cut, not rounded, which over thousands of chunks would add up.
  template <int NT>
  static __device__ __forceinline__ void product(float (&o)[NT][4], const uint32_t (&a)[4], const uint32_t (&b)[kParts][NT][2]) {
#pragma unroll
    for (int n = 0; n < NT; n++) {
      if constexpr (f32) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 2; w >= 0; w--) mma_16<B>(sum, a, b[w][n][0], b[w][n][1]);
#pragma unroll
        for (int e = 0; e < 4; e++) o[n][e] += sum[e];
      } else {
        mma_16<B>(o[n], a, b[0][n][0], b[0][n][1]);
      }
    }
  }
};

template <typename T, int D, int NT>
struct PackShape {
  using L = PackTile<T, D>;
  static constexpr int kRows = 8 * NT;
  static constexpr int kBlocks = NT == 1 ? 2 : 1;  // an SM
  static constexpr int kStages = kBlocks == 2 ? 4 : 6;  // chunks of a warp on their way or in use
  static constexpr int kRing = kTreeWarps * kStages * L::kStage;
  static constexpr int kJoin = kTreeWarps * 8 * D * 4;  // eight rows of every warp
  static constexpr int kQ = NT * L::kQBytes;
  static_assert(kQ >= kTreeThreads * 4, "the lengths are ranked there");
  static constexpr bool kQInRegs = NT == 1 && sizeof(T) == 2;
  static constexpr int kFactors = kRows * 4 * (1 + L::G);
  static constexpr int kSmem = kRing + kJoin + kQ + kFactors + kTreeWarps * kRows * 8 + kRows * 8 + 64 + kTreeWarps * 64 * 4 + kRows * 8;
};

template <typename T, int D, int NT, int CS>
__global__ void __launch_bounds__(kTreeThreads, (PackShape<T, D, NT>::kBlocks)) k_pack_attn(const TreeArgs a, int row_blocks) {
  using S = PackShape<T, D, NT>;
  using L = PackTile<T, D>;
  constexpr int ROWS = S::kRows, NS = S::kStages, G = L::G;
  namespace cg = cooperative_groups;
  extern __shared__ __align__(128) char sm[];
  char *ring = sm, *q_sm = sm + S::kRing + S::kJoin;
  float *join = (float *)(sm + S::kRing);
  char *p = q_sm + S::kQ;
  float *down_sm = (float *)p, *first_sm = down_sm + ROWS;  // [row]: 1 / up; [row][group]: 2^-24 * -8 times the sum of up q
  p += S::kFactors;
  float *ml = (float *)p;  // [warp][row][m, l]
  p += kTreeWarps * ROWS * 8;
  unsigned long long *seen = (unsigned long long *)p;  // [row]
  p += ROWS * 8;
  long long *plan = (long long *)p;
  p += 64;
  int *there = (int *)p;  // [warp][chunk % 64]: its positions that exist
  p += kTreeWarps * 64 * 4;
  float *part_ml = (float *)p;  // CS > 1: [row][m, l] of this block
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint32_t base = lifted_base<typename L::B>();
  asm("" : "+r"(base));  // stays in a register

  pdl_wait();
  WarpPiece cur;
  Walk walk;
  bool more = true;
  if constexpr (CS > 0) pdl_launch();
  if constexpr (CS == 0) {
    const bool any = walk.start(a, ROWS, plan, warp, lane, cur);
    pdl_launch();
    if (!any) return;
    cur.chunks_of(warp, kTileChunks);
  } else {
    const int seg = blockIdx.x / CS;
    cur.rb = seg % row_blocks, cur.head = seg / row_blocks % a.kv_heads, cur.b = seg / row_blocks / a.kv_heads;
    if (a.longest_first) {
      // Blocks are handed out in order, one an SM first: the longest sequences' come first, so that an SM's second block is
      // a short one's.  Every block ranks the lengths (at most one a thread) and takes the sequence of its rank.
      int *lens = (int *)q_sm;
      const int mine = tid < a.s.batch ? a.s.len(tid) : 0;
      if (tid < a.s.batch) lens[tid] = mine;
      __syncthreads();
      if (tid < a.s.batch) {
        int rank = 0;
        for (int i = 0; i < a.s.batch; i++) rank += lens[i] > mine || (lens[i] == mine && i < tid);
        if (rank == cur.b) plan[0] = tid;
      }
      __syncthreads();
      cur.b = (int)plan[0];
    }
    cur.sg = Segments(a, cur.b, ROWS);
    if (cur.rb >= cur.sg.blocks) return;  // the whole cluster alike
    cur.t0 = blockIdx.x % CS, cur.t1 = cur.sg.tiles;
    cur.chunks_of(warp, kTileChunks * CS);
  }
  // how many of the warp's chunks are cached ones; they come before those of drafts
  auto cached_of = [](const WarpPiece &x) {
    const int end = min(x.t1 * kTileChunks, x.sg.chunks_c);
    return x.c0 < end ? (end - x.c0 + x.step - 1) / x.step : 0;
  };

  const uint32_t my_ring = smem_addr(ring) + warp * (NS * L::kStage), q_at = smem_addr(q_sm);
  int *my_there = there + warp * 64;
  // Lane i: where the chunk 32 j + i lies, codes and scales, negative without a page.
  long long codes_at = -1, scales_at = -1;
  const char *from_k, *from_v, *from_s;  // of the piece's head: what the lane copies
  auto head_of = [&](const WarpPiece &x) {
    const long long at = x.head * a.c.head_bytes + lane * 16, at_s = x.head * a.scale_head;
    from_k = a.c.k + at, from_v = a.c.v + at;
    from_s = (lane < L::kScales / 16 ? a.k_scale + lane * 16 : a.v_scale + (lane - L::kScales / 16) * 16) + at_s;
  };
  head_of(cur);
  auto issue = [&](const WarpPiece &x, int nc, int k) {
    if (k < nc) {
      if ((k & 31) == 0) {
        const int c = x.c0 + (k + lane) * x.step, pos = c * kChunk;
        const long long in_page = pos & ((1 << a.c.page_shift) - 1);
        const int pg = c < x.sg.chunks_c ? a.c.table[x.b * a.c.table_stride + (pos >> a.c.page_shift)] : -1;
        const bool mapped = pg >= 0 && pg < a.c.num_pages;
        codes_at = mapped ? pg * a.c.page_bytes + in_page * (D / 2) : -1;
        scales_at = pg * a.scale_page + in_page * (G * 2);
        my_there[(k + lane) & 63] = mapped ? min(kChunk, x.sg.len - pos) : 0;
      }
      const long long at = __shfl_sync(~0u, codes_at, k & 31), at_s = __shfl_sync(~0u, scales_at, k & 31);
      // whole chunks: a page has room for them
      if (at >= 0) L::load(my_ring + k % NS * L::kStage, from_k + at, from_v + at, from_s + at_s, lane);
    }
    copy_commit();
  };
  // the query rows of a piece, their sums and the drafts that each sees
  auto load_query = [&](const WarpPiece &x) {
    const int rows = min(ROWS, x.sg.count * a.group - x.rb * ROWS);
    for (int i = tid; i < ROWS * G * 4; i += kTreeThreads) {  // (row, group, quarter): whole warps
      const int row = i / (G * 4), j = i / 4 % G, quarter = i % 4, at = x.rb * ROWS + row;
      float y[8] = {};
      if (row < rows) {
        Eight<T> e;
        e.load((const T *)a.q + (x.sg.first + at / a.group) * a.q_stride + (long long)(x.head * a.group + at % a.group) * D + 32 * j + 8 * quarter);
        e.floats(y);
      }
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 8; k++) most = fmaxf(most, fabsf(y[k]));
#pragma unroll
      for (int d = 1; d < G * 4; d <<= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
      // 2^13 over the largest value's power of two, within what has a reciprocal
      const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -100), 126);
      const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23), down = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
      uint32_t f[L::kQParts][4];
      L::pairs8(f, y, up);
#pragma unroll
      for (int w = 0; w < L::kQParts; w++)
        sts4u(q_at + row / 8 * L::kQBytes + (w * G + j) * 512 + (row % 8 * 4 + quarter) * 16, f[w][0], f[w][1], f[w][2], f[w][3]);
      if constexpr (!L::f32) {
        float q8 = 0.f;  // of the fragments, which may be rounded
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float2 z = unpack2<__half>(f[0][k]);
          q8 = fmaf(k & 1 ? L::kOdd : 1.f, z.x + z.y, q8);
        }
        q8 += __shfl_xor_sync(~0u, q8, 1);
        q8 += __shfl_xor_sync(~0u, q8, 2);
        if (quarter == 0) first_sm[row * G + j] = -8.f / L::kUnit * q8;
      }
      if (j + quarter == 0) down_sm[row] = down;
    }
    for (int r = tid; r < ROWS; r += kTreeThreads)
      seen[r] = r < rows ? (unsigned long long)a.mask[x.sg.first + (x.rb * ROWS + r) / a.group] : 0ull;
  };

  // The drafts of a piece that this warp takes, and the first one's key and value.
  int draft0, draft1;
  const int draft_step = CS > 1 ? kTreeWarps * CS : kTreeWarps;
  Four<T> key[G], value[G];
  auto load_draft = [&](const WarpPiece &x, int j) {
    const long long at = (x.sg.first + j) * a.kv_stride + (long long)x.head * D + 4 * g;
#pragma unroll
    for (int i = 0; i < G; i++) key[i].load((const T *)a.dk + at + 32 * i), value[i].load((const T *)a.dv + at + 32 * i);
  };
  auto drafts_of = [&](const WarpPiece &x) {
    const int c0 = CS > 0 ? 0 : x.t0 * kTileChunks - x.sg.chunks_c, c1 = x.t1 * kTileChunks - x.sg.chunks_c;
    // from the last warp down, which has the fewest chunks
    draft0 = max(0, c0) * kChunk + draft_step - 1 - warp - (CS > 1 ? blockIdx.x % CS * kTreeWarps : 0), draft1 = min(x.sg.count, c1 * kChunk);
    if (draft0 < draft1) load_draft(x, draft0);
  };

  int nc = cached_of(cur);
#pragma unroll 1
  for (int k = 0; k < NS - 1; k++) issue(cur, nc, k);
  drafts_of(cur);
  load_query(cur);
  __syncthreads();

  for (int piece = 0; more; piece++) {
    uint32_t qr[S::kQInRegs ? G : 1][4];
    float fr[S::kQInRegs ? G : 1][2];
    if constexpr (S::kQInRegs) {
#pragma unroll
      for (int j = 0; j < G; j++) {
        lds4u(qr[j], q_at + j * 512 + lane * 16);
        fr[j][0] = first_sm[2 * t * G + j], fr[j][1] = first_sm[(2 * t + 1) * G + j];
      }
    }
    // of rows 8 n + 2 t and + 1; factor: what makes scores of the products, in units of log2
    float o[L::kTiles][NT][4] = {}, ref[NT][2], sum[NT][2] = {}, low[NT][2] = {}, factor[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) ref[n][h] = -INFINITY, factor[n][h] = a.scale * L::kUnit * down_sm[n * 8 + 2 * t + h];

    // scores in units of log2 become weights, against the rows' references
    auto soften = [&](float (&s)[NT][4]) {
      bool above = false;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) above |= s[n][e] > ref[n][e & 1] + kSlack<T>;
      if (__any_sync(~0u, above)) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float top = fmaxf(s[n][h], s[n][2 + h]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
            const float now = fmaxf(ref[n][h], top - kLift<T>);
            const float alpha = now == -INFINITY ? 1.f : exp2_(ref[n][h] - now);
            ref[n][h] = now;
            sum[n][h] *= alpha, low[n][h] *= alpha;
#pragma unroll
            for (int i = 0; i < L::kTiles; i++) o[i][n][h] *= alpha, o[i][n][2 + h] *= alpha;
          }
      }
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float m = ref[n][h] == -INFINITY ? 0.f : ref[n][h];
          s[n][h] = exp2_(s[n][h] - m), s[n][2 + h] = exp2_(s[n][2 + h] - m);
          add_exactly(sum[n][h], low[n][h], s[n][h] + s[n][2 + h]);
        }
    };

    // Drafts first, while the first cached chunks are on their way: position by position, shared out over all warps, in 32
    // bits without the matrix instruction.  A lane has dims 32 j + 4 g .. + 3 of the key, the value and o.
    for (int j = draft0; j < draft1; j += draft_step) {
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int row = n * 8 + 2 * t + h;
          const float down = down_sm[row];
          float x = 0.f;
#pragma unroll
          for (int i = 0; i < G; i++) {
            const float4 q4 = L::four(q_at + n * L::kQBytes, 2 * t + h, i, g);
            const float4 k4 = key[i].floats();
            x = fmaf(q4.x * down, k4.x, fmaf(q4.y * down, k4.y, fmaf(q4.z * down, k4.z, fmaf(q4.w * down, k4.w, x))));
          }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(~0u, x, d);
          if (!(seen[row] >> j & 1)) continue;  // what a draft holds that is not seen stays out
          x *= a.scale;
          if (x > ref[n][h] + kSlack<T>) {
            const float now = x - kLift<T>, alpha = exp2_(ref[n][h] - now);
            ref[n][h] = now;
            sum[n][h] *= alpha, low[n][h] *= alpha;
#pragma unroll
            for (int i = 0; i < L::kTiles; i++) o[i][n][h] *= alpha, o[i][n][2 + h] *= alpha;
          }
          const float w = exp2_(x - (ref[n][h] == -INFINITY ? 0.f : ref[n][h]));
          if (g == 0) add_exactly(sum[n][h], low[n][h], w);
#pragma unroll
          for (int i = 0; i < G; i++) {
            const float4 v4 = value[i].floats();
            o[2 * i][n][h] = fmaf(w, v4.x, o[2 * i][n][h]), o[2 * i][n][2 + h] = fmaf(w, v4.y, o[2 * i][n][2 + h]);
            o[2 * i + 1][n][h] = fmaf(w, v4.z, o[2 * i + 1][n][h]), o[2 * i + 1][n][2 + h] = fmaf(w, v4.w, o[2 * i + 1][n][2 + h]);
          }
        }
      if (j + draft_step < draft1) load_draft(cur, j + draft_step);
    }

    for (int k = 0; k < nc; k++) {
      copy_wait<NS - 2>();
      __syncwarp();  // the stage before is read by all lanes too
      issue(cur, nc, k + NS - 1);
      const uint32_t st = my_ring + k % NS * L::kStage;
      const int valid = my_there[k & 63];
      if (valid == 0) continue;
      float s[NT][4];
      L::template scores<NT, S::kQInRegs>(s, qr, fr, q_at, first_sm, st, lane);
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[n][e] *= factor[n][e & 1];
      if (valid < kChunk) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (L::position(g) + (e >> 1) * 2 >= valid) s[n][e] = -INFINITY;
      }
      soften(s);
      uint32_t b[L::kParts][NT][2];
      L::template weights<NT>(b, s);
      L::template values<NT>(o, b, st, valid, lane, base);
    }
    // the next piece's first chunks are on their way while this one is joined
    const WarpPiece done = cur;
    if constexpr (CS == 0) {
      if (tid == 0) walk.tell(a, cur, row_blocks, 2 * blockIdx.x + (piece ? 1 : 0));
      more = walk.next(a, ROWS, cur);
      if (more) {
        cur.chunks_of(warp, kTileChunks);
        nc = cached_of(cur);
        __syncwarp();  // all lanes are done with the last stage
        head_of(cur);
#pragma unroll 1
        for (int k = 0; k < NS - 1; k++) issue(cur, nc, k);
        drafts_of(cur);
      }
    } else {
      more = false;
    }
    const int rows = min(ROWS, done.sg.count * a.group - done.rb * ROWS);
    const bool whole = CS == 0 ? done.t0 == 0 && done.t1 == done.sg.tiles : CS == 1;
    const long long slot = 2 * (long long)blockIdx.x + (piece ? 1 : 0);
    float *part = CS > 1 ? (float *)ring : a.part + slot * ROWS * D;
    float *to_ml = CS > 1 ? part_ml : a.part_ml + slot * ROWS * 2;
    // dim d of row r: exchanged so that a warp's stores hit different banks
    auto dim_of = [](int r, int d) { return d ^ (((r >> 1) & 3) << 3); };
#pragma unroll
    for (int n = 0; n < NT; n++) {
      __syncthreads();  // every warp is done with what the join, or the parts, lie over
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float l = sum[n][h] + low[n][h];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(~0u, l, d);
        const int r = 2 * t + h, row = n * 8 + r;
        if (g == 0) ml[(warp * ROWS + row) * 2] = ref[n][h], ml[(warp * ROWS + row) * 2 + 1] = l;
        float *to = join + (warp * 8 + r) * D;
#pragma unroll
        for (int j = 0; j < G; j++)
          *(float4 *)(to + dim_of(r, j * 32 + 4 * g)) = make_float4(o[2 * j][n][h], o[2 * j][n][2 + h], o[2 * j + 1][n][h], o[2 * j + 1][n][2 + h]);
      }
      if (n == NT - 1 && more) load_query(cur);
      __syncthreads();
      for (int i = tid; i < min(8, rows - n * 8) * (D / 4); i += kTreeThreads) {
        const int r = i / (D / 4), d = i % (D / 4), row = n * 8 + r;
        float top = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kTreeWarps; w++) top = fmaxf(top, ml[(w * ROWS + row) * 2]);
        const float base = top == -INFINITY ? 0.f : top;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kTreeWarps; w++) {
          const float f = exp2_(ml[(w * ROWS + row) * 2] - base);
          l = fmaf(f, ml[(w * ROWS + row) * 2 + 1], l);
          const float4 y = *(const float4 *)(join + (w * 8 + r) * D + dim_of(r, d * 4));
          x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
        }
        if (whole) {
          write_row<T, D>(a, done.sg, done.head, done.rb * ROWS + row, d * 4, x, top, l);
        } else {
          *(float4 *)(part + row * D + d * 4) = x;
          if (d == 0) *(float2 *)(to_ml + row * 2) = make_float2(top, l);
        }
      }
    }
    if constexpr (CS > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      for (int i = (int)cluster.block_rank() * kTreeThreads + tid; i < rows * (D / 4); i += CS * kTreeThreads) {
        const int row = i / (D / 4), d = i % (D / 4);
        float2 w[CS];
        float4 y[CS];
#pragma unroll
        for (int r = 0; r < CS; r++) {
          w[r] = *(const float2 *)(cluster.map_shared_rank(part_ml, r) + row * 2);
          y[r] = *(const float4 *)(cluster.map_shared_rank(part, r) + row * D + d * 4);
        }
        float top = -INFINITY, l = 0.f;
#pragma unroll
        for (int r = 0; r < CS; r++) top = fmaxf(top, w[r].x);
        const float base = top == -INFINITY ? 0.f : top;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < CS; r++) {
          const float f = exp2_(w[r].x - base);
          l = fmaf(f, w[r].y, l);
          x.x = fmaf(f, y[r].x, x.x), x.y = fmaf(f, y[r].y, x.y), x.z = fmaf(f, y[r].z, x.z), x.w = fmaf(f, y[r].w, x.w);
        }
        write_row<T, D>(a, cur.sg, cur.head, cur.rb * ROWS + row, d * 4, x, top, l);
      }
      cluster.sync();  // no block ends while another reads its part
    }
    __syncthreads();  // the join is read, the query rows are there
  }
}

}  // namespace paged
}  // namespace ocrvl
