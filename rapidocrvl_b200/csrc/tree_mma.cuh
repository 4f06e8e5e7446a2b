// Attention of drafted tokens over a paged cache for 16-bit types and many
// rows, on the tensor cores' fifth generation (ocrvl_op_tree_attn where a kv
// head has more than 16 rows; the mathematics, segments and runs are
// tree_attn.cuh's).
//
// One block an SM.  Its 128 x D query tile(s), the tiles of 128 positions of K
// and V (128-byte swizzled rows) lie in shared memory, S = Q K' and O += P V
// in tensor memory, and P goes back to tensor memory over S as the next product's
// operand, so the accumulators cost no registers and a row's softmax belongs
// to one thread: no shuffles, no join of warps.  Two streams of S, P and O keep the
// tensor cores busy while the other's softmax runs:
//   WIDE    up to 256 rows: each stream has 128 of them, both take every tile
//   narrow  up to 128 rows: both streams have them, and take tiles in turn
// Warps 0-3 and 4-7 are the streams' softmax (a thread a row), 8 to 11 copy K, V
// and Q (cp.async: pages of 16 positions are too small for tensor copies to
// pay), warp 12 issues the products.  All waits are bounded: a block that
// gives one up writes NaN.
//
// 131,071 positions, 64 drafts of 8 heads, bf16: 109 us, 630 TFLOP/s: tensor cores and
// exponentials (16 a cycle and SM) are each busy for 35 % of it, bound by the chain of a stream
// (S, its softmax by one warp an SM quarter, P, O) that the other one covers in part.
// 8 sequences of up to 8,448, 16 drafts: 29 us, 1.3 TB/s, four tiles a block: most of it is
// the start, the end and the join.  16 of 4,000, 64 drafts, a block a segment of 128 rows: 53 us.
//
// Over a packed cache (PACKED) warps 8 to 11 turn a chunk's codes into numbers of T on their way to shared memory:
// 16 bytes of a row are 8 consecutive dims of each of four pieces.  A tile's codes are loaded while the one before
// it is turned.  131,071 positions, 64 drafts, f16: 147 us, 468 TFLOP/s (a plain bf16 cache takes 114 us): a tile of 128
// rows takes 2.7 us, of which the turning is the longest part.  8 sequences of up to 8,448, 16
// drafts, bf16: 35 us.
#pragma once
#include "packed.cuh"
#include "tree_attn.cuh"

namespace ocrvl {
namespace paged {

constexpr int kCopyWarps = 4, kCopyThreads = kCopyWarps * 32;
constexpr int kMmaWarp = 8 + kCopyWarps;
constexpr int kMmaThreads = (kMmaWarp + 1) * 32;
constexpr int kMmaWaits = 1 << 20;  // polls, of up to some microseconds each, before a wait is given up
// The reference stands kMmaLift below the largest score when it is set, and rises once 32 weights
// sum to more than kMmaMost: half of f16's largest for f16, whose small weights need the room
// (kLift), with as much slack as there is left.
template <typename T>
constexpr float kMmaLift = std::is_same<T, __half>::value ? 6.f : 0.f;
template <typename T>
constexpr float kMmaMost = std::is_same<T, __half>::value ? 32768.f : 4096.f;

// ---- barriers and tensor memory ------------------------------------------

__device__ __forceinline__ void bar_init(uint64_t *b, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
// Waits for the end of the phase of that parity; false when given up (by
// anybody: *dead).
__device__ __forceinline__ bool bar_wait(uint64_t *b, uint32_t parity, volatile int *dead) {
  for (int i = 0; i < kMmaWaits; i++) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(b)), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((i & 63) == 63 && *dead) return false;
  }
  *dead = 1;
  return false;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t *b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(b)) : "memory");
}
// 32 columns of the warp's lanes; the values are there behind tc_load_wait.
__device__ __forceinline__ void tc_load32_start(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tc_load_wait(uint32_t (&v)[32]) {  // the operands tie the values' uses to the wait
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]),
                 "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]),
                 "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28])
               :
               : "memory");
  asm volatile("" : "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
__device__ __forceinline__ void tc_load32(uint32_t addr, uint32_t (&v)[32]) {
  tc_load32_start(addr, v);
  tc_load_wait(v);
}
__device__ __forceinline__ void tc_load16(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_store16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tc_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A whole sector of 32 bytes: rows lie in threads, so narrower stores would reach
// L2 as halves of sectors.
__device__ __forceinline__ void store_sector(float *p, const float *v) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ uint32_t times2(uint32_t two, float x, __half) {
  __half2 h = __hmul2(*reinterpret_cast<__half2 *>(&two), __float2half2_rn(x));
  return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t times2(uint32_t two, float x, __nv_bfloat16) {
  __nv_bfloat162 h = __hmul2(*reinterpret_cast<__nv_bfloat162 *>(&two), __float2bfloat162_rn(x));
  return *reinterpret_cast<uint32_t *>(&h);
}

// Meets the 256 threads of warps 0 to 7 and says whether x holds for any of them.
__device__ __forceinline__ bool softmax_any(bool x) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.pred.aligned p, 1, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(any)
      : "r"((uint32_t)x)
      : "memory");
  return any != 0;
}

// ---- products -----------------------------------------------------------------

// One lane of the converged warp.  Behind this predicate a product of N = 128 was measured at 64
// cycles, the tensor cores' own rate, against 80 to 88 behind a test of the lane.
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.b32 %0, 1, 0, P;\n\t}\n" : "=r"(p));
  return p != 0;
}

// Shared-memory matrix descriptor of rows of 128 bytes, 128-byte swizzle.
//   K-major (Q, K: a row's 64 dims are contracted): groups of 8 rows 1 KB apart
//   MN-major (V: a row is a position, its 64 dims are columns of the output):
//     groups of 8 positions 1 KB apart, the next 64 dims `next` bytes on
__device__ __forceinline__ uint64_t mma_desc(uint32_t addr, int next) {
  return (uint64_t)(addr >> 4 & 0x3fff) | (uint64_t)(next >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// Instruction descriptor: f32 accumulator, A and B of T, M = 128.
template <typename T>
__device__ __forceinline__ constexpr uint32_t mma_idesc(int n, bool b_mn_major) {
  const uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
  return 1u << 4 | type << 7 | type << 10 | (b_mn_major ? 1u : 0u) << 16 | (uint32_t)(n >> 3) << 17 | 128u >> 4 << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
               "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
               "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
               : "memory");
}

template <int D, bool WIDE>
struct MmaShape {
  static constexpr int kRows = WIDE ? 256 : 128;
  static constexpr int kHalves = D / 64;              // blocks of 128 rows x 128 bytes
  static constexpr int kBlock = kHalves * 16384;      // a tile of Q, K or V
  static constexpr int kStages = D == 64 ? 4 : WIDE ? 2 : 3;
  static constexpr int kQ = (WIDE ? 2 : 1) * kBlock;
  static constexpr int kMeta = 8;                     // tiles whose chunks are described at a time
  static constexpr int kTiles = kQ + 2 * kStages * kBlock;
  static constexpr int kSmem = kTiles + (4 * kStages + 9 + kMeta) * 8 + kMeta * 8 * 4 + 2 * 128 * 8 + 64 + 32;
};

// What a lane of a copying warp takes of a packed chunk: 16 bytes of codes of rows row(i), pieces of 8 dims
// which each hold, and the rows' scales.
template <typename T, int D>
struct PackedChunk {
  static constexpr int PER = D / 64;  // 16-byte runs a lane
  uint4 codes[PER];
  uint32_t scales[PER][D / 64];

  // Rows and runs so that the eight lanes of a store phase write to eight pieces of 16 bytes that lie in different banks.
  static __device__ __forceinline__ int run(int lane) { return D == 128 ? lane & 3 : lane & 1; }
  static __device__ __forceinline__ int row(int lane, int i) {
    return D == 128 ? (lane >> 3) + (lane >> 2 & 1) * 4 + i * 8 : (lane >> 1 & 1) + (lane >> 2 & 1) * 4 + (lane >> 3 & 1) * 2 + (lane >> 4) * 8;
  }
  __device__ __forceinline__ void load(const char *from, const char *from_s, int valid, int lane) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int r = row(lane, i);
      codes[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int w = 0; w < D / 64; w++) scales[i][w] = 0u;
      if (r < valid) {
        codes[i] = __ldg((const uint4 *)(from + r * (D / 2)) + run(lane));
        if constexpr (D == 128) {
          const uint2 s = __ldg((const uint2 *)(from_s + r * 8));
          scales[i][0] = s.x, scales[i][D / 64 - 1] = s.y;
        } else {
          scales[i][0] = __ldg((const uint32_t *)(from_s + r * 4));
        }
      }
    }
  }
  // To the chunk's rows of a tile.
  __device__ __forceinline__ void store(uint32_t to, int lane) const {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int r = row(lane, i), x = run(lane);
      const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int j = D == 128 ? q : q >> 1;  // the group
        const uint32_t c = D == 128 ? halves(w[q >> 1], w[2 + (q >> 1)], q & 1) : halves(w[2 * (q & 1)], w[2 * (q & 1) + 1], q >> 1);
        uint32_t s = __byte_perm(scales[i][j >> 1], 0, j & 1 ? 0x3232 : 0x1010);
        if constexpr (std::is_same<T, __half>::value) {
          const float f = __uint_as_float(s << 16);
          s = pack2(f, f, T());
        }
        const Scaled<T> by(s);
        uint32_t y[4];
#pragma unroll
        for (int k = 0; k < 4; k++) y[k] = by(c, k);
        const int piece = D == 128 ? (j & 1) * 4 + x : j * 4 + x * 2 + (q & 1);
        sts4u(to + (D == 128 ? j >> 1 : 0) * 16384 + r * 128 + ((piece ^ (r & 7)) * 16), low_halves(y[0], y[1]), low_halves(y[2], y[3]),
              high_halves(y[0], y[1]), high_halves(y[2], y[3]));
      }
    }
  }
};

template <typename T, int D, bool WIDE, bool SPLIT, bool PACKED>
__global__ void __launch_bounds__(kMmaThreads, 1) k_tree_mma(const TreeArgs a, int row_blocks) {
  using S = MmaShape<D, WIDE>;
  constexpr int NS = S::kStages;
  extern __shared__ __align__(1024) char sm_tiles[];  // the swizzle goes by address bits
  char *sm = sm_tiles;
  char *q_sm = sm, *k_sm = sm + S::kQ, *v_sm = k_sm + NS * S::kBlock;
  // behind the tiles, by falling alignment
  int *meta = (int *)(sm + S::kTiles);  // [tile % kMeta][chunk]: positions there | draft << 8 | not finite << 9 | first draft << 16
  float2 *ml = (float2 *)(meta + S::kMeta * 8);  // [stream][row]: reference and sum
  long long *plan = (long long *)(ml + 2 * 128);
  uint64_t *k_full = (uint64_t *)(plan + 8), *k_empty = k_full + NS, *v_full = k_empty + NS, *v_empty = v_full + NS;
  uint64_t *s_full = v_empty + NS, *p_ready = s_full + 2, *o_full = p_ready + 2, *meta_full = o_full + 2;
  uint64_t *o_free = meta_full + S::kMeta, *q_full = o_free + 1, *q_empty = q_full + 1;
  uint32_t *tmem_at = (uint32_t *)(q_empty + 1);
  volatile int *dead = (volatile int *)(tmem_at + 1);
  const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      bar_init(&k_full[i], kCopyThreads), bar_init(&v_full[i], kCopyThreads);
      bar_init(&k_empty[i], 1), bar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) bar_init(&s_full[i], 1), bar_init(&p_ready[i], 128), bar_init(&o_full[i], 1);
    for (int i = 0; i < S::kMeta; i++) bar_init(&meta_full[i], kCopyWarps);
    bar_init(o_free, 256), bar_init(q_full, kCopyThreads), bar_init(q_empty, 1);
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_at)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    tc_before();
  }
  if constexpr (PACKED) pdl_wait();
  Piece cur;
  Walk walk;
  bool more = true;
  if constexpr (PACKED && !SPLIT) pdl_launch();
  if constexpr (SPLIT) {
    more = walk.start(a, S::kRows, plan, warp, lane, cur);
    pdl_launch();
  } else {
    const int seg = blockIdx.x;
    cur.rb = seg % row_blocks, cur.head = seg / row_blocks % a.kv_heads, cur.b = seg / row_blocks / a.kv_heads;
    cur.sg = Segments(a, cur.b, S::kRows);
    cur.t0 = 0, cur.t1 = cur.sg.tiles;
    more = cur.rb < cur.sg.blocks;
  }
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_at;
  auto advance = [&]() {
    if constexpr (SPLIT)
      more = walk.next(a, S::kRows, cur);
    else
      more = false;
  };
  auto rows_of = [&](const Piece &x) { return min(S::kRows, x.sg.count * a.group - x.rb * S::kRows); };
  // tiles of stream s in a piece of n tiles
  auto tiles_of = [](int s, int n, int rows) { return WIDE ? (s * 128 < rows ? n : 0) : (n + 1 - s) / 2; };
  uint32_t T0 = 0;  // tiles of the pieces before

  if (warp < 8) {
    // ---- softmax: stream s, row r of its tile ---------------------------------
    const int s = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // the warp's 32 lanes of tensor memory
    const uint32_t s_at = tmem + lanes + s * 128, o_at = tmem + lanes + 256 + s * 128;
    uint32_t steps = 0, ends[2] = {0, 0};  // tiles of the stream, pieces that each stream had tiles in, so far
    for (int piece = 0; more; piece++) {
      const int rows = rows_of(cur), n = cur.t1 - cur.t0, n_s = tiles_of(s, n, rows);
      const int row = (WIDE ? s * 128 : 0) + r, first = cur.rb * S::kRows + row;
      const bool works = row - lane < rows;  // the warp has rows
      const unsigned long long seen = row < rows ? (unsigned long long)a.mask[cur.sg.first + first / a.group] : 0ull;
      float ref = -INFINITY, sum = 0.f, low = 0.f;
      bool ok = true, poison = false;
      for (int i = 0; i < n_s && ok; i++, steps++) {
        const uint32_t tile = T0 + (WIDE ? i : 2 * i + s);
        ok = bar_wait(&meta_full[tile % S::kMeta], tile / S::kMeta & 1, dead) && bar_wait(&s_full[s], steps & 1, dead);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        tc_after();
        if (works) {
          uint32_t v[2][32];
          tc_load32_start(s_at, v[0]);
          const int4 *m4 = (const int4 *)(meta + tile % S::kMeta * 8);
          const int4 ma = m4[0], mb = m4[1];
          const int m8[8] = {ma.x, ma.y, ma.z, ma.w, mb.x, mb.y, mb.z, mb.w};
          bool all = true;  // every position is there and seen
#pragma unroll
          for (int c = 0; c < 8; c++) all &= m8[c] == 16;
          uint32_t see[4] = {~0u, ~0u, ~0u, ~0u};  // which of the 128 positions the row sees
          if (!all) {
#pragma unroll
            for (int c = 0; c < 8; c++) {
              const int x = m8[c];
              uint32_t bits = (1u << (x & 31)) - 1;
              if (x >> 8 & 1) bits &= (uint32_t)(seen >> (x >> 16));
              poison |= x >> 9 & 1;
              see[c >> 1] = c & 1 ? (see[c >> 1] & 0xffff) | bits << 16 : bits & 0xffff;
            }
          }
          // 32 columns at a time, the next ones on their way meanwhile; P goes over
          // columns of S that were read.  The reference starts as the first tile's maximum
          // and rises, by a whole power of two so that what is there already is scaled
          // exactly, only once 32 weights sum to more than kMmaMost: no maximum
          // stands before the exponentials, which bound this loop (4 lanes a cycle
          // and SM quarter).
          if (__any_sync(~0u, ref == -INFINITY)) {
            tc_load_wait(v[0]);
            float top = -INFINITY;
#pragma unroll 1
            for (int q = 3; q >= 0; q--) {
              tc_load32(s_at + q * 32, v[0]);
              const uint32_t m = q < 2 ? (q ? see[1] : see[0]) : q == 2 ? see[2] : see[3];
#pragma unroll
              for (int j = 0; j < 32; j++)
                if (m >> j & 1) top = fmaxf(top, __uint_as_float(v[0][j]) * a.scale);
            }
            if (ref == -INFINITY) ref = top - kMmaLift<T>;  // and v[0] holds the first columns again
          }
          auto tile_pass = [&](auto masked) {
            constexpr bool MASKED = decltype(masked)::value;
#pragma unroll 1
            for (int q2 = 0; q2 < 4; q2 += 2)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const int q = q2 + e;
                const uint32_t m = e ? (q2 ? see[3] : see[1]) : q2 ? see[2] : see[0];
                uint32_t(&x)[32] = v[e];
                tc_load_wait(x);
                if (q < 3) tc_load32_start(s_at + (q + 1) * 32, v[e ^ 1]);
                uint32_t p16[16];
                float add;
                for (bool again = false;; again = true) {
                  const float base = ref == -INFINITY ? 0.f : ref;
                  // the exponentials follow one another without waiting for each other's
                  // results; what comes before and behind them goes in between
                  float add0 = 0.f, add1 = 0.f;
                  auto before = [&](int j) {
                    float y = fmaf(__uint_as_float(x[j]), a.scale, -base);
                    if (MASKED && !(m >> j & 1)) y = -INFINITY;
                    x[j] = __float_as_uint(y);
                  };
                  constexpr int AHEAD = 4, BEHIND = 6;
#pragma unroll
                  for (int j = 0; j < AHEAD; j++) before(j);
#pragma unroll
                  for (int j = 0; j < 32 + BEHIND; j++) {
                    if (j + AHEAD < 32) before(j + AHEAD);
                    if (j < 32) asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+r"(x[j]));
                    if (j >= BEHIND && (j - BEHIND) % 2 == 1) {
                      const int k = j - BEHIND - 1;
                      const float y = __uint_as_float(x[k]), z = __uint_as_float(x[k + 1]);
                      add0 += y, add1 += z;
                      p16[k / 2] = pack2(y, z, T());
                    }
                  }
                  add = add0 + add1;
                  if (again || !__any_sync(~0u, add > kMmaMost<T>)) break;
                  tc_store_wait();  // P's columns and O may have been stored a moment ago: loads are not ordered behind that
                  tc_load32(s_at + q * 32, x);  // still there
                  float top = 0.f;
#pragma unroll
                  for (int j = 0; j < 32; j++)
                    if (!MASKED || m >> j & 1) top = fmaxf(top, fmaf(__uint_as_float(x[j]), a.scale, -base));
                  const float down = add > kMmaMost<T> ? ceilf(top) - kMmaLift<T> : 0.f, alpha = exp2_(-down);
                  ref = down > 0.f ? base + down : ref;
                  sum *= alpha, low *= alpha;
                  uint32_t w[16];
#pragma unroll 1
                  for (int c = 0; c < q; c++) {
                    tc_load16(s_at + c * 16, w);
#pragma unroll
                    for (int k = 0; k < 16; k++) w[k] = times2(w[k], alpha, T());
                    tc_store16(s_at + c * 16, w);
                  }
#pragma unroll 1
                  for (int c = 0; c < (i > 0 ? D / 16 : 0); c++) {  // S is there, so the products before it are done: O rests
                    tc_load16(o_at + c * 16, w);
#pragma unroll
                    for (int k = 0; k < 16; k++) w[k] = __float_as_uint(__uint_as_float(w[k]) * alpha);
                    tc_store16(o_at + c * 16, w);
                  }
                }
                add_exactly(sum, low, add);
                tc_store16(s_at + q * 16, p16);
              }
          };
          if (all)
            tile_pass(std::false_type());
          else
            tile_pass(std::true_type());
          tc_store_wait();
        }
        tc_before();
        bar_arrive(&p_ready[s]);
      }
      // ---- the piece's end --------------------------------------------------
      sum += low;
      const int n_0 = tiles_of(0, n, rows), n_1 = tiles_of(1, n, rows);
      ends[0] += n_0 > 0, ends[1] += n_1 > 0;
      // A stream without tiles waits for the other's end: were it to arrive at o_free for pieces ahead, the
      // phase would end while the other still reads its O.
      if (n_0 && !(WIDE && s == 1 && n_1)) ok = ok && bar_wait(&o_full[0], (ends[0] - 1) & 1, dead);
      if (n_1 && !(WIDE && s == 0)) ok = ok && bar_wait(&o_full[1], (ends[1] - 1) & 1, dead);
      ok = __all_sync(~0u, ok);
      tc_after();
      const bool whole = cur.t0 == 0 && cur.t1 == cur.sg.tiles;
      const long long slot = 2 * (long long)blockIdx.x + (piece ? 1 : 0);
      if (SPLIT && tid == 0) walk.tell(a, cur, row_blocks, (int)slot);
      const int tok = cur.sg.first + first / a.group, hd = cur.head * a.group + first % a.group;
      float f0 = 1.f, f1 = 0.f, top = ref, l = sum;  // weights of this stream's and the other's O
      if constexpr (!WIDE) {
        ml[s * 128 + r] = make_float2(ref, sum);
        poison = softmax_any(poison);  // a thread adds up half the dims of both streams' tiles
        const float2 x = ml[r], y = ml[128 + r];
        top = n_1 ? fmaxf(x.x, y.x) : x.x;
        const float base = top == -INFINITY ? 0.f : top;
        f0 = exp2_(x.x - base), f1 = n_1 ? exp2_(y.x - base) : 0.f;
        l = f0 * x.y + f1 * (n_1 ? y.y : 0.f);
      }
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
      f0 *= inv, f1 *= inv;
      constexpr int kMine = WIDE ? D / 32 : D / 64;  // groups of 32 dims that this thread writes
      if (works && (WIDE ? n_s > 0 : true)) {
#pragma unroll
        for (int q = 0; q < kMine; q++) {
          const int d0 = (WIDE ? 0 : s * (D / 2)) + q * 32;
          const uint32_t at = tmem + lanes + 256 + (WIDE ? s * 128 : 0) + d0;
          uint32_t v[32];
          float o[32];
          tc_load32(at, v);
#pragma unroll
          for (int j = 0; j < 32; j++) o[j] = __uint_as_float(v[j]) * f0;
          if (!WIDE && n_1) {
            tc_load32(at + 128, v);
#pragma unroll
            for (int j = 0; j < 32; j++) o[j] = fmaf(__uint_as_float(v[j]), f1, o[j]);
          }
          if (row < rows) {
            if (poison) {  // values of drafts that are not finite, and that the row sees
              for (int t = 0; t < cur.sg.count; t++)
                if (seen >> t & 1 && t / kChunk + cur.sg.chunks_c >= cur.t0 * kTileChunks && t / kChunk + cur.sg.chunks_c < cur.t1 * kTileChunks) {
                  const T *x = (const T *)a.dv + (cur.sg.first + t) * a.kv_stride + (long long)cur.head * D + d0;
#pragma unroll
                  for (int j = 0; j < 32; j++) {
                    const float y = to_f(x[j]);
                    if (!isfinite(y)) o[j] += y;
                  }
                }
            }
            if (!ok) {
#pragma unroll
              for (int j = 0; j < 32; j++) o[j] = NAN;
            }
            if (whole) {
              T *to = (T *)a.out + tok * a.out_stride + (long long)hd * D + d0;
#pragma unroll
              for (int j = 0; j < 32; j += 8)
                *(uint4 *)(to + j) = make_uint4(pack2(o[j], o[j + 1], T()), pack2(o[j + 2], o[j + 3], T()), pack2(o[j + 4], o[j + 5], T()),
                                                pack2(o[j + 6], o[j + 7], T()));
            } else {
              float *to = a.part + (slot * S::kRows + row) * D + d0;
#pragma unroll
              for (int j = 0; j < 32; j += 8) store_sector(to + j, o + j);
            }
          }
        }
        if (row < rows && (WIDE || s == 0)) {
          if (!ok) l = NAN;
          if (!whole)
            *(float2 *)(a.part_ml + (slot * S::kRows + row) * 2) = make_float2(top, l);
          else if (a.lse)
            a.lse[(long long)tok * a.kv_heads * a.group + hd] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
        }
      }
      tc_before();
      bar_arrive(o_free);
      if constexpr (!WIDE) asm volatile("bar.sync 1, 256;" ::: "memory");  // ml is read
      T0 += n;
      advance();
    }
  } else if (warp < kMmaWarp) {
    // ---- copies -----------------------------------------------------------------
    const int w = warp - 8;
    constexpr int CH = kTileChunks / kCopyWarps;  // chunks of a tile that the warp copies
    constexpr int kPieces = D * 2 / 16;   // 16-byte pieces a row
    constexpr int kAtOnce = 32 / kPieces;  // rows a warp copies at once
    auto not_finite = [](uint32_t two) {  // either of two 16-bit values
      constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
      return (two & e) == e || (two >> 16 & e) == e;
    };
    bool ok = true;
    // a barrier's arrival once this thread's copies so far have landed
    auto landed = [](uint64_t *b) {
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(b)) : "memory");
    };
    const int piece16 = lane % kPieces, r0 = lane / kPieces;
    uint32_t to_off[kChunk / kAtOnce];  // where the lane's pieces of a chunk go
#pragma unroll
    for (int j = 0; j < kChunk / kAtOnce; j++) {
      const int row = j * kAtOnce + r0;
      to_off[j] = (piece16 >> 3) * 16384 + row * 128 + ((piece16 & 7) ^ (row & 7)) * 16;
    }
    for (int piece = 0; more && ok; piece++) {
      const int n = cur.t1 - cur.t0, rows = rows_of(cur);
      int pages = -1;  // lane i: the page of the warp's i-th chunk from the last look on
      auto of = [](const char *x, int h) { return (const char *)__shfl_sync(~0u, (unsigned long long)x, h); };
      // lane h < CH: where the warp's chunk h of a tile lies; the tiles are asked for in order
      struct Where {
        const char *k, *v, *ks, *vs;
        int row_bytes, valid, what;
      };
      auto where = [&](int i) {
        if (i % (32 / CH) == 0) {
          const int c = (cur.t0 + i + lane / CH) * kTileChunks + CH * w + lane % CH;
          pages = c < cur.sg.chunks_c ? a.c.table[cur.b * a.c.table_stride + ((c * kChunk) >> a.c.page_shift)] : -1;
        }
        const int c = (cur.t0 + i) * kTileChunks + CH * w + lane % CH;
        const int pg = __shfl_sync(~0u, pages, i % (32 / CH) * CH + lane % CH);
        Where x;
        x.what = 0, x.ks = x.vs = nullptr;
        if (c < cur.sg.chunks_c) {
          const int pos = c * kChunk;
          const bool mapped = pg >= 0 && pg < a.c.num_pages;
          x.valid = mapped ? min(kChunk, cur.sg.len - pos) : 0;
          x.row_bytes = a.c.token_bytes;
          const long long in_page = pos & ((1 << a.c.page_shift) - 1);
          const long long at = (mapped ? pg : 0) * a.c.page_bytes + cur.head * a.c.head_bytes + in_page * a.c.token_bytes;
          x.k = a.c.k + at, x.v = a.c.v + at;
          if constexpr (PACKED) {
            const long long at_s = (mapped ? pg : 0) * a.scale_page + cur.head * a.scale_head + in_page * (D / 16);
            x.ks = a.k_scale + at_s, x.vs = a.v_scale + at_s;
          }
        } else {
          const int j = (c - cur.sg.chunks_c) * kChunk;
          x.valid = max(0, min(kChunk, cur.sg.count - j));
          x.row_bytes = (int)(a.kv_stride * (long long)sizeof(T));
          const long long at = (cur.sg.first + (x.valid ? j : 0)) * a.kv_stride + (long long)cur.head * D;
          x.k = (const char *)((const T *)a.dk + at), x.v = (const char *)((const T *)a.dv + at);
          x.what = x.valid ? 1 << 8 | j << 16 : 0;
        }
        return x;
      };
      // PACKED: the warp's codes of a tile, the next one's fetched as soon as this one's are turned into numbers
      PackedChunk<T, D> codes_k[PACKED ? CH : 1], codes_v[PACKED ? CH : 1];
      auto fetch = [&](PackedChunk<T, D> *to, const Where &x, bool v) {
#pragma unroll
        for (int h = 0; h < CH; h++)
          to[h].load(of(v ? x.v : x.k, h), of(v ? x.vs : x.ks, h), __shfl_sync(~0u, x.what ? 0 : x.valid, h), lane);
      };
      Where at = where(0), at_next = at;
      if constexpr (PACKED) fetch(codes_k, at, false), fetch(codes_v, at, true);
      for (int i = 0; i < n && ok; i++) {
        const uint32_t tile = T0 + i, stage = tile % NS, use = tile / NS;
        if constexpr (PACKED) {
          at = at_next;
          if (i + 1 < n) at_next = where(i + 1);
        } else {
          if (i) at = where(i);
        }
        const char *src_k = at.k, *src_v = at.v;
        const int row_bytes = at.row_bytes, valid = at.valid, what = at.what;
        unsigned draft = __ballot_sync(~0u, what != 0 && lane < CH), odd = 0;  // chunks of drafts; those with values that are not finite
        for (; draft; draft &= draft - 1) {
          const int h = __ffs(draft) - 1, n_h = __shfl_sync(~0u, valid, h), row = __shfl_sync(~0u, row_bytes, h);
          const char *v = of(src_v, h);
          bool any = false;
          for (int x = lane; x < n_h * kPieces; x += 32) {
            const uint4 y = __ldg((const uint4 *)(v + (long long)(x / kPieces) * row) + x % kPieces);
            any |= not_finite(y.x) || not_finite(y.y) || not_finite(y.z) || not_finite(y.w);
          }
          odd |= (__any_sync(~0u, any) ? 1u : 0u) << h;
        }
        if (lane < CH) meta[tile % S::kMeta * 8 + CH * w + lane] = valid | what | (odd >> lane & 1 ? 1 << 9 : 0);
        __syncwarp();
        auto copy = [&](char *to, const char *src, const PackedChunk<T, D> *packed) {
          const uint32_t base = smem_addr(to) + CH * w * kChunk * 128;
          if constexpr (PACKED) {
#pragma unroll
            for (int h = 0; h < CH; h++)
              if (!__shfl_sync(~0u, what, h)) packed[h].store(base + h * kChunk * 128, lane);
            if (!__any_sync(~0u, what)) return;
          }
#pragma unroll 1
          for (int h = 0; h < CH; h++) {
            if (PACKED && !__shfl_sync(~0u, what, h)) continue;
            const int n_h = __shfl_sync(~0u, valid, h);
            const long long row_h = __shfl_sync(~0u, row_bytes, h);
            const char *from = of(src, h) + piece16 * 16 + r0 * row_h;
            if (n_h == kChunk) {
#pragma unroll
              for (int j = 0; j < kChunk / kAtOnce; j++) copy16(base + h * kChunk * 128 + to_off[j], from + j * kAtOnce * row_h, true);
            } else {
#pragma unroll
              for (int j = 0; j < kChunk / kAtOnce; j++) {
                const bool in = j * kAtOnce + r0 < n_h;
                copy16(base + h * kChunk * 128 + to_off[j], in ? from + j * kAtOnce * row_h : src, in);
              }
            }
          }
        };
        ok = __all_sync(~0u, use == 0 || bar_wait(&k_empty[stage], (use - 1) & 1, dead));
        if (!ok) break;
        if (lane == 0) bar_arrive(&meta_full[tile % S::kMeta]);
        copy(k_sm + stage * S::kBlock, src_k, codes_k);
        if constexpr (PACKED) {
          copy_commit();
          copy_wait<0>();
          bar_arrive(&k_full[stage]);
          if (i + 1 < n) fetch(codes_k, at_next, false);
        } else {
          landed(&k_full[stage]);
        }
        if (i == 0) {  // the query rows, once the piece before has no more use for its own
          ok = __all_sync(~0u, piece == 0 || bar_wait(q_empty, (piece - 1) & 1, dead));
          if (!ok) break;
          constexpr int kMine = S::kRows / kCopyWarps;  // the warp's rows; a lane works out every 32nd's address
#pragma unroll 1
          for (int x0 = 0; x0 < kMine; x0 += 32) {
            const int mine = w * kMine + x0 + lane, q = cur.rb * S::kRows + mine;
            const char *at = (const char *)((const T *)a.q + (cur.sg.first + q / a.group) * a.q_stride + (long long)(cur.head * a.group + q % a.group) * D);
            if (mine >= rows) at = nullptr;
#pragma unroll 8
            for (int x = 0; x < 32; x += kAtOnce) {
              const char *from = of(at, x + r0);
              const int row = w * kMine + x0 + x + r0;
              copy16(smem_addr(q_sm) + (row >> 7) * S::kBlock + (piece16 >> 3) * 16384 + (row & 127) * 128 + ((piece16 & 7) ^ (row & 7)) * 16,
                     from ? from + piece16 * 16 : (const char *)a.q, from != nullptr);
            }
          }
          landed(q_full);
        }
        ok = __all_sync(~0u, use == 0 || bar_wait(&v_empty[stage], (use - 1) & 1, dead));
        if (!ok) break;
        copy(v_sm + stage * S::kBlock, src_v, codes_v);
        if (!PACKED && !odd) {
          landed(&v_full[stage]);
        } else {  // what is not finite becomes 0 here (0 * NaN would reach rows that do not see it) and is added at the end
          copy_commit();
          copy_wait<0>();
          const uint32_t base = smem_addr(v_sm + stage * S::kBlock) + CH * w * kChunk * 128;
          for (unsigned left = odd; left; left &= left - 1)
#pragma unroll
            for (int j = 0; j < kChunk / kAtOnce; j++) {
              const uint32_t at = base + (__ffs(left) - 1) * kChunk * 128 + to_off[j];
              uint32_t x[4];
              lds4u(x, at);
#pragma unroll
              for (int k = 0; k < 4; k++) {
                if (not_finite(x[k] << 16)) x[k] &= 0xffff0000u;
                if (not_finite(x[k] & 0xffff0000u)) x[k] &= 0xffffu;
              }
              sts4u(at, x[0], x[1], x[2], x[3]);
            }
          bar_arrive(&v_full[stage]);
          if (PACKED && i + 1 < n) fetch(codes_v, at_next, true);
        }
      }
      if (!ok) break;
      T0 += n;
      advance();
    }
    copy_commit();
    copy_wait<0>();
  } else {
    // ---- products -----------------------------------------------------------------
    // The whole warp takes every step; one lane issues.
    // The copies were written like plain stores: to be seen by the products, which read
    // by another proxy, they need a fence behind the wait for them.
    auto wait_copies = [&](uint64_t *b, uint32_t parity) {
      const bool there = bar_wait(b, parity, dead);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      return there;
    };
    constexpr uint32_t i_s = mma_idesc<T>(128, false), i_o = mma_idesc<T>(D, true);
    const uint64_t q_desc = mma_desc(smem_addr(q_sm), 16), k_desc = mma_desc(smem_addr(k_sm), 16), v_desc = mma_desc(smem_addr(v_sm), 16384);
    uint32_t p_steps[2] = {0, 0};
    bool ok = true;
    for (int piece = 0; more && ok; piece++) {
      const int n = cur.t1 - cur.t0, rows = rows_of(cur);
      const int n_s[2] = {tiles_of(0, n, rows), tiles_of(1, n, rows)}, total = n_s[0] + n_s[1];
      const int last_stream = n_s[1] ? 1 : 0;
      int scored = 0;
      auto score = [&](int s, int i) {
        const uint32_t tile = T0 + (WIDE ? i : 2 * i + s), stage = tile % NS;
        if (!WIDE || s == 0) {
          if (!__all_sync(~0u, wait_copies(&k_full[stage], tile / NS & 1))) return false;
        }
        tc_after();
        const uint64_t q = q_desc + (WIDE ? s * S::kBlock : 0) / 16, k = k_desc + stage * (S::kBlock / 16);
        scored++;
        if (elected()) {
#pragma unroll
          for (int h = 0; h < S::kHalves; h++)
#pragma unroll
            for (int j = 0; j < 4; j++)
              mma_ss(tmem + s * 128, q + (h * 16384 + j * 32) / 16, k + (h * 16384 + j * 32) / 16, i_s, h + j > 0);
          tc_commit(&s_full[s]);
          if (!WIDE || s == last_stream) tc_commit(&k_empty[stage]);
          if (scored == total) tc_commit(q_empty);
        }
        __syncwarp();
        return true;
      };
      ok = __all_sync(~0u, wait_copies(q_full, piece & 1));
      for (int s = 0; s < 2 && ok; s++)
        if (n_s[s]) ok = score(s, 0);
      if (ok && piece) ok = __all_sync(~0u, bar_wait(o_free, (piece - 1) & 1, dead));
      for (int i = 0; i < n_s[0] && ok; i++)
#pragma unroll
        for (int s = 0; s < 2; s++) {
          if (i >= n_s[s] || !ok) continue;
          const uint32_t tile = T0 + (WIDE ? i : 2 * i + s), stage = tile % NS;
          ok = bar_wait(&p_ready[s], p_steps[s]++ & 1, dead) && wait_copies(&v_full[stage], tile / NS & 1);
          ok = __all_sync(~0u, ok);
          if (!ok) continue;
          tc_after();
          const uint64_t v = v_desc + stage * (S::kBlock / 16);
          if (elected()) {
#pragma unroll
            for (int j = 0; j < 8; j++)
              mma_ts(tmem + 256 + s * 128, tmem + s * 128 + j * 8, v + j * 2048 / 16, i_o, i > 0 || j > 0);
            if (!WIDE || s == last_stream) tc_commit(&v_empty[stage]);
            if (i == n_s[s] - 1) tc_commit(&o_full[s]);
          }
          __syncwarp();
          if (i + 1 < n_s[s]) ok = score(s, i + 1);
        }
      T0 += n;
      advance();
    }
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace paged
}  // namespace ocrvl
