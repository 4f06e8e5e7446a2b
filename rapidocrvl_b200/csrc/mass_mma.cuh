// The attention weight that cached positions got (attn_mass.cuh's mathematics) for
// 16-bit types and many rows, on the tensor cores' fifth generation.
//
// S' = K Q' of a tile of 128 positions and up to 128 rows in tensor memory has a position a lane
// and a row a column, so a thread has a position and adds its rows' weights by itself: no
// shuffles, no join.  A block keeps up to 256 rows of Q in shared memory (more: further passes over
// its run, each adding to what the one before wrote), streams K's tiles past them and has two
// groups of four warps take tiles by turns, each with two accumulators, so that a product
// runs while the last one's weights are summed.  Warps 8 to 11 copy, warp 12 issues.  Bound
// by the exponentials: 128 rows a tile take 1,024 cycles of an SM's 16 a cycle.  All waits are
// bounded: what a block gave up is NaN.
//
// bf16, 131,072 positions, 64 drafts of 8 heads: 62 us, 550 TFLOP/s (30 us of it exponentials; K is
// read twice); 64 sequences of 4,000, one token: 31 us, 4.2 TB/s; 4 of up to 8,448, 32 drafts:
// 12.7 us, a launch and the first loads of Q and K.
#pragma once
#include "attn_mass.cuh"
#include "tree_mma.cuh"

namespace ocrvl {
namespace paged {

template <int D>
struct MassMmaShape {
  static constexpr int kHalves = D / 64;
  static constexpr int kBlock = kHalves * 16384;  // 128 rows of Q, or positions of K
  static constexpr int kRows = 256;
  static constexpr int kStages = D == 64 ? 6 : 5;
  static constexpr int kTiles = (2 + kStages) * kBlock;
  static constexpr int kLoad = 12;
  static constexpr int kSmem = kTiles + kRows * 4 + 64 + (2 * kStages + 10) * 8 + 16;
};

template <typename T, int D>
__global__ void __launch_bounds__(kMmaThreads, 1) k_mass_mma(const MassArgs a) {
  using S = MassMmaShape<D>;
  constexpr int NS = S::kStages;
  extern __shared__ __align__(1024) char sm_tiles[];
  char *q_sm = sm_tiles, *k_sm = q_sm + 2 * S::kBlock;
  float *shift = (float *)(sm_tiles + S::kTiles);  // lse log2(e), +inf for rows that do not count
  long long *plan = (long long *)(shift + S::kRows);
  uint64_t *k_full = (uint64_t *)(plan + 8), *k_empty = k_full + NS, *s_full = k_empty + NS, *s_free = s_full + 4;
  uint64_t *q_full = s_free + 4, *q_empty = q_full + 1;
  uint32_t *tmem_at = (uint32_t *)(q_empty + 1);
  volatile int *dead = (volatile int *)(tmem_at + 1);
  const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < NS; i++) bar_init(&k_full[i], kCopyThreads), bar_init(&k_empty[i], 1);
    for (int i = 0; i < 4; i++) bar_init(&s_full[i], 1), bar_init(&s_free[i], 128);
    bar_init(q_full, kCopyThreads), bar_init(q_empty, 1);
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_at)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    tc_before();
  }
  if (warp == 0) mass_start(a, S::kLoad, blockIdx.x, gridDim.x, plan, lane);
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_at;

  // f(sequence, its share, head, tiles [t0, t1), first row, rows) for every pass over every segment
  // of the run; false ends it
  auto pieces = [&](auto f) {
    bool ok = true;
    mass_segments(a, S::kLoad, blockIdx.x, gridDim.x, plan, [&](const MassShare &sh, int b, int head, int t0, int t1) {
      const int rows = sh.count * a.group;
      for (int r0 = 0; ok && (r0 == 0 || r0 < rows); r0 += S::kRows) ok = f(b, sh, head, t0, t1, r0, min(S::kRows, rows - r0));
    });
  };
  // rows of a block of 128, in whole groups of 32
  auto columns = [](int rows, int rb) { return (min(128, rows - rb * 128) + 31) / 32 * 32; };

  if (warp < 8) {
    // ---- weights: a thread a position of the group's tile ----------------------------
    const int s = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    uint32_t items = 0;  // of this group
    bool ok = true;  // else all that is left becomes NaN: both groups take every piece to its end, they meet there
    pieces([&](int b, const MassShare &sh, int head, int t0, int t1, int r0, int rows) {
      const unsigned long long on = a.counted ? (unsigned long long)a.counted[b] : ~0ull;
      float l = INFINITY;
      if (tid < rows) {
        const int x = r0 + tid;
        if (on >> (x / a.group) & 1) {
          l = a.lse[(long long)(sh.first + x / a.group) * a.kv_heads * a.group + head * a.group + x % a.group] * kLog2e;
          if (l == -INFINITY) l = INFINITY;  // attended nothing
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the piece before is done with its own
      shift[tid] = l;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const float *acc = a.acc ? a.acc + ((long long)b * a.kv_heads + head) * a.acc_stride : nullptr;
      float *out = a.out + ((long long)b * a.kv_heads + head) * a.out_stride;
      const float keep = r0 ? 1.f : a.decay;
      for (int i = s; i < t1 - t0; i += 2) {
        const int pos = (t0 + i) * 128 + r;
        float old = 0.f, sum0 = 0.f, sum1 = 0.f;
        int pg = -1;
        if (pos < sh.len) {
          pg = a.c.table[b * a.c.table_stride + (pos >> a.c.page_shift)];
          old = r0 ? out[pos] : acc && pos < a.acc_width ? acc[pos] : 0.f;
        }
        for (int rb = 0; rb * 128 < rows && ok; rb++, items++) {
          const int buf = s * 2 + (items & 1), n = columns(rows, rb);
          ok = __all_sync(~0u, bar_wait(&s_full[buf], items >> 1 & 1, dead));
          if (!ok) break;
          tc_after();
          const uint32_t at = tmem + lanes + buf * 128;
          uint32_t v[2][32];
          tc_load32_start(at, v[0]);
          auto take = [&](int c, uint32_t(&x)[32]) {
            const float4 *l4 = (const float4 *)(shift + rb * 128 + c);
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 y = l4[j / 4];
              // a row that does not count adds nothing, whatever its query and the key hold
              auto weight = [&](uint32_t s, float l) { return exp2_(l == INFINITY ? -INFINITY : fmaf(__uint_as_float(s), a.scale, -l)); };
              sum0 += weight(x[j], y.x), sum1 += weight(x[j + 1], y.y);
              sum0 += weight(x[j + 2], y.z), sum1 += weight(x[j + 3], y.w);
            }
          };
#pragma unroll 1
          for (int c = 0; c < n; c += 64) {
            tc_load_wait(v[0]);
            if (c + 32 < n) tc_load32_start(at + c + 32, v[1]);
            take(c, v[0]);
            if (c + 32 < n) {
              tc_load_wait(v[1]);
              if (c + 64 < n) tc_load32_start(at + c + 64, v[0]);
              take(c + 32, v[1]);
            }
          }
          tc_before();
          bar_arrive(&s_free[buf]);
        }
        if (pos < sh.len) out[pos] = ok ? fmaf(keep, old, pg >= 0 && pg < a.c.num_pages ? sum0 + sum1 : 0.f) : NAN;
      }
      return true;
    });
  } else if (warp < kMmaWarp) {
    // ---- copies -----------------------------------------------------------------
    const int w = warp - 8;
    constexpr int CH = kTileChunks / kCopyWarps;  // chunks of a tile that the warp copies
    constexpr int kPieces = D * 2 / 16;   // 16-byte pieces a row
    constexpr int kAtOnce = 32 / kPieces;  // rows a warp copies at once
    // a barrier's arrival once this thread's copies so far have landed
    auto landed = [](uint64_t *b) {
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(b)) : "memory");
    };
    auto of = [](const char *x, int h) { return (const char *)__shfl_sync(~0u, (unsigned long long)x, h); };
    const int piece16 = lane % kPieces, r0_lane = lane / kPieces;
    uint32_t to_off[kChunk / kAtOnce];  // where the lane's pieces of a chunk go
#pragma unroll
    for (int j = 0; j < kChunk / kAtOnce; j++) {
      const int row = j * kAtOnce + r0_lane;
      to_off[j] = (piece16 >> 3) * 16384 + row * 128 + ((piece16 & 7) ^ (row & 7)) * 16;
    }
    uint32_t tile = 0, piece = 0;
    pieces([&](int b, const MassShare &sh, int head, int t0, int t1, int r0, int rows) {
      if (rows <= 0) return true;
      bool ok = true;
      const int chunks = (sh.len + kChunk - 1) / kChunk, n = t1 - t0;
      int pages = -1;  // lane i: the page of the warp's i-th chunk from the last look on
      for (int i = 0; i < n && ok; i++, tile++) {
        const uint32_t stage = tile % NS, use = tile / NS;
        if (i % (32 / CH) == 0) {
          const int c = (t0 + i + lane / CH) * kTileChunks + CH * w + lane % CH;
          pages = c < chunks ? a.c.table[b * a.c.table_stride + ((c * kChunk) >> a.c.page_shift)] : -1;
        }
        // lane h < CH: where the warp's chunk h lies
        const int pos = ((t0 + i) * kTileChunks + CH * w + lane % CH) * kChunk;
        const int pg = __shfl_sync(~0u, pages, i % (32 / CH) * CH + lane % CH);
        const bool mapped = pg >= 0 && pg < a.c.num_pages;
        const int valid = mapped ? max(0, min(kChunk, sh.len - pos)) : 0;
        const char *src = a.c.k + head * a.c.head_bytes +
                          (valid ? pg * a.c.page_bytes + (long long)(pos & ((1 << a.c.page_shift) - 1)) * a.c.token_bytes : 0);
        ok = __all_sync(~0u, use == 0 || bar_wait(&k_empty[stage], (use - 1) & 1, dead));
        if (!ok) break;
        const uint32_t base = smem_addr(k_sm) + stage * S::kBlock + CH * w * kChunk * 128;
#pragma unroll 1
        for (int h = 0; h < CH; h++) {
          const int n_h = __shfl_sync(~0u, valid, h);
          const char *at = of(src, h), *from = at + piece16 * 16 + r0_lane * (long long)a.c.token_bytes;
#pragma unroll
          for (int j = 0; j < kChunk / kAtOnce; j++) {
            const bool in = j * kAtOnce + r0_lane < n_h;
            copy16(base + h * kChunk * 128 + to_off[j], in ? from + j * kAtOnce * (long long)a.c.token_bytes : at, in);
          }
        }
        landed(&k_full[stage]);
        if (i == 0) {  // the rows, once the piece before has no more use for its own
          ok = __all_sync(~0u, piece == 0 || bar_wait(q_empty, (piece - 1) & 1, dead));
          if (!ok) break;
          const unsigned long long on = a.counted ? (unsigned long long)a.counted[b] : ~0ull;
          constexpr int kMine = S::kRows / kCopyWarps;  // the warp's rows; a lane works out every 32nd's address
#pragma unroll 1
          for (int x0 = 0; x0 < kMine; x0 += 32) {
            if (w * kMine + x0 >= rows) break;  // whole groups of 32
            const int mine = w * kMine + x0 + lane, q = r0 + mine;
            const char *at = nullptr;
            if (mine < rows && on >> (q / a.group) & 1)
              at = (const char *)((const T *)a.q + (sh.first + q / a.group) * a.q_stride + (long long)(head * a.group + q % a.group) * D);
#pragma unroll 8
            for (int x = 0; x < 32; x += kAtOnce) {
              const char *from = of(at, x + r0_lane);
              const int row = w * kMine + x0 + x + r0_lane;
              copy16(smem_addr(q_sm) + (row >> 7) * S::kBlock + (piece16 >> 3) * 16384 + (row & 127) * 128 + ((piece16 & 7) ^ (row & 7)) * 16,
                     from ? from + piece16 * 16 : (const char *)a.q, from != nullptr);
            }
          }
          landed(q_full);
        }
      }
      if (n > 0) piece++;
      return ok;
    });
    copy_commit();
    copy_wait<0>();
  } else {
    // ---- products: the whole warp takes every step; one lane issues ------------------
    auto wait_copies = [&](uint64_t *b, uint32_t parity) {
      const bool there = bar_wait(b, parity, dead);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the copies were plain stores
      return there;
    };
    const uint64_t q_desc = mma_desc(smem_addr(q_sm), 16), k_desc = mma_desc(smem_addr(k_sm), 16);
    uint32_t items[2] = {0, 0}, tile = 0, piece = 0;
    pieces([&](int b, const MassShare &sh, int head, int t0, int t1, int r0, int rows) {
      if (rows <= 0 || t1 <= t0) return true;
      bool ok = __all_sync(~0u, wait_copies(q_full, piece & 1));
      for (int i = 0; i < t1 - t0 && ok; i++, tile++) {
        const int s = i & 1;
        const uint32_t stage = tile % NS;
        ok = __all_sync(~0u, wait_copies(&k_full[stage], tile / NS & 1));
        for (int rb = 0; rb * 128 < rows && ok; rb++) {
          const uint32_t item = s ? items[1]++ : items[0]++, buf = s * 2 + (item & 1);
          ok = __all_sync(~0u, item < 2 || bar_wait(&s_free[buf], (item / 2 - 1) & 1, dead));
          if (!ok) break;
          tc_after();
          const bool last = (rb + 1) * 128 >= rows;
          const uint32_t idesc = mma_idesc<T>(columns(rows, rb), false);
          const uint64_t k = k_desc + stage * (S::kBlock / 16), q = q_desc + rb * (S::kBlock / 16);
          if (elected()) {
#pragma unroll
            for (int h = 0; h < S::kHalves; h++)
#pragma unroll
              for (int j = 0; j < 4; j++)
                mma_ss(tmem + buf * 128, k + (h * 16384 + j * 32) / 16, q + (h * 16384 + j * 32) / 16, idesc, h + j > 0);
            tc_commit(&s_full[buf]);
            if (last) tc_commit(&k_empty[stage]);
            if (last && i == t1 - t0 - 1) tc_commit(q_empty);
          }
          __syncwarp();
        }
      }
      piece++;
      return ok;
    });
  }
  mass_rest(a, kMmaThreads);
  __syncwarp();
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace paged
}  // namespace ocrvl
