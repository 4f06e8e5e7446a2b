// The attention weight that cached positions got from a set of tokens
// (ocrvl_op_attn_mass):
//   acc'[t] = decay acc[t] + sum over rows of 2^(scale log2(e) q . k_t - lse log2(e))
// with the rows' lse known, so one pass over K does: no maximum, no second
// pass.  Every position belongs to one warp, which adds its rows' weights in
// a fixed order: no atomics, the same sums every time.
//
// A block takes a run of tiles of 128 positions (16 a warp) of one
// (sequence, kv head) after another.  The fragments of 8 query rows stay in
// registers; those of more (f32 only: 16-bit types have mass_mma.cuh then) in shared
// memory, as many as fit, so more yet take several passes over the block's K.  Where
// a run has at most four chunks, two or four warps share one and its rows.  Calls
// of few tiles and many rows have a cluster of blocks a run, each with a part
// of the rows; the parts' sums are added in order over distributed shared memory.
//
// f32, 64 sequences of up to 4,096 positions, one token: 40.2 us, 3.7 TB/s, bound by a warp's
// work on a chunk (its split into pairs of tf32 and the three products).  131,072 positions, 64 drafts
// of 8 heads: 580 us, 59 TFLOP/s or 178 of products, of 276 that the instruction gives.
#pragma once
#include <cooperative_groups.h>

#include "paged.cuh"

namespace ocrvl {
namespace paged {

namespace cg = cooperative_groups;

constexpr int kMassWarps = 8;
constexpr int kMassThreads = kMassWarps * 32;

struct MassArgs {
  Cache c;
  Seqs s;
  int kv_heads, group;
  const void *q;
  long long q_stride;
  const long long *counted;
  const float *lse;
  float scale, decay;  // scale * log2(e)
  const float *acc;
  float *out;
  long long acc_stride, out_stride;
  int acc_width, out_width;
};

// A sequence's tiles and what one costs: K's load (about what `load` tiles of
// 8 rows take) and the rows' products.
struct MassShare {
  int first, count, len, tiles, cost;

  __device__ MassShare(const MassArgs &a, int b, int load) {
    count = a.s.tokens(b, &first);
    len = min(a.s.len(b), a.out_width);
    tiles = (len + kMassWarps * kChunk - 1) / (kMassWarps * kChunk);
    cost = load + (count * a.group + 7) / 8;
  }
  __device__ long long total(int kv_heads) const { return (long long)kv_heads * tiles * cost; }
  // The tiles [t0, t1) of a segment whose cost starts in [lo, hi); at: the cost below
  // it, then below the next one.
  __device__ bool tiles_in(long long lo, long long hi, long long &at, int *t0, int *t1) const {
    const long long from = max(lo - at, 0ll), to = hi - at;
    *t0 = (int)min((long long)tiles, (from + cost - 1) / cost);
    *t1 = to <= 0 ? 0 : (int)min((long long)tiles, (to + cost - 1) / cost);
    at += (long long)tiles * cost;
    return *t0 < *t1;
  }
};

// Where a run's share of the cost starts: plan[0] all of it, [1] the sequence, [2] the cost below it.
__device__ __forceinline__ void mass_start(const MassArgs &a, int load, int run, int runs, long long *plan, int lane) {
  long long all = 0;
  for (int b = lane; b < a.s.batch; b += 32) all += MassShare(a, b, load).total(a.kv_heads);
  for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(~0u, all, d);
  const long long lo = all * run / runs;
  if (lane == 0) plan[0] = all, plan[1] = a.s.batch, plan[2] = all;
  __syncwarp();
  long long below = 0;
  for (int b0 = 0; b0 < a.s.batch; b0 += 32) {
    const long long mine = b0 + lane < a.s.batch ? MassShare(a, b0 + lane, load).total(a.kv_heads) : 0;
    long long upto = mine;
    for (int d = 1; d < 32; d <<= 1) {
      const long long x = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += x;
    }
    const unsigned hit = __ballot_sync(~0u, below + upto > lo);
    if (hit) {
      if (lane == __ffs(hit) - 1) plan[1] = b0 + lane, plan[2] = below + upto - mine;
      break;
    }
    below += __shfl_sync(~0u, upto, 31);
  }
}

// f(share, sequence, head, t0, t1) for the tiles [t0, t1) of every segment whose cost starts in
// the run's share.
template <typename F>
__device__ __forceinline__ void mass_segments(const MassArgs &a, int load, int run, int runs, const long long *plan, F f) {
  const long long lo = plan[0] * run / runs, hi = plan[0] * (run + 1) / runs;
  long long at = plan[2];  // cost below the current segment
  for (int b = (int)plan[1]; b < a.s.batch && at < hi; b++) {
    const MassShare sh(a, b, load);
    for (int head = 0; head < a.kv_heads; head++) {
      int t0, t1;
      if (sh.tiles_in(lo, hi, at, &t0, &t1)) f(sh, b, head, t0, t1);
    }
  }
}

// 0 past the lengths: each row by the blocks that share its remainder
__device__ __forceinline__ void mass_rest(const MassArgs &a, int threads) {
  const int all_rows = a.s.batch * a.kv_heads, share = max(1, (int)gridDim.x / all_rows);
  for (int i = blockIdx.x; i < all_rows * share; i += gridDim.x) {
    const int r = i % all_rows, p = i / all_rows, len = min(a.s.len(r / a.kv_heads), a.out_width);
    for (int x = len + p * threads + threadIdx.x; x < a.out_width; x += share * threads) a.out[r * a.out_stride + x] = 0.f;
  }
}

template <typename T, int D, bool THIN>
struct MassShape {
  using L = Tile<T, D>;
  static constexpr int kUnits = L::kBytes >= 8192 ? (THIN ? 3 : 2) : L::kBytes >= 4096 ? 4 : 6;  // 16 positions each
  static constexpr int kRing = kMassWarps * kUnits * L::kBytes;
  static constexpr int kItems = 4;  // a thread's 16 bytes of half the rows in shared memory
  static constexpr int kHalf = THIN ? 1 : kItems * kMassThreads / L::kQItems;  // tiles of 8 rows
  static constexpr int kRowTiles = THIN ? 1 : 2 * kHalf;
  static constexpr int kLoad = L::f32 ? 4 : 12;
  static constexpr int kSmem = kRing + kRowTiles * (L::kQBytes + 8 * 4) + 64 + 2 * kMassWarps * kChunk * 4;
};

template <typename T, int D, bool THIN>
__global__ void __launch_bounds__(kMassThreads, 1) k_attn_mass(const MassArgs a, int blocks) {
  const int parts = THIN ? 1 : blocks;  // of the rows, a block each
  using S = MassShape<T, D, THIN>;
  using L = Tile<T, D>;
  constexpr int NU = S::kUnits;
  extern __shared__ __align__(128) char sm[];
  char *ring = sm, *q_sm = sm + S::kRing;
  float *shift = (float *)(q_sm + S::kRowTiles * L::kQBytes);  // lse log2(e), +inf for rows that do not count
  long long *plan = (long long *)(shift + S::kRowTiles * 8);
  float *joint = (float *)(plan + 8);  // [round & 1][warp][position]: sums of warps and blocks that share chunks
  const int runs = gridDim.x / parts, run = blockIdx.x / parts, rank = blockIdx.x % parts;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane & 3;

  if (warp == 0) mass_start(a, S::kLoad, run, runs, plan, lane);
  __syncthreads();

  const uint32_t my_ring = smem_addr(ring) + warp * NU * L::kBytes, q_at = smem_addr(q_sm);
  int flip = 0;
  const long long lo = plan[0] * run / runs, hi = plan[0] * (run + 1) / runs;
  long long at = plan[2];  // cost below the current segment
  for (int b = (int)plan[1]; b < a.s.batch && at < hi; b++) {
    const MassShare sh(a, b, S::kLoad);
    for (int head = 0; head < a.kv_heads; head++) {
      int t0, t1;
      if (!sh.tiles_in(lo, hi, at, &t0, &t1)) continue;
      // this block's rows: all, or a part of their tiles of eight
      const int all_tiles = (sh.count * a.group + 7) / 8, r0 = all_tiles * rank / parts * 8;
      const int rows = min(sh.count * a.group, all_tiles * (rank + 1) / parts * 8) - r0, row_tiles = (rows + 7) / 8;
      const int most = (all_tiles + parts - 1) / parts;  // of any block
      const int passes = THIN ? 1 : max(1, (most + S::kRowTiles - 1) / S::kRowTiles);
      const int chunks = (sh.len + kChunk - 1) / kChunk, c_end = min(t1 * kMassWarps, chunks);
      const int live = c_end - t0 * kMassWarps, rounds = (live + kMassWarps - 1) / kMassWarps;
      const int share = THIN || live > 4 ? 1 : live > 2 ? 2 : 4, part = warp % share;  // warps a chunk
      const int c0 = t0 * kMassWarps + warp / share;
      const int nk = c0 < c_end ? (share > 1 ? 1 : (c_end - c0 + kMassWarps - 1) / kMassWarps) : 0;
      const float *acc = a.acc ? a.acc + ((long long)b * a.kv_heads + head) * a.acc_stride : nullptr;
      float *out = a.out + ((long long)b * a.kv_heads + head) * a.out_stride;

      // the warp's chunks, all of them once a pass; the next ones' loads run across passes
      int pages = -1, ahead_k = 0, ahead_pass = 0;
      unsigned long long valids = 0;  // 8 bits a unit in flight
      auto issue = [&](int i) {  // the i-th one, in the ring's unit i % NU
        const int k = THIN ? i : ahead_k, unit = i % NU;
        if (THIN ? i < nk : ahead_pass < passes && nk > 0) {
          const int c = c0 + k * kMassWarps, pos = c * kChunk;
          if ((k & 31) == 0) {
            const int mine = c + lane * kMassWarps;
            pages = mine < chunks ? a.c.table[b * a.c.table_stride + ((mine * kChunk) >> a.c.page_shift)] : -1;
          }
          const int pg = __shfl_sync(~0u, pages, k & 31);
          const bool mapped = pg >= 0 && pg < a.c.num_pages;
          const int valid = mapped ? min(kChunk, sh.len - pos) : 0;
          valids |= (unsigned long long)valid << (8 * unit);
          L::template load<false>(my_ring + unit * L::kBytes,
                                  a.c.k + (mapped ? pg : 0) * a.c.page_bytes + head * a.c.head_bytes +
                                      (long long)(pos & ((1 << a.c.page_shift) - 1)) * a.c.token_bytes,
                                  a.c.token_bytes, valid, lane);
          if (!THIN && ++ahead_k == nk) ahead_k = 0, ahead_pass++;
        }
        copy_commit();
      };
      __syncthreads();  // the last segment is done with the query rows
#pragma unroll
      for (int i = 0; i < NU - 1; i++) issue(i);
      const unsigned long long on = a.counted ? (unsigned long long)a.counted[b] : ~0ull;
      auto counts = [&](int r) { return r < rows && (on >> ((r0 + r) / a.group) & 1); };
      auto query = [&](int r) -> const T * {
        const int x = r0 + r;
        return counts(r) ? (const T *)a.q + (sh.first + x / a.group) * a.q_stride + (long long)(head * a.group + x % a.group) * D : nullptr;
      };
      auto shift_of = [&](int r) {
        if (!counts(r)) return INFINITY;
        const int x = r0 + r;
        const float l = a.lse[(long long)(sh.first + x / a.group) * a.kv_heads * a.group + head * a.group + x % a.group] * kLog2e;
        return l == -INFINITY ? INFINITY : l;  // attended nothing
      };
      // whole pairs of tiles: rows past the last do not count
      auto tiles_of = [&](int pass) { return max(0, min(S::kRowTiles, (row_tiles - pass * S::kRowTiles + 1) / 2 * 2)); };
      if (!THIN || row_tiles) {
        const int tiles = THIN ? 1 : tiles_of(0);
        L::query(q_at, tiles, tid, kMassThreads, query);
        for (int r = tid; r < tiles * 8; r += kMassThreads) shift[r] = shift_of(r);
      }
      __syncthreads();

      uint32_t qr[THIN ? L::kTiles : 1][L::kQRegs];
      float l0 = INFINITY, l1 = INFINITY;
      if constexpr (THIN) {
        if (row_tiles) {
#pragma unroll
          for (int blk = 0; blk < L::kTiles; blk++) L::q_load(qr[blk], q_at, blk, lane);
          l0 = shift[2 * t], l1 = shift[2 * t + 1];
        }
      }
      float w[2] = {};  // of positions g and g + 8
      auto add = [&](const float(&s)[4], const float(&c)[2][4]) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = L::f32 ? s[e] + (c[0][e] + c[1][e]) : s[e];
        // a row that does not count adds nothing, whatever its query and the key hold
        auto weight = [&](float x, float l) { return l == INFINITY ? 0.f : exp2_(fmaf(x, a.scale, -l)); };
        w[0] += weight(y[0], l0) + weight(y[1], l1);
        w[1] += weight(y[2], l0) + weight(y[3], l1);
      };
      // a chunk's K with the tiles of rows from m on (the warp's share of them, two at once: a
      // chain of products of its own takes 11.5 ns a link)
      constexpr int AT = 2;
      auto weigh = [&](const typename L::KFrag(&f)[THIN ? 1 : L::kTiles], int m, int tiles) {
        if constexpr (!THIN) {
          for (m += part * AT; m < tiles; m += share * AT) {
            float s[AT][4] = {}, c[AT][2][4] = {};
#pragma unroll
            for (int blk = 0; blk < L::kTiles; blk++)
#pragma unroll
              for (int i = 0; i < AT; i++) {
                uint32_t x[L::kQRegs];
                L::q_load(x, q_at + (m + i) * L::kQBytes, blk, lane);
                L::k_product(s[i], c[i], x, f[blk]);
              }
#pragma unroll
            for (int i = 0; i < AT; i++) {
              l0 = shift[(m + i) * 8 + 2 * t], l1 = shift[(m + i) * 8 + 2 * t + 1];
              add(s[i], c[i]);
            }
          }
        }
      };
      int item = 0;  // chunks so far, over all passes
      for (int pass = 0; pass < passes; pass++) {
        const float keep = pass ? 1.f : a.decay;  // further passes add to what the first wrote
        auto sum_at = [&](int pos) {
          if (lane >= kChunk || pos >= sh.len) return 0.f;
          return pass ? out[pos] : acc && pos < a.acc_width ? acc[pos] : 0.f;
        };
        const bool alone = THIN || share * parts == 1;  // no other warp's sums go into this one's
        float ahead = alone && nk ? sum_at(c0 * kChunk + lane) : 0.f;
        for (int k = 0; k < (THIN ? nk : rounds); k++) {
          int valid = 0;
          w[0] = w[1] = 0.f;
          typename L::KFrag f[THIN ? 1 : L::kTiles];
          const uint32_t k_at = my_ring + item % NU * L::kBytes;
          const int pos = (c0 + k * kMassWarps) * kChunk + lane;
          float old = 0.f;
          if (THIN || k < nk) {
            copy_wait<NU - 2>();
            __syncwarp();
            valid = (int)(valids >> (8 * (item % NU))) & 31;
            valids &= ~(0xffull << (8 * (item % NU)));
            // lane j < 16 has position j; what the next chunk's sums were is on its way while
            // this one's products run
            old = ahead;
            ahead = alone && k + 1 < nk ? sum_at(pos + kMassWarps * kChunk) : 0.f;
            issue(item + NU - 1);
            item++;
            if constexpr (!THIN) {
#pragma unroll
              for (int blk = 0; blk < L::kTiles; blk++) L::k_load(f[blk], blk, k_at, lane);
            }
          }
          if constexpr (THIN) {
            if (row_tiles) {
              float s[4] = {}, c[2][4] = {};
#pragma unroll
              for (int blk = 0; blk < L::kTiles; blk++) {
                L::k_load(f[0], blk, k_at, lane);
                L::k_product(s, c, qr[blk], f[0]);
              }
              add(s, c);
            }
          } else if (k + 1 < rounds || pass + 1 == passes) {
            if (k < nk) weigh(f, 0, tiles_of(pass));
          } else {
            // the next pass's rows, a half at a time: fetched into registers before this pass's last
            // products with the half that they replace, put into place behind them
            const int tiles = tiles_of(pass);
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const int at = (pass + 1) * S::kRowTiles + h * S::kHalf;
              uint4 x[S::kItems];
              float l_next = INFINITY;
#pragma unroll
              for (int i = 0; i < S::kItems; i++) x[i] = L::q_fetch(at * L::kQItems + i * kMassThreads + tid, query);
              if (tid < S::kHalf * 8) l_next = shift_of(at * 8 + tid);
              if (k < nk) weigh(f, h * S::kHalf, min(tiles, (h + 1) * S::kHalf));
              __syncthreads();
#pragma unroll
              for (int i = 0; i < S::kItems; i++) L::q_put(q_at + h * S::kHalf * L::kQBytes, i * kMassThreads + tid, x[i]);
              if (tid < S::kHalf * 8) shift[h * S::kHalf * 8 + tid] = l_next;
            }
            __syncthreads();
          }
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) w[n] += __shfl_xor_sync(~0u, w[n], d);
          // lane j takes position j's sum from the lane that holds it
          const int j = lane & 15;
          const float w0 = __shfl_sync(~0u, w[0], (j & 7) * 4), w1 = __shfl_sync(~0u, w[1], (j & 7) * 4);
          float mine = j & 8 ? w1 : w0;
          if (j >= valid) mine = 0.f;
          if (alone) {
            if ((THIN || k < nk) && lane < kChunk && pos < sh.len) out[pos] = fmaf(keep, old, mine);
          } else {
            // thread i < 128 / share takes position i of the round, in the block that the
            // chunk falls to; a buffer is written again two rounds on, behind the next barrier
            float *buf = joint + flip * kMassWarps * kChunk;
            flip ^= 1;
            if (lane < kChunk) buf[warp * kChunk + lane] = mine;
            const int i = tid / kChunk, p = (t0 + k) * kMassWarps * kChunk + tid;
            const bool takes = i < kMassWarps / share && i % parts == rank && p < min(c_end * kChunk, sh.len);
            float sum = 0.f;
            if (takes) old = pass ? out[p] : acc && p < a.acc_width ? acc[p] : 0.f;
            if (parts > 1)
              cg::this_cluster().sync();
            else
              __syncthreads();
            if (takes) {
              for (int r = 0; r < parts; r++) {
                const float *from = parts > 1 ? cg::this_cluster().map_shared_rank(buf, r) : buf;
                for (int n = 0; n < share; n++) sum += from[(i * share + n) * kChunk + tid % kChunk];
              }
              out[p] = fmaf(keep, old, sum);
            }
          }
        }
      }
      copy_wait<0>();
    }
  }
  if (parts > 1) cg::this_cluster().sync();  // no block ends while another reads its sums
  mass_rest(a, kMassThreads);
}

}  // namespace paged
}  // namespace ocrvl
