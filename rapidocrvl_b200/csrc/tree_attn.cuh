// Attention of drafted tokens over a paged cache and over one another
// (ocrvl_op_tree_attn).
//
// For one kv head the rows are the sequence's drafted tokens times the query
// heads that share it.  A block takes 8 NT rows against a run of positions; its
// eight warps stream 16-position chunks of K and V of their own through private
// rings of shared memory (no block barrier on the way), each with a reference m,
// the sum l and the weighted values o of its own positions:
//   p = 2^(s - m),  l' = l + sum p,  o' = o + p v      (s = scale log2(e) q . k)
// m follows the running maximum, but only once a score passes it by kSlack:
//   m' = max(m, max s),  l and o times 2^(m - m')      (f16: max s - kLift)
// so most chunks need no maximum over lanes and no rescaling, and p stays below
// 2^kSlack; a value within that factor of the type's largest (f32 and bf16) may
// overflow its sum.  At the run's end the warps are joined: o = sum_w 2^(m_w - M) o_w,
// l likewise.
//
// A (sequence, kv head, row block) is a segment.  Two ways to share them out:
//   CS = 0  tiles of 128 positions over a persistent grid in equal runs,
//           whatever the lengths are: a run may cover several segments and a
//           segment several runs.  A segment within one run is written at
//           once, else its parts go to the workspace and k_tree_combine joins
//           them.  The first chunks of a run's next segment are fetched
//           before the warps join, so the memory does not idle.
//   CS > 0  a cluster of CS blocks a segment, joined over distributed shared
//           memory: one launch, no workspace, no search for the run's start.
//           For calls whose segments and lengths are few.
//
// 64 sequences of up to 4,096 positions, one token, f32: 60.3 us, 4.8 TB/s of K
// and V, bound by a warp's work on a chunk (the split into pairs of tf32 and three
// products of each, 1.2 us), bf16 39.0; 648 positions of one sequence: 9 us, bound by a
// launch and two loads behind one another; 8 sequences of up to 4,095 with 12 drafts: 41.4 us,
// 16 of 3,000 with 64 549, bound by the products of blocks of 32 rows, each of which reads
// and splits K and V again.
#pragma once
#include <cooperative_groups.h>

#include "paged.cuh"

namespace ocrvl {
namespace paged {

constexpr int kTreeWarps = 8;
constexpr int kTreeThreads = kTreeWarps * 32;
constexpr int kTileChunks = kTreeWarps;  // chunks a tile: one a warp
// A new reference stands kLift below its largest score, and stays while no score passes it by
// kSlack.  f16's weights below 2^-24 lose their last bits and those below 2^-25 are 0, which over
// 100,000 positions under one strong one adds up, so they start as 2^7 and may grow to 2^15, half
// of f16's largest: what is lost is below 2^-32 of the largest weight.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;
template <typename T>
constexpr float kSlack = std::is_same<T, __half>::value ? 15.f : 8.f;

struct TreeArgs {
  Cache c;
  Seqs s;
  int kv_heads, group;  // group: query heads a kv head
  const void *q, *dk, *dv;
  void *out;
  long long q_stride, kv_stride, out_stride;  // elements
  const long long *mask;
  float scale;    // scale * log2(e)
  float *lse;
  float *part;    // [2 grid][rows][D]
  float *part_ml; // [2 grid][rows][2]
  int4 *joint;    // [sequence][kv head][row block] of runs: the first part's slot (-1: the segment is whole), its run, the last run
  int start_cost; // of a segment's start (filling the rings, joining the warps), in tiles, in the split of runs
};

struct Segments {  // what a sequence's segments have in common
  int first, count, len, chunks_c, chunks, tiles, blocks, start;

  __device__ Segments() {}
  __device__ Segments(const TreeArgs &a, int b, int rows) {
    count = a.s.tokens(b, &first);
    len = a.s.len(b);
    chunks_c = (len + kChunk - 1) / kChunk;
    chunks = chunks_c + (count + kChunk - 1) / kChunk;
    tiles = (chunks + kTileChunks - 1) / kTileChunks;
    blocks = (count * a.group + rows - 1) / rows;
    start = a.start_cost;
  }
  __device__ int cost() const { return start + tiles; }
  // Its tiles that start below cost x, if the segment starts at `at`: behind its own cost.
  __device__ int tiles_below(long long x, long long at) const { return (int)max(0ll, min(x - at - start, (long long)tiles)); }
  __device__ long long total(int kv_heads) const { return (long long)kv_heads * blocks * cost(); }
};

// Cost of the sequences below b, and of all, by one warp.
__device__ __forceinline__ void count_cost(const TreeArgs &a, int rows, int b, int lane, long long *below, long long *all) {
  long long lo = 0, sum = 0;
  for (int i = lane; i < a.s.batch; i += 32) {
    const long long n = Segments(a, i, rows).total(a.kv_heads);
    sum += n;
    if (i < b) lo += n;
  }
  for (int d = 16; d; d >>= 1) {
    sum += __shfl_xor_sync(~0u, sum, d);
    lo += __shfl_xor_sync(~0u, lo, d);
  }
  *below = lo;
  *all = sum;
}

// Run c of n covers the costs from start(c) to start(c + 1) and takes the tiles
// that start there.
struct Runs {
  long long all, each;
  int n, rest;  // the first `rest` runs are one longer than `each`

  static __device__ long long over(long long x, long long d) {  // 32-bit division where that is enough
    return (x | d) >> 32 ? x / d : (long long)((unsigned)x / (unsigned)d);
  }
  __device__ Runs(long long all_, int grid) : all(all_) {
    n = (int)min((long long)grid, all);
    each = n ? over(all, n) : 0, rest = n ? (int)(all - each * n) : 0;
  }
  __device__ long long start(int c) const { return c * each + min(c, rest); }
  __device__ int of(long long x) const {  // the run that covers cost x
    const long long longer = rest * (each + 1);
    return x < longer ? (int)over(x, each + 1) : rest + (int)over(x - longer, each);
  }
};
// A part of a segment's positions: tiles t0 .. t1 - 1.
struct Piece {
  Segments sg;
  int b, head, rb, t0, t1;
};

// The runs of CS = 0: finds where this block's starts (one warp searches; plan: three
// words of shared memory), then steps through its pieces.
struct Walk {
  long long at, hi;  // cost at which the current segment starts; the run's end
  long long all;

  // False where the run is empty.  Called by the whole block.
  __device__ __forceinline__ bool start(const TreeArgs &a, int rows, long long *plan, int warp, int lane, Piece &x) {
    if (warp == 0) {
      long long below, all;
      count_cost(a, rows, 0, lane, &below, &all);
      const Runs runs(all, gridDim.x);
      if (lane == 0) plan[0] = all, plan[1] = a.s.batch;
      __syncwarp();
      if (blockIdx.x < runs.n) {
        const long long lo = runs.start(blockIdx.x);
        long long sum = 0;
        for (int b0 = 0; b0 < a.s.batch; b0 += 32) {
          const int b = b0 + lane;
          const long long mine = b < a.s.batch ? Segments(a, b, rows).total(a.kv_heads) : 0;
          long long upto = mine;
          for (int d = 1; d < 32; d <<= 1) {
            const long long y = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += y;
          }
          const unsigned hit = __ballot_sync(~0u, sum + upto > lo);
          if (hit) {
            if (lane == __ffs(hit) - 1) plan[1] = b, plan[2] = sum + upto - mine;
            break;
          }
          sum += __shfl_sync(~0u, upto, 31);
        }
      }
    }
    __syncthreads();
    all = plan[0];
    const Runs runs(all, gridDim.x);
    x.b = (int)plan[1];
    if ((int)blockIdx.x >= runs.n || x.b >= a.s.batch) return false;
    const long long lo = runs.start(blockIdx.x);
    hi = runs.start(blockIdx.x + 1);
    x.sg = Segments(a, x.b, rows);
    const int i = (int)Runs::over(lo - plan[2], x.sg.cost());
    at = plan[2] + (long long)i * x.sg.cost();
    x.head = i / x.sg.blocks, x.rb = i % x.sg.blocks;
    x.t0 = x.sg.tiles_below(lo, at);
    x.t1 = x.sg.tiles_below(hi, at);
    return x.t0 < x.t1 || next(a, rows, x);
  }
  // Says where the parts of a segment are, if its first one is this piece; by one thread,
  // while the walk is at the piece.
  __device__ __forceinline__ void tell(const TreeArgs &a, const Piece &x, int row_blocks, int slot) const {
    if (x.t0) return;
    const bool whole = x.t1 == x.sg.tiles;
    const int last = whole ? 0 : Runs(all, gridDim.x).of(at + x.sg.start + x.sg.tiles - 1);
    a.joint[((long long)x.b * a.kv_heads + x.head) * row_blocks + x.rb] = make_int4(whole ? -1 : slot, blockIdx.x, last, 0);
  }
  // The run's next piece that has tiles.
  __device__ __forceinline__ bool next(const TreeArgs &a, int rows, Piece &x) {
    while (true) {
      at += x.sg.cost();
      if (at >= hi) return false;
      if (++x.rb == x.sg.blocks) {
        x.rb = 0;
        if (++x.head == a.kv_heads) {
          x.head = 0;
          do {
            if (++x.b >= a.s.batch) return false;
            x.sg = Segments(a, x.b, rows);
          } while (x.sg.blocks == 0);
        }
      }
      x.t0 = 0;
      x.t1 = x.sg.tiles_below(hi, at);
      if (x.t1 > 0) return true;
    }
  }
};

// Sets non-finite values to 0: in the matrix product 0 * NaN would reach rows
// that do not see the draft they belong to.  The rows that see it get them
// added apart.
template <typename T, int D>
__device__ __noinline__ void drop_nonfinite(uint32_t v, int lane) {
  using L = Tile<T, D>;
  for (int i = lane; i < kChunk * L::kPieces; i += 32) {
    const uint32_t at = v + i * 16;
    uint32_t x[4];
    lds4u(x, at);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (sizeof(T) == 4) {
        if ((x[j] & 0x7f800000u) == 0x7f800000u) x[j] = 0u;
      } else {
        constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
        if ((x[j] & e) == e) x[j] &= 0xffff0000u;
        if ((x[j] >> 16 & e) == e) x[j] &= 0xffffu;
      }
    }
    sts4u(at, x[0], x[1], x[2], x[3]);
  }
  __syncwarp();
}

template <typename T, int D>
__device__ __forceinline__ bool any_nonfinite(uint32_t v, int lane) {
  using L = Tile<T, D>;
  bool bad = false;
  for (int i = lane; i < kChunk * L::kPieces; i += 32) {
    uint32_t x[4];
    lds4u(x, v + i * 16);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (sizeof(T) == 4) {
        bad |= (x[j] & 0x7f800000u) == 0x7f800000u;
      } else {
        constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
        bad |= (x[j] & e) == e || (x[j] >> 16 & e) == e;
      }
    }
  }
  return __any_sync(~0u, bad);
}

template <typename T, int D, int NT>
struct TreeShape {
  using L = Tile<T, D>;
  static constexpr int kRows = 8 * NT;
  // 16-bit types at up to 16 rows: two blocks an SM; else one
  static constexpr int kBlocks = sizeof(T) == 2 && NT <= 2 ? 2 : 1;
  // chunks of K or V in a warp's ring: about 192 KB an SM
  static constexpr int kUnits = L::kBytes * kBlocks >= 8192 ? 3 : 6;
  static constexpr int kSlot = kTreeWarps * L::kBytes;  // one unit of every warp
  // the join of 8 or 16 rows of eight warps in f32 lies over the last slots, so
  // the others can be filled meanwhile
  static constexpr int kJoinRows = NT == 1 ? 8 : 16;
  static constexpr int kJoinSlots = (kTreeWarps * kJoinRows * D * 4 + kSlot - 1) / kSlot;
  static constexpr int kEarly = kUnits - kJoinSlots < kUnits - 1 ? kUnits - kJoinSlots : kUnits - 1;
  static constexpr int kQ = NT * L::kQBytes;
  static constexpr bool kQInRegs = NT == 1;
  static constexpr int kSmem = kQ + kUnits * kSlot + kTreeWarps * kRows * 8 + kRows * 8 + 64 + kTreeWarps * 8 * 4 + kRows * 8;
  static_assert(kEarly >= 1, "");
};

// A warp's part of a piece.
struct WarpPiece : Piece {
  int c0, step, nk;  // chunks c0, c0 + step, ...: nk of them
  __device__ void chunks_of(int warp, int stride) {
    c0 = t0 * kTileChunks + warp, step = stride;
    const int end = min(t1 * kTileChunks, sg.chunks);
    nk = c0 < end ? (end - c0 + step - 1) / step : 0;
  }
};

template <typename T, int D>
__device__ __forceinline__ void write_row(const TreeArgs &a, const Segments &sg, int head, int r, int d, float4 x, float top, float l) {
  const int tok = sg.first + r / a.group, hd = head * a.group + r % a.group;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  store4((T *)a.out + tok * a.out_stride + (long long)hd * D + d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
  if (d == 0 && a.lse) a.lse[(long long)tok * a.kv_heads * a.group + hd] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
}

template <typename T, int D, int NT, int CS>
__global__ void __launch_bounds__(kTreeThreads, (TreeShape<T, D, NT>::kBlocks)) k_tree_attn(const TreeArgs a, int row_blocks) {
  using S = TreeShape<T, D, NT>;
  using L = Tile<T, D>;
  constexpr int ROWS = S::kRows, NU = S::kUnits;
  namespace cg = cooperative_groups;
  extern __shared__ __align__(128) char sm[];
  char *q_sm = sm, *ring = sm + S::kQ;
  char *p = ring + NU * S::kSlot;
  float *ml = (float *)p;  // [warp][row][m, l]
  p += kTreeWarps * ROWS * 8;
  unsigned long long *seen = (unsigned long long *)p;  // [row]
  p += ROWS * 8;
  long long *plan = (long long *)p;  // the cost of all; where this block's run starts: a sequence, the cost below it
  p += 64;
  int *there = (int *)p;  // [warp][unit]: positions of the chunk that exist
  p += kTreeWarps * 8 * 4;
  float *part_ml = (float *)p;  // CS > 1: [row][m, l] of this block
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

  WarpPiece cur;
  Walk walk;
  bool more = true;
  if constexpr (CS == 0) {
    const bool any = walk.start(a, ROWS, plan, warp, lane, cur);
    pdl_launch();
    if (!any) return;
    cur.chunks_of(warp, kTileChunks);
  } else {
    const int seg = blockIdx.x / CS;
    cur.rb = seg % row_blocks, cur.head = seg / row_blocks % a.kv_heads, cur.b = seg / row_blocks / a.kv_heads;
    cur.sg = Segments(a, cur.b, ROWS);
    if (cur.rb >= cur.sg.blocks) return;  // the whole cluster alike
    cur.t0 = blockIdx.x % CS, cur.t1 = cur.sg.tiles;
    cur.chunks_of(warp, kTileChunks * CS);
  }

  const uint32_t my_ring = smem_addr(ring) + warp * L::kBytes, q_at = smem_addr(q_sm);
  int *my_there = there + warp * NU;
  int pages = -1;  // lane i: the page of the chunk 32 j + i
  auto issue = [&](const WarpPiece &x, int u) {
    if (u < 2 * x.nk) {
      const int k = u >> 1, c = x.c0 + k * x.step, slot = u % NU;
      const uint32_t to = my_ring + slot * S::kSlot;
      const char *src;
      long long row_bytes;
      int valid;
      if (!(u & 1) && (k & 31) == 0) {
        const int mine = c + lane * x.step;
        const int pg = mine < x.sg.chunks_c ? (mine * kChunk) >> a.c.page_shift : -1;
        pages = pg >= 0 ? a.c.table[x.b * a.c.table_stride + pg] : -1;
      }
      if (c < x.sg.chunks_c) {
        const int pos = c * kChunk, pg = __shfl_sync(~0u, pages, k & 31);
        const bool mapped = pg >= 0 && pg < a.c.num_pages;
        valid = mapped ? min(kChunk, x.sg.len - pos) : 0;
        row_bytes = a.c.token_bytes;
        src = (u & 1 ? a.c.v : a.c.k) + (mapped ? pg : 0) * a.c.page_bytes + x.head * a.c.head_bytes +
              (long long)(pos & ((1 << a.c.page_shift) - 1)) * a.c.token_bytes;
      } else {
        const int j = (c - x.sg.chunks_c) * kChunk;
        valid = min(kChunk, x.sg.count - j);
        row_bytes = a.kv_stride * (long long)sizeof(T);
        src = (const char *)((const T *)(u & 1 ? a.dv : a.dk) + (x.sg.first + j) * a.kv_stride + (long long)x.head * D);
      }
      if (u & 1)
        L::template load<true>(to, src, row_bytes, valid, lane);
      else
        L::template load<false>(to, src, row_bytes, valid, lane);
      if (lane == 0) my_there[slot] = valid;
    }
    copy_commit();
  };
  // the query rows of a piece and the drafts that each sees
  auto load_query = [&](const WarpPiece &x) {
    const int rows = min(ROWS, x.sg.count * a.group - x.rb * ROWS);
    L::query(q_at, NT, tid, kTreeThreads, [&](int row) -> const T * {
      const int i = x.rb * ROWS + row;
      return row < rows ? (const T *)a.q + (x.sg.first + i / a.group) * a.q_stride + (long long)(x.head * a.group + i % a.group) * D
                        : nullptr;
    });
    for (int r = tid; r < ROWS; r += kTreeThreads)
      seen[r] = r < rows ? (unsigned long long)a.mask[x.sg.first + (x.rb * ROWS + r) / a.group] : 0ull;
  };

#pragma unroll
  for (int u = 0; u < S::kEarly; u++) issue(cur, u);
  load_query(cur);
  __syncthreads();

  for (int piece = 0; more; piece++) {
#pragma unroll
    for (int u = S::kEarly; u < NU - 1; u++) issue(cur, u);

    uint32_t qr[S::kQInRegs ? L::kTiles : 1][L::kQRegs];
    if constexpr (S::kQInRegs) {
#pragma unroll
      for (int blk = 0; blk < L::kTiles; blk++) L::q_load(qr[blk], q_at, blk, lane);
    }
    float o[L::kTiles][NT][4] = {}, ref[NT][2], sum[NT][2] = {}, low[NT][2] = {};  // of rows 8 n + 2 t and + 1
#pragma unroll
    for (int n = 0; n < NT; n++) ref[n][0] = ref[n][1] = -INFINITY;

    for (int k = 0; k < cur.nk; k++) {
      const int c = cur.c0 + k * cur.step, u = 2 * k;
      copy_wait<NU - 2>();
      __syncwarp();
      issue(cur, u + NU - 1);
      float s[NT][4];
      L::template scores<NT, S::kQInRegs>(s, qr, q_at, my_ring + (u % NU) * S::kSlot, lane);
      const int valid = my_there[u % NU];
      const bool draft = c >= cur.sg.chunks_c;
      const int j0 = (c - cur.sg.chunks_c) * kChunk;
      // scores in units of log2; -inf where there is nothing to see
      bool above = false;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[n][e] *= a.scale;
      if (draft || valid < kChunk) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int j = g + (e >> 1) * 8;
            if (j >= valid || (draft && !(seen[n * 8 + 2 * t + (e & 1)] >> (j0 + j) & 1))) s[n][e] = -INFINITY;
          }
      }
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
      copy_wait<NU - 2>();
      __syncwarp();
      issue(cur, u + NU);
      const uint32_t v = my_ring + ((u + 1) % NU) * S::kSlot;
      bool bad = false;
      if (draft) {
        bad = any_nonfinite<T, D>(v, lane);
        if (bad) drop_nonfinite<T, D>(v, lane);
      }
      L::template values<NT>(o, s, v, lane);
      if (bad) {
        for (int j = 0; j < valid; j++) {
          const T *row = (const T *)a.dv + (cur.sg.first + j0 + j) * a.kv_stride + (long long)cur.head * D;
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const float w = __shfl_sync(~0u, j >> 3 ? s[n][2 + h] : s[n][h], (j & 7) * 4 + t);
              const bool see = seen[n * 8 + 2 * t + h] >> (j0 + j) & 1;
#pragma unroll
              for (int i = 0; i < L::kTiles; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  const float x = to_f(row[L::out_dim(i, 2 * e, g)]);
                  if (!isfinite(x) && see) o[i][n][2 * e + h] += w * x;
                }
            }
        }
      }
    }
    // the next piece's first chunks are on their way while this one is joined
    const WarpPiece done = cur;
    if constexpr (CS == 0) {
      if (tid == 0) walk.tell(a, cur, row_blocks, 2 * blockIdx.x + (piece ? 1 : 0));
      more = walk.next(a, ROWS, cur);
      if (more) {
        cur.chunks_of(warp, kTileChunks);
#pragma unroll
        for (int u = 0; u < S::kEarly; u++) issue(cur, u);
      }
    } else {
      more = false;
    }
    const int rows = min(ROWS, done.sg.count * a.group - done.rb * ROWS);
    const bool whole = CS == 0 ? done.t0 == 0 && done.t1 == done.sg.tiles : CS == 1;
    const long long slot = 2 * (long long)blockIdx.x + (piece ? 1 : 0);
    float *join = (float *)(ring + S::kEarly * S::kSlot);
    float *part = CS > 1 ? (float *)ring : a.part + slot * ROWS * D;
    float *to_ml = CS > 1 ? part_ml : a.part_ml + slot * ROWS * 2;
    // dim d of row r: exchanged so that a warp's stores hit different banks
    auto dim_of = [](int r, int d) { return d ^ (((r >> 1) & 3) << 3); };
    constexpr int JR = S::kJoinRows;
#pragma unroll
    for (int m = 0; m < ROWS / JR; m++) {
      __syncthreads();  // every warp is done with what the join lies over
#pragma unroll
      for (int n = m * (JR / 8); n < (m + 1) * (JR / 8); n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float l = sum[n][h] + low[n][h];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(~0u, l, d);
          const int row = n * 8 + 2 * t + h, r = row - m * JR;
          if (g == 0) ml[(warp * ROWS + row) * 2] = ref[n][h], ml[(warp * ROWS + row) * 2 + 1] = l;
          float *to = join + (warp * JR + r) * D;
          if constexpr (L::f32) {
#pragma unroll
            for (int blk = 0; blk < D / 32; blk++)
              *(float4 *)(to + dim_of(r, blk * 32 + 4 * g)) =
                  make_float4(o[2 * blk][n][h], o[2 * blk][n][2 + h], o[2 * blk + 1][n][h], o[2 * blk + 1][n][2 + h]);
          } else {
#pragma unroll
            for (int i = 0; i < L::kTiles; i++)
              to[dim_of(r, i * 16 + g)] = o[i][n][h], to[dim_of(r, i * 16 + 8 + g)] = o[i][n][2 + h];
          }
        }
      if (m == ROWS / JR - 1 && more) load_query(cur);
      __syncthreads();
      for (int i = tid; i < min(JR, rows - m * JR) * (D / 4); i += kTreeThreads) {
        const int r = i / (D / 4), d = i % (D / 4), row = m * JR + r;
        float top = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kTreeWarps; w++) top = fmaxf(top, ml[(w * ROWS + row) * 2]);
        const float base = top == -INFINITY ? 0.f : top;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kTreeWarps; w++) {
          const float f = exp2_(ml[(w * ROWS + row) * 2] - base);
          l = fmaf(f, ml[(w * ROWS + row) * 2 + 1], l);
          const float4 y = *(const float4 *)(join + (w * JR + r) * D + dim_of(r, d * 4));
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
        const float ref = top == -INFINITY ? 0.f : top;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < CS; r++) {
          const float f = exp2_(w[r].x - ref);
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

// Joins the parts of the segments that several runs share.  A block takes
// `group` rows of one segment, 8 / group of its warps (at least one) a row.  All
// parts' maxima are read first, so that the sums over the parts are
// independent loads.
constexpr int kCombineWarps = 8;
constexpr int kMaxRuns = 512;

template <typename T, int D>
__global__ void __launch_bounds__(kCombineWarps * 32) k_tree_combine(const TreeArgs a, int rows_a_block, int row_blocks, int group) {
  __shared__ __align__(16) float o_sm[kCombineWarps][D];
  __shared__ float f_sm[kCombineWarps][kMaxRuns];
  const int b = blockIdx.z, head = blockIdx.y % a.kv_heads, rb = blockIdx.y / a.kv_heads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Segments sg;
  sg.count = a.s.tokens(b, &sg.first);
  const int rows = min(rows_a_block, sg.count * a.group - rb * rows_a_block), row0 = blockIdx.x * group;
  pdl_wait();  // on every path: this grid's end is to mean the main one's too
  if (row0 >= rows) return;
  const int4 where = a.joint[((long long)b * a.kv_heads + head) * row_blocks + rb];
  if (where.x < 0) return;  // written already
  const int n = where.z - where.y + 1;
  // part i: the first run's piece, then each next run's first
  auto slot_of = [&](int i) { return (long long)(i ? 2 * (where.y + i) : where.x); };
  const int share = max(1, kCombineWarps / group);  // warps a row
  const int mine = warp % share;
  float *f_mine = f_sm[warp];
  for (int r0 = 0; r0 < group; r0 += kCombineWarps / share) {
    const int row = row0 + r0 + warp / share;
    const bool there = r0 + warp / share < group && row < rows;
    constexpr int V = D / 32;
    float top = -INFINITY, l = 0.f, x[V] = {};
    if (there) {
      float sums[kMaxRuns / 32];  // of the parts lane, lane + 32, ...
#pragma unroll
      for (int j = 0; j < kMaxRuns / 32; j++) {
        const int i = j * 32 + lane;
        sums[j] = 0.f;
        if (j * 32 < n && i < n) {
          const float2 p = *(const float2 *)(a.part_ml + (slot_of(i) * rows_a_block + row) * 2);
          sums[j] = p.y, f_mine[i] = p.x;
          top = fmaxf(top, p.x);
        }
      }
      for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int j = 0; j < kMaxRuns / 32; j++) {
        const int i = j * 32 + lane;
        if (j * 32 < n && i < n) {
          const float f = exp2_(f_mine[i] - ref);
          f_mine[i] = f;
          l = fmaf(f, sums[j], l);
        }
      }
      for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(~0u, l, d);
      __syncwarp();
#pragma unroll 4
      for (int i = mine; i < n; i += share) {
        const float f = f_mine[i];
        const float *from = a.part + (slot_of(i) * rows_a_block + row) * D + lane * V;
        float y[V];
        if constexpr (V == 4)
          *(float4 *)y = *(const float4 *)from;
        else
          *(float2 *)y = *(const float2 *)from;
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = fmaf(f, y[j], x[j]);
      }
#pragma unroll
      for (int j = 0; j < V; j++) o_sm[warp][lane * V + j] = x[j];
    }
    if (share > 1)
      __syncthreads();
    else
      __syncwarp();
    if (there && mine == 0 && lane < D / 4) {
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < share; w++) {
        const float4 z = *(const float4 *)&o_sm[warp + w][lane * 4];
        y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
      }
      write_row<T, D>(a, sg, head, rb * rows_a_block + row, lane * 4, y, top, l);
    }
    __syncwarp();
  }
}

}  // namespace paged
}  // namespace ocrvl
