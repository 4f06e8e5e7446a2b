// The attention weight that cached positions got from a set of tokens
// (ocrvl_op_attn_mass):
//   acc'[t] = decay acc[t] + sum over rows of 2^(scale log2(e) q . k_t - lse log2(e))
// with the rows' lse known, so one pass over K does: no maximum, no second
// pass.  Every position belongs to one warp, which adds its rows' weights in
// a fixed order: no atomics, the same sums every time.
//
// A block takes a run of tiles of 128 positions (16 a warp) of one
// (sequence, kv head) after another; query fragments of up to kRowTiles x 8
// rows lie in shared memory (of 8 rows, in registers), more rows take further
// passes over the run's K.
#pragma once
#include "paged.cuh"

namespace ocrvl {
namespace paged {

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
};

template <typename T, int D, bool THIN>
struct MassShape {
  using L = Tile<T, D>;
  static constexpr int kUnits = L::kBytes >= 8192 ? 3 : L::kBytes >= 4096 ? 4 : 6;
  static constexpr int kRing = kMassWarps * kUnits * L::kBytes;
  static constexpr int kRowTiles = THIN ? 1 : L::f32 ? (D == 128 ? 4 : 16) : 32;
  static constexpr int kLoad = L::f32 ? 4 : 12;
  static constexpr int kSmem = kRing + kRowTiles * L::kQBytes + kRowTiles * 8 * 4 + 64;
};

template <typename T, int D, bool THIN>
__global__ void __launch_bounds__(kMassThreads) k_attn_mass(const MassArgs a) {
  using S = MassShape<T, D, THIN>;
  using L = Tile<T, D>;
  constexpr int NU = S::kUnits;
  extern __shared__ __align__(128) char sm[];
  char *ring = sm, *q_sm = sm + S::kRing;
  float *shift = (float *)(q_sm + S::kRowTiles * L::kQBytes);  // lse log2(e), +inf for rows that do not count
  long long *plan = (long long *)(shift + S::kRowTiles * 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane & 3;

  // where this block's share of the cost starts: a sequence, the cost below it
  if (warp == 0) {
    long long all = 0;
    for (int b = lane; b < a.s.batch; b += 32) all += MassShare(a, b, S::kLoad).total(a.kv_heads);
    for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(~0u, all, d);
    const long long lo = all * blockIdx.x / gridDim.x;
    if (lane == 0) plan[0] = all, plan[1] = a.s.batch, plan[2] = all;
    __syncwarp();
    long long below = 0;
    for (int b0 = 0; b0 < a.s.batch; b0 += 32) {
      const long long mine = b0 + lane < a.s.batch ? MassShare(a, b0 + lane, S::kLoad).total(a.kv_heads) : 0;
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
  __syncthreads();
  const long long lo = plan[0] * blockIdx.x / gridDim.x, hi = plan[0] * (blockIdx.x + 1) / gridDim.x;

  const uint32_t my_ring = smem_addr(ring) + warp * NU * L::kBytes, q_at = smem_addr(q_sm);
  long long at = plan[2];  // cost below the current segment
  for (int b = (int)plan[1]; b < a.s.batch && at < hi; b++) {
    const MassShare sh(a, b, S::kLoad);
    for (int head = 0; head < a.kv_heads; head++) {
      // the tiles whose cost starts in this block's share
      const long long from = max(lo - at, 0ll), to = hi - at;
      const int t0 = (int)min((long long)sh.tiles, (from + sh.cost - 1) / sh.cost);
      const int t1 = to <= 0 ? 0 : (int)min((long long)sh.tiles, (to + sh.cost - 1) / sh.cost);
      at += (long long)sh.tiles * sh.cost;
      if (t0 >= t1) continue;
      const int c0 = t0 * kMassWarps + warp, chunks = (sh.len + kChunk - 1) / kChunk;
      const int c_end = min(t1 * kMassWarps, chunks);
      const int nk = c0 < c_end ? (c_end - c0 + kMassWarps - 1) / kMassWarps : 0;
      const int rows = sh.count * a.group, row_tiles = (rows + 7) / 8;
      const float *acc = a.acc ? a.acc + ((long long)b * a.kv_heads + head) * a.acc_stride : nullptr;
      float *out = a.out + ((long long)b * a.kv_heads + head) * a.out_stride;

      for (int m0 = 0; m0 == 0 || m0 < row_tiles; m0 += S::kRowTiles) {
        const int mt = min(S::kRowTiles, (row_tiles - m0 + 3) / 4 * 4);  // rows past the last do not count
        int pages = -1;
        unsigned long long valids = 0;  // 8 bits a unit in flight, the next one lowest
        auto issue = [&](int k) {
          if (k < nk) {
            const int c = c0 + k * kMassWarps, pos = c * kChunk;
            if ((k & 31) == 0) {
              const int mine = c + lane * kMassWarps;
              pages = mine < chunks ? a.c.table[b * a.c.table_stride + ((mine * kChunk) >> a.c.page_shift)] : -1;
            }
            const int pg = __shfl_sync(~0u, pages, k & 31);
            const bool mapped = pg >= 0 && pg < a.c.num_pages;
            const int valid = mapped ? min(kChunk, sh.len - pos) : 0;
            valids |= (unsigned long long)valid << (8 * (k % NU));
            L::template load<false>(my_ring + k % NU * L::kBytes,
                                    a.c.k + (mapped ? pg : 0) * a.c.page_bytes + head * a.c.head_bytes +
                                        (long long)(pos & ((1 << a.c.page_shift) - 1)) * a.c.token_bytes,
                                    a.c.token_bytes, valid, lane);
          }
          copy_commit();
        };
        __syncthreads();  // the last pass is done with the query rows
#pragma unroll
        for (int k = 0; k < NU - 1; k++) issue(k);
        const unsigned long long on = a.counted ? (unsigned long long)a.counted[b] : ~0ull;
        auto counts = [&](int r) { return r < rows && (on >> (r / a.group) & 1); };
        L::query(q_at, mt, tid, kMassThreads, [&](int r) -> const T * {
          const int x = m0 * 8 + r;
          return counts(x) ? (const T *)a.q + (sh.first + x / a.group) * a.q_stride + (long long)(head * a.group + x % a.group) * D
                           : nullptr;
        });
        for (int r = tid; r < mt * 8; r += kMassThreads) {
          const int x = m0 * 8 + r;
          float l = INFINITY;
          if (counts(x)) {
            l = a.lse[(long long)(sh.first + x / a.group) * a.kv_heads * a.group + head * a.group + x % a.group] * kLog2e;
            if (l == -INFINITY) l = INFINITY;  // attended nothing
          }
          shift[r] = l;
        }
        __syncthreads();
        uint32_t qr[THIN ? L::kTiles : 1][L::kQRegs];
        const float keep = m0 ? 1.f : a.decay;  // further passes add to what the first wrote
        auto sum_at = [&](int pos) {
          if (lane >= kChunk || pos >= sh.len) return 0.f;
          return m0 ? out[pos] : acc && pos < a.acc_width ? acc[pos] : 0.f;
        };
        float ahead = nk ? sum_at(c0 * kChunk + lane) : 0.f;
        float l0 = INFINITY, l1 = INFINITY;
        if constexpr (THIN) {
          if (mt > 0) {
#pragma unroll
            for (int blk = 0; blk < L::kTiles; blk++) L::q_load(qr[blk], q_at, blk, lane);
            l0 = shift[2 * t], l1 = shift[2 * t + 1];
          }
        }
        for (int k = 0; k < nk; k++) {
          copy_wait<NU - 2>();
          __syncwarp();
          const int valid = (int)(valids >> (8 * (k % NU))) & 31;
          valids &= ~(0xffull << (8 * (k % NU)));
          issue(k + NU - 1);
          // lane j < 16 has position j; what the next chunk's sums were is on its way
          // while this one's products run
          const int pos = (c0 + k * kMassWarps) * kChunk + lane;
          const float old = ahead;
          ahead = k + 1 < nk ? sum_at(pos + kMassWarps * kChunk) : 0.f;
          const uint32_t k_at = my_ring + k % NU * L::kBytes;
          float w[2] = {0.f, 0.f};  // positions g and g + 8
          auto add = [&](const float(&s)[4], const float(&c)[2][4]) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = L::f32 ? s[e] + (c[0][e] + c[1][e]) : s[e];
            w[0] += exp2_(fmaf(y[0], a.scale, -l0)) + exp2_(fmaf(y[1], a.scale, -l1));
            w[1] += exp2_(fmaf(y[2], a.scale, -l0)) + exp2_(fmaf(y[3], a.scale, -l1));
          };
          if constexpr (THIN) {
            if (mt > 0) {
              float s[4] = {}, c[2][4] = {};
#pragma unroll
              for (int blk = 0; blk < L::kTiles; blk++) {
                typename L::KFrag f;
                L::k_load(f, blk, k_at, lane);
                L::k_product(s, c, qr[blk], f);
              }
              add(s, c);
            }
          } else {
            typename L::KFrag f[L::kTiles];
#pragma unroll
            for (int blk = 0; blk < L::kTiles; blk++) L::k_load(f[blk], blk, k_at, lane);
            // several tiles of rows at once: a chain of products of its own takes 11.5 ns a link
            constexpr int AT = L::f32 ? 2 : 4;
            for (int m = 0; m < mt; m += AT) {
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
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) w[n] += __shfl_xor_sync(~0u, w[n], d);
          // lane j takes position j's sum from the lane that holds it
          const int j = lane & 15;
          const float w0 = __shfl_sync(~0u, w[0], (j & 7) * 4), w1 = __shfl_sync(~0u, w[1], (j & 7) * 4);
          float mine = j & 8 ? w1 : w0;
          if (j >= valid) mine = 0.f;
          if (lane < kChunk && pos < sh.len) out[pos] = fmaf(keep, old, mine);
        }
        copy_wait<0>();
      }
    }
  }
  // 0 past the lengths: each row by the blocks that share its remainder
  const int all_rows = a.s.batch * a.kv_heads, share = max(1, (int)gridDim.x / all_rows);
  for (int i = blockIdx.x; i < all_rows * share; i += gridDim.x) {
    const int r = i % all_rows, p = i / all_rows, len = min(a.s.len(r / a.kv_heads), a.out_width);
    for (int x = len + p * kMassThreads + tid; x < a.out_width; x += share * kMassThreads) a.out[r * a.out_stride + x] = 0.f;
  }
}

}  // namespace paged
}  // namespace ocrvl
