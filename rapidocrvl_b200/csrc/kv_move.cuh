// Choosing the positions a cache keeps (ocrvl_op_kv_select), moving them
// together (ocrvl_op_kv_compact) and writing tokens behind a cache
// (ocrvl_op_kv_append).
#pragma once
#include <cooperative_groups.h>

#include "paged.cuh"

namespace ocrvl {
namespace paged {

// ---- select ---------------------------------------------------------------

constexpr int kSelThreads = 1024;
constexpr int kSelBins = 2048;
constexpr int kSelStage = 48 * 1024;  // sums a block holds in shared memory

struct SelectArgs {
  const float *acc;
  long long acc_stride;
  const int *lens;
  int batch, kv_heads, width, keep, sinks, recent;
  int *idx;
  float *sums;
  int *new_lens;
};

// A float's bits in an order that unsigned integers have; NaN lowest, -0 = 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One cluster of CS blocks a row, each with a contiguous slice of it.  The
// need-th largest key of the middle is found 11, 11 and 10 bits at a time from
// histograms that the blocks add up over distributed shared memory; then each
// block writes what it keeps, in order, behind what the blocks before it keep.
template <int CS, bool STAGED>
__global__ void __launch_bounds__(kSelThreads) k_kv_select(const SelectArgs a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) uint32_t keys[];  // STAGED: the slice's keys
  __shared__ uint32_t hist[kSelBins];
  __shared__ uint32_t warp_n[32];
  __shared__ uint32_t found[2];
  __shared__ uint32_t part[2];  // how many of the slice are above the threshold (or always kept), and at it
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CS == 1 ? 0 : (int)cluster.block_rank();
  const int row = blockIdx.x / CS, b = row / a.kv_heads % a.batch;
  const int n = min(max(a.lens[b], 0), a.width), held = min(n, a.keep);
  pdl_launch();
  const float *acc = a.acc + row * a.acc_stride;
  int *idx = a.idx + (long long)row * a.keep;
  float *sums = a.sums ? a.sums + (long long)row * a.keep : nullptr;
  if (a.new_lens && row < a.batch * a.kv_heads && row % a.kv_heads == 0 && rank == 0 && tid == 0) a.new_lens[b] = held;
  for (int j = held + rank * kSelThreads + tid; j < a.keep; j += CS * kSelThreads) {
    idx[j] = -1;
    if (sums) sums[j] = 0.f;
  }
  if (n <= a.keep) {
    for (int j = rank * kSelThreads + tid; j < n; j += CS * kSelThreads) {
      idx[j] = j;
      if (sums) sums[j] = acc[j];
    }
    return;  // the whole cluster alike
  }
  // the middle and the slice of all positions
  const int mid0 = a.sinks, mid1 = n - a.recent;
  const uint32_t need0 = a.keep - a.sinks - a.recent;
  const int slice = (n + CS - 1) / CS, s0 = min(n, rank * slice), s1 = min(n, s0 + slice);
  if (STAGED) {
    for (int i = s0 + tid; i < s1; i += kSelThreads) keys[i - s0] = order_key(acc[i]);
    __syncthreads();
  }
  auto key = [&](int i) { return STAGED ? keys[i - s0] : order_key(acc[i]); };
  const int m0 = max(s0, mid0), m1 = min(s1, mid1);

  uint32_t prefix = 0, need = need0;
#pragma unroll
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = m0 + tid; i < m1; i += kSelThreads) {
      const uint32_t k = key(i);
      if (pass == 0 || k >> (shift + bits) == prefix) atomicAdd(&hist[k >> shift & ((1u << bits) - 1)], 1u);
    }
    uint32_t c[2];
    if (CS > 1) {
      cluster.sync();
      c[0] = c[1] = 0;
      for (int r = 0; r < CS; r++) {
        const uint32_t *h = cluster.map_shared_rank(hist, r);
        c[0] += h[2 * tid], c[1] += h[2 * tid + 1];
      }
      cluster.sync();  // nobody reads this histogram any more
    } else {
      __syncthreads();
      c[0] = hist[2 * tid], c[1] = hist[2 * tid + 1];
    }
    // how many lie above this thread's two bins
    uint32_t mine = c[0] + c[1], above = mine;
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t x = __shfl_down_sync(~0u, above, d);
      if (lane + d < 32) above += x;
    }
    if (lane == 0) warp_n[warp] = above;
    __syncthreads();
    if (tid < 32) {
      uint32_t x = warp_n[lane], y = x;
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t z = __shfl_down_sync(~0u, y, d);
        if (lane + d < 32) y += z;
      }
      warp_n[lane] = y - x;  // of the warps above
    }
    __syncthreads();
    above += warp_n[warp] - mine;
    if (above < need && above + mine >= need) {  // exactly one thread, if need > 0
      const bool upper = above + c[1] >= need;
      found[0] = 2 * tid + (upper ? 1 : 0);
      found[1] = need - above - (upper ? 0 : c[1]);
    }
    __syncthreads();
    if (need > 0) prefix = prefix << bits | found[0], need = found[1];
    __syncthreads();
  }
  // kept: always kept ones, keys above prefix, and the first `need` at it
  const bool any = need0 > 0;
  auto above_it = [&](int i) { return i < mid0 || i >= mid1 || (any && key(i) > prefix); };
  auto at_it = [&](int i) { return any && i >= mid0 && i < mid1 && key(i) == prefix; };
  uint32_t n_above = 0, n_at = 0, base_above = 0, base_at = 0;
  if (CS > 1) {
    for (int i = s0 + tid; i < s1; i += kSelThreads) n_above += above_it(i), n_at += at_it(i);
    for (int d = 16; d; d >>= 1) n_above += __shfl_xor_sync(~0u, n_above, d), n_at += __shfl_xor_sync(~0u, n_at, d);
    if (tid < 2) part[tid] = 0;
    __syncthreads();
    if (lane == 0) atomicAdd(&part[0], n_above), atomicAdd(&part[1], n_at);
    cluster.sync();
    for (int r = 0; r < rank; r++) {
      const uint32_t *p = cluster.map_shared_rank(part, r);
      base_above += p[0], base_at += p[1];
    }
    cluster.sync();  // before any block of the cluster may end
  }
  // in order, 4 positions a thread, 4096 a step: 16 bits hold each count of a step
  for (int i0 = s0; i0 < s1; i0 += 4 * kSelThreads) {
    uint32_t up = 0, at = 0;
    const int i1 = i0 + 4 * tid;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (i1 + e < s1) up |= (uint32_t)above_it(i1 + e) << e, at |= (uint32_t)at_it(i1 + e) << e;
    const uint32_t mine = __popc(up) | __popc(at) << 16;
    uint32_t upto = mine;
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t x = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += x;
    }
    __syncthreads();
    if (lane == 31) warp_n[warp] = upto;
    __syncthreads();
    uint32_t before = 0, all = 0;
    {
      const uint32_t x = warp_n[lane];
      uint32_t y = x;
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t z = __shfl_up_sync(~0u, y, d);
        if (lane >= d) y += z;
      }
      before = __shfl_sync(~0u, y - x, warp);
      all = __shfl_sync(~0u, y, 31);
    }
    before += upto - mine;
    uint32_t na = base_above + (before & 0xffff), nt = base_at + (before >> 16);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const bool u = up >> e & 1, q = at >> e & 1;
      if (u || (q && nt < need)) {
        const uint32_t j = na + min(nt, need);
        idx[j] = i1 + e;
        if (sums) sums[j] = acc[i1 + e];
      }
      na += u, nt += q;
    }
    base_above += all & 0xffff, base_at += all >> 16;
  }
}

// ---- compact ----------------------------------------------------------------

struct CompactArgs {
  const char *src_k, *src_v;
  char *dst_k, *dst_v;
  const int *src_table, *dst_table, *idx;
  long long src_page, dst_page, src_layer, dst_layer, src_head, dst_head, src_table_stride, dst_table_stride;  // bytes; entries
  int src_token, dst_token, src_shift, dst_shift, src_pages, dst_pages, src_max, dst_max;
  int layers, batch, kv_heads, keep, row_bytes;
};

// Byte offset of a position's row in a pool, or -1.
__device__ __forceinline__ long long row_at(const int *table, long long table_stride, int b, int pos, int shift, int max_pages,
                                            int num_pages, long long page, int token) {
  const int e = pos >> shift;
  if (pos < 0 || e >= max_pages) return -1;
  const int pg = table[b * table_stride + e];
  return pg >= 0 && pg < num_pages ? pg * page + (long long)(pos & ((1 << shift) - 1)) * token : -1;
}

constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 64;  // rows a block moves at a time

// To other pages: blocks of 64 rows of K and V, in any order.
__global__ void __launch_bounds__(kMoveThreads) k_kv_compact(const CompactArgs a) {
  __shared__ long long from[kMoveRows], to[kMoveRows];
  const int j0 = blockIdx.y * kMoveRows, row = blockIdx.x;  // row: (layer, sequence, kv head)
  const int head = row % a.kv_heads, b = row / a.kv_heads % a.batch, layer = row / a.kv_heads / a.batch;
  pdl_wait();
  if (threadIdx.x < kMoveRows) {
    const int j = j0 + threadIdx.x, pos = j < a.keep ? a.idx[(long long)row * a.keep + j] : -1;
    const long long x = row_at(a.src_table, a.src_table_stride, b, pos, a.src_shift, a.src_max, a.src_pages, a.src_page, a.src_token);
    const long long y = pos < 0 ? -1 : row_at(a.dst_table, a.dst_table_stride, b, j, a.dst_shift, a.dst_max, a.dst_pages, a.dst_page, a.dst_token);
    from[threadIdx.x] = y < 0 ? -1 : x;
    to[threadIdx.x] = y;
  }
  __syncthreads();
  const long long s = layer * a.src_layer + head * a.src_head, d = layer * a.dst_layer + head * a.dst_head;
  const int pieces = a.row_bytes / 16;
#pragma unroll 4
  for (int i = threadIdx.x; i < 2 * kMoveRows * pieces; i += kMoveThreads) {
    const int p = i % pieces, r = i / pieces % kMoveRows, v = i / pieces / kMoveRows;
    if (from[r] >= 0)
      *(uint4 *)((v ? a.dst_v : a.dst_k) + d + to[r] + p * 16) =
          __ldg((const uint4 *)((v ? a.src_v : a.src_k) + s + from[r] + p * 16));
  }
}

// In place: a block moves one 64-byte column of one (layer, sequence, kv head)'s
// K or V, 64 rows at a time from the first on.  The indices rise, so what a
// step writes (rows j, from rows idx[j] >= j) no later step reads; within a
// step all is read before anything is written.
__global__ void __launch_bounds__(kMoveThreads) k_kv_compact_in_place(const CompactArgs a) {
  const int row = blockIdx.x, v = blockIdx.z, column = blockIdx.y * 64 + threadIdx.x % 4 * 16;
  const int head = row % a.kv_heads, b = row / a.kv_heads % a.batch, layer = row / a.kv_heads / a.batch;
  char *base = (v ? a.dst_v : a.dst_k) + layer * a.dst_layer + head * a.dst_head + column;
  pdl_wait();
  for (int j0 = 0; j0 < a.keep; j0 += kMoveRows) {
    const int j = j0 + threadIdx.x / 4, pos = j < a.keep ? a.idx[(long long)row * a.keep + j] : -1;
    long long x = -1, y = -1;
    if (pos > j) {
      x = row_at(a.src_table, a.src_table_stride, b, pos, a.src_shift, a.src_max, a.src_pages, a.src_page, a.src_token);
      y = row_at(a.src_table, a.src_table_stride, b, j, a.src_shift, a.src_max, a.src_pages, a.src_page, a.src_token);
    }
    uint4 z = make_uint4(0u, 0u, 0u, 0u);
    if (x >= 0 && y >= 0) z = *(const uint4 *)(base + x);
    __syncthreads();
    if (x >= 0 && y >= 0) *(uint4 *)(base + y) = z;
    __syncthreads();
  }
}

// ---- append -------------------------------------------------------------------

struct AppendArgs {
  char *k, *v;
  const char *src_k, *src_v;
  const int *table, *lens, *indptr, *path, *n_path;
  int *new_lens;
  long long page, layer, head, table_stride, src_token, src_layer;  // bytes; entries
  int token, shift, num_pages, max_pages, capacity;
  int layers, batch, kv_heads, n_tokens, max_path, row_bytes;
};

// A warp an item: one token of one layer, K or V, all heads.
__global__ void __launch_bounds__(kMoveThreads) k_kv_append(const AppendArgs a) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int first = min(max(a.indptr[b], 0), a.n_tokens), count = min(max(a.indptr[b + 1], first), a.n_tokens) - first;
  const int len = min(max(a.lens[b], 0), a.capacity);
  const int n = a.path ? min(max(a.n_path[b], 0), a.max_path) : count;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.new_lens[b] = min(len + n, a.capacity);
  const int pieces = a.row_bytes / 16 * a.kv_heads;
  const int items = n * a.layers * 2;
  for (int it = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); it < items; it += gridDim.x * (kMoveThreads / 32)) {
    const int v = it & 1, layer = (it >> 1) % a.layers, i = (it >> 1) / a.layers;
    const int node = a.path ? a.path[(long long)b * a.max_path + i] : i, pos = len + i;
    if (node < 0 || node >= count) continue;
    const long long at = row_at(a.table, a.table_stride, b, pos, a.shift, a.max_pages, a.num_pages, a.page, a.token);
    if (at < 0) continue;
    const char *src = (v ? a.src_v : a.src_k) + layer * a.src_layer + (first + node) * a.src_token;
    char *dst = (v ? a.v : a.k) + at + layer * a.layer;
    for (int p = lane; p < pieces; p += 32) {
      const int h = p / (a.row_bytes / 16), o = p % (a.row_bytes / 16);
      *(uint4 *)(dst + h * a.head + o * 16) = __ldg((const uint4 *)(src + (long long)p * 16));
    }
  }
}

}  // namespace paged
}  // namespace ocrvl
