// Choosing the positions a cache keeps (ocrvl_op_kv_select), moving them
// together (ocrvl_op_kv_compact) and writing tokens behind a cache
// (ocrvl_op_kv_append).
#pragma once
#include <cooperative_groups.h>

#include "paged.cuh"

namespace ocrvl {
namespace paged {

// ---- select ---------------------------------------------------------------

constexpr int kSelBins = 2048;
constexpr int kSelList = 256;  // keys that are ranked directly
constexpr int kSelStage = 48 * 1024;  // keys a block holds in shared memory: a multiple of its threads times four

struct SelectArgs {
  const float *acc;
  long long acc_stride;
  const int *lens;
  int batch, kv_heads, width, keep, sinks, recent;
  int *idx;
  float *sums;
  int *new_lens;
};

// A float's bits in an order that unsigned integers have, NaN lowest, -0 = 0,
// all of them between kNever (not a position) and kAlways (kept whatever its sum).
constexpr uint32_t kNever = 0u, kAlways = ~0u;
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 1u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One cluster of CS blocks a row, each with a contiguous slice of it, each
// warp with a contiguous part of the slice.  The need-th largest key of the
// middle is found from histograms of 2048 equal bins, first over the range
// from the smallest to the largest key, then over the bin that holds it, until a
// bin is one key, or holds so few that they are listed and ranked directly; the
// cluster's blocks add their filled bins to the first one's over distributed
// shared memory, which searches.
// Sums span many powers of two, so the range fills the bins evenly where the
// leading bits of the keys would send most of a warp's additions to one
// address.  Then each warp writes what it keeps, in order, behind what those
// before it keep.  Bound by latencies: the loads of a step go out together, and
// a round of the search takes 1 to 2 us.  36 rows of 1,257 sums, 512 kept: 8.4 us; 16
// rows of 131,072, 4,096 kept: 29 us.
template <int CS, bool STAGED, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_kv_select(const SelectArgs a) {
  namespace cg = cooperative_groups;
  constexpr int WARPS = THREADS / 32, OWN = kSelBins / THREADS;  // bins a thread looks after
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) uint32_t keys[];  // STAGED: the slice's keys
  __shared__ uint32_t hist[kSelBins], total[CS > 1 ? kSelBins : 1];
  __shared__ uint32_t warp_n[WARPS], warp_m[WARPS];
  __shared__ uint32_t found[3], list[kSelList], list_n;
  __shared__ uint32_t range[2], part[2];  // read by the cluster
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CS == 1 ? 0 : (int)cluster.block_rank();
  const int row = blockIdx.x / CS, b = row / a.kv_heads % a.batch;
  const int n = min(max(a.lens[b], 0), a.width), held = min(n, a.keep);
  pdl_launch();
  const float *acc = a.acc + row * a.acc_stride;
  int *idx = a.idx + (long long)row * a.keep;
  float *sums = a.sums ? a.sums + (long long)row * a.keep : nullptr;
  if (a.new_lens && row < a.batch * a.kv_heads && row % a.kv_heads == 0 && rank == 0 && tid == 0) a.new_lens[b] = held;
  for (int j = held + rank * THREADS + tid; j < a.keep; j += CS * THREADS) {
    idx[j] = -1;
    if (sums) sums[j] = 0.f;
  }
  if (n <= a.keep) {
    for (int j = rank * THREADS + tid; j < n; j += CS * THREADS) {
      idx[j] = j;
      if (sums) sums[j] = acc[j];
    }
    return;  // the whole cluster alike
  }
  // the middle, the block's slice of all positions and the warp's part of it,
  // in steps of 128
  const int mid0 = a.sinks, mid1 = n - a.recent;
  const int slice = ((n + CS - 1) / CS + 3) & ~3, s0 = min(n, rank * slice), s1 = min(n, s0 + slice);
  const int steps = (slice + THREADS * 4 - 1) / (THREADS * 4), w0 = s0 + warp * steps * 128;
  auto sum_of = [&](int i) { return i < s1 ? __ldg(acc + i) : 0.f; };
  auto key_of = [&](int i, float x) { return i >= s1 ? kNever : i < mid0 || i >= mid1 ? kAlways : order_key(x); };
  // the keys of positions i .. i + 3
  auto key4 = [&](int i) {
    if constexpr (STAGED)
      return *reinterpret_cast<const uint4 *>(keys + (i - s0));
    const float x[4] = {sum_of(i), sum_of(i + 1), sum_of(i + 2), sum_of(i + 3)};
    return make_uint4(key_of(i, x[0]), key_of(i + 1, x[1]), key_of(i + 2, x[2]), key_of(i + 3, x[3]));
  };

  uint32_t low = ~0u, high = 0u;
  if (STAGED) {  // all of the warp's sums on their way at once, then turned into keys where they lie
    const uint32_t at = smem_addr(keys);
    if (((uintptr_t)acc & 15) == 0) {  // then acc + s0 is too, but where the slice is empty
      for (int j = 0; j < steps; j++) {
        const int i = w0 + j * 128 + lane * 4, n4 = min(4, max(0, s1 - i));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + (i - s0) * 4), "l"(n4 ? acc + i : acc), "r"(n4 * 4) : "memory");
      }
    } else {
      for (int j = 0; j < steps * 4; j++) {
        const int i = w0 + j * 32 + lane;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(at + (i - s0) * 4), "l"(i < s1 ? acc + i : acc), "r"(i < s1 ? 4 : 0) : "memory");
      }
    }
    copy_commit();
    copy_wait<0>();
    __syncwarp();
  }
  for (int j = 0; j < steps; j++) {
    const int i = w0 + j * 128 + lane * 4;
    uint4 k;
    if constexpr (STAGED) {
      const float4 x = *reinterpret_cast<const float4 *>(keys + (i - s0));
      k = make_uint4(key_of(i, x.x), key_of(i + 1, x.y), key_of(i + 2, x.z), key_of(i + 3, x.w));
      *reinterpret_cast<uint4 *>(keys + (i - s0)) = k;
    } else {
      k = key4(i);
    }
    auto widen = [&](uint32_t x) {
      if (x != kNever && x != kAlways) low = min(low, x), high = max(high, x);
    };
    widen(k.x), widen(k.y), widen(k.z), widen(k.w);
  }
  low = __reduce_min_sync(~0u, low), high = __reduce_max_sync(~0u, high);
  if (lane == 0) warp_n[warp] = low, warp_m[warp] = high;
  if (tid == 0) list_n = 0;
  for (int i = tid; i < kSelBins; i += THREADS) {
    hist[i] = 0;
    if (CS > 1) total[i] = 0;
  }
  __syncthreads();
  low = __reduce_min_sync(~0u, lane < WARPS ? warp_n[lane] : ~0u), high = __reduce_max_sync(~0u, lane < WARPS ? warp_m[lane] : 0u);
  if (CS > 1) {
    if (tid == 0) range[0] = low, range[1] = high;
    cluster.sync();
    for (int r = 0; r < CS; r++) {
      const uint32_t *p = cluster.map_shared_rank(range, r);
      low = min(low, p[0]), high = max(high, p[1]);
    }
  }

  uint32_t need = a.keep - a.sinks - a.recent, base = kAlways - 1;
  if (need > 0) {
    uint32_t span = high - low;  // the key is in base .. base + span
    base = low;
    while (true) {
      const int shift = max(0, 32 - __clz(span) - 11);  // span >> shift < 2048
      for (int j = 0; j < steps; j++) {
        const uint4 k = key4(w0 + j * 128 + lane * 4);
        if (k.x - base <= span) atomicAdd(&hist[(k.x - base) >> shift], 1u);
        if (k.y - base <= span) atomicAdd(&hist[(k.y - base) >> shift], 1u);
        if (k.z - base <= span) atomicAdd(&hist[(k.z - base) >> shift], 1u);
        if (k.w - base <= span) atomicAdd(&hist[(k.w - base) >> shift], 1u);
      }
      __syncthreads();
      uint32_t c[OWN], mine = 0;
#pragma unroll
      for (int j = 0; j < OWN; j++) c[j] = hist[OWN * tid + j], hist[OWN * tid + j] = 0;
      if (CS > 1) {
        uint32_t *first = cluster.map_shared_rank(total, 0);
#pragma unroll
        for (int j = 0; j < OWN; j++)
          if (c[j]) atomicAdd(first + OWN * tid + j, c[j]);
        cluster.sync();
      }
      if (rank == 0) {
        if (CS > 1) {
#pragma unroll
          for (int j = 0; j < OWN; j++) c[j] = total[OWN * tid + j], total[OWN * tid + j] = 0;
        }
        // how many lie above this thread's bins
#pragma unroll
        for (int j = 0; j < OWN; j++) mine += c[j];
        uint32_t above = mine;
        for (int d = 1; d < 32; d <<= 1) {
          const uint32_t x = __shfl_down_sync(~0u, above, d);
          if (lane + d < 32) above += x;
        }
        if (lane == 0) warp_n[warp] = above;
        above -= mine;
        __syncthreads();
        above += __reduce_add_sync(~0u, lane > warp && lane < WARPS ? warp_n[lane] : 0u);
        if (above < need && above + mine >= need) {  // exactly one thread
          uint32_t over = above;
#pragma unroll
          for (int j = OWN - 1; j >= 0; j--) {
            if (over < need && over + c[j] >= need) {
              for (int r = 0; r < CS; r++) {
                uint32_t *to = CS > 1 ? cluster.map_shared_rank(found, r) : found;
                to[0] = OWN * tid + j, to[1] = need - over, to[2] = c[j];
              }
            }
            over += c[j];
          }
        }
      }
      if (CS > 1)
        cluster.sync();
      else
        __syncthreads();
      base += found[0] << shift, need = found[1];
      if (shift == 0) break;
      span = (1u << shift) - 1;
      const uint32_t count = found[2];
      if (count > kSelList) continue;
      uint32_t *to = CS > 1 ? cluster.map_shared_rank(list, 0) : list, *to_n = CS > 1 ? cluster.map_shared_rank(&list_n, 0) : &list_n;
      for (int j = 0; j < steps; j++) {
        const uint4 k = key4(w0 + j * 128 + lane * 4);
        if (k.x - base <= span) to[atomicAdd(to_n, 1u)] = k.x;
        if (k.y - base <= span) to[atomicAdd(to_n, 1u)] = k.y;
        if (k.z - base <= span) to[atomicAdd(to_n, 1u)] = k.z;
        if (k.w - base <= span) to[atomicAdd(to_n, 1u)] = k.w;
      }
      if (CS > 1)
        cluster.sync();
      else
        __syncthreads();
      if (rank == 0 && tid < count) {
        const uint32_t k = list[tid];
        uint32_t over = 0, same = 0;
        for (uint32_t i = 0; i < count; i++) over += list[i] > k, same += list[i] == k;
        if (over < need && over + same >= need) {  // the same values from every thread that has this key
          for (int r = 0; r < CS; r++) {
            uint32_t *f = CS > 1 ? cluster.map_shared_rank(found, r) : found;
            f[0] = k, f[1] = need - over;
          }
        }
      }
      if (CS > 1)
        cluster.sync();
      else
        __syncthreads();
      base = found[0], need = found[1];
      break;
    }
  }
  // kept: keys above base, and the first `need` equal to it
  uint32_t n_above = 0, n_at = 0;
  for (int j = 0; j < steps; j++) {
    const uint4 k = key4(w0 + j * 128 + lane * 4);
    n_above += (k.x > base) + (k.y > base) + (k.z > base) + (k.w > base);
    n_at += (k.x == base) + (k.y == base) + (k.z == base) + (k.w == base);
  }
  n_above = __reduce_add_sync(~0u, n_above), n_at = __reduce_add_sync(~0u, n_at);
  __syncthreads();
  if (lane == 0) warp_n[warp] = n_above, warp_m[warp] = n_at;
  __syncthreads();
  const uint32_t x = lane < WARPS ? warp_n[lane] : 0u, y = lane < WARPS ? warp_m[lane] : 0u;
  uint32_t before = __reduce_add_sync(~0u, lane < warp ? x : 0u), at = __reduce_add_sync(~0u, lane < warp ? y : 0u);
  if (CS > 1) {
    const uint32_t all_x = __reduce_add_sync(~0u, x), all_y = __reduce_add_sync(~0u, y);
    if (tid == 0) part[0] = all_x, part[1] = all_y;
    cluster.sync();
    for (int r = 0; r < rank; r++) {
      const uint32_t *p = cluster.map_shared_rank(part, r);
      before += p[0], at += p[1];
    }
    cluster.sync();  // before any block of the cluster may end
  }
  // the sum behind a key: from the key itself, unless that says too little
  auto sum_behind = [&](uint32_t k, int i) {
    if (k == kAlways || k == 1u || k == 0x80000000u) return __ldg(acc + i);
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  };
  const unsigned lower = (1u << lane) - 1;
  for (int j = 0; j < steps; j++) {
    const int i = w0 + j * 128 + lane * 4;
    const uint4 k4 = key4(i);
    const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
    uint32_t nu = before, nq = at;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const unsigned us = __ballot_sync(~0u, k[e] > base), qs = __ballot_sync(~0u, k[e] == base);
      nu += __popc(us & lower), nq += __popc(qs & lower);
      before += __popc(us), at += __popc(qs);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const bool u = k[e] > base, q = k[e] == base;
      if (u || (q && nq < need)) {
        const uint32_t to = nu + min(nq, need);
        idx[to] = i + e;
        if (sums) sums[to] = sum_behind(k[e], i + e);
      }
      nu += u, nq += q;
    }
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
constexpr int kMoveRows = 32;  // rows a block moves at a time

// To other pages: blocks of 32 rows of K and V of ROW bytes, in any order.  A
// thread's loads are all on their way before its first store.  With the choice before
// it, 4 layers of 8 sequences cut from up to 8,448 to 1,024 bf16 positions take 21 us, 3.3
// TB/s of what is read and written.
template <int ROW>
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
  constexpr int PIECES = ROW / 16, LANES = kMoveThreads / PIECES, STEPS = kMoveRows / LANES;  // rows at a time, and how often
  const int p = threadIdx.x % PIECES, r0 = threadIdx.x / PIECES;
  const long long s = layer * a.src_layer + head * a.src_head + p * 16, d = layer * a.dst_layer + head * a.dst_head + p * 16;
  uint4 k[STEPS], v[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; i++) {
    const long long x = from[r0 + i * LANES];
    if (x >= 0) k[i] = __ldg((const uint4 *)(a.src_k + s + x)), v[i] = __ldg((const uint4 *)(a.src_v + s + x));
  }
#pragma unroll
  for (int i = 0; i < STEPS; i++) {
    const long long y = to[r0 + i * LANES];
    if (from[r0 + i * LANES] >= 0) *(uint4 *)(a.dst_k + d + y) = k[i], *(uint4 *)(a.dst_v + d + y) = v[i];
  }
}

// In place: a block moves one 64-byte column of one (layer, sequence, kv head)'s
// K or V, 256 rows at a time from the first on.  The indices rise, so what a
// step writes (rows j, from rows idx[j] >= j) no later step reads; within a
// step all is read before anything is written.  Bound by a step's chain of loads (an
// index, two table entries, the row), so a thread has four rows on their way at once.  2 layers of
// 8 heads, 4,096 of 131,072 f16 positions: 43 us, where the move to other pages takes 10.5; 18 layers,
// 512 of 1,257 f32 positions: 10.4 and 6.6.
__global__ void __launch_bounds__(kMoveThreads) k_kv_compact_in_place(const CompactArgs a) {
  constexpr int AT = 4, ROWS = kMoveThreads / 4;
  const int row = blockIdx.x, v = blockIdx.z, column = blockIdx.y * 64 + threadIdx.x % 4 * 16;
  const int head = row % a.kv_heads, b = row / a.kv_heads % a.batch, layer = row / a.kv_heads / a.batch;
  char *base = (v ? a.dst_v : a.dst_k) + layer * a.dst_layer + head * a.dst_head + column;
  pdl_wait();
  for (int j0 = 0; j0 < a.keep; j0 += ROWS * AT) {
    long long x[AT], y[AT];
    uint4 z[AT];
#pragma unroll
    for (int i = 0; i < AT; i++) {
      const int j = j0 + i * ROWS + threadIdx.x / 4, pos = j < a.keep ? a.idx[(long long)row * a.keep + j] : -1;
      const bool moves = pos > j;
      x[i] = row_at(a.src_table, a.src_table_stride, b, moves ? pos : -1, a.src_shift, a.src_max, a.src_pages, a.src_page, a.src_token);
      y[i] = row_at(a.src_table, a.src_table_stride, b, moves ? j : -1, a.src_shift, a.src_max, a.src_pages, a.src_page, a.src_token);
    }
#pragma unroll
    for (int i = 0; i < AT; i++)
      if (x[i] >= 0 && y[i] >= 0) z[i] = *(const uint4 *)(base + x[i]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < AT; i++)
      if (x[i] >= 0 && y[i] >= 0) *(uint4 *)(base + y[i]) = z[i];
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

// A warp an item: K and V of one token in up to kAppendLayers layers, all heads: the
// token's place is looked up once, and the loads of all its layers are on their way
// before the first store (a layer, K or V an item: 12.4 us for the prompt below, bound by
// each item's divisions and look-ups).  1,241 tokens of 18 bf16 layers: 8.3 us, 5.5 TB/s
// read and written; 64 sequences' accepted tokens: 6.2 us, a launch and three loads
// behind one another.
constexpr int kAppendLayers = 3;
__global__ void __launch_bounds__(kMoveThreads) k_kv_append(const AppendArgs a) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int first = min(max(a.indptr[b], 0), a.n_tokens), count = min(max(a.indptr[b + 1], first), a.n_tokens) - first;
  const int len = min(max(a.lens[b], 0), a.capacity);
  const int n = a.path ? min(max(a.n_path[b], 0), a.max_path) : count;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.new_lens[b] = min(len + n, a.capacity);
  const int row_pieces = a.row_bytes / 16, pieces = row_pieces * a.kv_heads;
  const int groups = (a.layers + kAppendLayers - 1) / kAppendLayers, items = n * groups;
  for (int it = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); it < items; it += gridDim.x * (kMoveThreads / 32)) {
    const int i = it / groups, layer0 = it % groups * kAppendLayers;
    const int node = a.path ? a.path[(long long)b * a.max_path + i] : i, pos = len + i;
    if (node < 0 || node >= count) continue;
    const long long at = row_at(a.table, a.table_stride, b, pos, a.shift, a.max_pages, a.num_pages, a.page, a.token);
    if (at < 0) continue;
    const long long from = layer0 * a.src_layer + (first + node) * a.src_token, to = at + layer0 * a.layer;
    for (int p = lane; p < pieces; p += 32) {
      const char *src_k = a.src_k + from + (long long)p * 16, *src_v = a.src_v + from + (long long)p * 16;
      const long long dst = to + p / row_pieces * a.head + p % row_pieces * 16;
      uint4 k[kAppendLayers], v[kAppendLayers];
#pragma unroll
      for (int l = 0; l < kAppendLayers; l++)
        if (layer0 + l < a.layers) k[l] = __ldg((const uint4 *)(src_k + l * a.src_layer)), v[l] = __ldg((const uint4 *)(src_v + l * a.src_layer));
#pragma unroll
      for (int l = 0; l < kAppendLayers; l++)
        if (layer0 + l < a.layers) *(uint4 *)(a.k + dst + l * a.layer) = k[l], *(uint4 *)(a.v + dst + l * a.layer) = v[l];
    }
  }
}

}  // namespace paged
}  // namespace ocrvl
