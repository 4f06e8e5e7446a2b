// What the launches of attention over either kind of cache share: the
// workspace and the join of runs.
#pragma once
#include <cmath>

#include "entry.cuh"
#include "tree_mma.cuh"

namespace ocrvl {
namespace paged {

// The workspace: two parts a block, and 16 bytes a segment in front of them.
inline int64_t tree_joint_bytes(int batch, int kv_heads, int rows) { return ((int64_t)batch * kv_heads * ((rows + 7) / 8) * 16 + 127) / 128 * 128; }
inline int64_t tree_work_bytes(bool f32, int batch, int kv_heads, int dim, int sms, int rows) {
  const int64_t parts = 2ll * sms * (f32 || rows <= 16 ? 2 * 32 : rows > 128 ? 256 : 128);
  return tree_joint_bytes(batch, kv_heads, rows) + parts * (dim + 2) * 4;
}

// Tiles of the longest cache and of its drafts.
inline int tree_tiles(const TreeArgs &a) { return (a.s.capacity + a.s.max_draft + kChunk - 1 + kChunk * kTileChunks - 1) / (kChunk * kTileChunks); }

// What a call whose runs are joined must keep to, asked before its first launch.
inline int check_combine(const TreeArgs &a, int blocks) { return (long long)blocks * a.kv_heads > 65535 ? invalid("too many kv heads") : OCRVL_OK; }

// The join of runs' parts: eight rows a block, or fewer while the blocks would not fill
// the GPU, down to one (then eight warps share a row's parts).
template <typename T, int D>
int launch_combine(const TreeArgs &a, int sms, int rows_max, int rows_a_block, cudaStream_t stream) {
  const int blocks = (rows_max + rows_a_block - 1) / rows_a_block, rows = rows_max < rows_a_block ? rows_max : rows_a_block;
  int group = 8;
  while (group > 1 && (long long)((rows + group - 1) / group) * blocks * a.kv_heads * a.s.batch < 2 * sms) group /= 2;
  return launch("tree attention (join)", k_tree_combine<T, D>, dim3((rows + group - 1) / group, blocks * a.kv_heads, a.s.batch),
                kCombineWarps * 32, 0, stream, true, 1, a, rows_a_block, blocks, group);
}

// With blocks of 256 rows or 128, a block a segment or runs and their join.
template <typename T, int D, bool WIDE, bool SPLIT, bool PACKED>
int launch_tree_mma(TreeArgs a, int sms, int rows_max, char *work, cudaStream_t stream) {
  using S = MmaShape<D, WIDE>;
  const int blocks = (rows_max + S::kRows - 1) / S::kRows;
  const long long segments = (long long)blocks * a.kv_heads * a.s.batch;
  if (segments > 1 << 24) return invalid("too many sequences and kv heads");
  if constexpr (!SPLIT) {
    return launch("tree attention", k_tree_mma<T, D, WIDE, false, PACKED>, dim3((unsigned)segments), kMmaThreads, S::kSmem, stream, PACKED, 1, a, blocks);
  } else {
    if (int rc = check_combine(a, blocks)) return rc;
    const int grid = sms < kMaxRuns ? sms : kMaxRuns;
    a.start_cost = 3;
    a.joint = (int4 *)work;
    a.part = (float *)(work + tree_joint_bytes(a.s.batch, a.kv_heads, rows_max));
    a.part_ml = a.part + (int64_t)grid * 2 * S::kRows * D;
    if (int rc = launch("tree attention", k_tree_mma<T, D, WIDE, true, PACKED>, dim3(grid), kMmaThreads, S::kSmem, stream, PACKED, 1, a, blocks)) return rc;
    return launch_combine<T, D>(a, sms, rows_max, S::kRows, stream);
  }
}

// The shape of the fifth generation's kernel, by the time each takes in tiles of 128
// positions and 128 rows (1.25 us; what was measured at 1 to 74 sequences of 3,000 to
// 131,072 positions, bf16).  A block a segment: its tiles and a start and an end of
// 6, once a wave; with 256 rows twice the tiles.  Runs: the tiles shared out evenly (a narrow
// one takes a third longer there), the start, the join and the parts that go through
// memory: 13 and 0.15 a segment, 21 and 0.3 with 256 rows.  16 sequences of 8,000, 64 drafts
// of 8 heads: 95 us a block a segment of 128 rows, 160 of 256, 130 and 123 in runs; one of
// 131,072: 1178, 2274, 120 and 108.
template <typename T, int D>
int launch_tree_mma_shape(const TreeArgs &a, int sms, int rows_max, char *work, cudaStream_t stream) {
  const double tiles = tree_tiles(a), heads = (double)a.kv_heads * a.s.batch;
  const double narrow = (rows_max + 127) / 128 * heads, wide = (rows_max + 255) / 256 * heads;  // segments
  const double narrow_whole = std::ceil(narrow / sms) * (tiles + 6), wide_whole = std::ceil(wide / sms) * 2 * (tiles + 2);
  const double narrow_runs = narrow * tiles / sms * 4 / 3 + 13 + 0.15 * narrow, wide_runs = wide * tiles / sms * 2 + 21 + 0.3 * wide;
  if (rows_max <= 128)
    return narrow_whole <= narrow_runs ? launch_tree_mma<T, D, false, false, false>(a, sms, rows_max, work, stream)
                                       : launch_tree_mma<T, D, false, true, false>(a, sms, rows_max, work, stream);
  if (narrow_whole <= wide_whole && narrow_whole <= wide_runs) return launch_tree_mma<T, D, false, false, false>(a, sms, rows_max, work, stream);
  return wide_whole <= wide_runs ? launch_tree_mma<T, D, true, false, false>(a, sms, rows_max, work, stream)
                                 : launch_tree_mma<T, D, true, true, false>(a, sms, rows_max, work, stream);
}

}  // namespace paged
}  // namespace ocrvl
