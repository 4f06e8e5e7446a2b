// What the launches of attention over either kind of cache share: the
// workspace and the join of runs.
#pragma once
#include "entry.cuh"
#include "tree_attn.cuh"

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

}  // namespace paged
}  // namespace ocrvl
