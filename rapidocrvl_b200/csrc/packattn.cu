// C ABI of attention over a packed cache (include/ocrvl_cuda.h): argument checks
// and launches.
#include <cmath>

#include "../../include/ocrvl_cuda.h"
#include "pack_attn.cuh"
#include "packed_entry.cuh"
#include "tree_launch.cuh"

using namespace ocrvl;
using namespace ocrvl::paged;

namespace {

template <typename T, int D, int NT>
int launch_pack(TreeArgs a, int sms, int rows_max, char *work, cudaStream_t stream) {
  using S = PackShape<T, D, NT>;
  const int blocks = (rows_max + S::kRows - 1) / S::kRows;
  const long long segments = (long long)blocks * a.kv_heads * a.s.batch;
  if (segments > 1 << 24) return invalid("too many sequences and kv heads");
  // Blocks (in clusters) a segment, as many as run at once; or equal runs of tiles over all blocks and a second launch
  // that joins them, where a warp then has so many fewer chunks (of the longest cache, which is all that the host knows) that
  // it makes up for the search, the parts and the join.
  constexpr int kRunsCost = 16;  // chunks
  const int tiles = tree_tiles(a);
  const long long room = (long long)sms * S::kBlocks;
  auto one = [&](auto kernel, int cs) {
    return launch("packed attention", kernel, dim3((unsigned)(segments * cs)), kTreeThreads, S::kSmem, stream, !a.longest_first, cs, a, blocks);
  };
  int cs = 1;
  while (cs < 8 && cs < tiles && segments * cs * 2 <= (cs == 1 ? room : (long long)cluster_room(sms) * S::kBlocks)) cs *= 2;
  const double whole = (double)((tiles + cs - 1) / cs) * ((segments * cs + room - 1) / room), runs = (double)segments * tiles / room;
  // Where an SM gets more than one block, in the order of lengths; then not ahead of the kernel before (which would hand
  // blocks out where that one ends first, several of the longest to an SM: 64 bf16 sequences of up to 4,096 27.6 us, 31.4 so).
  a.longest_first = a.s.batch > 1 && a.s.batch <= kTreeThreads && segments * cs > sms;
  if (whole <= runs + kRunsCost)
    return cs == 8 ? one(k_pack_attn<T, D, NT, 8>, 8) : cs == 4 ? one(k_pack_attn<T, D, NT, 4>, 4) : cs == 2 ? one(k_pack_attn<T, D, NT, 2>, 2) : one(k_pack_attn<T, D, NT, 1>, 1);

  if (int rc = check_combine(a, blocks)) return rc;
  const int grid = sms * S::kBlocks < kMaxRuns ? sms * S::kBlocks : kMaxRuns;
  a.start_cost = 1;
  a.joint = (int4 *)work;
  a.part = (float *)(work + tree_joint_bytes(a.s.batch, a.kv_heads, rows_max));
  a.part_ml = a.part + (int64_t)grid * 2 * S::kRows * D;
  if (int rc = launch("packed attention", k_pack_attn<T, D, NT, 0>, dim3(grid), kTreeThreads, S::kSmem, stream, true, 1, a, blocks)) return rc;
  return launch_combine<T, D>(a, sms, rows_max, S::kRows, stream);
}

// Rows a block, as for a plain cache: eight or sixteen where there are no more, or where the call's tiles are so few that
// the GPU is not filled otherwise; else 32 for f32, and the fifth generation's products for 16 bits.
template <typename T, int D>
int launch_pack_rows(const TreeArgs &a, int sms, int rows_max, char *work, cudaStream_t stream) {
  const int room = sizeof(T) == 4 ? sms : 2 * sms;  // blocks that run at once
  auto few = [&](int rows) { return (long long)((rows_max + rows - 1) / rows) * a.kv_heads * a.s.batch * tree_tiles(a) * 2 <= 3 * room; };
  if (rows_max <= 8 || few(8)) return launch_pack<T, D, 1>(a, sms, rows_max, work, stream);
  if (rows_max <= 16 || few(16)) return launch_pack<T, D, 2>(a, sms, rows_max, work, stream);
  if constexpr (sizeof(T) == 4)
    return launch_pack<T, D, 4>(a, sms, rows_max, work, stream);
  else
    return launch_tree_mma_shape<T, D, true>(a, sms, rows_max, work, stream);
}

template <typename T>
int launch_pack_dim(const TreeArgs &a, int dim, int sms, int rows_max, char *work, cudaStream_t stream) {
  return dim == 128 ? launch_pack_rows<T, 128>(a, sms, rows_max, work, stream) : launch_pack_rows<T, 64>(a, sms, rows_max, work, stream);
}

}  // namespace

extern "C" {

int ocrvl_op_packed_attn_workspace(const ocrvl_packed_cache *c, int type, int heads, int max_draft, int64_t *bytes) {
  if (!bytes) return invalid("null argument");
  if (int rc = check_packed(c)) return rc;
  if (!elem_bytes(type)) return invalid("type must be f32, f16 or bf16");
  if (heads < 1 || heads % c->num_kv_heads || max_draft < 1 || max_draft > 64) return invalid("heads must be a multiple of num_kv_heads, max_draft 1..64");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  *bytes = tree_work_bytes(type == OCRVL_F32, c->batch, c->num_kv_heads, c->head_dim, sms, heads / c->num_kv_heads * max_draft);
  return OCRVL_OK;
}

int ocrvl_op_packed_attn(const ocrvl_packed_cache *c, int type, int layer, int heads, int n_tokens, int max_draft,
                         const int32_t *lens, const int32_t *indptr, const int64_t *mask, const void *q, int64_t q_stride,
                         const void *k, const void *v, int64_t kv_stride, float scale, void *out, int64_t out_stride, float *lse,
                         void *work, int64_t work_bytes, void *stream) {
  if (int rc = check_packed(c)) return rc;
  const int es = elem_bytes(type), D = c->head_dim;
  if (!es) return invalid("type must be f32, f16 or bf16");
  if (layer < 0 || layer >= c->num_layers) return invalid("layer outside the cache");
  if (heads < 1 || heads % c->num_kv_heads || heads / c->num_kv_heads > 16)
    return invalid("heads must be a multiple of num_kv_heads, at most 16 times it");
  if (n_tokens < 0) return invalid("n_tokens must not be negative");
  if (max_draft < 1 || max_draft > 64) return invalid("max_draft must be 1..64");
  if (!std::isfinite(scale)) return invalid("scale must be finite");
  if (!lens || !indptr) return invalid("null argument");
  if (n_tokens == 0) return OCRVL_OK;
  if (!mask || !q || !k || !v || !out || !work) return invalid("null argument");
  if (!aligned16(q) || q_stride * es % 16 || q_stride < (int64_t)heads * D)
    return invalid("q must be 16-byte aligned rows of heads * head_dim elements");
  if (!aligned16(k) || !aligned16(v) || kv_stride * es % 16 || kv_stride < (int64_t)c->num_kv_heads * D || kv_stride * es > 0x7fffffff)
    return invalid("k and v must be 16-byte aligned rows of num_kv_heads * head_dim elements");
  if (!aligned16(out) || out_stride * es % 16 || out_stride < (int64_t)heads * D)
    return invalid("out must be 16-byte aligned rows of heads * head_dim elements");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int rows_max = max_draft * (heads / c->num_kv_heads);
  if (((uintptr_t)work & 127) || work_bytes < tree_work_bytes(type == OCRVL_F32, c->batch, c->num_kv_heads, D, sms, rows_max))
    return invalid("work is too small or not 128-byte aligned");
  TreeArgs a = {};
  a.c.k = (const char *)c->k + layer * c->layer_stride, a.c.v = (const char *)c->v + layer * c->layer_stride;
  a.c.table = c->table, a.c.table_stride = c->table_stride;
  a.c.page_bytes = c->page_stride, a.c.head_bytes = c->head_stride, a.c.token_bytes = D / 2;
  a.c.max_pages = c->max_pages, a.c.num_pages = c->num_pages, a.c.page_shift = log2i(c->page_size);
  a.k_scale = (const char *)c->k_scale + layer * c->scale_layer_stride * 2;
  a.v_scale = (const char *)c->v_scale + layer * c->scale_layer_stride * 2;
  a.scale_page = c->scale_page_stride * 2, a.scale_head = c->scale_head_stride * 2;
  a.s = Seqs{lens, indptr, c->batch, n_tokens, max_draft, c->max_pages * c->page_size};
  a.kv_heads = c->num_kv_heads, a.group = heads / c->num_kv_heads;
  a.q = q, a.dk = k, a.dv = v, a.out = out;
  a.q_stride = q_stride, a.kv_stride = kv_stride, a.out_stride = out_stride;
  a.mask = (const long long *)mask, a.scale = scale * kLog2e, a.lse = lse;
  cudaStream_t st = (cudaStream_t)stream;
  if (type == OCRVL_F32) return launch_pack_dim<float>(a, D, sms, rows_max, (char *)work, st);
  if (type == OCRVL_F16) return launch_pack_dim<__half>(a, D, sms, rows_max, (char *)work, st);
  return launch_pack_dim<__nv_bfloat16>(a, D, sms, rows_max, (char *)work, st);
}

}  // extern "C"
