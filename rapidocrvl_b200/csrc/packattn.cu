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

// What a call would take, in us, by the kernel's shape; all that the host knows of the lengths is the table's width.
//   8 NT rows a block, clusters of cs blocks a segment: tiles / cs at `tile` each (8 warps, a chunk each; no less than 0.85,
//     the latency of a chunk), as often as the blocks are waves of the SMs (of mean length), drafts at `draft` a position of a warp, and 10
//     for launch, start and join
//   runs (cs 0): all tiles over all SMs, and 22, with the search for a run's start, the parts and their join
//   the fifth generation's products, 128 or 256 rows: 2.7 (3.6 in runs) or 4.4 a tile, mostly the time of the warps that
//     unpack it, and 8, or 24 and 55 in runs
// Measured (bf16, 16 / 2 heads of 128, up to 4,096 positions, 37 sequences of one, two and four tokens; NT 1, 2, 4): 23.6,
// 35.8 and 60.4 us; 39.3, 27.0 and 45.3; 39.5, 39.2 and 42.0; fifth generation 92.  40 of up to 6,000, 12 tokens (96
// rows): 119.7, 86.9, 91.7; 135.5.  32 / 8 heads of 64, 103,991 positions, 5 tokens, runs: 74, 76, 60; clusters of eight
// with NT 1: 100.  f32, 5 of 95 with 50 drafts: 17.4, 19.5, 32.8.
constexpr double kMean = 0.75;  // of the lengths, over the longest: between equal and evenly spread ones
struct Shape {
  double us;
  int nt, cs;
};

template <typename T, int D, int NT>
Shape shape_of(const TreeArgs &a, int sms, int rows_max) {
  constexpr double wide = sizeof(T) == 4 ? (NT == 1 ? 1.0 : NT == 2 ? 1.6 : 3.0) : (NT == 1 ? 0.75 : NT == 2 ? 1.0 : 1.9);
  constexpr double tile = wide * (D == 64 ? 0.55 : 1), alone = tile > 0.85 ? tile : 0.85;
  constexpr double draft = (sizeof(T) == 4 ? 0.4 : 0.25) * NT;
  const int blocks_an_sm = PackShape<T, D, NT>::kBlocks, tiles = tree_tiles(a);
  const double segments = (double)((rows_max + 8 * NT - 1) / (8 * NT)) * a.kv_heads * a.s.batch;
  int cs = 1;
  while (cs < 8 && cs < tiles && segments * cs * 2 <= (cs == 1 ? sms : cluster_room(sms)) * blocks_an_sm) cs *= 2;
  const double drafts = (a.s.max_draft + 8 * cs - 1) / (8 * cs) * draft, waves = segments * cs / sms;
  const double whole = std::fmax(1, waves * kMean) * ((tiles + cs - 1) / cs * (waves < 2 ? alone : tile) + drafts) + 10;
  const double runs = segments * tiles / sms * tile * kMean + drafts + 22;
  return whole <= runs ? Shape{whole, NT, cs} : Shape{runs, NT, 0};
}

template <typename T, int D, int NT>
int launch_pack(TreeArgs a, const Shape &shape, int sms, int rows_max, char *work, cudaStream_t stream) {
  using S = PackShape<T, D, NT>;
  const int blocks = (rows_max + S::kRows - 1) / S::kRows;
  const long long segments = (long long)blocks * a.kv_heads * a.s.batch;
  if (segments > 1 << 24) return invalid("too many sequences and kv heads");
  const int cs = shape.cs;
  if (cs) {
    // Where an SM gets more than one block, in the order of lengths; then not ahead of the kernel before (which would hand
    // blocks out where that one ends first, several of the longest to an SM: 64 bf16 sequences of up to 4,096 27.6 us, 31.4 so).
    a.longest_first = a.s.batch > 1 && a.s.batch <= kTreeThreads && segments * cs > sms;
    auto go = [&](auto kernel) {
      return launch("packed attention", kernel, dim3((unsigned)(segments * cs)), kTreeThreads, S::kSmem, stream, !a.longest_first, cs, a, blocks);
    };
    return cs == 8 ? go(k_pack_attn<T, D, NT, 8>) : cs == 4 ? go(k_pack_attn<T, D, NT, 4>) : cs == 2 ? go(k_pack_attn<T, D, NT, 2>) : go(k_pack_attn<T, D, NT, 1>);
  }
  if (int rc = check_combine(a, blocks)) return rc;
  const int grid = sms * S::kBlocks < kMaxRuns ? sms * S::kBlocks : kMaxRuns;
  a.start_cost = 1;
  a.joint = (int4 *)work;
  a.part = (float *)(work + tree_joint_bytes(a.s.batch, a.kv_heads, rows_max));
  a.part_ml = a.part + (int64_t)grid * 2 * S::kRows * D;
  if (int rc = launch("packed attention", k_pack_attn<T, D, NT, 0>, dim3(grid), kTreeThreads, S::kSmem, stream, true, 1, a, blocks)) return rc;
  return launch_combine<T, D>(a, sms, rows_max, S::kRows, stream);
}

template <typename T, int D>
int launch_pack_rows(const TreeArgs &a, int sms, int rows_max, char *work, cudaStream_t stream) {
  Shape best = shape_of<T, D, 1>(a, sms, rows_max);
  if (rows_max > 8) {
    const Shape two = shape_of<T, D, 2>(a, sms, rows_max), four = shape_of<T, D, 4>(a, sms, rows_max);
    if (two.us < best.us) best = two;
    if (rows_max > 16 && four.us < best.us) best = four;
  }
  if constexpr (sizeof(T) == 2) {
    if (rows_max > 16) {  // the workspace of fewer rows has no room for the parts of these
      const double tiles = tree_tiles(a), heads = (double)a.kv_heads * a.s.batch, unit = D == 64 ? 0.67 : 1;
      const double narrow = (rows_max + 127) / 128 * heads, wide = (rows_max + 255) / 256 * heads;  // segments
      auto waves = [&](double n) { return n <= sms ? 1. : std::fmax(1, (std::ceil(n / sms) + n / sms) / 2 * kMean); };
      const double t[4] = {waves(narrow) * tiles * 2.7 * unit + 8, narrow * tiles / sms * 3.6 * unit * kMean + 24,
                           waves(wide) * tiles * 4.4 * unit + 8, wide * tiles / sms * 4.4 * unit * kMean + 55};
      int i = 0;
      for (int j = 1; j < (rows_max > 128 ? 4 : 2); j++)
        if (t[j] < t[i]) i = j;
      if (t[i] < best.us)
        return i == 0   ? launch_tree_mma<T, D, false, false, true>(a, sms, rows_max, work, stream)
               : i == 1 ? launch_tree_mma<T, D, false, true, true>(a, sms, rows_max, work, stream)
               : i == 2 ? launch_tree_mma<T, D, true, false, true>(a, sms, rows_max, work, stream)
                        : launch_tree_mma<T, D, true, true, true>(a, sms, rows_max, work, stream);
    }
  }
  if (best.nt == 4) return launch_pack<T, D, 4>(a, best, sms, rows_max, work, stream);
  if (best.nt == 2) return launch_pack<T, D, 2>(a, best, sms, rows_max, work, stream);
  return launch_pack<T, D, 1>(a, best, sms, rows_max, work, stream);
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
