// C ABI of the packed cache's operators and of the rotation
// (include/ocrvl_cuda.h): argument checks and launches.
#include <cmath>

#include "../../include/ocrvl_cuda.h"
#include "entry.cuh"
#include "pack_attn.cuh"
#include "packed.cuh"
#include "rotate.cuh"
#include "tree_launch.cuh"

using namespace ocrvl;
using namespace ocrvl::paged;

namespace {

int check_packed(const ocrvl_packed_cache *c) {
  if (!c) return invalid("null cache");
  if (c->head_dim != 64 && c->head_dim != 128) return invalid("head_dim must be 64 or 128");
  if (c->num_kv_heads < 1 || c->num_layers < 1 || c->batch < 1 || c->max_pages < 1 || c->num_pages < 1)
    return invalid("cache dimensions must be positive");
  if (c->batch > 65535) return invalid("at most 65535 sequences a call");
  if (c->page_size < 16 || c->page_size & (c->page_size - 1)) return invalid("page_size must be a power of two of at least 16");
  if ((long long)c->max_pages * c->page_size > 0x40000000ll) return invalid("at most 2^30 positions a sequence");
  if (c->reserved) return invalid("reserved must be 0");
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->table) return invalid("null cache pointer");
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale))
    return invalid("k, v and their scales must be 16-byte aligned");
  for (long long s : {c->page_stride, c->layer_stride, c->head_stride})
    if (s < 0 || s % 16) return invalid("strides of the codes must be non-negative multiples of 16 bytes");
  for (long long s : {c->scale_page_stride, c->scale_layer_stride, c->scale_head_stride})
    if (s < 0 || s % 8) return invalid("strides of the scales must be non-negative multiples of 16 bytes");
  if (c->table_stride < (c->batch > 1 ? c->max_pages : 0)) return invalid("table_stride is shorter than a row");
  return OCRVL_OK;
}

Packed packed_of(const ocrvl_packed_cache *c) {
  Packed p;
  p.k = (char *)c->k, p.v = (char *)c->v, p.k_scale = (char *)c->k_scale, p.v_scale = (char *)c->v_scale;
  p.table = c->table;
  p.page = c->page_stride, p.layer = c->layer_stride, p.head = c->head_stride;
  p.scale_page = c->scale_page_stride * 2, p.scale_layer = c->scale_layer_stride * 2, p.scale_head = c->scale_head_stride * 2;
  p.table_stride = c->table_stride;
  p.shift = log2i(c->page_size), p.num_pages = c->num_pages, p.max_pages = c->max_pages;
  return p;
}

// What append and read share.
int check_move(const ocrvl_packed_cache *c, int type, int n_tokens, const int32_t *lens, const int32_t *indptr, const void *k,
               const void *v, int64_t kv_stride, int64_t kv_layer_stride) {
  if (int rc = check_packed(c)) return rc;
  const int es = elem_bytes(type);
  if (!es) return invalid("type must be f32, f16 or bf16");
  if (n_tokens < 0) return invalid("n_tokens must not be negative");
  if (!lens || !indptr || (n_tokens > 0 && (!k || !v))) return invalid("null argument");
  if (!aligned16(k) || !aligned16(v) || kv_stride * es % 16 || kv_layer_stride * es % 16 || kv_layer_stride < 0 ||
      kv_stride < (int64_t)c->num_kv_heads * c->head_dim)
    return invalid("k and v must be 16-byte aligned rows of num_kv_heads * head_dim elements");
  return OCRVL_OK;
}

PackArgs pack_args(const ocrvl_packed_cache *c, int type, int n_tokens, const int32_t *lens, const int32_t *indptr, const void *k,
                   const void *v, int64_t kv_stride, int64_t kv_layer_stride) {
  const long long es = elem_bytes(type);
  PackArgs a = {};
  a.c = packed_of(c);
  a.k = (char *)k, a.v = (char *)v, a.lens = lens, a.indptr = indptr;
  a.token = kv_stride * es, a.layer = kv_layer_stride * es;
  a.capacity = c->max_pages * c->page_size;
  a.layers = c->num_layers, a.batch = c->batch, a.kv_heads = c->num_kv_heads, a.n_tokens = n_tokens;
  return a;
}

// A warp 16 positions of a (layer, K or V, head); as many blocks as the longest sequence can use, or some waves of them.
int move_grid(const PackArgs &a, int most_tokens, dim3 *grid) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const long long rows = 2ll * a.layers * a.kv_heads;
  if (rows > 1 << 30) return invalid("too many layers and kv heads");
  const long long z = (rows + kPackWarps - 1) / kPackWarps < 1024 ? (rows + kPackWarps - 1) / kPackWarps : 1024;
  const long long chunks = (long long)most_tokens / kChunk + 2, most = (sms * 32 + a.batch * z - 1) / (a.batch * z);
  *grid = dim3((unsigned)(chunks < most ? chunks : most), a.batch, (unsigned)z);
  return OCRVL_OK;
}

// ---- attention ----------------------------------------------------------------

template <typename T, int D, int NT>
int launch_pack(TreeArgs a, int sms, int rows_max, char *work, cudaStream_t stream) {
  using S = PackShape<T, D, NT>;
  const int blocks = (rows_max + S::kRows - 1) / S::kRows;
  const long long segments = (long long)blocks * a.kv_heads * a.s.batch;
  if (segments > 1 << 24) return invalid("too many sequences and kv heads");
  // A cluster (or, for the shortest, a block) a segment where a block then has at most kFew
  // tiles of the longest cache and all clusters run at once: saves the second launch.
  constexpr int kFew = 4;
  const int tiles = tree_tiles(a);
  auto one = [&](auto kernel, int cs) {
    return launch("packed attention", kernel, dim3((unsigned)(segments * cs)), kTreeThreads, S::kSmem, stream, false, cs, a, blocks);
  };
  const int clustered = cluster_room(sms) * S::kBlocks;
  if (tiles > 2 && tiles <= 4 * kFew && segments * 4 <= clustered)
    return tiles > 4 && segments * 8 <= clustered ? one(k_pack_attn<T, D, NT, 8>, 8) : one(k_pack_attn<T, D, NT, 4>, 4);
  if (tiles > kFew && tiles <= 8 * kFew && segments * 8 <= clustered) return one(k_pack_attn<T, D, NT, 8>, 8);
  if (tiles <= kFew) return one(k_pack_attn<T, D, NT, 1>, 1);

  if (int rc = check_combine(a, blocks)) return rc;
  const int grid = sms * S::kBlocks < kMaxRuns ? sms * S::kBlocks : kMaxRuns;
  a.start_cost = 1;
  a.joint = (int4 *)work;
  a.part = (float *)(work + tree_joint_bytes(a.s.batch, a.kv_heads, rows_max));
  a.part_ml = a.part + (int64_t)grid * 2 * S::kRows * D;
  if (int rc = launch("packed attention", k_pack_attn<T, D, NT, 0>, dim3(grid), kTreeThreads, S::kSmem, stream, false, 1, a, blocks)) return rc;
  return launch_combine<T, D>(a, sms, rows_max, S::kRows, stream);
}

template <typename T, int D>
int launch_pack_rows(const TreeArgs &a, int sms, int rows_max, char *work, cudaStream_t stream) {
  if (rows_max <= 8) return launch_pack<T, D, 1>(a, sms, rows_max, work, stream);
  if (rows_max <= 16 || sizeof(T) == 2) return launch_pack<T, D, 2>(a, sms, rows_max, work, stream);
  if constexpr (sizeof(T) == 4)
    return launch_pack<T, D, 4>(a, sms, rows_max, work, stream);
  else
    return OCRVL_OK;
}

template <typename T>
int launch_pack_dim(const TreeArgs &a, int dim, int sms, int rows_max, char *work, cudaStream_t stream) {
  return dim == 128 ? launch_pack_rows<T, 128>(a, sms, rows_max, work, stream) : launch_pack_rows<T, 64>(a, sms, rows_max, work, stream);
}

template <typename T, int V, int NORM>
int launch_rotate(RotateArgs &a, int sms, cudaStream_t stream) {
  a.lanes = a.pairs / V + (a.dim - 2 * a.pairs) / (2 * V);
  a.at_once = 32 / a.lanes, a.lane_factor = (65536 + a.lanes - 1) / a.lanes, a.one_dim = 1.f / a.dim;
  // Warps a token: one, or as many as its heads keep busy while the GPU is not full.
  const int steps = (a.heads + a.at_once - 1) / a.at_once, blocks = (a.n_tokens + kRotateWarps - 1) / kRotateWarps;
  const int room = sms * 2 / blocks, share = room < 1 ? 1 : room < steps ? room : steps;
  const dim3 grid(blocks, share);
  auto go = [&](auto kernel) { return launch("rotate", kernel, grid, kRotateWarps * 32, 0, stream, false, 1, a); };
  if (a.lanes == 8) return go(k_rotate<T, V, NORM, 8>);
  if (a.lanes == 16) return go(k_rotate<T, V, NORM, 16>);
  return go(k_rotate<T, V, NORM, 0>);
}

template <typename T, int V>
int launch_rotate_norm(RotateArgs &a, int norm, int sms, cudaStream_t stream) {
  if (norm == 0) return launch_rotate<T, V, 0>(a, sms, stream);
  if constexpr (sizeof(T) == 2)
    if (norm == 1) return launch_rotate<T, V, 1>(a, sms, stream);
  return launch_rotate<T, V, 2>(a, sms, stream);
}

}  // namespace

extern "C" {

int ocrvl_op_packed_append(const ocrvl_packed_cache *c, int type, int n_tokens, const int32_t *lens, const int32_t *indptr,
                           const int32_t *path, const int32_t *n_path, int max_path, const void *k, const void *v,
                           int64_t kv_stride, int64_t kv_layer_stride, int32_t *new_lens, void *stream) {
  if (int rc = check_move(c, type, n_tokens, lens, indptr, k, v, kv_stride, kv_layer_stride)) return rc;
  if (path && (!n_path || max_path < 1)) return invalid("a path needs n_path and max_path >= 1");
  if (!new_lens) return invalid("null argument");
  if (new_lens == lens) return invalid("new_lens must not be lens");
  PackArgs a = pack_args(c, type, n_tokens, lens, indptr, k, v, kv_stride, kv_layer_stride);
  a.path = path, a.n_path = n_path, a.max_path = max_path, a.new_lens = new_lens;
  dim3 grid;
  if (int rc = move_grid(a, path ? max_path : n_tokens, &grid)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto wide, auto narrow) {
    return launch("append, packed", c->head_dim == 128 ? wide : narrow, grid, kPackThreads, 0, st, false, 1, a);
  };
  if (type == OCRVL_F32) return go(k_packed_append<float, 128>, k_packed_append<float, 64>);
  if (type == OCRVL_F16) return go(k_packed_append<__half, 128>, k_packed_append<__half, 64>);
  return go(k_packed_append<__nv_bfloat16, 128>, k_packed_append<__nv_bfloat16, 64>);
}

int ocrvl_op_packed_read(const ocrvl_packed_cache *c, int type, int n_tokens, const int32_t *lens, const int32_t *indptr,
                         void *k, void *v, int64_t kv_stride, int64_t kv_layer_stride, void *stream) {
  if (int rc = check_move(c, type, n_tokens, lens, indptr, k, v, kv_stride, kv_layer_stride)) return rc;
  if (n_tokens == 0) return OCRVL_OK;
  const PackArgs a = pack_args(c, type, n_tokens, lens, indptr, k, v, kv_stride, kv_layer_stride);
  dim3 grid;
  if (int rc = move_grid(a, n_tokens, &grid)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto wide, auto narrow) {
    return launch("read, packed", c->head_dim == 128 ? wide : narrow, grid, kPackThreads, 0, st, false, 1, a);
  };
  if (type == OCRVL_F32) return go(k_packed_read<float, 128>, k_packed_read<float, 64>);
  if (type == OCRVL_F16) return go(k_packed_read<__half, 128>, k_packed_read<__half, 64>);
  return go(k_packed_read<__nv_bfloat16, 128>, k_packed_read<__nv_bfloat16, 64>);
}

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

int ocrvl_op_rotate(const ocrvl_rotary *r, int type, int n_tokens, const int32_t *pos, int64_t pos_stride, int heads,
                    const void *q, int64_t q_stride, void *q_out, int64_t q_out_stride, int kv_heads, const void *k,
                    int64_t k_stride, void *k_out, int64_t k_out_stride, int weight_type, const void *q_weight,
                    const void *k_weight, float eps, void *stream) {
  if (!r) return invalid("null rotary");
  const int es = elem_bytes(type), D = r->head_dim, P = r->pairs;
  if (!es) return invalid("type must be f32, f16 or bf16");
  if (D < 8 || D > 256 || D % 8) return invalid("head_dim must be a multiple of 8, at most 256");
  if (P < 4 || P % 4 || 2 * P > D) return invalid("pairs must be a multiple of 4, at most half of head_dim");
  if (r->num_axes < 1 || r->num_axes > 8) return invalid("num_axes must be 1..8");
  if (r->neighbours != 0 && r->neighbours != 1) return invalid("neighbours must be 0 or 1");
  for (int p = 0; p < P; p++) {
    if (r->axis[p] >= r->num_axes) return invalid("a pair's axis must be one of num_axes");
    if (!std::isfinite(r->freq[p])) return invalid("freq must be finite");
  }
  if (n_tokens < 0) return invalid("n_tokens must not be negative");
  if (!k) kv_heads = 0;
  if (heads < 1 || heads > 65536 || kv_heads < (k ? 1 : 0) || kv_heads > 65536) return invalid("heads must be 1..65536");
  if (n_tokens == 0) return OCRVL_OK;
  if (!pos || !q || !q_out || (k && !k_out)) return invalid("null argument");
  if (pos_stride < r->num_axes) return invalid("pos must have num_axes entries a token");
  auto rows = [&](const void *p, int64_t stride, int n) { return aligned16(p) && stride * es % 16 == 0 && stride >= (int64_t)n * D; };
  if (!rows(q, q_stride, heads) || !rows(q_out, q_out_stride, heads) ||
      (k && (!rows(k, k_stride, kv_heads) || !rows(k_out, k_out_stride, kv_heads))))
    return invalid("q, k and what they become must be 16-byte aligned rows of heads * head_dim elements");
  if ((q_out == q && q_out_stride != q_stride) || (k && k_out == k && k_out_stride != k_stride))
    return invalid("in place, the strides must be the same");
  if (k && (q_weight != nullptr) != (k_weight != nullptr)) return invalid("q_weight and k_weight go together");
  if (q_weight) {
    if (weight_type != OCRVL_F32 && weight_type != type) return invalid("weight_type must be f32 or q's type");
    if (!aligned16(q_weight) || !aligned16(k_weight)) return invalid("weights must be 16-byte aligned");
    if (!(eps >= 0.f) || std::isinf(eps)) return invalid("eps must be finite and not negative");
  }
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  RotateArgs a = {};
  a.q = (const char *)q, a.k = (const char *)k, a.q_out = (char *)q_out, a.k_out = (char *)k_out;
  a.q_weight = q_weight, a.k_weight = k_weight;
  a.pos = pos, a.pos_stride = pos_stride;
  a.q_stride = q_stride * es, a.k_stride = k_stride * es, a.q_out_stride = q_out_stride * es, a.k_out_stride = k_out_stride * es;
  a.n_tokens = n_tokens, a.heads = heads, a.kv_heads = kv_heads, a.dim = D, a.pairs = P, a.neighbours = r->neighbours, a.eps = eps;
  for (int p = 0; p < P; p++) a.turns[p] = r->freq[p] * 0.15915494309189535, a.axis[p] = r->axis[p];
  const int norm = !q_weight ? 0 : weight_type == OCRVL_F32 ? 2 : 1;
  cudaStream_t st = (cudaStream_t)stream;
  if (type == OCRVL_F32) return launch_rotate_norm<float, 4>(a, norm, sms, st);
  const bool eight = P % 8 == 0 && (D - 2 * P) % 16 == 0;
  if (type == OCRVL_F16) return eight ? launch_rotate_norm<__half, 8>(a, norm, sms, st) : launch_rotate_norm<__half, 4>(a, norm, sms, st);
  return eight ? launch_rotate_norm<__nv_bfloat16, 8>(a, norm, sms, st) : launch_rotate_norm<__nv_bfloat16, 4>(a, norm, sms, st);
}

}  // extern "C"
