// C ABI of the packed cache's append and read and of the rotation
// (include/ocrvl_cuda.h): argument checks and launches.
#include <cmath>

#include "../../include/ocrvl_cuda.h"
#include "packed.cuh"
#include "packed_entry.cuh"
#include "rotate.cuh"

using namespace ocrvl;
using namespace ocrvl::paged;

namespace {

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

// A warp 16 positions of a (layer, K or V, head) at a time; as many blocks as twice an even share of the tokens can use (a
// sequence has `most_tokens` at most, all have n_tokens), or the GPU holds `waves` times.
int move_grid(const PackArgs &a, int most_tokens, int waves, dim3 *grid) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const long long rows = 2ll * a.layers * a.kv_heads;
  if (rows > 1 << 30) return invalid("too many layers and kv heads");
  const long long z = (rows + kPackWarps - 1) / kPackWarps < 1024 ? (rows + kPackWarps - 1) / kPackWarps : 1024;
  const long long chunks = (long long)most_tokens / kChunk + 2, even = 2 * ((long long)a.n_tokens / a.batch / kChunk + 1);
  const long long most = (sms * 8 * waves + a.batch * z - 1) / (a.batch * z), x = chunks < even ? chunks : even;
  *grid = dim3((unsigned)(x < most ? x : most), a.batch, (unsigned)z);
  return OCRVL_OK;
}

template <typename T, int V, int NORM>
int launch_rotate(RotateArgs &a, int sms, cudaStream_t stream) {
  a.lanes = a.pairs / V + (a.dim - 2 * a.pairs) / (2 * V);
  a.at_once = 32 / a.lanes, a.lane_factor = (65536 + a.lanes - 1) / a.lanes, a.one_dim = 1.f / a.dim;
  // Rows a batch: all that the ring holds, or fewer while the GPU is not full, so that a token's batches keep
  // several warps busy.
  const int full = sms * kRotateBlocks, blocks = (a.n_tokens - 1) / kRotateWarps + 1, room = full / blocks;
  auto batches = [&](int rows) { return (rows + a.at_once * a.steps - 1) / (a.at_once * a.steps); };
  a.steps = kRotateSteps;
  while (a.steps > 1 && batches(a.heads) + batches(a.kv_heads) < room) a.steps--;
  a.q_batches = batches(a.heads), a.batches = a.q_batches + batches(a.kv_heads);
  const int share = room < 1 ? 1 : room < a.batches ? room : a.batches;
  const dim3 grid(blocks < full ? blocks : full, share);
  auto go = [&](auto kernel) { return launch("rotate", kernel, grid, kRotateWarps * 32, kRotateSmem<T, V>, stream, true, 1, a); };
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
  if (int rc = move_grid(a, path ? max_path : n_tokens, 8, &grid)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto wide, auto narrow) {
    return launch("append, packed", c->head_dim == 128 ? wide : narrow, grid, kPackThreads, 0, st, true, 1, a);
  };
  if (type == OCRVL_F32) return go(k_packed_append<float, 128>, k_packed_append<float, 64>);
  if (type == OCRVL_F16) return go(k_packed_append<__half, 128>, k_packed_append<__half, 64>);
  return go(k_packed_append<__nv_bfloat16, 128>, k_packed_append<__nv_bfloat16, 64>);
}

int ocrvl_op_packed_read(const ocrvl_packed_cache *c, int type, int n_tokens, const int32_t *lens, const int32_t *indptr,
                         void *k, void *v, int64_t kv_stride, int64_t kv_layer_stride, void *stream) {
  if (int rc = check_move(c, type, n_tokens, lens, indptr, k, v, kv_stride, kv_layer_stride)) return rc;
  if (n_tokens == 0) return OCRVL_OK;
  const int64_t row = (int64_t)c->num_kv_heads * c->head_dim, tokens = (n_tokens - 1) * kv_stride + row;
  if (k == v || (c->num_layers > 1 && kv_layer_stride < tokens && (kv_layer_stride < row || kv_stride < (c->num_layers - 1) * kv_layer_stride + row)))
    return invalid("what is read must not share memory (of K and V, of two layers)");
  const PackArgs a = pack_args(c, type, n_tokens, lens, indptr, k, v, kv_stride, kv_layer_stride);
  dim3 grid;
  if (int rc = move_grid(a, n_tokens, 4, &grid)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto wide, auto narrow) {
    return launch("read, packed", c->head_dim == 128 ? wide : narrow, grid, kPackThreads, 0, st, true, 1, a);
  };
  if (type == OCRVL_F32) return go(k_packed_read<float, 128>, k_packed_read<float, 64>);
  if (type == OCRVL_F16) return go(k_packed_read<__half, 128>, k_packed_read<__half, 64>);
  return go(k_packed_read<__nv_bfloat16, 128>, k_packed_read<__nv_bfloat16, 64>);
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
