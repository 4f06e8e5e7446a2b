// C ABI of the paged-cache operators (include/ocrvl_cuda.h): argument checks
// and launches.
#include <cmath>
#include <cstdio>

#include "../../include/ocrvl_cuda.h"
#include "attn_mass.cuh"
#include "mass_mma.cuh"
#include "capi.h"
#include "kv_move.cuh"
#include "tree_attn.cuh"
#include "tree_mma.cuh"

using namespace ocrvl;
using namespace ocrvl::paged;

namespace {

int invalid(const char *msg) { return api_fail(OCRVL_E_INVALID, msg); }

int cuda_fail(const char *what, cudaError_t e) {
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
  return api_fail(OCRVL_E_CUDA, msg);
}

#define PCK(call)                                        \
  do {                                                   \
    cudaError_t e_ = (call);                             \
    if (e_ != cudaSuccess) return cuda_fail(#call, e_);  \
  } while (0)

int elem_bytes(int type) { return type == OCRVL_F32 ? 4 : type == OCRVL_F16 || type == OCRVL_BF16 ? 2 : 0; }

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int check_cache(const ocrvl_kv_cache *c) {
  if (!c) return invalid("null cache");
  const int es = elem_bytes(c->type);
  if (!es) return invalid("cache type must be f32, f16 or bf16");
  if (c->head_dim != 64 && c->head_dim != 128) return invalid("head_dim must be 64 or 128");
  if (c->num_kv_heads < 1 || c->num_layers < 1 || c->batch < 1 || c->max_pages < 1 || c->num_pages < 1)
    return invalid("cache dimensions must be positive");
  if (c->batch > 65535) return invalid("at most 65535 sequences a call");
  if (c->page_size < 16 || c->page_size & (c->page_size - 1)) return invalid("page_size must be a power of two of at least 16");
  if ((long long)c->max_pages * c->page_size > 0x40000000ll) return invalid("at most 2^30 positions a sequence");
  if (!c->k || !c->v || !c->table) return invalid("null cache pointer");
  if (!aligned16(c->k) || !aligned16(c->v)) return invalid("k and v must be 16-byte aligned");
  const long long strides[] = {c->page_stride, c->layer_stride, c->head_stride, c->token_stride};
  for (long long s : strides)
    if (s < 0 || s * es % 16) return invalid("cache strides must be non-negative multiples of 16 bytes");
  if (c->token_stride < c->head_dim || c->token_stride * es > 0x7fffffffll / 16) return invalid("token_stride out of range");
  if (c->table_stride < (c->batch > 1 ? c->max_pages : 0)) return invalid("table_stride is shorter than a row");
  return OCRVL_OK;
}

int log2i(int x) {
  int n = 0;
  while (1 << n < x) n++;
  return n;
}

Cache layer_of(const ocrvl_kv_cache *c, int layer) {
  const long long es = elem_bytes(c->type);
  Cache r;
  r.k = (const char *)c->k + layer * c->layer_stride * es;
  r.v = (const char *)c->v + layer * c->layer_stride * es;
  r.table = c->table;
  r.page_bytes = c->page_stride * es;
  r.head_bytes = c->head_stride * es;
  r.table_stride = c->table_stride;
  r.token_bytes = (int)(c->token_stride * es);
  r.max_pages = c->max_pages;
  r.num_pages = c->num_pages;
  r.page_shift = log2i(c->page_size);
  return r;
}

// The streaming multiprocessors of the current device.
int sm_count(int *out) {
  static int known[64];  // 0: not asked yet (a race stores the same value twice)
  int dev = 0;
  PCK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return invalid("device index out of range");
  if (!known[dev]) {
    int n = 0;
    PCK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    known[dev] = n;
  }
  *out = known[dev];
  return OCRVL_OK;
}

// Blocks that run at once in clusters of up to eight, one an SM: clusters lie within
// one of the GPU's partitions, so some SMs stay over (15 clusters of eight
// were resident on 148 SMs).
int cluster_room(int sms) { return sms * 4 / 5; }

// Bytes of dynamic shared memory: of this call, and the most that any call of
// the kernel takes.  The limit that a kernel has leave for is shared by all host threads, so it
// is always set to the same value.
struct Smem {
  int bytes, most;
  Smem(int all) : bytes(all), most(all) {}
  Smem(int bytes_, int most_) : bytes(bytes_), most(most_) {}
};

// Launches with dynamic shared memory; dependent: may start
// before the kernel launched just before it on the stream ends (both wait for
// it with griddepcontrol).
template <typename... Params, typename... Args>
int launch(const char *name, void (*kernel)(Params...), dim3 grid, int threads, Smem smem, cudaStream_t stream, bool dependent,
           int cluster, Args... args) {
  if (smem.bytes > 24 * 1024) {  // with a kernel's static share possibly past the 48 KB that need no leave
    cudaError_t e = cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem.most);
    if (e != cudaSuccess) return cuda_fail(name, e);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem.bytes;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (dependent) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    n++;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return e == cudaSuccess ? OCRVL_OK : cuda_fail(name, e);
}

int check_tokens(const ocrvl_kv_cache *c, int layer, int heads, int n_tokens, int max_draft, const int32_t *lens,
                 const int32_t *indptr, const void *q, int64_t q_stride, float scale) {
  if (int rc = check_cache(c)) return rc;
  const int es = elem_bytes(c->type);
  if (layer < 0 || layer >= c->num_layers) return invalid("layer outside the cache");
  if (heads < 1 || heads % c->num_kv_heads || heads / c->num_kv_heads > 16)
    return invalid("heads must be a multiple of num_kv_heads, at most 16 times it");
  if (n_tokens < 0) return invalid("n_tokens must not be negative");
  if (max_draft < 1 || max_draft > 64) return invalid("max_draft must be 1..64");
  if (!lens || !indptr || (n_tokens > 0 && !q)) return invalid("null argument");
  if (!aligned16(q) || q_stride * es % 16 || q_stride < (int64_t)heads * c->head_dim)
    return invalid("q must be 16-byte aligned rows of heads * head_dim elements");
  if (!std::isfinite(scale)) return invalid("scale must be finite");
  return OCRVL_OK;
}

// ---- tree attention ----------------------------------------------------------

// The workspace: two parts a block, and 16 bytes a segment in front of them.
int64_t tree_joint_bytes(int batch, int kv_heads, int rows) { return ((int64_t)batch * kv_heads * ((rows + 7) / 8) * 16 + 127) / 128 * 128; }
int64_t tree_work_bytes(const ocrvl_kv_cache *c, int sms, int rows) {
  const int64_t parts = 2ll * sms * (c->type == OCRVL_F32 || rows <= 16 ? 2 * 32 : rows > 128 ? 256 : 128);
  return tree_joint_bytes(c->batch, c->num_kv_heads, rows) + parts * (c->head_dim + 2) * 4;
}

// Tiles of the longest cache and of its drafts.
int tree_tiles(const TreeArgs &a) { return (a.s.capacity + a.s.max_draft + kChunk - 1 + kChunk * kTileChunks - 1) / (kChunk * kTileChunks); }

// What a call whose runs are joined must keep to, asked before its first launch.
int check_combine(const TreeArgs &a, int blocks) { return (long long)blocks * a.kv_heads > 65535 ? invalid("too many kv heads") : OCRVL_OK; }

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
template <typename T, int D, bool WIDE, bool SPLIT>
int launch_tree_mma(TreeArgs a, int sms, int rows_max, char *work, cudaStream_t stream) {
  using S = MmaShape<D, WIDE>;
  const int blocks = (rows_max + S::kRows - 1) / S::kRows;
  const long long segments = (long long)blocks * a.kv_heads * a.s.batch;
  if (segments > 1 << 24) return invalid("too many sequences and kv heads");
  if constexpr (!SPLIT) {
    return launch("tree attention", k_tree_mma<T, D, WIDE, false>, dim3((unsigned)segments), kMmaThreads, S::kSmem, stream, false, 1, a, blocks);
  } else {
    if (int rc = check_combine(a, blocks)) return rc;
    const int grid = sms < kMaxRuns ? sms : kMaxRuns;
    a.start_cost = 3;
    a.joint = (int4 *)work;
    a.part = (float *)(work + tree_joint_bytes(a.s.batch, a.kv_heads, rows_max));
    a.part_ml = a.part + (int64_t)grid * 2 * S::kRows * D;
    if (int rc = launch("tree attention", k_tree_mma<T, D, WIDE, true>, dim3(grid), kMmaThreads, S::kSmem, stream, false, 1, a, blocks)) return rc;
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
    return narrow_whole <= narrow_runs ? launch_tree_mma<T, D, false, false>(a, sms, rows_max, work, stream)
                                       : launch_tree_mma<T, D, false, true>(a, sms, rows_max, work, stream);
  if (narrow_whole <= wide_whole && narrow_whole <= wide_runs) return launch_tree_mma<T, D, false, false>(a, sms, rows_max, work, stream);
  return wide_whole <= wide_runs ? launch_tree_mma<T, D, true, false>(a, sms, rows_max, work, stream)
                                 : launch_tree_mma<T, D, true, true>(a, sms, rows_max, work, stream);
}

template <typename T, int D, int NT>
int launch_tree(TreeArgs a, int sms, int rows_max, char *work, cudaStream_t stream) {
  using S = TreeShape<T, D, NT>;
  const int blocks = (rows_max + S::kRows - 1) / S::kRows;
  const long long segments = (long long)blocks * a.kv_heads * a.s.batch;
  if (segments > 1 << 24) return invalid("too many sequences and kv heads");
  // A cluster (or, for the shortest, a block) a segment where a block then has at most kFew
  // tiles of the longest cache and all clusters run at once: saves the second launch.
  constexpr int kFew = 4;
  const int tiles = tree_tiles(a);
  auto one = [&](auto kernel, int cs) {
    return launch("tree attention", kernel, dim3((unsigned)(segments * cs)), kTreeThreads, S::kSmem, stream, false, cs, a, blocks);
  };
  const int clustered = cluster_room(sms) * S::kBlocks;
  if (tiles > 2 && tiles <= 4 * kFew && segments * 4 <= clustered)
    return tiles > 4 && segments * 8 <= clustered ? one(k_tree_attn<T, D, NT, 8>, 8) : one(k_tree_attn<T, D, NT, 4>, 4);
  if (tiles > kFew && tiles <= 8 * kFew && segments * 8 <= clustered) return one(k_tree_attn<T, D, NT, 8>, 8);
  if (tiles <= kFew) return one(k_tree_attn<T, D, NT, 1>, 1);

  if (int rc = check_combine(a, blocks)) return rc;
  const int grid = sms * S::kBlocks < kMaxRuns ? sms * S::kBlocks : kMaxRuns;
  a.start_cost = 1;
  a.joint = (int4 *)work;
  a.part = (float *)(work + tree_joint_bytes(a.s.batch, a.kv_heads, rows_max));
  a.part_ml = a.part + (int64_t)grid * 2 * S::kRows * D;
  if (int rc = launch("tree attention", k_tree_attn<T, D, NT, 0>, dim3(grid), kTreeThreads, S::kSmem, stream, false, 1, a, blocks)) return rc;
  return launch_combine<T, D>(a, sms, rows_max, S::kRows, stream);
}

// Rows a block.  Eight or sixteen where there are no more, or where the calls'
// tiles are so few that the GPU is not filled otherwise: a warp's pass over
// its chunk takes 2 us with 8 f32 rows, 7 with 32 (one sequence of 20 positions
// and 4 drafts: 6.3 us against 8.3 with 16 and 12.4 with 32).  Else 32 for f32 (the
// accumulators' limit), and the fifth generation's products for 16 bits.
template <typename T, int D>
int launch_tree_rows(const TreeArgs &a, int sms, int rows_max, char *work, cudaStream_t stream) {
  const int room = sizeof(T) == 4 ? sms : 2 * sms;  // blocks that run at once
  auto few = [&](int rows) { return (long long)((rows_max + rows - 1) / rows) * a.kv_heads * a.s.batch * tree_tiles(a) * 2 <= 3 * room; };
  if (rows_max <= 8 || few(8)) return launch_tree<T, D, 1>(a, sms, rows_max, work, stream);
  if (rows_max <= 16 || few(16)) return launch_tree<T, D, 2>(a, sms, rows_max, work, stream);
  if constexpr (sizeof(T) == 4)
    return launch_tree<T, D, 4>(a, sms, rows_max, work, stream);
  else
    return launch_tree_mma_shape<T, D>(a, sms, rows_max, work, stream);
}

template <typename T>
int launch_tree_dim(const TreeArgs &a, int dim, int sms, int rows_max, char *work, cudaStream_t stream) {
  return dim == 128 ? launch_tree_rows<T, 128>(a, sms, rows_max, work, stream) : launch_tree_rows<T, 64>(a, sms, rows_max, work, stream);
}

template <typename T, int D>
int launch_mass(const MassArgs &a, int sms, cudaStream_t stream) {
  const int width = a.out_width < a.s.capacity ? a.out_width : a.s.capacity, row_tiles = (a.s.max_draft * a.group + 7) / 8;
  const long long tiles = (long long)a.s.batch * a.kv_heads * ((width + kMassWarps * kChunk - 1) / (kMassWarps * kChunk));
  // Up to eight rows (one token of up to eight heads, say) stay in registers.  More of 16 bits go
  // to the fifth generation's products (4 sequences of 8,448, 32 drafts: 18.5 us here, 12.7 there),
  // and so do eight where the blocks have many tiles each (bf16, 64 of 4,000: 40 and 31
  // us, one of 131,072: 18.7 and 16.6; but 16 of 2,000: 10.4 and 11.0, one of 700: 6.5 and 8.2).
  if constexpr (sizeof(T) == 2) {
    if (row_tiles > 1 || tiles > 6ll * sms)
      return launch("attention mass", k_mass_mma<T, D>, dim3(sms), kMmaThreads, MassMmaShape<D>::kSmem, stream, false, 1, a);
    return launch("attention mass", k_attn_mass<T, D, true>, dim3(sms), kMassThreads, MassShape<T, D, true>::kSmem, stream, false, 1, a, 1);
  } else {
    if (row_tiles == 1)
      return launch("attention mass", k_attn_mass<T, D, true>, dim3(sms), kMassThreads, MassShape<T, D, true>::kSmem, stream, false, 1, a, 1);
    // A cluster a run, each block with a part of the rows, while all the call's tiles of 128
    // positions are in one wave of blocks and a part has about four tiles of eight rows: one
    // sequence of 700, 64 drafts: 68 us alone, 41, 25 and 20.8 in clusters of 2, 4 and 8; of
    // 3000: 68 and 41, but 54 in 4, now two waves; 5 drafts: 13.5 and 12.3.
    int parts = 1;
    while (parts < 8 && tiles * parts * 2 <= (parts == 1 ? sms : cluster_room(sms)) && row_tiles + 3 >= parts * 2 * 4) parts *= 2;
    return launch("attention mass", k_attn_mass<T, D, false>, dim3(sms / parts * parts), kMassThreads, MassShape<T, D, false>::kSmem,
                  stream, false, parts, a, parts);
  }
}

template <int CS, int THREADS>
int launch_select(const SelectArgs &a, int rows, cudaStream_t stream) {
  const dim3 grid((unsigned)(rows * CS));
  const long long step = THREADS * 4, n = (((a.width + CS - 1) / CS + 3) / 4 * 4 + step - 1) / step * step;
  return n <= kSelStage ? launch("select", k_kv_select<CS, true, THREADS>, grid, THREADS, Smem((int)n * 4, kSelStage * 4), stream, false, CS, a)
                        : launch("select", k_kv_select<CS, false, THREADS>, grid, THREADS, 0, stream, false, CS, a);
}

int check_move(const ocrvl_kv_cache *from, const ocrvl_kv_cache *to, const int32_t *idx, int keep) {
  if (int rc = check_cache(from)) return rc;
  if (int rc = check_cache(to)) return rc;
  if (from->type != to->type || from->head_dim != to->head_dim || from->num_kv_heads != to->num_kv_heads ||
      from->num_layers != to->num_layers || from->batch != to->batch)
    return invalid("the caches must have the same type, head_dim, heads, layers and batch");
  if (keep < 1 || keep > 65535 * kMoveRows) return invalid("keep must be 1..2,097,120");
  const long long room = (long long)to->max_pages * to->page_size, held = (long long)from->max_pages * from->page_size;
  if (keep > room && held > room) return invalid("to has no room for the positions that are kept");
  if (!idx) return invalid("null argument");
  if ((long long)from->num_layers * from->batch * from->num_kv_heads > 1 << 24) return invalid("too many rows");
  return OCRVL_OK;
}

// dependent: right behind the kernel that writes idx
int compact(const ocrvl_kv_cache *from, const ocrvl_kv_cache *to, const int32_t *idx, int keep, cudaStream_t st, bool dependent) {
  if (int rc = check_move(from, to, idx, keep)) return rc;
  const long long rows = (long long)from->num_layers * from->batch * from->num_kv_heads;
  const long long es = elem_bytes(from->type);
  CompactArgs a;
  a.src_k = (const char *)from->k, a.src_v = (const char *)from->v;
  a.dst_k = (char *)to->k, a.dst_v = (char *)to->v;
  a.src_table = from->table, a.dst_table = to->table, a.idx = idx;
  a.src_page = from->page_stride * es, a.dst_page = to->page_stride * es;
  a.src_layer = from->layer_stride * es, a.dst_layer = to->layer_stride * es;
  a.src_head = from->head_stride * es, a.dst_head = to->head_stride * es;
  a.src_table_stride = from->table_stride, a.dst_table_stride = to->table_stride;
  a.src_token = (int)(from->token_stride * es), a.dst_token = (int)(to->token_stride * es);
  a.src_shift = log2i(from->page_size), a.dst_shift = log2i(to->page_size);
  a.src_pages = from->num_pages, a.dst_pages = to->num_pages;
  a.src_max = from->max_pages, a.dst_max = to->max_pages;
  a.layers = from->num_layers, a.batch = from->batch, a.kv_heads = from->num_kv_heads, a.keep = keep;
  a.row_bytes = (int)(from->head_dim * es);
  if (from->k == to->k || from->v == to->v) {
    if (from->table == to->table) {
      if (from->v != to->v || from->k != to->k || a.src_page != a.dst_page || a.src_layer != a.dst_layer ||
          a.src_head != a.dst_head || a.src_token != a.dst_token || a.src_shift != a.dst_shift ||
          a.src_table_stride != a.dst_table_stride)
        return invalid("in place, both descriptors must be the same");
      return launch("compact in place", k_kv_compact_in_place, dim3((unsigned)rows, a.row_bytes / 64, 2), kMoveThreads, 0, st,
                    dependent, 1, a);
    }
  }
  const int blocks = (keep + kMoveRows - 1) / kMoveRows;
  auto kernel = a.row_bytes == 512 ? k_kv_compact<512> : a.row_bytes == 256 ? k_kv_compact<256> : k_kv_compact<128>;
  return launch("compact", kernel, dim3((unsigned)rows, blocks), kMoveThreads, 0, st, dependent, 1, a);
}

}  // namespace

extern "C" {

int ocrvl_op_tree_attn_workspace(const ocrvl_kv_cache *c, int heads, int max_draft, int64_t *bytes) {
  if (!bytes) return invalid("null argument");
  if (int rc = check_cache(c)) return rc;
  if (heads < 1 || heads % c->num_kv_heads || max_draft < 1 || max_draft > 64) return invalid("heads must be a multiple of num_kv_heads, max_draft 1..64");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  *bytes = tree_work_bytes(c, sms, heads / c->num_kv_heads * max_draft);
  return OCRVL_OK;
}

int ocrvl_op_tree_attn(const ocrvl_kv_cache *c, int layer, int heads, int n_tokens, int max_draft, const int32_t *lens,
                       const int32_t *indptr, const int64_t *mask, const void *q, int64_t q_stride, const void *k,
                       const void *v, int64_t kv_stride, float scale, void *out, int64_t out_stride, float *lse, void *work,
                       int64_t work_bytes, void *stream) {
  if (int rc = check_tokens(c, layer, heads, n_tokens, max_draft, lens, indptr, q, q_stride, scale)) return rc;
  const int es = elem_bytes(c->type), D = c->head_dim;
  if (n_tokens == 0) return OCRVL_OK;
  if (!mask || !k || !v || !out || !work) return invalid("null argument");
  if (!aligned16(k) || !aligned16(v) || kv_stride * es % 16 || kv_stride < (int64_t)c->num_kv_heads * D)
    return invalid("k and v must be 16-byte aligned rows of num_kv_heads * head_dim elements");
  if (kv_stride * es > 0x7fffffff) return invalid("kv_stride is too large");
  if (!aligned16(out) || out_stride * es % 16 || out_stride < (int64_t)heads * D)
    return invalid("out must be 16-byte aligned rows of heads * head_dim elements");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  if (((uintptr_t)work & 127) || work_bytes < tree_work_bytes(c, sms, heads / c->num_kv_heads * max_draft)) return invalid("work is too small or not 128-byte aligned");
  TreeArgs a;
  a.c = layer_of(c, layer);
  a.s = Seqs{lens, indptr, c->batch, n_tokens, max_draft, c->max_pages * c->page_size};
  a.kv_heads = c->num_kv_heads;
  a.group = heads / c->num_kv_heads;
  a.q = q, a.dk = k, a.dv = v, a.out = out;
  a.q_stride = q_stride, a.kv_stride = kv_stride, a.out_stride = out_stride;
  a.mask = (const long long *)mask;
  a.scale = scale * kLog2e;
  a.lse = lse;
  const int rows_max = max_draft * a.group;
  cudaStream_t st = (cudaStream_t)stream;
  if (c->type == OCRVL_F32) return launch_tree_dim<float>(a, D, sms, rows_max, (char *)work, st);
  if (c->type == OCRVL_F16) return launch_tree_dim<__half>(a, D, sms, rows_max, (char *)work, st);
  return launch_tree_dim<__nv_bfloat16>(a, D, sms, rows_max, (char *)work, st);
}

int ocrvl_op_attn_mass(const ocrvl_kv_cache *c, int layer, int heads, int n_tokens, int max_draft, const int32_t *lens,
                       const int32_t *indptr, const int64_t *counted, const void *q, int64_t q_stride, const float *lse,
                       float scale, float decay, const float *acc, int acc_width, int64_t acc_stride, float *acc_out,
                       int out_width, int64_t out_stride, void *stream) {
  if (int rc = check_tokens(c, layer, heads, n_tokens, max_draft, lens, indptr, q, q_stride, scale)) return rc;
  if (!acc_out || (n_tokens > 0 && !lse)) return invalid("null argument");
  if (!std::isfinite(decay)) return invalid("decay must be finite");
  if (out_width < 1 || out_stride < out_width) return invalid("acc_out rows must hold out_width >= 1 values");
  if (acc && (acc_width < 0 || acc_stride < acc_width)) return invalid("acc rows must hold acc_width values");
  if (acc == acc_out && acc_stride != out_stride) return invalid("acc in place needs the stride of acc_out");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  MassArgs a;
  a.c = layer_of(c, layer);
  a.s = Seqs{lens, indptr, c->batch, n_tokens, max_draft, c->max_pages * c->page_size};
  a.kv_heads = c->num_kv_heads;
  a.group = heads / c->num_kv_heads;
  a.q = q, a.q_stride = q_stride, a.counted = (const long long *)counted, a.lse = lse;
  a.scale = scale * kLog2e, a.decay = decay;
  a.acc = acc, a.out = acc_out;
  a.acc_stride = acc_stride, a.out_stride = out_stride;
  a.acc_width = acc ? acc_width : 0, a.out_width = out_width;
  cudaStream_t st = (cudaStream_t)stream;
  const bool wide = c->head_dim == 128;
  if (c->type == OCRVL_F32) return wide ? launch_mass<float, 128>(a, sms, st) : launch_mass<float, 64>(a, sms, st);
  if (c->type == OCRVL_F16) return wide ? launch_mass<__half, 128>(a, sms, st) : launch_mass<__half, 64>(a, sms, st);
  return wide ? launch_mass<__nv_bfloat16, 128>(a, sms, st) : launch_mass<__nv_bfloat16, 64>(a, sms, st);
}

int ocrvl_op_kv_select(int num_layers, int batch, int num_kv_heads, const float *acc, int acc_width, int64_t acc_stride,
                       const int32_t *lens, int keep, int sinks, int recent, int32_t *idx, float *sums, int32_t *new_lens,
                       void *stream) {
  if (num_layers < 1 || batch < 1 || num_kv_heads < 1) return invalid("num_layers, batch and num_kv_heads must be positive");
  const long long rows = (long long)num_layers * batch * num_kv_heads;
  if (rows > 1 << 24) return invalid("too many rows");
  if (acc_width < 1 || acc_width > 0x40000000 || acc_stride < acc_width) return invalid("acc rows must hold acc_width >= 1 values");
  if (keep < 1 || keep > 0x40000000) return invalid("keep must be positive");
  if (sinks < 0 || recent < 0 || (long long)sinks + recent > keep) return invalid("sinks + recent must be 0..keep");
  if (!acc || !lens || !idx) return invalid("null argument");
  if (new_lens == lens) return invalid("new_lens must not be lens");
  SelectArgs a{acc, acc_stride, lens, batch, num_kv_heads, acc_width, keep, sinks, recent, idx, sums, new_lens};
  cudaStream_t st = (cudaStream_t)stream;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  // Blocks a row: enough to hold the row's keys where that is possible, and more
  // while they all run at once (two an SM) and have 4096 sums each.
  int cs = 1;
  while (cs < 8 && ((acc_width + cs - 1) / cs > kSelStage || (rows * cs * 2 <= 2 * cluster_room(sms) && acc_width / cs > 4096))) cs *= 2;
  if (cs == 2) return launch_select<2, 512>(a, (int)rows, st);
  if (cs == 4) return launch_select<4, 512>(a, (int)rows, st);
  if (cs == 8) return launch_select<8, 512>(a, (int)rows, st);
  return acc_width <= 2048 ? launch_select<1, 256>(a, (int)rows, st) : launch_select<1, 512>(a, (int)rows, st);
}

int ocrvl_op_kv_compact(const ocrvl_kv_cache *from, const ocrvl_kv_cache *to, const int32_t *idx, int keep, void *stream) {
  return compact(from, to, idx, keep, (cudaStream_t)stream, false);
}

int ocrvl_op_kv_evict(const ocrvl_kv_cache *from, const ocrvl_kv_cache *to, const float *acc, int acc_width, int64_t acc_stride,
                      const int32_t *lens, int keep, int sinks, int recent, int32_t *idx, float *sums, int32_t *new_lens,
                      void *stream) {
  if (int rc = check_move(from, to, idx, keep)) return rc;
  if (int rc = ocrvl_op_kv_select(from->num_layers, from->batch, from->num_kv_heads, acc, acc_width, acc_stride, lens, keep, sinks,
                                  recent, idx, sums, new_lens, stream))
    return rc;
  return compact(from, to, idx, keep, (cudaStream_t)stream, true);
}

int ocrvl_op_kv_append(const ocrvl_kv_cache *c, int n_tokens, const int32_t *lens, const int32_t *indptr, const int32_t *path,
                       const int32_t *n_path, int max_path, const void *k, const void *v, int64_t kv_stride,
                       int64_t kv_layer_stride, int32_t *new_lens, void *stream) {
  if (int rc = check_cache(c)) return rc;
  const long long es = elem_bytes(c->type);
  if (n_tokens < 0) return invalid("n_tokens must not be negative");
  if (!lens || !indptr || !new_lens || (n_tokens > 0 && (!k || !v))) return invalid("null argument");
  if (path && (!n_path || max_path < 1)) return invalid("a path needs n_path and max_path >= 1");
  if (new_lens == lens) return invalid("new_lens must not be lens");
  if (!aligned16(k) || !aligned16(v) || kv_stride * es % 16 || kv_layer_stride * es % 16 || kv_layer_stride < 0 ||
      kv_stride < (int64_t)c->num_kv_heads * c->head_dim)
    return invalid("k and v must be 16-byte aligned rows of num_kv_heads * head_dim elements");
  AppendArgs a;
  a.k = (char *)c->k, a.v = (char *)c->v, a.src_k = (const char *)k, a.src_v = (const char *)v;
  a.table = c->table, a.lens = lens, a.indptr = indptr, a.path = path, a.n_path = n_path, a.new_lens = new_lens;
  a.page = c->page_stride * es, a.layer = c->layer_stride * es, a.head = c->head_stride * es;
  a.table_stride = c->table_stride;
  a.src_token = kv_stride * es, a.src_layer = kv_layer_stride * es;
  a.token = (int)(c->token_stride * es), a.shift = log2i(c->page_size), a.num_pages = c->num_pages, a.max_pages = c->max_pages;
  a.capacity = c->max_pages * c->page_size;
  a.layers = c->num_layers, a.batch = c->batch, a.kv_heads = c->num_kv_heads, a.n_tokens = n_tokens, a.max_path = max_path;
  a.row_bytes = (int)(c->head_dim * es);
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  // a warp an item, as many blocks as the longest path can use or the GPU holds
  const long long items = (c->num_layers + kAppendLayers - 1) / kAppendLayers * (long long)(path ? max_path : n_tokens);
  const long long blocks = (items + kMoveThreads / 32 - 1) / (kMoveThreads / 32), most = (sms * 16 + c->batch - 1) / c->batch;
  const unsigned gx = (unsigned)(blocks < 1 ? 1 : blocks < most ? blocks : most);
  return launch("append", k_kv_append, dim3(gx, c->batch), kMoveThreads, 0, (cudaStream_t)stream, false, 1, a);
}

}  // extern "C"
