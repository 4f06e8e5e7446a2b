// The torch side of the paged-cache operators (rapidocrvl_b200/kvops.py):
// checks torch tensors, takes outputs from torch's allocator and calls the C
// ABI on torch's current stream.  A call from Python through ctypes with the
// same checks took 16 to 24 us on the host, more than most single-token calls
// take on the GPU; this takes a third of that.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <string>

#include "../../include/ocrvl_cuda.h"

namespace {

PyObject *ocrvl_error;  // _lib.OcrvlError

struct Wrong {  // becomes a ValueError
  std::string text;
};

struct Refused {  // becomes an OcrvlError
  int code;
};

void ok(int rc) {
  if (rc < 0) throw Refused{rc};
}

// The operators have no backward pass: a result without a gradient is not to be taken for one.
const at::Tensor &no_gradient(const at::Tensor &t, const char *name) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    throw Wrong{std::string(name) + " requires a gradient, which this operator does not have (call it under torch.no_grad())"};
  return t;
}

const at::Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) throw Wrong{std::string(name) + " must be a tensor"};
  return no_gradient(THPVariable_Unpack(o), name);
}

// Tells autograd that a tensor of the caller's was written.
void wrote(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool none(PyObject *o) { return o == Py_None; }

int64_t whole(PyObject *o, const char *name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Wrong{std::string(name) + " must be an integer"};
  }
  return v;
}

int small(PyObject *o, const char *name) {
  const int64_t v = whole(o, name);
  if (v < INT32_MIN || v > INT32_MAX) throw Wrong{std::string(name) + " is out of range"};
  return (int)v;
}

float real(PyObject *o, const char *name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Wrong{std::string(name) + " must be a number"};
  }
  return (float)v;
}

int narrow(int64_t n, const char *name) {
  if (n > INT32_MAX) throw Wrong{std::string(name) + " is too large"};
  return (int)n;
}

struct Cache {
  const ocrvl_kv_cache *c;
  int device;
  at::ScalarType dtype;
  PyObject *pools[2];  // k and v, None where the engine holds them

  // a PagedCache's (address of the descriptor, device, k, v)
  explicit Cache(PyObject *o) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) throw Wrong{"cache must be a PagedCache"};
    c = (const ocrvl_kv_cache *)(uintptr_t)whole(PyTuple_GET_ITEM(o, 0), "cache");
    device = small(PyTuple_GET_ITEM(o, 1), "device");
    for (int i = 0; i < 2; i++) {
      pools[i] = PyTuple_GET_ITEM(o, 2 + i);
      if (!none(pools[i])) tensor(pools[i], i ? "the cache's v" : "the cache's k");
    }
    dtype = c->type == OCRVL_F32 ? at::kFloat : c->type == OCRVL_F16 ? at::kHalf : at::kBFloat16;
  }
  void written() const {
    for (PyObject *o : pools)
      if (!none(o)) wrote(THPVariable_Unpack(o));
  }
  std::string where() const { return "cuda:" + std::to_string(device); }
  void on_device(const at::Tensor &t, const char *name) const {
    if (!t.is_cuda() || t.get_device() != device) throw Wrong{std::string(name) + " must be on " + where()};
  }
  at::TensorOptions options(at::ScalarType type) const {
    return at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (c10::DeviceIndex)device));
  }
  void *stream() const {
    const int now = c10::cuda::current_device();
    if (now != device)
      throw Wrong{"the tensors are on " + where() + ", the current device is cuda:" + std::to_string(now)};
    return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  }
  // a contiguous tensor of `size` values
  void *flat(const at::Tensor &t, const char *name, at::ScalarType type, int64_t size) const {
    on_device(t, name);
    if (t.scalar_type() != type || !t.is_contiguous() || t.numel() != size)
      throw Wrong{std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor of " + std::to_string(size) + " values"};
    return t.data_ptr();
  }
  const int32_t *ints(PyObject *o, const char *name, int64_t size) const {
    return (const int32_t *)flat(tensor(o, name), name, at::kInt, size);
  }
  // The stride between the tokens of [tokens, heads, head_dim], the last three
  // dimensions of t.
  int64_t tokens(const at::Tensor &t, const char *name, int64_t heads, int64_t dims = 3) const {
    on_device(t, name);
    const int64_t i = dims - 3;
    if (t.scalar_type() != dtype || t.dim() != dims || (heads && t.size(i + 1) != heads) || t.size(i + 2) != c->head_dim ||
        t.stride(i + 2) != 1 || (t.size(i + 1) > 1 && t.stride(i + 1) != c->head_dim))
      throw Wrong{std::string(name) + " must be a " + (i ? "[layers, " : "[") + "tokens, " + (heads ? std::to_string(heads) : "heads") +
                  ", " + std::to_string(c->head_dim) + "] " + c10::toString(dtype) + " tensor with the heads of a token contiguous"};
    return t.size(i) > 1 ? t.stride(i) : t.size(i + 1) * c->head_dim;
  }
  // The stride between the rows of a f32 tensor [layers (if any), batch, kv heads, width].
  int64_t rows(const at::Tensor &t, const char *name, bool layers) const {
    on_device(t, name);
    const int64_t d = t.dim(), lead[3] = {c->num_layers, c->batch, c->num_kv_heads};
    bool fine = t.scalar_type() == at::kFloat && d == (layers ? 4 : 3) && t.stride(d - 1) == 1;
    int64_t size = 1, row = -1;
    for (int64_t i = d - 2, j = 2; fine && i >= 0; i--, j--) {
      fine = t.size(i) == lead[j];
      if (lead[j] > 1) {
        if (row < 0) row = t.stride(i) % size ? -2 : t.stride(i) / size;
        fine = fine && row >= 0 && t.stride(i) == row * size;
      }
      size *= lead[j];
    }
    if (!fine)
      throw Wrong{std::string(name) + " must be a [" + (layers ? "layers, " : "") + "batch, kv heads, width] float32 tensor of the cache's " +
                  "shape whose rows are one stride apart"};
    return row < 0 ? t.size(d - 1) : row;
  }
};

float scale_of(PyObject *o, const Cache &c) { return none(o) ? (float)(1.0 / std::sqrt((double)c.c->head_dim)) : real(o, "scale"); }

int draft_of(PyObject *o, int64_t n) { return none(o) ? (int)std::min<int64_t>(64, std::max<int64_t>(1, n)) : small(o, "max_draft"); }

PyObject *pack(std::initializer_list<at::Tensor> ts) {
  PyObject *t = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const at::Tensor &x : ts) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(x));
  return t;
}

// (cache, q, k, v, lens, indptr, mask, layer, max_draft, scale, out, lse, work)
PyObject *tree_attention(PyObject *const *a) {
  const Cache c(a[0]);
  const at::Tensor &q = tensor(a[1], "q"), &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
  const int64_t q_stride = c.tokens(q, "q", 0), kv_stride = c.tokens(k, "k", c.c->num_kv_heads);
  const int64_t n = q.size(0), heads = q.size(1);
  if (c.tokens(v, "v", c.c->num_kv_heads) != kv_stride || k.size(0) != n || v.size(0) != n)
    throw Wrong{"k and v must have q's tokens and the same stride"};
  const int32_t *lens = c.ints(a[4], "lens", c.c->batch), *indptr = c.ints(a[5], "indptr", c.c->batch + 1);
  const void *mask = c.flat(tensor(a[6], "mask"), "mask", at::kLong, n);
  void *stream = c.stream();
  const int max_draft = draft_of(a[8], n);
  int64_t bytes = 0;
  ok(ocrvl_op_tree_attn_workspace(c.c, narrow(heads, "heads"), max_draft, &bytes));
  const at::Tensor out = none(a[10]) ? at::empty({n, heads, c.c->head_dim}, c.options(c.dtype)) : tensor(a[10], "out");
  const int64_t out_stride = c.tokens(out, "out", heads);
  if (out.size(0) != n) throw Wrong{"out must have q's shape"};
  const at::Tensor lse = none(a[11]) ? at::empty({n, heads}, c.options(at::kFloat)) : tensor(a[11], "lse");
  const at::Tensor work = none(a[12]) ? at::empty({bytes}, c.options(at::kByte)) : tensor(a[12], "work");
  ok(ocrvl_op_tree_attn(c.c, small(a[7], "layer"), narrow(heads, "heads"), narrow(n, "tokens"), max_draft, lens, indptr,
                        (const int64_t *)mask, q.data_ptr(), q_stride, k.data_ptr(), v.data_ptr(), kv_stride, scale_of(a[9], c),
                        out.data_ptr(), out_stride, (float *)c.flat(lse, "lse", at::kFloat, n * heads),
                        c.flat(work, "work", at::kByte, work.numel()), work.numel(), stream));
  wrote(out), wrote(lse), wrote(work);
  return pack({out, lse});
}

// (cache, q, lse, lens, indptr, layer, max_draft, scale, counted, acc, decay, out)
PyObject *attention_mass(PyObject *const *a) {
  const Cache c(a[0]);
  const at::Tensor &q = tensor(a[1], "q"), &lse = tensor(a[2], "lse");
  const int64_t q_stride = c.tokens(q, "q", 0), n = q.size(0), heads = q.size(1);
  const float *lse_at = (const float *)c.flat(lse, "lse", at::kFloat, n * heads);
  const int32_t *lens = c.ints(a[3], "lens", c.c->batch), *indptr = c.ints(a[4], "indptr", c.c->batch + 1);
  const int64_t *counted = none(a[8]) ? nullptr : (const int64_t *)c.flat(tensor(a[8], "counted"), "counted", at::kLong, c.c->batch);
  const float *acc = nullptr;
  int64_t acc_width = 0, acc_stride = 0, width = (int64_t)c.c->max_pages * c.c->page_size;
  if (!none(a[9])) {
    const at::Tensor &t = tensor(a[9], "acc");
    acc_stride = c.rows(t, "acc", false);
    acc = (const float *)t.data_ptr(), acc_width = width = t.size(2);
  }
  void *stream = c.stream();
  const at::Tensor out = none(a[11]) ? at::empty({c.c->batch, c.c->num_kv_heads, width}, c.options(at::kFloat)) : tensor(a[11], "out");
  const int64_t out_stride = c.rows(out, "out", false);
  ok(ocrvl_op_attn_mass(c.c, small(a[5], "layer"), narrow(heads, "heads"), narrow(n, "tokens"), draft_of(a[6], n), lens, indptr, counted,
                        q.data_ptr(), q_stride, lse_at, scale_of(a[7], c), real(a[10], "decay"), acc, narrow(acc_width, "acc"),
                        acc_stride, (float *)out.data_ptr(), narrow(out.size(2), "out"), out_stride, stream));
  wrote(out);
  return THPVariable_Wrap(out);
}

// The shared part of select and evict: to is NULL for select.
PyObject *choose(const Cache &c, const Cache *to, PyObject *const *a) {
  const at::Tensor &acc = tensor(a[1], "acc");
  const int64_t stride = c.rows(acc, "acc", true);
  const int keep = small(a[3], "keep"), sinks = small(a[4], "sinks"), recent = small(a[5], "recent");
  const int32_t *lens = c.ints(a[2], "lens", c.c->batch);
  const float *from = (const float *)acc.data_ptr();
  const int width = narrow(acc.size(3), "acc");
  void *stream = c.stream();
  const int64_t shape[4] = {c.c->num_layers, c.c->batch, c.c->num_kv_heads, std::max(keep, 0)};
  const at::Tensor idx = at::empty(shape, c.options(at::kInt)), sums = at::empty(shape, c.options(at::kFloat));
  const at::Tensor new_lens = at::empty({c.c->batch}, c.options(at::kInt));
  int32_t *i = (int32_t *)idx.data_ptr(), *l = (int32_t *)new_lens.data_ptr();
  float *s = (float *)sums.data_ptr();
  ok(to ? ocrvl_op_kv_evict(c.c, to->c, from, width, stride, lens, keep, sinks, recent, i, s, l, stream)
        : ocrvl_op_kv_select(c.c->num_layers, c.c->batch, c.c->num_kv_heads, from, width, stride, lens, keep, sinks, recent, i, s, l, stream));
  if (to) to->written();
  return pack({idx, sums, new_lens});
}

// (cache, acc, lens, keep, sinks, recent)
PyObject *select(PyObject *const *a) { return choose(Cache(a[0]), nullptr, a); }

// (cache, acc, lens, keep, sinks, recent, into)
PyObject *evict(PyObject *const *a) {
  const Cache to(a[6]);
  return choose(Cache(a[0]), &to, a);
}

// (cache, idx, into)
PyObject *compact(PyObject *const *a) {
  const Cache c(a[0]), to(a[2]);
  const at::Tensor &idx = tensor(a[1], "idx");
  if (idx.dim() != 4 || idx.size(0) != c.c->num_layers || idx.size(1) != c.c->batch || idx.size(2) != c.c->num_kv_heads)
    throw Wrong{"idx must be [layers, batch, kv heads, keep] of the cache's shape"};
  ok(ocrvl_op_kv_compact(c.c, to.c, (const int32_t *)c.flat(idx, "idx", at::kInt, idx.numel()), narrow(idx.size(3), "keep"), c.stream()));
  to.written();
  Py_RETURN_NONE;
}

// (cache, k, v, lens, indptr, path, n_path)
PyObject *append(PyObject *const *a) {
  const Cache c(a[0]);
  const at::Tensor &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
  const int64_t stride = c.tokens(k, "k", c.c->num_kv_heads, 4);
  if (c.tokens(v, "v", c.c->num_kv_heads, 4) != stride || v.sizes() != k.sizes() || k.size(0) != c.c->num_layers ||
      (k.size(0) > 1 && v.stride(0) != k.stride(0)))
    throw Wrong{"k and v must be [" + std::to_string(c.c->num_layers) + ", tokens, kv heads, head_dim] of the same strides"};
  const int32_t *lens = c.ints(a[3], "lens", c.c->batch), *indptr = c.ints(a[4], "indptr", c.c->batch + 1);
  const int32_t *path = nullptr, *n_path = nullptr;
  int64_t most = 0;
  if (none(a[5]) != none(a[6])) throw Wrong{"path and n_path go together"};
  if (!none(a[5])) {
    const at::Tensor &p = tensor(a[5], "path");
    if (p.dim() != 2 || p.size(0) != c.c->batch) throw Wrong{"path must be [batch, most]"};
    path = (const int32_t *)c.flat(p, "path", at::kInt, p.numel()), most = p.size(1);
    n_path = c.ints(a[6], "n_path", c.c->batch);
  }
  void *stream = c.stream();
  const at::Tensor new_lens = at::empty({c.c->batch}, c.options(at::kInt));
  ok(ocrvl_op_kv_append(c.c, narrow(k.size(1), "tokens"), lens, indptr, path, n_path, narrow(most, "path"), k.data_ptr(), v.data_ptr(),
                        stride, k.size(0) > 1 ? k.stride(0) : 0, (int32_t *)new_lens.data_ptr(), stream));
  c.written();
  return THPVariable_Wrap(new_lens);
}

template <PyObject *(*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Wrong &w) {
    PyErr_SetString(PyExc_ValueError, w.text.c_str());
  } catch (const Refused &r) {
    PyObject *e = PyObject_CallFunction(ocrvl_error, "is", r.code, ocrvl_last_error());
    if (e) PyErr_SetObject(ocrvl_error, e), Py_DECREF(e);
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

#define ENTRY(f, n) {#f, (PyCFunction)(void (*)(void))entry<f, n>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(tree_attention, 13), ENTRY(attention_mass, 12), ENTRY(select, 6), ENTRY(compact, 3),
                         ENTRY(evict, 7),           ENTRY(append, 7),          {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kvops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kvops(void) {
  PyObject *lib = PyImport_ImportModule("rapidocrvl_b200._lib");
  if (!lib) return nullptr;
  ocrvl_error = PyObject_GetAttrString(lib, "OcrvlError");
  Py_DECREF(lib);
  return ocrvl_error ? PyModule_Create(&module) : nullptr;
}
