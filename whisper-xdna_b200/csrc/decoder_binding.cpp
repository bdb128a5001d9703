// The Python binding of the decoder operators (wxb200.ops): argument checks, output
// and workspace allocation and the call of the C ABI, on torch tensors.
//
// A decoder calls these operators once a layer and token, on work of a few
// microseconds, so what the host spends counts: checked and allocated in Python and
// called through ctypes, a call cost 10 to 24 us; here it costs 3 to 7 (B200 host).
// Everything computed is in libwxb200.so, whose entry points check sizes and
// strides themselves.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/wxb200.h"

namespace {

using at::Tensor;

struct Refused : std::runtime_error {   // a ValueError
  using std::runtime_error::runtime_error;
};
struct Failed {   // a status of the C ABI
  int status;
};
struct Raised {};   // a Python error is set

[[noreturn]] void refuse(const std::string& s) { throw Refused(s); }

std::string sizes(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); i++) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + ")";
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a torch tensor");
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised();
  return v == 1;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}

// `t` on device dev, of dtype, contiguous, of the shape given.
void* plain(int dev, const Tensor& t, const char* name, at::ScalarType dtype,
            at::IntArrayRef shape) {
  if (!t.is_cuda() || t.get_device() != dev)
    refuse(std::string(name) + " must be a CUDA tensor on the device of the others");
  if (t.scalar_type() != dtype || t.sizes() != shape || !t.is_contiguous())
    refuse(std::string(name) + " must be a contiguous " + c10::toString(dtype) +
           " tensor of shape " + sizes(shape) + ", got " + c10::toString(t.scalar_type()) + " " +
           sizes(t.sizes()) + " with strides " + sizes(t.strides()));
  return t.data_ptr();
}
void* plain_or_null(int dev, PyObject* o, const char* name, at::ScalarType dtype,
                    at::IntArrayRef shape) {
  return o == Py_None ? nullptr : plain(dev, tensor(o, name), name, dtype, shape);
}
int32_t* ints(void* p) { return static_cast<int32_t*>(p); }

int dtype_code(const Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return WX_DTYPE_BF16;
  if (t.scalar_type() == at::kFloat) return WX_DTYPE_F32;
  refuse(std::string(name) + " dtype " + c10::toString(t.scalar_type()) +
         " not in (BFloat16, Float)");
}

// A cache's two pools: (..., pages, page, heads, head_dim) with `dim` dimensions.
struct Pools {
  const Tensor &k, &v;
  int dev, dtype;
  int64_t n_layers, layer_stride, n_pages, page, n_heads, hd, page_stride, tok_stride,
      head_stride;

  Pools(PyObject* ko, PyObject* vo, int dim) : k(tensor(ko, "k_cache")), v(tensor(vo, "v_cache")) {
    if (!k.is_cuda() || !v.is_cuda()) refuse("k_cache and v_cache must be CUDA tensors");
    if (k.dim() != dim)
      refuse("the cache must have " + std::to_string(dim) + " dimensions, got " +
             std::to_string(k.dim()));
    dtype = dtype_code(k, "cache");
    if (v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes() ||
        v.strides() != k.strides())
      refuse("k_cache and v_cache must have the same dtype, shape and strides");
    dev = k.get_device();
    if (v.get_device() != dev || dev != c10::cuda::current_device())
      refuse("the cache must be on the current CUDA device");
    const auto n = k.sizes(), s = k.strides();
    const int o = dim - 4;
    n_layers = o ? n[0] : 1;
    layer_stride = o ? s[0] : 0;
    n_pages = n[o];
    page = n[o + 1];
    n_heads = n[o + 2];
    hd = n[o + 3];
    page_stride = s[o];
    tok_stride = s[o + 1];
    head_stride = s[o + 2];
    if (s[o + 3] != 1) refuse("the cache's head_dim must be contiguous");
  }
};

struct Table {
  int64_t n, width;
  int32_t* p;
  Table(int dev, PyObject* o) {
    const Tensor& t = tensor(o, "table");
    if (t.dim() != 2 || t.size(1) == 0) refuse("table must be a (n_seqs, width) tensor");
    n = t.size(0);
    width = t.size(1);
    p = ints(plain(dev, t, "table", at::kInt, t.sizes()));
  }
};

Tensor empty(int dev, at::IntArrayRef shape, at::ScalarType dtype) {
  return at::detail::empty_cuda(shape, dtype, at::Device(at::kCUDA, (c10::DeviceIndex)dev),
                                std::nullopt);
}
// Several outputs in one allocation: an allocation costs the host as much as a launch
// does. Each starts on 16 bytes.
class Outputs {
 public:
  explicit Outputs(int dev) : dev_(dev) {}
  // the place of an output of `bytes` bytes
  int64_t add(int64_t bytes) {
    const int64_t at = total_;
    total_ += (bytes + 15) / 16 * 16;
    return at;
  }
  void allocate() { all_ = empty(dev_, {total_}, at::kByte); }
  char* at(int64_t place) const { return static_cast<char*>(all_.data_ptr()) + place; }
  // a contiguous tensor on the output at `place`
  Tensor tensor(int64_t place, at::IntArrayRef shape, at::ScalarType dtype,
                at::OptionalIntArrayRef strides = {}) const {
    const auto meta = c10::scalarTypeToTypeMeta(dtype);
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all_.storage()),
                                                        all_.key_set(), meta);
    t.unsafeGetTensorImpl()->set_storage_offset(place / (int64_t)meta.itemsize());
    if (strides)
      t.unsafeGetTensorImpl()->set_sizes_and_strides(shape, *strides);
    else
      t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    return t;
  }

 private:
  int dev_;
  int64_t total_ = 0;
  Tensor all_;
};

void* stream(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }
void check(int status) {
  if (status != WX_OK) throw Failed{status};
}

// (q's rows) as the C ABI takes them: strides of sequence, cache head and group.
struct Rows {
  int64_t seq, head, group;
  Rows(const Tensor& t, int64_t g) {
    const auto s = t.strides();
    seq = s[0];
    head = t.dim() == 3 ? s[1] * g : s[1];
    group = t.dim() == 3 ? s[1] : s[2];
  }
};

// paged_attention(q, k_cache, v_cache, table, lens, scale, starts, max_len, out, return_lse)
PyObject* paged_attention(PyObject* const* a) {
  const Pools c(a[1], a[2], 4);
  const Table table(c.dev, a[3]);
  const int32_t* lens = ints(plain(c.dev, tensor(a[4], "lens"), "lens", at::kInt, {table.n}));
  const Tensor& q = tensor(a[0], "q");
  if (!q.is_cuda() || q.get_device() != c.dev || q.scalar_type() != c.k.scalar_type())
    refuse("q must be a CUDA tensor on the cache's device, of its dtype");
  if (q.dim() != 3 && q.dim() != 4) refuse("q must have 3 or 4 dimensions");
  const auto n = q.sizes();
  if (q.dim() == 3 && (c.n_heads == 0 || n[1] % c.n_heads))
    refuse(std::to_string(n[1]) + " query heads are no multiple of " + std::to_string(c.n_heads) +
           " cache heads");
  if (q.dim() == 4 && n[1] != c.n_heads)
    refuse("q has " + std::to_string(n[1]) + " cache heads, the cache " +
           std::to_string(c.n_heads));
  const int64_t group = q.dim() == 3 ? n[1] / c.n_heads : n[2];
  if (n[0] != table.n || n[q.dim() - 1] != c.hd || q.stride(-1) != 1)
    refuse("q of shape " + sizes(n) + " does not fit " + std::to_string(table.n) +
           " sequences of head_dim " + std::to_string(c.hd) + " (contiguous)");
  const bool own = a[8] == Py_None, want_lse = truth(a[9]);
  Tensor out, lse;
  if (!own) {
    out = tensor(a[8], "out");
    if (out.sizes() != n || out.scalar_type() != q.scalar_type() || !out.is_cuda() ||
        out.get_device() != c.dev || out.stride(-1) != 1)
      refuse("out must be like q, with a contiguous head_dim");
  }
  Outputs outputs(c.dev);
  const int64_t rows = table.n * c.n_heads * group;
  const int64_t o_at = outputs.add(own ? q.numel() * (int64_t)q.element_size() : 0),
                lse_at = outputs.add(want_lse ? 4 * rows : 0);
  if (own || want_lse) outputs.allocate();
  if (own) {
    // q dense and without overlap: its strides; else its order of dimensions
    if (q.is_non_overlapping_and_dense())
      out = outputs.tensor(o_at, n, q.scalar_type(), q.strides());
    else
      out = outputs.tensor(o_at, n, q.scalar_type());
  }
  if (want_lse) lse = outputs.tensor(lse_at, n.slice(0, q.dim() - 1), at::kFloat);
  const int32_t* starts = ints(plain_or_null(c.dev, a[6], "starts", at::kInt, {table.n}));
  const int64_t max_len = a[7] == Py_None ? table.width * c.page : integer(a[7]);
  const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)c.hd) : number(a[5]);
  Tensor ws;
  const int64_t space =
      wx_paged_attention_workspace(table.n, c.n_heads, group, c.hd, max_len, c.dtype);
  if (space < 0) throw Failed{(int)space};
  if (space) ws = empty(c.dev, {space}, at::kByte);
  const Rows qr(q, group), orow(out, group);
  check(wx_paged_attention(
      q.data_ptr(), qr.seq, qr.head, qr.group, c.k.data_ptr(), c.v.data_ptr(), c.page_stride,
      c.tok_stride, c.head_stride, table.p, table.width, lens, starts, out.data_ptr(), orow.seq,
      orow.head, orow.group, want_lse ? lse.data_ptr<float>() : nullptr, table.n, c.n_heads,
      group, c.hd, c.n_pages, c.page, max_len, (float)scale, c.dtype,
      space ? ws.data_ptr() : nullptr, space, stream(c.dev)));
  PyObject* o = a[8];
  if (own)
    o = THPVariable_Wrap(out);
  else
    Py_INCREF(o);
  if (!want_lse) return o;
  return Py_BuildValue("(NN)", o, THPVariable_Wrap(lse));
}

// kv_append(k, v, k_cache, v_cache, table, lens, counts)
PyObject* kv_append(PyObject* const* a) {
  const Pools c(a[2], a[3], 4);
  const Table table(c.dev, a[4]);
  const int32_t* lens = ints(plain(c.dev, tensor(a[5], "lens"), "lens", at::kInt, {table.n}));
  const Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v");
  for (const Tensor* t : {&k, &v})
    if (!t->is_cuda() || t->get_device() != c.dev || t->scalar_type() != c.k.scalar_type())
      refuse("k and v must be CUDA tensors on the cache's device, of its dtype");
  if (v.sizes() != k.sizes() || v.strides() != k.strides())
    refuse("k and v must have the same shape and strides");
  const auto n = k.sizes(), s = k.strides();
  const int o = (int)k.dim() - 3;   // (sequences, [tokens,] heads, head_dim)
  if ((o != 0 && o != 1) || n[0] != table.n || n[o + 1] != c.n_heads || n[o + 2] != c.hd ||
      s[o + 2] != 1)
    refuse("k of shape " + sizes(n) + " does not fit " + std::to_string(table.n) +
           " sequences of " + std::to_string(c.n_heads) + " heads of " + std::to_string(c.hd) +
           " (contiguous)");
  const int32_t* counts = ints(plain_or_null(c.dev, a[6], "counts", at::kInt, {table.n}));
  check(wx_kv_append(k.data_ptr(), v.data_ptr(), s[0], o ? s[1] : 0, s[o + 1], c.k.data_ptr(),
                     c.v.data_ptr(), c.page_stride, c.tok_stride, c.head_stride, table.p,
                     table.width, lens, counts, table.n, o ? n[1] : 1, c.n_heads, c.hd, c.n_pages,
                     c.page, c.dtype, stream(c.dev)));
  Py_RETURN_NONE;
}

// A plan's workspace: beside the outputs where it is small, since an allocation costs as
// much host time as the rest of the call, else apart, so that it does not live as long
// as they do.
struct PlanSpace {
  int64_t bytes, place = -1;
  Tensor apart;
  PlanSpace(Outputs& out, int64_t n_seqs, int64_t n_pages)
      : bytes(wx_kv_workspace(n_seqs, n_pages)) {
    if (bytes <= 1 << 18) place = out.add(bytes);
  }
  void* get(const Outputs& out, int dev) {
    if (place >= 0) return out.at(place);
    apart = empty(dev, {bytes}, at::kByte);
    return apart.data_ptr();
  }
};

// kv_fork(k_cache, v_cache, table, lens, refs, parents, grow)
PyObject* kv_fork(PyObject* const* a) {
  const Pools c(a[0], a[1], 5);
  const Table table(c.dev, a[2]);
  const int32_t* lens = ints(plain(c.dev, tensor(a[3], "lens"), "lens", at::kInt, {table.n}));
  const int32_t* refs = ints(plain(c.dev, tensor(a[4], "refs"), "refs", at::kInt, {c.n_pages}));
  const int32_t* parents = ints(plain_or_null(c.dev, a[5], "parents", at::kInt, {table.n}));
  const int32_t* grow = ints(plain_or_null(c.dev, a[6], "grow", at::kInt, {table.n}));
  Outputs out(c.dev);
  PlanSpace ws(out, table.n, c.n_pages);
  const int64_t t = out.add(4 * table.n * table.width), l = out.add(4 * table.n),
                r = out.add(4 * c.n_pages), g = out.add(4 * table.n), s = out.add(8);
  out.allocate();
  check(wx_kv_fork(c.k.data_ptr(), c.v.data_ptr(), c.n_layers, c.layer_stride, c.page_stride,
                   c.tok_stride, c.head_stride, c.n_heads, c.hd, c.n_pages, c.page, c.dtype,
                   table.p, lens, refs, parents, grow, table.n, table.width, ints(out.at(t)),
                   ints(out.at(l)), ints(out.at(r)), ints(out.at(g)), ints(out.at(s)),
                   ws.get(out, c.dev), ws.bytes, stream(c.dev)));
  return Py_BuildValue("(NNNNN)",
                       THPVariable_Wrap(out.tensor(t, {table.n, table.width}, at::kInt)),
                       THPVariable_Wrap(out.tensor(l, {table.n}, at::kInt)),
                       THPVariable_Wrap(out.tensor(r, {c.n_pages}, at::kInt)),
                       THPVariable_Wrap(out.tensor(g, {table.n}, at::kInt)),
                       THPVariable_Wrap(out.tensor(s, {2}, at::kInt)));
}

// kv_compact(k_cache, v_cache, table, refs)
PyObject* kv_compact(PyObject* const* a) {
  const Pools c(a[0], a[1], 5);
  const Table table(c.dev, a[2]);
  const int32_t* refs = ints(plain(c.dev, tensor(a[3], "refs"), "refs", at::kInt, {c.n_pages}));
  Outputs out(c.dev);
  PlanSpace ws(out, table.n, c.n_pages);
  const int64_t t = out.add(4 * table.n * table.width), r = out.add(4 * c.n_pages),
                s = out.add(8);
  out.allocate();
  check(wx_kv_compact(c.k.data_ptr(), c.v.data_ptr(), c.n_layers, c.layer_stride, c.page_stride,
                      c.tok_stride, c.head_stride, c.n_heads, c.hd, c.n_pages, c.page, c.dtype,
                      table.p, refs, table.n, table.width, ints(out.at(t)), ints(out.at(r)),
                      ints(out.at(s)), ws.get(out, c.dev), ws.bytes, stream(c.dev)));
  return Py_BuildValue("(NNN)",
                       THPVariable_Wrap(out.tensor(t, {table.n, table.width}, at::kInt)),
                       THPVariable_Wrap(out.tensor(r, {c.n_pages}, at::kInt)),
                       THPVariable_Wrap(out.tensor(s, {2}, at::kInt)));
}

// token_logprobs(logits, tokens, top_k, temperature)
PyObject* token_logprobs(PyObject* const* a) {
  const Tensor& x = tensor(a[0], "logits");
  if (!x.is_cuda()) refuse("logits must be a CUDA tensor");
  if (x.dim() != 2 || x.stride(1) != 1)
    refuse("logits must be 2-D with a contiguous last dimension");
  const int dtype = dtype_code(x, "logits"), dev = x.get_device();
  if (dev != c10::cuda::current_device()) refuse("logits must be on the current CUDA device");
  const int64_t rows = x.size(0), vocab = x.size(1), top_k = integer(a[2]);
  const int64_t* tokens =
      static_cast<int64_t*>(plain(dev, tensor(a[1], "tokens"), "tokens", at::kLong, {rows}));
  if (top_k < 0 || top_k > 32 || top_k > vocab)
    refuse("top_k " + std::to_string(top_k) + " not in [0, min(32, vocabulary " +
           std::to_string(vocab) + ")]");
  const double temperature = number(a[3]);
  Outputs out(dev);
  const int64_t logprob = out.add(4 * rows), entropy = out.add(4 * rows),
                top = out.add(4 * rows * top_k), index = out.add(4 * rows * top_k);
  out.allocate();
  auto floats = [&](int64_t place) { return reinterpret_cast<float*>(out.at(place)); };
  check(wx_token_logprobs(x.data_ptr(), dtype, rows, vocab, x.stride(0), tokens, top_k,
                          (float)temperature, floats(logprob), floats(entropy),
                          top_k ? floats(top) : nullptr, top_k ? ints(out.at(index)) : nullptr,
                          stream(dev)));
  return Py_BuildValue("(NNNN)", THPVariable_Wrap(out.tensor(logprob, {rows}, at::kFloat)),
                       THPVariable_Wrap(out.tensor(entropy, {rows}, at::kFloat)),
                       THPVariable_Wrap(out.tensor(top, {rows, top_k}, at::kFloat)),
                       THPVariable_Wrap(out.tensor(index, {rows, top_k}, at::kInt)));
}

// A function of `count` positional arguments; its errors as Python's.
template <PyObject* (*f)(PyObject* const*), int count>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != count) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", count, n);
    return nullptr;
  }
  try {
    return f(args);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const Raised&) {
  } catch (const Failed& e) {
    // wxb200._lib.check raises what the status stands for
    PyObject* lib = PyImport_ImportModule("wxb200._lib");
    PyObject* r = lib ? PyObject_CallMethod(lib, "check", "i", e.status) : nullptr;
    Py_XDECREF(lib);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "wxb200: a call failed");
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*f)(PyObject* const*), int count>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<f, count>)),
          METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<paged_attention, 10>("paged_attention"),
                         method<kv_append, 7>("kv_append"),
                         method<kv_fork, 7>("kv_fork"),
                         method<kv_compact, 4>("kv_compact"),
                         method<token_logprobs, 4>("token_logprobs"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decoder", "The decoder operators on torch tensors.",
                      -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decoder() { return PyModule_Create(&module); }
