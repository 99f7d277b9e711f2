// Python binding of the paged cache's entry points (the module ntilang_b200._paged behind
// ntilang_b200/paged.py): argument checks, output and workspace allocation, and the C-ABI call on torch's
// current stream.  In C++ because small calls waited for their checks in Python and the ctypes conversions: host
// time of a window attention 14 -> 8 us, of an append and an accept 22 -> 10, of a tree's mask and attention
// 21 -> 12, against 8 to 15 us on the device at their smallest.
//
// The C ABI itself is libntl_kernels.so, which this module links; nothing here launches kernels.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <map>
#include <string>

#include "../../include/ntl_kernels.h"

namespace {

using at::Tensor;

// A Python exception that is already set; caught at the module's functions.
struct Raised {};

[[noreturn]] void raise(PyObject* type, const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  PyErr_SetString(type, text);
  throw Raised();
}

std::string shape_text(at::IntArrayRef shape) {
  std::string s = "(";
  for (size_t i = 0; i < shape.size(); ++i)
    s += (i ? ", " : "") + (shape[i] < 0 ? std::string("any") : std::to_string(shape[i]));
  return s + (shape.size() == 1 ? ",)" : ")");
}

const char* type_name(const Tensor& x) { return c10::toString(x.scalar_type()); }

// ------------------------------------------------------------------------------ arguments

const Tensor& tensor_of(const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s must be a CUDA tensor", name);
  const Tensor& x = THPVariable_Unpack(o);
  if (!x.is_cuda()) raise(PyExc_TypeError, "%s must be a CUDA tensor", name);
  return x;
}

int64_t int_of(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}

void same_device(const Tensor& x, int index) {
  if (x.get_device() != index) raise(PyExc_ValueError, "All tensor arguments must be on the same CUDA device");
}

// An int32 CUDA tensor of the given sizes (-1: any), last dimension dense.
const Tensor& ints(const char* name, PyObject* o, int index, std::initializer_list<int64_t> shape) {
  const Tensor& x = tensor_of(name, o);
  if (x.scalar_type() != at::kInt) raise(PyExc_ValueError, "%s: expected dtype int32, got %s", name, type_name(x));
  bool ok = x.dim() == static_cast<int64_t>(shape.size());
  int64_t d = 0;
  for (int64_t want : shape) {
    ok = ok && (want < 0 || x.size(d) == want);
    ++d;
  }
  if (!ok)
    raise(PyExc_ValueError, "%s: expected shape %s, got %s", name, shape_text({shape.begin(), shape.size()}).c_str(),
          shape_text(x.sizes()).c_str());
  if (x.size(-1) > 1 && x.stride(-1) != 1) raise(PyExc_ValueError, "%s must be dense along its last dimension", name);
  same_device(x, index);
  return x;
}
// A table whose rows are written.
const Tensor& written_table(const char* name, const Tensor& x) {
  if (x.size(0) > 1 && x.stride(0) < x.size(1))
    raise(PyExc_ValueError, "%s must not be broadcast: its rows are written", name);
  return x;
}
int32_t* int_ptr(const Tensor& x) { return x.data_ptr<int32_t>(); }

// A 16-bit CUDA tensor that the kernels can read 16 bytes at a time along its last dimension.
const Tensor& values(const char* name, PyObject* o) {
  const Tensor& x = tensor_of(name, o);
  if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16)
    raise(PyExc_ValueError, "%s: expected dtype float16 or bfloat16, got %s", name, type_name(x));
  if (x.numel()) {
    const auto stride = x.strides();
    bool ok = !stride.empty() && stride.back() == 1;
    for (size_t i = 0; i + 1 < stride.size(); ++i) ok = ok && stride[i] % 8 == 0;
    if (!ok) raise(PyExc_ValueError, "%s must be dense along its last dimension, its other strides multiples of 8", name);
  }
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16)
    raise(PyExc_ValueError, "%s requires a tensor with an inspectable, 16-byte-aligned data pointer", name);
  return x;
}

struct Cache {
  ntl_cache_t c;
  int index;
  const Tensor *k, *v;
  bool layered;
};

Cache cache_of(PyObject* ko, PyObject* vo, bool layers_allowed, bool written) {
  const Tensor& k = values("k", ko);
  const Tensor& v = values("v", vo);
  if (k.dim() != 4 && !(layers_allowed && k.dim() == 5))
    raise(PyExc_ValueError, "k: expected %s dimensions, got shape %s", layers_allowed ? "4 or 5" : "4",
          shape_text(k.sizes()).c_str());
  if (v.sizes() != k.sizes() || v.strides() != k.strides() || v.scalar_type() != k.scalar_type())
    raise(PyExc_ValueError, "k and v must have the same shape, strides and dtype");
  Cache r;
  r.index = k.get_device();
  same_device(v, r.index);
  r.k = &k;
  r.v = &v;
  r.layered = k.dim() == 5;
  const int64_t at = r.layered ? 1 : 0;  // first dimension after the layers
  if (written)
    for (int64_t d = 0; d < k.dim(); ++d)
      if (k.size(d) > 1 && k.stride(d) == 0)
        raise(PyExc_ValueError, "k and v must not be broadcast: their rows are written");
  const int64_t dim = k.size(at + 3), page_size = k.size(at + 1);
  if (dim == 0 || dim % 8) raise(PyExc_ValueError, "k: head_dim %lld is not a multiple of 8", (long long)dim);
  if (page_size == 0) raise(PyExc_ValueError, "k: page_size is 0");
  r.c = {k.data_ptr(), v.data_ptr(), r.layered ? k.size(0) : 1, k.size(at), page_size, k.size(at + 2), dim,
         r.layered ? k.stride(0) : 0, k.stride(at), k.stride(at + 1), k.stride(at + 2),
         k.scalar_type() == at::kBFloat16 ? NTL_BF16 : NTL_F16};
  return r;
}

// ------------------------------------------------------------------------------ calls

// Makes `index` the current device for the scope of a call.
struct Device {
  c10::cuda::OptionalCUDAGuard guard;
  explicit Device(int index) {
    if (c10::cuda::current_device() != index) guard.set_index(static_cast<c10::DeviceIndex>(index));
  }
};

ntl_stream_t stream_of(int index) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream(); }

void check(const char* name, int code) {
  if (code == NTL_OK) return;
  PyObject* module = PyImport_ImportModule("ntilang_b200._lib");
  PyObject* type = module ? PyObject_GetAttrString(module, "KernelError") : nullptr;
  PyObject* error = type ? PyObject_CallFunction(type, "sis", name, code, ntl_last_error()) : nullptr;
  if (error) PyErr_SetObject(type, error);
  Py_XDECREF(error);
  Py_XDECREF(type);
  Py_XDECREF(module);
  throw Raised();
}

Tensor new_ints(at::IntArrayRef shape, int index) {
  return at::empty(shape, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, static_cast<c10::DeviceIndex>(index)));
}

// At least `bytes` of workspace for a call on device `index`'s current stream.  Calls on one stream follow
// each other, so they share a buffer; a call that is captured in a graph, which may be replayed on any
// stream, gets its own.  (Under the GIL; never freed, so that nothing runs at the interpreter's end.)
Tensor workspace(int64_t bytes, int index) {
  const auto options = at::TensorOptions().dtype(at::kByte).device(at::kCUDA, static_cast<c10::DeviceIndex>(index));
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return at::empty({bytes}, options);
  static auto* kept = new std::map<std::pair<int, ntl_stream_t>, Tensor>();
  if (kept->size() > 64) kept->clear();
  Tensor& work = (*kept)[{index, stream_of(index)}];
  if (!work.defined() || work.numel() < bytes) work = at::empty({bytes}, options);
  return work;
}

Tensor pool_workspace(const char* name, int64_t pages, int64_t n, int index, uint64_t* bytes) {
  check(name, ntl_cache_workspace_size(pages, n, bytes));
  return workspace(static_cast<int64_t>(*bytes), index);
}

PyObject* wrap(Tensor x) { return THPVariable_Wrap(std::move(x)); }

// ------------------------------------------------------------------------------ attention

bool overlaps(const Tensor& out, const Tensor& x) {
  if (!x.numel() || !out.numel()) return false;
  const char* begin = static_cast<const char*>(out.data_ptr());
  const char* from = static_cast<const char*>(x.data_ptr());
  int64_t reach = 1;
  for (int64_t d = 0; d < x.dim(); ++d) reach += (x.size(d) - 1) * x.stride(d);
  return from < begin + out.numel() * 2 && begin < from + reach * 2;
}

// (q, k, v, table, lens, q_lens or None, tree or None, window, sinks, scale or None, out or None)
PyObject* attend(PyObject* const* a) {
  const Cache cache = cache_of(a[1], a[2], false, false);
  const ntl_cache_t& c = cache.c;
  const Tensor& q = values("q", a[0]);
  const int index = cache.index;
  if (q.dim() != 4)
    raise(PyExc_ValueError, "q: expected 4 dimensions [seqs, tokens, heads, head_dim], got shape %s",
          shape_text(q.sizes()).c_str());
  const int64_t seqs = q.size(0), tokens = q.size(1), heads = q.size(2), dim = q.size(3);
  if (q.scalar_type() != cache.k->scalar_type())
    raise(PyExc_ValueError, "q: expected dtype %s like the cache, got %s", type_name(*cache.k), type_name(q));
  if (dim != c.head_dim || (dim != 64 && dim != 128))
    raise(PyExc_ValueError, "head_dim must be 64 or 128, the same for q (%lld) and the cache (%lld)", (long long)dim,
          (long long)c.head_dim);
  if (c.page_size % 8) raise(PyExc_ValueError, "page_size %lld is not a multiple of 8", (long long)c.page_size);
  if (!c.kv_heads || heads % c.kv_heads || heads / c.kv_heads > 128)
    raise(PyExc_ValueError, "%lld query heads cannot share %lld key heads (a whole number, up to 128 each)",
          (long long)heads, (long long)c.kv_heads);
  same_device(q, index);
  const Tensor& table = ints("table", a[3], index, {seqs, -1});
  const Tensor& lens = ints("lens", a[4], index, {seqs});
  const int32_t* q_lens = a[5] == Py_None ? nullptr : int_ptr(ints("q_lens", a[5], index, {seqs}));
  const Tensor* tree = nullptr;
  int64_t tree_stride = 0;
  if (a[6] != Py_None) {
    const int64_t words = (tokens + 31) / 32;
    const Tensor& x = tensor_of("tree", a[6]);
    const bool shared = x.dim() == 3 && x.size(0) == 1;
    tree = &ints("tree", a[6], index, {shared ? 1 : seqs, tokens, words});
    if (tokens > 1 && x.stride(1) != words) raise(PyExc_ValueError, "tree must be dense along its last two dimensions");
    tree_stride = shared ? 0 : x.stride(0);
  }
  double scale = 1.0 / std::sqrt(static_cast<double>(dim));
  if (a[9] != Py_None) {
    scale = PyFloat_AsDouble(a[9]);
    if (scale == -1.0 && PyErr_Occurred()) throw Raised();
    if (!(scale > 0 && scale < 1e30)) raise(PyExc_ValueError, "scale must be positive and finite, got %g", scale);
  }
  Device device(index);
  Tensor out;
  if (a[10] == Py_None) {
    out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  } else {
    out = values("out", a[10]);
    if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !out.is_contiguous() || out.get_device() != index)
      raise(PyExc_ValueError, "out must be a contiguous %s tensor of shape %s on q's device", type_name(q),
            shape_text(q.sizes()).c_str());
    const Tensor* others[3] = {&q, cache.k, cache.v};
    const char* names[3] = {"q", "k", "v"};
    for (int i = 0; i < 3; ++i)
      if (overlaps(out, *others[i]))
        raise(PyExc_ValueError, "Tensor arguments %s and out must have disjoint storage", names[i]);
  }
  if (!out.numel()) return wrap(out);
  const ntl_query_t query = {q.data_ptr(), out.data_ptr(), int_ptr(table), int_ptr(lens), q_lens, seqs, tokens, heads,
                             q.stride(0), q.stride(1), q.stride(2), table.stride(0), table.size(1), scale};
  uint64_t bytes = 0;
  check("ntl_cache_attention_workspace", ntl_cache_attention_workspace(&c, &query, &bytes));
  const Tensor work = workspace(static_cast<int64_t>(bytes), index);
  if (tree)
    check("ntl_tree_attention", ntl_tree_attention(&c, &query, reinterpret_cast<const uint32_t*>(int_ptr(*tree)), tree_stride,
                                                   work.data_ptr(), bytes, stream_of(index)));
  else
    check("ntl_window_attention",
          ntl_window_attention(&c, &query, int_of(a[7]), int_of(a[8]), work.data_ptr(), bytes, stream_of(index)));
  return wrap(out);
}

// (parents)
PyObject* tree_mask(PyObject* const* a) {
  const int index = tensor_of("parents", a[0]).get_device();
  const Tensor& parents = ints("parents", a[0], index, {-1, -1});
  Device device(index);
  const int64_t seqs = parents.size(0), tokens = parents.size(1);
  Tensor words = new_ints({seqs, tokens, (tokens + 31) / 32}, index);
  check("ntl_tree_mask", ntl_tree_mask(int_ptr(parents), parents.stride(0), seqs, tokens,
                                       reinterpret_cast<uint32_t*>(int_ptr(words)), stream_of(index)));
  return wrap(words);
}

// ------------------------------------------------------------------------------ cache operators

// (k, v, k_new, v_new, table, lens, counts or None) -> new lengths
PyObject* append_tokens(PyObject* const* a) {
  const Cache cache = cache_of(a[0], a[1], true, true);
  const ntl_cache_t& c = cache.c;
  const Tensor& k_new = values("k_new", a[2]);
  const Tensor& v_new = values("v_new", a[3]);
  const int index = cache.index;
  if (k_new.dim() != cache.k->dim())
    raise(PyExc_ValueError, "k_new: expected %lld dimensions, got shape %s", (long long)cache.k->dim(),
          shape_text(k_new.sizes()).c_str());
  const int64_t at = cache.layered ? 1 : 0, seqs = k_new.size(at), tokens = k_new.size(at + 1);
  if ((cache.layered && k_new.size(0) != c.layers) || k_new.size(at + 2) != c.kv_heads || k_new.size(at + 3) != c.head_dim ||
      k_new.scalar_type() != cache.k->scalar_type())
    raise(PyExc_ValueError, "k_new: expected %s rows of the cache's layers, heads and head_dim, got %s %s",
          type_name(*cache.k), type_name(k_new), shape_text(k_new.sizes()).c_str());
  if (v_new.sizes() != k_new.sizes() || v_new.strides() != k_new.strides() || v_new.scalar_type() != k_new.scalar_type())
    raise(PyExc_ValueError, "k_new and v_new must have the same shape, strides and dtype");
  same_device(k_new, index);
  same_device(v_new, index);
  const Tensor& table = ints("table", a[4], index, {seqs, -1});
  const Tensor& lens = ints("lens", a[5], index, {seqs});
  const int32_t* counts = a[6] == Py_None ? nullptr : int_ptr(ints("counts", a[6], index, {seqs}));
  Device device(index);
  Tensor out = new_ints({seqs}, index);
  check("ntl_cache_append",
        ntl_cache_append(&c, k_new.data_ptr(), v_new.data_ptr(), cache.layered ? k_new.stride(0) : 0, k_new.stride(at),
                         k_new.stride(at + 1), k_new.stride(at + 2), int_ptr(table), table.stride(0), seqs, table.size(1),
                         int_ptr(lens), counts, tokens, int_ptr(out), stream_of(index)));
  return wrap(out);
}

// (k, v, table, lens, path, counts, drafts: int or tensor) -> new lengths
PyObject* accept_path(PyObject* const* a) {
  const Cache cache = cache_of(a[0], a[1], true, true);
  const int index = cache.index;
  const Tensor& lens = ints("lens", a[3], index, {-1});
  const int64_t seqs = lens.size(0);
  const Tensor& table = ints("table", a[2], index, {seqs, -1});
  const Tensor& path = ints("path", a[4], index, {seqs, -1});
  const Tensor& counts = ints("counts", a[5], index, {seqs});
  const int32_t* each = nullptr;
  int64_t common = 0;
  if (THPVariable_Check(a[6])) {
    each = int_ptr(ints("drafts", a[6], index, {seqs}));
  } else if ((common = int_of(a[6])) < 0) {
    raise(PyExc_ValueError, "drafts must be at least 0, got %lld", (long long)common);
  }
  Device device(index);
  Tensor out = new_ints({seqs}, index);
  check("ntl_cache_accept",
        ntl_cache_accept(&cache.c, int_ptr(table), table.stride(0), seqs, table.size(1), int_ptr(lens), each, common,
                         int_ptr(path), path.stride(0), path.size(1), int_ptr(counts), int_ptr(out), stream_of(index)));
  return wrap(out);
}

// (k, v, src, dst)
PyObject* copy_pages(PyObject* const* a) {
  const Cache cache = cache_of(a[0], a[1], true, true);
  const Tensor& src = ints("src", a[2], cache.index, {-1});
  const Tensor& dst = ints("dst", a[3], cache.index, {src.size(0)});
  Device device(cache.index);
  check("ntl_cache_copy_pages",
        ntl_cache_copy_pages(&cache.c, int_ptr(src), int_ptr(dst), src.size(0), stream_of(cache.index)));
  Py_RETURN_NONE;
}

struct Sequences {
  const Tensor &table, &lens, &refs;
};

Sequences sequences_of(PyObject* table, PyObject* lens, PyObject* refs, int64_t pages, int index) {
  const Tensor& t = written_table("table", ints("table", table, index, {-1, -1}));
  return {t, ints("lens", lens, index, {t.size(0)}), ints("refs", refs, index, {pages})};
}

// (k, v, table, lens, refs, src, dst) -> granted
PyObject* fork(PyObject* const* a) {
  const Cache cache = cache_of(a[0], a[1], true, true);
  const int index = cache.index;
  const Sequences s = sequences_of(a[2], a[3], a[4], cache.c.pages, index);
  const Tensor& src = ints("src", a[5], index, {-1});
  const int64_t n = src.size(0);
  const Tensor& dst = ints("dst", a[6], index, {n});
  Device device(index);
  Tensor granted = new_ints({n}, index);
  uint64_t bytes = 0;
  const Tensor work = pool_workspace("ntl_cache_workspace_size", cache.c.pages, n, index, &bytes);
  check("ntl_cache_fork",
        ntl_cache_fork(&cache.c, int_ptr(s.table), s.table.stride(0), s.table.size(0), s.table.size(1), int_ptr(s.lens),
                       int_ptr(s.refs), int_ptr(src), int_ptr(dst), n, int_ptr(granted), work.data_ptr(), bytes,
                       stream_of(index)));
  return wrap(granted);
}

// (table, lens, refs, seqs, extra: int or tensor, page_size) -> granted
PyObject* reserve(PyObject* const* a) {
  const int index = tensor_of("table", a[0]).get_device();
  const Sequences s = sequences_of(a[0], a[1], a[2], -1, index);
  const Tensor& seqs = ints("seqs", a[3], index, {-1});
  const int64_t n = seqs.size(0), pages = s.refs.size(0), page_size = int_of(a[5]);
  const int32_t* each = nullptr;
  int64_t common = 0;
  if (THPVariable_Check(a[4])) {
    each = int_ptr(ints("extra", a[4], index, {n}));
  } else if ((common = int_of(a[4])) < 0) {
    raise(PyExc_ValueError, "extra must be at least 0, got %lld", (long long)common);
  }
  if (page_size < 1) raise(PyExc_ValueError, "page_size must be at least 1, got %lld", (long long)page_size);
  Device device(index);
  Tensor granted = new_ints({n}, index);
  uint64_t bytes = 0;
  const Tensor work = pool_workspace("ntl_cache_workspace_size", pages, n, index, &bytes);
  check("ntl_cache_reserve",
        ntl_cache_reserve(pages, page_size, int_ptr(s.table), s.table.stride(0), s.table.size(0), s.table.size(1),
                          int_ptr(s.lens), int_ptr(s.refs), int_ptr(seqs), n, common, each, int_ptr(granted),
                          work.data_ptr(), bytes, stream_of(index)));
  return wrap(granted);
}

// (table, lens, refs, seqs)
PyObject* free_sequences(PyObject* const* a) {
  const int index = tensor_of("table", a[0]).get_device();
  const Sequences s = sequences_of(a[0], a[1], a[2], -1, index);
  const Tensor& seqs = ints("seqs", a[3], index, {-1});
  Device device(index);
  check("ntl_cache_free",
        ntl_cache_free(s.refs.size(0), int_ptr(s.table), s.table.stride(0), s.table.size(0), s.table.size(1), int_ptr(s.lens),
                       int_ptr(s.refs), int_ptr(seqs), seqs.size(0), stream_of(index)));
  Py_RETURN_NONE;
}

// (k, v, table, refs, table_out, refs_out) -> live pages
PyObject* compact(PyObject* const* a) {
  const Cache cache = cache_of(a[0], a[1], true, true);
  const int index = cache.index;
  const Tensor& table = ints("table", a[2], index, {-1, -1});
  const Tensor& refs = ints("refs", a[3], index, {cache.c.pages});
  const Tensor& table_out = written_table("table_out", ints("table_out", a[4], index, {table.size(0), table.size(1)}));
  const Tensor& refs_out = ints("refs_out", a[5], index, {cache.c.pages});
  Device device(index);
  Tensor live = new_ints({1}, index);
  uint64_t bytes = 0;
  const Tensor work = pool_workspace("ntl_cache_workspace_size", cache.c.pages, 0, index, &bytes);
  check("ntl_cache_compact",
        ntl_cache_compact(&cache.c, int_ptr(table), table.stride(0), int_ptr(table_out), table_out.stride(0), table.size(0),
                          table.size(1), int_ptr(refs), int_ptr(refs_out), int_ptr(live), work.data_ptr(), bytes,
                          stream_of(index)));
  return wrap(live);
}

// A module function of exactly N positional arguments, with C++ exceptions turned into Python's.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, received %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define NTL_ENTRY(name, function, n) \
  {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<function, n>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {NTL_ENTRY("attend", attend, 11),
                         NTL_ENTRY("tree_mask", tree_mask, 1),
                         NTL_ENTRY("append_tokens", append_tokens, 7),
                         NTL_ENTRY("accept_path", accept_path, 7),
                         NTL_ENTRY("copy_pages", copy_pages, 4),
                         NTL_ENTRY("fork", fork, 7),
                         NTL_ENTRY("reserve", reserve, 6),
                         NTL_ENTRY("free", free_sequences, 4),
                         NTL_ENTRY("compact", compact, 6),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged() { return PyModule_Create(&module); }
