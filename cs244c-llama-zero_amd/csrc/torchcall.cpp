// Tensor-level entry of generation's operators (lzhip/ops.py: kv_cache_write,
// kv_cache_read, paged_attention, process_logits, and for drafted tokens
// cache_tables, verify_draft, kv_cache_keep): arguments checked, outputs
// and workspaces allocated and the C ABI called in compiled code.  A decoded
// token's kernels run for 4 to 5 us each; with the checks and allocations in
// Python a call took 9.6 us of host time, so it takes 4.8, 3 of them the launch.
//
// bind(addresses, raw_stream, get_device, set_device, error) hands over the
// library's entry points ({name: address}), torch's current-stream and device
// functions and the exception of a failed call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>

#include "../../include/llamazero_hip.h"

namespace {

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(PyObject* type, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  PyErr_FormatV(type, fmt, ap);
  va_end(ap);
  throw Refused{};
}

decltype(&lz_kv_write) p_write = nullptr;
decltype(&lz_kv_read) p_read = nullptr;
decltype(&lz_paged_attn) p_attn = nullptr;
decltype(&lz_paged_attn_workspace) p_attn_ws = nullptr;
decltype(&lz_process_logits) p_logits = nullptr;
decltype(&lz_kv_write_at) p_write_at = nullptr;
decltype(&lz_kv_keep) p_keep = nullptr;
decltype(&lz_tree_attn) p_tree = nullptr;
decltype(&lz_tree_attn_workspace) p_tree_ws = nullptr;
decltype(&lz_cache_tables) p_tables = nullptr;
decltype(&lz_verify_draft) p_verify = nullptr;
decltype(&lz_verify_workspace) p_verify_ws = nullptr;
decltype(&lz_copy2d) p_copy = nullptr;
decltype(&lz_fill) p_fill = nullptr;
decltype(&lz_last_error) p_error = nullptr;
PyObject *g_stream = nullptr, *g_get = nullptr, *g_set = nullptr, *g_failure = nullptr;

// ---- arguments ------------------------------------------------------------

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

void require_gpu(const at::Tensor& t) {
  if (!t.is_cuda())
    refuse(PyExc_RuntimeError,
           "llama-zero HIP kernels run on a ROCm GPU; got a tensor on %s. Move the model and inputs to 'cuda'.",
           t.device().str().c_str());
}

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{};
  return v;
}

PyObject* item(PyObject* tuple, Py_ssize_t i, Py_ssize_t n, const char* name) {
  if (!PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) != n)
    refuse(PyExc_TypeError, "expected a %s, got %s", name, Py_TYPE(tuple)->tp_name);
  return PyTuple_GET_ITEM(tuple, i);
}

std::string shape(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

const char* type_name(const at::Tensor& t) { return c10::toString(t.scalar_type()); }

int code_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return LZ_F32;
    case at::kBFloat16: return LZ_BF16;
    case at::kHalf: return LZ_F16;
    default:
      refuse(PyExc_TypeError, "llama-zero HIP kernels support float32, bfloat16 and float16 tensors, got %s", type_name(t));
  }
}

template <typename T = void>
T* address(const at::Tensor* t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// The device and stream of a call; other arguments must be on the device, and
// it is the current one until the call ends (a kernel goes to the current
// device, whatever its stream belongs to).
struct Place {
  c10::DeviceIndex index;
  int64_t back = -1;
  void* stream = nullptr;

  explicit Place(const at::Tensor& t) {
    require_gpu(t);
    index = t.get_device();
    PyObject* now = PyObject_CallNoArgs(g_get);
    if (!now) throw Refused{};
    const long current = PyLong_AsLong(now);
    Py_DECREF(now);
    if (current != index) {
      set(index);
      back = current;
    }
    PyObject* i = PyLong_FromLong(index);
    PyObject* s = i ? PyObject_CallOneArg(g_stream, i) : nullptr;
    Py_XDECREF(i);
    if (!s) {
      leave();
      throw Refused{};
    }
    stream = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
  }
  ~Place() { leave(); }
  Place(const Place&) = delete;
  Place& operator=(const Place&) = delete;

  static void set(long i) {
    PyObject* r = PyObject_CallFunction(g_set, "l", i);
    if (!r) throw Refused{};
    Py_DECREF(r);
  }
  void leave() {
    if (back < 0) return;
    PyObject *type, *value, *trace;
    PyErr_Fetch(&type, &value, &trace);
    PyObject* r = PyObject_CallFunction(g_set, "l", (long)back);
    Py_XDECREF(r);
    PyErr_Restore(type, value, trace);
    back = -1;
  }
  bool here(const at::Tensor& t) const { return t.is_cuda() && t.get_device() == index; }
};

template <typename F, typename... A>
void call(const char* name, F* fn, A... args) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(args...);
  Py_END_ALLOW_THREADS
  if (rc != 0) refuse(g_failure, "%s failed (%d): %s", name, rc, p_error());
}

at::Tensor fresh(const at::Tensor& like, at::IntArrayRef size, at::ScalarType type) {
  return at::empty(size, like.options().dtype(type));
}

void int32_table(const at::Tensor& t, const char* name, const Place& at, int64_t dim) {
  if (t.scalar_type() == at::kInt && t.dim() == dim && t.is_contiguous() && at.here(t)) return;
  require_gpu(t);
  refuse(PyExc_ValueError, "%s must be a contiguous int32 tensor of %d dimension(s) on cuda:%d, got %s %s on %s", name,
         (int)dim, (int)at.index, type_name(t), shape(t).c_str(), t.device().str().c_str());
}

// A LayerCache, checked against rows of `type`.
struct Cache {
  const at::Tensor *k, *v, *ke, *ve;
  int code;
  int64_t pages, KV, size, hd;

  Cache(PyObject* layer, at::ScalarType type, const Place& at) {
    k = &tensor(item(layer, 0, 4, "LayerCache"), "layer.k");
    v = &tensor(item(layer, 1, 4, "LayerCache"), "layer.v");
    ke = maybe(item(layer, 2, 4, "LayerCache"), "layer.k_exp");
    ve = maybe(item(layer, 3, 4, "LayerCache"), "layer.v_exp");
    for (const at::Tensor* t : {k, v, ke, ve})
      if (t && !at.here(*t)) {
        require_gpu(*t);
        refuse(PyExc_ValueError, "the cache is on %s, the rows on cuda:%d", t->device().str().c_str(), (int)at.index);
      }
    const at::ScalarType stored = k->scalar_type();
    if (k->dim() != 4 || v->sizes() != k->sizes() || v->scalar_type() != stored || !k->is_contiguous() || !v->is_contiguous())
      refuse(PyExc_ValueError,
             "cache pages must be two contiguous [pages, KV heads, page size, head dim] tensors of one dtype, got %s %s "
             "and %s %s", type_name(*k), shape(*k).c_str(), type_name(*v), shape(*v).c_str());
    if (stored == at::kFloat8_e4m3fn) {
      for (const at::Tensor* e : {ke, ve})
        if (!e || e->scalar_type() != at::kChar || e->sizes() != k->sizes().slice(0, 3) || !e->is_contiguous())
          refuse(PyExc_ValueError, "a float8_e4m3fn cache needs contiguous int8 exponents [pages, KV heads, page size] "
                                   "beside it");
      code = LZ_E4M3;
    } else {
      if (stored != type || ke || ve)
        refuse(PyExc_TypeError, "a cache of %s %s exponents does not hold %s rows", type_name(*k),
               ke || ve ? "with" : "without", c10::toString(type));
      code = code_of(*k);
    }
    pages = k->size(0);
    KV = k->size(1);
    size = k->size(2);
    hd = k->size(3);
  }
};

constexpr Py_ssize_t kDraft = 10;  // fields of a DraftStep
bool is_draft(PyObject* step) { return PyTuple_Check(step) && PyTuple_GET_SIZE(step) == kDraft; }

// A CacheStep or a DraftStep, checked.
struct Step {
  const at::Tensor *start, *len, *table;
  const at::Tensor *base = nullptr, *positions = nullptr, *mask = nullptr;  // of a DraftStep
  int64_t rows, max_new, max_len, B, width;

  // x: the call's rows, of which there may be more than the step has
  Step(PyObject* step, const at::Tensor& x, const Place& at) {
    const bool draft = is_draft(step);
    const Py_ssize_t fields = draft ? kDraft : 6;
    const char* type = draft ? "DraftStep" : "CacheStep";
    start = &tensor(item(step, 0, fields, type), "row_start");
    len = &tensor(item(step, 1, fields, type), "kv_len");
    table = &tensor(item(step, 2, fields, type), "page_table");
    rows = integer(item(step, 3, fields, type));
    max_new = integer(item(step, 4, fields, type));
    max_len = integer(item(step, 5, fields, type));
    int32_table(*start, "row_start", at, 1);
    int32_table(*len, "kv_len", at, 1);
    int32_table(*table, "page_table", at, 2);
    B = len->size(0);
    width = table->size(1);
    if (B == 0 || width == 0 || start->size(0) != B + 1 || table->size(0) != B)
      refuse(PyExc_ValueError, "a step of %lld sequences needs %lld row starts and a page table of %lld rows, got %lld and "
                               "%s", (long long)B, (long long)B + 1, (long long)B, (long long)start->size(0),
             shape(*table).c_str());
    const int64_t n = x.dim() == 2 ? x.size(0) : INT64_MAX;  // other shapes are refused as rows
    if (rows < 0 || rows > n || max_new < 0 || max_len < 0 || (max_new < rows && B * max_new < rows))
      refuse(PyExc_ValueError, "a step of %lld rows, at most %lld of each of %lld sequences and %lld cached, does not fit "
                               "rows %s", (long long)rows, (long long)max_new, (long long)B, (long long)max_len,
             shape(x).c_str());
    if (!draft) return;
    base = &tensor(PyTuple_GET_ITEM(step, 6), "base");
    positions = &tensor(PyTuple_GET_ITEM(step, 7), "positions");
    mask = maybe(PyTuple_GET_ITEM(step, 9), "mask");
    int32_table(*base, "base", at, 1);
    int32_table(*positions, "positions", at, 1);
    if (mask) int32_table(*mask, "mask", at, 2);
    if (base->size(0) != B || positions->size(0) < rows || (mask && (mask->size(0) < rows || mask->size(1) == 0)))
      refuse(PyExc_ValueError, "a draft of %lld sequences and %lld rows does not fit base %s, positions %s and mask %s",
             (long long)B, (long long)rows, shape(*base).c_str(), shape(*positions).c_str(),
             mask ? shape(*mask).c_str() : "None");
  }
};

// 2-D rows of `cols` whose starts are 16-byte aligned: t's, or a copy.
struct Rows {
  at::Tensor t;
  int64_t rows, ld;

  Rows(const at::Tensor& x, const char* name, int64_t cols, int code, const Place& at) : t(x) {
    if (x.dim() != 2 || x.size(1) != cols || (cols > 1 && x.stride(1) != 1))
      refuse(PyExc_ValueError, "%s must be rows of %lld adjacent values, got %s", name, (long long)cols, shape(x).c_str());
    rows = x.size(0);
    ld = rows > 1 ? x.stride(0) : cols;
    if (ld < cols) refuse(PyExc_ValueError, "%s: rows overlap (stride %lld)", name, (long long)ld);
    if (rows > 0 && (!aligned(x) || ld * x.element_size() % 16)) {
      t = fresh(x, {rows, cols}, x.scalar_type());
      call("lz_copy2d", p_copy, (const void*)x.data_ptr(), ld, t.data_ptr(), cols, rows, cols, code, at.stream);
      ld = cols;
    }
  }
};

// The output rows: the caller's, whose rows of no sequence are left as they
// are, or new ones, where those are zeros.
struct Out {
  at::Tensor t;
  int64_t ld;

  Out(PyObject* given, const at::Tensor& like, int64_t rows, int64_t cols, int64_t used, int code, const Place& at) {
    ld = cols;
    if (given == Py_None) {
      t = fresh(like, {rows, cols}, like.scalar_type());
      if (used != rows && rows > 0) call("lz_fill", p_fill, t.data_ptr(), code, rows * cols, 0.0, at.stream);
      return;
    }
    t = tensor(given, "out");
    require_gpu(t);
    const bool rows_fit = t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.stride(1) == 1;
    if (rows_fit && rows > 1) ld = t.stride(0);
    if (!rows_fit || t.scalar_type() != like.scalar_type() || !at.here(t) || ld < cols || !aligned(t) ||
        ld * t.element_size() % 16)
      refuse(PyExc_ValueError, "out must be %s rows [%lld, %lld] on cuda:%d, 16-byte aligned", type_name(like),
             (long long)rows, (long long)cols, (int)at.index);
  }
};

// Refuses an output that lies over values of the input rows x which other
// threads may read after it is written.  The same rows from their first column
// on are fine (a thread reads what it writes there first: `first` columns), and so
// are columns beside x's.
void require_apart(const Out& out, const Rows& x, int64_t cols, int64_t first) {
  const at::Tensor &o = out.t, &t = x.t;
  const int64_t n = o.size(1), esz = t.element_size();
  if (x.rows == 0 || n == 0) return;
  const char *a = static_cast<const char*>(t.data_ptr()), *b = static_cast<const char*>(o.data_ptr());
  const int64_t a_end = ((x.rows - 1) * x.ld + cols) * esz, b_end = ((x.rows - 1) * out.ld + n) * esz;
  if (a + a_end <= b || b + b_end <= a) return;
  if (x.ld == out.ld || x.rows == 1) {
    if (a == b && n <= first) return;
    const int64_t ld = x.ld * esz, off = ((b - a) % ld + ld) % ld;
    if (x.rows > 1 && off >= cols * esz && off + n * esz <= ld) return;
  }
  refuse(PyExc_ValueError, "out overlaps the rows that the call reads");
}

// Runs a call's body; nothing but a Python exception leaves it.
template <typename F>
PyObject* guarded(const F& body) {
  try {
    return body();
  } catch (const Refused&) {
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());  // torch's classes for its allocator's errors
  }
  return nullptr;
}

void expect(Py_ssize_t got, Py_ssize_t want) {
  if (p_write == nullptr) refuse(PyExc_RuntimeError, "bind() first");
  if (got != want) refuse(PyExc_TypeError, "this function takes %zd arguments (%zd given)", want, got);
}

// ---- the cache's and the logits' calls -------------------------------------------------------

PyObject* kv_cache_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 7);
    const at::Tensor& x = tensor(a[0], "qkv");
    const Place at(x);
    const int code = code_of(x);
    const Cache c(a[1], x.scalar_type(), at);
    const Step s(a[2], x, at);
    const int64_t H = integer(a[3]);
    const at::Tensor &cos = tensor(a[4], "cos"), &sin = tensor(a[5], "sin");
    const Rows qkv(x, "qkv", (H + 2 * c.KV) * c.hd, code, at);
    for (const at::Tensor* t : {&cos, &sin}) {
      require_gpu(*t);
      if (t->scalar_type() != x.scalar_type() || t->dim() != 2 || t->size(1) != c.hd || !t->is_contiguous() ||
          !at.here(*t) || !aligned(*t) || t->size(0) < s.max_len || t->size(0) != cos.size(0))
        refuse(PyExc_ValueError, "RoPE tables must be contiguous %s [%lld or more, %lld] on cuda:%d, got %s %s", type_name(x),
               (long long)s.max_len, (long long)c.hd, (int)at.index, type_name(*t), shape(*t).c_str());
    }
    const Out q(a[6], x, qkv.rows, H * c.hd, s.rows, code, at);
    require_apart(q, qkv, (H + 2 * c.KV) * c.hd, H * c.hd);
    if (s.positions) {
      call("lz_kv_write_at", p_write_at, (const void*)qkv.t.data_ptr(), qkv.ld, code, s.rows, (const void*)cos.data_ptr(),
           (const void*)sin.data_ptr(), cos.size(0), q.t.data_ptr(), q.ld, address(c.k), address(c.v), address(c.ke),
           address(c.ve), c.code, c.pages, c.size, (const int32_t*)address<int32_t>(s.table), s.width,
           (const int32_t*)address<int32_t>(s.start), (const int32_t*)address<int32_t>(s.len),
           (const int32_t*)address<int32_t>(s.positions), s.B, H, c.KV, c.hd, at.stream);
      return THPVariable_Wrap(q.t);
    }
    call("lz_kv_write", p_write, (const void*)qkv.t.data_ptr(), qkv.ld, code, qkv.rows, (const void*)cos.data_ptr(),
         (const void*)sin.data_ptr(), cos.size(0), q.t.data_ptr(), q.ld, address(c.k), address(c.v), address(c.ke),
         address(c.ve), c.code, c.pages, c.size, (const int32_t*)address<int32_t>(s.table), s.width,
         (const int32_t*)address<int32_t>(s.start), (const int32_t*)address<int32_t>(s.len), s.B, H, c.KV, c.hd, at.stream);
    return THPVariable_Wrap(q.t);
  });
}

PyObject* kv_cache_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 5);
    const at::Tensor &table = tensor(a[1], "page_table"), &start = tensor(a[2], "start");
    const Place at(table);
    const int64_t rows = integer(a[3]);
    if (!THPDtype_Check(a[4])) refuse(PyExc_TypeError, "dtype must be a torch dtype, got %s", Py_TYPE(a[4])->tp_name);
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    if (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf)
      refuse(PyExc_TypeError, "a cache is read back in float32, bfloat16 or float16, not in %s", c10::toString(type));
    const Cache c(a[0], type, at);
    int32_table(table, "page_table", at, 2);
    int32_table(start, "start", at, 1);
    const int64_t B = table.size(0), width = table.size(1);
    if (start.size(0) != B + 1 || B == 0 || width == 0 || rows < 0)
      refuse(PyExc_ValueError, "%lld sequences need %lld starts, got %lld", (long long)B, (long long)B + 1,
             (long long)start.size(0));
    const at::Tensor k = fresh(table, {rows, c.KV * c.hd}, type), v = fresh(table, {rows, c.KV * c.hd}, type);
    call("lz_kv_read", p_read, (const void*)address(c.k), (const void*)address(c.v), (const void*)address(c.ke),
         (const void*)address(c.ve), c.code, c.pages, c.size, (const int32_t*)address<int32_t>(&table), width,
         (const int32_t*)address<int32_t>(&start), B, c.KV, c.hd, k.data_ptr(), v.data_ptr(), code_of(k), rows, at.stream);
    PyObject* two = PyTuple_New(2);
    if (!two) throw Refused{};
    PyTuple_SET_ITEM(two, 0, THPVariable_Wrap(k));
    PyTuple_SET_ITEM(two, 1, THPVariable_Wrap(v));
    return two;
  });
}

PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 6);
    const at::Tensor& x = tensor(a[0], "q");
    const Place at(x);
    const int code = code_of(x);
    const Cache c(a[1], x.scalar_type(), at);
    const Step s(a[2], x, at);
    const int64_t H = integer(a[3]);
    const double scale = PyFloat_AsDouble(a[4]);
    if (scale == -1.0 && PyErr_Occurred()) throw Refused{};
    if (H <= 0 || c.KV == 0 || H % c.KV)
      refuse(PyExc_ValueError, "%lld query heads do not divide over %lld key/value heads", (long long)H, (long long)c.KV);
    const Rows q(x, "q", H * c.hd, code, at);
    const Out o(a[5], x, q.rows, H * c.hd, s.rows, code, at);
    require_apart(o, q, H * c.hd, H * c.hd);
    const int64_t bytes = s.mask ? p_tree_ws(code, c.code, s.rows, s.B, H, c.KV, c.hd, s.max_new, s.max_len)
                                 : p_attn_ws(code, c.code, q.rows, s.B, H, c.KV, c.hd, s.max_new, s.max_len);
    at::Tensor ws;
    if (bytes) ws = fresh(x, {(bytes + 3) / 4}, at::kFloat);
    if (s.mask) {
      call("lz_tree_attn", p_tree, (const void*)q.t.data_ptr(), q.ld, code, s.rows, (const void*)address(c.k),
           (const void*)address(c.v), (const void*)address(c.ke), (const void*)address(c.ve), c.code, c.pages, c.size,
           (const int32_t*)address<int32_t>(s.table), s.width, (const int32_t*)address<int32_t>(s.start),
           (const int32_t*)address<int32_t>(s.len), (const int32_t*)address<int32_t>(s.base),
           (const int32_t*)address<int32_t>(s.mask), s.mask->size(1), s.B, H, c.KV, c.hd, s.max_new, s.max_len,
           (float)scale, o.t.data_ptr(), o.ld, bytes ? ws.data_ptr() : nullptr, bytes, at.stream);
      return THPVariable_Wrap(o.t);
    }
    call("lz_paged_attn", p_attn, (const void*)q.t.data_ptr(), q.ld, code, q.rows, (const void*)address(c.k),
         (const void*)address(c.v), (const void*)address(c.ke), (const void*)address(c.ve), c.code, c.pages, c.size,
         (const int32_t*)address<int32_t>(s.table), s.width, (const int32_t*)address<int32_t>(s.start),
         (const int32_t*)address<int32_t>(s.len), s.B, H, c.KV, c.hd, s.max_new, s.max_len, (float)scale, o.t.data_ptr(),
         o.ld, bytes ? ws.data_ptr() : nullptr, bytes, at.stream);
    return THPVariable_Wrap(o.t);
  });
}

// A penalty: one fp32 value a row, or one for all.
struct Penalty {
  const float* rows = nullptr;
  float all = 0.f;

  Penalty(PyObject* o, const char* name, int64_t B, bool positive, const Place& at) {
    if (THPVariable_Check(o)) {
      const at::Tensor& t = THPVariable_Unpack(o);
      if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != B || !t.is_contiguous() || !at.here(t)) {
        require_gpu(t);
        refuse(PyExc_ValueError, "%s must be a number or a contiguous float32 [%lld] tensor on cuda:%d", name, (long long)B,
               (int)at.index);
      }
      rows = static_cast<const float*>(t.data_ptr());
      return;
    }
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused{};
    all = (float)v;
    if (!std::isfinite(all) || (positive && all <= 0.f))
      refuse(PyExc_ValueError, "%s must be finite%s in float32, got %R", name, positive ? " and positive" : "", o);
  }
};

at::Tensor row_lengths(const at::Tensor* t, const char* name, int64_t B, const Place& at) {
  if (!t) return {};
  const bool narrow = t->scalar_type() == at::kInt;
  if ((!narrow && t->scalar_type() != at::kLong) || t->dim() != 1 || t->size(0) != B || !at.here(*t)) {
    require_gpu(*t);
    refuse(PyExc_ValueError, "%s must be an int32 or int64 [%lld] tensor on cuda:%d", name, (long long)B, (int)at.index);
  }
  if (narrow) return t->contiguous();
  return t->clamp(0, INT32_MAX).to(at::kInt).contiguous();  // a text is shorter than that
}

// Rows of `cols` of a [cols] or [B, cols] tensor: their stride, 0 for one row
// that serves all, -1 where the tensor is neither.
int64_t row_stride(const at::Tensor& t, int64_t B, int64_t cols) {
  const bool one = t.dim() == 1 && t.size(0) == cols, each = t.dim() == 2 && t.size(0) == B && t.size(1) == cols;
  if (!one && !each) return -1;
  if (cols > 1 && t.stride(-1) != 1) return -1;
  return one ? 0 : t.stride(0);
}

PyObject* process_logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 9);
    const at::Tensor& x = tensor(a[0], "logits");
    const Place at(x);
    const int code = code_of(x);
    if (x.dim() != 2) refuse(PyExc_ValueError, "logits must be [B, V], got %s", shape(x).c_str());
    const int64_t B = x.size(0), V = x.size(1);
    if ((V > 1 && x.stride(1) != 1) || (B > 1 && x.stride(0) < V))
      refuse(PyExc_ValueError, "logits rows must be adjacent values, got strides (%lld, %lld)", (long long)x.stride(0),
             (long long)x.stride(1));
    const at::Tensor *tokens = maybe(a[1], "tokens"), *len = maybe(a[2], "lengths"), *prompt = maybe(a[3], "prompt_lengths");
    int64_t T = 0, ldt = 0;
    if (tokens) {
      if (tokens->scalar_type() != at::kLong || tokens->dim() != 2 || tokens->size(0) != B || !at.here(*tokens) ||
          (tokens->size(1) > 1 && tokens->stride(1) != 1)) {
        require_gpu(*tokens);
        refuse(PyExc_ValueError, "tokens must be int64 [%lld, T] rows on cuda:%d", (long long)B, (int)at.index);
      }
      T = tokens->size(1);
      ldt = tokens->stride(0);
    } else if (len || prompt) {
      refuse(PyExc_ValueError, "lengths and prompt_lengths say which tokens count: there are none");
    }
    const at::Tensor lengths = row_lengths(len, "lengths", B, at), prompts = row_lengths(prompt, "prompt_lengths", B, at);
    const Penalty rep(a[4], "repetition_penalty", B, true, at), pres(a[5], "presence_penalty", B, false, at),
        freq(a[6], "frequency_penalty", B, false, at);
    const at::Tensor *bias = maybe(a[7], "bias"), *mask = maybe(a[8], "mask");
    int64_t ldb = 0, ldm = 0;
    int kind = 0;
    if (bias) {
      ldb = row_stride(*bias, B, V);
      if (bias->scalar_type() != at::kFloat || ldb < 0 || !at.here(*bias)) {
        require_gpu(*bias);
        refuse(PyExc_ValueError, "bias must be float32 [%lld] or [%lld, %lld] on cuda:%d", (long long)V, (long long)B,
               (long long)V, (int)at.index);
      }
    }
    if (mask) {
      kind = mask->scalar_type() == at::kBool ? 1 : mask->scalar_type() == at::kInt ? 2 : 0;
      const int64_t words = (V + 31) / 32;
      ldm = row_stride(*mask, B, kind == 2 ? words : V);
      if (!kind || ldm < 0 || !at.here(*mask)) {
        require_gpu(*mask);
        refuse(PyExc_ValueError, "mask must be bool [%lld] or [%lld, %lld], or int32 words of %lld, on cuda:%d",
               (long long)V, (long long)B, (long long)V, (long long)words, (int)at.index);
      }
    }
    const at::Tensor out = fresh(x, {B, V}, at::kFloat);
    call("lz_process_logits", p_logits, (const void*)x.data_ptr(), B > 1 ? x.stride(0) : V, code, B, V,
         (const int64_t*)address<int64_t>(tokens), ldt, T,
         lengths.defined() ? (const int32_t*)lengths.data_ptr() : nullptr,
         prompts.defined() ? (const int32_t*)prompts.data_ptr() : nullptr, rep.rows, rep.all, pres.rows, pres.all, freq.rows,
         freq.all, (const float*)address<float>(bias), ldb, (const void*)address(mask), kind, ldm,
         static_cast<float*>(out.data_ptr()), V, at.stream);
    return THPVariable_Wrap(out);
  });
}

// ---- drafted tokens -------------------------------------------------------

// An int32 [B] tensor.
const at::Tensor& per_sequence(const at::Tensor& t, const char* name, int64_t B, const Place& at) {
  int32_table(t, name, at, 1);
  if (t.size(0) != B) refuse(PyExc_ValueError, "%s must hold %lld values, got %lld", name, (long long)B, (long long)t.size(0));
  return t;
}

// The parents of trees: int32 [nodes], for all sequences, or [B, nodes].
struct Parents {
  const int32_t* at = nullptr;
  int64_t nodes = 0, ld = 0;

  Parents(PyObject* o, int64_t B, int64_t max_new, const Place& place) {
    const at::Tensor* t = maybe(o, "parents");
    if (!t) return;
    int32_table(*t, "parents", place, t->dim() == 1 ? 1 : 2);
    nodes = t->size(-1);
    if (nodes == 0 || nodes < max_new || (t->dim() == 2 && t->size(0) != B))
      refuse(PyExc_ValueError, "parents must be [nodes] or [%lld, nodes], of at least %lld nodes, got %s", (long long)B,
             (long long)max_new, shape(*t).c_str());
    at = static_cast<const int32_t*>(t->data_ptr());
    ld = t->dim() == 2 ? nodes : 0;
  }
};

PyObject* tuple_of(std::initializer_list<const at::Tensor*> tensors) {
  PyObject* t = PyTuple_New((Py_ssize_t)tensors.size());
  if (!t) throw Refused{};
  Py_ssize_t i = 0;
  for (const at::Tensor* x : tensors) {
    PyObject* o = x->defined() ? THPVariable_Wrap(*x) : Py_NewRef(Py_None);
    if (!o) {
      Py_DECREF(t);
      throw Refused{};
    }
    PyTuple_SET_ITEM(t, i++, o);
  }
  return t;
}

PyObject* cache_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 8);
    const at::Tensor &table = tensor(item(a[0], 0, 5, "PageTables"), "page_table"),
                     &lengths = tensor(item(a[0], 1, 5, "PageTables"), "lengths"),
                     &free = tensor(item(a[0], 2, 5, "PageTables"), "free"),
                     &n_free = tensor(item(a[0], 3, 5, "PageTables"), "n_free");
    const int64_t size = integer(item(a[0], 4, 5, "PageTables"));
    const Place at(table);
    int32_table(table, "page_table", at, 2);
    int32_table(free, "free", at, 1);
    const int64_t B = table.size(0), width = table.size(1);
    if (B == 0 || width == 0 || free.size(0) == 0)
      refuse(PyExc_ValueError, "tables of %lld sequences, %lld pages each, %lld in all", (long long)B, (long long)width,
             (long long)free.size(0));
    per_sequence(lengths, "lengths", B, at);
    per_sequence(n_free, "n_free", 1, at);
    const at::Tensor& add = per_sequence(tensor(a[1], "new"), "new", B, at);
    const int64_t rows = integer(a[2]), max_new = integer(a[3]), max_len = integer(a[4]);
    if (rows < 0 || max_new < 0 || max_len < 0)
      refuse(PyExc_ValueError, "a step of %lld rows, %lld new tokens a sequence and %lld in all", (long long)rows,
             (long long)max_new, (long long)max_len);
    const at::Tensor *keep = maybe(a[5], "keep"), *first = maybe(a[6], "base");
    if (keep) per_sequence(*keep, "keep", B, at);
    if (first) per_sequence(*first, "base", B, at);
    const Parents parents(a[7], B, first ? 0 : max_new, at);
    const int64_t words = (parents.nodes + 31) / 32;
    const at::Tensor start = fresh(table, {B + 1}, at::kInt), len = fresh(table, {B}, at::kInt),
                     base = fresh(table, {B}, at::kInt), positions = fresh(table, {rows}, at::kInt),
                     slots = fresh(table, {rows}, at::kLong);
    at::Tensor mask;
    if (parents.at) mask = fresh(table, {rows, words}, at::kInt);
    // an empty mask has no address, and is asked for all the same
    int32_t* mask_at = parents.at ? (rows ? static_cast<int32_t*>(mask.data_ptr()) : start.data_ptr<int32_t>()) : nullptr;
    call("lz_cache_tables", p_tables, address<int32_t>(&table), width, address<int32_t>(&lengths), address<int32_t>(&free),
         free.size(0), address<int32_t>(&n_free), size, (const int32_t*)address<int32_t>(&add),
         (const int32_t*)address<int32_t>(keep), (const int32_t*)address<int32_t>(first), parents.at, parents.ld,
         parents.nodes, B, rows, max_new, max_len, address<int32_t>(&start), address<int32_t>(&len),
         address<int32_t>(&base), address<int32_t>(&positions), address<int64_t>(&slots), mask_at, words, at.stream);
    return tuple_of({&start, &len, &base, &positions, &slots, &mask});
  });
}

PyObject* verify_draft(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 8);
    const at::Tensor& x = tensor(a[0], "logits");
    const Place at(x);
    const int code = code_of(x);
    if (x.dim() != 2 || x.size(1) == 0) refuse(PyExc_ValueError, "logits must be [rows, V], got %s", shape(x).c_str());
    const int64_t rows = x.size(0), V = x.size(1);
    if ((V > 1 && x.stride(1) != 1) || (rows > 1 && x.stride(0) < V))
      refuse(PyExc_ValueError, "logits rows must be adjacent values, got strides (%lld, %lld)", (long long)x.stride(0),
             (long long)x.stride(1));
    const at::Tensor &tokens = tensor(a[1], "tokens"), &start = tensor(a[2], "row_start"), &uniform = tensor(a[4], "uniform");
    const int64_t max_new = integer(a[3]);
    int32_table(start, "row_start", at, 1);
    const int64_t B = start.size(0) - 1;
    if (B < 1 || max_new < 1) refuse(PyExc_ValueError, "no sequence's tokens to verify");
    if (tokens.scalar_type() != at::kLong || tokens.dim() != 1 || tokens.size(0) != rows || !tokens.is_contiguous() ||
        !at.here(tokens)) {
      require_gpu(tokens);
      refuse(PyExc_ValueError, "tokens must be a contiguous int64 [%lld] tensor on cuda:%d, got %s %s", (long long)rows,
             (int)at.index, type_name(tokens), shape(tokens).c_str());
    }
    const bool wide = uniform.scalar_type() == at::kDouble;
    if ((!wide && uniform.scalar_type() != at::kFloat) || uniform.dim() != 1 || uniform.size(0) != rows ||
        !uniform.is_contiguous() || !at.here(uniform)) {
      require_gpu(uniform);
      refuse(PyExc_ValueError, "uniform must be a contiguous float32 or float64 [%lld] tensor on cuda:%d, got %s %s",
             (long long)rows, (int)at.index, type_name(uniform), shape(uniform).c_str());
    }
    const Penalty heat(a[5], "temperature", B, false, at);
    const Parents parents(a[6], B, max_new, at);
    const at::Tensor* probs = maybe(a[7], "draft_probs");
    if (probs) {
      if (parents.at) refuse(PyExc_ValueError, "draft_probs are for chains: with parents, tokens are matched");
      if (probs->scalar_type() != at::kFloat || probs->dim() != 2 || probs->size(0) != rows || probs->size(1) != V ||
          (V > 1 && probs->stride(1) != 1) || (rows > 1 && probs->stride(0) < V) || !at.here(*probs)) {
        require_gpu(*probs);
        refuse(PyExc_ValueError, "draft_probs must be float32 rows [%lld, %lld] on cuda:%d, got %s %s", (long long)rows,
               (long long)V, (int)at.index, type_name(*probs), shape(*probs).c_str());
      }
    }
    const at::Tensor counts = fresh(x, {B}, at::kInt), kept = fresh(x, {B, max_new}, at::kInt),
                     chosen = fresh(x, {B, max_new}, at::kLong);
    const int64_t bytes = p_verify_ws(rows, B, V, probs != nullptr);
    at::Tensor ws;
    if (bytes) ws = fresh(x, {(bytes + 7) / 8}, at::kLong);
    call("lz_verify_draft", p_verify, (const void*)x.data_ptr(), rows > 1 ? x.stride(0) : V, code, rows, V,
         (const int64_t*)address<int64_t>(&tokens), (const void*)uniform.data_ptr(), (int)wide,
         (const int32_t*)address<int32_t>(&start), B, max_new, heat.rows, heat.all, parents.at, parents.ld, parents.nodes,
         (const float*)address<float>(probs), probs && rows > 1 ? probs->stride(0) : V, address<int32_t>(&counts),
         address<int32_t>(&kept), address<int64_t>(&chosen), bytes ? ws.data_ptr() : nullptr, bytes, at.stream);
    return tuple_of({&counts, &kept, &chosen});
  });
}

PyObject* kv_cache_keep(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 4);
    const at::Tensor &k = tensor(item(a[0], 0, 4, "LayerCache"), "layers.k"),
                     &v = tensor(item(a[0], 1, 4, "LayerCache"), "layers.v");
    const at::Tensor *ke = maybe(item(a[0], 2, 4, "LayerCache"), "layers.k_exp"),
                     *ve = maybe(item(a[0], 3, 4, "LayerCache"), "layers.v_exp");
    const Place at(k);
    for (const at::Tensor* t : {&v, ke, ve})
      if (t && !at.here(*t)) {
        require_gpu(*t);
        refuse(PyExc_ValueError, "the cache is on cuda:%d and on %s", (int)at.index, t->device().str().c_str());
      }
    const int64_t d = k.dim();
    if ((d != 4 && d != 5) || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() || !k.is_contiguous() ||
        !v.is_contiguous())
      refuse(PyExc_ValueError, "cache pages must be two contiguous tensors [pages, KV heads, page size, head dim], or of "
                               "several layers [layers, pages, ...], got %s %s and %s %s", type_name(k), shape(k).c_str(),
             type_name(v), shape(v).c_str());
    const bool e8 = k.scalar_type() == at::kFloat8_e4m3fn;
    for (const at::Tensor* e : {ke, ve}) {
      if (e8 && (!e || e->scalar_type() != at::kChar || e->sizes() != k.sizes().slice(0, d - 1) || !e->is_contiguous()))
        refuse(PyExc_ValueError, "a float8_e4m3fn cache needs contiguous int8 exponents of a token and head beside it");
      if (!e8 && e) refuse(PyExc_TypeError, "a cache of %s has no exponents", type_name(k));
    }
    if (!is_draft(a[1])) refuse(PyExc_TypeError, "expected a DraftStep, got %s", Py_TYPE(a[1])->tp_name);
    const at::Tensor &start = tensor(PyTuple_GET_ITEM(a[1], 0), "row_start"), &slots = tensor(PyTuple_GET_ITEM(a[1], 8), "slots");
    const int64_t rows = integer(PyTuple_GET_ITEM(a[1], 3));
    int32_table(start, "row_start", at, 1);
    const int64_t B = start.size(0) - 1;
    if (B < 1 || rows < 0 || slots.scalar_type() != at::kLong || slots.dim() != 1 || slots.size(0) < rows ||
        !slots.is_contiguous() || !at.here(slots)) {
      require_gpu(slots);
      refuse(PyExc_ValueError, "slots must be a contiguous int64 tensor of the step's %lld rows on cuda:%d, got %s %s",
             (long long)rows, (int)at.index, type_name(slots), shape(slots).c_str());
    }
    const at::Tensor &kept = tensor(a[2], "kept"), &counts = per_sequence(tensor(a[3], "counts"), "counts", B, at);
    int32_table(kept, "kept", at, 2);
    if (kept.size(0) != B)
      refuse(PyExc_ValueError, "kept must be [%lld, nodes], got %s", (long long)B, shape(kept).c_str());
    call("lz_kv_keep", p_keep, k.data_ptr(), v.data_ptr(), address(ke), address(ve), e8 ? LZ_E4M3 : code_of(k),
         d == 5 ? k.size(0) : 1, k.size(d - 4), k.size(d - 2), k.size(d - 3), k.size(d - 1),
         (const int64_t*)address<int64_t>(&slots), rows, (const int32_t*)address<int32_t>(&start), B,
         (const int32_t*)address<int32_t>(&kept), kept.size(1), kept.size(1), (const int32_t*)address<int32_t>(&counts),
         at.stream);
    Py_RETURN_NONE;
  });
}

template <typename P>
void take(PyObject* addresses, const char* name, P& p) {
  PyObject* o = PyDict_GetItemString(addresses, name);
  void* at = o ? PyLong_AsVoidPtr(o) : nullptr;
  if (!at) refuse(PyExc_ValueError, "no address of %s", name);
  p = reinterpret_cast<P>(at);
}

PyObject* bind(PyObject*, PyObject* args) {
  return guarded([&]() -> PyObject* {
    PyObject *addresses, *stream, *get, *set, *failure;
    if (!PyArg_ParseTuple(args, "O!OOOO", &PyDict_Type, &addresses, &stream, &get, &set, &failure)) throw Refused{};
    take(addresses, "lz_kv_read", p_read);
    take(addresses, "lz_paged_attn", p_attn);
    take(addresses, "lz_paged_attn_workspace", p_attn_ws);
    take(addresses, "lz_process_logits", p_logits);
    take(addresses, "lz_copy2d", p_copy);
    take(addresses, "lz_fill", p_fill);
    take(addresses, "lz_last_error", p_error);
    take(addresses, "lz_kv_write_at", p_write_at);
    take(addresses, "lz_kv_keep", p_keep);
    take(addresses, "lz_tree_attn", p_tree);
    take(addresses, "lz_tree_attn_workspace", p_tree_ws);
    take(addresses, "lz_cache_tables", p_tables);
    take(addresses, "lz_verify_draft", p_verify);
    take(addresses, "lz_verify_workspace", p_verify_ws);
    take(addresses, "lz_kv_write", p_write);
    for (auto& [slot, o] : {std::pair<PyObject*&, PyObject*>{g_stream, stream}, {g_get, get}, {g_set, set}, {g_failure, failure}}) {
      Py_INCREF(o);
      Py_XDECREF(slot);
      slot = o;
    }
    Py_RETURN_NONE;
  });
}

#define METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {METHOD(kv_cache_write), METHOD(kv_cache_read), METHOD(paged_attention), METHOD(process_logits),
                          METHOD(cache_tables), METHOD(verify_draft), METHOD(kv_cache_keep),
                          {"bind", bind, METH_VARARGS, "bind(addresses, raw_stream, get_device, set_device, error)"},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torchcall", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torchcall(void) { return PyModule_Create(&kModule); }
