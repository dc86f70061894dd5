// The paged cache's and drafting's calls without the interpreter.
//
// A decode step makes several of these for each layer, and a kernel for one short
// sequence runs for 3 to 10 us; the Python bodies of the same calls (kernels/paged.py,
// kernels/verify.py: a table of rules, a ctypes call of up to 28 arguments) take 20 us
// each.  A function here takes what its Python namesake was given, unchecked.  Where all of
// the rules hold it makes the call; where one does not, or where it is not sure, it
// returns None and does nothing (append_kv without q returns True), and the Python body finds the rule that is broken and says so.
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstddef>
#include <cstring>

#include "calls.h"

namespace {

namespace py = pybind11;

constexpr int64_t kHeadDim = 128;

// An argument as a tensor; None is one that is not defined.
struct Argument {
  Tensor t;
  bool ok;
  explicit Argument(py::handle h) : ok(h.is_none()) {
    if (THPVariable_Check(h.ptr())) {
      t = THPVariable_Unpack(h.ptr());
      ok = t.layout() == at::kStrided;
    }
  }
};

// The tensors of a call: set to false by the first one that breaks a rule.
struct Checked {
  at::Device device;
  bool ok = true;
  explicit Checked(const Tensor& first) : device(first.device()), ok(first.is_cuda()) {}
  void that(bool holds) { ok = ok && holds; }
  Tensor take(py::handle h, at::ScalarType dtype, int64_t dims) {
    Argument a(h);
    that(a.ok && a.t.defined() && a.t.scalar_type() == dtype && a.t.dim() == dims &&
         a.t.device() == device);
    return ok ? std::move(a.t) : Tensor();
  }
  Tensor take_or_none(py::handle h, at::ScalarType dtype, int64_t dims) {
    return h.is_none() ? Tensor() : take(h, dtype, dims);
  }
};

bool whole(py::handle h, int64_t minimum, int64_t limit, int64_t* out) {
  if (!PyLong_CheckExact(h.ptr())) return false;
  int overflow = 0;
  *out = PyLong_AsLongLongAndOverflow(h.ptr(), &overflow);
  return !overflow && *out >= minimum && *out < limit;
}

bool number(py::handle h, double* out) {
  if (PyFloat_CheckExact(h.ptr())) *out = PyFloat_AS_DOUBLE(h.ptr());
  else if (PyLong_CheckExact(h.ptr())) {
    int overflow = 0;
    *out = (double)PyLong_AsLongLongAndOverflow(h.ptr(), &overflow);
    if (overflow) return false;
  } else return false;
  return std::isfinite(*out);
}

// 16-byte aligned base, unit last stride, other strides multiples of 16 bytes.
bool strided(const Tensor& t) {
  const int64_t unit = 16 / t.element_size();
  if ((uintptr_t)t.data_ptr() % 16 || t.stride(-1) != 1) return false;
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    if (t.stride(d) % unit) return false;
  return true;
}

int code_of(const Tensor& t) {
  return t.scalar_type() == at::kHalf ? SS_F16 : t.scalar_type() == at::kFloat ? SS_F32 : SS_BF16;
}

// A block table and the lengths of its lines.
struct Table {
  Tensor table, lengths;
  int64_t rows = 0, width = 0, stride = 0;
  Table(Checked& c, py::handle table_arg, py::handle lengths_arg)
      : table(c.take(table_arg, at::kInt, 2)), lengths(c.take(lengths_arg, at::kInt, 1)) {
    if (!c.ok) return;
    rows = table.size(0);
    width = table.size(1);
    stride = std::max(table.stride(0), width);
    c.that(rows > 0 && width > 0 && (table.stride(1) == 1 || width == 1) &&
           (table.stride(0) >= width || rows <= 1) && rows < INT32_MAX && width < INT32_MAX &&
           lengths.size(0) == rows && lengths.is_contiguous());
  }
};

bool packed(const Tensor& t, int64_t heads) {
  return t.size(2) == kHeadDim && t.size(0) > 0 && (heads < 0 || t.size(1) == heads) &&
         !t.requires_grad() && strided(t);
}

// A cache by its struct's address: of 16 bits, or of 4 (whose memory is bytes).
struct Cache {
  const ss_paged_cache* wide = nullptr;
  const ss_paged_cache4* four = nullptr;
  int kv_heads, page_size;
  at::ScalarType dtype;
  Cache(int64_t pointer, bool is_four) {
    if (is_four) {
      four = reinterpret_cast<const ss_paged_cache4*>(pointer);
      set(*four);
    } else {
      wide = reinterpret_cast<const ss_paged_cache*>(pointer);
      set(*wide);
    }
  }
  template <class C>
  void set(const C& c) {
    kv_heads = c.kv_heads;
    page_size = c.page_size;
    dtype = c.dtype == SS_F16 ? at::kHalf : at::kBFloat16;
  }
};

py::object append_kv(int64_t cache_pointer, const Tensor& pages, bool is_four, py::handle k_arg,
                     py::handle v_arg, py::handle table_arg, py::handle lengths_arg,
                     py::handle cu_arg, py::handle q_arg, py::handle cos_arg,
                     py::handle sin_arg) {
  const Cache cache(cache_pointer, is_four);
  const at::ScalarType dtype = cache.dtype;
  Checked c(pages);
  const Table rows(c, table_arg, lengths_arg);
  const Tensor cu = c.take(cu_arg, at::kInt, 1);
  const Tensor k = c.take(k_arg, dtype, 3), v = c.take(v_arg, dtype, 3);
  const Tensor q = c.take_or_none(q_arg, dtype, 3);
  at::ScalarType angles = dtype;
  if (THPVariable_Check(cos_arg.ptr()) &&
      THPVariable_Unpack(cos_arg.ptr()).scalar_type() == at::kFloat)
    angles = at::kFloat;
  const Tensor cos = c.take_or_none(cos_arg, angles, 2), sin = c.take_or_none(sin_arg, angles, 2);
  if (!c.ok) return py::none();
  const int64_t tokens = k.size(0);
  auto turns = [&](const Tensor& t) {
    return t.size(0) == tokens && t.size(1) == kHeadDim && strided(t);
  };
  if (!(cu.size(0) == rows.rows + 1 && cu.is_contiguous() && packed(k, cache.kv_heads) &&
        packed(v, cache.kv_heads) && v.size(0) == tokens && cos.defined() == sin.defined() &&
        (!cos.defined() || (turns(cos) && turns(sin))) &&
        (!q.defined() || (cos.defined() && packed(q, -1) && q.size(0) == tokens && q.size(1) > 0))))
    return py::none();
  Tensor out;
  {
    py::gil_scoped_release unlocked;
    c10::DeviceGuard guard(pages.device());
    if (q.defined()) out = at::empty(q.sizes(), q.options());
    const bool turned = cos.defined(), queries = q.defined();
    auto append = [&](auto* call, const auto* to, const char* name) {
      check(call(to, ptr<void>(k), k.stride(0), k.stride(1), ptr<void>(v), v.stride(0),
                         v.stride(1), ptr<void>(q), queries ? q.stride(0) : 0,
                         queries ? q.stride(1) : 0, queries ? (int)q.size(1) : 0, ptr<void>(cos),
                         turned ? cos.stride(0) : 0, ptr<void>(sin), turned ? sin.stride(0) : 0,
                         turned ? code_of(cos) : SS_F32, ptr<int32_t>(rows.table), rows.stride,
                         (int)rows.width, ptr<int32_t>(rows.lengths), ptr<int32_t>(cu),
                         (int)rows.rows, tokens, ptr<void>(out), queries ? out.stride(0) : 0,
                         queries ? out.stride(1) : 0, stream_of(pages)),
            name);
    };
    if (is_four) append(&ss_kv_append4, cache.four, "ss_kv_append4");
    else append(&ss_kv_append, cache.wide, "ss_kv_append");
  }
  return q.defined() ? py::cast(out) : py::bool_(true);
}

bool weights_fit(const Tensor& t, const Table& rows, int kv_heads, int page_size) {
  return t.size(0) == rows.rows && t.size(1) == kv_heads &&
         t.size(2) == rows.width * page_size && t.is_contiguous();
}

py::object cached_attention(int64_t cache_pointer, const Tensor& pages, bool is_four, py::handle q_arg,
                            py::handle table_arg, py::handle lengths_arg, py::handle cu_arg,
                            py::handle max_new_arg, py::handle max_length_arg,
                            py::handle scale_arg, py::handle window_arg, py::handle sinks_arg,
                            py::handle weights_arg, py::handle weights_out_arg) {
  const Cache cache(cache_pointer, is_four);
  int64_t max_new, max_length, window = 0, sinks;
  double scale;
  if (!whole(max_new_arg, 1, (int64_t)1 << 31, &max_new) ||
      !whole(max_length_arg, 0, (int64_t)1 << 31, &max_length) || !number(scale_arg, &scale) ||
      (!window_arg.is_none() && !whole(window_arg, 1, (int64_t)1 << 62, &window)) ||
      !whole(sinks_arg, 0, (int64_t)1 << 62, &sinks))
    return py::none();
  Checked c(pages);
  const Table rows(c, table_arg, lengths_arg);
  const Tensor cu = c.take(cu_arg, at::kInt, 1);
  const Tensor q = c.take(q_arg, cache.dtype, 3);
  const Tensor weights = c.take_or_none(weights_arg, at::kFloat, 3);
  const Tensor weights_out = c.take_or_none(weights_out_arg, at::kFloat, 3);
  if (!c.ok) return py::none();
  const int64_t tokens = q.size(0), heads = q.size(1);
  if (!(cu.size(0) == rows.rows + 1 && cu.is_contiguous() && packed(q, -1) && heads > 0 &&
        heads % cache.kv_heads == 0 && heads < INT32_MAX &&
        (!weights.defined() || (weights_out.defined() && weights_fit(weights, rows, cache.kv_heads, cache.page_size))) &&
        (!weights_out.defined() || !is_four) &&
        (!weights_out.defined() || weights_fit(weights_out, rows, cache.kv_heads, cache.page_size))))
    return py::none();
  Tensor out;
  {
    py::gil_scoped_release unlocked;
    c10::DeviceGuard guard(pages.device());
    out = at::empty(q.sizes(), q.options());
    if (is_four) {
      const size_t size = ss_cached_attention4_workspace_size(
          (int)rows.rows, tokens, (int)heads, cache.kv_heads, (int)max_new, max_length);
      const Tensor scratch = workspace(size, q);
      check(ss_cached_attention4(cache.four, ptr<void>(q), q.stride(0), q.stride(1), (int)heads,
                                 ptr<int32_t>(rows.table), rows.stride, (int)rows.width,
                                 ptr<int32_t>(rows.lengths), ptr<int32_t>(cu), (int)rows.rows,
                                 tokens, (int)max_new, max_length, (float)scale, window, sinks,
                                 ptr<void>(out), out.stride(0), out.stride(1),
                                 ptr<void>(scratch), size, stream_of(pages)),
            "ss_cached_attention4");
    } else {
      const size_t size = ss_cached_attention_workspace_size(
          (int)rows.rows, tokens, (int)heads, cache.kv_heads, (int)max_new, max_length,
          weights_out.defined());
      const Tensor scratch = workspace(size, q);
      check(ss_cached_attention(cache.wide, ptr<void>(q), q.stride(0), q.stride(1), (int)heads,
                                ptr<int32_t>(rows.table), rows.stride, (int)rows.width,
                                ptr<int32_t>(rows.lengths), ptr<int32_t>(cu), (int)rows.rows,
                                tokens, (int)max_new, max_length, (float)scale, window, sinks,
                                ptr<float>(weights), ptr<float>(weights_out), ptr<void>(out),
                                out.stride(0), out.stride(1), ptr<void>(scratch), size,
                                stream_of(pages)),
            "ss_cached_attention");
    }
  }
  return py::cast(out);
}

py::object evict_kv(int64_t cache_pointer, const Tensor& pages, py::handle table_arg,
                    py::handle lengths_arg, py::handle weights_arg, py::handle out_table_arg,
                    py::handle budget_arg, py::handle max_length_arg, py::handle sinks_arg,
                    py::handle recent_arg) {
  const auto* cache = reinterpret_cast<const ss_paged_cache*>(cache_pointer);
  int64_t budget, max_length, sinks, recent;
  constexpr int64_t top = (int64_t)1 << 31;
  if (!whole(budget_arg, 1, top, &budget) || !whole(max_length_arg, 0, top, &max_length) ||
      !whole(sinks_arg, 0, top, &sinks) || !whole(recent_arg, 0, top, &recent) ||
      sinks + recent > budget)
    return py::none();
  Checked c(pages);
  const Table rows(c, table_arg, lengths_arg);
  const Table out(c, out_table_arg, lengths_arg);
  const Tensor weights = c.take(weights_arg, at::kFloat, 3);
  if (!c.ok || out.rows != rows.rows || budget > out.width * cache->page_size ||
      !weights_fit(weights, rows, cache->kv_heads, cache->page_size))
    return py::none();
  Tensor out_lengths, out_weights;
  {
    py::gil_scoped_release unlocked;
    c10::DeviceGuard guard(pages.device());
    out_lengths = empty({rows.rows}, weights, at::kInt);
    out_weights = empty({rows.rows, cache->kv_heads, out.width * cache->page_size}, weights,
                        at::kFloat);
    const size_t size = ss_kv_evict_workspace_size((int)rows.rows, cache->kv_heads, budget);
    const Tensor scratch = workspace(size, weights);
    check(ss_kv_evict(cache, ptr<int32_t>(rows.table), rows.stride, (int)rows.width,
                      ptr<int32_t>(rows.lengths), (int)rows.rows, max_length, ptr<float>(weights),
                      ptr<int32_t>(out.table), out.stride, (int)out.width, budget, sinks, recent,
                      ptr<int32_t>(out_lengths), ptr<float>(out_weights), ptr<void>(scratch),
                      size, stream_of(pages)),
          "ss_kv_evict");
  }
  return py::make_tuple(out_lengths, out_weights);
}

// The caches of a call, a list or tuple of one class: their structs' addresses (`_pointer`) and
// devices (`_index`) by attribute, as a call for each layer's cache would cost more than its kernel.
struct Caches {
  py::object held;  // while the call runs without the lock, whatever becomes of a list
  std::vector<int64_t> pointers;
  bool ok = false, four = false;
  int64_t index = -1;
  Caches(py::handle caches, py::handle wide_type, py::handle four_type) {
    static PyObject* const pointer_name = PyUnicode_InternFromString("_pointer");
    static PyObject* const index_name = PyUnicode_InternFromString("_index");
    if (PyList_Check(caches.ptr()))
      held = py::reinterpret_steal<py::object>(PyList_AsTuple(caches.ptr()));
    else if (PyTuple_Check(caches.ptr()))
      held = py::reinterpret_borrow<py::object>(caches);
    if (!held) {
      PyErr_Clear();
      return;
    }
    const Py_ssize_t n = PyTuple_GET_SIZE(held.ptr());
    if (n == 0 || n >= INT32_MAX) return;
    pointers.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* cache = PyTuple_GET_ITEM(held.ptr(), i);
      const bool is_four = (PyObject*)Py_TYPE(cache) == four_type.ptr();
      if (!is_four && (PyObject*)Py_TYPE(cache) != wide_type.ptr()) return;
      int64_t pointer, device;
      if (!number_of(cache, pointer_name, &pointer) || !number_of(cache, index_name, &device))
        return;
      if (i == 0) four = is_four, index = device;
      if (is_four != four || device != index || device < 0) return;
      pointers.push_back(pointer);
      if (!(four ? alike<ss_paged_cache4>(offsetof(ss_paged_cache4, page), 3)
                 : alike<ss_paged_cache>(offsetof(ss_paged_cache, k_page), 3)))
        return;
    }
    ok = true;
  }
  static bool number_of(PyObject* of, PyObject* name, int64_t* out) {
    PyObject* value = PyObject_GetAttr(of, name);
    const bool good = value && PyLong_CheckExact(value);
    if (good) *out = PyLong_AsLongLong(value);
    Py_XDECREF(value);
    PyErr_Clear();
    return good;
  }
  // Everything but the bases (the C entries compare the strides of v).
  template <class C>
  bool alike(size_t from, size_t strides) const {
    const auto *a = reinterpret_cast<const C*>(pointers[0]),
               *b = reinterpret_cast<const C*>(pointers.back());
    return a->pages == b->pages && a->page_size == b->page_size && a->kv_heads == b->kv_heads &&
           a->dtype == b->dtype &&
           !memcmp((const char*)a + from, (const char*)b + from, strides * sizeof(int64_t));
  }
  template <class C>
  const C* const* all() const {
    return reinterpret_cast<const C* const*>(pointers.data());
  }
  int count() const { return (int)pointers.size(); }
  bool on(const Tensor& t) const { return t.is_cuda() && t.device().index() == index; }
};

// The block table of a call, whose device the others are checked against.
bool table_of(py::handle arg, Tensor* out) {
  const Argument a(arg);
  *out = a.t;
  return a.ok && a.t.defined();
}

py::object read_kv(py::handle caches_arg, py::handle wide_type, py::handle four_type,
                   py::handle table_arg, py::handle lengths_arg, py::handle cu_arg,
                   py::handle tokens_arg, bool several) {
  int64_t tokens;
  Tensor pages;
  const Caches caches(caches_arg, wide_type, four_type);
  if (!caches.ok || !whole(tokens_arg, 1, (int64_t)1 << 31, &tokens) ||
      !table_of(table_arg, &pages) || !caches.on(pages))
    return py::none();
  const Cache cache(caches.pointers[0], caches.four);
  Checked c(pages);
  const Table rows(c, table_arg, lengths_arg);
  const Tensor cu = c.take(cu_arg, at::kInt, 1);
  if (!c.ok || cu.size(0) != rows.rows + 1 || !cu.is_contiguous()) return py::none();
  Tensor k, v;
  {
    py::gil_scoped_release unlocked;
    c10::DeviceGuard guard(pages.device());
    k = several ? empty({caches.count(), tokens, cache.kv_heads, kHeadDim}, pages, cache.dtype)
                : empty({tokens, cache.kv_heads, kHeadDim}, pages, cache.dtype);
    v = at::empty_like(k);
    auto read = [&](auto* call, auto* const* all, const char* name) {
      check(call(all, caches.count(), ptr<int32_t>(rows.table), rows.stride, (int)rows.width,
                 ptr<int32_t>(rows.lengths), ptr<int32_t>(cu), (int)rows.rows, tokens,
                 ptr<void>(k), ptr<void>(v), stream_of(pages)),
            name);
    };
    if (caches.four) read(&ss_kv_read4, caches.all<ss_paged_cache4>(), "ss_kv_read4");
    else read(&ss_kv_read, caches.all<ss_paged_cache>(), "ss_kv_read");
  }
  return py::make_tuple(k, v);
}

py::object fork_kv(py::handle caches_arg, py::handle wide_type, py::handle four_type,
                   py::handle table_arg, py::handle lengths_arg, py::handle parents_arg,
                   py::handle spare_arg) {
  Tensor pages;
  const Caches caches(caches_arg, wide_type, four_type);
  if (!caches.ok || !table_of(table_arg, &pages) || !caches.on(pages)) return py::none();
  Checked c(pages);
  const Table rows(c, table_arg, lengths_arg);
  const Tensor parents = c.take(parents_arg, at::kInt, 1), spare = c.take(spare_arg, at::kInt, 1);
  if (!c.ok || parents.size(0) == 0 || parents.size(0) >= INT32_MAX ||
      spare.size(0) != parents.size(0) || !parents.is_contiguous() || !spare.is_contiguous())
    return py::none();
  Tensor table, lengths;
  {
    py::gil_scoped_release unlocked;
    c10::DeviceGuard guard(pages.device());
    table = empty({parents.size(0), rows.width}, parents, at::kInt);
    lengths = empty({parents.size(0)}, parents, at::kInt);
    auto fork = [&](auto* call, auto* const* all, const char* name) {
      check(call(all, caches.count(), ptr<int32_t>(rows.table), rows.stride, (int)rows.width,
                 ptr<int32_t>(rows.lengths), (int)rows.rows, ptr<int32_t>(parents),
                 ptr<int32_t>(spare), (int)parents.size(0), ptr<int32_t>(table),
                 ptr<int32_t>(lengths), stream_of(pages)),
            name);
    };
    if (caches.four) fork(&ss_kv_fork4, caches.all<ss_paged_cache4>(), "ss_kv_fork4");
    else fork(&ss_kv_fork, caches.all<ss_paged_cache>(), "ss_kv_fork");
  }
  return py::make_tuple(table, lengths);
}

py::object select_beams(py::handle logits_arg, py::handle scores_arg, py::handle count_arg) {
  int64_t count;
  const Argument first(logits_arg);
  if (!first.ok || !first.t.defined() || first.t.dim() != 3 || first.t.requires_grad() ||
      !whole(count_arg, 1, 65, &count))
    return py::none();
  const Tensor& logits = first.t;
  const at::ScalarType dtype = logits.scalar_type();
  if (dtype != at::kHalf && dtype != at::kBFloat16 && dtype != at::kFloat) return py::none();
  Checked c(logits);
  const Tensor scores = c.take(scores_arg, at::kFloat, 2);
  if (!c.ok) return py::none();
  const int64_t rows = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
  if (!(rows > 0 && rows <= 65535 && beams > 0 && beams <= 64 && vocab > 0 &&
        vocab < INT32_MAX - 65536 && count <= beams * vocab && beams * count <= 2048 &&
        (logits.stride(2) == 1 || vocab == 1) && scores.size(0) == rows &&
        scores.size(1) == beams && scores.is_contiguous()))
    return py::none();
  Tensor out, parents, tokens;
  {
    py::gil_scoped_release unlocked;
    c10::DeviceGuard guard(logits.device());
    out = empty({rows, count}, logits, at::kFloat);
    parents = empty({rows, count}, logits, at::kInt);
    tokens = empty({rows, count}, logits, at::kLong);
    const size_t size = ss_select_beams_workspace_size((int)rows, (int)beams, vocab, (int)count,
                                                       code_of(logits));
    const Tensor scratch = workspace(size, logits);
    check(ss_select_beams(ptr<void>(logits), logits.stride(0), logits.stride(1), code_of(logits),
                          ptr<float>(scores), (int)rows, (int)beams, vocab, (int)count,
                          ptr<float>(out), ptr<int32_t>(parents), ptr<int64_t>(tokens),
                          ptr<void>(scratch), size, stream_of(logits)),
          "ss_select_beams");
  }
  return py::make_tuple(out, parents, tokens);
}

py::object verify_drafts(py::handle target_arg, py::handle tokens_arg, py::handle uniform_arg,
                         py::handle draft_arg, py::handle counts_arg,
                         py::handle temperature_arg) {
  double temperature;
  const Argument first(target_arg);
  if (!first.ok || !first.t.defined() || first.t.dim() != 3 || !number(temperature_arg, &temperature) ||
      temperature < 0.0)
    return py::none();
  const Tensor& target = first.t;
  const at::ScalarType dtype = target.scalar_type();
  if (dtype != at::kHalf && dtype != at::kBFloat16 && dtype != at::kFloat) return py::none();
  Checked c(target);
  const Tensor tokens = c.take(tokens_arg, at::kLong, 2);
  const Tensor uniform = c.take_or_none(uniform_arg, at::kFloat, 2);
  const Tensor draft = c.take_or_none(draft_arg, dtype, 3);
  const Tensor counts = c.take_or_none(counts_arg, at::kInt, 1);
  if (!c.ok) return py::none();
  const int64_t rows = target.size(0), length = target.size(1), vocab = target.size(2);
  if (!(rows > 0 && length > 0 && vocab > 0 && vocab < INT32_MAX - 8192 &&
        rows * (2 * length - 1) <= 65535 && (target.stride(2) == 1 || vocab == 1) &&
        tokens.size(0) == rows && tokens.size(1) == length - 1 && tokens.is_contiguous() &&
        (uniform.defined() ? uniform.size(0) == rows && uniform.size(1) == length &&
                                 uniform.is_contiguous()
                           : temperature == 0.0) &&
        (!draft.defined() || (draft.size(0) == rows && draft.size(1) == length - 1 &&
                              draft.size(2) == vocab && (draft.stride(2) == 1 || vocab == 1))) &&
        (!counts.defined() || (counts.size(0) == rows && counts.is_contiguous()))))
    return py::none();
  Tensor accepted, out;
  {
    py::gil_scoped_release unlocked;
    c10::DeviceGuard guard(target.device());
    accepted = empty({rows}, target, at::kInt);
    out = empty({rows, length}, target, at::kLong);
    const bool drafted = draft.defined() && length > 1;
    const size_t size = ss_verify_drafts_workspace_size((int)rows, (int)length - 1, vocab, drafted);
    const Tensor scratch = workspace(size, target);
    check(ss_verify_drafts(ptr<void>(target), target.stride(0), target.stride(1),
                           drafted ? ptr<void>(draft) : nullptr, drafted ? draft.stride(0) : 0,
                           drafted ? draft.stride(1) : 0, code_of(target), ptr<int64_t>(tokens),
                           ptr<int32_t>(counts), ptr<float>(uniform), (int)rows, (int)length - 1,
                           vocab, temperature, ptr<int32_t>(accepted), ptr<int64_t>(out),
                           ptr<void>(scratch), size, stream_of(target)),
          "ss_verify_drafts");
  }
  return py::make_tuple(accepted, out);
}

}  // namespace

void define_serving(py::module_& m) {
  m.def("append_kv", &append_kv);
  m.def("cached_attention", &cached_attention);
  m.def("evict_kv", &evict_kv);
  m.def("read_kv", &read_kv);
  m.def("fork_kv", &fork_kv);
  m.def("select_beams", &select_beams);
  m.def("verify_drafts", &verify_drafts);
}
