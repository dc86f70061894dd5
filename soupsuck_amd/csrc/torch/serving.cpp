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

py::object append_kv(int64_t cache_pointer, const Tensor& pages, py::handle k_arg,
                     py::handle v_arg, py::handle table_arg, py::handle lengths_arg,
                     py::handle cu_arg, py::handle q_arg, py::handle cos_arg,
                     py::handle sin_arg) {
  const auto* cache = reinterpret_cast<const ss_paged_cache*>(cache_pointer);
  const at::ScalarType dtype = pages.scalar_type();
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
  if (!(cu.size(0) == rows.rows + 1 && cu.is_contiguous() && packed(k, cache->kv_heads) &&
        packed(v, cache->kv_heads) && v.size(0) == tokens && cos.defined() == sin.defined() &&
        (!cos.defined() || (turns(cos) && turns(sin))) &&
        (!q.defined() || (cos.defined() && packed(q, -1) && q.size(0) == tokens && q.size(1) > 0))))
    return py::none();
  Tensor out;
  {
    py::gil_scoped_release unlocked;
    c10::DeviceGuard guard(pages.device());
    if (q.defined()) out = at::empty(q.sizes(), q.options());
    const bool turned = cos.defined(), queries = q.defined();
    check(ss_kv_append(cache, ptr<void>(k), k.stride(0), k.stride(1), ptr<void>(v), v.stride(0),
                       v.stride(1), ptr<void>(q), queries ? q.stride(0) : 0,
                       queries ? q.stride(1) : 0, queries ? (int)q.size(1) : 0, ptr<void>(cos),
                       turned ? cos.stride(0) : 0, ptr<void>(sin), turned ? sin.stride(0) : 0,
                       turned ? code_of(cos) : SS_F32, ptr<int32_t>(rows.table), rows.stride,
                       (int)rows.width, ptr<int32_t>(rows.lengths), ptr<int32_t>(cu),
                       (int)rows.rows, tokens, ptr<void>(out), queries ? out.stride(0) : 0,
                       queries ? out.stride(1) : 0, stream_of(pages)),
          "ss_kv_append");
  }
  return q.defined() ? py::cast(out) : py::bool_(true);
}

bool weights_fit(const Tensor& t, const Table& rows, const ss_paged_cache* cache) {
  return t.size(0) == rows.rows && t.size(1) == cache->kv_heads &&
         t.size(2) == rows.width * cache->page_size && t.is_contiguous();
}

py::object cached_attention(int64_t cache_pointer, const Tensor& pages, py::handle q_arg,
                            py::handle table_arg, py::handle lengths_arg, py::handle cu_arg,
                            py::handle max_new_arg, py::handle max_length_arg,
                            py::handle scale_arg, py::handle window_arg, py::handle sinks_arg,
                            py::handle weights_arg, py::handle weights_out_arg) {
  const auto* cache = reinterpret_cast<const ss_paged_cache*>(cache_pointer);
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
  const Tensor q = c.take(q_arg, pages.scalar_type(), 3);
  const Tensor weights = c.take_or_none(weights_arg, at::kFloat, 3);
  const Tensor weights_out = c.take_or_none(weights_out_arg, at::kFloat, 3);
  if (!c.ok) return py::none();
  const int64_t tokens = q.size(0), heads = q.size(1);
  if (!(cu.size(0) == rows.rows + 1 && cu.is_contiguous() && packed(q, -1) && heads > 0 &&
        heads % cache->kv_heads == 0 && heads < INT32_MAX &&
        (!weights.defined() || (weights_out.defined() && weights_fit(weights, rows, cache))) &&
        (!weights_out.defined() || weights_fit(weights_out, rows, cache))))
    return py::none();
  Tensor out;
  {
    py::gil_scoped_release unlocked;
    c10::DeviceGuard guard(pages.device());
    out = at::empty(q.sizes(), q.options());
    const size_t size = ss_cached_attention_workspace_size(
        (int)rows.rows, tokens, (int)heads, cache->kv_heads, (int)max_new, max_length,
        weights_out.defined());
    const Tensor scratch = workspace(size, q);
    check(ss_cached_attention(cache, ptr<void>(q), q.stride(0), q.stride(1), (int)heads,
                              ptr<int32_t>(rows.table), rows.stride, (int)rows.width,
                              ptr<int32_t>(rows.lengths), ptr<int32_t>(cu), (int)rows.rows,
                              tokens, (int)max_new, max_length, (float)scale, window, sinks,
                              ptr<float>(weights), ptr<float>(weights_out), ptr<void>(out),
                              out.stride(0), out.stride(1), ptr<void>(scratch), size,
                              stream_of(pages)),
          "ss_cached_attention");
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
      !weights_fit(weights, rows, cache))
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
  m.def("verify_drafts", &verify_drafts);
}
