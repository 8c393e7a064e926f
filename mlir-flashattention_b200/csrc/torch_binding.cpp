// torch_binding.cpp — the serving calls of include/attn_rt.h on torch tensors.
//
// A step of a served model makes these calls for a few microseconds of GPU work
// each; checking shapes and filling a descriptor from Python took 8 to 14 us a
// call, here it takes about two.  serving.py documents the calls and passes
// their arguments on by position; nothing here looks at device data.
#include <Python.h>
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <optional>
#include <sstream>
#include <string>

#include "../../include/attn_rt.h"

namespace {

using at::Tensor;
using Ints = c10::IntArrayRef;

struct Refused {  // becomes VerifyError
  std::string message;
};
struct Failed {  // becomes AttentionError
  int code;
};
struct Raised {};  // a Python error is set

// The interpreter's lock, given up while memory is allocated and kernels are
// launched: with a full launch queue either may wait for the GPU, which in turn
// may wait for what another Python thread has yet to do.  Nothing in such a
// scope touches Python objects.
class Unlocked {
 public:
  Unlocked() : state_(PyEval_SaveThread()) {}
  ~Unlocked() { PyEval_RestoreThread(state_); }
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;

 private:
  PyThreadState* state_;
};

PyObject* g_verify_error = nullptr;
PyObject* g_attention_error = nullptr;
decltype(&attn_cache_plan) g_plan = nullptr;
decltype(&attn_cache_append) g_append = nullptr;
decltype(&attn_rotary) g_rotary = nullptr;
decltype(&attn_tree_fwd) g_tree = nullptr;
decltype(&attn_rt_last_error) g_last_error = nullptr;
decltype(&attn_rt_status_string) g_status_string = nullptr;

template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Refused{s.str()};
}

std::string text(Ints shape) {
  std::ostringstream s;
  s << "[";
  for (size_t i = 0; i < shape.size(); ++i) s << (i ? ", " : "") << shape[i];
  s << "]";
  return s.str();
}

const char* name_of(at::ScalarType t) { return c10::toString(t); }

// ---------------------------------------------------------------- arguments
const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor, not %s", name, Py_TYPE(o)->tp_name);
    throw Raised{};
  }
  return THPVariable_Unpack(o);
}

const Tensor* optional_tensor(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

int64_t integer(PyObject* o) {
  PyObject* i = PyNumber_Index(o);
  if (!i) throw Raised{};
  const int64_t v = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}

float number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return static_cast<float>(v);
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}

void need_count(Py_ssize_t have, Py_ssize_t want) {
  if (have != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", have, want);
    throw Raised{};
  }
}

void on_device(const Tensor& t, const char* name, c10::Device d) {
  if (t.device() != d) refuse(name, " must be a CUDA tensor on ", d.str(), " (got ", t.device().str(), ")");
}

template <typename T = int32_t>
T* ints(const Tensor& t, const char* name, Ints shape, c10::Device d) {
  constexpr auto type = sizeof(T) == 8 ? at::kLong : at::kInt;
  if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous())
    refuse(name, " must be a contiguous ", sizeof(T) == 8 ? "int64" : "int32", " tensor of shape ", text(shape),
           " (got ", name_of(t.scalar_type()), " ", text(t.sizes()), ")");
  on_device(t, name, d);
  return static_cast<T*>(t.data_ptr());
}

bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }

void no_grad(const char* what, std::initializer_list<const Tensor*> list) {
  for (const Tensor* t : list) {
    if (!t) continue;
    if (c10::GradMode::is_enabled() && t->requires_grad())
      refuse(what, " has no backward pass: call it under torch.no_grad()");
    if (has_tangent(*t)) refuse(what, " has no forward-mode derivative");
  }
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return ATTN_F32;
    case at::kBFloat16: return ATTN_BF16;
    case at::kHalf: return ATTN_F16;
    case at::kFloat8_e4m3fn:
    case at::kByte: return ATTN_E4M3;
    default: return -1;
  }
}

Tensor empty(Ints shape, at::ScalarType type, c10::Device d) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(d));
}

// A tensor that was written in place: autograd then knows that what it saved of
// it is no longer there.
void written(std::initializer_list<const Tensor*> list) {
  for (const Tensor* t : list)
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

const Tensor* maybe(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// Runs an entry on the current stream of `d`.
template <typename F, typename D>
void launch(F f, D& desc, c10::Device d) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != d.index()) guard.set_index(d.index());
  const int rc = f(&desc, at::cuda::getCurrentCUDAStream(d.index()).stream());
  if (rc != 0) throw Failed{rc};
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused& e) {
    PyErr_SetString(g_verify_error, e.message.c_str());
  } catch (const Failed& e) {
    const char* m = g_last_error();
    PyObject* args = Py_BuildValue("(is)", e.code, *m ? m : g_status_string(e.code));
    if (args) {
      PyErr_SetObject(g_attention_error, args);
      Py_DECREF(args);
    }
  } catch (const Raised&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// ------------------------------------------------------------------- planner
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_count(n, 12);
    const Tensor &lengths = tensor(a[0], "lengths"), &targets = tensor(a[1], "targets"),
                 &table = tensor(a[2], "block_table"), &free_pages = tensor(a[3], "free_pages"),
                 &free_count = tensor(a[4], "free_count");
    if (lengths.dim() != 1 || table.dim() != 2 || free_pages.dim() != 1)
      refuse("lengths must be [B], block_table [B, W] and free_pages [num_pages]");
    const c10::Device d = lengths.device();
    if (!d.is_cuda()) refuse("lengths must be a CUDA tensor");
    const int64_t B = table.size(0), W = table.size(1), tokens = integer(a[6]);
    if (lengths.size(0) != B) refuse("lengths and block_table must have one row per request");
    if (table.scalar_type() != at::kInt || (W > 1 && table.stride(1) != 1))
      refuse("block_table must be int32 with unit-stride columns");
    on_device(table, "block_table", d);
    if (tokens < 0) refuse("tokens must not be negative");
    AttnCachePlan p{};
    p.flags = ATTN_FLAG_DEVICE_POINTERS;
    const int64_t page = integer(a[5]);
    p.page_size = page > 0 && page <= 1024 ? static_cast<int32_t>(page) : 0;
    p.B = B, p.W = W, p.num_pages = free_pages.size(0), p.tokens = tokens;
    p.table_stride = B > 1 ? table.stride(0) : W;
    p.lengths = ints(lengths, "lengths", {B}, d);
    p.targets = ints(targets, "targets", {B}, d);
    p.block_table = static_cast<int32_t*>(table.data_ptr());
    p.free_pages = ints(free_pages, "free_pages", {p.num_pages}, d);
    p.free_count = ints(free_count, "free_count", {1}, d);
    constexpr const char* names[5] = {"lengths_out", "free_count_out", "slots", "positions", "starts"};
    const Tensor* given[5];
    for (int i = 0; i < 5; ++i) given[i] = optional_tensor(a[7 + i], names[i]);
    Tensor lengths_out, count_out, slots, positions, starts;
    {
      Unlocked unlocked;
      auto out = [&](int i, int64_t size, at::ScalarType type) { return given[i] ? *given[i] : empty({size}, type, d); };
      lengths_out = out(0, B, at::kInt), count_out = out(1, 1, at::kInt), slots = out(2, tokens, at::kLong);
      positions = out(3, tokens, at::kInt), starts = out(4, B + 1, at::kInt);
      p.lengths_out = ints(lengths_out, names[0], {B}, d);
      p.free_count_out = ints(count_out, names[1], {1}, d);
      p.slots = ints<int64_t>(slots, names[2], {tokens}, d);
      p.positions = ints(positions, names[3], {tokens}, d);
      p.starts = ints(starts, names[4], {B + 1}, d);
      launch(g_plan, p, d);
    }
    written({&table, &free_pages, given[0], given[1], given[2], given[3], given[4]});
    PyObject* r = PyTuple_New(5);
    const Tensor* parts[5] = {&slots, &positions, &starts, &lengths_out, &count_out};
    for (int i = 0; r && i < 5; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(*parts[i]));
    return r;
  });
}

// -------------------------------------------------------------------- writer
// A descale: a number, or one f32 value per key head.
void descale(PyObject* o, const char* name, int64_t heads, c10::Device d, float& value, const float*& list) {
  if (!THPVariable_Check(o)) {
    value = number(o);
    return;
  }
  const Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != at::kFloat || t.sizes() != Ints{heads} || !t.is_contiguous() || t.device() != d)
    refuse(name, " must be a number or a contiguous f32 tensor of ", heads, " heads on ", d.str());
  value = 1.f;
  list = static_cast<const float*>(t.data_ptr());
}

void check_cache(const Tensor& kc, const Tensor& vc, int64_t heads, int64_t dim, int code, c10::Device d) {
  if (kc.dim() != 4 || kc.sizes() != vc.sizes() || kc.size(1) != heads || kc.size(3) != dim)
    refuse("k_cache and v_cache must be [num_pages, ", heads, ", page_size, ", dim, "] (got ", text(kc.sizes()), " and ",
           text(vc.sizes()), ")");
  const int c = code_of(kc.scalar_type());
  if (kc.scalar_type() != vc.scalar_type() || (c != code && c != ATTN_E4M3))
    refuse("k_cache and v_cache must share one type: that of the keys, or float8_e4m3fn (got ",
           name_of(kc.scalar_type()), " and ", name_of(vc.scalar_type()), ")");
  if (kc.device() != d || vc.device() != d) refuse("k_cache and v_cache must be CUDA tensors on ", d.str());
  if (kc.stride(3) != 1 || vc.stride(3) != 1) refuse("the cache's head_dim must be unit-stride");
}

int32_t page_size(const Tensor& cache) {
  return cache.size(2) <= 1024 ? static_cast<int32_t>(cache.size(2)) : 0;
}

template <typename Desc>
void cache_fields(Desc& p, const Tensor& kc, const Tensor& vc) {
  p.cache_dtype = code_of(kc.scalar_type());
  p.page_size = page_size(kc);
  p.num_pages = kc.size(0);
  for (int i = 0; i < 3; ++i) p.k_cache_stride[i] = kc.stride(i), p.v_cache_stride[i] = vc.stride(i);
  p.k_cache = kc.data_ptr(), p.v_cache = vc.data_ptr();
}

PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_count(n, 8);
    const Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &kc = tensor(a[2], "k_cache"),
                 &vc = tensor(a[3], "v_cache"), &slots = tensor(a[4], "slots");
    const Tensor* rows = optional_tensor(a[5], "rows");
    if (k.dim() != 3 || k.sizes() != v.sizes()) refuse("k and v must both be [tokens, heads, head_dim]");
    const int64_t T = k.size(0), H = k.size(1), D = k.size(2);
    const c10::Device d = k.device();
    const int code = code_of(k.scalar_type());
    if (!d.is_cuda() || v.device() != d) refuse("k and v must be CUDA tensors on one device");
    if (v.scalar_type() != k.scalar_type() || (code != ATTN_BF16 && code != ATTN_F16))
      refuse("k and v must both be bfloat16 or both float16");
    if (k.stride(2) != 1 || v.stride(2) != 1) refuse("head_dim must be unit-stride");
    check_cache(kc, vc, H, D, code, d);
    no_grad("cache_append", {&k, &v, &kc, &vc, maybe(a[6]), maybe(a[7])});
    AttnCacheAppend p{};
    p.flags = ATTN_FLAG_DEVICE_POINTERS;
    p.dtype = code;
    cache_fields(p, kc, vc);
    p.N = slots.dim() ? slots.size(0) : 0, p.T = T, p.Hkv = H, p.D = D;
    for (int i = 0; i < 2; ++i) p.k_stride[i] = k.stride(i), p.v_stride[i] = v.stride(i);
    p.k = k.data_ptr(), p.v = v.data_ptr();
    p.slots = ints<int64_t>(slots, "slots", {p.N}, d);
    if (rows) p.rows = ints(*rows, "rows", {p.N}, d);
    descale(a[6], "k_descale", H, d, p.k_descale, p.k_descale_heads);
    descale(a[7], "v_descale", H, d, p.v_descale, p.v_descale_heads);
    {
      Unlocked unlocked;
      launch(g_append, p, d);
    }
    written({&kc, &vc});
    Py_RETURN_NONE;
  });
}

// -------------------------------------------------------------------- rotary
struct View {
  int64_t B, H, N, D;
  std::array<int64_t, 3> stride;  // batch, head, token
};

// [T, H, D] or [B, H, N, D].
View view(const Tensor& x, const char* name, c10::Device d, at::ScalarType type) {
  if (x.device() != d || x.scalar_type() != type)
    refuse(name, " must be a ", name_of(type), " tensor on ", d.str());
  View r{};
  if (x.dim() == 4)
    r = {x.size(0), x.size(1), x.size(2), x.size(3), {x.stride(0), x.stride(1), x.stride(2)}};
  else if (x.dim() == 3)
    r = {1, x.size(1), x.size(0), x.size(2), {0, x.stride(1), x.stride(0)}};
  else
    refuse(name, " must be [tokens, heads, head_dim] or [batch, heads, tokens, head_dim]");
  if (x.size(-1) > 1 && x.stride(-1) != 1) refuse(name, " head_dim must be unit-stride");
  return r;
}

PyObject* rotate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_count(n, 7);
    const Tensor *q = optional_tensor(a[0], "Q"), *k = optional_tensor(a[1], "K"),
                 *axes = optional_tensor(a[4], "axes");
    if (!q && !k) refuse("rotary needs Q or K");
    const Tensor &pos = tensor(a[2], "positions"), &freqs = tensor(a[3], "freqs"), &first = q ? *q : *k;
    const c10::Device d = first.device();
    const at::ScalarType type = first.scalar_type();
    if (!d.is_cuda()) refuse("Q and K must be CUDA tensors");
    AttnRotary p{};
    p.flags = ATTN_FLAG_DEVICE_POINTERS;
    p.dtype = code_of(type);
    if (p.dtype != ATTN_F32 && p.dtype != ATTN_BF16 && p.dtype != ATTN_F16)
      refuse("rotary takes float32, bfloat16 or float16 (got ", name_of(type), ")");
    p.neighbours = truth(a[5]);
    p.inverse = truth(a[6]);
    Tensor q_out, k_out;
    View f{};
    auto operand = [&](const Tensor* x, const char* name, int64_t& heads, int64_t (&stride)[3], int64_t (&out_stride)[3],
                       const void*& src, void*& dst, Tensor& out) {
      if (!x) return;
      const View v = view(*x, name, d, type);
      if (x != &first && (v.B != f.B || v.N != f.N || v.D != f.D || x->dim() != first.dim()))
        refuse("Q and K must have the same tokens and head_dim");
      if (x == &first) f = v;
      {
        Unlocked unlocked;
        out = at::empty_like(*x);
      }
      const View o = view(out, name, d, type);
      heads = v.H;
      for (int i = 0; i < 3; ++i) stride[i] = v.stride[i], out_stride[i] = o.stride[i];
      src = x->data_ptr(), dst = out.data_ptr();
    };
    operand(q, "Q", p.Hq, p.q_stride, p.qo_stride, p.q, p.qo, q_out);
    operand(k, "K", p.Hk, p.k_stride, p.ko_stride, p.k, p.ko, k_out);
    p.B = f.B, p.N = f.N, p.D = f.D;
    const int64_t half = freqs.dim() ? freqs.size(0) : 0;
    if (freqs.scalar_type() != at::kDouble || freqs.dim() != 1 || !freqs.is_contiguous())
      refuse("freqs must be a contiguous float64 tensor [dim / 2]");
    if (2 * half > f.D) refuse("freqs turn ", 2 * half, " values of a head_dim of ", f.D);
    on_device(freqs, "freqs", d);
    on_device(pos, "positions", d);
    p.R = 2 * half;
    p.freqs = static_cast<const double*>(freqs.data_ptr());
    if (axes) p.axes = ints(*axes, "axes", {half}, d);
    if (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong) refuse("positions must be int32 or int64");
    p.positions_64 = pos.scalar_type() == at::kLong;
    if (pos.dim() == 1 && pos.size(0) == f.N) {
      p.num_axes = 1;
      p.pos_stride[2] = pos.stride(0);
    } else if (pos.dim() == 2 && pos.size(1) == f.N) {
      p.num_axes = static_cast<int32_t>(pos.size(0));
      p.pos_stride[0] = pos.stride(0), p.pos_stride[2] = pos.stride(1);
    } else if (pos.dim() == 3 && first.dim() == 4 && pos.size(1) == f.B && pos.size(2) == f.N) {
      p.num_axes = static_cast<int32_t>(pos.size(0));
      for (int i = 0; i < 3; ++i) p.pos_stride[i] = pos.stride(i);
    } else {
      refuse("positions must be [axes, ", f.N, "]", first.dim() == 4 ? " or [axes, batch, tokens]" : "", " (got ",
             text(pos.sizes()), ")");
    }
    if (p.num_axes == 0) refuse("positions need an axis");
    p.positions = pos.data_ptr();
    {
      Unlocked unlocked;
      launch(g_rotary, p, d);
    }
    PyObject* r = PyTuple_New(2);
    if (!r) throw Raised{};
    const Tensor* outs[2] = {q ? &q_out : nullptr, k ? &k_out : nullptr};
    for (int i = 0; i < 2; ++i) {
      PyObject* o = outs[i] ? THPVariable_Wrap(*outs[i]) : Py_NewRef(Py_None);
      PyTuple_SET_ITEM(r, i, o);
    }
    return r;
  });
}

// Whether Q or K carries a forward-mode tangent.
PyObject* dual(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_count(n, 2);
    const Tensor *q = maybe(a[0]), *k = maybe(a[1]);
    return Py_NewRef((q && has_tangent(*q)) || (k && has_tangent(*k)) ? Py_True : Py_False);
  });
}

// ----------------------------------------------------------------- attention
PyObject* tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_count(n, 15);
    const Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k_new"), &v = tensor(a[2], "v_new");
    if (q.dim() != 3 || k.dim() != 3 || k.sizes() != v.sizes()) refuse("Q, K and V must be [tokens, heads, head_dim]");
    const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), H = k.size(1);
    if (k.size(0) != T) refuse("K seq_len must equal Q seq_len");
    if (k.size(2) != D) refuse("K head_dim must equal Q head_dim");
    const c10::Device d = q.device();
    const int code = code_of(q.scalar_type());
    if (!d.is_cuda() || k.device() != d || v.device() != d) refuse("Q, K and V must be CUDA tensors on one device");
    if ((code != ATTN_BF16 && code != ATTN_F16) || k.scalar_type() != q.scalar_type() ||
        v.scalar_type() != q.scalar_type())
      refuse("Q, K and V must share one element type, bfloat16 or float16");
    if (q.stride(2) != 1 || k.stride(2) != 1 || v.stride(2) != 1) refuse("head_dim must be unit-stride");
    const Tensor &kc = tensor(a[3], "k_cache"), &vc = tensor(a[4], "v_cache"), &table = tensor(a[5], "block_table"),
                 &lengths = tensor(a[6], "lengths"), &starts = tensor(a[7], "starts");
    check_cache(kc, vc, H, D, code, d);
    if (table.dim() != 2 || table.scalar_type() != at::kInt || (table.size(1) > 1 && table.stride(1) != 1))
      refuse("block_table must be int32 [B, W] with unit-stride columns");
    on_device(table, "block_table", d);
    const int64_t B = table.size(0), W = table.size(1);
    AttnTree p{};
    p.flags = ATTN_FLAG_DEVICE_POINTERS;
    p.dtype = code;
    cache_fields(p, kc, vc);
    p.B = B, p.T = T, p.Hq = Hq, p.Hkv = H, p.D = D, p.W = W;
    p.max_new = a[10] == Py_None ? T : integer(a[10]);
    p.table_stride = B > 1 ? table.stride(0) : W;
    p.block_table = static_cast<const int32_t*>(table.data_ptr());
    p.lengths = ints(lengths, "lengths", {B}, d);
    p.starts = ints(starts, "starts", {B + 1}, d);
    p.scale = number(a[8]);
    if (const Tensor* mask = optional_tensor(a[9], "mask")) {
      const auto type = mask->scalar_type();
      if (mask->dim() != 2 || (type != at::kBool && type != at::kByte) || mask->size(0) != T ||
          mask->size(1) < p.max_new || (mask->size(1) > 1 && mask->stride(1) != 1))
        refuse("mask must be bool [", T, ", at least max_new = ", p.max_new, "] with unit-stride columns");
      on_device(*mask, "mask", d);
      p.mask = static_cast<const uint8_t*>(mask->data_ptr());
      p.mask_stride = T > 1 ? mask->stride(0) : mask->size(1);
    }
    no_grad("fused_tree", {&q, &k, &v, &kc, &vc, maybe(a[8]), maybe(a[11]), maybe(a[12]), maybe(a[13]), maybe(a[14])});
    Tensor out;
    if (const Tensor* o = optional_tensor(a[11], "output")) {
      if (o->sizes() != q.sizes() || o->scalar_type() != q.scalar_type() || o->stride(2) != 1)
        refuse("output must have Q's shape and type, head_dim unit-stride");
      on_device(*o, "output", d);
      out = *o;
    } else {
      Unlocked unlocked;
      out = empty({T, Hq, D}, q.scalar_type(), d);
    }
    if (const Tensor* lse = optional_tensor(a[12], "lse")) {
      if (lse->scalar_type() != at::kFloat || lse->sizes() != Ints{T, Hq} || !lse->is_contiguous())
        refuse("lse must be a contiguous f32 tensor [tokens, heads]");
      on_device(*lse, "lse", d);
      p.lse = static_cast<float*>(lse->data_ptr());
    }
    descale(a[13], "k_descale", H, d, p.k_descale, p.k_descale_heads);
    descale(a[14], "v_descale", H, d, p.v_descale, p.v_descale_heads);
    for (int i = 0; i < 2; ++i) {
      p.q_stride[i] = q.stride(i), p.k_stride[i] = k.stride(i), p.v_stride[i] = v.stride(i);
      p.o_stride[i] = out.stride(i);
    }
    p.q = q.data_ptr(), p.k_new = k.data_ptr(), p.v_new = v.data_ptr(), p.o = out.data_ptr();
    {
      Unlocked unlocked;
      launch(g_tree, p, d);
    }
    written({maybe(a[11]), maybe(a[12])});
    return THPVariable_Wrap(out);
  });
}

// ---------------------------------------------------------------------- module
// setup(path of libattnrt.so, VerifyError, AttentionError)
PyObject* setup(PyObject*, PyObject* args) {
  const char* path;
  PyObject *verify, *attention;
  if (!PyArg_ParseTuple(args, "sOO", &path, &verify, &attention)) return nullptr;
  void* lib = dlopen(path, RTLD_NOW);
  if (!lib) return PyErr_Format(PyExc_RuntimeError, "%s", dlerror());
  auto get = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(lib, name));
    return f != nullptr;
  };
  if (!get(g_plan, "attn_cache_plan") || !get(g_append, "attn_cache_append") || !get(g_rotary, "attn_rotary") ||
      !get(g_tree, "attn_tree_fwd") || !get(g_last_error, "attn_rt_last_error") ||
      !get(g_status_string, "attn_rt_status_string"))
    return PyErr_Format(PyExc_RuntimeError, "%s lacks an entry of the serving calls", path);
  Py_XSETREF(g_verify_error, Py_NewRef(verify));
  Py_XSETREF(g_attention_error, Py_NewRef(attention));
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<plan>("plan"), method<append>("append"), method<rotate>("rotate"), method<dual>("dual"),
                           method<tree>("tree"), {"setup", setup, METH_VARARGS, nullptr},
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&g_module); }
