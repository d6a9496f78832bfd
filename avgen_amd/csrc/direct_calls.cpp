// Ordinary eager calls of the paged cache and of the gated norm, from Python's
// arguments to the C call without Python's own steps in between.
//
// Each function takes what the public function was given and either does the
// whole call or returns NotImplemented, having done nothing: for any argument that
// is not as the kernels read it (a layout to be copied, another device than the
// current one, a shape or type to be refused), and for whatever the registered ops
// exist for (modes, tracing, function transforms, subclasses).  The callers then
// go through those, which also raise every error; so nothing is refused here.
//
// Where kernels take a few microseconds the host decides: one token's attention
// (8 heads of 64) 16 us a call through Python, a norm forward and backward of
// 8 rows 195.
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/profiler/api.h>
#include <torch/types.h>

#include <cmath>

#include "avattn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

// ---------------------------------------------------------------------------
// What bind() is given: the loaded library's functions and the ops' limits
// ---------------------------------------------------------------------------

struct Bound {
  decltype(&avattn_append_paged) append_paged = nullptr;
  decltype(&avattn_page_values) page_values = nullptr;
  decltype(&avattn_paged_attention_workspace_size) attention_workspace = nullptr;
  decltype(&avattn_paged_attention) attention = nullptr;
  decltype(&avattn_gated_add_rms_norm) norm = nullptr;
  decltype(&avattn_gated_add_rms_norm_bwd_workspace_size) norm_bwd_workspace = nullptr;
  decltype(&avattn_gated_add_rms_norm_bwd) norm_bwd = nullptr;
  PyObject* parameter = nullptr;  // torch.nn.Parameter
  int64_t max_window = 0, max_slope_group = 0;
  double max_softcap = 0;
};
Bound bound;

// ---------------------------------------------------------------------------
// Ordinary tensors
// ---------------------------------------------------------------------------

// No mode, tracing or profiler.  (Python's part asks for function transforms and
// forward-mode tangents; the transforms' key is for the backward, which it does not
// see.)
bool ordinary_state() {
  return c10::impl::TorchDispatchModeTLS::stack_len() == 0 && at::impl::PythonTorchFunctionTLS::stack_len() == 0 &&
         !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !torch::jit::tracer::isTracing() && !torch::profiler::impl::profilerEnabled();
}

// On the current device, with the key set of an ordinary tensor (made in or out of
// inference mode; process constants).
bool ordinary(const Tensor& t, c10::Device device) {
  if (!t.is_cuda() || t.device() != device) return false;
  static const std::array<uint64_t, 2> plain = [&] {
    std::array<uint64_t, 2> keys{};
    for (bool inference : {false, true}) {
      c10::InferenceMode mode(inference);
      keys[inference] = at::empty({0}, t.options().requires_grad(std::nullopt)).key_set().raw_repr();
    }
    return keys;
  }();
  const uint64_t keys = t.key_set().raw_repr();
  return keys == plain[0] || keys == plain[1];
}
bool ordinary(const MaybeTensor& t, c10::Device device) { return !t || ordinary(*t, device); }

c10::Device current_device() { return c10::Device(c10::kCUDA, c10::hip::current_device()); }
void* current_stream(c10::Device d) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(d.index()).stream();
}

// Python's tensor arguments: exactly torch.Tensor or torch.nn.Parameter, or None.
bool take(PyObject* o, MaybeTensor& t) {
  t.reset();
  if (o == Py_None) return true;
  auto* type = reinterpret_cast<PyObject*>(Py_TYPE(o));
  if (type != THPVariableClass && type != bound.parameter) return false;
  t = THPVariable_Unpack(o);
  return true;
}
template <size_t N>
bool take(PyObject* const* args, std::array<MaybeTensor, N>& ts) {
  for (size_t i = 0; i < N; ++i)
    if (!take(args[i], ts[i])) return false;
  return true;
}
template <size_t N>
bool wants_grad(const std::array<MaybeTensor, N>& ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto& t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}

const void* data(const MaybeTensor& t) { return t ? t->data_ptr() : nullptr; }
template <class T>
T* data_as(const MaybeTensor& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Rows of heads, (batch, heads, length, dim) with whole 16-byte strides.
struct Strides3 {
  int64_t s[3];
};
bool head_strides(const Tensor& t, Strides3& s) {
  for (int i = 0; i < 3; ++i) s.s[i] = t.stride(i);
  return t.stride(3) == 1 && (s.s[0] | s.s[1] | s.s[2]) % 8 == 0 && aligned(t);
}

// ---------------------------------------------------------------------------
// Pools and tables
// ---------------------------------------------------------------------------

struct Pool {
  int32_t pages, heads, page, dim;
  bool e4m3;
  void *key, *value;
  int8_t *ke, *ve;
  Strides3 ks, vs;
  int64_t kes, ves;
};

bool read_pool(const MaybeTensor& key, const MaybeTensor& value, const MaybeTensor& ke, const MaybeTensor& ve,
               c10::Device device, Pool& p) {
  if (!key || !value || key->dim() != 4 || key->sizes() != value->sizes() || ke.has_value() != ve.has_value())
    return false;
  const auto sizes = key->sizes();
  const auto type = key->scalar_type();
  p.e4m3 = ke.has_value();
  if (value->scalar_type() != type || type != (p.e4m3 ? at::kFloat8_e4m3fn : at::kBFloat16)) return false;
  for (int64_t n : sizes)
    if (n < 1 || n > INT32_MAX) return false;
  p.pages = (int32_t)sizes[0], p.heads = (int32_t)sizes[1], p.page = (int32_t)sizes[2], p.dim = (int32_t)sizes[3];
  if (p.page < 16 || p.page > 256 || (p.page & (p.page - 1)) || (p.dim != 64 && p.dim != 128)) return false;
  auto pool = [&](const Tensor& t, void*& at, Strides3& s) {
    if (!ordinary(t, device) || !aligned(t)) return false;
    const int64_t unit = p.e4m3 ? 16 : 8, least = (int64_t)p.page * p.dim;
    // (Nothing steps by the strides of sizes of one.)
    const int64_t sp = p.pages > 1 ? t.stride(0) : 0, sh = p.heads > 1 ? t.stride(1) : 0;
    if (t.stride(3) != 1 || t.stride(2) != p.dim || sp % unit || sh % unit) return false;
    // Pages and heads in either order, none in another's place.
    const bool pages_in = p.heads <= 1 || (p.pages > 1 && sp <= sh);
    const int64_t inner = pages_in ? sp : sh, n = pages_in ? p.pages : p.heads;
    const int64_t outer = pages_in ? sh : sp, m = pages_in ? p.heads : p.pages;
    if (n > 1 && inner < least) return false;
    if (m > 1 && outer < (n > 1 ? inner * n : least)) return false;
    at = t.data_ptr();
    s = {{sp, sh, p.dim}};
    return true;
  };
  if (!pool(*key, p.key, p.ks) || !pool(*value, p.value, p.vs)) return false;
  auto exponents = [&](const MaybeTensor& t, int8_t*& at, int64_t& s) {
    at = nullptr, s = 0;
    if (!t) return true;
    if (!ordinary(*t, device) || t->scalar_type() != at::kChar || t->dim() != 2 || t->size(0) != p.pages ||
        t->size(1) != p.heads)
      return false;
    s = p.pages > 1 ? t->stride(0) : 0;
    at = static_cast<int8_t*>(t->data_ptr());
    return (p.heads == 1 || t->stride(1) == 1) && (p.pages == 1 || s >= p.heads);
  };
  return exponents(ke, p.ke, p.kes) && exponents(ve, p.ve, p.ves);
}

struct Tables {
  const int32_t *table, *lengths, *counts;
  int64_t stride;
  int32_t blocks;
};
bool read_tables(const MaybeTensor& table, const MaybeTensor& lengths, const MaybeTensor& counts, int64_t B,
                 c10::Device device, Tables& t) {
  if (!table || !lengths || table->dim() != 2 || table->size(0) != B || table->scalar_type() != at::kInt ||
      !ordinary(*table, device))
    return false;
  const int64_t blocks = table->size(1);
  if (blocks < 1 || blocks > INT32_MAX || (blocks > 1 && table->stride(1) != 1)) return false;
  t.stride = B > 1 ? table->stride(0) : blocks;
  if (0 < t.stride && t.stride < blocks) return false;
  t.blocks = (int32_t)blocks;
  t.table = static_cast<const int32_t*>(table->data_ptr());
  auto vector = [&](const MaybeTensor& v, const int32_t*& at) {
    at = nullptr;
    if (!v) return true;
    at = static_cast<const int32_t*>(v->data_ptr());
    return ordinary(*v, device) && v->scalar_type() == at::kInt && v->dim() == 1 && v->size(0) == B &&
           v->is_contiguous();
  };
  return vector(lengths, t.lengths) && vector(counts, t.counts);
}

// (batch, heads, length, dim) in bf16, of a size that is not empty.
bool heads_of(const MaybeTensor& t, int64_t dim, c10::Device device) {
  if (!t || !ordinary(*t, device) || t->scalar_type() != at::kBFloat16 || t->dim() != 4 || t->size(3) != dim)
    return false;
  for (int i = 0; i < 3; ++i)
    if (t->size(i) < 1 || t->size(i) > INT32_MAX) return false;
  return true;
}

PyObject* not_here() { Py_RETURN_NOTIMPLEMENTED; }

// paged_attention(query, key pages, value pages, key exponents, value exponents,
// block table, lengths, counts, slopes, window, scale, softcap): the output.
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  std::array<MaybeTensor, 9> ts;
  if (n != 12 || !ordinary_state() || !take(args, ts) || wants_grad(ts)) return not_here();
  const auto& [q, kp, vp, ke, ve, table, lengths, counts, slopes] = ts;
  const long long window = PyLong_AsLongLong(args[9]);
  const double scale = PyFloat_AsDouble(args[10]), softcap = PyFloat_AsDouble(args[11]);
  if (PyErr_Occurred()) return nullptr;
  Tensor out;
  auto go = [&] {
    pybind11::gil_scoped_release no_gil;
    const c10::Device device = current_device();
    Pool p;
    Tables t;
    Strides3 qs, os;
    if (!read_pool(kp, vp, ke, ve, device, p) || !heads_of(q, p.dim, device) || !head_strides(*q, qs)) return false;
    const int64_t B = q->size(0), H = q->size(1), L = q->size(2);
    if (H % p.heads || !read_tables(table, lengths, counts, B, device, t) || window < 0 ||
        window > bound.max_window || !(std::isfinite(scale) && scale > 0) ||
        !(softcap >= 0 && softcap <= bound.max_softcap))
      return false;
    if (slopes && (!ordinary(*slopes, device) || slopes->scalar_type() != at::kFloat || slopes->dim() != 1 ||
                   slopes->size(0) != H || !slopes->is_contiguous() || H / p.heads > bound.max_slope_group))
      return false;
    at::AutoDispatchBelowADInplaceOrView below;
    out = at::empty_like(*q);
    if (!head_strides(out, os)) return false;
    const size_t need = bound.attention_workspace((int32_t)B, (int32_t)H, p.heads, (int32_t)L, p.dim, t.blocks, p.page,
                                                  (int32_t)window, p.e4m3);
    // (Behind the workspace, which is whole 16 bytes, the rows' lse.)
    Tensor scratch = at::empty({(int64_t)need + 4 * B * H * L}, q->options().dtype(at::kByte));
    char* at = static_cast<char*>(scratch.data_ptr());
    return bound.attention(q->data_ptr(), qs.s, (int32_t)B, (int32_t)H, p.heads, (int32_t)L, p.dim, t.table, t.stride,
                           t.blocks, t.lengths, t.counts, p.key, p.ks.s, p.value, p.vs.s, p.ke, p.kes, p.ve, p.ves,
                           p.pages, p.page, (int32_t)window, (float)scale, (float)softcap,
                           data_as<const float>(slopes), out.data_ptr(), os.s, reinterpret_cast<float*>(at + need), at,
                           need, current_stream(device)) == AVATTN_OK;
  };
  return go() ? THPVariable_Wrap(out) : not_here();
  END_HANDLE_TH_ERRORS
}

// append_paged(key, value, query, cos, sin, block table, lengths, counts, key
// pages, value pages, key exponents, value exponents, start, half): the rotated
// query, or None.
PyObject* append_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  std::array<MaybeTensor, 12> ts;
  if (n != 14 || !ordinary_state() || !take(args, ts) || wants_grad(ts)) return not_here();
  const auto& [k, v, q, cos, sin, table, lengths, counts, kp, vp, ke, ve] = ts;
  const long long start = PyLong_AsLongLong(args[12]);
  const int half = PyObject_IsTrue(args[13]);
  if (PyErr_Occurred()) return nullptr;
  Tensor out;
  auto go = [&] {
    pybind11::gil_scoped_release no_gil;
    const c10::Device device = current_device();
    Pool p;
    Tables t;
    Strides3 ks, vs, qs{}, os{};
    if (!read_pool(kp, vp, ke, ve, device, p) || !heads_of(k, p.dim, device) || !heads_of(v, p.dim, device) ||
        k->sizes() != v->sizes() || k->size(1) != p.heads || !head_strides(*k, ks) || !head_strides(*v, vs) ||
        cos.has_value() != sin.has_value())
      return false;
    const int64_t B = k->size(0), L = k->size(2);
    if (!read_tables(table, lengths, counts, B, device, t)) return false;
    if (q && (!heads_of(q, p.dim, device) || q->size(0) != B || q->size(2) != L || !head_strides(*q, qs)))
      return false;
    int64_t pairs = 0, tsb = 0;
    if (cos) {
      for (const MaybeTensor* x : {&cos, &sin})
        if (!ordinary(**x, device) || (*x)->scalar_type() != at::kFloat || (*x)->dim() != 4 ||
            (*x)->sizes() != cos->sizes() || !(*x)->is_contiguous())
          return false;
      pairs = cos->size(3);
      if (pairs < 1 || pairs > p.dim || start < 0 || start > p.dim || start + 2 * pairs > p.dim ||
          cos->size(2) != L || cos->size(1) != 1 || (cos->size(0) != 1 && cos->size(0) != B))
        return false;
      tsb = cos->size(0) == 1 ? 0 : L * pairs;
    }
    at::AutoDispatchBelowADInplaceOrView below;
    if (q) {
      out = at::empty_like(*q);
      if (!head_strides(out, os)) return false;
    }
    if (bound.append_paged(k->data_ptr(), ks.s, v->data_ptr(), vs.s, data(q), q ? qs.s : nullptr,
                           q ? (int32_t)q->size(1) : 0, q ? out.data_ptr() : nullptr, q ? os.s : nullptr, (int32_t)B,
                           p.heads, (int32_t)L, p.dim, data_as<const float>(cos), data_as<const float>(sin), tsb,
                           (int32_t)pairs, cos ? (int32_t)start : 0, half, t.table, t.stride, t.blocks, t.lengths,
                           t.counts, p.key, p.ks.s, p.value, p.vs.s, p.ke, p.kes, p.ve, p.ves, p.pages, p.page,
                           current_stream(device)) != AVATTN_OK)
      return false;
    for (const MaybeTensor* w : {&kp, &vp, &ke, &ve})  // written in place
      if (*w && !(*w)->is_inference()) (*w)->unsafeGetTensorImpl()->bump_version();
    return true;
  };
  if (!go()) return not_here();
  if (!out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// page_values(key pages, value pages, key exponents, value exponents): both pools'
// values in bf16.
PyObject* page_values(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  std::array<MaybeTensor, 4> ts;
  if (n != 4 || !ordinary_state() || !take(args, ts) || wants_grad(ts)) return not_here();
  const auto& [kp, vp, ke, ve] = ts;
  Tensor key, value;
  bool done = false;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::Device device = current_device();
    Pool p;
    if (read_pool(kp, vp, ke, ve, device, p) && p.e4m3) {
      at::AutoDispatchBelowADInplaceOrView below;
      const auto options = kp->options().dtype(at::kBFloat16);
      key = at::empty(kp->sizes(), options);
      value = at::empty(kp->sizes(), options);
      done = bound.page_values(p.key, p.ks.s, p.ke, p.kes, key.data_ptr(), p.value, p.vs.s, p.ve, p.ves,
                               value.data_ptr(), p.pages, p.heads, p.page, p.dim,
                               current_stream(device)) == AVATTN_OK;
    }
  }
  if (!done) return not_here();
  return Py_BuildValue("(NN)", THPVariable_Wrap(key), THPVariable_Wrap(value));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// The gated norm
// ---------------------------------------------------------------------------

// `t` (..., width) as rows of contiguous values, their stride apart.
bool rows_of(const Tensor& t, int64_t W, int64_t& stride) {
  stride = W;
  if (t.is_contiguous()) return true;
  if (t.stride(-1) != 1 && W > 1) return false;
  if (t.dim() == 1 || t.numel() <= W) return true;
  int64_t expect = -1;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (expect < 0)
      stride = t.stride(d);
    else if (t.stride(d) != expect)
      return false;
    expect = t.stride(d) * t.size(d);
  }
  return true;
}

struct NormCall {
  c10::Device device{c10::kCUDA};
  int64_t rows, width, group, xs, rs, gs = 0, ss = 0, ts = 0;
  bool f32, w32 = false, p32 = false, m32 = false;
};

// Whether the call is one for here, and its layout.
bool read_norm(const Tensor& x, const Tensor& r, const MaybeTensor& w, const MaybeTensor& p, const MaybeTensor& gate,
               const MaybeTensor& scale, const MaybeTensor& shift, NormCall& c) {
  c.device = current_device();
  if (!ordinary(x, c.device) || !ordinary(r, c.device) || x.dim() < 1 || x.numel() == 0) return false;
  const auto type = x.scalar_type();
  c.f32 = type == at::kFloat;
  if ((!c.f32 && type != at::kBFloat16) || r.scalar_type() != type || r.sizes() != x.sizes()) return false;
  c.width = x.size(-1);
  c.rows = c.group = x.numel() / c.width;
  if (!rows_of(x, c.width, c.xs) || !rows_of(r, c.width, c.rs)) return false;
  auto gain = [&](const MaybeTensor& t, bool& t32) {
    if (!t) return true;
    t32 = t->scalar_type() == at::kFloat;
    return ordinary(*t, c.device) && (t32 || t->scalar_type() == type) && t->dim() == 1 && t->size(0) == c.width &&
           t->is_contiguous();
  };
  if (!gain(w, c.w32) || !gain(p, c.p32)) return false;
  const MaybeTensor& first = gate ? gate : scale ? scale : shift;
  if (!first) return true;
  auto modulation = [&](const MaybeTensor& t, int64_t& stride) {
    if (!t) return true;
    return ordinary(*t, c.device) && t->scalar_type() == first->scalar_type() && t->sizes() == first->sizes() &&
           rows_of(*t, c.width, stride);
  };
  c.m32 = first->scalar_type() == at::kFloat;
  if (!c.m32 && first->scalar_type() != type) return false;
  if (first->dim() < 1 || first->dim() > x.dim() || first->size(-1) != c.width) return false;
  // One row, one for each sample, or one for each row of x.
  const bool one = first->numel() == c.width;
  const bool sample = first->dim() == 3 && x.dim() == 3 && first->size(1) == 1 && first->size(0) == x.size(0);
  if (!one && !sample && first->sizes() != x.sizes()) return false;
  c.group = x.numel() / first->numel();
  return modulation(gate, c.gs) && modulation(scale, c.ss) && modulation(shift, c.ts);
}

bool norm_forward(const NormCall& c, const Tensor& x, const Tensor& r, const MaybeTensor& w, const MaybeTensor& p,
                  const MaybeTensor& gate, const MaybeTensor& scale, const MaybeTensor& shift, double factor,
                  double eps, Tensor& norm, Tensor& sum, Tensor* stats) {
  at::AutoDispatchBelowADInplaceOrView below;
  sum = at::empty(x.sizes(), x.options());
  norm = at::empty(x.sizes(), x.options());
  if (stats != nullptr) *stats = at::empty({c.rows, 2}, x.options().dtype(at::kFloat));
  return bound.norm(x.data_ptr(), c.xs, r.data_ptr(), c.rs, data(w), c.w32, data(p), c.p32, data(gate), c.gs,
                    data(scale), c.ss, data(shift), c.ts, c.m32, c.rows, c.width, c.group, c.f32, (float)factor,
                    (float)eps, sum.data_ptr(), norm.data_ptr(),
                    stats != nullptr ? static_cast<float*>(stats->data_ptr()) : nullptr,
                    current_stream(c.device)) == AVATTN_OK;
}

struct Refused {};

class GatedNorm : public torch::autograd::Function<GatedNorm> {
 public:
  static variable_list forward(AutogradContext* ctx, const NormCall* c, const Tensor& x, const Tensor& r,
                               const MaybeTensor& w, const MaybeTensor& p, const MaybeTensor& gate,
                               const MaybeTensor& scale, const MaybeTensor& shift, double factor, double eps) {
    Tensor norm, sum, stats;
    if (!norm_forward(*c, x, r, w, p, gate, scale, shift, factor, eps, norm, sum, &stats)) throw Refused();
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, r, stats, w.value_or(Tensor()), p.value_or(Tensor()), gate.value_or(Tensor()),
                            scale.value_or(Tensor()), shift.value_or(Tensor())});
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["eps"] = eps;
    return {norm, sum};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(10);
    Tensor dn = grads[0], dh = grads[1];
    if (!dn.defined() && !dh.defined()) return result;
    const variable_list saved = ctx->get_saved_variables();
    if (!dn.defined()) dn = at::zeros_like(saved[0]);  // the sum alone was used
    const double factor = ctx->saved_data["factor"].toDouble(), eps = ctx->saved_data["eps"].toDouble();
    auto maybe = [](const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
    const Tensor &x = saved[0], &r = saved[1], &stats = saved[2];
    const std::array<MaybeTensor, 5> vec = {maybe(saved[3]), maybe(saved[4]), maybe(saved[5]), maybe(saved[6]),
                                            maybe(saved[7])};
    const bool alike = !vec[1] && !vec[2] && factor == 1.0;
    std::array<Tensor, 7> d;  // of x, the residual and the vectors
    if (!run(dn, dh, x, r, stats, vec, factor, eps, alike, d)) {
      // Whatever is not ordinary: the op (which a backward of this one refuses).
      static const auto op = c10::Dispatcher::singleton()
                                 .findSchemaOrThrow("avgen_amd::gated_add_rms_norm_bwd", "")
                                 .typed<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>(
                                     const Tensor&, const MaybeTensor&, const Tensor&, const Tensor&, const Tensor&,
                                     const MaybeTensor&, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&,
                                     const MaybeTensor&, double, double)>();
      std::tie(d[0], d[1], d[2], d[3], d[4], d[5], d[6]) =
          op.call(dn, maybe(dh), x, r, stats, vec[0], vec[1], vec[2], vec[3], vec[4], factor, eps);
      if (alike) d[1] = d[0];
    }
    result[1] = d[0];
    result[2] = d[1];
    for (int i = 0; i < 5; ++i)
      if (vec[i]) result[3 + i] = d[2 + i];
    return result;
  }

 private:
  static bool run(const Tensor& dn, const Tensor& dh, const Tensor& x, const Tensor& r, const Tensor& stats,
                  const std::array<MaybeTensor, 5>& vec, double factor, double eps, bool alike,
                  std::array<Tensor, 7>& d) {
    NormCall c;
    if (at::GradMode::is_enabled() || !ordinary_state() ||
        !read_norm(x, r, vec[0], vec[1], vec[2], vec[3], vec[4], c))
      return false;
    int64_t dns = 0, dhs = 0;
    for (const Tensor* g : {&dn, &dh})
      if (g->defined() &&
          (!ordinary(*g, c.device) || g->scalar_type() != x.scalar_type() || g->sizes() != x.sizes() ||
           !rows_of(*g, c.width, g == &dn ? dns : dhs)))
        return false;
    if (!ordinary(stats, c.device) || stats.scalar_type() != at::kFloat || !stats.is_contiguous() ||
        stats.numel() != 2 * c.rows)
      return false;
    at::AutoDispatchBelowADInplaceOrView below;
    d[0] = at::empty(x.sizes(), x.options());
    d[1] = alike ? d[0] : at::empty(x.sizes(), x.options());
    for (int i = 0; i < 5; ++i)
      if (vec[i]) d[2 + i] = at::empty(vec[i]->sizes(), vec[i]->options());
    const bool modulated = vec[2] || vec[3] || vec[4];
    const size_t need = bound.norm_bwd_workspace(c.rows, c.width, c.group, modulated);
    Tensor ws = at::empty({(int64_t)std::max<size_t>(need, 256)}, x.options().dtype(at::kByte));
    auto out = [&](int i) { return d[i].defined() ? d[i].data_ptr() : nullptr; };
    return bound.norm_bwd(dn.data_ptr(), dns, dh.defined() ? dh.data_ptr() : nullptr, dhs, x.data_ptr(), c.xs,
                          r.data_ptr(), c.rs, static_cast<const float*>(stats.data_ptr()), data(vec[0]), c.w32,
                          data(vec[1]), c.p32, data(vec[2]), c.gs, data(vec[3]), c.ss, data(vec[4]), c.ts, c.m32,
                          c.rows, c.width, c.group, c.f32, (float)factor, (float)eps, d[0].data_ptr(),
                          alike ? nullptr : d[1].data_ptr(), out(2), out(3), out(4), out(5), out(6), ws.data_ptr(),
                          (size_t)ws.numel(), current_stream(c.device)) == AVATTN_OK;
  }
};

// gated_add_rms_norm(x, residual, weight, post weight, gate, scale, shift,
// residual factor, eps): (norm, sum).
PyObject* gated_add_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  std::array<MaybeTensor, 7> ts;
  if (n != 9 || !ordinary_state() || !take(args, ts) || !ts[0] || !ts[1]) return not_here();
  const auto& [x, r, w, p, gate, scale, shift] = ts;
  const double factor = PyFloat_AsDouble(args[7]), eps = PyFloat_AsDouble(args[8]);
  if (PyErr_Occurred()) return nullptr;
  Tensor norm, sum;
  bool done = false;
  {
    pybind11::gil_scoped_release no_gil;
    NormCall c;
    if (std::isfinite(factor) && std::isfinite(eps) && eps >= 0 && read_norm(*x, *r, w, p, gate, scale, shift, c)) {
      if (wants_grad(ts)) {
        try {
          variable_list both = GatedNorm::apply(&c, *x, *r, w, p, gate, scale, shift, factor, eps);
          norm = std::move(both[0]), sum = std::move(both[1]);
          done = true;
        } catch (const Refused&) {
        }
      } else {
        done = norm_forward(c, *x, *r, w, p, gate, scale, shift, factor, eps, norm, sum, nullptr);
      }
    }
  }
  if (!done) return not_here();
  return Py_BuildValue("(NN)", THPVariable_Wrap(norm), THPVariable_Wrap(sum));
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the C functions in Bound's order, torch.nn.Parameter, largest
// window, largest softcap, largest group of heads with slopes)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long f[7];
  PyObject* parameter;
  long long window, group;
  double softcap;
  if (!PyArg_ParseTuple(args, "(KKKKKKK)OLdL", f, f + 1, f + 2, f + 3, f + 4, f + 5, f + 6, &parameter, &window,
                        &softcap, &group))
    return nullptr;
  auto set = [](auto& fn, unsigned long long at) {
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(static_cast<uintptr_t>(at));
  };
  set(bound.append_paged, f[0]);
  set(bound.page_values, f[1]);
  set(bound.attention_workspace, f[2]);
  set(bound.attention, f[3]);
  set(bound.norm, f[4]);
  set(bound.norm_bwd_workspace, f[5]);
  set(bound.norm_bwd, f[6]);
  Py_INCREF(parameter);
  bound.parameter = parameter;
  bound.max_window = window, bound.max_softcap = softcap, bound.max_slope_group = group;
  Py_RETURN_NONE;
}

template <class F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"paged_attention", fast(paged_attention), METH_FASTCALL, nullptr},
    {"append_paged", fast(append_paged), METH_FASTCALL, nullptr},
    {"page_values", fast(page_values), METH_FASTCALL, nullptr},
    {"gated_add_rms_norm", fast(gated_add_rms_norm), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_direct_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__direct_calls() { return PyModule_Create(&module); }
