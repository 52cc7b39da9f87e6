// torch_operators.cpp -- the operators around self-attention for Python: torch tensors to the C ABI
// (include/fattn.h), with their checks, allocations and autograd nodes.
//
// Their smallest calls, a decoding token's, are bound by the host, so what lies between Python and the
// launch is compiled: fused_rotary of one token takes 7.5 us a call, 12.8 with these steps in Python;
// paged_append 5.1 for 13.7; paged_attention over 240 tokens 7.5 for 11.2. With the nodes in
// Python a small training call takes 15 us more: fused_rotary and its gradient 77 us, 60 so, where an
// elementwise product and its gradient take 52; fused_cross_attention 78, 62.
//
// Every entry takes its positional arguments from candle_fused_attn/{rotary,paged,cross}.py, whose
// docstrings say what they mean. A refused argument raises the package's FusedAttentionError.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>
#include <vector>

#include "fattn.h"

namespace {

using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
typedef std::vector<Tensor> Tensors;

PyObject* g_error = nullptr;  // candle_fused_attn.FusedAttentionError

// A refused argument or a failed launch; `code` as the C ABI returned it (0: refused here).
struct OpError : std::runtime_error {
  explicit OpError(const std::string& msg, int c = 0) : std::runtime_error(msg), code(c) {}
  int code;
};

void set_python(const OpError& e) {
  PyObject* x = PyObject_CallFunction(g_error, "si", e.what(), e.code);
  if (!x) return;  // (with that call's own error set)
  PyErr_SetObject(g_error, x);
  Py_DECREF(x);
}
// fn() inside a backward, which may be any thread without the interpreter's lock: an OpError leaves as
// the Python exception that the engine hands to its caller.
template <typename F>
auto in_backward(F fn) -> decltype(fn()) {
  try {
    return fn();
  } catch (const OpError& e) {
    const PyGILState_STATE state = PyGILState_Ensure();
    set_python(e);
    python_error error;
    error.persist();
    PyGILState_Release(state);
    throw error;
  }
}
bool records(std::initializer_list<const Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts) {
    if (t->defined() && t->requires_grad()) return true;
  }
  return false;
}
// No operand may have a tangent of forward-mode differentiation: a result without one would be a derivative
// of 0. (Tensors that are absent have none.)
void no_tangents(const char* who, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) {
    if (t->defined() && t->_fw_grad(0).defined()) {
      throw OpError(std::string(who) + ": no forward-mode derivative");
    }
  }
}

std::string shape_of(at::IntArrayRef x) {
  std::string out = "[";
  for (size_t i = 0; i < x.size(); ++i) out += (i ? ", " : "") + std::to_string(x[i]);
  return out + "]";
}
const char* name_of(ScalarType t) {
  switch (t) {
    case ScalarType::Float: return "float32";
    case ScalarType::Half: return "float16";
    case ScalarType::BFloat16: return "bfloat16";
    case ScalarType::Double: return "float64";
    case ScalarType::Int: return "int32";
    case ScalarType::Long: return "int64";
    default: return c10::toString(t);
  }
}

// The element types an operand may have.
typedef std::initializer_list<ScalarType> Types;
constexpr ScalarType kF32 = ScalarType::Float, kF16 = ScalarType::Half, kBF16 = ScalarType::BFloat16;
constexpr ScalarType kI32 = ScalarType::Int, kI64 = ScalarType::Long, kF64 = ScalarType::Double;

// A tensor of `rank` dimensions on a HIP device (that of `like`), of one of `types`.
void require(const char* who, const char* name, const Tensor& t, int64_t rank, const Tensor* like,
             Types types) {
  bool known = false;
  for (ScalarType x : types) known = known || t.scalar_type() == x;
  if (known && t.dim() == rank && t.is_cuda() && (!like || t.get_device() == like->get_device())) return;
  const std::string what = std::string(who) + ": " + name;
  if (!known) {
    std::string takes;
    for (ScalarType x : types) takes += (takes.empty() ? "" : ", ") + std::string(name_of(x));
    throw OpError(what + " must be " + takes + ", got " + name_of(t.scalar_type()));
  }
  if (t.dim() != rank) {
    throw OpError(what + " must have " + std::to_string(rank) + " dimensions, got shape " +
                  shape_of(t.sizes()));
  }
  if (!t.is_cuda()) throw OpError(what + " is not on a HIP device (this operator has no CPU path)");
  throw OpError(what + " is on " + t.device().str() + ", the first operand on " + like->device().str());
}

int type_code(const Tensor& t) {
  return t.scalar_type() == kF32 ? FATTN_F32 : t.scalar_type() == kF16 ? FATTN_F16 : FATTN_BF16;
}
// `t` itself where its last dimension is contiguous, else a contiguous copy.
Tensor rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
// A four-dimensional `t` itself where its rows are contiguous and 16-byte aligned, else a contiguous copy.
Tensor aligned_rows(const Tensor& t) {
  const int64_t per = 16 / t.element_size();
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.stride(i) % per == 0 || t.size(i) <= 1);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// fn(stream) on torch's current stream of t's device, with that device current.
template <typename F>
void launch(const Tensor& t, F fn) {
  const c10::OptionalDeviceGuard guard(t.device());
  const int rc = fn(static_cast<void*>(c10::hip::getCurrentHIPStream(t.get_device()).stream()));
  if (rc != 0) throw OpError(fattn_last_error(), rc);
}
// An empty tensor laid out like t, whose rows are contiguous, and its own contiguous too. (A contiguous one
// by one call of the dispatcher instead of two. Where rows of t overlap, in windows of a longer row, torch
// may order the dimensions otherwise.)
Tensor like(const Tensor& t) {
  if (!t.is_contiguous()) {
    Tensor y = at::empty_like(t);
    if (y.stride(-1) == 1) return y;
  }
  return at::empty(t.sizes(), t.options());
}
// A workspace from torch's allocator (undefined for 0 bytes).
Tensor workspace(const Tensor& t, size_t bytes) {
  return bytes == 0 ? Tensor()
                    : at::empty({static_cast<int64_t>(bytes)}, t.options().dtype(ScalarType::Byte));
}
void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// --- Rotary positions ------------------------------------------------------------------------------

struct Turn {
  Tensor positions, frequencies;
  int64_t heads;  // 0: [b, h, s, d] operands; else of the one [b, s, 3 h d] projection
  bool interleaved;
  double magnitude;
  bool inverse;
};

// The frequencies get no gradient: those that ask for one are refused where a graph would be recorded.
void not_learned(const char* who, const Tensor& f) {
  if (records({&f})) {
    throw OpError(std::string(who) + ": no gradient of the frequencies (detach them, or call it under "
                  "torch.no_grad())");
  }
}
int64_t check_frequencies(const char* who, const Tensor& f, int64_t d, const Tensor& like) {
  require(who, "frequencies", f, 1, &like, {kF64});
  if (2 * f.size(0) > d || !f.is_contiguous()) {
    throw OpError(std::string(who) + ": contiguous frequencies of at most " + std::to_string(d / 2) +
                  " pairs expected, got " + std::to_string(f.size(0)));
  }
  return 2 * f.size(0);
}
void check_positions(const char* who, const Tensor& p, int64_t b, int64_t s, const Tensor& like) {
  if (p.dim() != 1 && p.dim() != 2) {
    throw OpError(std::string(who) + ": positions must be a [s] or [b, s] tensor");
  }
  require(who, "positions", p, p.dim(), &like, {kI64, kI32});
  if (p.size(-1) != s || (p.dim() == 2 && p.size(0) != 1 && p.size(0) != b)) {
    throw OpError(std::string(who) + ": positions [" + std::to_string(s) + "] or [" + std::to_string(b) +
                  ", " + std::to_string(s) + "] expected, got shape " + shape_of(p.sizes()));
  }
}

// The turned tensors: one or two operands, or the one projection, whose q and k are turned and v copied.
Tensors turned(const Tensors& xs, const Turn& how) {
  Tensors ys;
  for (const Tensor& x : xs) ys.push_back(like(x));
  const Tensor& x = xs[0];
  int64_t heads[3] = {0, 0, 0}, xst[9] = {}, yst[9] = {}, pst[2] = {};
  const void* xp[3] = {};
  void* yp[3] = {};
  int64_t b, s, d;
  int mask = 0b111;
  if (how.heads > 0) {
    b = x.size(0), s = x.size(1), d = x.size(2) / (3 * how.heads);
    const int64_t step = how.heads * d * x.element_size();
    for (int i = 0; i < 3; ++i) {
      heads[i] = how.heads;
      xp[i] = static_cast<const char*>(x.data_ptr()) + i * step;
      yp[i] = static_cast<char*>(ys[0].data_ptr()) + i * step;
      xst[3 * i] = x.stride(0), xst[3 * i + 1] = d, xst[3 * i + 2] = x.stride(1);
      yst[3 * i] = ys[0].stride(0), yst[3 * i + 1] = d, yst[3 * i + 2] = ys[0].stride(1);
    }
    mask = 0b011;
  } else {
    b = x.size(0), s = x.size(2), d = x.size(3);
    for (size_t i = 0; i < xs.size(); ++i) {
      heads[i] = xs[i].size(1);
      xp[i] = xs[i].data_ptr(), yp[i] = ys[i].data_ptr();
      for (int k = 0; k < 3; ++k) xst[3 * i + k] = xs[i].stride(k), yst[3 * i + k] = ys[i].stride(k);
    }
  }
  const Tensor& p = how.positions;
  pst[0] = p.dim() == 1 || p.size(0) == 1 ? 0 : p.stride(0);
  pst[1] = p.stride(-1);
  launch(x, [&](void* stream) {
    return fattn_rotary(type_code(x), b, s, d, heads, xp, yp, xst, yst, mask, p.data_ptr(),
                        p.scalar_type() == kI64 ? 64 : 32, pst,
                        static_cast<const double*>(how.frequencies.data_ptr()), 2 * how.frequencies.size(0),
                        how.interleaved, how.magnitude, how.inverse, stream);
  });
  return ys;
}

// The turn as a node, of one operand or two; its gradient is the turn back, the same node again where a
// graph of it is asked for (so it can be differentiated again).
void remember(AutogradContext* ctx, const Turn& how) {
  ctx->save_for_backward({how.positions, how.frequencies});
  ctx->saved_data["heads"] = how.heads;
  ctx->saved_data["interleaved"] = how.interleaved;
  ctx->saved_data["magnitude"] = how.magnitude;
  ctx->saved_data["inverse"] = how.inverse;
  ctx->set_materialize_grads(false);
}
Turn turn_back(AutogradContext* ctx, const Tensor& grad) {
  const Tensors saved = ctx->get_saved_variables();
  const Turn how{saved[0],
                 saved[1],
                 ctx->saved_data["heads"].toInt(),
                 ctx->saved_data["interleaved"].toBool(),
                 ctx->saved_data["magnitude"].toDouble(),
                 !ctx->saved_data["inverse"].toBool()};
  // (Hooks on saved tensors may have replaced them.)
  if (how.heads > 0) {
    check_positions("fused_rotary_qkv", how.positions, grad.size(0), grad.size(1), grad);
    check_frequencies("fused_rotary_qkv", how.frequencies, grad.size(2) / 3 / how.heads, grad);
  } else {
    check_positions("fused_rotary", how.positions, grad.size(0), grad.size(2), grad);
    check_frequencies("fused_rotary", how.frequencies, grad.size(3), grad);
  }
  return how;
}
Tensor turn_one(const Tensor& x, const Turn& how);
Tensors turn_two(const Tensor& q, const Tensor& k, const Turn& how);

struct TurnOne : Function<TurnOne> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Turn& how) {
    remember(ctx, how);
    return turned({rows(x)}, how)[0];
  }
  static Tensors backward(AutogradContext* ctx, const Tensors& grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    return in_backward([&]() -> Tensors {
      const Turn how = turn_back(ctx, grads[0]);
      no_tangents(how.heads > 0 ? "fused_rotary_qkv" : "fused_rotary", {&grads[0]});
      return {turn_one(grads[0], how), Tensor()};
    });
  }
};
struct TurnTwo : Function<TurnTwo> {
  static Tensors forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Turn& how) {
    remember(ctx, how);
    return turned({rows(q), rows(k)}, how);
  }
  static Tensors backward(AutogradContext* ctx, const Tensors& grads) {
    const bool gq = grads[0].defined() && ctx->needs_input_grad(0);
    const bool gk = grads[1].defined() && ctx->needs_input_grad(1);
    if (!gq && !gk) return {Tensor(), Tensor(), Tensor()};
    return in_backward([&]() -> Tensors {
      const Turn how = turn_back(ctx, gq ? grads[0] : grads[1]);
      no_tangents("fused_rotary", {&grads[0], &grads[1]});
      if (gq && gk) {
        const Tensors both = turn_two(grads[0], grads[1], how);
        return {both[0], both[1], Tensor()};
      }
      return {gq ? turn_one(grads[0], how) : Tensor(), gk ? turn_one(grads[1], how) : Tensor(), Tensor()};
    });
  }
};
Tensor turn_one(const Tensor& x, const Turn& how) {
  return records({&x}) ? TurnOne::apply(x, how) : turned({rows(x)}, how)[0];
}
Tensors turn_two(const Tensor& q, const Tensor& k, const Turn& how) {
  return records({&q, &k}) ? TurnTwo::apply(q, k, how) : turned({rows(q), rows(k)}, how);
}

Tensors fused_rotary(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& f,
                     bool interleaved, double magnitude) {
  const char* who = "fused_rotary";
  no_tangents(who, {&q, &k, &f});
  not_learned(who, f);
  require(who, "q", q, 4, nullptr, {kF32, kF16, kBF16});
  require(who, "k", k, 4, &q, {q.scalar_type()});
  if (k.size(0) != q.size(0) || k.size(2) != q.size(2) || k.size(3) != q.size(3)) {
    throw OpError(std::string(who) + ": q and k must agree but for their heads, got " + shape_of(q.sizes()) +
                  " and " + shape_of(k.sizes()));
  }
  check_positions(who, positions, q.size(0), q.size(2), q);
  check_frequencies(who, f, q.size(3), q);
  return turn_two(q, k, Turn{positions, f, 0, interleaved, magnitude, false});
}

Tensor fused_rotary_qkv(const Tensor& qkv, int64_t heads, const Tensor& positions, const Tensor& f,
                        bool interleaved, double magnitude) {
  const char* who = "fused_rotary_qkv";
  no_tangents(who, {&qkv, &f});
  not_learned(who, f);
  require(who, "qkv", qkv, 3, nullptr, {kF32, kF16, kBF16});
  const int64_t w = qkv.size(2);
  if (heads <= 0 || heads > w / 3 || w % (3 * heads) != 0) {
    throw OpError(std::string(who) + ": last dimension " + std::to_string(w) + " is not 3 x " +
                  std::to_string(heads) + " heads x head_dim");
  }
  check_positions(who, positions, qkv.size(0), qkv.size(1), qkv);
  check_frequencies(who, f, w / 3 / heads, qkv);
  return turn_one(qkv, Turn{positions, f, heads, interleaved, magnitude, false});
}

// --- The paged cache -------------------------------------------------------------------------------

void check_cache(const char* who, const Tensor& x, const Tensor& kp, const Tensor& vp, const Tensor& table,
                 const Tensor& lengths, int64_t b, int64_t d) {
  require(who, "k_pages", kp, 4, &x, {kF32, kF16, kBF16});
  require(who, "v_pages", vp, 4, &x, {kp.scalar_type()});
  if (vp.sizes() != kp.sizes() || kp.size(3) != d) {
    throw OpError(std::string(who) + ": k_pages and v_pages [pages, kv_heads, page_size, " +
                  std::to_string(d) + "] expected, got " + shape_of(kp.sizes()) + " and " +
                  shape_of(vp.sizes()));
  }
  if (d > 1 && (kp.stride(3) != 1 || vp.stride(3) != 1)) {
    throw OpError(std::string(who) + ": k_pages and v_pages must have a contiguous last dimension, strides " +
                  shape_of(kp.strides()) + " and " + shape_of(vp.strides()));
  }
  require(who, "page_table", table, 2, &x, {kI32});
  require(who, "lengths", lengths, 1, &x, {kI32});
  if (table.size(0) != b || lengths.size(0) != b || !lengths.is_contiguous() ||
      (table.stride(1) != 1 && table.size(1) > 1)) {
    throw OpError(std::string(who) + ": a page table [" + std::to_string(b) +
                  ", width] with contiguous rows and contiguous lengths [" + std::to_string(b) +
                  "] expected, got " + shape_of(table.sizes()) + " and " + shape_of(lengths.sizes()));
  }
}
const int32_t* ints(const Tensor& t) { return t.defined() ? static_cast<const int32_t*>(t.data_ptr()) : nullptr; }
void no_graph(const char* who, std::initializer_list<const Tensor*> ts) {
  if (records(ts)) throw OpError(std::string(who) + ": not differentiable (call it under torch.no_grad())");
}
// The pages were written: a graph that saved them before must not run on them. (Tensors of inference mode
// have no versions.)
void wrote(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
bool broadcast(const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.stride(i) == 0 && t.size(i) > 1) return true;
  }
  return false;
}

// counts, q, f: undefined where absent. The turned q, undefined without one.
Tensor paged_append(const Tensor& k0, const Tensor& v0, const Tensor& kp, const Tensor& vp,
                    const Tensor& table, const Tensor& lengths, const Tensor& counts, const Tensor& q0,
                    const Tensor& f, bool interleaved, double magnitude) {
  const char* who = "paged_append";
  no_tangents(who, {&k0, &v0, &kp, &vp, &q0, &f});
  not_learned(who, f);
  require(who, "k", k0, 4, nullptr, {kF32, kF16, kBF16});
  require(who, "v", v0, 4, &k0, {k0.scalar_type()});
  const int64_t b = k0.size(0), hk = k0.size(1), s = k0.size(2), d = k0.size(3);
  if (v0.sizes() != k0.sizes()) {
    throw OpError(std::string(who) + ": k and v must share one shape, got " + shape_of(k0.sizes()) +
                  " and " + shape_of(v0.sizes()));
  }
  check_cache(who, k0, kp, vp, table, lengths, b, d);
  if (kp.size(1) != hk) {
    throw OpError(std::string(who) + ": the cache has " + std::to_string(kp.size(1)) + " key heads, k has " +
                  std::to_string(hk));
  }
  no_graph(who, {&k0, &v0, &q0, &kp, &vp});
  if (broadcast(kp) || broadcast(vp)) {
    throw OpError(std::string(who) + ": k_pages or v_pages is a broadcast view, whose slots share memory");
  }
  if (kp.numel() > 0 && kp.data_ptr() == vp.data_ptr()) {
    throw OpError(std::string(who) + ": k_pages and v_pages are the same memory");
  }
  Tensor q, out;
  int64_t heads = 0;
  if (q0.defined()) {
    require(who, "q", q0, 4, &k0, {k0.scalar_type()});
    if (q0.size(0) != b || q0.size(2) != s || q0.size(3) != d) {
      throw OpError(std::string(who) + ": q and k must agree but for their heads, got " +
                    shape_of(q0.sizes()) + " and " + shape_of(k0.sizes()));
    }
    q = rows(q0), out = like(q), heads = q.size(1);
  }
  if (counts.defined()) {
    require(who, "counts", counts, 1, &k0, {kI32});
    if (counts.size(0) != b || !counts.is_contiguous()) {
      throw OpError(std::string(who) + ": contiguous counts [" + std::to_string(b) + "] expected, got " +
                    shape_of(counts.sizes()));
    }
  }
  const int64_t dim = f.defined() ? check_frequencies(who, f, d, k0) : 0;
  const Tensor k = rows(k0), v = rows(v0);
  launch(k, [&](void* stream) {
    return fattn_paged_append(
        type_code(k), type_code(kp), b, heads, hk, s, d, address(q), heads ? q.strides().data() : nullptr,
        address(out), heads ? out.strides().data() : nullptr, k.data_ptr(), k.strides().data(), v.data_ptr(),
        v.strides().data(), kp.data_ptr(), kp.strides().data(), vp.data_ptr(), vp.strides().data(),
        kp.size(0), kp.size(2), ints(table), table.stride(0), table.size(1), ints(lengths), ints(counts),
        static_cast<const double*>(address(f)), dim, interleaved, magnitude, stream);
  });
  wrote(kp), wrote(vp);
  return out;
}

Tensor paged_attention(const Tensor& q0, const Tensor& kp, const Tensor& vp, const Tensor& table,
                       const Tensor& lengths, double scale) {
  const char* who = "paged_attention";
  no_tangents(who, {&q0, &kp, &vp});
  require(who, "q", q0, 4, nullptr, {kF32, kF16, kBF16});
  const int64_t b = q0.size(0), h = q0.size(1), d = q0.size(3);
  if (q0.size(2) != 1) {
    throw OpError(std::string(who) + ": q [b, h, 1, d] expected, got shape " + shape_of(q0.sizes()));
  }
  check_cache(who, q0, kp, vp, table, lengths, b, d);
  no_graph(who, {&q0, &kp, &vp});
  const Tensor q = aligned_rows(q0);
  Tensor out = at::empty(q.sizes(), q.options());
  const int64_t hk = kp.size(1), page = kp.size(2), width = table.size(1);
  const size_t bytes = fattn_paged_attention_workspace_bytes(b, h, hk, d, width * page);
  const Tensor ws = workspace(q, bytes);
  launch(q, [&](void* stream) {
    return fattn_paged_attention(type_code(q), type_code(kp), b, h, hk, d, q.data_ptr(), q.strides().data(),
                                 out.data_ptr(), kp.data_ptr(), kp.strides().data(), vp.data_ptr(),
                                 vp.strides().data(), kp.size(0), page, ints(table), table.stride(0), width,
                                 ints(lengths), static_cast<float>(scale), address(ws), bytes, stream);
  });
  return out;
}

// --- Cross attention -------------------------------------------------------------------------------

constexpr const char* kCross = "fused_cross_attention";
const float* f32(const Tensor& t) { return static_cast<const float*>(t.data_ptr()); }

void check_cross(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths) {
  require(kCross, "q", q, 4, nullptr, {kF32});
  require(kCross, "k", k, 4, &q, {kF32});
  require(kCross, "v", v, 4, &q, {kF32});
  const int64_t b = q.size(0);
  if (k.sizes() != v.sizes() || k.size(0) != b || k.size(3) != q.size(3)) {
    throw OpError(std::string(kCross) + ": q [b, h, sq, d] and k, v [b, kv_heads, sk, d] expected, got " +
                  shape_of(q.sizes()) + " " + shape_of(k.sizes()) + " " + shape_of(v.sizes()));
  }
  if (!lengths.defined()) return;
  require(kCross, "key_lengths", lengths, 1, &q, {kI32});
  if (lengths.size(0) != b || !lengths.is_contiguous()) {
    throw OpError(std::string(kCross) + ": contiguous key_lengths [" + std::to_string(b) +
                  "] expected, got " + shape_of(lengths.sizes()));
  }
}
// A [b, h, s, d] tensor itself where it lies over a contiguous [b, s, h, d] buffer, else a copy that does.
Tensor merged(const Tensor& t) {
  const int64_t h = t.size(1), s = t.size(2), d = t.size(3);
  const bool ok = t.stride(3) == 1 && (h <= 1 || t.stride(1) == d) && (s <= 1 || t.stride(2) == h * d) &&
                  (t.size(0) <= 1 || t.stride(0) == s * h * d);
  return ok ? t : t.transpose(1, 2).contiguous().transpose(1, 2);
}

// The output, [b, h, sq, d] over a contiguous [b, sq, h, d] buffer, and the [b, h, sq] log-sums.
Tensors cross_forward(const Tensor& q, const Tensor& k, const Tensor& v, double scale, const Tensor& lengths) {
  const int64_t b = q.size(0), h = q.size(1), sq = q.size(2), d = q.size(3), hk = k.size(1), sk = k.size(2);
  Tensor out = at::empty_strided({b, h, sq, d}, {sq * h * d, d, h * d, 1}, q.options());
  Tensor lse = at::empty({b, h, sq}, q.options());
  const size_t bytes = fattn_cross_workspace_bytes(b, h, hk, sq, sk, d);
  const Tensor ws = workspace(q, bytes);
  launch(q, [&](void* stream) {
    return fattn_cross_forward(f32(q), q.strides().data(), f32(k), k.strides().data(), f32(v),
                               v.strides().data(), b, h, hk, sq, sk, d, ints(lengths),
                               static_cast<float>(scale), static_cast<float*>(out.data_ptr()),
                               static_cast<float*>(lse.data_ptr()), address(ws), bytes, stream);
  });
  return {out, lse};
}

// dq over a contiguous [b, sq, h, d] buffer, dk and dv over one contiguous [b, sk, 2, kv_heads, d].
Tensors cross_backward(const Tensor& q, const Tensor& k, const Tensor& v, double scale, const Tensor& lengths,
                       const Tensor& out, const Tensor& lse, const Tensor& grad) {
  const int64_t b = q.size(0), h = q.size(1), sq = q.size(2), d = q.size(3), hk = k.size(1), sk = k.size(2);
  const Tensor g = aligned_rows(grad);
  Tensor dq = at::empty_strided({b, h, sq, d}, {sq * h * d, d, h * d, 1}, q.options());
  Tensor dkv = at::empty({b, sk, 2, hk, d}, q.options());
  const size_t bytes = fattn_cross_backward_workspace_bytes(b, h, hk, sq, sk, d);
  const Tensor ws = workspace(q, bytes);
  launch(q, [&](void* stream) {
    return fattn_cross_backward(f32(q), q.strides().data(), f32(k), k.strides().data(), f32(v),
                                v.strides().data(), b, h, hk, sq, sk, d, ints(lengths),
                                static_cast<float>(scale), f32(out), f32(lse), f32(g), g.strides().data(),
                                static_cast<float*>(dq.data_ptr()), static_cast<float*>(dkv.data_ptr()),
                                address(ws), bytes, stream);
  });
  return {dq, dkv.select(2, 0).transpose(1, 2), dkv.select(2, 1).transpose(1, 2)};
}

// Gradients that were asked for with a graph: they are not differentiable, and say so when it is tried
// (without this they would look like constants).
struct NotTwice : Function<NotTwice> {
  static Tensors forward(AutogradContext*, const Tensor& dq, const Tensor& dk, const Tensor& dv,
                         const Tensor&, const Tensor&, const Tensor&, const Tensor&) {
    return {dq.view_as(dq), dk.view_as(dk), dv.view_as(dv)};
  }
  static Tensors backward(AutogradContext*, const Tensors&) {
    return in_backward([]() -> Tensors {
      throw OpError(std::string(kCross) + ": its gradient is not differentiable");
    });
  }
};
struct How {
  double scale;
  Tensor lengths;  // (may be undefined: not among a node's tensors)
};
struct CrossNode : Function<CrossNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const How& how) {
    const Tensors out = cross_forward(q, k, v, how.scale, how.lengths);
    ctx->save_for_backward({q, k, v, how.lengths, out[0], out[1]});
    ctx->saved_data["scale"] = how.scale;
    return out[0];
  }
  static Tensors backward(AutogradContext* ctx, const Tensors& grads) {
    const Tensors s = ctx->get_saved_variables();
    return in_backward([&]() -> Tensors {
      no_tangents(kCross, {&grads[0]});
      // (Hooks on saved tensors may have replaced them: save_on_cpu brings them back in another layout.)
      check_cross(s[0], s[1], s[2], s[3]);
      require(kCross, "the saved output", s[4], 4, &s[0], {kF32});
      require(kCross, "the saved log-sums", s[5], 3, &s[0], {kF32});
      if (s[4].sizes() != s[0].sizes() || s[5].sizes() != s[0].sizes().slice(0, 3) ||
          grads[0].sizes() != s[0].sizes()) {
        throw OpError(std::string(kCross) + ": saved tensors came back in other shapes");
      }
      Tensors to;
      {
        const c10::AutoGradMode off(false);
        to = cross_backward(aligned_rows(s[0]), aligned_rows(s[1]), aligned_rows(s[2]),
                            ctx->saved_data["scale"].toDouble(), s[3], merged(s[4]), s[5].contiguous(), grads[0]);
      }
      if (c10::GradMode::is_enabled()) to = NotTwice::apply(to[0], to[1], to[2], s[0], s[1], s[2], grads[0]);
      to.resize(4);  // (none for `how`)
      return to;
    });
  }
};

Tensor fused_cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, double scale,
                              const Tensor& lengths) {
  no_tangents(kCross, {&q, &k, &v});
  check_cross(q, k, v, lengths);
  const Tensor qa = aligned_rows(q), ka = aligned_rows(k), va = aligned_rows(v);
  return records({&qa, &ka, &va}) ? CrossNode::apply(qa, ka, va, How{scale, lengths})
                                  : cross_forward(qa, ka, va, scale, lengths)[0];
}

// --- Python ----------------------------------------------------------------------------------------

// The positional arguments of a call, read in turn.
struct Args {
  const char* who;
  PyObject* const* at;
  Py_ssize_t left;

  PyObject* next() {
    if (left == 0) throw OpError(std::string(who) + ": too few arguments");
    --left;
    return *at++;
  }
  const Tensor& tensor(const char* name, PyObject* x) const {
    if (!THPVariable_Check(x)) throw OpError(std::string(who) + ": " + name + " must be a tensor");
    return THPVariable_Unpack(x);
  }
  const Tensor& tensor(const char* name) { return tensor(name, next()); }
  Tensor maybe(const char* name) {
    PyObject* x = next();
    return x == Py_None ? Tensor() : tensor(name, x);
  }
  bool truth() {
    const int x = PyObject_IsTrue(next());
    if (x < 0) throw python_error();
    return x == 1;
  }
  double number() {
    const double x = PyFloat_AsDouble(next());
    if (x == -1.0 && PyErr_Occurred()) throw python_error();
    return x;
  }
  int64_t integer() {
    const long long x = PyLong_AsLongLong(next());
    if (x == -1 && PyErr_Occurred()) throw python_error();
    return x;
  }
};

// Without the interpreter's lock while it lives, as every call of torch's is.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// (Undefined: None.)
PyObject* one(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
PyObject* all(const Tensors& ts) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!out) throw python_error();
  for (size_t i = 0; i < ts.size(); ++i) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(ts[i]));
  return out;
}

// body(args) with what it throws as Python's exceptions: OpError as FusedAttentionError, torch's errors
// as torch raises them.
template <typename F>
PyObject* entry(const char* who, PyObject* const* args, Py_ssize_t n, F body) {
  HANDLE_TH_ERRORS
  try {
    Args a{who, args, n};
    return body(a);
  } catch (const OpError& e) {
    set_python(e);
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("fused_rotary", args, n, [](Args& a) {
    const Tensor &q = a.tensor("q"), &k = a.tensor("k"), &p = a.tensor("positions"),
                 &f = a.tensor("frequencies");
    const bool interleaved = a.truth();
    const double magnitude = a.number();
    Tensors out;
    {
      const Unlocked unlocked;
      out = fused_rotary(q, k, p, f, interleaved, magnitude);
    }
    return all(out);
  });
}

PyObject* py_rotary_qkv(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("fused_rotary_qkv", args, n, [](Args& a) {
    const Tensor& x = a.tensor("qkv");
    const int64_t heads = a.integer();
    const Tensor &p = a.tensor("positions"), &f = a.tensor("frequencies");
    const bool interleaved = a.truth();
    const double magnitude = a.number();
    Tensor out;
    {
      const Unlocked unlocked;
      out = fused_rotary_qkv(x, heads, p, f, interleaved, magnitude);
    }
    return one(out);
  });
}

PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("paged_append", args, n, [](Args& a) {
    const Tensor &k = a.tensor("k"), &v = a.tensor("v"), &kp = a.tensor("k_pages"),
                 &vp = a.tensor("v_pages"), &table = a.tensor("page_table"), &lengths = a.tensor("lengths");
    const Tensor counts = a.maybe("counts"), q = a.maybe("q"), f = a.maybe("frequencies");
    const bool interleaved = a.truth();
    const double magnitude = a.number();
    Tensor out;
    {
      const Unlocked unlocked;
      out = paged_append(k, v, kp, vp, table, lengths, counts, q, f, interleaved, magnitude);
    }
    return one(out);
  });
}

PyObject* py_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("paged_attention", args, n, [](Args& a) {
    const Tensor &q = a.tensor("q"), &kp = a.tensor("k_pages"), &vp = a.tensor("v_pages"),
                 &table = a.tensor("page_table"), &lengths = a.tensor("lengths");
    const double scale = a.number();
    Tensor out;
    {
      const Unlocked unlocked;
      out = paged_attention(q, kp, vp, table, lengths, scale);
    }
    return one(out);
  });
}

PyObject* py_cross_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return entry("fused_cross_attention", args, n, [](Args& a) {
    const Tensor &q = a.tensor("q"), &k = a.tensor("k"), &v = a.tensor("v");
    const double scale = a.number();
    const Tensor lengths = a.maybe("key_lengths");
    Tensor out;
    {
      const Unlocked unlocked;
      out = fused_cross_attention(q, k, v, scale, lengths);
    }
    return one(out);
  });
}

PyMethodDef g_methods[] = {
#define ENTRY(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, ""}
    ENTRY("rotary", py_rotary),
    ENTRY("rotary_qkv", py_rotary_qkv),
    ENTRY("paged_append", py_append),
    ENTRY("paged_attention", py_paged_attention),
    ENTRY("cross_attention", py_cross_attention),
#undef ENTRY
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "torch_operators", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_torch_operators() {
  PyObject* package = PyImport_ImportModule("candle_fused_attn._lib");
  if (!package) return nullptr;
  g_error = PyObject_GetAttrString(package, "FusedAttentionError");
  Py_DECREF(package);
  return g_error ? PyModule_Create(&g_module) : nullptr;
}
