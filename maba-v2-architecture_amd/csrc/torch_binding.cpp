// The feed-forward operators as native autograd functions for torch: what the Python path does (maba_sparse/kernels/
// feed_forward.py over hip_backend.py), without Python in the call or in the autograd engine's thread.
//
// Bound by the host: a training step of 1,777 x 555 to 1,001, whose kernels take 74 us, takes 95 us here and took 177 by the
// Python path (an empty autograd function in Python: 78); a forward call 9 and 19.
//
// A call that is not plain (other dtypes or devices, shapes that do not fit, tensor subclasses, tangents of forward-mode
// derivatives, sizes that the library refuses) is declined: the function returns None and the caller takes the Python
// path, which checks, raises or falls back.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <cstdlib>
#include <strings.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "../../include/maba_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

#define MABA_ENTRIES(X)                                                                                                 \
  X(gated_ffn_workspace_size) X(gated_ffn) X(gated_ffn_backward_workspace_size) X(gated_ffn_backward)                   \
  X(linear_epilogue_workspace_size) X(linear_epilogue) X(linear_epilogue_backward_workspace_size)                       \
  X(linear_epilogue_backward) X(checkpoint_pack) X(checkpoint_unpack) X(last_error)

// The entry points of the library that the Python side has loaded.
#define X(name) decltype(&maba_hip_##name) name = nullptr;
struct Library { MABA_ENTRIES(X) };
#undef X
Library lib;

void bind(const std::map<std::string, uintptr_t>& address) {
#define X(name) lib.name = (decltype(lib.name))address.at(#name);
  MABA_ENTRIES(X)
#undef X
}

struct Declined {};
void take(int rc) {
  if (rc != MABA_OK) throw Declined();
}

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MABA_F32;
    case at::kHalf: return MABA_F16;
    case at::kBFloat16: return MABA_BF16;
    case at::kFloat8_e4m3fn: return MABA_E4M3;
    case at::kByte: return MABA_U8;
    default: throw Declined();
  }
}

// A tensor [..., C] as [rows, C] with unit column stride (a view where the strides allow it), or a vector.
struct Desc {
  Tensor keep;
  maba_tensor d = {};
  bool there = false;
  Desc() = default;
  explicit Desc(const Tensor& t, bool vector = false) {
    if (!t.defined()) return;
    keep = t;
    if (vector) {
      if (!keep.is_contiguous()) keep = keep.contiguous();
    } else {
      if (keep.dim() != 2) keep = keep.reshape({-1, keep.size(-1)});
      if (keep.size(1) != 1 && keep.stride(1) != 1) keep = keep.contiguous();
    }
    d.data = keep.data_ptr();
    d.dtype = code_of(keep);
    d.ndim = (int)keep.dim();
    for (int i = 0; i < 4; ++i) {
      d.shape[i] = i < d.ndim ? keep.size(i) : 1;
      d.stride[i] = i < d.ndim ? keep.stride(i) : 0;
    }
    there = true;
  }
  maba_tensor* operator&() { return there ? &d : nullptr; }
};

Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Everything below runs on the tensors' device, below autograd.
struct Scope {
  c10::DeviceGuard device;
  at::AutoDispatchBelowADInplaceOrView below;
  explicit Scope(const Tensor& t) : device(t.device()) {}
};

// Plain tensors of one 16-bit dtype on one GPU, without a tangent.
bool plain(const Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t._fw_grad(0).defined() &&
         !t.unsafeGetTensorImpl()->key_set().has_any(
             c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                  c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize}));
}
bool alike(const Tensor& first, std::initializer_list<const Tensor*> others) {
  if (!plain(first) || (first.scalar_type() != at::kHalf && first.scalar_type() != at::kBFloat16)) return false;
  for (const Tensor* t : others)
    if (t->defined() && (!plain(*t) || t->scalar_type() != first.scalar_type() || t->device() != first.device())) return false;
  return true;
}
bool needs_grad(std::initializer_list<const Tensor*> all) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : all)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
std::vector<int64_t> outer(const Tensor& x, int64_t last) {
  auto s = x.sizes().vec();
  s.back() = last;
  return s;
}
bool needs(const Tensor& t) { return t.defined() && t.requires_grad(); }

// ---------------------------------------------------------------- the calls

Tensor gated_call(const Tensor& x, const Tensor& wg, const Tensor& wu) {
  Scope scope(x);
  Desc dx(x), dg(wg), du(wu);
  Tensor out = at::empty(outer(x, wg.size(0)), x.options());
  Desc dout(out);
  void* s = stream_of(x);
  int rc = lib.gated_ffn(&dx, &dg, &du, &dout, nullptr, 0, s);
  if (rc == MABA_ERR_WORKSPACE) {
    Tensor ws = workspace(lib.gated_ffn_workspace_size(&dx, &dg, &du), x);
    rc = lib.gated_ffn(&dx, &dg, &du, &dout, ws.data_ptr(), ws.numel(), s);
  }
  take(rc);
  return out;
}

Tensor linear_call(const Tensor& x, const Tensor& w, const Tensor& bias, int act, const Tensor& res, const Tensor& gate) {
  Scope scope(x);
  Desc dx(x), dw(w), db(bias, true), dr(res), dg(gate, true);
  Tensor out = at::empty(outer(x, w.size(0)), x.options());
  Desc dout(out);
  void* s = stream_of(x);
  int rc = lib.linear_epilogue(&dx, &dw, &db, act, &dr, &dg, &dout, nullptr, 0, s);
  if (rc == MABA_ERR_WORKSPACE) {
    Tensor ws = workspace(lib.linear_epilogue_workspace_size(&dx, &dw), x);
    rc = lib.linear_epilogue(&dx, &dw, &db, act, &dr, &dg, &dout, ws.data_ptr(), ws.numel(), s);
  }
  take(rc);
  return out;
}

std::pair<Tensor, Tensor> pack_call(const Tensor& x) {
  Scope scope(x);
  Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  Tensor scales = at::empty(outer(x, (x.size(-1) + 31) / 32), x.options().dtype(at::kByte));
  Desc dx(x), dc(codes), ds(scales);
  take(lib.checkpoint_pack(&dx, &dc, &ds, stream_of(x)));
  return {codes, scales};
}

void check_backward(int rc, const char* who) {
  TORCH_CHECK(rc == MABA_OK, who, " failed (", rc, "): ", lib.last_error());
}

// What a backward pass returns where a second derivative may be asked for: gradients that raise in it.
void once(std::initializer_list<Tensor*> grads) {
  if (!at::GradMode::is_enabled()) return;
  variable_list live;
  for (Tensor* t : grads)
    if (t->defined()) {
      *t = t->detach();
      t->set_requires_grad(true);
      live.push_back(*t);
    }
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)live.size());
  live = (*error)(std::move(live));
  size_t i = 0;
  for (Tensor* t : grads)
    if (t->defined()) *t = live[i++];
}

struct GatedFFN : public torch::autograd::Function<GatedFFN> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, bool packed) {
    variable_list kept = {wg, wu};
    if (packed) {
      auto p = pack_call(x);
      kept.push_back(p.first);
      kept.push_back(p.second);
    } else {
      kept.push_back(x);
    }
    ctx->save_for_backward(kept);
    ctx->saved_data["needs"] = (int64_t)(needs(x) | needs(wg) << 1 | needs(wu) << 2);
    return gated_call(x, wg, wu);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto kept = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["needs"].toInt();
    const Tensor &dh = grads[0], &wg = kept[0], &wu = kept[1], &x = kept[2];
    Tensor dx, dwg, dwu;
    {
      Scope scope(wg);
      Desc ddh(dh), ddx_in(x), ds(kept.size() > 3 ? kept[3] : Tensor()), dg(wg), du(wu);
      if (need & 1) dx = at::empty(x.sizes(), wg.options());
      if (need & 2) dwg = at::empty(wg.sizes(), wg.options());
      if (need & 4) dwu = at::empty(wu.sizes(), wg.options());
      Desc odx(dx), odg(dwg), odu(dwu);
      Tensor ws = workspace(lib.gated_ffn_backward_workspace_size(&ddx_in, &ds, &dg, &du, (need & 1) | (need & 6 ? 2 : 0)), wg);
      check_backward(lib.gated_ffn_backward(&ddh, &ddx_in, &ds, &dg, &du, &odx, &odg, &odu, ws.data_ptr(), ws.numel(),
                                            stream_of(wg)), "gated_ffn_backward");
    }
    once({&dx, &dwg, &dwu});
    return {dx, dwg, dwu, Tensor()};
  }
};

struct LinearEpilogue : public torch::autograd::Function<LinearEpilogue> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& bias_, const Maybe& res_,
                        const Maybe& gate_, int64_t act, bool packed) {
    const Tensor bias = bias_.value_or(Tensor()), res = res_.value_or(Tensor()), gate = gate_.value_or(Tensor());
    const bool dx = needs(x), dw = needs(w), db = needs(bias), dg = needs(gate);
    // x is read by dW and dgate and, with an activation, to make z again
    const bool keeps_x = dw || dg || ((dx || db) && act != 0);
    if (dx || dw || db || dg) {
      variable_list kept = {w};
      if (bias.defined()) kept.push_back(bias);
      if (gate.defined()) kept.push_back(gate);
      if (keeps_x && packed) {
        auto p = pack_call(x);
        kept.push_back(p.first);
        kept.push_back(p.second);
      } else if (keeps_x) {
        kept.push_back(x);
      }
      ctx->save_for_backward(kept);
    }
    ctx->saved_data["flags"] = (int64_t)(dx | dw << 1 | db << 2 | dg << 3 | needs(res) << 4 | bias.defined() << 5 |
                                         gate.defined() << 6 | keeps_x << 7 | (keeps_x && packed) << 8 | act << 9);
    ctx->saved_data["shape"] = x.sizes().vec();
    return linear_call(x, w, bias, (int)act, res, gate);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const int64_t f = ctx->saved_data["flags"].toInt();
    const int need = (int)(f & 15), act = (int)(f >> 9);
    const Tensor& dy = grads[0];
    Tensor dx, dw, dbias, dgate, dres;
    if (f >> 4 & 1) dres = dy;
    if (need) {
      const auto kept = ctx->get_saved_variables();
      const auto shape = ctx->saved_data["shape"].toIntVector();
      size_t at_ = 0;
      const Tensor w = kept[at_++], bias = f >> 5 & 1 ? kept[at_++] : Tensor(), gate = f >> 6 & 1 ? kept[at_++] : Tensor();
      Scope scope(w);
      // where x is not read, a view of its shape over one weight row takes its place
      const Tensor x = f >> 7 & 1 ? kept[at_++] : w.select(0, 0).expand(shape);
      Desc ddy(dy), ix(x), is(f >> 8 & 1 ? kept[at_++] : Tensor()), iw(w), ib(bias, true), ig(gate, true);
      if (need & 1) dx = at::empty(shape, w.options());
      if (need & 2) dw = at::empty(w.sizes(), w.options());
      if (need & 4) dbias = at::empty({w.size(0)}, w.options());
      if (need & 8) dgate = at::empty({w.size(0)}, w.options());
      Desc odx(dx), odw(dw), odb(dbias, true), odg(dgate, true);
      Tensor ws = workspace(lib.linear_epilogue_backward_workspace_size(&ddy, &ix, &is, &iw, act, bias.defined(), gate.defined(),
                                                                        need), w);
      check_backward(lib.linear_epilogue_backward(&ddy, &ix, &is, &iw, &ib, act, &ig, &odx, &odw, &odb, &odg, ws.data_ptr(),
                                                  ws.numel(), stream_of(w)), "linear_epilogue_backward");
    }
    once({&dx, &dw, &dbias, &dgate});
    return {dx, dw, dbias, dres, dgate, Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------- the module's functions

// Whether the dispatcher's backend for GPU tensors is this library: MABA_BACKEND as its get_backend reads it, without the
// 1.3 us that takes in Python.  Any other value is declined, and the Python path routes or refuses it.  Called with the
// interpreter's lock held: a write to os.environ in another thread holds it too.
bool routed_here() {
  const char* e = std::getenv("MABA_BACKEND");
  if (!e || !*e) return true;
  for (const char* name : {"auto", "hip", "triton", "cuda", "gpu"})
    if (!strcasecmp(e, name)) return true;
  return false;
}

Maybe gated_ffn(const Tensor& x, const Tensor& wg, const Tensor& wu, bool packed) {
  if (!alike(x, {&wg, &wu}) || x.dim() < 1 || wg.dim() != 2 || wg.size(0) == 0 || x.size(-1) == 0 || wg.size(1) != x.size(-1) ||
      wu.sizes() != wg.sizes())
    return std::nullopt;
  try {
    if (needs_grad({&x, &wg, &wu})) return GatedFFN::apply(x, wg, wu, packed);
    return gated_call(x, wg, wu);
  } catch (const Declined&) {
    return std::nullopt;
  }
}

Maybe linear_epilogue(const Tensor& x, const Tensor& w, const Maybe& bias_, int64_t act, const Maybe& res_, const Maybe& gate_,
                      bool packed) {
  const Tensor bias = bias_.value_or(Tensor()), res = res_.value_or(Tensor()), gate = gate_.value_or(Tensor());
  if (!alike(x, {&w, &bias, &res, &gate}) || x.dim() < 1 || w.dim() != 2 || w.size(0) == 0 || x.size(-1) == 0 ||
      w.size(1) != x.size(-1))
    return std::nullopt;
  for (const Tensor* v : {&bias, &gate})
    if (v->defined() && (v->dim() != 1 || v->size(0) != w.size(0))) return std::nullopt;
  if (res.defined() && res.sizes() != at::IntArrayRef(outer(x, w.size(0)))) return std::nullopt;
  try {
    if (needs_grad({&x, &w, &bias, &res, &gate})) return LinearEpilogue::apply(x, w, bias_, res_, gate_, act, packed);
    return linear_call(x, w, bias, (int)act, res, gate);
  } catch (const Declined&) {
    return std::nullopt;
  }
}

std::optional<std::pair<Tensor, Tensor>> checkpoint_pack(const Tensor& x) {
  if (!plain(x) || x.dim() < 1 || x.size(-1) == 0) return std::nullopt;
  try {
    return pack_call(x.requires_grad() ? x.detach() : x);
  } catch (const Declined&) {
    return std::nullopt;
  }
}

Maybe checkpoint_unpack(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
  if (!plain(codes) || !plain(scales) || codes.device() != scales.device() || codes.dim() < 1 || codes.size(-1) == 0 ||
      codes.scalar_type() != at::kFloat8_e4m3fn || scales.scalar_type() != at::kByte ||
      scales.sizes() != at::IntArrayRef(outer(codes, (codes.size(-1) + 31) / 32)))
    return std::nullopt;
  try {
    Scope scope(codes);
    Tensor out = at::empty(codes.sizes(), codes.options().dtype(dtype));
    Desc dc(codes), ds(scales), dout(out);
    take(lib.checkpoint_unpack(&dc, &ds, &dout, stream_of(codes)));
    return out;
  } catch (const Declined&) {
    return std::nullopt;
  }
}

// Whether a leaf that `out` was made from, by itself or cast to another type, keeps its autograd node from another stream
// than the current one: the stream that was current when the eager graph it belongs to was made, by whatever op.
bool leaf_of_another_stream(const Tensor& out) {
  const auto fn = out.grad_fn();
  if (!fn) return false;
  const auto now = c10::hip::getCurrentHIPStream(out.device().index());
  for (const auto& edge : fn->next_edges()) {
    torch::autograd::Node* node = edge.function.get();
    while (node && node->num_outputs() > 0 && node->name() == "ToCopyBackward0") node = node->next_edge(0).function.get();
    if (!dynamic_cast<torch::autograd::AccumulateGrad*>(node)) continue;
    const auto made = node->stream();
    if (made && (made->id() != now.id() || made->device_index() != now.device_index())) return true;
  }
  return false;
}

// `f` without the interpreter's lock, where the backend is this library.
template <class R, class... A>
auto unlocked(R (*f)(A...)) {
  return [f](A... a) -> R {
    if (!routed_here()) return std::nullopt;
    py::gil_scoped_release free;
    return f(a...);
  };
}

}  // namespace

PYBIND11_MODULE(maba_torch, m) {
  m.def("bind", &bind);
  m.def("leaf_of_another_stream", &leaf_of_another_stream);
  m.def("gated_ffn", unlocked(&gated_ffn));
  m.def("linear_epilogue", unlocked(&linear_epilogue));
  m.def("checkpoint_pack", unlocked(&checkpoint_pack));
  m.def("checkpoint_unpack", unlocked(&checkpoint_unpack));
}
