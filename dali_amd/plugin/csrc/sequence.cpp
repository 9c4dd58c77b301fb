// dali_amd.sequence for PyTorch: argument checks, outputs and automatic differentiation around the C entries of
// libdali_amd_kernels.so (include/dali_amd_kernels.h).  In C++ because the same in Python takes longer than most of the kernels:
// 80 to 150 us of the host's time for a forward and a backward pass.
//
// The kernel library is not linked but bound at run time (bind()), so that the module has no HIP runtime of its own choosing.
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <optional>
#include "dali_amd_kernels.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

// ---- the kernel library --------------------------------------------------------------------------------------------------
struct Library {
#define DALIAMD_ENTRY(name) decltype(&daliamd##name) name = nullptr;
  DALIAMD_ENTRY(GetLastErrorMessage)
  DALIAMD_ENTRY(RecurrenceSetup) DALIAMD_ENTRY(RecurrenceRun) DALIAMD_ENTRY(RecurrenceBackwardRun)
  DALIAMD_ENTRY(BlockNormSetup) DALIAMD_ENTRY(BlockNormRun) DALIAMD_ENTRY(BlockNormBackwardRun)
  DALIAMD_ENTRY(EmbeddingSetup) DALIAMD_ENTRY(EmbeddingRun) DALIAMD_ENTRY(EmbeddingBackwardRun)
#undef DALIAMD_ENTRY
};
Library lib;
bool host_memory = false;   // the library is a model of the kernels on the CPU: tensors are in host memory
py::object *error_class = nullptr;

struct KernelError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void Bind(const std::string &path, py::object error, bool host) {
  void *h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  if (!h) throw std::runtime_error(dlerror());
#define DALIAMD_ENTRY(name)                                                                            \
  lib.name = reinterpret_cast<decltype(lib.name)>(dlsym(h, "daliamd" #name));                          \
  if (!lib.name) throw std::runtime_error("daliamd" #name " is missing in " + path);
  DALIAMD_ENTRY(GetLastErrorMessage)
  DALIAMD_ENTRY(RecurrenceSetup) DALIAMD_ENTRY(RecurrenceRun) DALIAMD_ENTRY(RecurrenceBackwardRun)
  DALIAMD_ENTRY(BlockNormSetup) DALIAMD_ENTRY(BlockNormRun) DALIAMD_ENTRY(BlockNormBackwardRun)
  DALIAMD_ENTRY(EmbeddingSetup) DALIAMD_ENTRY(EmbeddingRun) DALIAMD_ENTRY(EmbeddingBackwardRun)
#undef DALIAMD_ENTRY
  host_memory = host;
  if (!error_class) error_class = new py::object(error);
}

void Check(daliamdResult_t r) {
  if (r != DALIAMD_SUCCESS)
    throw KernelError("[dali_amd kernels error " + std::to_string((int)r) + "] " + lib.GetLastErrorMessage());
}

// the device of a call and its current stream
struct OnDevice {
  c10::OptionalDeviceGuard guard;
  daliamdStream_t stream = nullptr;
  explicit OnDevice(const Tensor &t) {
    if (host_memory) return;
    guard.reset_device(t.device());
    stream = c10::hip::getCurrentHIPStream(t.device().index()).stream();
  }
};

// ---- checks --------------------------------------------------------------------------------------------------------------
std::string Shape(c10::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}
const char *TypeName(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "float32";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    case at::kInt: return "int32";
    case at::kLong: return "int64";
    default: return c10::toString(t);
  }
}
bool IsValueType(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }
int DType(at::ScalarType t) {
  return t == at::kFloat ? DALIAMD_FLOAT : t == at::kHalf ? DALIAMD_FLOAT16 : t == at::kBFloat16 ? DALIAMD_BFLOAT16 : t == at::kInt ? DALIAMD_INT32 : DALIAMD_INT64;
}
void CheckValues(const char *name, const Tensor &t) {
  TORCH_CHECK_TYPE(IsValueType(t.scalar_type()), name, " must be float32 or float16 or bfloat16, got ", TypeName(t.scalar_type()));
}
// x's type or float32
void CheckWide(const char *name, const Tensor &t, at::ScalarType x) {
  TORCH_CHECK_TYPE(t.scalar_type() == x || t.scalar_type() == at::kFloat, name, " must be ", x == at::kFloat ? "" : TypeName(x),
                   x == at::kFloat ? "" : " or ", "float32, got ", TypeName(t.scalar_type()));
}
void CheckIndex(const char *name, const Tensor &t) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64, got ", TypeName(t.scalar_type()));
}
void CheckShape(const char *name, const Tensor &t, c10::IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have the shape ", Shape(shape), ", got ", Shape(t.sizes()));
}
void CheckDevice(const char *name, const Tensor &t, const Tensor &x) {
  TORCH_CHECK_VALUE(t.is_cuda() || host_memory, name, " must be on the GPU: the sequence operators have no CPU fallback");
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", the other tensors on ", x.device());
}
void CheckDevice(const char *name, const Maybe &t, const Tensor &x) {
  if (t) CheckDevice(name, *t, x);
}
// What looks at a call through torch's operators sees the outputs' allocation and not the kernels that write them: a trace would
// hold the former alone, a tangent would be lost.
void CheckNotTraced(const char *what) {
  const bool traced = torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
                      (c10::impl::TorchDispatchModeTLS::any_modes_set() &&
                       c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
  TORCH_CHECK(!traced, what, " cannot be traced: its kernels are not torch operators");
}
void CheckNoTangent(const char *what, const Tensor &t) {
  // (without autograd's data, which a tensor has that requires a gradient or has a tangent, there is none)
  TORCH_CHECK(!t.defined() || !t.unsafeGetTensorImpl()->autograd_meta() || !t._fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}
void CheckNoTangent(const char *what, const Maybe &t) {
  if (t) CheckNoTangent(what, *t);
}
template <typename... T> void CheckSeen(const char *what, const T &...inputs) {
  CheckNotTraced(what);
  (CheckNoTangent(what, inputs), ...);
}

// ---- plumbing ------------------------------------------------------------------------------------------------------------
void *Ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *FloatPtr(const Tensor &t) { return static_cast<float *>(Ptr(t)); }
Tensor Get(const Maybe &t) { return t ? *t : Tensor(); }
// t with its values in memory: a view that is negated in name only (of a conjugate's imaginary part) is copied
Tensor Dense(const Tensor &t) { return t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous(); }
// t with adjacent channels: itself if its last dimension is dense, else a copy
Tensor Rows(const Tensor &t) { return !t.is_neg() && (t.stride(-1) == 1 || t.size(-1) == 1) ? t : Dense(t); }
// t as [rows, channels]: in place where all leading dimensions are one, else a copy
Tensor Flat(const Tensor &t) {
  const Tensor r = Rows(t);
  return r.dim() == 2 ? r : r.reshape({t.numel() / t.size(-1), t.size(-1)});
}
Tensor Workspace(size_t bytes, const Tensor &like) { return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor(); }
Tensor EmptyLike(const Tensor &t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }
bool Tracked(std::initializer_list<Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor &t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
Maybe AsMaybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }
// Gradients that cannot be differentiated again: asked for with create_graph, they say so if that is tried.  They depend on
// `inputs` and on the gradients of the outputs, so that a second differentiation with respect to any of these finds the error.
variable_list Once(variable_list grads, const variable_list &inputs, const variable_list &outputs, const char *what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list all;
  for (const Tensor &g : grads)
    if (g.defined()) all.push_back(g.detach().requires_grad_(true));
  for (const variable_list *list : {&inputs, &outputs})
    for (const Tensor &t : *list)
      if (t.defined() && t.requires_grad()) all.push_back(t);
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " cannot be differentiated twice", (int64_t)all.size());
  all = (*error)(std::move(all));
  size_t k = 0;
  for (Tensor &g : grads)
    if (g.defined()) g = all[k++];
  return grads;
}

// ---- linear recurrence ---------------------------------------------------------------------------------------------------
daliamdRecurrenceArgs RecurrenceArgs(const Tensor &x, const Tensor &decay, const Tensor &initial, const Tensor &offsets, const Tensor &lengths, int64_t form) {
  daliamdRecurrenceArgs a = {};
  a.channels = (int32_t)x.size(-1);
  a.dtype = DType(x.scalar_type());
  a.decay_dtype = DType(decay.scalar_type());
  a.form = (int32_t)form;
  a.per_channel = decay.dim() == 1;
  if (offsets.defined()) {
    a.seq.offsets = offsets.data_ptr();
    a.seq.index_dtype = DType(offsets.scalar_type());
    a.seq.rows = x.size(0);
    a.seq.sequences = (int32_t)(offsets.size(0) - 1);
    a.x_row = x.stride(0);
    if (!a.per_channel) a.decay_row = decay.stride(0);
  } else {
    a.seq.sequences = (int32_t)x.size(0);
    a.seq.steps = x.size(1);
    a.seq.rows = x.size(0) * x.size(1);
    a.x_seq = x.stride(0), a.x_row = x.stride(1);
    if (!a.per_channel) a.decay_seq = decay.stride(0), a.decay_row = decay.stride(1);
    if (lengths.defined()) {
      a.seq.lengths = lengths.data_ptr();
      a.seq.index_dtype = DType(lengths.scalar_type());
    }
  }
  a.x = Ptr(x);
  a.decay = Ptr(decay);
  a.initial = FloatPtr(initial);
  return a;
}

// y, state, saved
std::tuple<Tensor, Tensor, Tensor> RecurrenceForward(const Tensor &x, const Tensor &decay, const Tensor &initial, const Tensor &offsets, const Tensor &lengths,
                                                     int64_t form, Tensor state, bool save) {
  OnDevice on(x);
  daliamdRecurrenceArgs a = RecurrenceArgs(x, decay, initial, offsets, lengths, form);
  const auto floats = x.options().dtype(at::kFloat);
  if (!state.defined()) state = at::empty({a.seq.sequences, a.channels}, floats);
  a.final_state = FloatPtr(state);
  daliamdRecurrencePlan plan;
  Check(lib.RecurrenceSetup(&a, &plan));
  Tensor y = at::empty(x.sizes(), x.options()), saved;
  if (save) saved = at::empty({(int64_t)(plan.saved_bytes / sizeof(float))}, floats);
  a.y = Ptr(y);
  a.saved = FloatPtr(saved);
  const Tensor ws = Workspace(plan.forward_workspace_bytes, x);
  Check(lib.RecurrenceRun(on.stream, &a, Ptr(ws), plan.forward_workspace_bytes));
  return {y, state, saved};
}

struct RecurrenceFunction : torch::autograd::Function<RecurrenceFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &decay, const Maybe &initial, const Maybe &offsets, const Maybe &lengths,
                               int64_t form) {
    auto [y, state, saved] = RecurrenceForward(x, decay, Get(initial), Get(offsets), Get(lengths), form, Tensor(), true);
    ctx->save_for_backward({x, decay, Get(initial), Get(offsets), Get(lengths), saved});
    ctx->saved_data["form"] = form;
    ctx->set_materialize_grads(false);
    return {y, state};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    const Tensor &x = v[0], &decay = v[1], &initial = v[2], &offsets = v[3], &lengths = v[4], &saved = v[5];
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(6);
    CheckSeen("linear_recurrence", grads[0], grads[1]);
    at::AutoDispatchBelowADInplaceOrView below;
    OnDevice on(x);
    daliamdRecurrenceArgs a = RecurrenceArgs(x, decay, initial, offsets, lengths, ctx->saved_data["form"].toInt());
    daliamdRecurrencePlan plan;
    Check(lib.RecurrenceSetup(&a, &plan));
    Tensor dx = EmptyLike(x), ddecay = EmptyLike(decay), dinitial = EmptyLike(initial), dy, dstate;
    if (grads[0].defined()) {
      dy = Rows(grads[0]);
      a.dy = Ptr(dy);
      if (offsets.defined()) a.dy_row = dy.stride(0);
      else a.dy_seq = dy.stride(0), a.dy_row = dy.stride(1);
    }
    if (grads[1].defined()) {
      dstate = Dense(grads[1]);
      a.dfinal = FloatPtr(dstate);
    }
    a.saved = FloatPtr(saved);
    a.dx = Ptr(dx);
    a.ddecay = Ptr(ddecay);
    a.dinitial = FloatPtr(dinitial);
    const Tensor ws = Workspace(plan.backward_workspace_bytes, x);
    Check(lib.RecurrenceBackwardRun(on.stream, &a, Ptr(ws), plan.backward_workspace_bytes));
    return Once({dx, ddecay, dinitial, Tensor(), Tensor(), Tensor()}, {x, decay, initial}, grads, "linear_recurrence");
  }
};

std::tuple<Tensor, Tensor> Recurrence(const Tensor &x0, const Tensor &decay0, const std::string &form_name, const Maybe &initial_state, const Maybe &offsets,
                                      const Maybe &lengths, const Maybe &final_state) {
  CheckSeen("linear_recurrence", x0, decay0, initial_state);
  TORCH_CHECK_VALUE(form_name == "decay" || form_name == "gate", "form must be \"decay\" or \"gate\", got \"", form_name, "\"");
  const int64_t form = form_name == "gate" ? DALIAMD_RECURRENCE_GATE : DALIAMD_RECURRENCE_DECAY;
  CheckValues("x", x0);
  int64_t sequences;
  if (offsets) {
    TORCH_CHECK_VALUE(!lengths, "offsets and lengths exclude each other");
    CheckIndex("offsets", *offsets);
    TORCH_CHECK_VALUE(offsets->dim() == 1 && offsets->size(0) >= 1, "offsets must be [sequences + 1], got the shape ", Shape(offsets->sizes()));
    TORCH_CHECK_VALUE(x0.dim() == 2, "x must be [rows, channels] with offsets, got the shape ", Shape(x0.sizes()));
    sequences = offsets->size(0) - 1;
    TORCH_CHECK_VALUE(sequences > 0 || x0.size(0) == 0, "offsets name no sequence but x has rows");
  } else {
    TORCH_CHECK_VALUE(x0.dim() == 3, "x must be [batch, steps, channels] (or [rows, channels] with offsets), got the shape ", Shape(x0.sizes()));
    sequences = x0.size(0);
    if (lengths) {
      CheckIndex("lengths", *lengths);
      CheckShape("lengths", *lengths, {sequences});
    }
  }
  const int64_t channels = x0.size(-1);
  TORCH_CHECK_VALUE(channels >= 1 && channels <= DALIAMD_RECURRENCE_MAX_CHANNELS && x0.numel() / channels <= DALIAMD_SEQUENCE_MAX_ROWS &&
                        sequences <= DALIAMD_SEQUENCE_MAX_ROWS,
                    "x must have between 1 and ", (int)DALIAMD_RECURRENCE_MAX_CHANNELS, " channels and at most ", (int)DALIAMD_SEQUENCE_MAX_ROWS,
                    " rows, got the shape ", Shape(x0.sizes()));
  CheckWide("decay", decay0, x0.scalar_type());
  TORCH_CHECK_VALUE((decay0.dim() == 1 && decay0.size(0) == channels) || decay0.sizes() == x0.sizes(), "decay must have x's shape ", Shape(x0.sizes()), " or [",
                    channels, "], got ", Shape(decay0.sizes()));
  for (const auto &[name, t] : {std::pair<const char *, const Maybe &>("initial_state", initial_state), {"final_state", final_state}}) {
    if (!t) continue;
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, name, " must be float32, got ", TypeName(t->scalar_type()));
    CheckShape(name, *t, {sequences, channels});
  }
  TORCH_CHECK_VALUE(!final_state || (final_state->is_contiguous() && !final_state->is_neg()), "final_state must be contiguous, and no view that is negated in name only");
  const bool tracked = Tracked({x0, decay0, Get(initial_state)});
  TORCH_CHECK_VALUE(!(tracked && final_state), "final_state cannot be given while gradients are recorded");
  CheckDevice("x", x0, x0);
  CheckDevice("decay", decay0, x0);
  CheckDevice("initial_state", initial_state, x0);
  CheckDevice("offsets", offsets, x0);
  CheckDevice("lengths", lengths, x0);
  CheckDevice("final_state", final_state, x0);
  const Tensor x = Rows(x0), decay = Rows(decay0), initial = initial_state ? Dense(*initial_state) : Tensor();
  const Tensor off = offsets ? Dense(*offsets) : Tensor(), len = lengths ? Dense(*lengths) : Tensor();
  if (tracked) {
    const variable_list out = RecurrenceFunction::apply(x, decay, AsMaybe(initial), AsMaybe(off), AsMaybe(len), form);
    return {out[0], out[1]};
  }
  auto [y, state, saved] = RecurrenceForward(x, decay, initial, off, len, form, Get(final_state), false);
  // written in place: a backward pass that saved the tensor has to notice
  if (final_state && !final_state->is_inference()) final_state->unsafeGetTensorImpl()->bump_version();
  return {y, state};
}

// ---- norms around a block ------------------------------------------------------------------------------------------------
struct NormTensors {
  Tensor x, gate, residual, post, scale, pre;
};
daliamdBlockNormArgs BlockNormArgs(const NormTensors &t, double eps) {
  daliamdBlockNormArgs a = {};
  a.rows = t.x.size(0);
  a.channels = (int32_t)t.x.size(1);
  a.eps = (float)eps;
  a.dtype = DType(t.x.scalar_type());
  a.residual_dtype = t.residual.defined() ? DType(t.residual.scalar_type()) : a.dtype;
  const Tensor &w = t.post.defined() ? t.post : t.scale.defined() ? t.scale : t.pre;
  a.weight_dtype = w.defined() ? DType(w.scalar_type()) : a.dtype;
  a.x = Ptr(t.x), a.x_row = t.x.stride(0);
  if (t.gate.defined()) a.gate = Ptr(t.gate), a.gate_row = t.gate.stride(0);
  if (t.residual.defined()) a.residual = Ptr(t.residual), a.residual_row = t.residual.stride(0);
  a.post_weight = Ptr(t.post), a.scale = Ptr(t.scale), a.pre_weight = Ptr(t.pre);
  return a;
}
// hidden, normed, rstd of both norms
std::tuple<Tensor, Tensor, Tensor> BlockNormForward(const NormTensors &t, double eps, bool save) {
  OnDevice on(t.x);
  daliamdBlockNormArgs a = BlockNormArgs(t, eps);
  Tensor hidden = at::empty(t.x.sizes(), t.residual.defined() ? t.residual.options() : t.x.options()), normed, rstd;
  if (t.pre.defined()) normed = at::empty(t.x.sizes(), t.x.options());
  if (save) rstd = at::empty({2, a.rows}, t.x.options().dtype(at::kFloat));
  a.hidden = Ptr(hidden), a.normed = Ptr(normed);
  if (save) a.rstd_post = FloatPtr(rstd), a.rstd_pre = FloatPtr(rstd) + a.rows;
  Check(lib.BlockNormRun(on.stream, &a));
  return {hidden, normed, rstd};
}

struct BlockNormFunction : torch::autograd::Function<BlockNormFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Maybe &gate, const Maybe &residual, const Maybe &post, const Maybe &scale,
                               const Maybe &pre, double eps) {
    const NormTensors t = {x, Get(gate), Get(residual), Get(post), Get(scale), Get(pre)};
    auto [hidden, normed, rstd] = BlockNormForward(t, eps, true);
    ctx->save_for_backward({t.x, t.gate, t.residual, t.post, t.scale, t.pre, rstd});
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    if (!normed.defined()) return {hidden};
    return {hidden, normed};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    const NormTensors t = {v[0], v[1], v[2], v[3], v[4], v[5]};
    const Tensor &rstd = v[6];
    if (!grads[0].defined() && !(grads.size() > 1 && grads[1].defined())) return variable_list(7);
    CheckSeen("block_norm", grads[0], grads.size() > 1 ? grads[1] : Tensor());
    at::AutoDispatchBelowADInplaceOrView below;
    OnDevice on(t.x);
    daliamdBlockNormArgs a = BlockNormArgs(t, ctx->saved_data["eps"].toDouble());
    daliamdBlockNormPlan plan;
    Check(lib.BlockNormSetup(&a, &plan));
    a.rstd_post = FloatPtr(rstd), a.rstd_pre = FloatPtr(rstd) + a.rows;
    Tensor dh, dn;
    if (grads[0].defined()) {
      dh = Rows(grads[0]);
      a.dhidden = Ptr(dh), a.dhidden_row = dh.stride(0);
    }
    if (grads.size() > 1 && grads[1].defined()) {
      dn = Rows(grads[1]);
      a.dnormed = Ptr(dn), a.dnormed_row = dn.stride(0);
    }
    Tensor dx = EmptyLike(t.x), dgate = EmptyLike(t.gate), dresidual = EmptyLike(t.residual);
    Tensor dpost = EmptyLike(t.post), dscale = EmptyLike(t.scale), dpre = EmptyLike(t.pre);
    a.dx = Ptr(dx), a.dgate = Ptr(dgate), a.dresidual = Ptr(dresidual);
    a.dpost_weight = Ptr(dpost), a.dscale = Ptr(dscale), a.dpre_weight = Ptr(dpre);
    const Tensor ws = Workspace(plan.backward_workspace_bytes, t.x);
    Check(lib.BlockNormBackwardRun(on.stream, &a, Ptr(ws), plan.backward_workspace_bytes));
    return Once({dx, dgate, dresidual, dpost, dscale, dpre, Tensor()}, {t.x, t.gate, t.residual, t.post, t.scale, t.pre}, grads, "block_norm");
  }
};

std::tuple<Tensor, Maybe> BlockNorm(const Tensor &x, const Maybe &gate, const Maybe &residual, const Maybe &post, const Maybe &scale, const Maybe &pre, double eps) {
  CheckSeen("block_norm", x, gate, residual, post, scale, pre);
  CheckValues("x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must be [..., channels]");
  const int64_t channels = x.size(-1);
  TORCH_CHECK_VALUE(channels >= 1 && channels <= DALIAMD_BLOCK_NORM_MAX_CHANNELS, "x must have between 1 and ", (int)DALIAMD_BLOCK_NORM_MAX_CHANNELS,
                    " channels, got ", channels);
  TORCH_CHECK_VALUE(x.numel() / channels <= DALIAMD_SEQUENCE_MAX_ROWS, "x must have at most ", (int)DALIAMD_SEQUENCE_MAX_ROWS, " rows");
  if (gate) {
    TORCH_CHECK_TYPE(gate->scalar_type() == x.scalar_type(), "gate must be ", TypeName(x.scalar_type()), ", got ", TypeName(gate->scalar_type()));
    CheckShape("gate", *gate, x.sizes());
  }
  if (residual) {
    CheckWide("residual", *residual, x.scalar_type());
    CheckShape("residual", *residual, x.sizes());
  }
  const Tensor *first = nullptr;
  for (const auto &[name, w] : {std::pair<const char *, const Maybe &>("post_weight", post), {"scale", scale}, {"pre_weight", pre}}) {
    if (!w) continue;
    CheckWide(name, *w, x.scalar_type());
    CheckShape(name, *w, {channels});
    if (!first) first = &*w;
    TORCH_CHECK_TYPE(w->scalar_type() == first->scalar_type(), "the weights must have one type: one is ", TypeName(first->scalar_type()), ", ", name, " is ",
                     TypeName(w->scalar_type()));
  }
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
  CheckDevice("x", x, x);
  CheckDevice("gate", gate, x);
  CheckDevice("residual", residual, x);
  CheckDevice("post_weight", post, x);
  CheckDevice("scale", scale, x);
  CheckDevice("pre_weight", pre, x);
  NormTensors t = {Flat(x), gate ? Flat(*gate) : Tensor(), residual ? Flat(*residual) : Tensor(), post ? Dense(*post) : Tensor(),
                   scale ? Dense(*scale) : Tensor(), pre ? Dense(*pre) : Tensor()};
  Tensor hidden, normed;
  if (Tracked({t.x, t.gate, t.residual, t.post, t.scale, t.pre})) {
    const variable_list out =
        BlockNormFunction::apply(t.x, AsMaybe(t.gate), AsMaybe(t.residual), AsMaybe(t.post), AsMaybe(t.scale), AsMaybe(t.pre), eps);
    hidden = out[0];
    if (out.size() > 1) normed = out[1];
  } else {
    std::tie(hidden, normed, std::ignore) = BlockNormForward(t, eps, false);
  }
  if (x.dim() != 2) {
    hidden = hidden.view(x.sizes());
    if (normed.defined()) normed = normed.view(x.sizes());
  }
  return {hidden, AsMaybe(normed)};
}

// ---- embedding lookup ----------------------------------------------------------------------------------------------------
daliamdEmbeddingArgs EmbeddingArgs(const Tensor &ids, c10::IntArrayRef table, at::ScalarType dtype, double scale, int64_t padding, at::ScalarType out) {
  daliamdEmbeddingArgs a = {};
  a.ids = Ptr(ids), a.index_dtype = DType(ids.scalar_type()), a.tokens = ids.numel();
  a.vocab = table[0], a.channels = (int32_t)table[1];
  a.dtype = DType(dtype), a.out_dtype = DType(out);
  a.padding = padding, a.scale = (float)scale;
  return a;
}
Tensor EmbeddingForward(const Tensor &ids, const Tensor &table, double scale, int64_t padding, at::ScalarType type) {
  OnDevice on(table);
  daliamdEmbeddingArgs a = EmbeddingArgs(ids, table.sizes(), table.scalar_type(), scale, padding, type);
  a.table = Ptr(table), a.table_row = table.stride(0);
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(table.size(1));
  Tensor out = at::empty(shape, table.options().dtype(type));
  a.out = Ptr(out);
  Check(lib.EmbeddingRun(on.stream, &a));
  return out;
}

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &table, const Tensor &ids, double scale, int64_t padding, at::ScalarType type) {
    // The gradient takes the table's size and type, not its values, which may change before the backward pass.
    ctx->save_for_backward({ids});
    ctx->saved_data["table"] = table;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["type"] = (int64_t)type;
    return EmbeddingForward(ids, table, scale, padding, type);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const Tensor ids = ctx->get_saved_variables()[0], table = ctx->saved_data["table"].toTensor();
    CheckSeen("embedding_lookup", grads[0]);
    at::AutoDispatchBelowADInplaceOrView below;
    OnDevice on(ids);
    const Tensor dout = Flat(grads[0]);
    const std::array<int64_t, 2> sizes = {table.size(0), dout.size(1)};
    daliamdEmbeddingArgs a = EmbeddingArgs(ids, sizes, table.scalar_type(), ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(),
                                           (at::ScalarType)ctx->saved_data["type"].toInt());
    daliamdEmbeddingPlan plan;
    Check(lib.EmbeddingSetup(&a, &plan));
    Tensor dtable = at::empty(sizes, ids.options().dtype(table.scalar_type()));
    a.dout = Ptr(dout), a.dout_row = dout.stride(0), a.dtable = Ptr(dtable);
    const Tensor ws = Workspace(plan.backward_workspace_bytes, ids);
    Check(lib.EmbeddingBackwardRun(on.stream, &a, Ptr(ws), plan.backward_workspace_bytes));
    return Once({dtable, Tensor(), Tensor(), Tensor(), Tensor()}, {table}, grads, "embedding_lookup");
  }
};

Tensor Embedding(const Tensor &ids0, const Tensor &table0, double scale, std::optional<int64_t> padding_idx, std::optional<at::ScalarType> dtype) {
  CheckSeen("embedding_lookup", table0);
  CheckValues("table", table0);
  TORCH_CHECK_VALUE(table0.dim() == 2 && table0.size(0) >= 1 && table0.size(1) >= 1 && table0.size(0) < ((int64_t)1 << 31) && table0.size(1) <= (1 << 24),
                    "table must be [vocab, channels], got the shape ", Shape(table0.sizes()));
  CheckIndex("ids", ids0);
  TORCH_CHECK_VALUE(ids0.numel() < ((int64_t)1 << 31), "ids must be fewer than 2^31");
  const at::ScalarType type = dtype ? *dtype : table0.scalar_type();
  TORCH_CHECK_TYPE(IsValueType(type), "dtype must be float32, float16 or bfloat16, got ", TypeName(type));
  int64_t padding = -1;
  if (padding_idx) {
    const int64_t vocab = table0.size(0);
    TORCH_CHECK_VALUE(*padding_idx >= -vocab && *padding_idx < vocab, "padding_idx must be a row of the table, got ", *padding_idx, " of ", vocab);
    padding = *padding_idx < 0 ? *padding_idx + vocab : *padding_idx;
  }
  CheckDevice("table", table0, table0);
  CheckDevice("ids", ids0, table0);
  const Tensor ids = Dense(ids0), table = Rows(table0);
  if (Tracked({table})) return EmbeddingFunction::apply(table, ids, scale, padding, type);
  return EmbeddingForward(ids, table, scale, padding, type);
}

}  // namespace

PYBIND11_MODULE(_sequence, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const KernelError &e) {
      PyErr_SetString(error_class->ptr(), e.what());
    }
  });
  m.def("bind", &Bind);
  m.def("linear_recurrence", &Recurrence, py::call_guard<py::gil_scoped_release>());
  m.def("block_norm", &BlockNorm, py::call_guard<py::gil_scoped_release>());
  m.def("embedding_lookup", &Embedding, py::call_guard<py::gil_scoped_release>());
}
