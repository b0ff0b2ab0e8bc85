// causal_conv, selective_scan and their single-token steps as PyTorch sees them: argument checks, allocation, the C-ABI calls and
// the autograd nodes, in native code (a step's kernel takes a few microseconds: the host sets its pace).
#include <optional>
#include <tuple>
#include <vector>

#include "torch_common.h"

namespace {

using at::Tensor;
using lasp_torch::check_status;
using lasp_torch::lasp_dtype_of;
using lasp_torch::Range;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

bool have(const Maybe& t) { return t.has_value() && t->defined(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

// ---- checks --------------------------------------------------------------------------------------------------------------------
void check_plain(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "lasp_b200 has no forward-mode derivative");
  TORCH_CHECK(t.is_cuda(), "lasp_b200 runs on CUDA tensors only (there is no CPU fallback); ", name, " is a tensor on ", t.device());
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", but the inputs are on ", like.device());
  TORCH_CHECK_TYPE(t.layout() == at::kStrided, name, " must be an ordinary (strided) tensor");
}
void check_of(const char* name, const Tensor& t, const Tensor& like, at::IntArrayRef sizes) {
  TORCH_CHECK_VALUE(t.sizes() == sizes, name, " has shape ", t.sizes(), "; expected ", sizes);
  TORCH_CHECK_TYPE(t.scalar_type() == like.scalar_type(), name, " is ", t.scalar_type(), "; expected ", like.scalar_type(), " as the inputs are");
  check_plain(name, t, like);
}
void check_param(const char* name, const Tensor& t, const Tensor& like, at::IntArrayRef sizes) {
  TORCH_CHECK_VALUE(t.sizes() == sizes, name, " has shape ", t.sizes(), "; expected ", sizes);
  TORCH_CHECK_TYPE(at::isFloatingType(t.scalar_type()), name, " is ", t.scalar_type(), "; expected a floating type");
  check_plain(name, t, like);
}
void check_state(const char* name, const Tensor& t, const Tensor& like, at::ScalarType type, at::IntArrayRef sizes) {
  TORCH_CHECK_VALUE(t.sizes() == sizes, name, " has shape ", t.sizes(), "; expected ", sizes);
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " is ", t.scalar_type(), "; expected ", type);
  check_plain(name, t, like);
}
void check_index(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK_VALUE(t.dim() == 1, name, " has shape ", t.sizes(), "; expected one dimension");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " is ", t.scalar_type(), "; expected int32 or int64");
  check_plain(name, t, like);
}
int64_t check_sequences(const Maybe& cu, const Tensor& x) {   // how many sequences there are
  if (!have(cu)) return x.size(0);
  check_index("cu_seqlens", *cu, x);
  TORCH_CHECK_VALUE(x.size(0) == 1, "packed sequences (cu_seqlens) need a batch of one row; got ", x.size(0));
  TORCH_CHECK_VALUE(cu->numel() >= 2, "cu_seqlens holds where each sequence begins and where the last one ends; got ", cu->numel(), " numbers");
  return cu->numel() - 1;
}
constexpr int64_t kMost = 2147480000;   // tokens, channels
void check_tokens(const char* name, const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() == 3, name, " has shape ", x.sizes(), "; expected (batch, tokens, channels)");
  lasp_dtype_of(x.scalar_type());
  TORCH_CHECK_VALUE(x.size(2) > 0, name, " has no channels");
  TORCH_CHECK_VALUE(x.size(1) <= kMost && x.size(2) <= kMost && x.size(0) <= INT32_MAX, name, " of shape ", x.sizes(), " is too large");
}
void check_step(const char* name, const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() == 2, name, " has shape ", x.sizes(), "; expected (batch, channels): one token of every row");
  lasp_dtype_of(x.scalar_type());
  TORCH_CHECK_VALUE(x.size(1) > 0 && x.size(1) <= kMost, name, " has ", x.size(1), " channels");
  TORCH_CHECK_VALUE(x.size(0) <= 65535, "a step of ", x.size(0), " rows exceeds 65535");
}
void check_slots(const Maybe& slots, const Tensor& x, const Tensor& state) {
  TORCH_CHECK_VALUE(state.size(0) <= INT32_MAX, "state holds too many slots");
  if (!have(slots)) {
    TORCH_CHECK_VALUE(state.size(0) == x.size(0), "state holds ", state.size(0), " sequences for ", x.size(0), " rows; name their slots");
    return;
  }
  check_index("slots", *slots, x);
  TORCH_CHECK_VALUE(slots->numel() == x.size(0), "slots names ", slots->numel(), " rows of ", x.size(0));
}
// A state that a step writes: in place, so it is what it is or the call is refused.
void check_written(const Tensor& state) {
  TORCH_CHECK_VALUE(state.is_contiguous(), "state is written in place and must be contiguous");
  TORCH_CHECK(!(at::GradMode::is_enabled() && state.requires_grad()), "state is written in place and must not require grad");
}
void refuse_gradients(const char* name, std::initializer_list<const Maybe> inputs) {
  if (!at::GradMode::is_enabled()) return;
  for (const Maybe& t : inputs)
    TORCH_CHECK(!have(t) || !t->requires_grad(), name, " has no backward pass: call it under torch.no_grad()");
}
int32_t activation_of(int64_t act) { return act ? LASP_ACT_SILU : LASP_ACT_NONE; }

// ---- layout --------------------------------------------------------------------------------------------------------------------
// The kernels take any pitches, with the channels (or states) of a token side by side.
Tensor side_by_side(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
lasp_tokens tokens_of(const Tensor& t) {   // (batch, tokens, channels) or (batch, tokens, groups, states)
  return t.defined() ? lasp_tokens{t.data_ptr(), t.stride(0), t.stride(1), t.dim() > 3 ? t.stride(2) : 0} : lasp_tokens{};
}
lasp_tokens rows_of(const Tensor& t) {   // (batch, channels) or (batch, groups, states)
  return t.defined() ? lasp_tokens{t.data_ptr(), t.stride(0), 0, t.dim() > 2 ? t.stride(1) : 0} : lasp_tokens{};
}
const void* data_of(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
Tensor contiguous(const Maybe& t) { return have(t) ? t->contiguous() : Tensor(); }
int32_t bits_of(const Tensor& t) { return t.defined() && t.scalar_type() == at::kLong ? 64 : 32; }

// Parameters are read as they are where they are all fp32 or all of the inputs' type; otherwise as fp32 (a cast that autograd sees).
bool as_inputs(const Tensor& x, const Tensor& p, const Maybe& q) {
  return p.scalar_type() == x.scalar_type() && (!have(q) || q->scalar_type() == x.scalar_type());
}
Tensor in_fp32(const Tensor& t) { return t.scalar_type() == at::kFloat ? t : t.to(at::kFloat); }

// A tensor taken out of a graph again: it may have been through a saved-tensor hook.
Tensor saved(const Tensor& t, const char* name, at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
  TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == device, "lasp_b200: the saved tensor ", name,
              " did not come back as what it was");
  return t;
}
void first_order_only() { TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "lasp_b200 has no second derivative (create_graph)"); }

// ---- convolution ----------------------------------------------------------------------------------------------------------------
lasp_conv_args conv_args(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& state, const Tensor& cu, int64_t act) {
  lasp_conv_args a = {};
  a.rows = (int32_t)x.size(0), a.tokens = (int32_t)x.size(1), a.channels = (int32_t)x.size(2), a.width = (int32_t)weight.size(1);
  a.dtype = lasp_dtype_of(x.scalar_type()), a.param_dtype = lasp_dtype_of(weight.scalar_type()), a.activation = activation_of(act);
  a.sequences = cu.defined() ? (int32_t)cu.numel() - 1 : 0, a.index_bits = bits_of(cu), a.offsets = data_of(cu);
  a.x = tokens_of(x), a.weight = weight.data_ptr(), a.bias = data_of(bias), a.state_in = data_of(state);
  return a;
}

variable_list run_conv(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& state, const Tensor& cu, int64_t act, bool want_state) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t sequences = cu.defined() ? cu.numel() - 1 : x.size(0);
  Tensor y = at::empty(x.sizes(), x.options()), last;
  if (want_state) last = at::empty({sequences, weight.size(1) - 1, x.size(2)}, x.options());
  if (x.size(0) == 0 || (x.size(1) == 0 && !want_state)) return {y, last};
  lasp_conv_args a = conv_args(x, weight, bias, state, cu, act);
  a.y = tokens_of(y), a.state_out = want_state ? last.data_ptr() : nullptr;
  Range range("lasp_b200_conv_forward");
  check_status("lasp_b200_conv_forward", lasp_b200_conv_forward(&a, at::cuda::getCurrentCUDAStream().stream()));
  return {y, last};
}

class Conv : public torch::autograd::Function<Conv> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias, const Maybe& state, const Maybe& cu,
                               int64_t act, bool want_state) {
    const Tensor xs = side_by_side(x), w = weight.contiguous(), b = contiguous(bias), s = contiguous(state), c = contiguous(cu);
    variable_list out = run_conv(xs, w, b, s, c, act, want_state);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, bias.value_or(Tensor()), state.value_or(Tensor()), cu.value_or(Tensor())});
    ctx->saved_data["act"] = act;
    ctx->saved_data["x"] = x.sizes().vec();
    ctx->saved_data["weight"] = weight.sizes().vec();
    ctx->saved_data["sequences"] = have(cu) ? cu->numel() : 0;
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->saved_data["param_type"] = (int64_t)weight.scalar_type();
    ctx->saved_data["device"] = (int64_t)x.device().index();
    if (!want_state) out.pop_back();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const variable_list in = ctx->get_saved_variables();
    variable_list out(7);
    const Tensor d_state = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !d_state.defined()) return out;
    const auto sizes = ctx->saved_data["x"].toIntVector(), wsizes = ctx->saved_data["weight"].toIntVector();
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt(), ptype = (at::ScalarType)ctx->saved_data["param_type"].toInt();
    const at::Device device(at::kCUDA, (c10::DeviceIndex)ctx->saved_data["device"].toInt());
    const int64_t cu_count = ctx->saved_data["sequences"].toInt(), sequences = cu_count ? cu_count - 1 : sizes[0];
    const c10::cuda::CUDAGuard guard(device);
    const Tensor x = side_by_side(saved(in[0], "x", sizes, type, device)), weight = saved(in[1], "weight", wsizes, ptype, device).contiguous();
    const Tensor bias = in[2].defined() ? saved(in[2], "bias", {wsizes[0]}, ptype, device).contiguous() : Tensor();
    const Tensor state = in[3].defined() ? saved(in[3], "initial_state", {sequences, wsizes[1] - 1, wsizes[0]}, type, device).contiguous() : Tensor();
    Tensor cu;
    if (cu_count) {
      TORCH_CHECK(in[4].defined() && in[4].numel() == cu_count && in[4].device() == device && !at::isFloatingType(in[4].scalar_type()),
                  "lasp_b200: the saved tensor cu_seqlens did not come back as what it was");
      cu = in[4].scalar_type() == at::kInt ? in[4].contiguous() : in[4].to(at::kLong).contiguous();
    }
    const Tensor dy = side_by_side(grads[0].defined() ? grads[0] : at::zeros(sizes, x.options()));
    const Tensor d_last = contiguous(maybe(d_state));
    Tensor dx = at::empty(sizes, x.options()), dw = at::empty(wsizes, weight.options()), db, d_first;
    if (bias.defined()) db = at::empty(bias.sizes(), bias.options());
    if (state.defined()) d_first = at::empty(state.sizes(), state.options());
    if (sizes[0] == 0) {
      dw.zero_();
      if (db.defined()) db.zero_();
    } else {
      lasp_conv_args a = conv_args(x, weight, bias, state, cu, ctx->saved_data["act"].toInt());
      a.dy = tokens_of(dy), a.dx = tokens_of(dx), a.dstate_out = data_of(d_last);
      a.dstate_in = d_first.defined() ? d_first.data_ptr() : nullptr, a.dweight = dw.data_ptr(), a.dbias = db.defined() ? db.data_ptr() : nullptr;
      const Tensor ws = at::empty({(int64_t)lasp_b200_conv_workspace_bytes(&a)}, x.options().dtype(at::kByte));
      a.ws = ws.data_ptr(), a.ws_bytes = (size_t)ws.numel();
      Range range("lasp_b200_conv_backward");
      check_status("lasp_b200_conv_backward", lasp_b200_conv_backward(&a, at::cuda::getCurrentCUDAStream().stream()));
    }
    out[0] = dx, out[1] = dw, out[2] = db, out[3] = d_first;
    return out;
  }
};

std::tuple<Tensor, Tensor> causal_conv(const Tensor& x, const Tensor& weight, const Maybe& bias, int64_t act, const Maybe& state, const Maybe& cu,
                                       bool want_state) {
  check_tokens("x", x);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) == x.size(2) && weight.size(1) >= 2 && weight.size(1) <= 4, "weight has shape ",
                    weight.sizes(), "; expected (", x.size(2), ", 2 to 4 taps)");
  check_plain("x", x, x);
  check_param("weight", weight, x, weight.sizes());
  if (have(bias)) check_param("bias", *bias, x, {x.size(2)});
  const int64_t sequences = check_sequences(cu, x);
  TORCH_CHECK_VALUE(x.size(0) <= 65535 && sequences <= (1 << 17), "batch of ", x.size(0), " rows, ", sequences, " sequences: at most 65535 and 131072");
  if (have(state)) check_state("initial_state", *state, x, x.scalar_type(), {sequences, weight.size(1) - 1, x.size(2)});
  const bool plain = as_inputs(x, weight, bias);
  const Tensor w = plain ? weight : in_fp32(weight);
  const Maybe b = have(bias) && !plain ? Maybe(in_fp32(*bias)) : bias;
  variable_list out;
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (have(b) && b->requires_grad()) || (have(state) && state->requires_grad())))
    out = Conv::apply(x, w, b, state, cu, act, want_state);
  else
    out = run_conv(side_by_side(x), w.contiguous(), contiguous(b), contiguous(state), contiguous(cu), act, want_state);
  return {out[0], want_state ? out[1] : Tensor()};
}

Tensor causal_conv_step(const Tensor& state, const Tensor& x, const Tensor& weight, const Maybe& bias, int64_t act, const Maybe& slots) {
  check_step("x", x);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) == x.size(1) && weight.size(1) >= 2 && weight.size(1) <= 4, "weight has shape ",
                    weight.sizes(), "; expected (", x.size(1), ", 2 to 4 taps)");
  TORCH_CHECK_VALUE(state.dim() == 3, "state has shape ", state.sizes(), "; expected (slots, taps - 1, channels)");
  check_plain("x", x, x);
  check_param("weight", weight, x, weight.sizes());
  if (have(bias)) check_param("bias", *bias, x, {x.size(1)});
  check_state("state", state, x, x.scalar_type(), {state.size(0), weight.size(1) - 1, x.size(1)});
  check_slots(slots, x, state);
  check_written(state);
  refuse_gradients("causal_conv_step", {x, weight, bias});
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  if (x.size(0) == 0) return y;
  const bool plain = as_inputs(x, weight, bias);
  const Tensor xs = side_by_side(x), w = (plain ? weight : in_fp32(weight)).contiguous();
  const Tensor b = have(bias) ? (plain ? *bias : in_fp32(*bias)).contiguous() : Tensor(), named = contiguous(slots);
  lasp_conv_step_args a = {};
  a.rows = (int32_t)x.size(0), a.channels = (int32_t)x.size(1), a.width = (int32_t)weight.size(1);
  a.dtype = lasp_dtype_of(x.scalar_type()), a.param_dtype = lasp_dtype_of(w.scalar_type()), a.activation = activation_of(act);
  a.slot_count = (int32_t)state.size(0), a.index_bits = bits_of(named), a.slots = data_of(named);
  a.x = rows_of(xs), a.y = rows_of(y), a.weight = w.data_ptr(), a.bias = data_of(b), a.state = state.data_ptr();
  Range range("lasp_b200_conv_step");
  check_status("lasp_b200_conv_step", lasp_b200_conv_step(&a, at::cuda::getCurrentCUDAStream().stream()));
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return y;
}

// ---- scan -------------------------------------------------------------------------------------------------------------------------
struct ScanInputs {   // laid out as the kernels take them; B and C (batch, tokens, [groups,] states)
  Tensor u, dt, A, B, C, D, z, bias, state, cu;
  bool softplus;
  int64_t sequences() const { return cu.defined() ? cu.numel() - 1 : u.size(0); }
  Tensor new_state() const { return at::empty({sequences(), u.size(2), A.size(1)}, A.options()); }
};

lasp_scan_args scan_args(const ScanInputs& s) {
  lasp_scan_args a = {};
  a.rows = (int32_t)s.u.size(0), a.tokens = (int32_t)s.u.size(1), a.channels = (int32_t)s.u.size(2), a.states = (int32_t)s.A.size(1);
  a.groups = s.B.dim() > 3 ? (int32_t)s.B.size(2) : 1, a.dtype = lasp_dtype_of(s.u.scalar_type()), a.softplus = s.softplus ? 1 : 0;
  const Tensor& p = s.D.defined() ? s.D : s.bias;
  a.param_dtype = p.defined() ? lasp_dtype_of(p.scalar_type()) : LASP_F32;
  a.sequences = s.cu.defined() ? (int32_t)s.cu.numel() - 1 : 0, a.index_bits = bits_of(s.cu), a.offsets = data_of(s.cu);
  a.u = tokens_of(s.u), a.dt = tokens_of(s.dt), a.z = tokens_of(s.z), a.B = tokens_of(s.B), a.C = tokens_of(s.C);
  a.A = s.A.const_data_ptr<float>(), a.D = data_of(s.D), a.dt_bias = data_of(s.bias);
  a.state_in = s.state.defined() ? s.state.const_data_ptr<float>() : nullptr;
  return a;
}

variable_list run_scan(const ScanInputs& s, bool want_state, bool keep) {   // y, last states, what the backward pass takes
  const c10::cuda::CUDAGuard guard(s.u.device());
  Tensor y = at::empty(s.u.sizes(), s.u.options()), last, kept;
  if (want_state) last = s.new_state();
  if (s.u.size(0) == 0) return {y, last, keep ? at::empty({0}, s.u.options().dtype(at::kByte)) : kept};
  lasp_scan_args a = scan_args(s);
  a.y = tokens_of(y), a.state_out = want_state ? last.data_ptr<float>() : nullptr;
  if (keep) {
    kept = at::empty({(int64_t)lasp_b200_scan_kept_bytes(&a)}, s.u.options().dtype(at::kByte));
    a.kept = kept.data_ptr(), a.kept_bytes = (size_t)kept.numel();
  }
  Tensor ws;
  if (const size_t need = lasp_b200_scan_forward_workspace_bytes(&a)) {
    ws = at::empty({(int64_t)need}, s.u.options().dtype(at::kByte));
    a.ws = ws.data_ptr(), a.ws_bytes = need;
  }
  Range range("lasp_b200_scan_forward");
  check_status("lasp_b200_scan_forward", lasp_b200_scan_forward(&a, at::cuda::getCurrentCUDAStream().stream()));
  return {y, last, kept};
}

class Scan : public torch::autograd::Function<Scan> {
 public:
  static ScanInputs laid_out(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Maybe& D, const Maybe& z,
                             const Maybe& bias, const Maybe& state, const Maybe& cu, bool softplus) {
    return {side_by_side(u), side_by_side(dt), A.contiguous(), side_by_side(B), side_by_side(C), contiguous(D),
            have(z) ? side_by_side(*z) : Tensor(), contiguous(bias), contiguous(state), contiguous(cu), softplus};
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                               const Maybe& D, const Maybe& z, const Maybe& bias, const Maybe& state, const Maybe& cu, bool softplus, bool want_state) {
    variable_list out = run_scan(laid_out(u, dt, A, B, C, D, z, bias, state, cu, softplus), want_state, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({u, dt, A, B, C, D.value_or(Tensor()), z.value_or(Tensor()), bias.value_or(Tensor()), cu.value_or(Tensor()), out[2]});
    ctx->saved_data["u"] = u.sizes().vec();
    ctx->saved_data["B"] = B.sizes().vec(), ctx->saved_data["C"] = C.sizes().vec();
    ctx->saved_data["sequences"] = have(cu) ? cu->numel() : 0;
    ctx->saved_data["kept"] = out[2].numel();
    ctx->saved_data["type"] = (int64_t)u.scalar_type();
    ctx->saved_data["param_type"] = (int64_t)(have(D) ? D->scalar_type() : have(bias) ? bias->scalar_type() : at::kFloat);
    ctx->saved_data["device"] = (int64_t)u.device().index();
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["state"] = have(state);
    out.resize(want_state ? 2 : 1);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const variable_list in = ctx->get_saved_variables();
    variable_list out(12);
    const Tensor d_state = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !d_state.defined()) return out;
    const auto sizes = ctx->saved_data["u"].toIntVector(), bsizes = ctx->saved_data["B"].toIntVector(), csizes = ctx->saved_data["C"].toIntVector();
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt(), ptype = (at::ScalarType)ctx->saved_data["param_type"].toInt();
    const at::Device device(at::kCUDA, (c10::DeviceIndex)ctx->saved_data["device"].toInt());
    const int64_t cu_count = ctx->saved_data["sequences"].toInt(), channels = sizes[2], states = bsizes.back();
    const c10::cuda::CUDAGuard guard(device);
    const auto param = [&](const Tensor& t, const char* name) { return t.defined() ? Maybe(saved(t, name, {channels}, ptype, device)) : Maybe(); };
    Maybe cu;
    if (cu_count) {
      TORCH_CHECK(in[8].defined() && in[8].numel() == cu_count && in[8].device() == device && !at::isFloatingType(in[8].scalar_type()),
                  "lasp_b200: the saved tensor cu_seqlens did not come back as what it was");
      cu = in[8].scalar_type() == at::kInt ? in[8] : in[8].to(at::kLong);
    }
    const ScanInputs s = laid_out(saved(in[0], "u", sizes, type, device), saved(in[1], "dt", sizes, type, device),
                                  saved(in[2], "A", {channels, states}, at::kFloat, device), saved(in[3], "B", bsizes, type, device),
                                  saved(in[4], "C", csizes, type, device), param(in[5], "D"),
                                  in[6].defined() ? Maybe(saved(in[6], "z", sizes, type, device)) : Maybe(), param(in[7], "dt_bias"), Maybe(), cu,
                                  ctx->saved_data["softplus"].toBool());
    const Tensor kept = saved(in[9], "of the kept states", {ctx->saved_data["kept"].toInt()}, at::kByte, device).contiguous();
    const Tensor dy = side_by_side(grads[0].defined() ? grads[0] : at::zeros(sizes, s.u.options()));
    const Tensor d_last = contiguous(maybe(d_state));
    Tensor du = at::empty(sizes, s.u.options()), ddt = at::empty(sizes, s.u.options()), dA = at::empty(s.A.sizes(), s.A.options());
    Tensor dB = at::empty(bsizes, s.u.options()), dC = at::empty(bsizes, s.u.options()), dD, dz, dbias, d_first;
    if (s.D.defined()) dD = at::empty({channels}, s.D.options());
    if (s.z.defined()) dz = at::empty(sizes, s.u.options());
    if (s.bias.defined()) dbias = at::empty({channels}, s.bias.options());
    if (ctx->saved_data["state"].toBool()) d_first = s.new_state();
    if (sizes[0] == 0) {
      for (Tensor* t : {&dA, &dD, &dbias})
        if (t->defined()) t->zero_();
    } else {
      lasp_scan_args a = scan_args(s);
      a.dy = tokens_of(dy), a.du = tokens_of(du), a.ddt = tokens_of(ddt), a.dz = tokens_of(dz), a.dB = tokens_of(dB), a.dC = tokens_of(dC);
      a.dstate_out = d_last.defined() ? d_last.const_data_ptr<float>() : nullptr;
      a.dstate_in = d_first.defined() ? d_first.data_ptr<float>() : nullptr;
      a.dA = dA.data_ptr<float>(), a.dD = dD.defined() ? dD.data_ptr() : nullptr, a.ddt_bias = dbias.defined() ? dbias.data_ptr() : nullptr;
      a.kept = kept.data_ptr(), a.kept_bytes = (size_t)kept.numel();
      const Tensor ws = at::empty({(int64_t)lasp_b200_scan_workspace_bytes(&a)}, s.u.options().dtype(at::kByte));
      a.ws = ws.data_ptr(), a.ws_bytes = (size_t)ws.numel();
      Range range("lasp_b200_scan_backward");
      check_status("lasp_b200_scan_backward", lasp_b200_scan_backward(&a, at::cuda::getCurrentCUDAStream().stream()));
    }
    out[0] = du, out[1] = ddt, out[2] = dA, out[3] = dB, out[4] = dC, out[5] = dD, out[6] = dz, out[7] = dbias, out[8] = d_first;
    return out;
  }
};

void check_scan_params(const Tensor& u, const Tensor& A, const Maybe& D, const Maybe& bias) {
  const int64_t c = u.size(-1);
  TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == c && A.size(1) >= 1 && A.size(1) <= 64, "A has shape ", A.sizes(), "; expected (", c, ", 1 to 64 states)");
  check_state("A", A, u, at::kFloat, A.sizes());
  if (have(D)) check_param("D", *D, u, {c});
  if (have(bias)) check_param("dt_bias", *bias, u, {c});
}
// How many groups of channels B or C has: (..., states) is one
int64_t groups_of(const char* name, const Tensor& t, const Tensor& u, int64_t states) {
  TORCH_CHECK_VALUE((t.dim() == u.dim() || t.dim() == u.dim() + 1) && t.sizes().slice(0, u.dim() - 1) == u.sizes().slice(0, u.dim() - 1) && t.size(-1) == states,
                    name, " has shape ", t.sizes(), "; expected (", u.sizes().slice(0, u.dim() - 1), ", [groups,] ", states, " states)");
  check_of(name, t, u, t.sizes());
  if (t.dim() == u.dim()) return 1;
  TORCH_CHECK_VALUE(t.size(-2) >= 1 && t.size(-2) <= 65535 && u.size(-1) % t.size(-2) == 0, name, " has ", t.size(-2), " groups, which must divide ", u.size(-1), " channels");
  return t.size(-2);
}
void check_groups(const Tensor& B, const Tensor& C, const Tensor& u, int64_t states) {
  const int64_t of_B = groups_of("B", B, u, states), of_C = groups_of("C", C, u, states);
  TORCH_CHECK_VALUE(of_B == of_C, "C has ", of_C, " groups, B has ", of_B);
}

std::tuple<Tensor, Tensor> selective_scan(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Maybe& D,
                                          const Maybe& z, const Maybe& bias, bool softplus, const Maybe& state, const Maybe& cu, bool want_state) {
  check_tokens("u", u);
  check_plain("u", u, u);
  check_of("dt", dt, u, u.sizes());
  check_scan_params(u, A, D, bias);
  check_groups(B, C, u, A.size(1));
  if (have(z)) check_of("z", *z, u, u.sizes());
  const int64_t sequences = check_sequences(cu, u);
  if (have(state)) check_state("initial_state", *state, u, at::kFloat, {sequences, u.size(2), A.size(1)});
  const bool plain = have(D) ? as_inputs(u, *D, bias) : have(bias) && bias->scalar_type() == u.scalar_type();
  const Maybe skip = have(D) && !plain ? Maybe(in_fp32(*D)) : D, b = have(bias) && !plain ? Maybe(in_fp32(*bias)) : bias;
  bool graph = false;
  if (at::GradMode::is_enabled()) {
    for (const Tensor* t : {&u, &dt, &A, &B, &C}) graph |= t->requires_grad();
    for (const Maybe* t : {&skip, &z, &b, &state}) graph |= have(*t) && (*t)->requires_grad();
  }
  variable_list out;
  if (graph)
    out = Scan::apply(u, dt, A, B, C, skip, z, b, state, cu, softplus, want_state);
  else
    out = run_scan(Scan::laid_out(u, dt, A, B, C, skip, z, b, state, cu, softplus), want_state, false);
  return {out[0], want_state ? out[1] : Tensor()};
}

Tensor selective_scan_step(const Tensor& state, const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Maybe& D,
                           const Maybe& z, const Maybe& bias, bool softplus, const Maybe& slots) {
  check_step("u", u);
  check_plain("u", u, u);
  check_of("dt", dt, u, u.sizes());
  check_scan_params(u, A, D, bias);
  check_groups(B, C, u, A.size(1));
  if (have(z)) check_of("z", *z, u, u.sizes());
  TORCH_CHECK_VALUE(state.dim() == 3, "state has shape ", state.sizes(), "; expected (slots, channels, states)");
  check_state("state", state, u, at::kFloat, {state.size(0), u.size(1), A.size(1)});
  check_slots(slots, u, state);
  check_written(state);
  refuse_gradients("selective_scan_step", {u, dt, A, B, C, D, z, bias});
  const c10::cuda::CUDAGuard guard(u.device());
  Tensor y = at::empty(u.sizes(), u.options());
  if (u.size(0) == 0) return y;
  const bool plain = have(D) ? as_inputs(u, *D, bias) : have(bias) && bias->scalar_type() == u.scalar_type();
  const auto param = [&](const Maybe& t) { return have(t) ? (plain ? *t : in_fp32(*t)).contiguous() : Tensor(); };
  const Tensor us = side_by_side(u), dts = side_by_side(dt), As = A.contiguous(), skip = param(D), b = param(bias), named = contiguous(slots);
  const Tensor zs = have(z) ? side_by_side(*z) : Tensor(), Bs = side_by_side(B), Cs = side_by_side(C);
  lasp_scan_step_args a = {};
  a.rows = (int32_t)u.size(0), a.channels = (int32_t)u.size(1), a.states = (int32_t)A.size(1), a.groups = Bs.dim() > 2 ? (int32_t)Bs.size(1) : 1;
  const Tensor& p = skip.defined() ? skip : b;
  a.dtype = lasp_dtype_of(u.scalar_type()), a.param_dtype = p.defined() ? lasp_dtype_of(p.scalar_type()) : LASP_F32, a.softplus = softplus ? 1 : 0;
  a.slot_count = (int32_t)state.size(0), a.index_bits = bits_of(named), a.slots = data_of(named);
  a.u = rows_of(us), a.dt = rows_of(dts), a.z = rows_of(zs), a.B = rows_of(Bs), a.C = rows_of(Cs), a.y = rows_of(y);
  a.A = As.const_data_ptr<float>(), a.D = data_of(skip), a.dt_bias = data_of(b), a.state = state.data_ptr<float>();
  Range range("lasp_b200_scan_step");
  check_status("lasp_b200_scan_step", lasp_b200_scan_step(&a, at::cuda::getCurrentCUDAStream().stream()));
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return y;
}

// As nodes of a traced graph (see torch_ops.cpp); other calls spare themselves the dispatcher.
TORCH_LIBRARY_FRAGMENT(lasp_b200, m) {
  m.def("causal_conv(Tensor x, Tensor weight, Tensor? bias, int activation, Tensor? initial_state, Tensor? cu_seqlens, bool return_state) -> (Tensor, Tensor)");
  m.impl("causal_conv", c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(causal_conv));
  m.def("causal_conv_step(Tensor(a!) state, Tensor x, Tensor weight, Tensor? bias, int activation, Tensor? slots) -> Tensor");
  m.impl("causal_conv_step", c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(causal_conv_step));
  m.def("selective_scan(Tensor u, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, bool dt_softplus, "
        "Tensor? initial_state, Tensor? cu_seqlens, bool return_state) -> (Tensor, Tensor)");
  m.impl("selective_scan", c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(selective_scan));
  m.def("selective_scan_step(Tensor(a!) state, Tensor u, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, "
        "bool dt_softplus, Tensor? slots) -> Tensor");
  m.impl("selective_scan_step", c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(selective_scan_step));
}
template <typename F, typename... Args>
auto call(const char* name, F* fn, const Args&... args) {
  if (!torch::jit::tracer::isTracing()) return fn(args...);
  return c10::Dispatcher::singleton().findSchemaOrThrow((std::string("lasp_b200::") + name).c_str(), "").template typed<F>().call(args...);
}

// ---- the module's methods: positional arguments, None for what is left out --------------------------------------------------------
const Tensor& tensor(PyObject* p, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(p), name, " must be a tensor");
  return THPVariable_Unpack(p);
}
Maybe optional(PyObject* p, const char* name) { return p == Py_None ? Maybe() : Maybe(tensor(p, name)); }
bool flag(PyObject* p) {
  const int v = PyObject_IsTrue(p);
  if (v < 0) throw python_error();
  return v != 0;
}
PyObject* outputs(std::tuple<Tensor, Tensor>&& got, bool want_state) {
  if (!want_state) return THPVariable_Wrap(std::move(std::get<0>(got)));
  PyObject *y = THPVariable_Wrap(std::move(std::get<0>(got))), *s = y ? THPVariable_Wrap(std::move(std::get<1>(got))) : nullptr;
  PyObject* both = s ? PyTuple_Pack(2, y, s) : nullptr;
  Py_XDECREF(y);
  Py_XDECREF(s);
  return both;
}

}  // namespace

namespace lasp_torch {

PyObject* py_causal_conv(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 7, "causal_conv takes 7 arguments");
  const Tensor &x = tensor(args[0], "x"), &weight = tensor(args[1], "weight");
  const Maybe bias = optional(args[2], "bias"), state = optional(args[4], "initial_state"), cu = optional(args[5], "cu_seqlens");
  const int64_t act = flag(args[3]);
  const bool want_state = flag(args[6]);
  std::tuple<Tensor, Tensor> got;
  {
    pybind11::gil_scoped_release no_gil;
    got = call("causal_conv", causal_conv, x, weight, bias, act, state, cu, want_state);
  }
  return outputs(std::move(got), want_state);
  END_HANDLE_TH_ERRORS
}

PyObject* py_causal_conv_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 6, "causal_conv_step takes 6 arguments");
  const Tensor &state = tensor(args[0], "state"), &x = tensor(args[1], "x"), &weight = tensor(args[2], "weight");
  const Maybe bias = optional(args[3], "bias"), slots = optional(args[5], "slots");
  const int64_t act = flag(args[4]);
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    y = call("causal_conv_step", causal_conv_step, state, x, weight, bias, act, slots);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

PyObject* py_selective_scan(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 12, "selective_scan takes 12 arguments");
  const Tensor &u = tensor(args[0], "u"), &dt = tensor(args[1], "dt"), &A = tensor(args[2], "A"), &B = tensor(args[3], "B"), &C = tensor(args[4], "C");
  const Maybe D = optional(args[5], "D"), z = optional(args[6], "z"), bias = optional(args[7], "dt_bias");
  const bool softplus = flag(args[8]);
  const Maybe state = optional(args[9], "initial_state"), cu = optional(args[10], "cu_seqlens");
  const bool want_state = flag(args[11]);
  std::tuple<Tensor, Tensor> got;
  {
    pybind11::gil_scoped_release no_gil;
    got = call(
        "selective_scan", selective_scan, u, dt, A, B, C, D, z, bias, softplus, state, cu, want_state);
  }
  return outputs(std::move(got), want_state);
  END_HANDLE_TH_ERRORS
}

PyObject* py_selective_scan_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 11, "selective_scan_step takes 11 arguments");
  const Tensor &state = tensor(args[0], "state"), &u = tensor(args[1], "u"), &dt = tensor(args[2], "dt"), &A = tensor(args[3], "A"),
               &B = tensor(args[4], "B"), &C = tensor(args[5], "C");
  const Maybe D = optional(args[6], "D"), z = optional(args[7], "z"), bias = optional(args[8], "dt_bias"), slots = optional(args[10], "slots");
  const bool softplus = flag(args[9]);
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    y = call(
        "selective_scan_step", selective_scan_step, state, u, dt, A, B, C, D, z, bias, softplus, slots);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

}  // namespace lasp_torch
