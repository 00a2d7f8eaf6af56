// The recurrent mixers' operators over the C ABI: the short convolution, the selective
// state space scan and the group norm, with their autograd nodes, on the tensors' own
// device and its current stream.
//
// kernels.py checks the arguments; here are types, layouts, outputs, workspaces, launches
// and the graph nodes.  A call computes in bf16 where all its activations are, else in
// fp32; outputs come in x's type, gradients in their input's.  Activations may be slices
// of wider rows; anything else is copied.
#include <c10/core/DeviceGuard.h>

#include <limits>
#include <optional>

#include "torch_common.hpp"

namespace {

using Opt = std::optional<Tensor>;

Tensor get(const Opt& t) { return t ? *t : Tensor(); }
Tensor cast(const Tensor& t, at::ScalarType dtype) { return t.defined() ? t.to(dtype) : t; }
Tensor params(const Tensor& t) { return t.defined() ? f32(t) : t; }

// bf16 where every one given is
at::ScalarType common(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t->defined() && t->scalar_type() != at::kBFloat16) return at::kFloat;
  return at::kBFloat16;
}

// t itself where its last dimension is contiguous and the strides between are ones the
// library takes (up to `limit`), else a contiguous copy
Tensor rows(const Tensor& t, int64_t limit = LZ_MIXER_MAX_STRIDE) {
  if (!t.defined()) return t;
  const int64_t last = t.dim() - 1;
  bool ok = t.size(last) <= 1 || t.stride(last) == 1;
  for (int64_t d = 1; d < last; ++d) ok = ok && (t.size(d) <= 1 || t.stride(d) <= limit);
  return ok ? t : t.contiguous();
}

// Elements from one entry of a dimension to the next; 0 where there is one entry
long long step_of(const Tensor& t, int64_t d) {
  return t.defined() && t.size(d) > 1 ? t.stride(d) : 0;
}

// A backward may run on a stream that is being captured though its forward ran eagerly:
// refused, as kernels.py refuses the calls
void refuse_capture(const Tensor& t) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(static_cast<hipStream_t>(stream_of(t)), &status) != hipSuccess ||
      status != hipStreamCaptureStatusNone)
    throw std::runtime_error("lizard_reproduction_amd kernels: calls under HIP graph capture are "
                             "not supported (run the kernels eagerly)");
}

// Lengths of sequences as the library takes them; 64-bit ones into [0, most] before they lose
// their upper half
Tensor int_lengths(const Opt& lengths, int64_t most) {
  if (!lengths) return {};
  return as(lengths->scalar_type() == at::kInt ? *lengths : lengths->clamp(0, most), at::kInt);
}

// Contiguous, of t's sizes and type; not given where t is not
Tensor like(const Tensor& t) {
  return t.defined() ? at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous))
                     : Tensor();
}
// the gradient of a call's output of t's sizes and type, zeros where there is none
Tensor upstream(const Tensor& grad, const Tensor& t) {
  return grad.defined() ? as(grad, t.scalar_type()) : like(t).zero_();
}
void zero(const variable_list& tensors) {
  for (const Tensor& t : tensors)
    if (t.defined()) t.zero_();
}

int64_t i64(at::ScalarType t) { return static_cast<int64_t>(t); }

// Outputs' types as an autograd node keeps them; -1 for an input that was not given
std::vector<int64_t> types(std::initializer_list<const Tensor*> tensors) {
  std::vector<int64_t> out;
  for (const Tensor* t : tensors) out.push_back(t->defined() ? i64(t->scalar_type()) : -1);
  return out;
}

// Gradients in their inputs' types, none for an input that was not given
variable_list as_inputs(variable_list grads, const std::vector<int64_t>& types) {
  for (size_t i = 0; i < types.size(); ++i)
    grads[i] = types[i] < 0 ? Tensor() : grads[i].to(static_cast<at::ScalarType>(types[i]));
  return grads;
}

// ---------------------------------------------------------------------------
// selective state space scan
// ---------------------------------------------------------------------------

// x, dt, z [B, L, E] (a step: L = 1), B, C [B, L, G, N], A [E, N]
struct SsmCall {
  Tensor x, dt, A, B, C, D, z, bias;
  bool softplus;

  lz_ssm_args args() const {
    lz_ssm_args a = {};
    a.x = ptr(x), a.dt = ptr(dt), a.z = ptr(z), a.B = ptr(B), a.C = ptr(C);
    a.A = ptr<float>(A), a.D = ptr<float>(D), a.dt_bias = ptr<float>(bias);
    a.x_batch = step_of(x, 0), a.dt_batch = step_of(dt, 0), a.z_batch = step_of(z, 0);
    a.B_batch = step_of(B, 0), a.C_batch = step_of(C, 0);
    a.x_token = step_of(x, 1), a.dt_token = step_of(dt, 1), a.z_token = step_of(z, 1);
    a.B_token = step_of(B, 1), a.C_token = step_of(C, 1);
    a.B_group = step_of(B, 2), a.C_group = step_of(C, 2);
    a.batch = i32(x.size(0)), a.length = i32(x.size(1)), a.channels = i32(x.size(2));
    a.state = i32(A.size(1)), a.groups = i32(B.size(2));
    a.softplus = softplus, a.bf16 = x.scalar_type() == at::kBFloat16;
    return a;
  }

  Tensor forward(const Tensor& state_in, const Tensor& state_out, const Tensor& lengths,
                 const Tensor& states) const {
    Tensor y = like(x);
    if (!y.numel()) return y;
    const lz_ssm_args a = args();
    const size_t need =
        lz_ssm_fwd_workspace_bytes(a.batch, a.length, a.channels, a.state, a.groups);
    const Tensor ws = bytes(need ? need : 1, x);
    check(lz_ssm_fwd(&a, ptr<float>(state_in), ptr<float>(state_out), ptr<int>(lengths), ptr(y),
                     ptr<float>(states), ptr(ws), need, stream_of(x)),
          "lz_ssm_fwd");
    return y;
  }
};

SsmCall ssm_call(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                 const Tensor& C, const Tensor& D, const Tensor& z, const Tensor& bias,
                 bool softplus) {
  const auto t = common({&x, &dt, &B, &C, &z});
  return {rows(cast(x, t)), rows(cast(dt, t)), params(A), rows(cast(B, t)), rows(cast(C, t)),
          params(D), rows(cast(z, t)), params(bias), softplus};
}

struct SsmNode : torch::autograd::Function<SsmNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A,
                        const Tensor& B, const Tensor& C, const Opt& D_, const Opt& z_,
                        const Opt& bias_, bool softplus) {
    const Tensor D = get(D_), z = get(z_), bias = get(bias_);
    const c10::DeviceGuard guard(x.device());
    const SsmCall c = ssm_call(x, dt, A, B, C, D, z, bias, softplus);
    const lz_ssm_args a = c.args();
    const Tensor states = at::empty(
        {static_cast<int64_t>(lz_ssm_states_bytes(a.batch, a.length, a.channels, a.state, a.z != nullptr) / 4)},
        c.A.options());
    const Tensor y = c.forward({}, {}, {}, states);
    ctx->save_for_backward({c.x, c.dt, c.A, c.B, c.C, c.D, c.z, c.bias, states});
    ctx->saved_data["types"] = types({&x, &dt, &A, &B, &C, &D, &z, &bias});
    ctx->saved_data["softplus"] = softplus;
    return y.to(x.scalar_type());
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    const SsmCall c{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7],
                    ctx->saved_data["softplus"].toBool()};
    const Tensor& states = s[8];
    const c10::DeviceGuard guard(c.x.device());
    refuse_capture(c.x);
    const lz_ssm_args a = c.args();
    const Tensor dy = upstream(grads[0], c.x);
    const Tensor dx = like(c.x), ddt = like(c.dt), dA = like(c.A),
                 dB = like(c.B), dC = like(c.C), dD = like(c.D),
                 dz = like(c.z), dbias = like(c.bias);
    const variable_list all{dx, ddt, dA, dB, dC, dD, dz, dbias};
    if (dy.numel()) {
      const size_t need =
          lz_ssm_bwd_workspace_bytes(a.batch, a.length, a.channels, a.state, a.groups);
      const Tensor ws = bytes(need, c.x);
      check(lz_ssm_bwd(&a, ptr<float>(states), ptr(dy), ptr(dx), ptr(ddt), ptr(dz), ptr(dB),
                       ptr(dC), ptr<float>(dA), ptr<float>(dD), ptr<float>(dbias), ptr(ws), need,
                       stream_of(c.x)),
            "lz_ssm_bwd");
    } else {
      zero(all);
    }
    variable_list out = as_inputs(all, ctx->saved_data["types"].toIntVector());
    out.emplace_back();
    return out;
  }
};

Tensor ssm(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
           const Opt& D_, const Opt& z_, const Opt& bias_, bool softplus) {
  const Tensor D = get(D_), z = get(z_), bias = get(bias_);
  if (any_grad({&x, &dt, &A, &B, &C, &D, &z, &bias}))
    return SsmNode::apply(x, dt, A, B, C, D_, z_, bias_, softplus);
  const c10::DeviceGuard guard(x.device());
  return ssm_call(x, dt, A, B, C, D, z, bias, softplus).forward({}, {}, {}, {}).to(x.scalar_type());
}

std::tuple<Tensor, Tensor> ssm_prefill(const Tensor& x, const Tensor& dt, const Tensor& A,
                                       const Tensor& B, const Tensor& C, const Opt& D, const Opt& z,
                                       const Opt& bias, bool softplus, const Opt& state,
                                       const Opt& lengths_) {
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(x.device());
  const SsmCall c = ssm_call(x, dt, A, B, C, get(D), get(z), get(bias), softplus);
  const Tensor in = params(get(state));
  const Tensor lengths = int_lengths(lengths_, x.size(1));
  Tensor out = at::empty({x.size(0), x.size(2), A.size(1)}, c.A.options());
  const Tensor y = c.forward(in, out, lengths, {});
  return {y.to(x.scalar_type()), out};
}

// x, dt, z [B, 1, E], B, C [B, 1, G, N], state fp32 [B, E, N], updated in place
Tensor ssm_step(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                const Tensor& C, const Tensor& state, const Opt& D, const Opt& z, const Opt& bias,
                bool softplus) {
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(x.device());
  const SsmCall c = ssm_call(x, dt, A, B, C, get(D), get(z), get(bias), softplus);
  const Tensor y = like(c.x);
  const lz_ssm_args a = c.args();
  if (y.numel())
    check(lz_ssm_decode_step(&a, ptr<float>(state), ptr(y), stream_of(x)), "lz_ssm_decode_step");
  return y.to(x.scalar_type());
}

// Whether a decode step's launch takes t as it is: on x's device, of the given type and
// sizes, its last dimension contiguous (all of it, with whole)
bool fits(const Tensor& t, const Tensor& x, at::ScalarType dtype, at::IntArrayRef sizes, bool whole) {
  const int64_t last = t.dim() - 1;
  return t.is_cuda() && t.device() == x.device() && t.scalar_type() == dtype &&
         t.sizes() == sizes && (whole ? t.is_contiguous() : t.size(last) == 1 || t.stride(last) == 1);
}
bool fits(const Opt& t, const Tensor& x, at::ScalarType dtype, at::IntArrayRef sizes, bool whole) {
  return !t || fits(*t, x, dtype, sizes, whole);
}
// x's own form, and a state that may be written in place
bool fits_step(const Tensor& x, const Tensor& state) {
  return x.dim() == 2 && x.is_cuda() && x.numel() && x.numel() < (1LL << 31) &&
         (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat) &&
         (x.size(1) == 1 || x.stride(1) == 1) &&
         !(at::GradMode::is_enabled() && state.requires_grad());
}

// The step of operands that its launch takes as they are, checked here once and not in
// Python (a step of one sequence: 17 -> 6.3 us, its kernel takes 3.0); no output for others,
// which go through ssm_step after Python's checks.
Opt ssm_step_direct(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                    const Tensor& C, const Tensor& state, const Opt& D, const Opt& z,
                    const Opt& bias, bool softplus) {
  if (!fits_step(x, state) || A.dim() != 2 || (B.dim() != 2 && B.dim() != 3)) return {};
  const auto t = x.scalar_type();
  const int64_t b = x.size(0), e = x.size(1), n = A.size(1), g = B.dim() == 3 ? B.size(1) : 1;
  const auto bc = B.dim() == 3 ? std::vector<int64_t>{b, g, n} : std::vector<int64_t>{b, n};
  if (n < 1 || n > LZ_SSM_MAX_STATE || g < 1 || e % g || !fits(dt, x, t, {b, e}, false) ||
      !fits(A, x, at::kFloat, {e, n}, true) || !fits(B, x, t, bc, false) ||
      !fits(C, x, t, bc, false) || !fits(state, x, at::kFloat, {b, e, n}, true) ||
      !fits(D, x, at::kFloat, {e}, true) || !fits(z, x, t, {b, e}, false) ||
      !fits(bias, x, at::kFloat, {e}, true))
    return {};
  const c10::DeviceGuard guard(x.device());
  const Tensor y = at::empty({b, e}, x.options());
  lz_ssm_args a = {};
  a.x = ptr(x), a.dt = ptr(dt), a.z = z ? ptr(*z) : nullptr, a.B = ptr(B), a.C = ptr(C);
  a.A = ptr<float>(A), a.D = D ? ptr<float>(*D) : nullptr;
  a.dt_bias = bias ? ptr<float>(*bias) : nullptr;
  a.x_batch = step_of(x, 0), a.dt_batch = step_of(dt, 0), a.z_batch = z ? step_of(*z, 0) : 0;
  a.B_batch = step_of(B, 0), a.C_batch = step_of(C, 0);
  if (B.dim() == 3) a.B_group = step_of(B, 1), a.C_group = step_of(C, 1);
  a.batch = i32(b), a.channels = i32(e), a.state = i32(n), a.groups = i32(g);
  a.softplus = softplus, a.bf16 = t == at::kBFloat16;
  check(lz_ssm_decode_step(&a, ptr<float>(state), ptr(y), stream_of(x)), "lz_ssm_decode_step");
  return y;
}

// ---------------------------------------------------------------------------
// short causal convolution
// ---------------------------------------------------------------------------

struct ConvCall {
  Tensor x, w, bias;
  bool silu;
  int bf16() const { return x.scalar_type() == at::kBFloat16; }

  Tensor forward(const Tensor& state_in, const Tensor& state_out, const Tensor& lengths) const {
    Tensor y = like(x);
    if (y.numel())
      check(lz_short_conv_fwd(ptr(x), step_of(x, 0), step_of(x, 1), ptr<float>(w), ptr<float>(bias),
                            ptr(state_in), ptr(state_out), ptr<int>(lengths), ptr(y),
                            i32(x.size(0)), i32(x.size(1)), i32(x.size(2)), i32(w.size(1)), silu,
                            bf16(), stream_of(x)),
          "lz_short_conv_fwd");
    return y;
  }
};

ConvCall conv_call(const Tensor& x, const Tensor& w, const Tensor& bias, bool silu) {
  return {rows(cast(x, common({&x}))), params(w), params(bias), silu};
}

struct ConvNode : torch::autograd::Function<ConvNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opt& bias_,
                        bool silu) {
    const Tensor bias = get(bias_);
    const c10::DeviceGuard guard(x.device());
    const ConvCall c = conv_call(x, w, bias, silu);
    ctx->save_for_backward({c.x, c.w, c.bias});
    ctx->saved_data["types"] = types({&x, &w, &bias});
    ctx->saved_data["silu"] = silu;
    return c.forward({}, {}, {});
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    const ConvCall c{s[0], s[1], s[2], ctx->saved_data["silu"].toBool()};
    const c10::DeviceGuard guard(c.x.device());
    refuse_capture(c.x);
    const Tensor dy = upstream(grads[0], c.x);
    const Tensor dx = like(c.x), dw = like(c.w), dbias = like(c.bias);
    const int b = i32(c.x.size(0)), n = i32(c.x.size(1)), ch = i32(c.x.size(2)), k = i32(c.w.size(1));
    if (dy.numel()) {
      const size_t need = lz_short_conv_bwd_workspace_bytes(b, n, ch, k);
      const Tensor ws = bytes(need, c.x);
      check(lz_short_conv_bwd(ptr(c.x), step_of(c.x, 0), step_of(c.x, 1), ptr<float>(c.w),
                              ptr<float>(c.bias), ptr(dy), ptr(dx), ptr<float>(dw),
                              ptr<float>(dbias), b, n, ch, k, c.silu, c.bf16(), ptr(ws), need,
                              stream_of(c.x)),
            "lz_short_conv_bwd");
    } else {
      zero({dx, dw, dbias});
    }
    variable_list out = as_inputs({dx, dw, dbias}, ctx->saved_data["types"].toIntVector());
    out.emplace_back();
    return out;
  }
};

Tensor short_conv(const Tensor& x, const Tensor& w, const Opt& bias_, bool silu) {
  const Tensor bias = get(bias_);
  if (any_grad({&x, &w, &bias})) return ConvNode::apply(x, w, bias_, silu);
  const c10::DeviceGuard guard(x.device());
  return conv_call(x, w, bias, silu).forward({}, {}, {});
}

std::tuple<Tensor, Tensor> short_conv_prefill(const Tensor& x, const Tensor& w, const Opt& bias,
                                              bool silu, const Opt& state, const Opt& lengths_) {
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(x.device());
  const ConvCall c = conv_call(x, w, get(bias), silu);
  const Tensor in = state ? as(*state, c.x.scalar_type()) : Tensor();
  const Tensor lengths = int_lengths(lengths_, x.size(1));
  const auto options = c.x.options().memory_format(at::MemoryFormat::Contiguous);
  Tensor out = at::empty({x.size(0), w.size(1) - 1, x.size(2)}, options);
  const Tensor y = c.forward(in, out, lengths);
  return {y, out};
}

// x [B, 1, C], state [B, K - 1, C] of x's type, moved up in place
Tensor short_conv_step(const Tensor& x, const Tensor& w, const Tensor& state, const Opt& bias,
                       bool silu) {
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(x.device());
  const ConvCall c = conv_call(x, w, get(bias), silu);
  const Tensor y = like(c.x);
  if (y.numel())
    check(lz_short_conv_decode_step(ptr(c.x), step_of(c.x, 0), ptr<float>(c.w), ptr<float>(c.bias),
                                  ptr(state), ptr(y), i32(x.size(0)), i32(x.size(2)),
                                  i32(c.w.size(1)), silu, c.bf16(), stream_of(x)),
        "lz_short_conv_decode_step");
  return y;
}

// as ssm_step_direct
Opt short_conv_step_direct(const Tensor& x, const Tensor& w, const Tensor& state, const Opt& bias,
                           bool silu) {
  if (!fits_step(x, state) || w.dim() != 2) return {};
  const int64_t b = x.size(0), c = x.size(1), k = w.size(1);
  if (k < 1 || k > LZ_CONV_MAX_TAPS || !fits(w, x, at::kFloat, {c, k}, true) ||
      !fits(state, x, x.scalar_type(), {b, k - 1, c}, true) || !fits(bias, x, at::kFloat, {c}, true))
    return {};
  const c10::DeviceGuard guard(x.device());
  const Tensor y = at::empty({b, c}, x.options());
  check(lz_short_conv_decode_step(ptr(x), step_of(x, 0), ptr<float>(w),
                                  bias ? ptr<float>(*bias) : nullptr, ptr(state), ptr(y), i32(b),
                                  i32(c), i32(k), silu, x.scalar_type() == at::kBFloat16,
                                  stream_of(x)),
        "lz_short_conv_decode_step");
  return y;
}

// ---------------------------------------------------------------------------
// group norm
// ---------------------------------------------------------------------------

// x, gate [B, L, G, W]
struct NormCall {
  Tensor x, w, bias, gate;
  bool silu;
  double eps;

  lz_group_norm_args args() const {
    lz_group_norm_args a = {};
    a.x = ptr(x), a.gate = ptr(gate), a.weight = ptr<float>(w), a.bias = ptr<float>(bias);
    a.x_batch = step_of(x, 0), a.x_token = step_of(x, 1), a.x_group = step_of(x, 2);
    a.gate_batch = step_of(gate, 0), a.gate_token = step_of(gate, 1), a.gate_group = step_of(gate, 2);
    a.batch = i32(x.size(0)), a.length = i32(x.size(1)), a.groups = i32(x.size(2));
    a.width = i32(x.size(3)), a.silu = silu, a.bf16 = x.scalar_type() == at::kBFloat16;
    a.eps = static_cast<float>(eps);
    return a;
  }

  Tensor forward() const {
    Tensor y = like(x);
    if (!y.numel()) return y;
    const lz_group_norm_args a = args();
    check(lz_group_norm_fwd(&a, ptr(y), stream_of(x)), "lz_group_norm_fwd");
    return y;
  }
};

NormCall norm_call(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& gate,
                   bool silu, double eps) {
  const auto t = common({&x, &gate});
  const int64_t any = std::numeric_limits<int64_t>::max();
  return {rows(cast(x, t), any), params(w), params(bias), rows(cast(gate, t), any), silu, eps};
}

struct NormNode : torch::autograd::Function<NormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Opt& w_, const Opt& bias_,
                        const Opt& gate_, bool silu, double eps) {
    const Tensor w = get(w_), bias = get(bias_), gate = get(gate_);
    const c10::DeviceGuard guard(x.device());
    const NormCall c = norm_call(x, w, bias, gate, silu, eps);
    ctx->save_for_backward({c.x, c.w, c.bias, c.gate});
    ctx->saved_data["types"] = types({&x, &w, &bias, &gate});
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["eps"] = eps;
    return c.forward().to(x.scalar_type());
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    const NormCall c{s[0], s[1], s[2], s[3], ctx->saved_data["silu"].toBool(),
                     ctx->saved_data["eps"].toDouble()};
    const c10::DeviceGuard guard(c.x.device());
    refuse_capture(c.x);
    const lz_group_norm_args a = c.args();
    const Tensor dy = upstream(grads[0], c.x);
    const Tensor dx = like(c.x), dgate = like(c.gate), dw = like(c.w),
                 dbias = like(c.bias);
    if (dy.numel()) {
      const size_t need =
          dw.defined() || dbias.defined()
              ? lz_group_norm_bwd_workspace_bytes(a.batch, a.length, a.groups, a.width)
              : 0;
      const Tensor ws = bytes(need ? need : 1, c.x);
      check(lz_group_norm_bwd(&a, ptr(dy), ptr(dx), ptr(dgate), ptr<float>(dw), ptr<float>(dbias),
                              ptr(ws), need, stream_of(c.x)),
            "lz_group_norm_bwd");
    } else {
      zero({dx, dgate, dw, dbias});
    }
    variable_list out = as_inputs({dx, dw, dbias, dgate}, ctx->saved_data["types"].toIntVector());
    out.emplace_back();
    out.emplace_back();
    return out;
  }
};

Tensor group_norm(const Tensor& x, const Opt& w_, const Opt& bias_, const Opt& gate_, bool silu,
                  double eps) {
  const Tensor w = get(w_), bias = get(bias_), gate = get(gate_);
  if (any_grad({&x, &w, &bias, &gate})) return NormNode::apply(x, w_, bias_, gate_, silu, eps);
  const c10::DeviceGuard guard(x.device());
  return norm_call(x, w, bias, gate, silu, eps).forward().to(x.scalar_type());
}

}  // namespace

void bind_mixers(py::module_& m) {
  const auto nogil = py::call_guard<py::gil_scoped_release>();
  m.def("ssm", &ssm, nogil);
  m.def("ssm_prefill", &ssm_prefill, nogil);
  m.def("ssm_step", &ssm_step, nogil);
  m.def("ssm_step_direct", &ssm_step_direct, nogil);
  m.def("short_conv_step_direct", &short_conv_step_direct, nogil);
  m.def("short_conv", &short_conv, nogil);
  m.def("short_conv_prefill", &short_conv_prefill, nogil);
  m.def("short_conv_step", &short_conv_step, nogil);
  m.def("group_norm", &group_norm, nogil);
  m.attr("SSM_MAX_STATE") = LZ_SSM_MAX_STATE;
  m.attr("CONV_MAX_TAPS") = LZ_CONV_MAX_TAPS;
  m.attr("NORM_MAX_WIDTH") = LZ_NORM_MAX_WIDTH;
}
