// torch.ops.paraconv2d_b200: the sequence operators (dropout, causal
// convolution, state space scan) on top of the C ABI of libpc2d_sm100.so.
//
// As for the other ops of the package: CUDA dispatch key only, every invalid
// call raises, non-contiguous inputs are made contiguous (and a view that
// starts off a 16-byte boundary is copied), work runs on torch's current
// stream of the tensors' device, scratch comes from torch's caching allocator.
// A state that a step moves on in place is never copied: it has to be
// contiguous.
//
// The gradients are registered here as well (Autograd key): a training step of
// a small layer is bound by the host, and going through Python functions took
// it about twice as long.  The backward passes are differentiable once.  The
// Autograd kernels go on through the dispatcher (0.3 us a call), as whatever
// stands in between has to see the calls.
#include "pc2d_op_common.h"

namespace {

using namespace pc2d_ops;

// ------------------------------------------------------------------- dropout

Tensor dropout_cuda(const Tensor &input_, const Tensor &key_, double p, const OptTensor &residual_) {
  const Call call{"paraconv2d_b200.dropout", input_.device()};
  const int dt = seq_dtype_code(input_, call.what, true);
  const c10::cuda::CUDAGuard guard(input_.device());
  const Tensor input = dense(input_);
  const Tensor key = call.need(key_, "key", at::kLong, {2});
  const Tensor residual = call.maybe(residual_, "residual", input.scalar_type(), input.sizes());
  Tensor out = at::empty(input.sizes(), input.options());
  check_status(pc2d_dropout(dt, ptr(input), ptr(residual), ptr<int64_t>(key), p, input.numel(), ptr(out), stream_now()),
               call.what);
  return out;
}

Tensor dropout_next_key_cuda(Tensor state) {
  const Call call{"paraconv2d_b200.dropout_next_key", state.device()};
  const c10::cuda::CUDAGuard guard(state.device());
  call.in_place(state, "state", at::kLong, {2});
  Tensor key = at::empty({2}, state.options());
  check_status(pc2d_dropout_next_key(ptr<int64_t>(state), ptr<int64_t>(key), stream_now()), call.what);
  changed(state);
  return key;
}

// -------------------------------------------------------- causal convolution

struct ConvCall {
  Call call;
  int dt, wdt, batch, channels, length, taps;
  Tensor input, weight, bias, initial, lengths;
};

ConvCall conv_call(const char *what, const Tensor &input, const Tensor &weight, const OptTensor &bias,
                   const OptTensor &initial, const OptTensor &lengths) {
  ConvCall c{{what, input.device()}};
  c.dt = seq_dtype_code(input, what);
  TORCH_CHECK(input.dim() == 3, what, ": input must be [batch, channels, length], got ", input.sizes());
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) == input.size(1), what, ": weight must be [", input.size(1),
              ", taps], got ", weight.sizes());
  c.batch = as_int(input.size(0), what, "batch");
  c.channels = as_int(input.size(1), what, "channels");
  c.length = as_int(input.size(2), what, "length");
  c.taps = as_int(weight.size(1), what, "taps");
  c.wdt = seq_dtype_code(weight, what);
  c.input = dense(input);
  c.weight = c.call.need(weight, "weight", weight.scalar_type(), weight.sizes());
  c.bias = c.call.maybe(bias, "bias", weight.scalar_type(), {c.channels});
  c.initial = c.call.maybe(initial, "initial_state", input.scalar_type(), {c.batch, c.channels, c.taps - 1});
  c.lengths = c.call.maybe(lengths, "lengths", at::kInt, {c.batch});
  return c;
}

std::vector<Tensor> causal_conv_forward_cuda(const Tensor &input, const Tensor &weight, const OptTensor &bias,
                                             const OptTensor &initial, const OptTensor &lengths, bool silu,
                                             bool final_state) {
  const c10::cuda::CUDAGuard guard(input.device());
  const ConvCall c = conv_call("paraconv2d_b200.causal_conv_forward", input, weight, bias, initial, lengths);
  const auto opts = c.input.options();
  std::vector<Tensor> outs{at::empty({c.batch, c.channels, c.length}, opts)};
  if (final_state) outs.push_back(at::empty({c.batch, c.channels, c.taps - 1}, opts));
  check_status(pc2d_causal_conv_forward(c.dt, c.wdt, ptr(c.input), ptr(c.weight), ptr(c.bias), ptr(c.initial),
                                        ptr<int>(c.lengths), c.batch, c.channels, c.length, c.taps, silu, ptr(outs[0]),
                                        final_state ? ptr(outs[1]) : nullptr, stream_now()),
               c.call.what);
  return outs;
}

std::vector<Tensor> causal_conv_backward_cuda(const Tensor &grad_, const OptTensor &grad_final_, const Tensor &input,
                                              const Tensor &weight, const OptTensor &bias, const OptTensor &initial,
                                              const OptTensor &lengths, bool silu) {
  const c10::cuda::CUDAGuard guard(input.device());
  const ConvCall c = conv_call("paraconv2d_b200.causal_conv_backward", input, weight, bias, initial, lengths);
  const Tensor grad = c.call.need(grad_, "grad", input.scalar_type(), c.input.sizes());
  const Tensor grad_final = c.call.maybe(grad_final_, "grad_final", input.scalar_type(),
                                         {c.batch, c.channels, c.taps - 1});
  const auto opts = c.input.options();
  Tensor dx = at::empty({c.batch, c.channels, c.length}, opts);
  Tensor dw = at::empty({c.channels, c.taps}, c.weight.options());
  Tensor db = c.bias.defined() ? at::empty({c.channels}, c.weight.options()) : at::empty({0}, c.weight.options());
  Tensor di = c.initial.defined() ? at::empty({c.batch, c.channels, c.taps - 1}, opts) : at::empty({0}, opts);
  const size_t bytes = pc2d_causal_conv_backward_workspace_size(c.batch, c.channels, c.length, c.taps);
  const Tensor ws = workspace(bytes, c.input);
  check_status(pc2d_causal_conv_backward(c.dt, c.wdt, ptr(grad), ptr(grad_final), ptr(c.input), ptr(c.weight),
                                         ptr(c.bias), ptr(c.initial), ptr<int>(c.lengths), c.batch, c.channels,
                                         c.length, c.taps, silu, ptr(dx), ptr(dw), c.bias.defined() ? ptr(db) : nullptr,
                                         c.initial.defined() ? ptr(di) : nullptr, ptr(ws), bytes, stream_now()),
               c.call.what);
  return {dx, dw, db, di};
}

Tensor causal_conv_step_cuda(const Tensor &input_, const Tensor &state, const Tensor &weight_, const OptTensor &bias_,
                             const OptTensor &slots_, bool silu) {
  const Call call{"paraconv2d_b200.causal_conv_step", input_.device()};
  const c10::cuda::CUDAGuard guard(input_.device());
  const int dt = seq_dtype_code(input_, call.what), wdt = seq_dtype_code(weight_, call.what);
  TORCH_CHECK(input_.dim() == 2, call.what, ": input must be [batch, channels], got ", input_.sizes());
  const int batch = as_int(input_.size(0), call.what, "batch"), channels = as_int(input_.size(1), call.what, "channels");
  TORCH_CHECK(weight_.dim() == 2 && weight_.size(0) == channels && weight_.size(1) >= 1, call.what, ": weight must be [",
              channels, ", taps], got ", weight_.sizes());
  const int taps = as_int(weight_.size(1), call.what, "taps");
  TORCH_CHECK(state.dim() == 3, call.what, ": state must be [places, ", channels, ", ", taps - 1, "], got ",
              state.sizes());
  const int places = as_int(state.size(0), call.what, "places");
  call.in_place(state, "state", input_.scalar_type(), {places, channels, taps - 1});
  const Tensor input = dense(input_);
  const Tensor weight = call.need(weight_, "weight", weight_.scalar_type(), weight_.sizes());
  const Tensor bias = call.maybe(bias_, "bias", weight_.scalar_type(), {channels});
  const Tensor slots = call.maybe(slots_, "slots", at::kInt, {batch});
  call.apart(state, {&input, &weight, &bias, &slots});
  Tensor out = at::empty({batch, channels}, input.options());
  check_status(pc2d_causal_conv_step(dt, wdt, ptr(input), ptr(state), ptr(weight), ptr(bias), ptr<int>(slots), batch,
                                     places, channels, taps, silu, ptr(out), stream_now()),
               call.what);
  changed(state);
  return out;
}

// ---------------------------------------------------------- state space scan

struct ScanCall {
  Call call;
  int dt, batch, channels, length, states, groups;
  Tensor u, delta, A, B, C, skip, z, bias, lengths;
};

ScanCall scan_call(const char *what, const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &B,
                   const Tensor &C, const OptTensor &skip, const OptTensor &z, const OptTensor &bias,
                   const OptTensor &lengths) {
  ScanCall c{{what, u.device()}};
  const auto type = u.scalar_type();
  c.dt = seq_dtype_code(u, what);
  TORCH_CHECK(u.dim() == 3, what, ": u must be [batch, channels, length], got ", u.sizes());
  c.batch = as_int(u.size(0), what, "batch");
  c.channels = as_int(u.size(1), what, "channels");
  c.length = as_int(u.size(2), what, "length");
  TORCH_CHECK(A.dim() == 2 && A.size(0) == c.channels, what, ": A must be [", c.channels, ", states], got ", A.sizes());
  c.states = as_int(A.size(1), what, "states");
  TORCH_CHECK(B.dim() == 4, what, ": B must be [batch, groups, states, length], got ", B.sizes());
  c.groups = as_int(B.size(1), what, "groups");
  c.u = dense(u);
  c.delta = c.call.need(delta, "delta", type, u.sizes());
  c.A = c.call.need(A, "A", at::kFloat, A.sizes());
  c.B = c.call.need(B, "B", type, {c.batch, c.groups, c.states, c.length});
  c.C = c.call.need(C, "C", type, {c.batch, c.groups, c.states, c.length});
  c.skip = c.call.maybe(skip, "D", at::kFloat, {c.channels});
  c.z = c.call.maybe(z, "z", type, u.sizes());
  c.bias = c.call.maybe(bias, "delta_bias", at::kFloat, {c.channels});
  c.lengths = c.call.maybe(lengths, "lengths", at::kInt, {c.batch});
  return c;
}

std::vector<Tensor> ssm_scan_forward_cuda(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &B,
                                          const Tensor &C, const OptTensor &D, const OptTensor &z,
                                          const OptTensor &delta_bias, const OptTensor &initial_,
                                          const OptTensor &lengths, bool delta_softplus, bool final_state,
                                          bool checkpoints) {
  const c10::cuda::CUDAGuard guard(u.device());
  const ScanCall c = scan_call("paraconv2d_b200.ssm_scan_forward", u, delta, A, B, C, D, z, delta_bias, lengths);
  const Tensor initial = c.call.maybe(initial_, "initial_state", at::kFloat, {c.batch, c.channels, c.states});
  Tensor out = at::empty({c.batch, c.channels, c.length}, c.u.options());
  Tensor last = at::empty(final_state ? at::IntArrayRef({c.batch, c.channels, c.states}) : at::IntArrayRef({0}),
                          c.A.options());
  const size_t ck = checkpoints ? pc2d_ssm_scan_checkpoint_size(c.batch, c.channels, c.length, c.states) : 0;
  Tensor kept = at::empty({(int64_t)(ck / 4)}, c.A.options());
  const size_t bytes = pc2d_ssm_scan_forward_workspace_size(c.batch, c.channels, c.length, c.states, c.groups);
  const Tensor ws = workspace(bytes, c.u);
  check_status(
      pc2d_ssm_scan_forward(c.dt, ptr(c.u), ptr(c.delta), ptr<float>(c.A), ptr(c.B), ptr(c.C), ptr<float>(c.skip),
                            ptr(c.z), ptr<float>(c.bias), ptr<float>(initial), ptr<int>(c.lengths), delta_softplus,
                            c.batch, c.channels, c.length, c.states, c.groups, ptr(out),
                            final_state ? ptr<float>(last) : nullptr, ck ? ptr<float>(kept) : nullptr, ptr(ws), bytes,
                            stream_now()),
      c.call.what);
  return {out, last, kept};
}

std::vector<Tensor> ssm_scan_backward_cuda(const Tensor &grad_, const OptTensor &grad_final_, const Tensor &u,
                                           const Tensor &delta, const Tensor &A, const Tensor &B, const Tensor &C,
                                           const OptTensor &D, const OptTensor &z, const OptTensor &delta_bias,
                                           const OptTensor &lengths, const Tensor &checkpoints_, bool delta_softplus,
                                           bool initial_grad) {
  const c10::cuda::CUDAGuard guard(u.device());
  const ScanCall c = scan_call("paraconv2d_b200.ssm_scan_backward", u, delta, A, B, C, D, z, delta_bias, lengths);
  const Tensor grad = c.call.need(grad_, "grad", u.scalar_type(), c.u.sizes());
  const Tensor grad_final = c.call.maybe(grad_final_, "grad_final", at::kFloat, {c.batch, c.channels, c.states});
  const int64_t ck = (int64_t)(pc2d_ssm_scan_checkpoint_size(c.batch, c.channels, c.length, c.states) / 4);
  const Tensor kept = c.call.need(checkpoints_, "checkpoints", at::kFloat, {ck});
  const auto opts = c.u.options(), fopts = c.A.options();
  auto like = [](const Tensor &t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); };
  Tensor du = like(c.u), dd = like(c.delta), dA = like(c.A), dB = like(c.B), dC = like(c.C);
  Tensor dskip = like(c.skip), dz = like(c.z), dbias = like(c.bias);
  Tensor dinit = initial_grad ? at::empty({c.batch, c.channels, c.states}, fopts) : Tensor();
  const size_t bytes = pc2d_ssm_scan_backward_workspace_size(c.batch, c.channels, c.length, c.states, c.groups);
  const Tensor ws = workspace(bytes, c.u);
  check_status(
      pc2d_ssm_scan_backward(c.dt, ptr(grad), ptr<float>(grad_final), ptr(c.u), ptr(c.delta), ptr<float>(c.A),
                             ptr(c.B), ptr(c.C), ptr<float>(c.skip), ptr(c.z), ptr<float>(c.bias), ptr<int>(c.lengths),
                             ptr<float>(kept), delta_softplus, c.batch, c.channels, c.length, c.states, c.groups,
                             ptr(du), ptr(dd), ptr<float>(dA), ptr(dB), ptr(dC), ptr<float>(dskip), ptr(dz),
                             ptr<float>(dbias), ptr<float>(dinit), ptr(ws), bytes, stream_now()),
      c.call.what);
  auto given = [&](const Tensor &t) { return t.defined() ? t : at::empty({0}, opts); };
  return {du, dd, dA, dB, dC, given(dskip), given(dz), given(dbias), given(dinit)};
}

Tensor ssm_scan_step_cuda(const Tensor &u_, const Tensor &delta_, const Tensor &state, const Tensor &A_, const Tensor &B_,
                          const Tensor &C_, const OptTensor &D_, const OptTensor &z_, const OptTensor &bias_,
                          const OptTensor &slots_, bool delta_softplus) {
  const Call call{"paraconv2d_b200.ssm_scan_step", u_.device()};
  const c10::cuda::CUDAGuard guard(u_.device());
  const auto type = u_.scalar_type();
  const int dt = seq_dtype_code(u_, call.what);
  TORCH_CHECK(u_.dim() == 2, call.what, ": u must be [batch, channels], got ", u_.sizes());
  const int batch = as_int(u_.size(0), call.what, "batch"), channels = as_int(u_.size(1), call.what, "channels");
  TORCH_CHECK(A_.dim() == 2 && A_.size(0) == channels, call.what, ": A must be [", channels, ", states], got ",
              A_.sizes());
  const int states = as_int(A_.size(1), call.what, "states");
  TORCH_CHECK(B_.dim() == 3, call.what, ": B must be [batch, groups, states], got ", B_.sizes());
  const int groups = as_int(B_.size(1), call.what, "groups");
  TORCH_CHECK(state.dim() == 3, call.what, ": state must be [places, ", channels, ", ", states, "], got ",
              state.sizes());
  const int places = as_int(state.size(0), call.what, "places");
  call.in_place(state, "state", at::kFloat, {places, channels, states});
  const Tensor u = dense(u_);
  const Tensor delta = call.need(delta_, "delta", type, u.sizes()), A = call.need(A_, "A", at::kFloat, A_.sizes());
  const Tensor B = call.need(B_, "B", type, {batch, groups, states}), C = call.need(C_, "C", type, {batch, groups, states});
  const Tensor skip = call.maybe(D_, "D", at::kFloat, {channels}), z = call.maybe(z_, "z", type, u.sizes());
  const Tensor bias = call.maybe(bias_, "delta_bias", at::kFloat, {channels});
  const Tensor slots = call.maybe(slots_, "slots", at::kInt, {batch});
  call.apart(state, {&u, &delta, &A, &B, &C, &skip, &z, &bias, &slots});
  Tensor out = at::empty({batch, channels}, u.options());
  check_status(pc2d_ssm_scan_step(dt, ptr(u), ptr(delta), ptr<float>(state), ptr<float>(A), ptr(B), ptr(C),
                                  ptr<float>(skip), ptr(z), ptr<float>(bias), ptr<int>(slots), delta_softplus, batch,
                                  places, channels, states, groups, ptr(out), stream_now()),
               call.what);
  changed(state);
  return out;
}

// ------------------------------------------------------------------ autograd

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &input, const Tensor &key, double p,
                        const OptTensor &residual) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({key});
    ctx->saved_data["p"] = p;
    ctx->saved_data["input"] = input.requires_grad();
    ctx->saved_data["residual"] = residual.has_value() && residual->defined() && residual->requires_grad();
    return PC2D_BELOW(dropout).call(input, key, p, residual);
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const Tensor key = ctx->get_saved_variables()[0];
    // (linear: its gradient is the same operation, which may be differentiated again)
    // (through Autograd again)
    Tensor dx;
    if (ctx->saved_data["input"].toBool())
      dx = PC2D_BELOW(dropout).call(grads[0], key, ctx->saved_data["p"].toDouble(), OptTensor());
    return {dx, Tensor(), Tensor(), ctx->saved_data["residual"].toBool() ? grads[0] : Tensor()};
  }
};

Tensor dropout_autograd(const Tensor &input, const Tensor &key, double p, const OptTensor &residual) {
  no_forward_mode("dropout", {&input}, {&residual});
  check_cuda(input, "dropout");
  if (needs_grad({&input}, {&residual})) return DropoutFunction::apply(input, key, p, residual);
  at::AutoDispatchBelowADInplaceOrView below;
  return PC2D_BELOW(dropout).call(input, key, p, residual);
}

struct ConvFunction : torch::autograd::Function<ConvFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &input, const Tensor &weight, const OptTensor &bias,
                               const OptTensor &initial, const OptTensor &lengths, bool silu, bool final_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor x = input.contiguous();
    auto outs = PC2D_BELOW(causal_conv_forward).call(x, weight, bias, initial, lengths, silu, final_state);
    ctx->save_for_backward({x, weight, bias.value_or(Tensor()), initial.value_or(Tensor()), lengths.value_or(Tensor())});
    ctx->saved_data["silu"] = silu;
    ctx->set_materialize_grads(false);
    return outs;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    return once("causal_conv", [&]() -> variable_list {
      const auto saved = ctx->get_saved_variables();
      const Tensor grad = grads[0].defined() ? grads[0] : at::zeros_like(saved[0]);
      const auto g = PC2D_BELOW(causal_conv_backward)
                         .call(grad, grads.size() > 1 ? optional_of(grads[1]) : OptTensor(), saved[0], saved[1],
                               optional_of(saved[2]), optional_of(saved[3]), optional_of(saved[4]),
                               ctx->saved_data["silu"].toBool());
      return {g[0], g[1], saved[2].defined() ? g[2] : Tensor(), saved[3].defined() ? g[3] : Tensor(),
              Tensor(), Tensor(), Tensor()};
    });
  }
};

std::vector<Tensor> causal_conv_forward_autograd(const Tensor &input, const Tensor &weight, const OptTensor &bias,
                                                 const OptTensor &initial, const OptTensor &lengths, bool silu,
                                                 bool final_state) {
  no_forward_mode("causal_conv", {&input, &weight}, {&bias, &initial});
  check_cuda(input, "causal_conv");
  if (needs_grad({&input, &weight}, {&bias, &initial}))
    return ConvFunction::apply(input, weight, bias, initial, lengths, silu, final_state);
  at::AutoDispatchBelowADInplaceOrView below;
  return PC2D_BELOW(causal_conv_forward).call(input, weight, bias, initial, lengths, silu, final_state);
}

struct ScanFunction : torch::autograd::Function<ScanFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &u_, const Tensor &delta_, const Tensor &A_,
                               const Tensor &B_, const Tensor &C_, const OptTensor &D, const OptTensor &z_,
                               const OptTensor &delta_bias, const OptTensor &initial, const OptTensor &lengths,
                               bool delta_softplus, bool final_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor u = u_.contiguous(), delta = delta_.contiguous(), A = A_.contiguous(), B = B_.contiguous(),
                 C = C_.contiguous();
    const Tensor z = z_.has_value() && z_->defined() ? z_->contiguous() : Tensor();
    auto outs = PC2D_BELOW(ssm_scan_forward).call(u, delta, A, B, C, D, optional_of(z), delta_bias, initial, lengths,
                                                  delta_softplus, final_state, true);
    ctx->save_for_backward({u, delta, A, B, C, D.value_or(Tensor()), z, delta_bias.value_or(Tensor()),
                            lengths.value_or(Tensor()), outs[2]});
    ctx->saved_data["softplus"] = delta_softplus;
    ctx->saved_data["initial"] = initial.has_value() && initial->defined() && initial->requires_grad();
    ctx->set_materialize_grads(false);
    outs.pop_back();
    if (!final_state) outs.pop_back();
    return outs;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    return once("ssm_scan", [&]() -> variable_list {
      const auto s = ctx->get_saved_variables();
      const Tensor grad = grads[0].defined() ? grads[0] : at::zeros_like(s[0]);
      const bool initial = ctx->saved_data["initial"].toBool();
      const auto g = PC2D_BELOW(ssm_scan_backward)
                         .call(grad, grads.size() > 1 ? optional_of(grads[1]) : OptTensor(), s[0], s[1], s[2], s[3],
                               s[4], optional_of(s[5]), optional_of(s[6]), optional_of(s[7]), optional_of(s[8]), s[9],
                               ctx->saved_data["softplus"].toBool(), initial);
      return {g[0], g[1], g[2], g[3], g[4], s[5].defined() ? g[5] : Tensor(), s[6].defined() ? g[6] : Tensor(),
              s[7].defined() ? g[7] : Tensor(), initial ? g[8] : Tensor(), Tensor(), Tensor(), Tensor()};
    });
  }
};

// With gradients the checkpoints are the graph's own: the third result is empty.
std::vector<Tensor> ssm_scan_forward_autograd(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &B,
                                              const Tensor &C, const OptTensor &D, const OptTensor &z,
                                              const OptTensor &delta_bias, const OptTensor &initial,
                                              const OptTensor &lengths, bool delta_softplus, bool final_state,
                                              bool checkpoints) {
  no_forward_mode("ssm_scan", {&u, &delta, &A, &B, &C}, {&D, &z, &delta_bias, &initial});
  check_cuda(u, "ssm_scan");
  if (needs_grad({&u, &delta, &A, &B, &C}, {&D, &z, &delta_bias, &initial})) {
    auto outs = ScanFunction::apply(u, delta, A, B, C, D, z, delta_bias, initial, lengths, delta_softplus, final_state);
    while (outs.size() < 3) outs.push_back(at::empty({0}, A.options()));
    return outs;
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return PC2D_BELOW(ssm_scan_forward).call(u, delta, A, B, C, D, z, delta_bias, initial, lengths, delta_softplus,
                                           final_state, checkpoints);
}

Tensor causal_conv_step_autograd(const Tensor &input, const Tensor &state, const Tensor &weight, const OptTensor &bias,
                                 const OptTensor &slots, bool silu) {
  no_forward_mode("causal_conv_step", {&input, &state, &weight}, {&bias});
  no_step_grad("causal_conv_step", needs_grad({&input, &state, &weight}, {&bias}));
  check_cuda(input, "causal_conv_step");
  at::AutoDispatchBelowADInplaceOrView below;
  return PC2D_BELOW(causal_conv_step).call(input, state, weight, bias, slots, silu);
}

Tensor ssm_scan_step_autograd(const Tensor &u, const Tensor &delta, const Tensor &state, const Tensor &A, const Tensor &B,
                              const Tensor &C, const OptTensor &D, const OptTensor &z, const OptTensor &delta_bias,
                              const OptTensor &slots, bool delta_softplus) {
  no_forward_mode("ssm_scan_step", {&u, &delta, &state, &A, &B, &C}, {&D, &z, &delta_bias});
  no_step_grad("ssm_scan_step", needs_grad({&u, &delta, &state, &A, &B, &C}, {&D, &z, &delta_bias}));
  check_cuda(u, "ssm_scan_step");
  at::AutoDispatchBelowADInplaceOrView below;
  return PC2D_BELOW(ssm_scan_step).call(u, delta, state, A, B, C, D, z, delta_bias, slots, delta_softplus);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(paraconv2d_b200, m) {
  m.def("dropout(Tensor input, Tensor key, float p, Tensor? residual) -> Tensor");
  m.def("dropout_next_key(Tensor(a!) state) -> Tensor");
  m.def(
      "causal_conv_forward(Tensor input, Tensor weight, Tensor? bias, Tensor? initial_state, Tensor? lengths, bool "
      "silu, bool final_state) -> Tensor[]");
  m.def(
      "causal_conv_backward(Tensor grad, Tensor? grad_final, Tensor input, Tensor weight, Tensor? bias, Tensor? "
      "initial_state, Tensor? lengths, bool silu) -> Tensor[]");
  m.def(
      "causal_conv_step(Tensor input, Tensor(a!) state, Tensor weight, Tensor? bias, Tensor? slots, bool silu) -> "
      "Tensor");
  m.def(
      "ssm_scan_forward(Tensor u, Tensor delta, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? "
      "delta_bias, Tensor? initial_state, Tensor? lengths, bool delta_softplus, bool final_state, bool checkpoints) -> "
      "Tensor[]");
  m.def(
      "ssm_scan_backward(Tensor grad, Tensor? grad_final, Tensor u, Tensor delta, Tensor A, Tensor B, Tensor C, "
      "Tensor? D, Tensor? z, Tensor? delta_bias, Tensor? lengths, Tensor checkpoints, bool delta_softplus, bool "
      "initial_grad) -> Tensor[]");
  m.def(
      "ssm_scan_step(Tensor u, Tensor delta, Tensor(a!) state, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, "
      "Tensor? delta_bias, Tensor? slots, bool delta_softplus) -> Tensor");
}

TORCH_LIBRARY_IMPL(paraconv2d_b200, CUDA, m) {
  m.impl("dropout", dropout_cuda);
  m.impl("dropout_next_key", dropout_next_key_cuda);
  m.impl("causal_conv_forward", causal_conv_forward_cuda);
  m.impl("causal_conv_backward", causal_conv_backward_cuda);
  m.impl("causal_conv_step", causal_conv_step_cuda);
  m.impl("ssm_scan_forward", ssm_scan_forward_cuda);
  m.impl("ssm_scan_backward", ssm_scan_backward_cuda);
  m.impl("ssm_scan_step", ssm_scan_step_cuda);
}

TORCH_LIBRARY_IMPL(paraconv2d_b200, Autograd, m) {
  m.impl("dropout", dropout_autograd);
  m.impl("causal_conv_forward", causal_conv_forward_autograd);
  m.impl("causal_conv_step", causal_conv_step_autograd);
  m.impl("ssm_scan_forward", ssm_scan_forward_autograd);
  m.impl("ssm_scan_step", ssm_scan_step_autograd);
}
