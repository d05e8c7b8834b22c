// torch.ops.paraconv2d_b200: group norm, linear attention and the AdamW step
// over many tensors, on top of the C ABI of libpc2d_sm100.so.  Argument checks, streams, scratch
// and gradients as for the sequence operators.
#include <algorithm>

#include "pc2d_op_common.h"

namespace {

using namespace pc2d_ops;

// Whether two tensors of the same sizes have their elements in the same order.
bool same_layout(const Tensor &a, const Tensor &b) {
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// Byte ranges of one call: one that is written may share nothing with another.
struct Ranges {
  struct Range {
    uintptr_t first, last;
    bool written;
  };
  std::vector<Range> all;
  void add(const Tensor &t, bool written) {
    if (!t.defined() || !t.numel()) return;
    const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
    all.push_back({at, at + t.nbytes(), written});
  }
  void check(const char *what) {
    std::sort(all.begin(), all.end(), [](const Range &a, const Range &b) { return a.first < b.first; });
    uintptr_t read_to = 0, written_to = 0;
    for (const Range &r : all) {
      TORCH_CHECK(r.first >= written_to && (!r.written || r.first >= read_to), what,
                  ": a tensor that is updated in place shares memory with another one of the call");
      auto &to = r.written ? written_to : read_to;
      to = std::max(to, r.last);
    }
  }
};

// --------------------------------------------------------------------- AdamW

void adamw_step_cuda(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs, at::TensorList exp_avg_sqs,
                     at::TensorList masters, at::TensorList scales, const Tensor &step, const OptTensor &lr_tensor,
                     double lr, double beta1, double beta2, double eps, double weight_decay,
                     const OptTensor &grad_scale_, at::IntArrayRef splits, at::ArrayRef<double> factors, int64_t seed,
                     at::IntArrayRef numbers) {
  const Call call{"paraconv2d_b200.adamw_step", step.device()};
  const c10::cuda::CUDAGuard guard(step.device());
  const size_t count = params.size();
  TORCH_CHECK(grads.size() == count && exp_avgs.size() == count && exp_avg_sqs.size() == count, call.what,
              ": params, grads, exp_avgs and exp_avg_sqs must be of equal length");
  TORCH_CHECK((masters.empty() || masters.size() == count) && (scales.empty() || scales.size() == count), call.what,
              ": masters and scales must be as many as params, or none");
  TORCH_CHECK((splits.empty() && factors.empty()) || (splits.size() == count && factors.size() == 3 * count), call.what,
              ": a split and three factors for each of params, or none");
  TORCH_CHECK(numbers.empty() || numbers.size() == count, call.what, ": a number for each of params, or none");
  TORCH_CHECK(count <= INT_MAX, call.what, ": too many tensors");
  call.in_place_any(step, "step", at::kLong, {1});
  Ranges ranges;
  ranges.add(step, true);
  auto scalar = [&](const OptTensor &t, const char *name) {
    if (!t.has_value() || !t->defined()) return Tensor();
    TORCH_CHECK(t->device() == call.device && t->scalar_type() == at::kFloat && t->numel() == 1, call.what, ": ", name,
                " must be one float32 number on ", call.device);
    ranges.add(*t, false);
    return *t;
  };
  const Tensor rate = scalar(lr_tensor, "lr"), grad_scale = scalar(grad_scale_, "grad_scale");
  const bool bits8 = count && exp_avgs[0].scalar_type() == at::kByte;
  TORCH_CHECK(bits8 ? scales.size() == count : scales.empty(), call.what, ": scales go with moments of 8 bits (uint8)");
  std::vector<pc2d_adamw_tensor> items(count);
  std::vector<Tensor> copies;  // gradients brought into their parameters' order
  for (size_t i = 0; i < count; ++i) {
    const Tensor &p = params[i], &m = exp_avgs[i], &v = exp_avg_sqs[i];
    auto like = [&](const Tensor &t, const char *name, at::ScalarType type) {
      TORCH_CHECK(t.device() == call.device && t.scalar_type() == type && t.sizes() == p.sizes(), call.what, ": ", name,
                  "[", i, "] must be ", type, " ", p.sizes(), " on ", call.device, ", got ", t.scalar_type(), " ",
                  t.sizes(), " on ", t.device());
    };
    auto ordered = [&](const Tensor &t, const char *name) {
      TORCH_CHECK(same_layout(p, t), call.what, ": ", name, "[", i, "] must have the strides of its parameter");
      ranges.add(t, true);
    };
    pc2d_adamw_tensor &it = items[i];
    it = {};
    like(p, "params", p.scalar_type());
    it.dtype = seq_dtype_code(p, call.what);
    TORCH_CHECK(p.is_non_overlapping_and_dense(), call.what, ": params[", i, "] is updated in place and must be dense");
    ranges.add(p, true);
    it.param = p.data_ptr();
    it.n = p.numel();
    Tensor g = grads[i];
    TORCH_CHECK(g.scalar_type() == p.scalar_type() || g.scalar_type() == at::kFloat, call.what, ": grads[", i,
                "] must be of the parameter's type or float32, got ", g.scalar_type());
    like(g, "grads", g.scalar_type());
    if (!same_layout(p, g) || !g.is_non_overlapping_and_dense()) {
      g = at::empty_strided(p.sizes(), p.strides(), g.options()).copy_(g);
      copies.push_back(g);
    }
    ranges.add(g, false);
    it.grad_dtype = seq_dtype_code(g, call.what);
    it.grad = g.data_ptr();
    if (bits8) {
      const int64_t blocks = (it.n + 255) / 256;
      call.in_place_any(m, "exp_avgs", at::kByte, {it.n});
      call.in_place_any(v, "exp_avg_sqs", at::kByte, {it.n});
      call.in_place_any(scales[i], "scales", at::kByte, {blocks, 2});
      ranges.add(m, true);
      ranges.add(v, true);
      ranges.add(scales[i], true);
      it.scales = ptr<unsigned char>(scales[i]);
    } else {
      like(m, "exp_avgs", at::kFloat);
      like(v, "exp_avg_sqs", at::kFloat);
      ordered(m, "exp_avgs");
      ordered(v, "exp_avg_sqs");
    }
    it.exp_avg = m.data_ptr();
    it.exp_avg_sq = v.data_ptr();
    if (!masters.empty() && masters[i].numel()) {
      TORCH_CHECK(p.scalar_type() != at::kFloat, call.what, ": params[", i, "] is float32 and needs no master");
      like(masters[i], "masters", at::kFloat);
      ordered(masters[i], "masters");
      it.master = ptr<float>(masters[i]);
    } else {
      TORCH_CHECK(masters.empty() || !it.n || p.scalar_type() == at::kFloat, call.what, ": masters[", i, "] is missing");
    }
    it.split = splits.empty() ? it.n : splits[i];
    it.rate_first = factors.empty() ? 1.0 : factors[3 * i];
    it.rate_rest = factors.empty() ? 1.0 : factors[3 * i + 1];
    it.decay = factors.empty() ? 1.0 : factors[3 * i + 2];
  }
  ranges.check(call.what);
  const size_t bytes = pc2d_adamw_workspace_size();
  const Tensor ws = workspace(bytes, step);
  check_status(pc2d_adamw_step_numbered(bits8 ? 8 : 32, items.data(), (int)count,
                                        numbers.empty() ? nullptr : numbers.data(), ptr<int64_t>(step), ptr<float>(rate),
                                        lr, beta1, beta2, eps, weight_decay, ptr<float>(grad_scale), seed, ptr(ws),
                                        bytes, stream_now()),
               call.what);
  changed(step);
  for (const auto &list : {params, exp_avgs, exp_avg_sqs, masters, scales})
    for (const Tensor &t : list) changed(t);
}

// (The parameters need gradients; the step is not differentiated.)
void adamw_step_autograd(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs,
                         at::TensorList exp_avg_sqs, at::TensorList masters, at::TensorList scales, const Tensor &step,
                         const OptTensor &lr_tensor, double lr, double beta1, double beta2, double eps,
                         double weight_decay, const OptTensor &grad_scale, at::IntArrayRef splits,
                         at::ArrayRef<double> factors, int64_t seed, at::IntArrayRef numbers) {
  check_cuda(step, "adamw_step");
  at::AutoDispatchBelowADInplaceOrView below;
  PC2D_BELOW(adamw_step)
      .call(params, grads, exp_avgs, exp_avg_sqs, masters, scales, step, lr_tensor, lr, beta1, beta2, eps, weight_decay,
            grad_scale, splits, factors, seed, numbers);
}

std::vector<Tensor> adamw_state_values_cuda(at::TensorList exp_avgs, at::TensorList exp_avg_sqs, at::TensorList scales,
                                            at::ScalarType dtype) {
  const size_t count = exp_avgs.size();
  TORCH_CHECK(count && exp_avg_sqs.size() == count && scales.size() == count && count <= INT_MAX,
              "paraconv2d_b200.adamw_state_values: exp_avgs, exp_avg_sqs and scales must be of equal length");
  const Call call{"paraconv2d_b200.adamw_state_values", exp_avgs[0].device()};
  const c10::cuda::CUDAGuard guard(call.device);
  TORCH_CHECK(dtype == at::kFloat || dtype == at::kBFloat16, call.what, ": float32 or bfloat16, got ", dtype);
  std::vector<pc2d_adamw_tensor> items(count);
  std::vector<Tensor> outs(2 * count);
  std::vector<void *> m(count), v(count);
  std::vector<Tensor> kept;
  for (size_t i = 0; i < count; ++i) {
    pc2d_adamw_tensor &it = items[i];
    it = {};
    it.n = exp_avgs[i].numel();
    auto given = [&](const Tensor &t, const char *name, at::IntArrayRef shape) {
      kept.push_back(call.need(t, name, at::kByte, shape));
      return kept.back().data_ptr();
    };
    it.exp_avg = given(exp_avgs[i], "exp_avgs", {it.n});
    it.exp_avg_sq = given(exp_avg_sqs[i], "exp_avg_sqs", {it.n});
    it.scales = (unsigned char *)given(scales[i], "scales", {(it.n + 255) / 256, 2});
    for (size_t k : {i, count + i}) outs[k] = at::empty({it.n}, exp_avgs[i].options().dtype(dtype));
    m[i] = outs[i].data_ptr();
    v[i] = outs[count + i].data_ptr();
  }
  check_status(pc2d_adamw_state_values(dtype == at::kFloat ? PC2D_DTYPE_F32 : PC2D_DTYPE_BF16, items.data(), (int)count,
                                       m.data(), v.data(), stream_now()),
               call.what);
  return outs;
}

// ---------------------------------------------------------------- group norm

struct NormCall {
  Call call;
  int dt, wdt, last, batch, channels, length, groups;
  Tensor input, weight, bias, lengths;
};

// Channels last: the order in which dimension 1 is the innermost one.
bool is_last(const Tensor &t) {
  if (t.dim() < 3) return false;
  int64_t stride = t.size(1);
  if (t.size(1) > 1 && t.stride(1) != 1) return false;
  for (int64_t d = t.dim() - 1; d != 1; d = d == 2 ? 0 : d - 1) {
    if (t.size(d) > 1 && t.stride(d) != stride) return false;
    stride *= t.size(d);
    if (d == 0) break;
  }
  return true;
}

NormCall norm_call(const char *what, const Tensor &input, const OptTensor &weight, const OptTensor &bias,
                   const OptTensor &lengths, int64_t groups) {
  NormCall c{{what, input.device()}};
  c.dt = seq_dtype_code(input, what);
  TORCH_CHECK(input.dim() >= 2, what, ": input must be [batch, channels, ...], got ", input.sizes());
  c.batch = as_int(input.size(0), what, "batch");
  c.channels = as_int(input.size(1), what, "channels");
  int64_t length = 1;
  for (int64_t d = 2; d < input.dim(); ++d) length *= input.size(d);
  c.length = as_int(length, what, "the number of positions");
  c.groups = as_int(groups, what, "groups");
  c.last = !input.is_contiguous() && is_last(input);
  const auto wtype = weight.has_value() && weight->defined() ? weight->scalar_type()
                     : bias.has_value() && bias->defined()   ? bias->scalar_type()
                                                             : input.scalar_type();
  TORCH_CHECK(wtype == input.scalar_type() || wtype == at::kFloat, what,
              ": weight and bias must be of the input's type or float32, got ", wtype);
  c.wdt = wtype == at::kFloat ? PC2D_DTYPE_F32 : c.dt;
  c.input = c.last ? input : input.contiguous();
  c.weight = c.call.maybe(weight, "weight", wtype, {c.channels});
  c.bias = c.call.maybe(bias, "bias", wtype, {c.channels});
  TORCH_CHECK(!(lengths.has_value() && lengths->defined()) || input.dim() == 3, what,
              ": lengths go with [batch, channels, length] only, got ", input.sizes());
  c.lengths = c.call.maybe(lengths, "lengths", at::kInt, {c.batch});
  return c;
}

// A result in the order of dimensions of the input.
Tensor norm_result(const NormCall &c) { return at::empty_strided(c.input.sizes(), c.input.strides(), c.input.options()); }

std::vector<Tensor> group_norm_forward_cuda(const Tensor &input, const OptTensor &weight, const OptTensor &bias,
                                            const OptTensor &lengths, int64_t groups, double eps, bool silu,
                                            bool keep_stats) {
  const c10::cuda::CUDAGuard guard(input.device());
  const NormCall c = norm_call("paraconv2d_b200.group_norm_forward", input, weight, bias, lengths, groups);
  Tensor out = norm_result(c);
  Tensor stats = at::empty(keep_stats ? at::IntArrayRef({c.batch, c.groups, 2}) : at::IntArrayRef({0}),
                           input.options().dtype(at::kFloat));
  const size_t bytes = pc2d_group_norm_workspace_size(c.dt, c.last, c.batch, c.channels, c.length, c.groups, 0);
  const Tensor ws = workspace(bytes, input);
  check_status(pc2d_group_norm_forward(c.dt, c.wdt, c.last, ptr(c.input), ptr(c.weight), ptr(c.bias),
                                       ptr<int>(c.lengths), c.batch, c.channels, c.length, c.groups, eps, silu, ptr(out),
                                       keep_stats ? ptr<float>(stats) : nullptr, ptr(ws), bytes, stream_now()),
               c.call.what);
  return {out, stats};
}

std::vector<Tensor> group_norm_backward_cuda(const Tensor &grad_, const Tensor &input, const OptTensor &weight,
                                             const OptTensor &bias, const OptTensor &lengths, const Tensor &stats_,
                                             int64_t groups, bool silu) {
  const c10::cuda::CUDAGuard guard(input.device());
  const NormCall c = norm_call("paraconv2d_b200.group_norm_backward", input, weight, bias, lengths, groups);
  TORCH_CHECK(grad_.device() == input.device() && grad_.scalar_type() == input.scalar_type() &&
                  grad_.sizes() == input.sizes(),
              c.call.what, ": grad must be like the input");
  const Tensor grad = same_layout(c.input, grad_) ? grad_ : norm_result(c).copy_(grad_);
  const Tensor stats = c.call.need(stats_, "stats", at::kFloat, {c.batch, c.groups, 2});
  Tensor dx = norm_result(c);
  auto like = [&](const Tensor &t) { return at::empty(t.defined() ? t.sizes() : at::IntArrayRef({0}),
                                                      t.defined() ? t.options() : input.options()); };
  Tensor dw = like(c.weight), db = like(c.bias);
  const size_t bytes = pc2d_group_norm_workspace_size(c.dt, c.last, c.batch, c.channels, c.length, c.groups, 1);
  const Tensor ws = workspace(bytes, input);
  check_status(pc2d_group_norm_backward(c.dt, c.wdt, c.last, ptr(grad), ptr(c.input), ptr(c.weight), ptr(c.bias),
                                        ptr<int>(c.lengths), ptr<float>(stats), c.batch, c.channels, c.length, c.groups,
                                        silu, ptr(dx), c.weight.defined() ? ptr(dw) : nullptr,
                                        c.bias.defined() ? ptr(db) : nullptr, ptr(ws), bytes, stream_now()),
               c.call.what);
  return {dx, dw, db};
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &input, const OptTensor &weight, const OptTensor &bias,
                        const OptTensor &lengths, int64_t groups, double eps, bool silu) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto outs = PC2D_BELOW(group_norm_forward).call(input, weight, bias, lengths, groups, eps, silu, true);
    ctx->save_for_backward({input, weight.value_or(Tensor()), bias.value_or(Tensor()), lengths.value_or(Tensor()),
                            outs[1]});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["silu"] = silu;
    return outs[0];
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    return once("group_norm", [&]() -> variable_list {
      const auto s = ctx->get_saved_variables();
      const auto g = PC2D_BELOW(group_norm_backward)
                         .call(grads[0], s[0], optional_of(s[1]), optional_of(s[2]), optional_of(s[3]), s[4],
                               ctx->saved_data["groups"].toInt(), ctx->saved_data["silu"].toBool());
      return {g[0], s[1].defined() ? g[1] : Tensor(), s[2].defined() ? g[2] : Tensor(), Tensor(), Tensor(), Tensor(),
              Tensor()};
    });
  }
};

// With gradients the statistics are the graph's own: the second result is empty.
std::vector<Tensor> group_norm_forward_autograd(const Tensor &input, const OptTensor &weight, const OptTensor &bias,
                                                const OptTensor &lengths, int64_t groups, double eps, bool silu,
                                                bool keep_stats) {
  no_forward_mode("group_norm", {&input}, {&weight, &bias});
  check_cuda(input, "group_norm");
  if (needs_grad({&input}, {&weight, &bias}))
    return {NormFunction::apply(input, weight, bias, lengths, groups, eps, silu),
            at::empty({0}, input.options().dtype(at::kFloat))};
  at::AutoDispatchBelowADInplaceOrView below;
  return PC2D_BELOW(group_norm_forward).call(input, weight, bias, lengths, groups, eps, silu, keep_stats);
}

// ---------------------------------------------------------- linear attention

struct AttentionCall {
  Call call;
  int dt, batch, heads, groups, length, dk, dv;
  bool per_token;
  Tensor q, k, v, decay, lengths;
};

AttentionCall attention_call(const char *what, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &decay,
                             const OptTensor &lengths) {
  AttentionCall c{{what, v.device()}};
  const auto type = v.scalar_type();
  c.dt = seq_dtype_code(v, what);
  TORCH_CHECK(v.dim() == 4, what, ": v must be [batch, heads, values, length], got ", v.sizes());
  TORCH_CHECK(q.dim() == 4, what, ": q must be [batch, groups, keys, length], got ", q.sizes());
  c.batch = as_int(v.size(0), what, "batch");
  c.heads = as_int(v.size(1), what, "heads");
  c.dv = as_int(v.size(2), what, "values");
  c.length = as_int(v.size(3), what, "length");
  c.groups = as_int(q.size(1), what, "groups");
  c.dk = as_int(q.size(2), what, "keys");
  c.q = c.call.need(q, "q", type, {c.batch, c.groups, c.dk, c.length});
  c.k = c.call.need(k, "k", type, {c.batch, c.groups, c.dk, c.length});
  c.v = dense(v);
  c.per_token = decay.dim() != 1;
  c.decay = c.per_token ? c.call.need(decay, "log_decay", at::kFloat, {c.batch, c.heads, c.length})
                        : c.call.need(decay, "log_decay", at::kFloat, {c.heads});
  c.lengths = c.call.maybe(lengths, "lengths", at::kInt, {c.batch});
  return c;
}

std::vector<Tensor> linear_attention_forward_cuda(const Tensor &q, const Tensor &k, const Tensor &v,
                                                  const Tensor &log_decay, const OptTensor &initial_,
                                                  const OptTensor &lengths, double scale, bool final_state,
                                                  bool keep_states) {
  const c10::cuda::CUDAGuard guard(v.device());
  const AttentionCall c = attention_call("paraconv2d_b200.linear_attention_forward", q, k, v, log_decay, lengths);
  const Tensor initial = c.call.maybe(initial_, "initial_state", at::kFloat, {c.batch, c.heads, c.dk, c.dv});
  Tensor out = at::empty(c.v.sizes(), c.v.options());
  const auto fopts = c.decay.options();
  Tensor last = at::empty(final_state ? at::IntArrayRef({c.batch, c.heads, c.dk, c.dv}) : at::IntArrayRef({0}), fopts);
  const size_t size =
      keep_states ? pc2d_linear_attention_states_size(c.dt, c.batch, c.heads, c.length, c.dk, c.dv) : 0;
  Tensor states = at::empty({(int64_t)(size / 4)}, fopts);
  const size_t bytes =
      pc2d_linear_attention_workspace_size(c.dt, c.batch, c.heads, c.groups, c.length, c.dk, c.dv, 0);
  const Tensor ws = workspace(bytes, c.v);
  check_status(pc2d_linear_attention_forward(c.dt, ptr(c.q), ptr(c.k), ptr(c.v), ptr<float>(c.decay), c.per_token,
                                             ptr<float>(initial), ptr<int>(c.lengths), c.batch, c.heads, c.groups,
                                             c.length, c.dk, c.dv, scale, ptr(out),
                                             final_state ? ptr<float>(last) : nullptr,
                                             size ? ptr<float>(states) : nullptr, ptr(ws), bytes, stream_now()),
               c.call.what);
  return {out, last, states};
}

std::vector<Tensor> linear_attention_backward_cuda(const Tensor &grad_, const OptTensor &grad_final_, const Tensor &q,
                                                   const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                                   const Tensor &states_, const OptTensor &lengths, double scale,
                                                   bool initial_grad) {
  const c10::cuda::CUDAGuard guard(v.device());
  const AttentionCall c = attention_call("paraconv2d_b200.linear_attention_backward", q, k, v, log_decay, lengths);
  const Tensor grad = c.call.need(grad_, "grad", v.scalar_type(), v.sizes());
  const Tensor grad_final = c.call.maybe(grad_final_, "grad_final", at::kFloat, {c.batch, c.heads, c.dk, c.dv});
  const int64_t kept =
      (int64_t)(pc2d_linear_attention_states_size(c.dt, c.batch, c.heads, c.length, c.dk, c.dv) / 4);
  const Tensor states = c.call.need(states_, "states", at::kFloat, {kept});
  auto like = [](const Tensor &t) { return at::empty(t.sizes(), t.options()); };
  Tensor dq = like(c.q), dk = like(c.k), dv = like(c.v), dg = like(c.decay);
  Tensor dinit = initial_grad ? at::empty({c.batch, c.heads, c.dk, c.dv}, c.decay.options()) : Tensor();
  const size_t bytes =
      pc2d_linear_attention_workspace_size(c.dt, c.batch, c.heads, c.groups, c.length, c.dk, c.dv, 1);
  const Tensor ws = workspace(bytes, c.v);
  check_status(pc2d_linear_attention_backward(c.dt, ptr(grad), ptr<float>(grad_final), ptr(c.q), ptr(c.k), ptr(c.v),
                                              ptr<float>(c.decay), c.per_token, ptr<float>(states),
                                              ptr<int>(c.lengths), c.batch, c.heads, c.groups, c.length, c.dk, c.dv,
                                              scale, ptr(dq), ptr(dk), ptr(dv), ptr<float>(dg), ptr<float>(dinit),
                                              ptr(ws), bytes, stream_now()),
               c.call.what);
  return {dq, dk, dv, dg, dinit.defined() ? dinit : at::empty({0}, c.decay.options())};
}

Tensor linear_attention_step_cuda(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &log_decay,
                                  const Tensor &state, const OptTensor &slots_, double scale) {
  const Call call{"paraconv2d_b200.linear_attention_step", v_.device()};
  const c10::cuda::CUDAGuard guard(v_.device());
  const auto type = v_.scalar_type();
  const int dt = seq_dtype_code(v_, call.what);
  TORCH_CHECK(v_.dim() == 3, call.what, ": v must be [batch, heads, values], got ", v_.sizes());
  TORCH_CHECK(q_.dim() == 3, call.what, ": q must be [batch, groups, keys], got ", q_.sizes());
  const int batch = as_int(v_.size(0), call.what, "batch"), heads = as_int(v_.size(1), call.what, "heads");
  const int dv = as_int(v_.size(2), call.what, "values"), groups = as_int(q_.size(1), call.what, "groups");
  const int dk = as_int(q_.size(2), call.what, "keys");
  TORCH_CHECK(state.dim() == 4, call.what, ": state must be [places, ", heads, ", ", dk, ", ", dv, "], got ",
              state.sizes());
  const int places = as_int(state.size(0), call.what, "places");
  call.in_place(state, "state", at::kFloat, {places, heads, dk, dv});
  const Tensor q = call.need(q_, "q", type, {batch, groups, dk}), k = call.need(k_, "k", type, {batch, groups, dk});
  const Tensor v = dense(v_);
  const bool per_row = log_decay.dim() != 1;
  const Tensor decay = per_row ? call.need(log_decay, "log_decay", at::kFloat, {batch, heads})
                               : call.need(log_decay, "log_decay", at::kFloat, {heads});
  const Tensor slots = call.maybe(slots_, "slots", at::kInt, {batch});
  call.apart(state, {&q, &k, &v, &decay, &slots});
  Tensor out = at::empty({batch, heads, dv}, v.options());
  check_status(pc2d_linear_attention_step(dt, ptr(q), ptr(k), ptr(v), ptr<float>(decay), per_row, ptr<float>(state),
                                          ptr<int>(slots), batch, places, heads, groups, dk, dv, scale, ptr(out),
                                          stream_now()),
               call.what);
  changed(state);
  return out;
}

struct AttentionFunction : torch::autograd::Function<AttentionFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q_, const Tensor &k_, const Tensor &v_,
                               const Tensor &log_decay, const OptTensor &initial, const OptTensor &lengths, double scale,
                               bool final_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor q = q_.contiguous(), k = k_.contiguous(), v = v_.contiguous(), g = log_decay.contiguous();
    auto outs = PC2D_BELOW(linear_attention_forward).call(q, k, v, g, initial, lengths, scale, final_state, true);
    ctx->save_for_backward({q, k, v, g, outs[2], lengths.value_or(Tensor())});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["initial"] = initial.has_value() && initial->defined() && initial->requires_grad();
    ctx->set_materialize_grads(false);
    outs.pop_back();
    if (!final_state) outs.pop_back();
    return outs;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    return once("linear_attention", [&]() -> variable_list {
      const auto s = ctx->get_saved_variables();
      const Tensor grad = grads[0].defined() ? grads[0] : at::zeros_like(s[2]);
      const bool initial = ctx->saved_data["initial"].toBool();
      const auto g = PC2D_BELOW(linear_attention_backward)
                         .call(grad, grads.size() > 1 ? optional_of(grads[1]) : OptTensor(), s[0], s[1], s[2], s[3],
                               s[4], optional_of(s[5]), ctx->saved_data["scale"].toDouble(), initial);
      return {g[0], g[1], g[2], g[3], initial ? g[4] : Tensor(), Tensor(), Tensor(), Tensor()};
    });
  }
};

// With gradients the states are the graph's own: the third result is empty.
std::vector<Tensor> linear_attention_forward_autograd(const Tensor &q, const Tensor &k, const Tensor &v,
                                                      const Tensor &log_decay, const OptTensor &initial,
                                                      const OptTensor &lengths, double scale, bool final_state,
                                                      bool keep_states) {
  no_forward_mode("linear_attention", {&q, &k, &v, &log_decay}, {&initial});
  check_cuda(v, "linear_attention");
  if (needs_grad({&q, &k, &v, &log_decay}, {&initial})) {
    auto outs = AttentionFunction::apply(q, k, v, log_decay, initial, lengths, scale, final_state);
    while (outs.size() < 3) outs.push_back(at::empty({0}, log_decay.options()));
    return outs;
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return PC2D_BELOW(linear_attention_forward).call(q, k, v, log_decay, initial, lengths, scale, final_state, keep_states);
}

Tensor linear_attention_step_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                      const Tensor &state, const OptTensor &slots, double scale) {
  no_forward_mode("linear_attention_step", {&q, &k, &v, &log_decay, &state}, {});
  no_step_grad("linear_attention_step", needs_grad({&q, &k, &v, &log_decay, &state}, {}));
  check_cuda(v, "linear_attention_step");
  at::AutoDispatchBelowADInplaceOrView below;
  return PC2D_BELOW(linear_attention_step).call(q, k, v, log_decay, state, slots, scale);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(paraconv2d_b200, m) {
  m.def(
      "adamw_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, "
      "Tensor(d!)[] masters, Tensor(e!)[] scales, Tensor(f!) step, Tensor? lr_tensor, float lr, float beta1, "
      "float beta2, float eps, float weight_decay, Tensor? grad_scale, int[] splits, float[] factors, int seed, "
      "int[] numbers=[]) -> ()");
  m.def(
      "group_norm_forward(Tensor input, Tensor? weight, Tensor? bias, Tensor? lengths, int groups, float eps, bool "
      "silu, bool keep_stats) -> Tensor[]");
  m.def(
      "group_norm_backward(Tensor grad, Tensor input, Tensor? weight, Tensor? bias, Tensor? lengths, Tensor stats, "
      "int groups, bool silu) -> Tensor[]");
  m.def(
      "linear_attention_forward(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? initial_state, Tensor? lengths, "
      "float scale, bool final_state, bool keep_states) -> Tensor[]");
  m.def(
      "linear_attention_backward(Tensor grad, Tensor? grad_final, Tensor q, Tensor k, Tensor v, Tensor log_decay, "
      "Tensor states, Tensor? lengths, float scale, bool initial_grad) -> Tensor[]");
  m.def(
      "linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, Tensor? slots, float "
      "scale) -> Tensor");
  m.def("adamw_state_values(Tensor[] exp_avgs, Tensor[] exp_avg_sqs, Tensor[] scales, ScalarType dtype) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(paraconv2d_b200, CUDA, m) {
  m.impl("adamw_step", adamw_step_cuda);
  m.impl("adamw_state_values", adamw_state_values_cuda);
  m.impl("group_norm_forward", group_norm_forward_cuda);
  m.impl("group_norm_backward", group_norm_backward_cuda);
  m.impl("linear_attention_forward", linear_attention_forward_cuda);
  m.impl("linear_attention_backward", linear_attention_backward_cuda);
  m.impl("linear_attention_step", linear_attention_step_cuda);
}

TORCH_LIBRARY_IMPL(paraconv2d_b200, Autograd, m) {
  m.impl("adamw_step", adamw_step_autograd);
  m.impl("group_norm_forward", group_norm_forward_autograd);
  m.impl("linear_attention_forward", linear_attention_forward_autograd);
  m.impl("linear_attention_step", linear_attention_step_autograd);
}
