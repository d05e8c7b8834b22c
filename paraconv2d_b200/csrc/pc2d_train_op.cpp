// torch.ops.paraconv2d_b200: the AdamW step over many tensors, on top of the C
// ABI of libpc2d_sm100.so.  Argument checks, streams and scratch as for the
// sequence operators.
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

void adamw_step_cuda(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs, at::TensorList exp_avg_sqs,
                     at::TensorList masters, at::TensorList scales, const Tensor &step, const OptTensor &lr_tensor,
                     double lr, double beta1, double beta2, double eps, double weight_decay,
                     const OptTensor &grad_scale_, at::IntArrayRef splits, at::ArrayRef<double> factors, int64_t seed) {
  const Call call{"paraconv2d_b200.adamw_step", step.device()};
  const c10::cuda::CUDAGuard guard(step.device());
  const size_t count = params.size();
  TORCH_CHECK(grads.size() == count && exp_avgs.size() == count && exp_avg_sqs.size() == count, call.what,
              ": params, grads, exp_avgs and exp_avg_sqs must be of equal length");
  TORCH_CHECK((masters.empty() || masters.size() == count) && (scales.empty() || scales.size() == count), call.what,
              ": masters and scales must be as many as params, or none");
  TORCH_CHECK((splits.empty() && factors.empty()) || (splits.size() == count && factors.size() == 3 * count), call.what,
              ": a split and three factors for each of params, or none");
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
  check_status(pc2d_adamw_step(bits8 ? 8 : 32, items.data(), (int)count, ptr<int64_t>(step), ptr<float>(rate), lr,
                               beta1, beta2, eps, weight_decay, ptr<float>(grad_scale), seed, ptr(ws), bytes,
                               stream_now()),
               call.what);
  changed(step);
  for (const auto &list : {params, exp_avgs, exp_avg_sqs, masters, scales})
    for (const Tensor &t : list) changed(t);
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

}  // namespace

TORCH_LIBRARY_FRAGMENT(paraconv2d_b200, m) {
  m.def(
      "adamw_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, "
      "Tensor(d!)[] masters, Tensor(e!)[] scales, Tensor(f!) step, Tensor? lr_tensor, float lr, float beta1, "
      "float beta2, float eps, float weight_decay, Tensor? grad_scale, int[] splits, float[] factors, int seed) -> ()");
  m.def("adamw_state_values(Tensor[] exp_avgs, Tensor[] exp_avg_sqs, Tensor[] scales, ScalarType dtype) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(paraconv2d_b200, CUDA, m) {
  m.impl("adamw_step", adamw_step_cuda);
  m.impl("adamw_state_values", adamw_state_values_cuda);
}
