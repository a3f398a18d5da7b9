// The autograd nodes of group_norm_act and dropout (sfm_amd/norm.py checks their arguments and calls this module).
//
// A small call of these operators is bound by the host: their kernels take about five microseconds each.  autograd runs a backward on a
// thread of its own, where Python costs several times what it costs in the loop of a program: a forward and backward of an [8, 8, 26, 512]
// tensor through torch.autograd.Function took 118 us for 25 us of kernels.  So these two are nodes in C++.  All compute
// stays in the C ABI (include/sfm_amd.h), which this file only calls.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cstdint>
#include <mutex>
#include <optional>
#include <string>
#include <vector>

#include "../../include/sfm_amd.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// what a failed C-ABI call raises everywhere in the package, from whichever thread it failed on
void check(const char* name, int rc) {
  if (rc == 0) return;
  pybind11::gil_scoped_acquire gil;
  pybind11::object type = pybind11::module_::import("sfm_amd._lib").attr("SfmAmdError");
  PyErr_SetString(type.ptr(), (std::string(name) + " failed: " + (rc < 0 ? "argument rejected " : "hipError_t ") + std::to_string(rc)).c_str());
  python_error e;
  e.persist();
  throw std::move(e);
}

void refuse_second_order(const char* name) {  // a backward runs with gradients on under create_graph=True alone
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " is differentiable once: its backward was called with create_graph=True");
}

// These nodes are no operators of torch's dispatcher: a tracer would record nothing of them but the allocation of their results, and
// its program would return memory as it found it.
void refuse_tracing(const char* name) {
  TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
              name, " cannot be traced (torch.jit.trace, torch.fx): its kernels would not be in the traced program");
}

int dtype_of(const Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return SFM_F32;
    case at::kBFloat16: return SFM_BF16;
    case at::kHalf: return SFM_F16;
    default: TORCH_CHECK_TYPE(false, "float32, bfloat16 or float16 is needed, got ", x.scalar_type());
  }
}

void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.get_device()).stream(); }

// x [B, ..., C] as rows of C channels ld elements apart: itself if it is dense or a channel slice of a dense buffer, else a copy.  A
// slice's rows are at least C elements apart in every dimension that has more than one of them: a stride of 0, as expanded tensors
// and the gradients of sums have, is none (the kernels would read rows that are not there).
struct Rows {
  Tensor t;
  int64_t ld;
};
Rows rows_of(const Tensor& x) {
  const int64_t d = x.dim(), C = x.size(d - 1);
  if (x.is_contiguous()) return {x, C};
  if (C == 1 || x.stride(d - 1) == 1) {
    int64_t ld = C, want = 0;
    bool seen = false, even = true;  // seen: a dimension of more than one row has set ld
    for (int64_t k = d - 2; k >= 0 && even; --k) {
      if (x.size(k) == 1) continue;
      if (seen) {
        even = x.stride(k) == want;
      } else {
        seen = true;
        ld = want = x.stride(k);
        even = ld >= C && ld <= INT32_MAX / x.element_size();  // (the kernels' limit: rows farther apart are copied)
      }
      want *= x.size(k);
    }
    if (even) return {x, ld};
  }
  return {x.contiguous(), C};
}

struct Mask {
  std::optional<Tensor> rng;
  uint64_t seed;
  uint32_t step, layer, item0;
  int threshold;
  bool per_channel;
  const void* state(const Tensor& unpacked) const { return rng.has_value() ? unpacked.data_ptr() : nullptr; }
};

struct Shape {
  int64_t B, N;
  int C, G, dt, act;
  int64_t stats, fwd, bwd;  // floats: statistics (an even number, so that the workspace behind them is aligned), workspace of either direction
};

struct GroupNormActBackward : public torch::autograd::Node {
  SavedVariable x_, gamma_, beta_, buf_, rng_;
  Shape s{};
  Mask m{};
  std::mutex lock_;

  std::string name() const override { return "GroupNormActBackward"; }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(lock_);
    refuse_second_order("group_norm_act");
    refuse_tracing("group_norm_act");
    variable_list out(3);
    const Tensor x = x_.unpack(), gamma = gamma_.unpack(), beta = beta_.unpack();
    if (!grads[0].defined()) return out;
    const bool need_x = task_should_compute_output(0), need_p = task_should_compute_output(1) || task_should_compute_output(2);
    if (!need_x && !need_p) return out;
    if (s.fwd == 0) return {at::zeros_like(x), at::zeros_like(gamma), at::zeros_like(beta)};
    const Tensor buf = buf_.unpack();
    const Tensor rng = m.rng.has_value() ? rng_.unpack() : Tensor();  // (checks that it is what the forward read)
    const c10::DeviceGuard guard(x.device());
    const Rows xr = rows_of(x), gr = rows_of(grads[0]);
    if (need_x) out[0] = at::empty(x.sizes(), x.options());
    if (need_p) {
      out[1] = at::empty({s.C}, gamma.options());
      out[2] = at::empty({s.C}, gamma.options());
    }
    const void* gy[1] = {gr.t.data_ptr()};
    const long long ld[1] = {gr.ld};
    // a workspace of this pass alone: the node's other passes may be running beside it, as replays of graphs that they were captured into
    const Tensor ws = at::empty({s.bwd}, gamma.options());
    const float* at = buf.data_ptr<float>();
    check("sfm_group_norm_act_bwd",
          sfm_group_norm_act_bwd(xr.t.data_ptr(), xr.ld, s.dt, gy, ld, 1, gamma.data_ptr<float>(), beta.data_ptr<float>(), at,
                                 at + s.stats / 2, s.B, s.N, s.C, s.G, s.act, m.state(rng), m.seed, m.step, m.layer, m.item0,
                                 m.threshold, m.per_channel, need_x ? out[0].data_ptr() : nullptr,
                                 need_p ? out[1].data_ptr<float>() : nullptr, need_p ? out[2].data_ptr<float>() : nullptr,
                                 ws.data_ptr<float>(), stream_of(x)));
    return out;
  }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(lock_);
    for (SavedVariable* v : {&x_, &gamma_, &beta_, &buf_, &rng_}) v->reset_data();
  }
};

struct DropoutBackward : public torch::autograd::Node {
  SavedVariable rng_;
  Mask m{};
  std::mutex lock_;

  std::string name() const override { return "DropoutBackward"; }
  variable_list apply(variable_list&& grads) override;
  void release_variables() override {
    std::lock_guard<std::mutex> lock(lock_);
    rng_.reset_data();
  }
};

Tensor run_dropout(const Tensor& x_, const Mask& m, const Tensor& rng) {
  const Tensor x = x_.contiguous();
  Tensor y = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return y;
  const c10::DeviceGuard guard(x.device());
  check("sfm_dropout", sfm_dropout(x.data_ptr(), dtype_of(x), x.size(0), x.numel() / x.size(0), (int)x.size(-1), m.state(rng), m.seed,
                                   m.step, m.layer, m.item0, m.threshold, m.per_channel, y.data_ptr(), stream_of(x)));
  return y;
}

variable_list DropoutBackward::apply(variable_list&& grads) {
  std::lock_guard<std::mutex> lock(lock_);
  refuse_second_order("dropout");
  refuse_tracing("dropout");
  const Tensor rng = m.rng.has_value() ? rng_.unpack() : Tensor();
  if (!grads[0].defined()) return {Tensor()};
  return {run_dropout(grads[0], m, rng)};
}

void refuse_forward_mode(const char* name, const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), name, " has no forward-mode derivative");
}

// A backward that is captured into a graph hands its gradients to the leaves on the stream on which autograd first met them.  While an
// eager graph of the same leaves lives (or a hook on them) that is a stream outside the capture, which cannot be ended
// then: the call is refused before anything of it is recorded.
void refuse_foreign_leaf(const char* name, const Tensor& t, const Tensor& x) {
  if (!t.requires_grad() || !t.is_leaf()) return;
  const auto leaf = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!leaf) return;
  const auto current = c10::hip::getCurrentHIPStream(x.get_device());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(current.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  const auto met = leaf->stream();
  TORCH_CHECK(!met.has_value() || *met == current.unwrap(), name, ": a stream capture, and a tensor that requires gradients and that autograd knows from "
              "another stream: let go of what was computed from it outside of the capture (and of hooks on it), or give a detached copy");
}

template <typename NodeT, typename... T> std::shared_ptr<NodeT> make_node(const T&... inputs) {
  std::shared_ptr<NodeT> node(new NodeT(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}

Tensor group_norm_act(const Tensor& x, const Tensor& gamma, const Tensor& beta, int64_t groups, double epsilon, int act,
                      std::optional<Tensor> rng, uint64_t seed, uint32_t step, uint32_t layer, uint32_t item0, int threshold,
                      bool per_channel) {
  refuse_tracing("group_norm_act");
  Shape s{};
  s.dt = dtype_of(x);
  s.act = act;
  s.C = (int)x.size(-1);
  s.G = (int)groups;
  s.B = x.size(0);
  s.N = s.B ? x.numel() / (s.B * s.C) : 0;
  Mask m{std::move(rng), seed, step, layer, item0, threshold, per_channel};
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || gamma.requires_grad() || beta.requires_grad());
  for (const Tensor* t : {&x, &gamma, &beta}) {
    refuse_forward_mode("group_norm_act", *t);
    if (grad) refuse_foreign_leaf("group_norm_act", *t, x);
  }
  Tensor y, buf;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    y = at::empty(x.sizes(), x.options());
    if (x.numel()) {
      s.fwd = sfm_group_norm_workspace_floats(s.B, s.N, s.C, s.G, s.dt, 0);
      s.bwd = sfm_group_norm_workspace_floats(s.B, s.N, s.C, s.G, s.dt, 1);
      TORCH_CHECK_VALUE(s.fwd > 0 && s.bwd > 0, "unsupported group-norm shape ", x.sizes(), " with ", groups, " groups (rc ",
                        std::min(s.fwd, s.bwd), ")");
      s.stats = 2 * s.B * s.G;
      // one buffer for the statistics, where a backward may come, and the workspace
      buf = at::empty({grad ? s.stats + s.fwd : s.fwd}, gamma.options());
      float* at = buf.data_ptr<float>();
      const Rows xr = rows_of(x);
      check("sfm_group_norm_act_fwd",
            sfm_group_norm_act_fwd(xr.t.data_ptr(), xr.ld, s.dt, gamma.data_ptr<float>(), beta.data_ptr<float>(), s.B, s.N, s.C, s.G,
                                   (float)epsilon, act, m.rng.has_value() ? m.rng->data_ptr() : nullptr, seed, step, layer, item0,
                                   threshold, per_channel, y.data_ptr(), s.C, grad ? at : nullptr, grad ? at + s.stats / 2 : nullptr,
                                   grad ? at + s.stats : at, stream_of(x)));
    }
  }
  if (grad) {
    auto node = make_node<GroupNormActBackward>(x, gamma, beta);
    node->x_ = SavedVariable(x, false);
    node->gamma_ = SavedVariable(gamma, false);
    node->beta_ = SavedVariable(beta, false);
    if (buf.defined()) node->buf_ = SavedVariable(buf, false);
    if (m.rng.has_value()) node->rng_ = SavedVariable(*m.rng, false);
    node->s = s;
    node->m = std::move(m);
    torch::autograd::set_history(y, node);
  }
  return y;
}

Tensor dropout(const Tensor& x, std::optional<Tensor> rng, uint64_t seed, uint32_t step, uint32_t layer, uint32_t item0, int threshold,
               bool per_channel) {
  refuse_tracing("dropout");
  Mask m{std::move(rng), seed, step, layer, item0, threshold, per_channel};
  refuse_forward_mode("dropout", x);
  const bool grad = at::GradMode::is_enabled() && x.requires_grad();
  if (grad) refuse_foreign_leaf("dropout", x, x);
  Tensor y;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    y = run_dropout(x, m, m.rng.has_value() ? *m.rng : Tensor());
  }
  if (grad) {
    auto node = make_node<DropoutBackward>(x);
    if (m.rng.has_value()) node->rng_ = SavedVariable(*m.rng, false);
    node->m = std::move(m);
    torch::autograd::set_history(y, node);
  }
  return y;
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
  m.doc() = "autograd nodes of sfm_amd.norm";
  m.def("group_norm_act", torch::wrap_pybind_function_no_gil(&group_norm_act));
  m.def("dropout", torch::wrap_pybind_function_no_gil(&dropout));
  // x as rows -> (the tensor itself or a dense copy, elements between rows)
  m.def("rows_of", [](const Tensor& x) {
    Rows r = rows_of(x);
    return pybind11::make_tuple(std::move(r.t), r.ld);
  });
  m.def("refuse_tracing", [](const std::string& name) { refuse_tracing(name.c_str()); });
  m.def("refuse_foreign_leaves", [](const std::string& name, const std::vector<Tensor>& inputs, const Tensor& x) {
    for (const Tensor& t : inputs) refuse_foreign_leaf(name.c_str(), t, x);
  });
}
