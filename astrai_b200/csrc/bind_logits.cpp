// Python bindings of the kernels over rows of logits (distill.cu, top_logits.cu, sample_given.cu): every tensor check is here.
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "bind_util.h"

namespace astrai_host {
int distill_max_k();
int distill_max_vocab(int elem);
void distill(const void* x, long long ldx, void* dx, long long lddx, const void* ids, bool ids64, const void* values,
             int values_type, const float* rest, const long long* target, long long ignore, int rows, int V, int K,
             double tau, double hard, const float* grad, float expected, bool unless_expected, float* row_loss,
             float* count, bool have_count, float* loss, int dtype, int device, cudaStream_t s);
int top_logits_max_k();
void top_logits(const void* x, long long ldx, int rows, int V, int k, float tau, int* ids, void* values, float* rest,
                int dtype, cudaStream_t s);
void sample_given(const void* x, long long ldx, int rows, int V, const void* uniform, bool uniform64,
                  const float* temperature, const int* top_k, const float* top_p, const float* min_p, long long* token,
                  float* logprob, int dtype, int device, cudaStream_t s);
}  // namespace astrai_host

namespace {

using namespace astrai_bind;

int dtype_code(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, what, " must be bfloat16, float16 or float32, got ", t.scalar_type());
  }
  return -1;
}

void check_cuda(const at::Tensor& t, const at::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), what, " must be on the logits' device");
}

void no_tangent(const at::Tensor& t, const char* op) {
  TORCH_CHECK(!t._fw_grad(0).defined(), op, " has no forward-mode derivative");
}

// [rows, vocab] with a contiguous last dimension, a view where the strides allow it
at::Tensor rows_of(const at::Tensor& t) {
  const auto r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}
long long row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// ------------------------------------------------------------------------------------------ top logits
std::tuple<at::Tensor, at::Tensor, at::Tensor> top_logits(const at::Tensor& logits, int64_t k, double tau) {
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "top_logits: logits must be [..., vocab]");
  const int64_t V = logits.size(-1);
  TORCH_CHECK_VALUE(k >= 1 && k <= V && k <= astrai_host::top_logits_max_k(), "top_logits: k must be in 1 .. ",
                    std::to_string(std::min<int64_t>(V, astrai_host::top_logits_max_k())), ", got ", std::to_string(k));
  TORCH_CHECK_VALUE(tau > 0. && std::isfinite(tau), "top_logits: temperature must be positive");
  const int code = dtype_code(logits, "top_logits: logits");
  TORCH_CHECK_VALUE(V < (1LL << 30), "top_logits: vocabulary too large");
  no_tangent(logits, "top_logits");
  TORCH_CHECK(!(at::GradMode::is_enabled() && logits.requires_grad()), "top_logits has no gradient: call it under no_grad");
  const c10::cuda::CUDAGuard guard(logits.device());
  const at::Tensor x = rows_of(logits);
  const int64_t rows = x.size(0);
  TORCH_CHECK_VALUE(rows < (1LL << 27), "top_logits: too many rows");
  auto lead = logits.sizes().vec();
  lead.pop_back();
  auto ids = new_like(x, {rows, k}, at::kInt), values = new_like(x, {rows, k}, x.scalar_type()),
       rest = new_like(x, {rows}, at::kFloat);
  if (rows > 0) {
    astrai_host::top_logits(x.data_ptr(), row_stride(x), (int)rows, (int)V, (int)k, (float)tau, ids.data_ptr<int>(),
                            values.data_ptr(), rest.data_ptr<float>(), code, stream());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  if (logits.dim() != 2) {
    rest = rest.view(lead);
    lead.push_back(k);
    ids = ids.view(lead), values = values.view(lead);
  }
  return {ids, values, rest};
}

// ------------------------------------------------------------------------------------------ sampling
std::pair<at::Tensor, OptTensor> sample_given(const at::Tensor& logits, const at::Tensor& uniform_in,
                                              const at::Tensor& temperature_in, const at::Tensor& top_k_in,
                                              const at::Tensor& top_p_in, const at::Tensor& min_p_in, bool logprobs) {
  TORCH_CHECK_VALUE(logits.dim() == 2 && logits.size(1) >= 1, "sample_given: logits must be [batch, vocab]");
  const int64_t rows = logits.size(0), V = logits.size(1);
  const int code = dtype_code(logits, "sample_given: logits");
  TORCH_CHECK_VALUE(V <= (1LL << 22), "sample_given: a vocabulary of at most 2^22");
  TORCH_CHECK_VALUE(rows < (1LL << 27), "sample_given: too many rows");
  TORCH_CHECK(uniform_in.scalar_type() == at::kFloat || uniform_in.scalar_type() == at::kDouble,
              "sample_given: uniform must be float32 or float64, got ", uniform_in.scalar_type());
  const c10::cuda::CUDAGuard guard(logits.device());
  // one number per row, or one for all
  const auto per_row = [&](const at::Tensor& t, at::ScalarType type, const char* name) {
    TORCH_CHECK_VALUE(t.numel() == rows || t.numel() == 1, "sample_given: ", name, " must have one number or one per row");
    TORCH_CHECK(t.is_cuda() && t.device() == logits.device(), "sample_given: ", name, " must be on the logits' device");
    if (t.scalar_type() == type && t.numel() == rows && t.is_contiguous()) return t;
    return t.to(type).reshape({-1}).expand({rows}).contiguous();
  };
  const at::NoGradGuard off;
  const at::Tensor uniform = per_row(uniform_in, uniform_in.scalar_type(), "uniform"),
                   temperature = per_row(temperature_in, at::kFloat, "temperature"),
                   top_k = per_row(top_k_in, at::kInt, "top_k"), top_p = per_row(top_p_in, at::kFloat, "top_p"),
                   min_p = per_row(min_p_in, at::kFloat, "min_p");
  const at::Tensor x = rows_of(logits);
  auto token = new_like(x, {rows}, at::kLong);
  OptTensor logprob;
  if (logprobs) logprob = new_like(x, {rows}, at::kFloat);
  if (rows > 0) {
    astrai_host::sample_given(x.data_ptr(), row_stride(x), (int)rows, (int)V, uniform.data_ptr(),
                              uniform.scalar_type() == at::kDouble, temperature.data_ptr<float>(), top_k.data_ptr<int>(),
                              top_p.data_ptr<float>(), min_p.data_ptr<float>(), (long long*)token.data_ptr<int64_t>(),
                              logprobs ? logprob->data_ptr<float>() : nullptr, code, logits.get_device(), stream());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {token, logprob};
}

// ------------------------------------------------------------------------------------------ distillation
struct Distill {
  at::Tensor x, ids, values, rest, target, count;  // rest and target: undefined if not given; count: with a target
  double tau, hard;
  int64_t ignore;
};

void launch(const Distill& d, const at::Tensor& dx, const float* grad, double expected, bool unless_expected,
            const at::Tensor& row_loss, bool have_count, const at::Tensor& loss) {
  const auto f32 = [](const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
  astrai_host::distill(d.x.data_ptr(), row_stride(d.x), dx.defined() ? dx.data_ptr() : nullptr,
                       dx.defined() ? row_stride(dx) : 0, d.ids.data_ptr(), d.ids.scalar_type() == at::kLong,
                       d.values.data_ptr(), dtype_code(d.values, "distill_loss: the teacher's values"), f32(d.rest),
                       d.target.defined() ? (const long long*)d.target.data_ptr<int64_t>() : nullptr, d.ignore,
                       (int)d.x.size(0), (int)d.x.size(1), (int)d.ids.size(1), d.tau, d.hard, grad,
                       (float)expected, unless_expected, f32(row_loss), f32(d.count), have_count, f32(loss),
                       dtype_code(d.x, "distill_loss: logits"), d.x.get_device(), stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Memory for the gradient of `x`: each row starts as far off the 16-byte grid as x's does, as the kernel wants it.
at::Tensor grad_like(const at::Tensor& x) {
  const int64_t rows = x.size(0), V = x.size(1), E = 16 / x.element_size();
  const int64_t head = (int64_t)(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) / x.element_size();
  const int64_t ld = V + (((row_stride(x) - V) % E) + E) % E;
  if (head == 0 && ld == V) return new_like(x, {rows, V}, x.scalar_type());
  return new_like(x, {head + rows * ld}, x.scalar_type()).as_strided({rows, V}, {ld, 1}, head);
}

// The capture that the current stream is part of; 0: none.
unsigned long long current_capture() {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream(), &status, &id));
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

// The forward pass leaves the gradient for an upstream gradient of `expected`; the backward hands it out after a launch
// that does nothing on the device where that came true and computes the pass again where it did not. A second backward
// through a retained graph computes it into new memory: the first one's belongs to its receiver. A backward that is not in the
// forward's capture may run again where the forward does not, or before it: it takes neither the gradient nor the rows' number
// from there.
struct DistillLossBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable x, ids, values, rest, target;
  at::Tensor count, ready;
  double tau = 1., hard = 0., expected = 1.;
  int64_t ignore = -100;
  unsigned long long capture = 0;  // the forward's
  std::vector<int64_t> sizes;
  std::string name() const override { return "DistillLossBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* v : {&x, &ids, &values, &rest, &target}) v->reset_data();
    ready.reset();
  }
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    TORCH_CHECK(!at::GradMode::is_enabled(), "distill_loss has no second derivative (create_graph)");
    std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list out(1);
    if (!grads[0].defined()) return out;
    no_tangent(grads[0], "distill_loss's backward");
    Distill d{x.unpack(), ids.unpack(), values.unpack(), rest.unpack(), target.unpack(), count, tau, hard, ignore};
    const c10::cuda::CUDAGuard guard(d.x.device());
    const at::Tensor g = grads[0].to(at::kFloat);
    const bool same = capture == current_capture(), given = ready.defined() && same;
    if (d.target.defined() && !same) d.count = new_like(d.x, {1}, at::kFloat);
    at::Tensor dx = given ? std::move(ready) : grad_like(d.x);
    ready = at::Tensor();
    if (d.x.size(0) > 0) launch(d, dx, g.data_ptr<float>(), expected, given, {}, same, {});
    out[0] = dx.view(sizes);
    return out;
  }
};

at::Tensor distill_loss(const at::Tensor& logits, const at::Tensor& ids_in, const at::Tensor& values_in,
                        const OptTensor& rest_in, double tau, const OptTensor& target_in, double hard, int64_t ignore,
                        double expected) {
  const char* op = "distill_loss";
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "distill_loss: logits must be [..., vocab]");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  for (const auto* t : {&ids_in, &values_in})
    TORCH_CHECK_VALUE(t->dim() == logits.dim() && t->sizes().slice(0, t->dim() - 1) == lead && t->size(-1) >= 1 &&
                          t->sizes() == ids_in.sizes(),
                      "distill_loss: the teacher's ids and values must be [..., k] with the logits' leading sizes");
  TORCH_CHECK_VALUE(ids_in.size(-1) <= astrai_host::distill_max_k(), "distill_loss: at most ",
                    std::to_string(astrai_host::distill_max_k()), " entries of the teacher");
  TORCH_CHECK_VALUE(!given(rest_in) || rest_in->sizes() == lead, "distill_loss: rest must have the logits' leading sizes");
  TORCH_CHECK_VALUE(!given(target_in) || target_in->sizes() == lead,
                    "distill_loss: target must have the logits' leading sizes");
  TORCH_CHECK_VALUE(tau > 0. && std::isfinite(tau), "distill_loss: temperature must be positive");
  TORCH_CHECK_VALUE(hard >= 0. && hard <= 1., "distill_loss: hard_weight must be in [0, 1]");
  TORCH_CHECK_VALUE(hard == 0. || given(target_in), "distill_loss: hard_weight needs a target");
  const int64_t V = logits.size(-1);
  dtype_code(logits, "distill_loss: logits");
  dtype_code(values_in, "distill_loss: the teacher's values");
  TORCH_CHECK_VALUE(V <= astrai_host::distill_max_vocab((int)logits.element_size()), "distill_loss: a vocabulary of ",
                    std::to_string(V), " is too large for this type");
  TORCH_CHECK(ids_in.scalar_type() == at::kInt || ids_in.scalar_type() == at::kLong,
              "distill_loss: ids must be int32 or int64, got ", ids_in.scalar_type());
  TORCH_CHECK(!given(rest_in) || rest_in->scalar_type() == at::kFloat, "distill_loss: rest must be float32");
  check_cuda(ids_in, logits, "distill_loss: ids");
  check_cuda(values_in, logits, "distill_loss: values");
  if (given(rest_in)) check_cuda(*rest_in, logits, "distill_loss: rest");
  if (given(target_in)) {
    check_cuda(*target_in, logits, "distill_loss: target");
    TORCH_CHECK(at::isIntegralType(target_in->scalar_type(), false), "distill_loss: target must hold whole numbers");
  }
  no_tangent(logits, op);
  no_tangent(values_in, op);
  if (given(rest_in)) no_tangent(*rest_in, op);
  TORCH_CHECK(!(at::GradMode::is_enabled() &&
                (values_in.requires_grad() || (given(rest_in) && rest_in->requires_grad()))),
              "distill_loss has no gradient of the teacher");

  const c10::cuda::CUDAGuard guard(logits.device());
  const bool train = at::GradMode::is_enabled() && logits.requires_grad();
  Distill d;
  at::Tensor loss, dx;
  {
    const at::NoGradGuard off;
    d = {rows_of(logits), ids_in.reshape({-1, ids_in.size(-1)}).contiguous(),
         values_in.reshape({-1, ids_in.size(-1)}).contiguous(), {}, {}, {}, tau, hard, ignore};
    if (given(rest_in)) d.rest = rest_in->reshape({-1}).contiguous();
    if (given(target_in)) {
      d.target = target_in->reshape({-1}).to(at::kLong).contiguous();
      d.count = new_like(logits, {1}, at::kFloat);
    }
    const int64_t rows = d.x.size(0);
    TORCH_CHECK_VALUE(rows < (1LL << 27), "distill_loss: too many rows");
    loss = new_like(logits, {}, at::kFloat);
    const auto row_loss = new_like(logits, {rows}, at::kFloat);
    if (train) dx = grad_like(d.x);
    launch(d, dx, nullptr, expected, false, row_loss, false, loss);
  }
  if (train) {
    std::shared_ptr<DistillLossBackward> node(new DistillLossBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->x = {d.x, false}, node->ids = {d.ids, false}, node->values = {d.values, false};
    node->rest = {d.rest, false}, node->target = {d.target, false};
    node->count = d.count, node->ready = dx;
    node->tau = tau, node->hard = hard, node->expected = expected, node->ignore = ignore;
    node->capture = current_capture();
    node->sizes = logits.sizes().vec();
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

}  // namespace

void register_logits(pybind11::module& m) {
  namespace py = pybind11;
  m.def("top_logits", &top_logits, py::arg("logits"), py::arg("k"), py::arg("temperature"));
  m.def("sample_given", &sample_given, py::arg("logits"), py::arg("uniform"), py::arg("temperature"), py::arg("top_k"),
        py::arg("top_p"), py::arg("min_p"), py::arg("return_logprobs"));
  m.def("distill_loss", &distill_loss, py::arg("logits"), py::arg("ids"), py::arg("values"), py::arg("rest"),
        py::arg("temperature"), py::arg("target"), py::arg("hard_weight"), py::arg("ignore_index"),
        py::arg("expected_grad"));
}
