// Python bindings of the per-head norm + rotation kernels (qk_norm.cu): every tensor check is here.
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <cuda_runtime.h>

#include "bind_util.h"

namespace astrai_host {
void qk_norm_fwd(const void* x, long long ldx, void* y, long long ldy, int rows, int hq, int hkv, int D,
                 const void* table, int max_pos, const int* pos, int seq_len, const void* wq, const void* wk, int rot,
                 int rot_off, bool half_layout, int norm, int inverse, float eps, int dtype, int device,
                 cudaStream_t s);
long long qk_norm_bwd_scratch(int rows, int heads, int D, int rot, int elem, int device);
void qk_norm_bwd(const void* dy, long long lddy, const void* x, long long ldx, void* dx, long long lddx, int rows,
                 int hq, int hkv, int D, const void* table, int max_pos, const int* pos, int seq_len, const void* wq,
                 const void* wk, int rot, int rot_off, bool half_layout, int norm, float eps, void* dwq, void* dwk,
                 float* scratch, int dtype, int device, cudaStream_t s);
}  // namespace astrai_host

namespace {

using namespace astrai_bind;

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, "qk_norm_rope: bfloat16, float16 or float32, got ", t.scalar_type());
  }
  return -1;
}

bool rows_on_grid(const at::Tensor& t) {
  return t.stride(1) == 1 && (t.size(0) <= 1 || (t.stride(0) * t.element_size()) % 16 == 0) && on_grid(t);
}
// The first `used` columns as the kernels can read them: t itself, or a copy (contiguous() would return a contiguous
// tensor as it is, wherever its rows start).
at::Tensor rows_of(const at::Tensor& t, int64_t used) {
  return rows_on_grid(t) ? t : t.narrow(1, 0, used).clone(at::MemoryFormat::Contiguous);
}
OptTensor weight_of(const OptTensor& w) {
  return given(w) && !(w->is_contiguous() && on_grid(*w)) ? OptTensor(w->clone(at::MemoryFormat::Contiguous)) : w;
}

// rows of at least `width` columns, of like's type and device, each on a 16-byte boundary
void check_rows(const at::Tensor& t, const at::Tensor& like, int64_t width, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == like.scalar_type(), "qk_norm_rope: ",
              name, " must be a CUDA tensor of the input's type and device");
  TORCH_CHECK(t.dim() == 2 && t.size(0) == like.size(0) && t.size(1) >= width, "qk_norm_rope: ", name,
              " must be [rows, >= (n_heads + n_kv_heads) * head_dim]");
  TORCH_CHECK(rows_on_grid(t), "qk_norm_rope: ", name, " needs a contiguous inner dimension and 16-byte aligned rows");
}
void check_output(const at::Tensor& t, const at::Tensor& like, int64_t width, const char* name) {
  check_rows(t, like, width, name);
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= width, "qk_norm_rope: rows of ", name, " overlap");
}

struct Shape {
  int rows, hq, hkv, D, max_pos, rot, rot_off, dtype, device;
  const int* pos;
};

Shape check(const at::Tensor& x, int64_t hq, int64_t hkv, int64_t D, const at::Tensor& table, const OptTensor& pos,
            int64_t seq_len, const OptTensor& wq, const OptTensor& wk, int64_t rot, int64_t rot_off, int64_t norm) {
  TORCH_CHECK(x.is_cuda(), "qk_norm_rope: x must be a CUDA tensor");
  Shape s{};
  s.dtype = dtype_code(x);
  TORCH_CHECK(hq >= 1 && hkv >= 0 && hq + hkv <= 65536, "qk_norm_rope: head counts");
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "qk_norm_rope: head_dim must be a multiple of 8, at most 256");
  TORCH_CHECK(rot >= 8 && rot % 8 == 0 && rot_off >= 0 && rot_off % 8 == 0 && rot + rot_off <= D,
              "qk_norm_rope: rot_dim and rot_off must be multiples of 8 inside head_dim");
  TORCH_CHECK(norm >= 0 && norm <= 2, "qk_norm_rope: norm mode");
  TORCH_CHECK(x.size(0) <= (1LL << 30), "qk_norm_rope: too many rows");
  check_rows(x, x, (hq + hkv) * D, "x");
  TORCH_CHECK(table.is_cuda() && table.device() == x.device() && table.scalar_type() == at::kFloat &&
                  table.is_contiguous() && table.dim() == 3 && table.size(1) == rot / 2 && table.size(2) == 2 &&
                  on_grid(table),
              "qk_norm_rope: table must be contiguous fp32 [max_pos, rot_dim / 2, 2] on x's device, 16-byte aligned");
  s.pos = nullptr;
  if (given(pos)) {
    TORCH_CHECK(pos->is_cuda() && pos->device() == x.device() && pos->scalar_type() == at::kInt &&
                    pos->is_contiguous() && pos->numel() == x.size(0),
                "qk_norm_rope: positions must be contiguous int32 with one entry per row");
    s.pos = pos->data_ptr<int>();
  } else {
    TORCH_CHECK(seq_len >= 1 && seq_len < (1LL << 31), "qk_norm_rope: seq_len is needed without positions");
  }
  if (norm != 0) {
    for (const auto* w : {&wq, &wk}) {
      TORCH_CHECK(given(*w) && (*w)->device() == x.device() && (*w)->scalar_type() == x.scalar_type() &&
                      (*w)->is_contiguous() && (*w)->numel() == D && on_grid(**w),
                  "qk_norm_rope: weights must be contiguous [head_dim], of x's type and device, 16-byte aligned");
    }
  }
  s.rows = (int)x.size(0), s.hq = (int)hq, s.hkv = (int)hkv, s.D = (int)D, s.max_pos = (int)table.size(0);
  s.rot = (int)rot, s.rot_off = (int)rot_off, s.device = x.device().index();
  return s;
}

struct Options {
  int64_t hq, hkv, D, seq_len, rot, rot_off, norm;
  bool half_layout;
  double eps;
};

// y may be x itself
void forward_into(const at::Tensor& x, const at::Tensor& y, const at::Tensor& table, const OptTensor& pos,
                  const OptTensor& wq_in, const OptTensor& wk_in, const Options& o, bool inverse) {
  const OptTensor wq = weight_of(wq_in), wk = weight_of(wk_in);
  const Shape s = check(x, o.hq, o.hkv, o.D, table, pos, o.seq_len, wq, wk, o.rot, o.rot_off, o.norm);
  check_output(y, x, (o.hq + o.hkv) * o.D, "y");
  const c10::cuda::CUDAGuard g(x.device());
  astrai_host::qk_norm_fwd(x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), s.rows, s.hq, s.hkv, s.D,
                           table.data_ptr(), s.max_pos, s.pos, (int)o.seq_len, o.norm ? wq->data_ptr() : nullptr,
                           o.norm ? wk->data_ptr() : nullptr, s.rot, s.rot_off, o.half_layout, (int)o.norm, inverse,
                           (float)o.eps, s.dtype, s.device, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Fills the query and key columns of dx; -> gradients of the weights (undefined without a norm).
std::pair<at::Tensor, at::Tensor> backward_into(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& dx,
                                                const at::Tensor& table, const OptTensor& pos,
                                                const OptTensor& wq_in, const OptTensor& wk_in, const Options& o) {
  const OptTensor wq = weight_of(wq_in), wk = weight_of(wk_in);
  if (o.norm == 0) {  // the transposed rotation
    forward_into(dy, dx, table, pos, wq, wk, o, true);
    return {};
  }
  const Shape s = check(x, o.hq, o.hkv, o.D, table, pos, o.seq_len, wq, wk, o.rot, o.rot_off, o.norm);
  check_rows(dy, x, (o.hq + o.hkv) * o.D, "dy");
  check_output(dx, x, (o.hq + o.hkv) * o.D, "dx");
  const c10::cuda::CUDAGuard g(x.device());
  if (s.rows == 0) return {at::zeros_like(*wq), at::zeros_like(*wk)};
  auto dwq = new_like(x, wq->sizes(), x.scalar_type()), dwk = new_like(x, wk->sizes(), x.scalar_type());
  const int64_t need = astrai_host::qk_norm_bwd_scratch(s.rows, s.hq + s.hkv, s.D, s.rot, (int)x.element_size(), s.device);
  auto scratch = new_like(x, {need}, at::kFloat);
  astrai_host::qk_norm_bwd(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), dx.data_ptr(), dx.stride(0), s.rows,
                           s.hq, s.hkv, s.D, table.data_ptr(), s.max_pos, s.pos, (int)o.seq_len, wq->data_ptr(),
                           wk->data_ptr(), s.rot, s.rot_off, o.half_layout, (int)o.norm, (float)o.eps, dwq.data_ptr(),
                           dwk.data_ptr(), scratch.data_ptr<float>(), s.dtype, s.device, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dwq, dwk};
}

// The autograd node, in C++ and a Node of its own: a training step of short kernels would otherwise wait for Python,
// and for the list and dictionary in which torch::autograd::Function keeps what it was given.
struct QkNormRopeBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable x, wq, wk, table, pos;  // x and the weights: undefined without a norm
  Options o;
  int64_t width = 0;  // columns of x
  std::string name() const override { return "QkNormRopeBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* v : {&x, &wq, &wk, &table, &pos}) v->reset_data();
  }
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    TORCH_CHECK(!at::GradMode::is_enabled(), "qk_norm_rope has no second derivative (create_graph)");
    std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list out(3);
    if (!grads[0].defined()) return out;
    TORCH_CHECK(!grads[0]._fw_grad(0).defined(), "qk_norm_rope has no second derivative (a tangent in its backward)");
    const at::Tensor table_ = table.unpack(), dy = rows_of(grads[0], grads[0].size(1)),
                     x_ = o.norm ? x.unpack() : dy;
    const auto given_or_none = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const int64_t used = (o.hq + o.hkv) * o.D;
    const int64_t grid = 16 / dy.element_size();  // rows of dx start on the 16-byte grid, whatever x's width is
    auto dx = new_like(dy, {dy.size(0), (width + grid - 1) / grid * grid}, dy.scalar_type()).narrow(1, 0, width);
    if (width > used) dx.narrow(1, used, width - used).zero_();  // columns behind the keys are not an input
    auto dw = backward_into(dy, x_, dx, table_, given_or_none(pos.unpack()), given_or_none(wq.unpack()),
                            given_or_none(wk.unpack()), o);
    out[0] = std::move(dx), out[1] = std::move(dw.first), out[2] = std::move(dw.second);
    return out;
  }
};

at::Tensor with_gradient(const at::Tensor& x, const OptTensor& wq, const OptTensor& wk, const at::Tensor& table,
                         const OptTensor& pos, const Options& o) {
  const auto or_none = [](const OptTensor& t) { return given(t) ? *t : at::Tensor(); };
  at::Tensor rows, y;
  {
    const at::NoGradGuard off;
    rows = rows_of(x, (o.hq + o.hkv) * o.D);
    y = new_like(x, {x.size(0), (o.hq + o.hkv) * o.D}, x.scalar_type());
    forward_into(rows, y, table, pos, wq, wk, o, false);
  }
  std::shared_ptr<QkNormRopeBackward> node(new QkNormRopeBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, or_none(wq), or_none(wk)));
  if (o.norm) node->x = {rows, false};  // a rotation's gradient does not depend on its input
  node->wq = {or_none(wq), false}, node->wk = {or_none(wk), false};
  node->table = {table, false}, node->pos = {or_none(pos), false};
  node->o = o, node->width = x.size(1);
  torch::autograd::set_history(y, node);
  return y;
}

// The user's call: argument errors are ValueErrors here, wrong tensors RuntimeErrors in check().
at::Tensor qk_norm_rope(const at::Tensor& x, int64_t hq, int64_t hkv, int64_t D, const at::Tensor& table,
                        OptTensor wq, OptTensor wk, OptTensor pos, int64_t seq_len, double eps, bool half_layout,
                        int64_t norm, int64_t rot, int64_t rot_off, bool in_place) {
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) >= (hq + hkv) * D,
                    "qk_norm_rope: x must be [rows, >= (n_heads + n_kv_heads) * head_dim]");
  TORCH_CHECK_VALUE(rot > 0 && rot % 2 == 0 && rot_off >= 0 && rot + rot_off <= D,
                    "qk_norm_rope: rot_dim at rot_off is no even part of head_dim");
  TORCH_CHECK_VALUE(table.dim() == 3 && table.size(1) * 2 == rot && table.size(2) == 2,
                    "qk_norm_rope: table must be [max_pos, rot_dim / 2, 2]");
  if (norm == 0) wq = wk = OptTensor();
  TORCH_CHECK_VALUE(norm == 0 || (given(wq) && given(wk) && wq->numel() == D && wk->numel() == D),
                    "qk_norm_rope: the norm needs q_weight and k_weight of head_dim entries");
  TORCH_CHECK_VALUE(given(pos) || seq_len > 0, "qk_norm_rope: positions or seq_len must be given");
  if (given(pos)) {
    TORCH_CHECK_VALUE(pos->numel() == x.size(0), "qk_norm_rope: positions must have one entry per row");
    if (pos->scalar_type() != at::kInt || !pos->is_contiguous()) pos = pos->to(at::kInt).contiguous();
  }
  // a dual number need not require a gradient, and GradMode does not stop tangents
  const at::Tensor* const inputs[] = {&x, &table, given(wq) ? &*wq : nullptr, given(wk) ? &*wk : nullptr};
  for (const at::Tensor* t : inputs)
    TORCH_CHECK(!t || !t->_fw_grad(0).defined(), "qk_norm_rope has no forward-mode derivative");
  TORCH_CHECK(!(at::GradMode::is_enabled() && table.requires_grad()), "qk_norm_rope has no gradient of the table");
  const bool grad = at::GradMode::is_enabled() &&
                    (x.requires_grad() || (norm && (wq->requires_grad() || wk->requires_grad())));
  const Options o{hq, hkv, D, seq_len, rot, rot_off, norm, half_layout, eps};
  if (in_place) {
    TORCH_CHECK(!grad, "qk_norm_rope_ has no gradient (of x or the weights): use qk_norm_rope");
    forward_into(x, x, table, pos, wq, wk, o, false);
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();  // a backward that saved x has to notice
    return x;
  }
  if (grad)
    return with_gradient(x, wq, wk, table, pos, o);
  auto y = new_like(x, {x.size(0), (hq + hkv) * D}, x.scalar_type());
  forward_into(rows_of(x, (hq + hkv) * D), y, table, pos, wq, wk, o, false);
  return y;
}

}  // namespace

void register_qk_norm(pybind11::module& m) {
  namespace py = pybind11;
  m.def("qk_norm_rope", &qk_norm_rope, py::arg("x"), py::arg("n_heads"), py::arg("n_kv_heads"), py::arg("head_dim"),
        py::arg("table"), py::arg("q_weight"), py::arg("k_weight"), py::arg("positions"), py::arg("seq_len"),
        py::arg("eps"), py::arg("half_layout"), py::arg("norm"), py::arg("rot_dim"), py::arg("rot_off"),
        py::arg("in_place"));
  // on row buffers, for callers with an autograd node of their own
  m.def("qk_norm_fwd", [](const at::Tensor& x, const at::Tensor& y, int64_t hq, int64_t hkv, int64_t D,
                          const at::Tensor& table, const OptTensor& pos, int64_t seq_len, const OptTensor& wq,
                          const OptTensor& wk, int64_t rot, int64_t rot_off, bool half_layout, int64_t norm, double eps) {
    forward_into(x, y, table, pos, wq, wk, Options{hq, hkv, D, seq_len, rot, rot_off, norm, half_layout, eps}, false);
  }, py::arg("x"), py::arg("y"), py::arg("n_heads"), py::arg("n_kv_heads"), py::arg("head_dim"), py::arg("table"),
     py::arg("positions"), py::arg("seq_len"), py::arg("q_weight"), py::arg("k_weight"), py::arg("rot_dim"),
     py::arg("rot_off"), py::arg("half_layout"), py::arg("norm"), py::arg("eps"));
  m.def("qk_norm_bwd", [](const at::Tensor& dy, const at::Tensor& x, const at::Tensor& dx, int64_t hq, int64_t hkv,
                          int64_t D, const at::Tensor& table, const OptTensor& pos, int64_t seq_len, const OptTensor& wq,
                          const OptTensor& wk, int64_t rot, int64_t rot_off, bool half_layout, int64_t norm, double eps) {
    auto dw = backward_into(dy, x, dx, table, pos, wq, wk,
                            Options{hq, hkv, D, seq_len, rot, rot_off, norm, half_layout, eps});
    auto or_none = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    return std::make_pair(or_none(dw.first), or_none(dw.second));
  }, py::arg("dy"), py::arg("x"), py::arg("dx"), py::arg("n_heads"), py::arg("n_kv_heads"), py::arg("head_dim"),
     py::arg("table"), py::arg("positions"), py::arg("seq_len"), py::arg("q_weight"), py::arg("k_weight"),
     py::arg("rot_dim"), py::arg("rot_off"), py::arg("half_layout"), py::arg("norm"), py::arg("eps"));
}
