// Python bindings of the per-head norm + rotation kernels (qk_norm.cu): every tensor check is here.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cuda_runtime.h>

namespace astrai_host {
void qk_norm_fwd(const void* x, long long ldx, void* y, long long ldy, int rows, int hq, int hkv, int D,
                 const void* table, int max_pos, const int* pos, int seq_len, const void* wq, const void* wk, int rot,
                 int rot_off, bool half_layout, int norm, int inverse, float eps, int dtype, int device,
                 cudaStream_t s);
int qk_norm_bwd_blocks(int rows, int device);
void qk_norm_bwd(const void* dy, long long lddy, const void* x, long long ldx, void* dx, long long lddx, int rows,
                 int hq, int hkv, int D, const void* table, int max_pos, const int* pos, int seq_len, const void* wq,
                 const void* wk, int rot, int rot_off, bool half_layout, int norm, float eps, void* dwq, void* dwk,
                 float* scratch, int dtype, int device, cudaStream_t s);
}  // namespace astrai_host

namespace {

using OptTensor = c10::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, "qk_norm_rope: bfloat16, float16 or float32, got ", t.scalar_type());
  }
  return -1;
}

// rows of at least `width` columns, of like's type and device, each on a 16-byte boundary
void check_rows(const at::Tensor& t, const at::Tensor& like, int64_t width, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == like.scalar_type(), "qk_norm_rope: ",
              name, " must be a CUDA tensor of the input's type and device");
  TORCH_CHECK(t.dim() == 2 && t.size(0) == like.size(0) && t.size(1) >= width, "qk_norm_rope: ", name,
              " must be [rows, >= (n_heads + n_kv_heads) * head_dim]");
  TORCH_CHECK(t.stride(1) == 1 && (t.stride(0) * t.element_size()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              "qk_norm_rope: ", name, " needs a contiguous inner dimension and 16-byte aligned rows");
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
  TORCH_CHECK(x.size(0) < (1LL << 31), "qk_norm_rope: too many rows");
  check_rows(x, x, (hq + hkv) * D, "x");
  TORCH_CHECK(table.is_cuda() && table.device() == x.device() && table.scalar_type() == at::kFloat &&
                  table.is_contiguous() && table.dim() == 3 && table.size(1) == rot / 2 && table.size(2) == 2 &&
                  reinterpret_cast<uintptr_t>(table.data_ptr()) % 16 == 0,
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
                      (*w)->is_contiguous() && (*w)->numel() == D &&
                      reinterpret_cast<uintptr_t>((*w)->data_ptr()) % 16 == 0,
                  "qk_norm_rope: weights must be contiguous [head_dim], of x's type and device, 16-byte aligned");
    }
  }
  s.rows = (int)x.size(0), s.hq = (int)hq, s.hkv = (int)hkv, s.D = (int)D, s.max_pos = (int)table.size(0);
  s.rot = (int)rot, s.rot_off = (int)rot_off, s.device = x.device().index();
  return s;
}

// y may be x itself
void qk_norm_fwd(const at::Tensor& x, at::Tensor& y, int64_t hq, int64_t hkv, int64_t D, const at::Tensor& table,
                 const OptTensor& pos, int64_t seq_len, const OptTensor& wq, const OptTensor& wk, int64_t rot,
                 int64_t rot_off, bool half_layout, int64_t norm, bool inverse, double eps) {
  const Shape s = check(x, hq, hkv, D, table, pos, seq_len, wq, wk, rot, rot_off, norm);
  check_rows(y, x, (hq + hkv) * D, "y");
  const c10::cuda::CUDAGuard g(x.device());
  astrai_host::qk_norm_fwd(x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), s.rows, s.hq, s.hkv, s.D,
                           table.data_ptr(), s.max_pos, s.pos, (int)seq_len, norm ? wq->data_ptr() : nullptr,
                           norm ? wk->data_ptr() : nullptr, s.rot, s.rot_off, half_layout, (int)norm, inverse,
                           (float)eps, s.dtype, s.device, at::cuda::getCurrentCUDAStream().stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

int64_t qk_norm_bwd_scratch(int64_t rows, int64_t D, int64_t device) {
  return astrai_host::qk_norm_bwd_blocks((int)rows, (int)device) * 2 * D;
}

void qk_norm_bwd(const at::Tensor& dy, const at::Tensor& x, at::Tensor& dx, int64_t hq, int64_t hkv, int64_t D,
                 const at::Tensor& table, const OptTensor& pos, int64_t seq_len, const OptTensor& wq,
                 const OptTensor& wk, int64_t rot, int64_t rot_off, bool half_layout, int64_t norm, double eps,
                 at::Tensor& dwq, at::Tensor& dwk, at::Tensor& scratch) {
  TORCH_CHECK(norm == 1 || norm == 2, "qk_norm_bwd: norm mode");
  const Shape s = check(x, hq, hkv, D, table, pos, seq_len, wq, wk, rot, rot_off, norm);
  check_rows(dy, x, (hq + hkv) * D, "dy");
  check_rows(dx, x, (hq + hkv) * D, "dx");
  for (const auto* w : {&dwq, &dwk})
    TORCH_CHECK(w->device() == x.device() && w->scalar_type() == x.scalar_type() && w->is_contiguous() &&
                    w->numel() == D,
                "qk_norm_bwd: weight gradients must be contiguous [head_dim] of x's type");
  TORCH_CHECK(scratch.device() == x.device() && scratch.scalar_type() == at::kFloat && scratch.is_contiguous() &&
                  scratch.numel() >= qk_norm_bwd_scratch(s.rows, D, s.device),
              "qk_norm_bwd: scratch too small");
  const c10::cuda::CUDAGuard g(x.device());
  astrai_host::qk_norm_bwd(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), dx.data_ptr(), dx.stride(0), s.rows,
                           s.hq, s.hkv, s.D, table.data_ptr(), s.max_pos, s.pos, (int)seq_len, wq->data_ptr(),
                           wk->data_ptr(), s.rot, s.rot_off, half_layout, (int)norm, (float)eps, dwq.data_ptr(),
                           dwk.data_ptr(), scratch.data_ptr<float>(), s.dtype, s.device,
                           at::cuda::getCurrentCUDAStream().stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace

void register_qk_norm(pybind11::module& m) {
  namespace py = pybind11;
  m.def("qk_norm_fwd", &qk_norm_fwd, py::arg("x"), py::arg("y"), py::arg("n_heads"), py::arg("n_kv_heads"),
        py::arg("head_dim"), py::arg("table"), py::arg("positions"), py::arg("seq_len"), py::arg("q_weight"),
        py::arg("k_weight"), py::arg("rot_dim"), py::arg("rot_off"), py::arg("half_layout"), py::arg("norm"),
        py::arg("inverse"), py::arg("eps"));
  m.def("qk_norm_bwd_scratch", &qk_norm_bwd_scratch);
  m.def("qk_norm_bwd", &qk_norm_bwd, py::arg("dy"), py::arg("x"), py::arg("dx"), py::arg("n_heads"),
        py::arg("n_kv_heads"), py::arg("head_dim"), py::arg("table"), py::arg("positions"), py::arg("seq_len"),
        py::arg("q_weight"), py::arg("k_weight"), py::arg("rot_dim"), py::arg("rot_off"), py::arg("half_layout"),
        py::arg("norm"), py::arg("eps"), py::arg("dq_weight"), py::arg("dk_weight"), py::arg("scratch"));
}
