// Python bindings of the 8-bit paged KV cache kernels (kv8.cu): every tensor check is here.
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cuda_runtime.h>

#include "bind_util.h"

namespace astrai_host {
bool kv8_block_supported(int block);
void kv8_append(const void* k, const long long* ks, const void* v, const long long* vs, void* kc, void* vc, float* ka,
                float* va, const int* table, const int* starts, const int* lens, int B, int S, int Hkv, int D,
                int page_size, int n_pages, int max_pages, int block, int dtype, cudaStream_t s);
void kv8_gather(const void* kc, const void* vc, const float* ka, const float* va, const int* table, const int* starts,
                const int* lens, void* ko, void* vo, int B, int total, int Hkv, int D, int page_size, int n_pages,
                int max_pages, int block, int dtype, cudaStream_t s);
long long kv8_attend_workspace(int B, int S, int Hq, int Hkv, int D, int page_size, int max_pages, int device);
void kv8_attend(const void* q, const long long* qs, const void* kc, const void* vc, const float* ka, const float* va,
                const int* table, const int* lens, const int* starts, void* out, float* workspace, int B, int S,
                int Hq, int Hkv, int D, int page_size, int n_pages, int max_pages, int block, float scale, int dtype,
                int device, cudaStream_t s);
}  // namespace astrai_host

namespace {

using namespace astrai_bind;

// Numbers enter messages as text made here: a build whose compiler links its own static libstdc++ must not
// stream them through the locale of the one that torch loaded.
std::string text(int64_t n) { return std::to_string(n); }
std::string text(at::IntArrayRef sizes) {
  std::string s = "[";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + "]";
}

struct Cache {
  int n_pages, Hkv, page_size, D, block;
};

Cache check_cache(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ka, const at::Tensor& va) {
  for (const auto* t : {&kc, &vc})
    TORCH_CHECK(t->is_cuda() && t->device() == kc.device() && t->scalar_type() == at::kChar && t->dim() == 4 &&
                    t->is_contiguous() && t->sizes() == kc.sizes(),
                "kv8: the caches must be contiguous CUDA int8 [n_pages, n_kv_heads, page_size, head_dim]");
  for (const auto* t : {&ka, &va})
    TORCH_CHECK(t->is_cuda() && t->device() == kc.device() && t->scalar_type() == at::kFloat && t->dim() == 3 &&
                    t->is_contiguous() && t->sizes() == ka.sizes(),
                "kv8: the magnitudes must be contiguous CUDA fp32 [n_pages, n_kv_heads, page_size / block]");
  TORCH_CHECK(kc.size(3) == 64 || kc.size(3) == 128, "kv8: head_dim must be 64 or 128, got ", text(kc.size(3)));
  TORCH_CHECK(kc.size(1) >= 1 && ka.size(0) == kc.size(0) && ka.size(1) == kc.size(1) && ka.size(2) >= 1 &&
                  kc.size(2) % ka.size(2) == 0,
              "kv8: cache ", text(kc.sizes()), " and magnitudes ", text(ka.sizes()), " do not belong together");
  const int64_t block = kc.size(2) / ka.size(2);
  TORCH_CHECK(astrai_host::kv8_block_supported((int)block), "kv8: block must be 16, 32, 64 or 128 tokens, got ", text(block));
  TORCH_CHECK(kc.size(0) < (1LL << 31) && kc.size(1) < 65536 && kc.size(2) < (1LL << 30), "kv8: cache too large");
  for (const auto* t : {&kc, &vc})
    TORCH_CHECK(on_grid(*t), "kv8: the caches must be 16-byte aligned");
  return {(int)kc.size(0), (int)kc.size(1), (int)kc.size(2), (int)kc.size(3), (int)block};
}

const int* check_i32(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous() &&
                  t.numel() == n,
              "kv8: ", name, " must be a contiguous CUDA int32 tensor of ", text(n), " entries");
  return t.data_ptr<int>();
}

// page_table [B, max_pages] -> max_pages
int check_table(const at::Tensor& table, const at::Tensor& like, int64_t B, const Cache& c) {
  TORCH_CHECK(table.dim() == 2 && table.size(0) == B && table.size(1) >= 1, "kv8: page_table must be [batch, pages >= 1]");
  check_i32(table, like, table.numel(), "page_table");
  TORCH_CHECK(table.size(1) * c.page_size < (1LL << 30), "kv8: rows of at most 2^30 tokens");
  return (int)table.size(1);
}

int dtype_code(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, "kv8: ", name,
              " must be bfloat16 or float16, got ", t.scalar_type());
  return t.scalar_type() == at::kHalf;
}

// [B, S, H, D] as the kernels read it: a contiguous last dimension and 16-byte aligned rows of any stride;
// copied if it is not (contiguous() would return a contiguous tensor as it is, wherever it starts)
at::Tensor heads_of(const at::Tensor& t) {
  if (t.dim() != 4) return t;  // refused by check_heads
  bool ok = t.stride(3) == 1 && on_grid(t);
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
at::Tensor int32_of(const at::Tensor& t) {
  return t.scalar_type() == at::kInt && t.is_contiguous() ? t : t.to(at::kInt).contiguous();
}

// strides of the batch, token and head dimensions
void check_heads(const at::Tensor& t, const at::Tensor& like, const char* name, long long* strides) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.dim() == 4, "kv8: ", name,
              " must be a CUDA [batch, tokens, heads, head_dim] tensor on the cache's device");
  TORCH_CHECK(t.stride(3) == 1 && on_grid(t), "kv8: ", name,
              " needs a contiguous last dimension and a 16-byte aligned start");
  for (int i = 0; i < 3; ++i) {
    TORCH_CHECK(t.size(i) <= 1 || t.stride(i) % 8 == 0, "kv8: ", name, " rows must be 16-byte aligned");
    strides[i] = t.stride(i);
  }
}

void kv8_append(const at::Tensor& k_in, const at::Tensor& v_in, at::Tensor& kc, at::Tensor& vc, at::Tensor& ka,
                at::Tensor& va, const at::Tensor& table_in, const at::Tensor& starts_in, const at::Tensor& lens_in) {
  const Cache c = check_cache(kc, vc, ka, va);
  const at::Tensor k = heads_of(k_in), v = heads_of(v_in);
  const at::Tensor table = int32_of(table_in), starts = int32_of(starts_in), lens = int32_of(lens_in);
  long long ks[3], vs[3];
  check_heads(k, kc, "k", ks);
  check_heads(v, kc, "v", vs);
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), "kv8_append: k and v differ");
  TORCH_CHECK(k.size(2) == c.Hkv && k.size(3) == c.D, "kv8_append: k ", text(k.sizes()),
              " does not fit the cache ", text(kc.sizes()));
  const int dt = dtype_code(k, "k");
  const int64_t B = k.size(0), S = k.size(1);
  const int mp = check_table(table, kc, B, c);
  const int* st = check_i32(starts, kc, B, "starts");
  const int* ln = check_i32(lens, kc, B, "lens");
  TORCH_CHECK(S < (1LL << 30) && 2 * B * c.Hkv * (S / c.block + 2) < (1LL << 31), "kv8_append: too many tokens");
  const c10::cuda::CUDAGuard g(k.device());
  astrai_host::kv8_append(k.data_ptr(), ks, v.data_ptr(), vs, kc.data_ptr(), vc.data_ptr(), ka.data_ptr<float>(),
                          va.data_ptr<float>(), table.data_ptr<int>(), st, ln, (int)B, (int)S, c.Hkv, c.D, c.page_size,
                          c.n_pages, mp, c.block, dt, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

std::pair<at::Tensor, at::Tensor> kv8_gather(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ka,
                                             const at::Tensor& va, const at::Tensor& table_in,
                                             const OptTensor& starts_in, const at::Tensor& lens_in, int64_t total,
                                             at::ScalarType dtype) {
  const Cache c = check_cache(kc, vc, ka, va);
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kHalf, "kv8_gather: bfloat16 or float16, got ", dtype);
  TORCH_CHECK(total >= 0 && total < (1LL << 30), "kv8_gather: total must be in [0, 2^30)");
  TORCH_CHECK(table_in.size(0) < 65536, "kv8_gather: at most 65535 rows");
  const at::Tensor table = int32_of(table_in), lens = int32_of(lens_in);
  const int64_t B = table.dim() == 2 ? table.size(0) : -1;
  const int mp = check_table(table, kc, B, c);
  at::Tensor starts;
  const int* st = nullptr;
  if (given(starts_in)) {
    starts = int32_of(*starts_in);
    st = check_i32(starts, kc, B, "starts");
  }
  const int* ln = check_i32(lens, kc, B, "lens");
  const c10::cuda::CUDAGuard g(kc.device());
  const int64_t sizes[4] = {B, total, c.Hkv, c.D};
  auto ko = new_like(kc, sizes, dtype), vo = new_like(kc, sizes, dtype);
  astrai_host::kv8_gather(kc.data_ptr(), vc.data_ptr(), ka.data_ptr<float>(), va.data_ptr<float>(),
                          table.data_ptr<int>(), st, ln, ko.data_ptr(), vo.data_ptr(), (int)B, (int)total, c.Hkv, c.D,
                          c.page_size, c.n_pages, mp, c.block, dtype == at::kHalf, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {ko, vo};
}

// fp32 elements of workspace that kv8_attend needs for these sizes (0: none)
int64_t kv8_attend_workspace(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, int64_t page_size,
                             int64_t max_pages, int64_t device) {
  TORCH_CHECK(B >= 0 && S >= 0 && Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && page_size >= 1 && max_pages >= 1 &&
                  max_pages * page_size < (1LL << 30) && S * (Hq / Hkv) < (1LL << 24),
              "kv8_attend_workspace: sizes");
  if (B == 0 || S == 0) return 0;
  return astrai_host::kv8_attend_workspace((int)B, (int)S, (int)Hq, (int)Hkv, (int)D, (int)page_size, (int)max_pages,
                                           (int)device);
}

at::Tensor kv8_attend(const at::Tensor& q_in, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ka,
                      const at::Tensor& va, const at::Tensor& table_in, const at::Tensor& lens_in,
                      const OptTensor& starts_in, const OptTensor& workspace, double scale) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && q_in.requires_grad()), "kv8_attention has no gradient: detach the query");
  TORCH_CHECK(!q_in._fw_grad(0).defined(), "kv8_attention has no forward-mode derivative");
  const Cache c = check_cache(kc, vc, ka, va);
  const at::Tensor q = heads_of(q_in), table = int32_of(table_in), lens = int32_of(lens_in);
  long long qs[3];
  check_heads(q, kc, "q", qs);
  const int dt = dtype_code(q, "q");
  const int64_t B = q.size(0), S = q.size(1), Hq = q.size(2);
  TORCH_CHECK(q.size(3) == c.D && Hq % c.Hkv == 0 && Hq >= 1, "kv8_attention: q ", text(q.sizes()),
              " does not fit the cache ", text(kc.sizes()));
  const int mp = check_table(table, kc, B, c);
  const int* ln = check_i32(lens, kc, B, "lens");
  at::Tensor starts;
  const int* st = nullptr;
  if (given(starts_in)) {
    starts = int32_of(*starts_in);
    st = check_i32(starts, kc, B, "starts");
  }
  const int64_t units = ((int64_t)mp * c.page_size + 127) / 128, rows = S * (Hq / c.Hkv);
  TORCH_CHECK(rows < (1LL << 24) && (units + 8) * 1024 < (1LL << 31) && (units + 8) * c.Hkv * (rows / 8 + 1) < (1LL << 31) &&
                  B * c.Hkv * (rows + 16) < (1LL << 31),
              "kv8_attention: too many rows or pages");
  const int64_t need = kv8_attend_workspace(B, S, Hq, c.Hkv, c.D, c.page_size, mp, q.device().index());
  const c10::cuda::CUDAGuard g(q.device());
  auto out = new_like(q, {B, S, Hq, c.D}, q.scalar_type());
  at::Tensor ws;
  float* wp = nullptr;
  if (need > 0) {
    if (given(workspace)) {
      ws = *workspace;
      TORCH_CHECK(ws.device() == q.device() && ws.scalar_type() == at::kFloat && ws.is_contiguous() && ws.numel() >= need &&
                      on_grid(ws),
                  "kv8_attention: workspace must be contiguous fp32 of at least ", text(need), " elements");
    } else {
      ws = new_like(q, {need}, at::kFloat);
    }
    wp = ws.data_ptr<float>();
  }
  astrai_host::kv8_attend(q.data_ptr(), qs, kc.data_ptr(), vc.data_ptr(), ka.data_ptr<float>(), va.data_ptr<float>(),
                          table.data_ptr<int>(), ln, st, out.data_ptr(), wp, (int)B, (int)S, (int)Hq, c.Hkv, c.D,
                          c.page_size, c.n_pages, mp, c.block, (float)scale, dt, q.device().index(), stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

}  // namespace

void register_kv8(pybind11::module& m) {
  namespace py = pybind11;
  m.def("kv8_append", &kv8_append, py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("k_absmax"), py::arg("v_absmax"), py::arg("page_table"), py::arg("starts"), py::arg("lens"));
  m.def("kv8_gather", &kv8_gather, py::arg("k_cache"), py::arg("v_cache"), py::arg("k_absmax"), py::arg("v_absmax"),
        py::arg("page_table"), py::arg("starts"), py::arg("lens"), py::arg("total"), py::arg("dtype"));
  m.def("kv8_attend_workspace", &kv8_attend_workspace, py::arg("batch"), py::arg("tokens"), py::arg("n_heads"),
        py::arg("n_kv_heads"), py::arg("head_dim"), py::arg("page_size"), py::arg("max_pages"), py::arg("device"));
  m.def("kv8_attend", &kv8_attend, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"), py::arg("k_absmax"),
        py::arg("v_absmax"), py::arg("page_table"), py::arg("lens"), py::arg("starts"),
        py::arg("workspace"), py::arg("scale"));
}
