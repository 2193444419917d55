// PyTorch extension `cuda_attn._C`: the reference's pybind entry points (csrc/bindings.cpp:40-54) with
// the same names, argument names and defaults, and the same input checks and error texts
// (bindings.cpp:12-22). Each entry allocates O with empty_like(q), as the reference wrappers did
// (csrc/attn_fused_tc.cu:15), and calls the C ABI of libphantom_attn on the current CUDA stream.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <climits>

#include "../../include/phantom_attn.h"

extern "C" void phantom_attn_pointers_checked(int on);  // capi.cu, between the library and this extension

namespace {

using CFn = int (*)(const void*, const void*, const void*, void*, int, int, int, int, int, void*);

int dtype_code(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PHANTOM_ATTN_F32;
    case at::kHalf: return PHANTOM_ATTN_F16;
    case at::kBFloat16: return PHANTOM_ATTN_BF16;
    default: return -1;
  }
}

void check_inputs(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v) {
  for (const auto* t : {&q, &k, &v}) {
    TORCH_CHECK(t->is_cuda(), "inputs must be CUDA tensors");
    TORCH_CHECK(t->is_contiguous(), "inputs must be contiguous");
    TORCH_CHECK(t->dim() == 4, "inputs must be shaped (B, H, N, d)");
    TORCH_CHECK(t->scalar_type() == q.scalar_type(), "q, k, v must share a dtype");
  }
  TORCH_CHECK(q.sizes() == k.sizes() && q.sizes() == v.sizes(), "q, k, v must have the same shape");
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "q, k, v must be on the same device");
  TORCH_CHECK(q.numel() > 0, "inputs must be non-empty");
  TORCH_CHECK(dtype_code(q) >= 0, "inputs must be float32, float16 or bfloat16 (got ", q.scalar_type(), ")");
}

torch::Tensor call(CFn fn, const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, bool causal) {
  const c10::cuda::CUDAGuard guard(q.device());
  auto o = torch::empty_like(q);
  const int B = (int)q.size(0), H = (int)q.size(1), N = (int)q.size(2), d = (int)q.size(3);
  const int rc = fn(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), B * H, N, d, dtype_code(q),
                    causal ? 1 : 0, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == PHANTOM_ATTN_OK, phantom_attn_last_error());
  return o;
}

template <CFn F>
torch::Tensor checked(torch::Tensor q, torch::Tensor k, torch::Tensor v, bool causal) {
  check_inputs(q, k, v);
  return call(F, q, k, v, causal);
}

torch::Tensor checked_tuned(torch::Tensor q, torch::Tensor k, torch::Tensor v, bool causal, bool double_buffer,
                            int64_t br, int64_t bc) {
  check_inputs(q, k, v);
  const c10::cuda::CUDAGuard guard(q.device());
  auto o = torch::empty_like(q);
  const int B = (int)q.size(0), H = (int)q.size(1), N = (int)q.size(2), d = (int)q.size(3);
  const int rc = phantom_attn_fused_tuned(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), B * H, N, d,
                                          dtype_code(q), causal ? 1 : 0, double_buffer ? 1 : 0, (int)br, (int)bc,
                                          at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == PHANTOM_ATTN_OK, phantom_attn_last_error());
  return o;
}

// ---- paged cache. k_cache, v_cache: (pages, heads, page size, d); page_table (batch, width), kv_lens (batch) and cu_new
// (batch + 1) int32; k_scale, v_scale (pages, heads, page size) float32 with an int8 cache.
using OptTensor = c10::optional<torch::Tensor>;

// A stride that no index reaches (extent 1) may be anything in torch; the library gets one that passes its checks.
long long stride_of(const torch::Tensor& t, int dim, long long unused) { return t.size(dim) == 1 ? unused : t.stride(dim); }

phantom_paged_cache paged_cache(const torch::Tensor& kc, const torch::Tensor& vc, const torch::Tensor& table,
                                const torch::Tensor& lens, const torch::Tensor& cu, const OptTensor& ks, const OptTensor& vs) {
  for (const auto* t : {&kc, &vc, &table, &lens, &cu}) TORCH_CHECK(t->is_cuda(), "inputs must be CUDA tensors");
  for (const auto* t : {&vc, &table, &lens, &cu})
    TORCH_CHECK(t->device() == kc.device(), "all tensors must be on the same device");
  TORCH_CHECK(kc.dim() == 4 && kc.sizes() == vc.sizes(), "k_cache and v_cache must both be shaped (pages, heads, page size, d)");
  TORCH_CHECK(kc.numel() > 0, "inputs must be non-empty");
  TORCH_CHECK(kc.scalar_type() == vc.scalar_type(), "k_cache and v_cache must share a dtype");
  TORCH_CHECK(kc.stride(3) == 1 && vc.stride(3) == 1, "the caches' head dimension must be contiguous");
  const bool int8 = kc.scalar_type() == at::kChar;
  TORCH_CHECK(int8 || kc.scalar_type() == at::kHalf || kc.scalar_type() == at::kBFloat16,
              "the cache must be float16, bfloat16 or int8 (got ", kc.scalar_type(), ")");
  for (const auto* t : {&table, &lens, &cu})
    TORCH_CHECK(t->scalar_type() == at::kInt, "page_table, kv_lens and cu_new must be int32");
  TORCH_CHECK(table.dim() == 2 && lens.dim() == 1 && cu.dim() == 1 && lens.size(0) == table.size(0) &&
                  cu.size(0) == table.size(0) + 1,
              "page_table, kv_lens and cu_new must be shaped (batch, width), (batch) and (batch + 1)");
  TORCH_CHECK(table.numel() > 0, "inputs must be non-empty");
  TORCH_CHECK(lens.is_contiguous() && cu.is_contiguous() && (table.size(1) == 1 || table.stride(1) == 1),
              "page_table's rows, kv_lens and cu_new must be contiguous");
  TORCH_CHECK(kc.size(0) <= INT_MAX && table.size(0) <= INT_MAX && table.size(1) <= INT_MAX && kc.size(1) <= INT_MAX &&
                  kc.size(2) <= INT_MAX, "sizes must fit 32 bits");
  TORCH_CHECK(ks.has_value() == int8 && vs.has_value() == int8, "k_scale and v_scale go with an int8 cache, and only with it");
  phantom_paged_cache c = {};
  const long long d = kc.size(3), page = kc.size(2);
  c.k = kc.data_ptr(), c.v = vc.data_ptr();
  const torch::Tensor* caches[2] = {&kc, &vc};
  for (int t = 0; t < 2; ++t) {
    long long* st = t ? c.v_stride : c.k_stride;
    st[0] = stride_of(*caches[t], 0, kc.size(1) * page * d);
    st[1] = stride_of(*caches[t], 1, page * d);
    st[2] = stride_of(*caches[t], 2, d);
  }
  if (int8) {
    for (int t = 0; t < 2; ++t) {
      const torch::Tensor& s = t ? *vs : *ks;
      TORCH_CHECK(s.is_cuda() && s.device() == kc.device(), "all tensors must be on the same device");
      TORCH_CHECK(s.scalar_type() == at::kFloat && s.dim() == 3 && s.size(0) == kc.size(0) && s.size(1) == kc.size(1) &&
                      s.size(2) == page, "scales must be float32 and shaped (pages, heads, page size)");
      TORCH_CHECK(page == 1 || s.stride(2) == 1, "scales must be contiguous over a page");
      long long* st = t ? c.v_scale_stride : c.k_scale_stride;
      st[0] = stride_of(s, 0, kc.size(1) * page);
      st[1] = stride_of(s, 1, page);
    }
    c.k_scale = ks->data_ptr<float>(), c.v_scale = vs->data_ptr<float>();
  }
  c.page_table = table.data_ptr<int>(), c.kv_lens = lens.data_ptr<int>(), c.cu_new = cu.data_ptr<int>();
  c.batch = (int)table.size(0), c.table_width = (int)table.size(1);
  const long long row = stride_of(table, 0, table.size(1));
  TORCH_CHECK(row <= INT_MAX, "sizes must fit 32 bits");
  c.table_stride = (int)row;
  c.num_pages = (int)kc.size(0), c.page_size = (int)page, c.heads = (int)kc.size(1), c.head_dim = (int)d;
  c.dtype = int8 ? PHANTOM_ATTN_I8 : dtype_code(kc);
  return c;
}

// While it lives, the library takes this thread's pointers as checked (they are, by the tensors' devices).
struct PointersChecked {
  PointersChecked() { phantom_attn_pointers_checked(1); }
  ~PointersChecked() { phantom_attn_pointers_checked(0); }
};

// A packed (tokens, heads, d) tensor of new tokens.
void check_packed(const torch::Tensor& t, const torch::Tensor& kc, const char* what) {
  TORCH_CHECK(t.is_cuda(), "inputs must be CUDA tensors");
  TORCH_CHECK(t.device() == kc.device(), "all tensors must be on the same device");
  TORCH_CHECK(t.dim() == 3 && t.size(2) == kc.size(3), what, " must be shaped (tokens, heads, d) with the cache's d");
  TORCH_CHECK(t.stride(2) == 1, what, "'s head dimension must be contiguous");
  TORCH_CHECK(t.size(0) <= INT_MAX && t.size(1) <= INT_MAX, "sizes must fit 32 bits");
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, what, " must be float16 or bfloat16 (got ",
              t.scalar_type(), ")");
}

void paged_append(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& kc, const torch::Tensor& vc,
                  const torch::Tensor& table, const torch::Tensor& lens, const torch::Tensor& cu, const OptTensor& ks,
                  const OptTensor& vs) {
  const phantom_paged_cache c = paged_cache(kc, vc, table, lens, cu, ks, vs);
  check_packed(k, kc, "k");
  check_packed(v, kc, "v");
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), "k and v must have the same shape and dtype");
  TORCH_CHECK(k.size(1) == kc.size(1), "k and v must have the cache's heads");
  if (k.size(0) == 0) return;
  const c10::cuda::CUDAGuard guard(kc.device());
  const long long d = k.size(2), token = k.size(1) * d;
  const PointersChecked checked;
  const int rc = phantom_attn_paged_append(&c, k.data_ptr(), v.data_ptr(), stride_of(k, 0, token), stride_of(k, 1, d),
                                           stride_of(v, 0, token), stride_of(v, 1, d), (int)k.size(0), dtype_code(k),
                                           at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == PHANTOM_ATTN_OK, phantom_attn_last_error());
}

std::tuple<torch::Tensor, torch::Tensor> paged_read(const torch::Tensor& kc, const torch::Tensor& vc, const torch::Tensor& table,
                                                    const torch::Tensor& lens, const torch::Tensor& cu, int64_t total,
                                                    bool bf16, const OptTensor& ks, const OptTensor& vs) {
  const phantom_paged_cache c = paged_cache(kc, vc, table, lens, cu, ks, vs);
  TORCH_CHECK(total >= 0 && total <= INT_MAX, "total must be from 0 to 2^31 - 1 (got ", total, ")");
  const c10::cuda::CUDAGuard guard(kc.device());
  const auto opts = kc.options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
  auto k = torch::empty({total, kc.size(1), kc.size(3)}, opts), v = torch::empty_like(k);
  if (total == 0) return {k, v};
  const PointersChecked checked;
  const int rc = phantom_attn_paged_read(&c, k.data_ptr(), v.data_ptr(), (int)total, bf16 ? PHANTOM_ATTN_BF16 : PHANTOM_ATTN_F16,
                                         at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == PHANTOM_ATTN_OK, phantom_attn_last_error());
  return {k, v};
}

torch::Tensor paged_attn(const torch::Tensor& q, const torch::Tensor& kc, const torch::Tensor& vc, const torch::Tensor& table,
                         const torch::Tensor& lens, const torch::Tensor& cu, const OptTensor& ks, const OptTensor& vs,
                         bool causal, int64_t max_new, double scale) {
  const phantom_paged_cache c = paged_cache(kc, vc, table, lens, cu, ks, vs);
  check_packed(q, kc, "q");
  TORCH_CHECK(max_new >= 0 && max_new <= INT_MAX, "max_new must be from 0 to 2^31 - 1 (got ", max_new, ")");
  const c10::cuda::CUDAGuard guard(kc.device());
  auto o = torch::empty(q.sizes(), q.options());
  if (q.numel() == 0) return o;
  const long long d = q.size(2);
  const PointersChecked checked;
  const int rc = phantom_attn_paged(&c, q.data_ptr(), stride_of(q, 0, q.size(1) * d), stride_of(q, 1, d), o.data_ptr(),
                                    (int)q.size(0), (int)q.size(1), dtype_code(q), causal ? 1 : 0, (float)scale, (int)max_new,
                                    at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == PHANTOM_ATTN_OK, phantom_attn_last_error());
  return o;
}

int device_status() {
  int status = 0;
  const int rc = phantom_attn_device_status(&status);
  TORCH_CHECK(rc == PHANTOM_ATTN_OK || rc == PHANTOM_ATTN_ERR_DEVICE, phantom_attn_last_error());
  return status;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "B200 (sm_100a) attention kernels: naive, tiled, fused, fused_tuned, fused_tc";
  m.def("naive", &checked<phantom_attn_naive>, "v1 entry point (fp32 CUDA-core fused kernel on sm_100a)",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("causal") = false);
  m.def("tiled", &checked<phantom_attn_tiled>, "v2 entry point (fp32 CUDA-core fused kernel on sm_100a)",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("causal") = false);
  m.def("fused", &checked<phantom_attn_fused>, "v3 fused online-softmax attention (fp32 CUDA cores)",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("causal") = false);
  m.def("fused_tuned", &checked_tuned,
        "v3.1/v3.2 entry point; (br, bc) validated, runs on the tcgen05 tensor-core kernel (fp16/bf16)",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("causal") = false, py::arg("double_buffer") = true,
        py::arg("br") = 64, py::arg("bc") = 32);
  m.def("fused_tc", &checked<phantom_attn_fused_tc>,
        "v4 fused attention on tcgen05 tensor cores with TMEM accumulators (fp16/bf16, d 64/128)", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("causal") = false);
  m.def("paged_append", &paged_append, "write new tokens' keys and values into a paged cache", py::arg("k"), py::arg("v"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("page_table"), py::arg("kv_lens"), py::arg("cu_new"),
        py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none());
  m.def("paged_read", &paged_read, "read cached tokens back, packed", py::arg("k_cache"), py::arg("v_cache"),
        py::arg("page_table"), py::arg("kv_lens"), py::arg("cu_new"), py::arg("total"), py::arg("bf16"),
        py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none());
  m.def("paged_attn", &paged_attn, "attention of new tokens over a paged cache", py::arg("q"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("page_table"), py::arg("kv_lens"), py::arg("cu_new"), py::arg("k_scale") = py::none(),
        py::arg("v_scale") = py::none(), py::arg("causal") = true, py::arg("max_new") = 0, py::arg("scale") = 0.0);
  m.def("device_status", &device_status, "read and clear the device status word (0 = no wait expired)");
}
