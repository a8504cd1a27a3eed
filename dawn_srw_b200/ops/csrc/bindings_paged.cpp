// Python bindings of the paged key/value cache (see bindings.cpp).  Arguments are refused with ValueError
// before anything touches a device, so that a refusal reads the same with and without a GPU.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "dsb_api_paged.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

#define REFUSE_UNLESS(cond, ...) TORCH_CHECK_VALUE(cond, "paged cache: ", __VA_ARGS__)

bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

DsbPaged view(const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs, const Tensor& table,
              const Tensor& lengths, const OptTensor& starts, int64_t N, Tensor& status) {
  DsbPaged c = {};
  REFUSE_UNLESS(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
                "k and v pages must have one shape [n_pages, heads, page, dim] and one type");
  REFUSE_UNLESS(k.is_contiguous() && v.is_contiguous(), "pages must be contiguous");
  const auto type = k.scalar_type();
  REFUSE_UNLESS(type == torch::kBFloat16 || type == torch::kFloat8_e4m3fn || type == torch::kInt8,
                "pages must be bfloat16, float8_e4m3fn or int8");
  c.kind = type == torch::kBFloat16 ? 0 : type == torch::kFloat8_e4m3fn ? 1 : 2;
  const int64_t page = k.size(2), dh = k.size(3), H = k.size(1);
  REFUSE_UNLESS(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page size ", page,
                " is not a power of two from 16 to 256");
  REFUSE_UNLESS(dh >= 16 && dh <= 128 && dh % 16 == 0, "head dimension ", dh,
                " is not supported by the kernels (multiple of 16, at most 128)");
  REFUSE_UNLESS(H >= 1 && H <= 65535 && k.size(0) <= 0x7fffffffLL, "number of heads or pages");
  const bool scaled = c.kind != 0;
  REFUSE_UNLESS(ks.has_value() == scaled && vs.has_value() == scaled,
                "8-bit pages come with k_scale and v_scale, bf16 pages without");
  if (scaled) {
    for (const Tensor* s : {&*ks, &*vs})
      REFUSE_UNLESS(s->scalar_type() == torch::kFloat32 && s->is_contiguous() && s->dim() == 3 &&
                        s->size(0) == k.size(0) && s->size(1) == H && s->size(2) == page && s->device() == k.device(),
                    "scales must be contiguous float32 [n_pages, heads, page] on the pages' device");
    c.k_scale = ks->data_ptr<float>();
    c.v_scale = vs->data_ptr<float>();
  }
  REFUSE_UNLESS(table.dim() == 2 && table.scalar_type() == torch::kInt32 && table.is_contiguous() &&
                    table.size(1) <= (1 << 30) / page,
                "table must be a contiguous int32 [sequences, pages] of at most 2^30 positions each");
  const int64_t B = table.size(0);
  REFUSE_UNLESS(lengths.dim() == 1 && lengths.size(0) == B && lengths.scalar_type() == torch::kInt32 &&
                    lengths.is_contiguous(),
                "lengths must be a contiguous int32 [sequences]");
  if (starts.has_value()) {
    REFUSE_UNLESS(starts->dim() == 1 && starts->size(0) == B + 1 && starts->scalar_type() == torch::kInt32 &&
                      starts->is_contiguous() && starts->device() == k.device(),
                  "starts must be a contiguous int32 [sequences + 1] on the pages' device");
    c.starts = starts->data_ptr<int>();
  } else {
    REFUSE_UNLESS(N == B, "without starts every sequence has one new token: ", N, " rows for ", B, " sequences");
  }
  REFUSE_UNLESS(N <= (1 << 30) && B <= 65535, "more than 65535 sequences, or too many rows");
  REFUSE_UNLESS(v.device() == k.device() && table.device() == k.device() && lengths.device() == k.device(),
                "pages, table and lengths must be on one device");
  REFUSE_UNLESS(aligned(k) && aligned(v) && (!scaled || (aligned(*ks) && aligned(*vs))),
                "pages and scales must be 16-byte aligned for the kernels");
  REFUSE_UNLESS(k.is_cuda(), "the kernels need CUDA tensors");
  REFUSE_UNLESS(status.device() == k.device(), "status word on another device");
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.table = table.data_ptr<int>();
  c.lengths = lengths.data_ptr<int>();
  c.status = status.data_ptr<int>();
  c.n_pages = static_cast<int>(k.size(0));
  c.H = static_cast<int>(H);
  c.page = static_cast<int>(page);
  c.dh = static_cast<int>(dh);
  c.B = static_cast<int>(B);
  c.width = static_cast<int>(table.size(1));
  c.N = static_cast<int>(N);
  return c;
}

void check_rows(const Tensor& x, const Tensor& pages, const char* name) {
  REFUSE_UNLESS(x.dim() == 3 && x.size(2) == pages.size(3), name, " must be [rows, heads, dim] with the pages' head dimension");
  REFUSE_UNLESS(x.scalar_type() == torch::kFloat32 || x.scalar_type() == torch::kBFloat16, name,
                " must be float32 or bfloat16");
  REFUSE_UNLESS(x.device() == pages.device(), name, " must be on the pages' device");
}

// Unit inner stride and 16-byte aligned rows, as the kernels read them; anything else is copied.
Tensor rows_of(const Tensor& x) {
  const int64_t step = x.scalar_type() == torch::kBFloat16 ? 8 : 4;
  if (x.stride(2) == 1 && x.stride(0) % step == 0 && x.stride(1) % step == 0 && x.stride(0) >= 0 && x.stride(1) >= 0 &&
      aligned(x))
    return x;
  return x.clone(at::MemoryFormat::Contiguous);
}

void paged_write(const Tensor& k, const Tensor& v, const Tensor& kp, const Tensor& vp, const Tensor& table,
                 const Tensor& lengths, const OptTensor& starts, const OptTensor& ks, const OptTensor& vs, Tensor& status) {
  TORCH_CHECK_VALUE(kp.dim() == 4, "paged cache: pages must be [n_pages, heads, page, dim]");
  check_rows(k, kp, "k");
  check_rows(v, kp, "v");
  REFUSE_UNLESS(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.size(1) == kp.size(1),
                "k and v must have one type and one shape with the pages' heads");
  DsbPaged c = view(kp, vp, ks, vs, table, lengths, starts, k.size(0), status);
  const at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(kp.device());
  const Tensor kr = rows_of(k), vr = rows_of(v);
  const int rc = dsb_paged_write(&c, kr.data_ptr(), vr.data_ptr(), kr.scalar_type() == torch::kBFloat16, kr.stride(0),
                                 kr.stride(1), vr.stride(0), vr.stride(1), at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "dsb_paged_write failed with code ", rc);
}

std::vector<Tensor> paged_read(const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& lengths,
                               int64_t max_len, const OptTensor& ks, const OptTensor& vs, bool bf16, Tensor& status) {
  REFUSE_UNLESS(max_len >= 0 && max_len <= 0x7fffffffLL, "max_len ", max_len);
  const OptTensor none;
  const int64_t B = table.dim() == 2 ? table.size(0) : 0;
  DsbPaged c = view(kp, vp, ks, vs, table, lengths, none, B, status);
  REFUSE_UNLESS(B * kp.size(1) <= 0x7fffffffLL, "too many sequences");
  const at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(kp.device());
  const auto opt = kp.options().dtype(bf16 ? torch::kBFloat16 : torch::kFloat32);
  Tensor k = torch::empty({B, kp.size(1), max_len, kp.size(3)}, opt), v = torch::empty_like(k);
  const int rc = dsb_paged_read(&c, k.data_ptr(), v.data_ptr(), bf16, static_cast<int>(max_len),
                                at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "dsb_paged_read failed with code ", rc);
  return {k, v};
}

Tensor paged_attention(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& lengths,
                       const OptTensor& starts, const OptTensor& ks, const OptTensor& vs, c10::optional<int64_t> max_new,
                       c10::optional<int64_t> window, int64_t sinks, c10::optional<double> scale, Tensor& status) {
  TORCH_CHECK_VALUE(kp.dim() == 4, "paged cache: pages must be [n_pages, heads, page, dim]");
  check_rows(q, kp, "q");
  const int64_t Hq = q.size(1);
  REFUSE_UNLESS(Hq >= 1 && kp.size(1) >= 1 && Hq % kp.size(1) == 0, Hq, " query heads are no multiple of the pages' ",
                kp.size(1), " heads");
  REFUSE_UNLESS(q.size(0) * (Hq / kp.size(1)) <= (1 << 30), "too many rows");
  REFUSE_UNLESS(!window.has_value() || *window >= 1, "window must be at least 1 (None: no window)");
  REFUSE_UNLESS(sinks >= 0, "sinks must not be negative");
  REFUSE_UNLESS(!max_new.has_value() || *max_new >= 0, "max_new must not be negative");
  DsbPaged c = view(kp, vp, ks, vs, table, lengths, starts, q.size(0), status);
  const at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(kp.device());
  const Tensor qr = rows_of(q.scalar_type() == torch::kBFloat16 ? q : q.to(torch::kBFloat16));
  Tensor out = torch::empty({q.size(0), Hq, q.size(2)}, kp.options().dtype(torch::kBFloat16));
  const int64_t top = 0x7fffffffLL;
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(2)));
  const int hint = static_cast<int>(std::min<int64_t>(max_new.has_value() ? *max_new : starts.has_value() ? q.size(0) : 1, top));
  const int win = window.has_value() ? static_cast<int>(std::min(*window, top)) : 0, snk = static_cast<int>(std::min(sinks, top));
  const int64_t bytes = dsb_paged_attention_workspace(&c, static_cast<int>(Hq), hint, win, snk);
  Tensor ws;                    // of this call alone: captured graphs and streams share nothing
  if (bytes > 0) ws = torch::empty({bytes}, kp.options().dtype(torch::kUInt8));
  const int rc = dsb_paged_attention(&c, qr.data_ptr(), qr.stride(0), qr.stride(1), out.data_ptr(), static_cast<int>(Hq),
                                     hint, win, snk, static_cast<float>(s),
                                     bytes > 0 ? ws.data_ptr() : nullptr, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "dsb_paged_attention failed with code ", rc);
  return out;
}

}  // namespace

void register_paged(py::module_& m) {
  m.def("paged_write", &paged_write);
  m.def("paged_read", &paged_read);
  m.def("paged_attention", &paged_attention);
}
