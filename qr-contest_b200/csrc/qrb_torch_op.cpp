// qrb200 -- PyTorch operator registration: torch.ops.qrb200.geqrf(A) -> (H, tau, info), and the
// layer operators (rms_norm, quantize_rows, linear and their backward passes).
//
// geqrf is the operator form of the reference entry point custom_kernel(data) -> (H, tau)
// (reflection_no_reflectors.py:181-196) for callers that dispatch through the torch operator
// registry (torch.ops, TorchScript, torch.compile graphs).  It is a thin layer over the C ABI of
// libqrb200.so (include/qrb200.h): no kernel lives here.
//   * A: (..., n, n) CUDA tensor of any floating dtype; float32 / bfloat16 / float16 are read
//     and written natively, others are converted to float32 first and the factors back, like
//     the reference's .to(float32) / .to(dtype) (:183, :196).
//   * H (..., n, n) and tau (..., n) in A's dtype, info (...) int32 QRB200_INFO_* bits.
//   * Enqueued on the current CUDA stream of A's device; the workspace comes from torch's
//     caching allocator.  A bad argument or a CUDA error raises (TORCH_CHECK).
// A Meta kernel gives shapes and dtypes without running anything.
//
// The layer operators take rows in place where one row stride describes them (any leading shape,
// slices and expanded tensors included) and copy otherwise; a wrong argument raises ValueError or
// TypeError before anything is allocated.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "qrb200.h"
#include "qrb200_layer.h"
#include "qrb_torch_layers.h"

namespace {

bool native(at::ScalarType t) {
  return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf;
}

int32_t dtype_code(at::ScalarType t) {
  return t == at::kFloat ? QRB200_F32 : (t == at::kBFloat16 ? QRB200_BF16 : QRB200_F16);
}

std::vector<int64_t> lead_sizes(const at::Tensor& A) {
  return std::vector<int64_t>(A.sizes().begin(), A.sizes().end() - 2);
}

void check_square(const at::Tensor& A) {
  TORCH_CHECK(A.dim() >= 2 && A.size(-1) == A.size(-2),
              "qrb200::geqrf expects a (..., n, n) tensor, got ", A.sizes());
  TORCH_CHECK(at::isFloatingType(A.scalar_type()), "qrb200::geqrf expects a floating dtype");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> geqrf_cuda(const at::Tensor& data) {
  check_square(data);
  TORCH_CHECK(data.is_cuda(), "qrb200::geqrf: the CUDA kernel takes CUDA tensors");
  const c10::cuda::CUDAGuard guard(data.device());
  at::Tensor A = (native(data.scalar_type()) ? data : data.to(at::kFloat)).contiguous();
  const int64_t n = A.size(-1);
  auto lead = lead_sizes(A);
  int64_t batch = 1;
  for (int64_t d : lead) batch *= d;
  at::Tensor H = at::empty_like(A);
  auto tsz = lead;
  tsz.push_back(n);
  at::Tensor tau = at::empty(tsz, A.options());
  at::Tensor info = at::zeros(lead, A.options().dtype(at::kInt));
  if (batch > 0 && n > 0) {
    size_t ws_bytes = 0;
    int rc = qrb200_workspace_bytes(batch, (int32_t)n, &ws_bytes);
    TORCH_CHECK(rc == QRB200_OK, "qrb200_workspace_bytes: ", qrb200_status_string(rc));
    at::Tensor ws = at::empty({(int64_t)ws_bytes}, A.options().dtype(at::kByte));
    rc = qrb200_geqrf_batched(A.data_ptr(), H.data_ptr(), tau.data_ptr(),
                              info.data_ptr<int32_t>(), batch, (int32_t)n,
                              dtype_code(A.scalar_type()), ws_bytes ? ws.data_ptr() : nullptr,
                              ws_bytes, at::cuda::getCurrentCUDAStream().stream());
    TORCH_CHECK(rc == QRB200_OK, "qrb200_geqrf_batched: ", qrb200_status_string(rc),
                rc == QRB200_ERR_CUDA ? qrb200_last_cuda_error() : "");
  }
  if (!native(data.scalar_type())) {
    H = H.to(data.scalar_type());
    tau = tau.to(data.scalar_type());
  }
  return {H, tau, info};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> geqrf_meta(const at::Tensor& data) {
  check_square(data);
  auto lead = lead_sizes(data);
  auto tsz = lead;
  tsz.push_back(data.size(-1));
  return {at::empty_like(data), at::empty(tsz, data.options()),
          at::empty(lead, data.options().dtype(at::kInt))};
}

// ---------------------------------------------------------------- layer operators
using qrb200::OptTensor;

int32_t layer_code(at::ScalarType t) {
  return t == at::kFloat8_e4m3fn ? QRB200_E4M3 : dtype_code(t);
}

void check_rc(int rc, const char* where) {
  TORCH_CHECK(rc == QRB200_OK, where, ": ", qrb200_status_string(rc), " (status ", rc, ")",
              rc == QRB200_ERR_CUDA ? ": " : "", rc == QRB200_ERR_CUDA ? qrb200_last_cuda_error() : "");
}

void check_device(const at::Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.is_cuda() || x.is_meta(), "qrb200: ", name, " must be a CUDA tensor (got one on ", x.device(), ")");
}
void check_with(const at::Tensor& t, const at::Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.device() == x.device(), "qrb200: ", name, " is on ", t.device(), ", the input on ", x.device());
}
void check_type(bool ok, const char* name, at::ScalarType t) {
  TORCH_CHECK_TYPE(ok, "qrb200: ", name, " cannot be of type ", t);
}

// A tensor (..., d) as rows of d contiguous elements, `ld` apart: itself where one stride describes
// it, a contiguous copy otherwise.  apart: rows may not overlap (matrix-product operands).
struct Rows {
  at::Tensor t;
  int64_t rows, d, ld;
};
Rows as_rows(const at::Tensor& x, bool apart = false) {
  Rows r{x, 1, x.size(-1), x.size(-1)};
  for (int64_t i = 0; i < x.dim() - 1; ++i) r.rows *= x.size(i);
  if (r.rows == 0 || r.d == 0 || x.is_meta()) return r;
  bool fits = r.d == 1 || x.stride(-1) == 1;
  int64_t next = -1;  // the stride the next outer dimension must have
  for (int64_t i = x.dim() - 2; fits && i >= 0; --i) {
    if (x.size(i) == 1) continue;
    if (next < 0) r.ld = x.stride(i);
    else fits = x.stride(i) == next;
    next = x.stride(i) * x.size(i);
  }
  if (!fits || (apart && r.rows > 1 && r.ld < r.d)) {
    r.t = x.contiguous();
    r.ld = r.d;
  }
  return r;
}
std::vector<int64_t> with_last(const at::Tensor& x, int64_t d) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = d;
  return s;
}
// A new contiguous tensor beside `like`.
at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType t) {
  return like.is_cuda() ? at::detail::empty_cuda(sizes, t, like.device(), c10::nullopt)
                        : at::empty(sizes, like.options().dtype(t));
}
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* cur_stream(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The norm's weight: (d), contiguous, in x's type or float32.
at::Tensor norm_weight(const OptTensor& weight, const at::Tensor& x, at::ScalarType xt) {
  if (!weight) return {};
  check_with(*weight, x, "weight");
  TORCH_CHECK_VALUE(weight->dim() == 1 && weight->size(0) == x.size(-1), "qrb200: weight must have shape (", x.size(-1),
                    "), got ", weight->sizes());
  check_type(weight->scalar_type() == xt || weight->scalar_type() == at::kFloat, "weight", weight->scalar_type());
  return weight->contiguous();
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm(const at::Tensor& x, const OptTensor& weight,
                                                        const OptTensor& residual, double eps,
                                                        c10::optional<at::ScalarType> out_dtype) {
  check_device(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1, "qrb200: rms_norm takes a (..., d) tensor");
  const auto xt = x.scalar_type();
  check_type(native(xt), "x", xt);
  const auto ot = out_dtype.value_or(xt);
  check_type(ot == xt || ot == at::kFloat8_e4m3fn, "the output", ot);
  TORCH_CHECK_VALUE(eps >= 0, "qrb200: eps must not be negative");
  const at::Tensor w = norm_weight(weight, x, xt);
  if (residual) {
    check_with(*residual, x, "residual");
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "qrb200: residual must have x's shape ", x.sizes(), ", got ", residual->sizes());
    check_type(residual->scalar_type() == xt || residual->scalar_type() == at::kFloat, "residual", residual->scalar_type());
  }
  const c10::OptionalDeviceGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  const Rows rx = as_rows(x), rr = residual ? as_rows(*residual) : Rows{{}, 0, 0, 0};
  at::Tensor y = fresh(x.sizes(), x, ot), scale, h;
  if (ot == at::kFloat8_e4m3fn) scale = fresh(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
  if (residual) h = fresh(x.sizes(), x, residual->scalar_type());
  if (x.is_meta()) return {y, scale, h};
  check_rc(qrb200_rms_norm(rx.t.data_ptr(), rx.ld, ptr(w), w.defined() ? layer_code(w.scalar_type()) : 0, ptr(rr.t), rr.ld,
                           residual ? layer_code(residual->scalar_type()) : 0, y.data_ptr(),
                           static_cast<float*>(ptr(scale)), ptr(h), rx.rows, rx.d, (float)eps, layer_code(xt),
                           layer_code(ot), cur_stream(x)),
           "qrb200_rms_norm");
  return {y, scale, h};
}

std::tuple<at::Tensor, at::Tensor> quantize_rows(const at::Tensor& x) {
  check_device(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1, "qrb200: quantize_rows takes a (..., d) tensor");
  check_type(native(x.scalar_type()), "x", x.scalar_type());
  const c10::OptionalDeviceGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  const Rows r = as_rows(x);
  at::Tensor q = fresh(x.sizes(), x, at::kFloat8_e4m3fn);
  at::Tensor scale = fresh(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
  if (x.is_meta()) return {q, scale};
  check_rc(qrb200_quantize_rows(r.t.data_ptr(), r.ld, q.data_ptr(), scale.data_ptr<float>(), r.rows, r.d,
                                layer_code(x.scalar_type()), cur_stream(x)),
           "qrb200_quantize_rows");
  return {q, scale};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_backward(const at::Tensor& dy, const at::Tensor& h,
                                                                 const OptTensor& dh, const OptTensor& weight,
                                                                 double eps, bool want_dx, bool want_dresidual,
                                                                 bool want_dweight) {
  check_device(dy, "dy");
  const auto xt = dy.scalar_type(), ht = h.scalar_type();
  check_type(native(xt), "dy", xt);
  check_type(ht == xt || ht == at::kFloat, "h", ht);
  check_with(h, dy, "h");
  TORCH_CHECK_VALUE(dy.dim() >= 1 && h.sizes() == dy.sizes(), "qrb200: h must have dy's shape");
  TORCH_CHECK_VALUE(eps >= 0, "qrb200: eps must not be negative");
  if (dh) {
    check_with(*dh, dy, "dh");
    check_type(dh->scalar_type() == ht, "dh", dh->scalar_type());
    TORCH_CHECK_VALUE(dh->sizes() == dy.sizes(), "qrb200: dh must have dy's shape");
  }
  const at::Tensor w = norm_weight(weight, dy, xt);
  TORCH_CHECK_VALUE(!want_dweight || w.defined(), "qrb200: a weight's gradient needs the weight");
  const c10::OptionalDeviceGuard guard(dy.is_cuda() ? c10::optional<c10::Device>(dy.device()) : c10::nullopt);
  const Rows rg = as_rows(dy), rh = as_rows(h), rd = dh ? as_rows(*dh) : Rows{{}, 0, 0, 0};
  at::Tensor dx, dres, dw;
  if (want_dx || (want_dresidual && ht == xt)) dx = fresh(dy.sizes(), dy, xt);
  if (want_dresidual && ht != xt) dres = fresh(dy.sizes(), dy, ht);  // dx is it otherwise: no two outputs share memory
  if (want_dweight) dw = fresh(w.sizes(), dy, w.scalar_type());
  if (dy.is_meta()) return {dx, dres, dw};
  size_t bytes = 0;
  if (want_dweight) check_rc(qrb200_rms_norm_backward_workspace_bytes(rg.rows, rg.d, layer_code(xt), layer_code(ht), &bytes), "qrb200_rms_norm_backward_workspace_bytes");
  at::Tensor ws;
  if (bytes) ws = fresh({(int64_t)bytes}, dy, at::kByte);
  check_rc(qrb200_rms_norm_backward(rg.t.data_ptr(), rg.ld, rh.t.data_ptr(), rh.ld, ptr(rd.t), rd.ld, ptr(w),
                                    w.defined() ? layer_code(w.scalar_type()) : 0, ptr(dx), ptr(dres),
                                    ptr(dw), rg.rows, rg.d, (float)eps, layer_code(xt), layer_code(ht), ptr(ws), bytes,
                                    cur_stream(dy)),
           "qrb200_rms_norm_backward");
  return {dx, dres, dw};
}

// The product's weight (n, k): rows in place, or columns (a transposed view) for 16-bit types.
struct Weight {
  at::Tensor t;
  int64_t ld;
  int32_t transposed;
};
Weight as_weight(const at::Tensor& w, bool may_transpose) {
  if (w.is_meta() || w.numel() == 0) return {w, w.size(1), 0};
  const int64_t n = w.size(0), k = w.size(1);
  if ((k == 1 || w.stride(1) == 1) && (n == 1 || w.stride(0) >= k)) return {w, n == 1 ? k : w.stride(0), 0};
  if (may_transpose && (n == 1 || w.stride(0) == 1) && (k == 1 || w.stride(1) >= n)) return {w, k == 1 ? n : w.stride(1), 1};
  return {w.contiguous(), k, 0};
}
// Scales of the rows of an 8-bit operand: one each, or one for all.
at::Tensor row_scales(const OptTensor& s, const at::Tensor& x, int64_t rows, const char* name) {
  if (!s) return {};
  check_with(*s, x, name);
  check_type(s->scalar_type() == at::kFloat, name, s->scalar_type());
  TORCH_CHECK_VALUE(s->numel() == rows || s->numel() == 1, "qrb200: ", name, " must hold one scale or ", rows, ", got ", s->numel());
  return s->reshape({-1}).expand({rows}).contiguous();
}

std::tuple<at::Tensor, at::Tensor> linear(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                                          const OptTensor& residual, int64_t activation, const OptTensor& x_scale,
                                          const OptTensor& weight_scale, c10::optional<at::ScalarType> out_dtype,
                                          bool want_slope) {
  check_device(x, "x");
  const auto xt = x.scalar_type();
  const bool q8 = xt == at::kFloat8_e4m3fn;
  check_type(xt == at::kBFloat16 || xt == at::kHalf || q8, "x", xt);
  check_type(weight.scalar_type() == xt, "weight", weight.scalar_type());
  check_with(weight, x, "weight");
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1),
                    "qrb200: linear takes x (..., k) and weight (n, k), got ", x.sizes(), " and ", weight.sizes());
  const auto ot = out_dtype.value_or(q8 ? at::kBFloat16 : xt);
  check_type(q8 ? (ot == at::kBFloat16 || ot == at::kHalf) : ot == xt, "the output", ot);
  TORCH_CHECK_VALUE(activation >= QRB200_ACT_NONE && activation <= QRB200_ACT_SILU, "qrb200: unknown activation ", activation);
  TORCH_CHECK_VALUE(q8 || (!x_scale && !weight_scale), "qrb200: scales belong to 8-bit operands");
  TORCH_CHECK_VALUE(!(q8 && want_slope), "qrb200: the 8-bit product has no gradient");
  const int64_t n = weight.size(0), k = weight.size(1);
  const auto shape = with_last(x, n);
  if (bias) {
    check_with(*bias, x, "bias");
    check_type(bias->scalar_type() == ot, "bias", bias->scalar_type());
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == n, "qrb200: bias must have shape (", n, "), got ", bias->sizes());
  }
  if (residual) {
    check_with(*residual, x, "residual");
    check_type(residual->scalar_type() == ot, "residual", residual->scalar_type());
    TORCH_CHECK_VALUE(residual->sizes() == at::IntArrayRef(shape), "qrb200: residual must have the output's shape ", at::IntArrayRef(shape), ", got ", residual->sizes());
  }
  const c10::OptionalDeviceGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  const Rows rx = as_rows(x, true), rr = residual ? as_rows(*residual) : Rows{{}, 0, 0, 0};
  const Weight w = as_weight(weight, !q8);
  const at::Tensor b = bias ? bias->contiguous() : at::Tensor();
  const at::Tensor xs = row_scales(x_scale, x, rx.rows, "x_scale"), wsc = row_scales(weight_scale, x, n, "weight_scale");
  at::Tensor y = fresh(shape, x, ot), slope;
  if (want_slope) slope = fresh(shape, x, at::kShort);
  if (x.is_meta()) return {y, slope};
  size_t bytes = 0;
  check_rc(qrb200_linear_workspace_bytes(rx.t.data_ptr(), rx.ld, w.t.data_ptr(), w.ld, w.transposed, rx.rows, n, k, layer_code(xt), &bytes),
           "qrb200_linear_workspace_bytes");
  at::Tensor ws;
  if (bytes) ws = fresh({(int64_t)bytes}, x, at::kByte);
  check_rc(qrb200_linear(rx.t.data_ptr(), rx.ld, w.t.data_ptr(), w.ld, w.transposed, static_cast<const float*>(ptr(xs)),
                         static_cast<const float*>(ptr(wsc)), ptr(b), ptr(rr.t), rr.ld, y.data_ptr(), n,
                         static_cast<uint16_t*>(ptr(slope)), rx.rows, n, k, layer_code(xt), layer_code(ot), (int32_t)activation,
                         ptr(ws), bytes, cur_stream(x)),
           "qrb200_linear");
  return {y, slope};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_backward(const at::Tensor& dy, const OptTensor& slope,
                                                               const at::Tensor& x, const at::Tensor& weight, bool want_dx,
                                                               bool want_dweight, bool want_dbias) {
  check_device(dy, "dy");
  const auto t = dy.scalar_type();
  check_type(t == at::kBFloat16 || t == at::kHalf, "dy", t);
  check_type(x.scalar_type() == t, "x", x.scalar_type());
  check_type(weight.scalar_type() == t, "weight", weight.scalar_type());
  check_with(x, dy, "x");
  check_with(weight, dy, "weight");
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1), "qrb200: linear_backward takes x (..., k) and weight (n, k)");
  const int64_t n = weight.size(0), k = weight.size(1);
  const auto shape = with_last(x, n);
  TORCH_CHECK_VALUE(dy.sizes() == at::IntArrayRef(shape), "qrb200: dy must have shape ", at::IntArrayRef(shape), ", got ", dy.sizes());
  if (slope) {
    check_with(*slope, dy, "slope");
    check_type(slope->scalar_type() == at::kShort, "slope", slope->scalar_type());
    TORCH_CHECK_VALUE(slope->sizes() == dy.sizes() && slope->is_contiguous(), "qrb200: slope must be contiguous, in dy's shape");
  }
  const c10::OptionalDeviceGuard guard(dy.is_cuda() ? c10::optional<c10::Device>(dy.device()) : c10::nullopt);
  const Rows rg = as_rows(dy, true), rx = as_rows(x, true);
  const Weight w = as_weight(weight, true);
  at::Tensor dx, dw, db;
  if (want_dx) dx = fresh(x.sizes(), x, t);
  if (want_dweight) dw = fresh(weight.sizes(), x, t);
  if (want_dbias) db = fresh({n}, dy, t);
  if (dy.is_meta()) return {dx, dw, db};
  size_t bytes = 0;
  check_rc(qrb200_linear_backward_workspace_bytes(rg.t.data_ptr(), rg.ld, slope.has_value(), rx.t.data_ptr(), rx.ld, w.t.data_ptr(),
                                                  w.ld, w.transposed, want_dx, want_dweight, want_dbias, rg.rows, n, k, &bytes),
           "qrb200_linear_backward_workspace_bytes");
  at::Tensor ws;
  if (bytes) ws = fresh({(int64_t)bytes}, dy, at::kByte);
  check_rc(qrb200_linear_backward(rg.t.data_ptr(), rg.ld, slope ? static_cast<const uint16_t*>(slope->data_ptr()) : nullptr,
                                  rx.t.data_ptr(), rx.ld, w.t.data_ptr(), w.ld, w.transposed, ptr(dx), ptr(dw), ptr(db),
                                  rg.rows, n, k, layer_code(t), ptr(ws), bytes, cur_stream(dy)),
           "qrb200_linear_backward");
  return {dx, dw, db};
}

// ---- gradients ----
// The operators as they run below autograd: by way of the dispatcher where anything may be listening
// there (a dispatch mode, a fake tensor, a trace, another device), so that it sees the operator; as plain
// functions where nothing can: CUDA tensors of no other kind, no mode, no transform.  The dispatcher takes
// about 1 us a call: 4 of the 77 us of a small training step, which is bound by the host.
bool is_plain(const at::Tensor& t) {
  constexpr c10::DispatchKeySet plain = c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
                                        c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) |
                                        c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA);
  return !t.defined() || (t.key_set() - plain).empty();
}
bool is_plain(const OptTensor& t) { return !t || is_plain(*t); }
template <typename... T>
bool nothing_listens(const T&... ts) {
  return (is_plain(ts) && ...) && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         (c10::impl::tls_local_dispatch_key_set().included_ - c10::default_included_set).empty();
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_below(const at::Tensor& x, const OptTensor& weight, const OptTensor& residual,
                                                              double eps, c10::optional<at::ScalarType> out_dtype) {
  if (nothing_listens(x, weight, residual)) return rms_norm(x, weight, residual, eps, out_dtype);
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("qrb200::rms_norm", "").typed<decltype(rms_norm)>();
  return op.call(x, weight, residual, eps, out_dtype);
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_backward_below(const at::Tensor& dy, const at::Tensor& h, const OptTensor& dh,
                                                                       const OptTensor& weight, double eps, bool want_dx,
                                                                       bool want_dresidual, bool want_dweight) {
  if (nothing_listens(dy, h, dh, weight)) return rms_norm_backward(dy, h, dh, weight, eps, want_dx, want_dresidual, want_dweight);
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("qrb200::rms_norm_backward", "").typed<decltype(rms_norm_backward)>();
  return op.call(dy, h, dh, weight, eps, want_dx, want_dresidual, want_dweight);
}
std::tuple<at::Tensor, at::Tensor> linear_below(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                                                const OptTensor& residual, int64_t activation, const OptTensor& x_scale,
                                                const OptTensor& weight_scale, c10::optional<at::ScalarType> out_dtype,
                                                bool want_slope) {
  if (nothing_listens(x, weight, bias, residual, x_scale, weight_scale))
    return linear(x, weight, bias, residual, activation, x_scale, weight_scale, out_dtype, want_slope);
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("qrb200::linear", "").typed<decltype(linear)>();
  return op.call(x, weight, bias, residual, activation, x_scale, weight_scale, out_dtype, want_slope);
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_backward_below(const at::Tensor& dy, const OptTensor& slope, const at::Tensor& x,
                                                                     const at::Tensor& weight, bool want_dx, bool want_dweight,
                                                                     bool want_dbias) {
  if (nothing_listens(dy, slope, x, weight)) return linear_backward(dy, slope, x, weight, want_dx, want_dweight, want_dbias);
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("qrb200::linear_backward", "").typed<decltype(linear_backward)>();
  return op.call(dy, slope, x, weight, want_dx, want_dweight, want_dbias);
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

OptTensor given(const at::Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
bool requires_grad(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
bool requires_grad(const OptTensor& t) { return t && requires_grad(*t); }
template <typename... T>
bool wants_grad(const T&... ts) {
  return at::GradMode::is_enabled() && (requires_grad(ts) || ...);
}
// A tangent would be lost without a word below here: it hangs on a tensor that need not require a gradient.
bool has_tangent(const at::Tensor& t) {
  return t.defined() && t.unsafeGetTensorImpl()->autograd_meta() && t._fw_grad(/*level=*/0).defined();
}
bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }
template <typename... T>
void check_no_tangent(const T&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(ts) || ...), "qrb200: the layer operators have no forward-mode derivative");
}
void check_once() {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "qrb200: the layer operators are differentiable once (no create_graph)");
}

struct RmsNormGrad : torch::autograd::Function<RmsNormGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& weight,
                               const OptTensor& residual, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    auto [y, scale, h] = rms_norm_below(x, weight, residual, eps, c10::nullopt);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["type"] = x.scalar_type();
    ctx->save_for_backward({h.defined() ? h : x, weight.value_or(at::Tensor())});
    return h.defined() ? variable_list{y, h} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once();
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &h = saved[0], &weight = saved[1];
    at::Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : at::Tensor();
    check_no_tangent(dy, dh);
    // inputs that were given, in order, have an edge each
    size_t edge = 0;
    const bool want_x = ctx->needs_input_grad(edge++);
    const bool want_w = weight.defined() && ctx->needs_input_grad(edge++);
    const bool want_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(edge++);
    if (!dy.defined()) {
      if (!dh.defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
      dy = at::zeros(h.sizes(), h.options().dtype(ctx->saved_data["type"].toScalarType()));
    }
    auto [dx, dres, dw] =
        rms_norm_backward_below(dy, h, given(dh), given(weight), ctx->saved_data["eps"].toDouble(), want_x, want_r, want_w);
    if (want_r && !dres.defined()) dres = dx;
    return {want_x ? dx : at::Tensor(), dw, dres, at::Tensor()};
  }
};

// Below autograd with nothing to differentiate; otherwise with a node that can.  PLAIN: the caller knows
// that nothing listens.
template <bool PLAIN>
std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_grad(const at::Tensor& x, const OptTensor& weight, const OptTensor& residual,
                                                             double eps, c10::optional<at::ScalarType> out_dtype) {
  check_no_tangent(x, weight, residual);
  if (!wants_grad(x, weight, residual)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return PLAIN ? rms_norm(x, weight, residual, eps, out_dtype) : rms_norm_below(x, weight, residual, eps, out_dtype);
  }
  TORCH_CHECK_VALUE(!out_dtype || *out_dtype == x.scalar_type(), "qrb200: the 8-bit norm has no gradient (use torch.no_grad())");
  variable_list out = RmsNormGrad::apply(x, weight, residual, eps);
  return {out[0], at::Tensor(), out.size() > 1 ? out[1] : at::Tensor()};
}

struct LinearGrad : torch::autograd::Function<LinearGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                               const OptTensor& residual, int64_t activation, c10::optional<at::ScalarType> out_dtype,
                               bool want_slope) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    const bool sums = x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad());
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    auto [y, slope] = linear_below(x, weight, bias, residual, activation, c10::nullopt, c10::nullopt, out_dtype,
                                   want_slope || (sums && activation != QRB200_ACT_NONE));
    if (sums) ctx->save_for_backward({x, weight, activation == QRB200_ACT_NONE ? at::Tensor() : slope});
    if (!want_slope) return {y};
    ctx->mark_non_differentiable({slope});
    return {y, slope};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once();
    variable_list out(7);
    const at::Tensor& dy = grads[0];
    check_no_tangent(dy);
    if (!dy.defined()) return out;
    size_t edge = 0;
    const bool want_x = ctx->needs_input_grad(edge++), want_w = ctx->needs_input_grad(edge++);
    const bool want_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(edge++);
    const bool want_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(edge++);
    if (want_x || want_w || want_b) {
      const auto saved = ctx->get_saved_variables();
      std::tie(out[0], out[1], out[2]) =
          linear_backward_below(dy, given(saved[2]), saved[0], saved[1], want_x, want_w, want_b);
    }
    if (want_r) out[3] = dy;
    return out;
  }
};

template <bool PLAIN>
std::tuple<at::Tensor, at::Tensor> linear_grad(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                                               const OptTensor& residual, int64_t activation, const OptTensor& x_scale,
                                               const OptTensor& weight_scale, c10::optional<at::ScalarType> out_dtype,
                                               bool want_slope) {
  check_no_tangent(x, weight, bias, residual, x_scale, weight_scale);
  if (!wants_grad(x, weight, bias, residual)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return PLAIN ? linear(x, weight, bias, residual, activation, x_scale, weight_scale, out_dtype, want_slope)
                 : linear_below(x, weight, bias, residual, activation, x_scale, weight_scale, out_dtype, want_slope);
  }
  TORCH_CHECK_VALUE(x.scalar_type() != at::kFloat8_e4m3fn, "qrb200: the 8-bit product has no gradient (use torch.no_grad())");
  TORCH_CHECK_VALUE(!x_scale && !weight_scale, "qrb200: scales belong to 8-bit operands");
  variable_list out = LinearGrad::apply(x, weight, bias, residual, activation, out_dtype, want_slope);
  return {out[0], out.size() > 1 ? out[1] : at::Tensor()};
}

}  // namespace

// The short way from Python.
std::tuple<at::Tensor, at::Tensor, at::Tensor> qrb200::rms_norm(const at::Tensor& x, const OptTensor& weight,
                                                                const OptTensor& residual, double eps,
                                                                c10::optional<at::ScalarType> out_dtype) {
  return rms_norm_grad<true>(x, weight, residual, eps, out_dtype);
}
std::tuple<at::Tensor, at::Tensor> qrb200::linear(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                                                  const OptTensor& residual, int64_t activation, const OptTensor& x_scale,
                                                  const OptTensor& weight_scale, c10::optional<at::ScalarType> out_dtype,
                                                  bool want_slope) {
  return linear_grad<true>(x, weight, bias, residual, activation, x_scale, weight_scale, out_dtype, want_slope);
}

TORCH_LIBRARY(qrb200, m) {
  m.def("geqrf(Tensor A) -> (Tensor H, Tensor tau, Tensor info)");
  m.def("rms_norm(Tensor x, Tensor? weight, Tensor? residual, float eps, ScalarType? out_dtype) -> (Tensor y, Tensor scale, Tensor h)");
  m.def("rms_norm_backward(Tensor dy, Tensor h, Tensor? dh, Tensor? weight, float eps, bool want_dx, bool want_dresidual, bool want_dweight) -> (Tensor dx, Tensor dresidual, Tensor dweight)");
  m.def("quantize_rows(Tensor x) -> (Tensor q, Tensor scale)");
  m.def("linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int activation, Tensor? x_scale, Tensor? weight_scale, ScalarType? out_dtype, bool want_slope) -> (Tensor y, Tensor slope)");
  m.def("linear_backward(Tensor dy, Tensor? slope, Tensor x, Tensor weight, bool want_dx, bool want_dweight, bool want_dbias) -> (Tensor dx, Tensor dweight, Tensor dbias)");
}

namespace {
// A layer operator's function serves both keys: on meta tensors it returns before it runs anything.
void layer_impls(torch::Library& m) {
  m.impl("rms_norm", rms_norm);
  m.impl("rms_norm_backward", rms_norm_backward);
  m.impl("quantize_rows", quantize_rows);
  m.impl("linear", linear);
  m.impl("linear_backward", linear_backward);
}
}  // namespace

TORCH_LIBRARY_IMPL(qrb200, CUDA, m) {
  m.impl("geqrf", geqrf_cuda);
  layer_impls(m);
}

TORCH_LIBRARY_IMPL(qrb200, Meta, m) {
  m.impl("geqrf", geqrf_meta);
  layer_impls(m);
}

TORCH_LIBRARY_IMPL(qrb200, Autograd, m) {
  m.impl("rms_norm", rms_norm_grad<false>);
  m.impl("linear", linear_grad<false>);
  // no derivative of either mode: refused where one is asked for
  m.impl("quantize_rows", torch::autograd::autogradNotImplementedFallback());
  m.impl("rms_norm_backward", torch::autograd::autogradNotImplementedFallback());
  m.impl("linear_backward", torch::autograd::autogradNotImplementedFallback());
}

// Host tensors (and mixes of host and device tensors, which reach this key too) are refused by the
// functions themselves.
TORCH_LIBRARY_IMPL(qrb200, CPU, m) { layer_impls(m); }
