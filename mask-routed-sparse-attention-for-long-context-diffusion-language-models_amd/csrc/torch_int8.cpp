// The CUDA implementations of the 8-bit torch.ops.mrsa operators (schemas and fake kernels:
// mrsa/ops.py): tensors to the C entry points of libmrsa.so.  At one token a call of these
// operators is host time, and a public call costs half as much with this side of it and the checks
// in C++ as through ctypes (norm of one row 12.1 -> 6.1 us, rows 8.6 -> 5.1, product 10.9 -> 5.2;
// where the processor is faster 5.6, 4.7 and 4.8).
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <tuple>

#include "mrsa.h"

namespace {

using at::Tensor;

int32_t dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? MRSA_DTYPE_BF16 : t == at::kHalf ? MRSA_DTYPE_FP16 : MRSA_DTYPE_FP32;
}

// The exceptions of mrsa/_lib.py: check.
void check(int status, const char* op) {
  if (status == MRSA_OK) return;
  TORCH_CHECK_VALUE(status == MRSA_ERR_LAUNCH, op, ": ", mrsa_status_string(status), " (status ",
                    status, ")");
  TORCH_CHECK(false, op, ": ", mrsa_status_string(status), " (status ", status, ")");
}

// The checks of mrsa/int8_checks.py, in their words.
bool float_type(at::ScalarType t) {
  return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat;
}
void check_rows(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name,
                    " must have rows of at least one value, got ", t.sizes());
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(float_type(t.scalar_type()), name, " must be bf16, fp16 or fp32, got ",
                    t.scalar_type());
}
void check_values(const Tensor& values, const Tensor& scales, const char* name) {
  TORCH_CHECK_VALUE(values.scalar_type() == at::kChar && values.is_cuda() && values.dim() >= 1,
                    name, " must be CUDA int8 rows, got ", values.sizes(), " ",
                    values.scalar_type(), " on ", values.device());
  const auto want = values.sizes().slice(0, values.dim() - 1);
  TORCH_CHECK_VALUE(scales.sizes() == want && scales.scalar_type() == at::kFloat, name,
                    " of shape ", values.sizes(), " need fp32 scales of shape ", want, ", got ",
                    scales.sizes(), " ", scales.scalar_type());
  TORCH_CHECK_VALUE(scales.device() == values.device(), name,
                    " and their scales must be on one device");
}
void check_dtype(at::ScalarType dtype) {
  TORCH_CHECK_VALUE(float_type(dtype), "dtype must be bf16, fp16 or fp32, got ", dtype);
}

// t as rows [n, dim] whose last dim is dense (a copy only if no strides give that).
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}
// As rows_of, at strides that mrsa_int8_linear_fwd takes.
Tensor operand_rows(const Tensor& t) {
  Tensor r = rows_of(t);
  return r.size(0) > 1 && r.stride(0) >= (int64_t)1 << 31 ? r.contiguous() : r;
}
int64_t row_stride(const Tensor& rows) {  // (a single row's is arbitrary)
  return rows.size(0) > 1 ? rows.stride(0) : rows.size(1);
}
at::DimVector with_dim(const Tensor& t, int64_t dim) {
  at::DimVector sizes(t.sizes());
  sizes.back() = dim;
  return sizes;
}
// (as at::empty, without another pass through the dispatcher)
Tensor new_rows(const Tensor& t, int64_t dim, at::ScalarType dtype) {
  return at::detail::empty_cuda(with_dim(t, dim), dtype, t.device(), std::nullopt);
}
Tensor new_scales(const Tensor& t) {
  return at::detail::empty_cuda(t.sizes().slice(0, t.dim() - 1), at::kFloat, t.device(),
                                std::nullopt);
}

// The device of the tensors, current during the call, and its current stream.
struct Launch {
  c10::hip::HIPGuard guard;
  void* stream;
  explicit Launch(const Tensor& t)
      : guard(t.device().index()),
        stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  check_rows(x, "x");
  const Launch at(x);
  const Tensor rows = rows_of(x);
  const int64_t dim = rows.size(1);
  Tensor values = new_rows(x, dim, at::kChar), scales = new_scales(x);
  check(mrsa_quantize_rows_fwd(rows.data_ptr(), row_stride(rows), rows.size(0), dim,
                               dtype_code(x.scalar_type()), (int8_t*)values.data_ptr(),
                               (float*)scales.data_ptr(), at.stream),
        "quantize_rows");
  return {values, scales};
}

Tensor dequantize_rows(const Tensor& values, const Tensor& scales, at::ScalarType dtype) {
  check_values(values, scales, "values");
  TORCH_CHECK_VALUE(values.size(-1) >= 1, "values must have rows of at least one value, got ",
                    values.sizes());
  check_dtype(dtype);
  const Launch at(values);
  const Tensor rows = rows_of(values), s = scales.contiguous();
  const int64_t dim = rows.size(1);
  Tensor out = new_rows(values, dim, dtype);
  check(mrsa_dequantize_rows_fwd((const int8_t*)rows.data_ptr(), row_stride(rows),
                                 (const float*)s.data_ptr(), rows.size(0), dim, dtype_code(dtype),
                                 out.data_ptr(), at.stream),
        "dequantize_rows");
  return out;
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_int8(const Tensor& x,
                                                     const std::optional<Tensor>& residual,
                                                     const Tensor& weight, double eps) {
  check_rows(x, "x");
  if (residual) {
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() &&
                          residual->scalar_type() == x.scalar_type() &&
                          residual->device() == x.device(),
                      "residual must match x, got ", residual->sizes(), " ",
                      residual->scalar_type(), " on ", residual->device(), " for ", x.sizes(), " ",
                      x.scalar_type(), " on ", x.device());
  }
  TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(-1) &&
                        weight.scalar_type() == x.scalar_type() && weight.device() == x.device(),
                    "weight must be [", x.size(-1), "] ", x.scalar_type(), " on ", x.device(),
                    ", got ", weight.sizes(), " ", weight.scalar_type(), " on ", weight.device());
  TORCH_CHECK_VALUE(eps >= 1e-24 && eps <= 1e24, "eps must be in [1e-24, 1e24], got ", eps);
  const Launch at(x);
  const Tensor rows = rows_of(x), w = weight.contiguous();
  const int64_t dim = rows.size(1);
  Tensor res, total;
  if (residual) {
    res = rows_of(*residual);
    total = new_rows(x, dim, x.scalar_type());
  } else {
    total = at::detail::empty_cuda({0}, x.scalar_type(), x.device(), std::nullopt);
  }
  Tensor values = new_rows(x, dim, at::kChar), scales = new_scales(x);
  check(mrsa_add_rms_norm_int8_fwd(
            rows.data_ptr(), row_stride(rows), residual ? res.data_ptr() : nullptr,
            residual ? row_stride(res) : 0, w.data_ptr(), rows.size(0), dim, (float)eps,
            dtype_code(x.scalar_type()), residual ? total.data_ptr() : nullptr,
            (int8_t*)values.data_ptr(), (float*)scales.data_ptr(), at.stream),
        "add_rms_norm_int8");
  return {total, values, scales};
}

std::tuple<Tensor, Tensor> swiglu_int8(const Tensor& gate_up) {
  check_rows(gate_up, "gate_up");
  TORCH_CHECK_VALUE(gate_up.size(-1) % 2 == 0, "gate_up must have an even last dim, got ",
                    gate_up.sizes());
  const Launch at(gate_up);
  const Tensor rows = rows_of(gate_up);
  const int64_t dim = rows.size(1) / 2;
  Tensor values = new_rows(gate_up, dim, at::kChar), scales = new_scales(gate_up);
  check(mrsa_swiglu_int8_fwd(rows.data_ptr(), row_stride(rows), rows.size(0), dim,
                             dtype_code(gate_up.scalar_type()), (int8_t*)values.data_ptr(),
                             (float*)scales.data_ptr(), at.stream),
        "swiglu_int8");
  return {values, scales};
}

Tensor int8_linear(const Tensor& x, const Tensor& x_scales, const Tensor& weight,
                   const Tensor& weight_scales, const std::optional<Tensor>& bias,
                   at::ScalarType dtype) {
  check_values(x, x_scales, "x");
  check_values(weight, weight_scales, "weight");
  const int64_t dim = x.size(-1);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == dim, "weight must be [out_dim, ", dim,
                    "], got ", weight.sizes());
  TORCH_CHECK_VALUE(weight.device() == x.device(), "x and weight must be on one device");
  TORCH_CHECK_VALUE(dim >= 1 && dim <= 131071,
                    "rows of 1 to 131071 values have a sum in 32 bits, got ", dim);
  check_dtype(dtype);
  if (bias) {
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == weight.size(0) &&
                          bias->scalar_type() == dtype && bias->device() == x.device(),
                      "bias must be [", weight.size(0), "] ", dtype, " on ", x.device(), ", got ",
                      bias->sizes(), " ", bias->scalar_type(), " on ", bias->device());
  }
  const Launch at(x);
  const Tensor rows = operand_rows(x), w = operand_rows(weight);
  const Tensor sx = x_scales.contiguous(), sw = weight_scales.contiguous();
  const Tensor b = bias ? bias->contiguous() : Tensor();
  const int64_t n = rows.size(0), out_dim = w.size(0);
  Tensor out = new_rows(x, out_dim, dtype);
  const int64_t bytes = mrsa_int8_linear_workspace_bytes(n, out_dim, dim);
  Tensor space;
  if (bytes > 0) space = at::detail::empty_cuda({bytes}, at::kByte, x.device(), std::nullopt);
  check(mrsa_int8_linear_fwd((const int8_t*)rows.data_ptr(), row_stride(rows),
                             (const float*)sx.data_ptr(), (const int8_t*)w.data_ptr(),
                             row_stride(w), (const float*)sw.data_ptr(),
                             bias ? b.data_ptr() : nullptr, n, out_dim, dim, dtype_code(dtype),
                             bytes > 0 ? space.data_ptr() : nullptr, bytes, out.data_ptr(),
                             at.stream),
        "int8_linear");
  return out;
}

// ---- derivatives ---------------------------------------------------------------------------
// Tensors that ask for one are refused where autograd sees the call: below it those of torch.func's
// reverse transforms no longer ask, and a gradient of zeros would come back.

void no_derivative(const char* op, const Tensor& t) {
  TORCH_CHECK_VALUE(!t.requires_grad() || !at::GradMode::is_enabled(), op,
                    " has no gradient: call it under torch.no_grad()");
  TORCH_CHECK_VALUE(!t._fw_grad(0).defined(), op, " has no forward-mode derivative");
}
void no_derivative(const char* op, const std::optional<Tensor>& t) {
  if (t) no_derivative(op, *t);
}
void no_derivative(const char*, double) {}
void no_derivative(const char*, at::ScalarType) {}

constexpr const char* kOps[] = {"quantize_rows", "dequantize_rows", "add_rms_norm_int8",
                                "swiglu_int8", "int8_linear"};

// Operator OP of kOps for autograd: the refusals, and the call below.
template <int OP, class R, class... Args>
R below_autograd(c10::DispatchKeySet keys, Args... args) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow((std::string("mrsa::") + kOps[OP]).c_str(), "")
                             .template typed<R(Args...)>();
  (no_derivative(kOps[OP], args), ...);
  const at::AutoDispatchBelowADInplaceOrView guard;
  return op.redispatch(keys & c10::after_autograd_keyset, args...);
}
template <int OP, class R, class... Args>
void impl_autograd(torch::Library& m, R (*)(Args...)) {
  m.impl(kOps[OP], TORCH_FN((below_autograd<OP, R, Args...>)));
}

}  // namespace

TORCH_LIBRARY_IMPL(mrsa, CUDA, m) {
  m.impl("quantize_rows", &quantize_rows);
  m.impl("dequantize_rows", &dequantize_rows);
  m.impl("add_rms_norm_int8", &add_rms_norm_int8);
  m.impl("swiglu_int8", &swiglu_int8);
  m.impl("int8_linear", &int8_linear);
}

TORCH_LIBRARY_IMPL(mrsa, Autograd, m) {
  impl_autograd<0>(m, &quantize_rows);
  impl_autograd<1>(m, &dequantize_rows);
  impl_autograd<2>(m, &add_rms_norm_int8);
  impl_autograd<3>(m, &swiglu_int8);
  impl_autograd<4>(m, &int8_linear);
}
