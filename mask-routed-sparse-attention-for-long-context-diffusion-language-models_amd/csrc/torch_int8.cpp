// The CUDA implementations of the 8-bit torch.ops.mrsa operators (schemas and fake kernels:
// mrsa/ops.py): tensors to the C entry points of libmrsa.so.  At one token a call of these
// operators is host time, and a public call costs 2 to 4 us less with this side of it in C++ than
// through ctypes (norm of one row 12.1 -> 8.3 us, rows 8.6 -> 6.2, product 10.9 -> 7.0).
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "mrsa.h"

namespace {

using at::Tensor;

int32_t dtype_code(at::ScalarType t) {
  TORCH_CHECK_VALUE(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat,
                    "8-bit operators work on bf16, fp16 or fp32, got ", t);
  return t == at::kBFloat16 ? MRSA_DTYPE_BF16 : t == at::kHalf ? MRSA_DTYPE_FP16 : MRSA_DTYPE_FP32;
}

// The exceptions of mrsa/_lib.py: check.
void check(int status, const char* op) {
  if (status == MRSA_OK) return;
  TORCH_CHECK_VALUE(status == MRSA_ERR_LAUNCH, op, ": ", mrsa_status_string(status), " (status ",
                    status, ")");
  TORCH_CHECK(false, op, ": ", mrsa_status_string(status), " (status ", status, ")");
}

// What a compiler has traced, or calls the operators directly, reaches them past the checks of the
// public functions: what a kernel would read or write out of range for is refused here too.
void refuse_tangent(const Tensor& t, const char* op) {
  TORCH_CHECK_VALUE(!t._fw_grad(0).defined(), op, " has no forward-mode derivative here");
}

void need(const Tensor& t, int64_t numel, at::ScalarType dtype, const Tensor& like,
          const char* name) {
  TORCH_CHECK_VALUE(t.numel() == numel && t.scalar_type() == dtype && t.device() == like.device(),
                    name, " must hold ", numel, " elements of ", dtype, " on ", like.device(),
                    ", got ", t.sizes(), " ", t.scalar_type(), " on ", t.device());
}

// t as rows [n, dim] whose last dim is dense (a copy only if no strides give that).
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}
int64_t row_stride(const Tensor& rows) {  // (a single row's is arbitrary)
  return rows.size(0) > 1 ? rows.stride(0) : rows.size(1);
}
at::DimVector with_dim(const Tensor& t, int64_t dim) {
  at::DimVector sizes(t.sizes());
  sizes.back() = dim;
  return sizes;
}
Tensor new_rows(const Tensor& t, int64_t dim, at::ScalarType dtype) {
  return at::empty(with_dim(t, dim), t.options().dtype(dtype));
}
Tensor new_scales(const Tensor& t) {
  return at::empty(t.sizes().slice(0, t.dim() - 1), t.options().dtype(at::kFloat));
}

// The device of the tensors, current during the call, and its current stream.
struct Launch {
  c10::hip::HIPGuard guard;
  void* stream;
  explicit Launch(const Tensor& t)
      : guard(device_of(t)), stream(c10::hip::getCurrentHIPStream(device_of(t)).stream()) {}
  static c10::DeviceIndex device_of(const Tensor& t) {
    TORCH_CHECK_VALUE(t.is_cuda(), "8-bit operators need CUDA tensors, got one on ", t.device());
    return t.device().index();
  }
};

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  refuse_tangent(x, "mrsa::quantize_rows");
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
  refuse_tangent(scales, "mrsa::dequantize_rows");
  const Launch at(values);
  const Tensor rows = rows_of(values), s = scales.contiguous();
  const int64_t dim = rows.size(1);
  need(values, values.numel(), at::kChar, values, "values");
  need(s, rows.size(0), at::kFloat, values, "scales");
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
  refuse_tangent(x, "mrsa::add_rms_norm_int8");
  refuse_tangent(weight, "mrsa::add_rms_norm_int8");
  const Launch at(x);
  const Tensor rows = rows_of(x), w = weight.contiguous();
  const int64_t dim = rows.size(1);
  need(w, dim, x.scalar_type(), x, "weight");
  Tensor res, total;
  if (residual) {
    refuse_tangent(*residual, "mrsa::add_rms_norm_int8");
    need(*residual, x.numel(), x.scalar_type(), x, "residual");
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "residual must have the shape of x");
    res = rows_of(*residual);
    total = new_rows(x, dim, x.scalar_type());
  } else {
    total = at::empty({0}, x.options());
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
  refuse_tangent(gate_up, "mrsa::swiglu_int8");
  const Launch at(gate_up);
  const Tensor rows = rows_of(gate_up);
  const int64_t dim = rows.size(1) / 2;
  TORCH_CHECK_VALUE(rows.size(1) % 2 == 0, "gate_up must be [..., 2 * dim]");
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
  refuse_tangent(x_scales, "mrsa::int8_linear");
  refuse_tangent(weight_scales, "mrsa::int8_linear");
  if (bias) refuse_tangent(*bias, "mrsa::int8_linear");
  const Launch at(x);
  const Tensor rows = rows_of(x), w = rows_of(weight);
  const Tensor sx = x_scales.contiguous(), sw = weight_scales.contiguous();
  const Tensor b = bias ? bias->contiguous() : Tensor();
  const int64_t n = rows.size(0), dim = rows.size(1), out_dim = w.size(0);
  need(x, x.numel(), at::kChar, x, "x");
  need(weight, out_dim * dim, at::kChar, x, "weight");
  need(sx, n, at::kFloat, x, "x_scales");
  need(sw, out_dim, at::kFloat, x, "weight_scales");
  if (bias) need(b, out_dim, dtype, x, "bias");
  Tensor out = new_rows(x, out_dim, dtype);
  const int64_t bytes = mrsa_int8_linear_workspace_bytes(n, out_dim, dim);
  Tensor space;
  if (bytes > 0) space = at::empty({bytes}, x.options().dtype(at::kByte));
  check(mrsa_int8_linear_fwd((const int8_t*)rows.data_ptr(), row_stride(rows),
                             (const float*)sx.data_ptr(), (const int8_t*)w.data_ptr(),
                             row_stride(w), (const float*)sw.data_ptr(),
                             bias ? b.data_ptr() : nullptr, n, out_dim, dim, dtype_code(dtype),
                             bytes > 0 ? space.data_ptr() : nullptr, bytes, out.data_ptr(),
                             at.stream),
        "int8_linear");
  return out;
}

}  // namespace

TORCH_LIBRARY_IMPL(mrsa, CUDA, m) {
  m.impl("quantize_rows", &quantize_rows);
  m.impl("dequantize_rows", &dequantize_rows);
  m.impl("add_rms_norm_int8", &add_rms_norm_int8);
  m.impl("swiglu_int8", &swiglu_int8);
  m.impl("int8_linear", &int8_linear);
}
