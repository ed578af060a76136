// torch_binding.cpp - registers torch.ops.hp_rms_norm.* on top of the C ABI of
// libhprms.so.  This is the only host layer between PyTorch and the kernels:
// it checks tensors, flattens them to [rows, hidden] with a row stride, picks
// the current HIP stream of the tensor's device and calls the C ABI.
//
// Schemas follow the reference's registration
// (hp_rms_norm/csrc/hp_rms_norm.cpp:35-38) with the same names and argument
// order, plus alias annotations that declare the in-place writes, so that
// functionalisation and torch.compile see them.  Messages of the shape checks
// are the reference's (hp_rms_norm/csrc/cuda/hp_rms_norm.cu:12-24,48 and
// activation_kernels.cu:11-15,38).
//
// The library is the package's importable extension module `_C`, as the
// reference's is (hp_rms_norm/__init__.py:2): importing it loads the library,
// whose static initialisers at the end of this file register the operators.
#include <Python.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <algorithm>
#include <vector>

#include "hp_rms_norm_amd.h"

namespace {

int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return HPRMS_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return HPRMS_DTYPE_FP16;
  TORCH_CHECK(false, "dtype must be kFloat16 or kBFloat16");
  return -1;
}

// Rows and row stride of a [..., hidden] tensor whose leading dims collapse
// into one (the reference flattens with view({-1, hidden}),
// hp_rms_norm/csrc/cuda/hp_rms_norm.cu:26).  Rows of width 0 hold no
// element (the ops return at once); view cannot infer their count.
void rows_of(const at::Tensor& t, int64_t hidden, int64_t* rows, int64_t* stride) {
  if (hidden == 0) {
    *rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) *rows *= t.size(i);
    *stride = 0;
    return;
  }
  if (t.dim() == 2) {  // nothing to flatten
    *rows = t.size(0);
    *stride = *rows <= 1 ? hidden : t.stride(0);
  } else {
    const at::Tensor flat = t.view({-1, hidden});
    *rows = flat.size(0);
    *stride = *rows <= 1 ? hidden : flat.stride(0);
  }
  TORCH_CHECK(*stride >= hidden, "rows of the tensor overlap (row stride ", *stride, " < hidden ", hidden, ")");
}

void check_status(int rc) {
  TORCH_CHECK(rc == HPRMS_OK, "hp_rms_norm: ", hprms_last_error(), " (status ", rc, ")");
}

struct FusedShape {
  int64_t rows, hidden, in_stride, res_stride;
  int dtype;
};

FusedShape check_fused(const at::Tensor& input, const at::Tensor& weight, const at::Tensor& residual) {
  TORCH_CHECK(input.dim() >= 2, "input.dim() >= 2");
  TORCH_CHECK(input.dim() == residual.dim(), "input.dim() == residual.dim()");
  for (int64_t i = 0; i < input.dim(); ++i)
    TORCH_CHECK(input.size(i) == residual.size(i), "input.size(i) == residual.size(i)");
  TORCH_CHECK(weight.dim() == 1, "weight.dim() == 1");
  const int64_t hidden = weight.size(0);
  TORCH_CHECK(input.size(-1) == hidden, "input.size(-1) == hidden_dim");
  TORCH_CHECK(input.stride(-1) == 1, "input.stride(-1) == 1");
  TORCH_CHECK(residual.stride(-1) == 1, "residual.stride(-1) == 1");
  TORCH_CHECK(weight.stride(0) == 1 || hidden == 1, "weight.stride(0) == 1");
  FusedShape s;
  s.dtype = dtype_code(input);
  TORCH_CHECK(residual.scalar_type() == input.scalar_type(), "residual.dtype() == input.dtype()");
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(), "weight.dtype() == input.dtype()");
  TORCH_CHECK(residual.device() == input.device() && weight.device() == input.device(),
              "input, weight and residual must be on the same device");
  s.hidden = hidden;
  rows_of(input, hidden, &s.rows, &s.in_stride);
  int64_t rrows = 0;
  rows_of(residual, hidden, &rrows, &s.res_stride);
  if (s.rows > 0) at::assert_no_overlap(input, residual);
  return s;
}

void rms_norm_hip(at::Tensor& input, const at::Tensor& weight, at::Tensor& residual, double eps) {
  const FusedShape s = check_fused(input, weight, residual);
  if (s.rows == 0 || s.hidden == 0) return;
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  check_status(hprms_fused_add_rmsnorm(input.data_ptr(), weight.data_ptr(), residual.data_ptr(), s.rows,
                                       s.hidden, s.in_stride, s.res_stride, s.dtype, eps, stream));
}

void rms_norm_meta(at::Tensor& input, const at::Tensor& weight, at::Tensor& residual, double eps) {
  (void)check_fused(input, weight, residual);
  (void)eps;
}

struct StreamShape {
  int64_t rows, hidden, out_stride, in_stride;
  int dtype;
};

StreamShape check_stream(const at::Tensor& out, const at::Tensor& input) {
  TORCH_CHECK(input.dim() >= 2, "input.dim() >= 2");
  TORCH_CHECK(input.dim() == out.dim(), "input.dim() == out.dim()");
  for (int64_t i = 0; i < input.dim(); ++i)
    TORCH_CHECK(input.size(i) == out.size(i), "input.size(i) == out.size(i)");
  TORCH_CHECK(input.stride(-1) == 1, "input.stride(-1) == 1");
  TORCH_CHECK(out.stride(-1) == 1, "out.stride(-1) == 1");
  StreamShape s;
  s.dtype = dtype_code(input);
  TORCH_CHECK(out.scalar_type() == input.scalar_type(), "out.dtype() == input.dtype()");
  TORCH_CHECK(out.device() == input.device(), "out and input must be on the same device");
  s.hidden = input.size(-1);
  int64_t orows = 0;
  rows_of(input, s.hidden, &s.rows, &s.in_stride);
  rows_of(out, s.hidden, &orows, &s.out_stride);
  if (s.rows > 0 && s.hidden > 0) at::assert_no_partial_overlap(out, input);
  return s;
}

void stream_hip(at::Tensor& out, const at::Tensor& input, int op) {
  const StreamShape s = check_stream(out, input);
  if (s.rows == 0 || s.hidden == 0) return;
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  check_status(hprms_streamer(out.data_ptr(), input.data_ptr(), s.rows, s.hidden, s.out_stride, s.in_stride,
                              s.dtype, op, stream));
}

void relu_hip(at::Tensor& out, const at::Tensor& input) { stream_hip(out, input, HPRMS_STREAM_COPY); }
void relu_max0_hip(at::Tensor& out, const at::Tensor& input) { stream_hip(out, input, HPRMS_STREAM_RELU); }
void stream_meta(at::Tensor& out, const at::Tensor& input) { (void)check_stream(out, input); }

struct PlainShape {
  int64_t rows, hidden, out_stride, in_stride;
  int dtype;
};

PlainShape check_plain(const at::Tensor& out, const at::Tensor& input, const at::Tensor& weight) {
  TORCH_CHECK(input.dim() >= 2, "input.dim() >= 2");
  TORCH_CHECK(input.dim() == out.dim(), "input.dim() == out.dim()");
  for (int64_t i = 0; i < input.dim(); ++i)
    TORCH_CHECK(input.size(i) == out.size(i), "input.size(i) == out.size(i)");
  TORCH_CHECK(weight.dim() == 1, "weight.dim() == 1");
  const int64_t hidden = weight.size(0);
  TORCH_CHECK(input.size(-1) == hidden, "input.size(-1) == hidden_dim");
  TORCH_CHECK(input.stride(-1) == 1, "input.stride(-1) == 1");
  TORCH_CHECK(out.stride(-1) == 1, "out.stride(-1) == 1");
  TORCH_CHECK(weight.stride(0) == 1 || hidden == 1, "weight.stride(0) == 1");
  PlainShape s;
  s.dtype = dtype_code(input);
  TORCH_CHECK(out.scalar_type() == input.scalar_type(), "out.dtype() == input.dtype()");
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(), "weight.dtype() == input.dtype()");
  TORCH_CHECK(out.device() == input.device() && weight.device() == input.device(),
              "out, input and weight must be on the same device");
  s.hidden = hidden;
  int64_t orows = 0;
  rows_of(input, hidden, &s.rows, &s.in_stride);
  rows_of(out, hidden, &orows, &s.out_stride);
  if (s.rows > 0) at::assert_no_partial_overlap(out, input);
  return s;
}

void rms_norm_plain_hip(at::Tensor& out, const at::Tensor& input, const at::Tensor& weight, double eps) {
  const PlainShape s = check_plain(out, input, weight);
  if (s.rows == 0 || s.hidden == 0) return;
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  check_status(hprms_rmsnorm(out.data_ptr(), input.data_ptr(), weight.data_ptr(), s.rows, s.hidden,
                             s.out_stride, s.in_stride, s.dtype, eps, stream));
}

void rms_norm_plain_meta(at::Tensor& out, const at::Tensor& input, const at::Tensor& weight, double eps) {
  (void)check_plain(out, input, weight);
  (void)eps;
}

struct Fp8Shape {
  FusedShape f;
  int64_t out_stride;
};

Fp8Shape check_fp8(const at::Tensor& out, const at::Tensor& scale, const at::Tensor& input,
                   const at::Tensor& weight, const at::Tensor& residual) {
  Fp8Shape s;
  s.f = check_fused(input, weight, residual);
  TORCH_CHECK(out.scalar_type() == at::kFloat8_e4m3fn, "out.dtype() == float8_e4m3fn");
  TORCH_CHECK(scale.scalar_type() == at::kFloat, "scale.dtype() == float32");
  TORCH_CHECK(out.dim() == input.dim(), "out.dim() == input.dim()");
  for (int64_t i = 0; i < input.dim(); ++i) TORCH_CHECK(out.size(i) == input.size(i), "out.size(i) == input.size(i)");
  TORCH_CHECK(out.stride(-1) == 1, "out.stride(-1) == 1");
  TORCH_CHECK(scale.numel() == s.f.rows, "scale.numel() == number of rows");
  TORCH_CHECK(scale.is_contiguous(), "scale must be contiguous");
  TORCH_CHECK(out.device() == input.device() && scale.device() == input.device(),
              "out, scale and input must be on the same device");
  int64_t orows = 0;
  rows_of(out, s.f.hidden, &orows, &s.out_stride);
  if (s.f.rows > 0) {
    // the FP8 rows and the scales are written while input and residual are
    // read: no sharing between any two of them
    at::assert_no_overlap(out, residual);
    at::assert_no_overlap(out, input);
    at::assert_no_overlap(scale, residual);
    at::assert_no_overlap(scale, input);
    at::assert_no_overlap(scale, out);
  }
  return s;
}

void rms_norm_fp8_hip(at::Tensor& out, at::Tensor& scale, const at::Tensor& input, const at::Tensor& weight,
                      at::Tensor& residual, double eps) {
  const Fp8Shape s = check_fp8(out, scale, input, weight, residual);
  if (s.f.rows == 0 || s.f.hidden == 0) return;
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  check_status(hprms_fused_add_rmsnorm_fp8(out.data_ptr(), scale.data_ptr<float>(), input.data_ptr(),
                                           weight.data_ptr(), residual.data_ptr(), s.f.rows, s.f.hidden,
                                           s.out_stride, s.f.in_stride, s.f.res_stride, s.f.dtype, eps, stream));
}

void rms_norm_fp8_meta(at::Tensor& out, at::Tensor& scale, const at::Tensor& input, const at::Tensor& weight,
                       at::Tensor& residual, double eps) {
  (void)check_fp8(out, scale, input, weight, residual);
  (void)eps;
}

// ---- FP8 output with per-row scales bounded above ------------------------------------
Fp8Shape check_fp8_ub(const at::Tensor& out, const at::Tensor& scale, const at::Tensor& input,
                      const at::Tensor& weight, const at::Tensor& residual, const at::Tensor& scale_ub) {
  const Fp8Shape s = check_fp8(out, scale, input, weight, residual);
  TORCH_CHECK(scale_ub.scalar_type() == at::kFloat, "scale_ub.dtype() == float32");
  TORCH_CHECK(scale_ub.numel() == 1, "scale_ub must hold one element");
  TORCH_CHECK(scale_ub.device() == input.device(), "scale_ub and input must be on the same device");
  if (s.f.rows > 0) at::assert_no_overlap(scale, scale_ub);
  return s;
}

void rms_norm_fp8_ub_hip(at::Tensor& out, at::Tensor& scale, const at::Tensor& input, const at::Tensor& weight,
                         at::Tensor& residual, const at::Tensor& scale_ub, double eps) {
  const Fp8Shape s = check_fp8_ub(out, scale, input, weight, residual, scale_ub);
  if (s.f.rows == 0 || s.f.hidden == 0) return;
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  check_status(hprms_fused_add_rmsnorm_fp8_ub(out.data_ptr(), scale.data_ptr<float>(), scale_ub.data_ptr<float>(),
                                              input.data_ptr(), weight.data_ptr(), residual.data_ptr(), s.f.rows,
                                              s.f.hidden, s.out_stride, s.f.in_stride, s.f.res_stride, s.f.dtype,
                                              eps, stream));
}

void rms_norm_fp8_ub_meta(at::Tensor& out, at::Tensor& scale, const at::Tensor& input, const at::Tensor& weight,
                          at::Tensor& residual, const at::Tensor& scale_ub, double eps) {
  (void)check_fp8_ub(out, scale, input, weight, residual, scale_ub);
  (void)eps;
}

// ---- FP8 output with one given scale ---------------------------------------------------
Fp8Shape check_fp8_static(const at::Tensor& out, const at::Tensor& scale, const at::Tensor& input,
                          const at::Tensor& weight, const at::Tensor& residual) {
  Fp8Shape s;
  s.f = check_fused(input, weight, residual);
  TORCH_CHECK(out.scalar_type() == at::kFloat8_e4m3fn, "out.dtype() == float8_e4m3fn");
  TORCH_CHECK(scale.scalar_type() == at::kFloat, "scale.dtype() == float32");
  TORCH_CHECK(scale.numel() == 1, "scale must hold one element (one scale for every row)");
  TORCH_CHECK(out.dim() == input.dim(), "out.dim() == input.dim()");
  for (int64_t i = 0; i < input.dim(); ++i) TORCH_CHECK(out.size(i) == input.size(i), "out.size(i) == input.size(i)");
  TORCH_CHECK(out.stride(-1) == 1, "out.stride(-1) == 1");
  TORCH_CHECK(out.device() == input.device() && scale.device() == input.device(),
              "out, scale and input must be on the same device");
  int64_t orows = 0;
  rows_of(out, s.f.hidden, &orows, &s.out_stride);
  if (s.f.rows > 0) {
    // the FP8 rows are written while input, residual and the scale are read
    at::assert_no_overlap(out, residual);
    at::assert_no_overlap(out, input);
    at::assert_no_overlap(out, scale);
    at::assert_no_overlap(residual, scale);
  }
  return s;
}

void rms_norm_fp8_static_hip(at::Tensor& out, const at::Tensor& scale, const at::Tensor& input,
                             const at::Tensor& weight, at::Tensor& residual, double eps) {
  const Fp8Shape s = check_fp8_static(out, scale, input, weight, residual);
  if (s.f.rows == 0 || s.f.hidden == 0) return;
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  check_status(hprms_fused_add_rmsnorm_fp8_static(out.data_ptr(), scale.data_ptr<float>(), input.data_ptr(),
                                                  weight.data_ptr(), residual.data_ptr(), s.f.rows, s.f.hidden,
                                                  s.out_stride, s.f.in_stride, s.f.res_stride, s.f.dtype, eps,
                                                  stream));
}

void rms_norm_fp8_static_meta(at::Tensor& out, const at::Tensor& scale, const at::Tensor& input,
                              const at::Tensor& weight, at::Tensor& residual, double eps) {
  (void)check_fp8_static(out, scale, input, weight, residual);
  (void)eps;
}

// ---- FP8 output with a scale per 128 elements -------------------------------------------
struct GroupShape {
  FusedShape f;
  int64_t out_stride, scale_stride, scale_group_stride;
};

GroupShape check_fp8_group(const at::Tensor& out, const at::Tensor& scales, const at::Tensor& input,
                           const at::Tensor& weight, const at::Tensor& residual) {
  GroupShape s;
  s.f = check_fused(input, weight, residual);
  TORCH_CHECK(s.f.hidden % 128 == 0, "the FP8 output with a scale per 128 elements needs hidden_dim % 128 == 0");
  TORCH_CHECK(out.scalar_type() == at::kFloat8_e4m3fn, "out.dtype() == float8_e4m3fn");
  TORCH_CHECK(scales.scalar_type() == at::kFloat, "scales.dtype() == float32");
  for (const at::Tensor* t : {&out, &scales}) {
    TORCH_CHECK(t->dim() == input.dim(), "out and scales must have input.dim() dimensions");
    for (int64_t i = 0; i + 1 < input.dim(); ++i)
      TORCH_CHECK(t->size(i) == input.size(i), "out and scales must match input in the leading dimensions");
    TORCH_CHECK(t->device() == input.device(), "out, scales and input must be on the same device");
  }
  TORCH_CHECK(out.stride(-1) == 1, "out must be contiguous in the last dimension");
  TORCH_CHECK(out.size(-1) == s.f.hidden, "out.size(-1) == hidden_dim");
  TORCH_CHECK(scales.size(-1) == s.f.hidden / 128, "scales.size(-1) must be hidden / 128 = ", s.f.hidden / 128);
  int64_t r = 0;
  rows_of(out, s.f.hidden, &r, &s.out_stride);
  // scales: rows of scales or the column-major (token-minor) layout; the
  // leading dimensions must flatten to one row stride, and the C ABI rejects
  // strides under which two (row, group) pairs share a scale
  TORCH_CHECK(at::has_internal_overlap(scales) != at::MemOverlap::Yes, "scales must not overlap themselves");
  s.scale_stride = 0;
  s.scale_group_stride = 1;
  if (s.f.hidden > 0) {
    const at::Tensor flat = scales.view({-1, s.f.hidden / 128});
    s.scale_stride = flat.size(0) <= 1 ? s.f.hidden / 128 : flat.stride(0);
    s.scale_group_stride = flat.size(1) <= 1 ? 1 : flat.stride(1);
  }
  if (s.f.rows > 0) {
    at::assert_no_overlap(out, scales);
    at::assert_no_overlap(out, residual);
    at::assert_no_overlap(out, input);
    at::assert_no_overlap(scales, residual);
    at::assert_no_overlap(scales, input);
  }
  return s;
}

void rms_norm_fp8_group_hip(at::Tensor& out, at::Tensor& scales, const at::Tensor& input, const at::Tensor& weight,
                            at::Tensor& residual, double eps) {
  const GroupShape s = check_fp8_group(out, scales, input, weight, residual);
  if (s.f.rows == 0 || s.f.hidden == 0) return;
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  check_status(hprms_fused_add_rmsnorm_fp8_group(out.data_ptr(), scales.data_ptr<float>(), input.data_ptr(),
                                                 weight.data_ptr(), residual.data_ptr(), s.f.rows, s.f.hidden,
                                                 s.out_stride, s.scale_stride, s.scale_group_stride,
                                                 s.f.in_stride, s.f.res_stride, s.f.dtype, eps, stream));
}

void rms_norm_fp8_group_meta(at::Tensor& out, at::Tensor& scales, const at::Tensor& input, const at::Tensor& weight,
                             at::Tensor& residual, double eps) {
  (void)check_fp8_group(out, scales, input, weight, residual);
  (void)eps;
}

// ---- fused op out of place ----------------------------------------------------------
FusedShape check_fused_out(const at::Tensor& out, const at::Tensor& residual_out, const at::Tensor& input,
                           const at::Tensor& weight, const at::Tensor& residual) {
  TORCH_CHECK(input.dim() >= 2, "input.dim() >= 2");
  const int64_t hidden = weight.dim() == 1 ? weight.size(0) : -1;
  for (const at::Tensor* t : {&residual, &out, &residual_out}) {
    TORCH_CHECK(t->dim() == input.dim(), "all row tensors must have input.dim() dimensions");
    for (int64_t i = 0; i < input.dim(); ++i) TORCH_CHECK(t->size(i) == input.size(i), "input.size(i) == residual.size(i)");
    TORCH_CHECK(t->stride(-1) == 1, "rows must be contiguous (stride(-1) == 1)");
    TORCH_CHECK(t->scalar_type() == input.scalar_type(), "all tensors must have input.dtype()");
    TORCH_CHECK(t->device() == input.device(), "all tensors must be on input's device");
  }
  TORCH_CHECK(weight.dim() == 1, "weight.dim() == 1");
  TORCH_CHECK(input.size(-1) == hidden, "input.size(-1) == hidden_dim");
  TORCH_CHECK(input.stride(-1) == 1, "input.stride(-1) == 1");
  TORCH_CHECK(weight.stride(0) == 1 || hidden == 1, "weight.stride(0) == 1");
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(), "weight.dtype() == input.dtype()");
  TORCH_CHECK(weight.device() == input.device(), "weight must be on input's device");
  FusedShape s;
  s.dtype = dtype_code(input);
  s.hidden = hidden;
  rows_of(input, hidden, &s.rows, &s.in_stride);
  int64_t r = 0, st = 0;
  rows_of(residual, hidden, &r, &s.res_stride);
  rows_of(out, hidden, &r, &st);
  rows_of(residual_out, hidden, &r, &st);
  if (s.rows > 0) {
    // out may be input and residual_out may be residual (in place); no other sharing
    at::assert_no_overlap(out, residual_out);
    at::assert_no_overlap(out, residual);
    at::assert_no_overlap(residual_out, input);
    at::assert_no_partial_overlap(out, input);
    at::assert_no_partial_overlap(residual_out, residual);
  }
  return s;
}

void rms_norm_out_hip(at::Tensor& out, at::Tensor& residual_out, const at::Tensor& input, const at::Tensor& weight,
                      const at::Tensor& residual, double eps) {
  const FusedShape s = check_fused_out(out, residual_out, input, weight, residual);
  if (s.rows == 0 || s.hidden == 0) return;
  int64_t r = 0, out_stride = 0, res_out_stride = 0;
  rows_of(out, s.hidden, &r, &out_stride);
  rows_of(residual_out, s.hidden, &r, &res_out_stride);
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  check_status(hprms_fused_add_rmsnorm_out(out.data_ptr(), residual_out.data_ptr(), input.data_ptr(),
                                           residual.data_ptr(), weight.data_ptr(), s.rows, s.hidden, out_stride,
                                           res_out_stride, s.in_stride, s.res_stride, s.dtype, eps, stream));
}

void rms_norm_out_meta(at::Tensor& out, at::Tensor& residual_out, const at::Tensor& input, const at::Tensor& weight,
                       const at::Tensor& residual, double eps) {
  (void)check_fused_out(out, residual_out, input, weight, residual);
  (void)eps;
}

// ---- partial-sum reduction + fused op ----------------------------------------------------
struct ReduceShape {
  int64_t rows, hidden, out_stride, part_stride, res_stride;
  int dtype;
};

ReduceShape check_reduce(const at::Tensor& out, at::TensorList parts, const at::Tensor& weight,
                         const at::Tensor& residual) {
  TORCH_CHECK(!parts.empty() && (int64_t)parts.size() <= HPRMS_MAX_PARTS, "parts must hold 1 to ",
              HPRMS_MAX_PARTS, " tensors (got ", parts.size(), ")");
  TORCH_CHECK(residual.dim() >= 2, "input.dim() >= 2");
  TORCH_CHECK(weight.dim() == 1, "weight.dim() == 1");
  const int64_t hidden = weight.size(0);
  TORCH_CHECK(residual.size(-1) == hidden, "input.size(-1) == hidden_dim");
  TORCH_CHECK(weight.stride(0) == 1 || hidden == 1, "weight.stride(0) == 1");
  ReduceShape s;
  s.dtype = dtype_code(residual);
  s.hidden = hidden;
  TORCH_CHECK(weight.scalar_type() == residual.scalar_type(), "weight.dtype() == input.dtype()");
  TORCH_CHECK(weight.device() == residual.device(), "weight must be on residual's device");
  for (const at::Tensor* t : {&out, &parts[0]}) {
    TORCH_CHECK(t->dim() == residual.dim(), "all row tensors must have residual.dim() dimensions");
    for (int64_t i = 0; i < residual.dim(); ++i)
      TORCH_CHECK(t->size(i) == residual.size(i), "input.size(i) == residual.size(i)");
  }
  for (const at::Tensor* t : {&residual, &out}) {
    TORCH_CHECK(t->stride(-1) == 1, "rows must be contiguous (stride(-1) == 1)");
    TORCH_CHECK(t->scalar_type() == residual.scalar_type(), "all tensors must have residual.dtype()");
    TORCH_CHECK(t->device() == residual.device(), "all tensors must be on residual's device");
  }
  rows_of(residual, hidden, &s.rows, &s.res_stride);
  int64_t r = 0;
  rows_of(out, hidden, &r, &s.out_stride);
  for (size_t g = 0; g < parts.size(); ++g) {
    const at::Tensor& p = parts[g];
    TORCH_CHECK(p.sizes() == parts[0].sizes(), "every part must have the shape of the residual");
    TORCH_CHECK(p.stride(-1) == 1, "rows must be contiguous (stride(-1) == 1)");
    TORCH_CHECK(p.scalar_type() == residual.scalar_type(), "all tensors must have residual.dtype()");
    TORCH_CHECK(p.device() == residual.device(), "all tensors must be on residual's device");
    int64_t st = 0;
    rows_of(p, hidden, &r, &st);
    if (g == 0) s.part_stride = st;
    TORCH_CHECK(st == s.part_stride, "all parts must share one row stride");
    if (s.rows > 0) {
      at::assert_no_overlap(p, residual);
      at::assert_no_partial_overlap(out, p);
    }
  }
  if (s.rows > 0) at::assert_no_overlap(out, residual);
  return s;
}

void reduce_rms_norm_hip(at::Tensor& out, at::TensorList parts, const at::Tensor& weight, at::Tensor& residual,
                         double eps) {
  const ReduceShape s = check_reduce(out, parts, weight, residual);
  if (s.rows == 0 || s.hidden == 0) return;
  const void* ptrs[HPRMS_MAX_PARTS];
  for (size_t g = 0; g < parts.size(); ++g) ptrs[g] = parts[g].data_ptr();
  c10::DeviceGuard guard(residual.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(residual.device().index()).stream();
  check_status(hprms_reduce_add_rmsnorm(out.data_ptr(), ptrs, (int)parts.size(), weight.data_ptr(),
                                        residual.data_ptr(), s.rows, s.hidden, s.out_stride, s.part_stride,
                                        s.res_stride, s.dtype, eps, stream));
}

void reduce_rms_norm_meta(at::Tensor& out, at::TensorList parts, const at::Tensor& weight, at::Tensor& residual,
                          double eps) {
  (void)check_reduce(out, parts, weight, residual);
  (void)eps;
}

// ---- fused op with an OCP MX output ---------------------------------------------------
struct MxShape {
  FusedShape f;
  int64_t out_stride, scale_stride;
};

MxShape check_mx(const at::Tensor& out, const at::Tensor& scales, const at::Tensor& input, const at::Tensor& weight,
                 const at::Tensor& residual, int64_t format) {
  TORCH_CHECK(format == HPRMS_MX_FP8_E4M3 || format == HPRMS_MX_FP4_E2M1,
              "format must be 0 (MXFP8, E4M3) or 1 (MXFP4, E2M1)");
  MxShape s;
  s.f = check_fused(input, weight, residual);
  TORCH_CHECK(s.f.hidden % 32 == 0, "MX output needs hidden_dim % 32 == 0");
  const bool fp8 = format == HPRMS_MX_FP8_E4M3;
  TORCH_CHECK(out.scalar_type() == at::kByte ||
                  out.scalar_type() == (fp8 ? at::kFloat8_e4m3fn : at::kFloat4_e2m1fn_x2),
              fp8 ? "out.dtype() must be float8_e4m3fn or uint8" : "out.dtype() must be float4_e2m1fn_x2 or uint8");
  TORCH_CHECK(scales.scalar_type() == at::kByte || scales.scalar_type() == at::kFloat8_e8m0fnu,
              "scales.dtype() must be float8_e8m0fnu or uint8");
  const int64_t qw = fp8 ? s.f.hidden : s.f.hidden / 2;
  for (const at::Tensor* t : {&out, &scales}) {
    TORCH_CHECK(t->dim() == input.dim(), "out and scales must have input.dim() dimensions");
    for (int64_t i = 0; i + 1 < input.dim(); ++i)
      TORCH_CHECK(t->size(i) == input.size(i), "out and scales must match input in the leading dimensions");
    TORCH_CHECK(t->stride(-1) == 1, "out and scales must be contiguous in the last dimension");
    TORCH_CHECK(t->device() == input.device(), "out, scales and input must be on the same device");
  }
  TORCH_CHECK(out.size(-1) == qw, "out.size(-1) must be ", qw, " (", fp8 ? "hidden" : "hidden / 2", ")");
  TORCH_CHECK(scales.size(-1) == s.f.hidden / 32, "scales.size(-1) must be hidden / 32 = ", s.f.hidden / 32);
  int64_t r = 0;
  rows_of(out, qw, &r, &s.out_stride);
  rows_of(scales, s.f.hidden / 32, &r, &s.scale_stride);
  if (s.f.rows > 0) {
    at::assert_no_overlap(out, scales);
    at::assert_no_overlap(out, residual);
    at::assert_no_overlap(out, input);
    at::assert_no_overlap(scales, residual);
    at::assert_no_overlap(scales, input);
  }
  return s;
}

void rms_norm_mx_hip(at::Tensor& out, at::Tensor& scales, const at::Tensor& input, const at::Tensor& weight,
                     at::Tensor& residual, int64_t format, double eps) {
  const MxShape s = check_mx(out, scales, input, weight, residual, format);
  if (s.f.rows == 0 || s.f.hidden == 0) return;
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  check_status(hprms_fused_add_rmsnorm_mx(out.data_ptr(), scales.data_ptr(), input.data_ptr(), weight.data_ptr(),
                                          residual.data_ptr(), s.f.rows, s.f.hidden, s.out_stride, s.scale_stride,
                                          s.f.in_stride, s.f.res_stride, (int)format, s.f.dtype, eps, stream));
}

void rms_norm_mx_meta(at::Tensor& out, at::Tensor& scales, const at::Tensor& input, const at::Tensor& weight,
                      at::Tensor& residual, int64_t format, double eps) {
  (void)check_mx(out, scales, input, weight, residual, format);
  (void)eps;
}

// ---- training: gradients, the loss, clipping ------------------------------------------
// Workspace of a call on the current stream: from torch's allocator, which hands
// its memory out again only behind this call's work on that stream (and, in a
// captured graph, keeps it to the graph).
at::Tensor workspace_of(int64_t bytes, const at::Tensor& like) {
  TORCH_CHECK(bytes >= 0, "hp_rms_norm: ", hprms_last_error(), " (status ", bytes, ")");
  return at::empty({bytes > 0 ? bytes : 1}, like.options().dtype(at::kByte).requires_grad(false));
}

struct BackwardShape {
  int64_t rows, hidden, din_stride, dout_stride, in_stride, dres_stride;
  int dtype, dweight_dtype;
};

BackwardShape check_backward(const at::Tensor& dinput, const at::Tensor& dweight, const at::Tensor& dout,
                             const at::Tensor& input, const at::Tensor& weight,
                             const std::optional<at::Tensor>& dresidual) {
  TORCH_CHECK(input.dim() >= 2, "input.dim() >= 2");
  TORCH_CHECK(weight.dim() == 1, "weight.dim() == 1");
  BackwardShape s;
  s.hidden = weight.size(0);
  s.dtype = dtype_code(input);
  TORCH_CHECK(input.size(-1) == s.hidden, "input.size(-1) == hidden_dim");
  TORCH_CHECK(weight.stride(0) == 1 || s.hidden <= 1, "weight.stride(0) == 1");
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(), "weight.dtype() == input.dtype()");
  TORCH_CHECK(weight.device() == input.device(), "weight must be on input's device");
  TORCH_CHECK(dweight.dim() == 1 && dweight.size(0) == s.hidden, "dweight must be shaped like weight");
  TORCH_CHECK(dweight.stride(0) == 1 || s.hidden <= 1, "dweight.stride(0) == 1");
  TORCH_CHECK(dweight.scalar_type() == input.scalar_type() || dweight.scalar_type() == at::kFloat,
              "dweight.dtype() must be weight.dtype() or float32");
  TORCH_CHECK(dweight.device() == input.device(), "dweight must be on input's device");
  s.dweight_dtype = dweight.scalar_type() == at::kFloat ? HPRMS_DTYPE_FP32 : s.dtype;
  const at::Tensor* rows[4] = {&input, &dout, &dinput, dresidual ? &*dresidual : &input};
  for (const at::Tensor* t : rows) {
    TORCH_CHECK(t->sizes() == input.sizes(), "dinput, dout and dresidual must be shaped like input");
    TORCH_CHECK(t->stride(-1) == 1 || s.hidden <= 1, "rows must be contiguous (stride(-1) == 1)");
    TORCH_CHECK(t->scalar_type() == input.scalar_type(), "dinput, dout and dresidual must have input.dtype()");
    TORCH_CHECK(t->device() == input.device(), "all tensors must be on input's device");
  }
  int64_t r = 0;
  rows_of(input, s.hidden, &s.rows, &s.in_stride);
  rows_of(dout, s.hidden, &r, &s.dout_stride);
  rows_of(dinput, s.hidden, &r, &s.din_stride);
  rows_of(*rows[3], s.hidden, &r, &s.dres_stride);
  if (s.rows > 0 && s.hidden > 0) {
    // dinput may lie on any one of the row tensors exactly: a row is read before it is written
    for (const at::Tensor* t : rows)
      if (t != &dinput) at::assert_no_partial_overlap(dinput, *t);
    at::assert_no_overlap(dinput, weight);
    for (const at::Tensor* t : rows) at::assert_no_overlap(dweight, *t);
    at::assert_no_overlap(dweight, weight);
  }
  return s;
}

void rms_norm_backward_hip(at::Tensor& dinput, at::Tensor& dweight, const at::Tensor& dout, const at::Tensor& input,
                           const at::Tensor& weight, const std::optional<at::Tensor>& dresidual, double eps) {
  const BackwardShape s = check_backward(dinput, dweight, dout, input, weight, dresidual);
  if (s.hidden == 0) return;
  c10::DeviceGuard guard(input.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(input.device().index()).stream();
  const at::Tensor ws = workspace_of(hprms_rmsnorm_backward_workspace(s.rows, s.hidden), input);
  check_status(hprms_rmsnorm_backward(dinput.data_ptr(), dweight.data_ptr(), dout.data_ptr(), input.data_ptr(),
                                      weight.data_ptr(), dresidual ? dresidual->data_ptr() : nullptr, ws.data_ptr(),
                                      ws.numel(), s.rows, s.hidden, s.din_stride, s.dout_stride, s.in_stride,
                                      s.dres_stride, s.dtype, s.dweight_dtype, eps, stream));
}

void rms_norm_backward_meta(at::Tensor& dinput, at::Tensor& dweight, const at::Tensor& dout, const at::Tensor& input,
                            const at::Tensor& weight, const std::optional<at::Tensor>& dresidual, double eps) {
  (void)check_backward(dinput, dweight, dout, input, weight, dresidual);
  (void)eps;
}

struct LossShape {
  int64_t rows, hidden, vocab, hidden_stride, weight_stride;
  int dtype;
};

// Rows and row stride of a [vocab, hidden] matrix.
int64_t matrix_stride(const at::Tensor& t, int64_t hidden) {
  const int64_t stride = t.size(0) <= 1 ? hidden : t.stride(0);
  TORCH_CHECK(stride >= hidden, "rows of the tensor overlap (row stride ", stride, " < hidden ", hidden, ")");
  return stride;
}

LossShape check_loss(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target,
                     std::initializer_list<const at::Tensor*> per_row) {
  TORCH_CHECK(hidden.dim() >= 2, "hidden.dim() >= 2");
  TORCH_CHECK(weight.dim() == 2, "weight.dim() == 2");
  LossShape s;
  s.vocab = weight.size(0);
  s.hidden = weight.size(1);
  s.dtype = dtype_code(hidden);
  TORCH_CHECK(hidden.size(-1) == s.hidden, "hidden.size(-1) == weight.size(1)");
  TORCH_CHECK(s.hidden >= 1 && s.vocab >= 1, "weight must hold at least one element");
  TORCH_CHECK(hidden.stride(-1) == 1 || s.hidden == 1, "hidden.stride(-1) == 1");
  TORCH_CHECK(weight.stride(1) == 1 || s.hidden == 1, "weight.stride(1) == 1");
  TORCH_CHECK(weight.scalar_type() == hidden.scalar_type(), "weight.dtype() == hidden.dtype()");
  TORCH_CHECK(weight.device() == hidden.device() && target.device() == hidden.device(),
              "hidden, weight and target must be on the same device");
  TORCH_CHECK(target.scalar_type() == at::kLong, "target.dtype() == int64");
  TORCH_CHECK(target.sizes() == hidden.sizes().slice(0, hidden.dim() - 1), "target must have one element per row");
  TORCH_CHECK(target.is_contiguous(), "target must be contiguous");
  for (const at::Tensor* t : per_row) {
    TORCH_CHECK(t->scalar_type() == at::kFloat, "loss, lse and dloss must be float32");
    TORCH_CHECK(t->sizes() == target.sizes(), "loss, lse and dloss must be shaped like target");
    TORCH_CHECK(t->is_contiguous(), "loss, lse and dloss must be contiguous");
    TORCH_CHECK(t->device() == hidden.device(), "all tensors must be on hidden's device");
  }
  rows_of(hidden, s.hidden, &s.rows, &s.hidden_stride);
  s.weight_stride = matrix_stride(weight, s.hidden);
  return s;
}

LossShape check_loss_forward(const at::Tensor& loss, const at::Tensor& lse, const at::Tensor& hidden,
                             const at::Tensor& weight, const at::Tensor& target) {
  const LossShape s = check_loss(hidden, weight, target, {&loss, &lse});
  if (s.rows > 0) {
    at::assert_no_overlap(loss, lse);
    for (const at::Tensor* out : {&loss, &lse})
      for (const at::Tensor* in : {&hidden, &weight, &target}) at::assert_no_overlap(*out, *in);
  }
  return s;
}

void linear_cross_entropy_hip(at::Tensor& loss, at::Tensor& lse, const at::Tensor& hidden, const at::Tensor& weight,
                              const at::Tensor& target, int64_t ignore_index) {
  const LossShape s = check_loss_forward(loss, lse, hidden, weight, target);
  if (s.rows == 0) return;
  c10::DeviceGuard guard(hidden.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(hidden.device().index()).stream();
  const at::Tensor ws = workspace_of(
      hprms_linear_cross_entropy_workspace(s.rows, s.hidden, s.vocab, weight.data_ptr(), s.weight_stride), hidden);
  check_status(hprms_linear_cross_entropy(loss.data_ptr<float>(), lse.data_ptr<float>(), hidden.data_ptr(),
                                          weight.data_ptr(), target.data_ptr<int64_t>(), ws.data_ptr(), ws.numel(),
                                          s.rows, s.hidden, s.vocab, s.hidden_stride, s.weight_stride, ignore_index,
                                          s.dtype, stream));
}

void linear_cross_entropy_meta(at::Tensor& loss, at::Tensor& lse, const at::Tensor& hidden, const at::Tensor& weight,
                               const at::Tensor& target, int64_t ignore_index) {
  (void)check_loss_forward(loss, lse, hidden, weight, target);
  (void)ignore_index;
}

struct LossGradShape {
  LossShape f;
  int64_t dhidden_stride, dweight_stride;
};

LossGradShape check_loss_backward(const at::Tensor& dhidden, const at::Tensor& dweight, const at::Tensor& dloss,
                                  const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target,
                                  const at::Tensor& lse) {
  LossGradShape s;
  s.f = check_loss(hidden, weight, target, {&lse, &dloss});
  TORCH_CHECK(dhidden.sizes() == hidden.sizes(), "dhidden must be shaped like hidden");
  TORCH_CHECK(dweight.sizes() == weight.sizes(), "dweight must be shaped like weight");
  for (const at::Tensor* t : {&dhidden, &dweight}) {
    TORCH_CHECK(t->stride(-1) == 1 || s.f.hidden == 1, "rows must be contiguous (stride(-1) == 1)");
    TORCH_CHECK(t->scalar_type() == hidden.scalar_type(), "dhidden and dweight must have hidden.dtype()");
    TORCH_CHECK(t->device() == hidden.device(), "all tensors must be on hidden's device");
  }
  int64_t r = 0;
  rows_of(dhidden, s.f.hidden, &r, &s.dhidden_stride);
  s.dweight_stride = matrix_stride(dweight, s.f.hidden);
  at::assert_no_overlap(dweight, weight);
  if (s.f.rows > 0) {
    at::assert_no_overlap(dhidden, dweight);
    for (const at::Tensor* out : {&dhidden, &dweight})
      for (const at::Tensor* in : {&hidden, &weight, &target, &lse, &dloss}) at::assert_no_overlap(*out, *in);
  }
  return s;
}

void linear_cross_entropy_backward_hip(at::Tensor& dhidden, at::Tensor& dweight, const at::Tensor& dloss,
                                       const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target,
                                       const at::Tensor& lse, int64_t ignore_index) {
  const LossGradShape s = check_loss_backward(dhidden, dweight, dloss, hidden, weight, target, lse);
  c10::DeviceGuard guard(hidden.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(hidden.device().index()).stream();
  const at::Tensor ws = workspace_of(
      hprms_linear_cross_entropy_backward_workspace(s.f.rows, s.f.hidden, s.f.vocab, weight.data_ptr(),
                                                    s.f.weight_stride),
      hidden);
  check_status(hprms_linear_cross_entropy_backward(
      dhidden.data_ptr(), dweight.data_ptr(), dloss.data_ptr<float>(), hidden.data_ptr(), weight.data_ptr(),
      target.data_ptr<int64_t>(), lse.data_ptr<float>(), ws.data_ptr(), ws.numel(), s.f.rows, s.f.hidden, s.f.vocab,
      s.dhidden_stride, s.dweight_stride, s.f.hidden_stride, s.f.weight_stride, ignore_index, s.f.dtype, stream));
}

void linear_cross_entropy_backward_meta(at::Tensor& dhidden, at::Tensor& dweight, const at::Tensor& dloss,
                                        const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target,
                                        const at::Tensor& lse, int64_t ignore_index) {
  (void)check_loss_backward(dhidden, dweight, dloss, hidden, weight, target, lse);
  (void)ignore_index;
}

int grad_dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat) return HPRMS_DTYPE_FP32;
  if (t.scalar_type() == at::kBFloat16) return HPRMS_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return HPRMS_DTYPE_FP16;
  TORCH_CHECK(false, "gradients must be bfloat16, float16 or float32");
  return -1;
}

// [first, last) bytes of a dense tensor's elements
struct Span {
  uintptr_t first, last;
  size_t i;
};

Span span_of(const at::Tensor& t, size_t i) {
  const uintptr_t p = (uintptr_t)t.data_ptr();
  return {p, p + (uintptr_t)t.numel() * t.element_size(), i};
}

void check_grads(const at::Tensor& norm, at::TensorList grads) {
  TORCH_CHECK(!grads.empty(), "grads must hold at least one tensor");
  TORCH_CHECK(norm.scalar_type() == at::kFloat && norm.numel() == 1, "norm must hold one float32");
  for (const at::Tensor& g : grads) {
    (void)grad_dtype_code(g);
    TORCH_CHECK(g.device() == norm.device(), "all gradients must be on one device");
    TORCH_CHECK(g.is_non_overlapping_and_dense(), "gradients must be dense in memory");
  }
}

void check_outs(at::TensorList outs, at::TensorList grads) {
  TORCH_CHECK(outs.size() == grads.size(), "outs must hold one tensor per gradient");
  for (size_t i = 0; i < outs.size(); ++i) {
    TORCH_CHECK(outs[i].sizes() == grads[i].sizes(), "outs[i] must be shaped like grads[i]");
    TORCH_CHECK(outs[i].is_non_overlapping_and_dense() && (outs[i].strides() == grads[i].strides() ||
                                                           (outs[i].is_contiguous() && grads[i].is_contiguous())),
                "outs[i] must be laid out like grads[i]");
    TORCH_CHECK(outs[i].device() == grads[i].device(), "outs must be on the gradients' device");
    TORCH_CHECK(outs[i].scalar_type() == grads[i].scalar_type() || outs[i].scalar_type() == at::kFloat,
                "outs[i].dtype() must be grads[i].dtype() or float32");
  }
}

// No output shares memory with another output, with the norm or with a
// gradient other than its own (which it must then be, exactly).
void check_out_spans(const at::Tensor& norm, at::TensorList outs, at::TensorList grads) {
  std::vector<Span> spans;
  spans.reserve(outs.size());
  for (size_t i = 0; i < outs.size(); ++i)
    if (outs[i].numel() > 0) spans.push_back(span_of(outs[i], i));
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.first < b.first; });
  for (size_t i = 1; i < spans.size(); ++i)
    TORCH_CHECK(spans[i - 1].last <= spans[i].first, "two of the tensors to be written share memory");
  auto meets = [&](const Span& s, bool own) {
    // the first output that ends after s begins
    auto it = std::upper_bound(spans.begin(), spans.end(), s.first,
                               [](uintptr_t v, const Span& o) { return v < o.last; });
    for (; it != spans.end() && it->first < s.last; ++it)
      TORCH_CHECK(own && it->i == s.i && it->first == s.first && it->last == s.last,
                  "a tensor to be written shares memory with another tensor");
  };
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].numel() > 0) meets(span_of(grads[i], i), true);
  meets(span_of(norm, 0), false);
}

struct GradArrays {
  std::vector<void*> outs;
  std::vector<const void*> grads;
  std::vector<int> out_dtypes, dtypes;
  std::vector<int64_t> counts;
};

GradArrays grad_arrays(at::TensorList outs, at::TensorList grads) {
  GradArrays a;
  a.outs.reserve(outs.size());
  a.out_dtypes.reserve(outs.size());
  a.grads.reserve(grads.size());
  a.dtypes.reserve(grads.size());
  a.counts.reserve(grads.size());
  for (const at::Tensor& t : outs) {
    a.outs.push_back(t.data_ptr());
    a.out_dtypes.push_back(grad_dtype_code(t));
  }
  for (const at::Tensor& t : grads) {
    a.grads.push_back(t.data_ptr());
    a.dtypes.push_back(grad_dtype_code(t));
    a.counts.push_back(t.numel());
  }
  return a;
}

void grad_norm_hip(at::Tensor& norm, at::TensorList grads) {
  check_grads(norm, grads);
  const GradArrays a = grad_arrays({}, grads);
  const int n = (int)grads.size();
  c10::DeviceGuard guard(norm.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(norm.device().index()).stream();
  const at::Tensor ws = workspace_of(hprms_grad_norm_workspace(a.counts.data(), n), norm);
  check_status(hprms_grad_norm(norm.data_ptr<float>(), a.grads.data(), a.dtypes.data(), a.counts.data(), n,
                               ws.data_ptr(), ws.numel(), stream));
}

void grad_norm_meta(at::Tensor& norm, at::TensorList grads) { check_grads(norm, grads); }

void clip_grad_norm_out_hip(at::Tensor& norm, at::TensorList outs, at::TensorList grads, double max_norm) {
  check_grads(norm, grads);
  check_outs(outs, grads);
  check_out_spans(norm, outs, grads);
  const GradArrays a = grad_arrays(outs, grads);
  const int n = (int)grads.size();
  c10::DeviceGuard guard(norm.device());
  hipStream_t stream = c10::hip::getCurrentHIPStream(norm.device().index()).stream();
  const at::Tensor ws = workspace_of(hprms_grad_norm_workspace(a.counts.data(), n), norm);
  check_status(hprms_clip_grad_norm(norm.data_ptr<float>(), a.outs.data(), a.out_dtypes.data(), a.grads.data(),
                                    a.dtypes.data(), a.counts.data(), n, max_norm, ws.data_ptr(), ws.numel(), stream));
}

void clip_grad_norm_out_meta(at::Tensor& norm, at::TensorList outs, at::TensorList grads, double max_norm) {
  check_grads(norm, grads);
  check_outs(outs, grads);
  (void)max_norm;
}

void clip_grad_norm_hip_(at::Tensor& norm, at::TensorList grads, double max_norm) {
  clip_grad_norm_out_hip(norm, grads, grads, max_norm);
}

void clip_grad_norm_meta_(at::Tensor& norm, at::TensorList grads, double max_norm) {
  clip_grad_norm_out_meta(norm, grads, grads, max_norm);
}

// _C.set_batch_invariant(enable) -> previous setting; _C.batch_invariant()
// -> current setting (hprms_set_batch_invariant / hprms_batch_invariant).
PyObject* py_set_batch_invariant(PyObject*, PyObject* arg) {
  const int on = PyObject_IsTrue(arg);
  if (on < 0) return nullptr;
  const int previous = hprms_set_batch_invariant(on);
  if (previous < 0) {
    PyErr_SetString(PyExc_RuntimeError, hprms_last_error());
    return nullptr;
  }
  return PyBool_FromLong(previous);
}

PyObject* py_batch_invariant(PyObject*, PyObject*) { return PyBool_FromLong(hprms_batch_invariant()); }

PyMethodDef kMethods[] = {
    {"set_batch_invariant", py_set_batch_invariant, METH_O,
     "set_batch_invariant(enable) -> bool: choose each call's kernel shape by the width alone (a row's bits "
     "then do not depend on the call's row count); returns the previous setting"},
    {"batch_invariant", py_batch_invariant, METH_NOARGS, "batch_invariant() -> bool: the current setting"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

// Module init of `hp_rms_norm_amd._C`.  The operators live in torch's
// registry, so the module itself carries the C ABI version it was built
// against and the batch-invariant mode's setter and getter.
extern "C" PyObject* PyInit__C(void) {
  static PyModuleDef def = {PyModuleDef_HEAD_INIT, "_C",
                            "torch.ops.hp_rms_norm.* on the gfx950 kernels of libhprms.so", -1, kMethods};
  PyObject* m = PyModule_Create(&def);
  if (m && PyModule_AddIntConstant(m, "abi_version", hprms_abi_version()) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}

TORCH_LIBRARY(hp_rms_norm, m) {
  m.def("rms_norm(Tensor(a!) input, Tensor weight, Tensor(b!) residual, float eps) -> ()");
  m.def("relu(Tensor(a!) out, Tensor input) -> ()");
  m.def("relu_max0(Tensor(a!) out, Tensor input) -> ()");
  m.def("rms_norm_plain(Tensor(a!) out, Tensor input, Tensor weight, float eps) -> ()");
  m.def("rms_norm_fp8_quant(Tensor(a!) out, Tensor(b!) scale, Tensor input, Tensor weight, Tensor(c!) residual, "
        "float eps) -> ()");
  m.def("rms_norm_fp8_quant_ub(Tensor(a!) out, Tensor(b!) scale, Tensor input, Tensor weight, Tensor(c!) residual, "
        "Tensor scale_ub, float eps) -> ()");
  m.def("rms_norm_fp8_static_quant(Tensor(a!) out, Tensor scale, Tensor input, Tensor weight, Tensor(b!) residual, "
        "float eps) -> ()");
  m.def("rms_norm_fp8_group_quant(Tensor(a!) out, Tensor(b!) scales, Tensor input, Tensor weight, "
        "Tensor(c!) residual, float eps) -> ()");
  m.def("rms_norm_out(Tensor(a!) out, Tensor(b!) residual_out, Tensor input, Tensor weight, Tensor residual, "
        "float eps) -> ()");
  m.def("reduce_add_rms_norm(Tensor(a!) out, Tensor[] parts, Tensor weight, Tensor(b!) residual, float eps) -> ()");
  m.def("rms_norm_mx_quant(Tensor(a!) out, Tensor(b!) scales, Tensor input, Tensor weight, Tensor(c!) residual, "
        "int format, float eps) -> ()");
  m.def("rms_norm_backward(Tensor(a!) dinput, Tensor(b!) dweight, Tensor dout, Tensor input, Tensor weight, "
        "Tensor? dresidual, float eps) -> ()");
  m.def("linear_cross_entropy(Tensor(a!) loss, Tensor(b!) lse, Tensor hidden, Tensor weight, Tensor target, "
        "int ignore_index) -> ()");
  m.def("linear_cross_entropy_backward(Tensor(a!) dhidden, Tensor(b!) dweight, Tensor dloss, Tensor hidden, "
        "Tensor weight, Tensor target, Tensor lse, int ignore_index) -> ()");
  m.def("grad_norm(Tensor(a!) norm, Tensor[] grads) -> ()");
  m.def("clip_grad_norm_(Tensor(a!) norm, Tensor(b!)[] grads, float max_norm) -> ()");
  m.def("clip_grad_norm_out(Tensor(a!) norm, Tensor(b!)[] outs, Tensor[] grads, float max_norm) -> ()");
}

// ROCm builds of PyTorch expose HIP devices under the CUDA dispatch key.
TORCH_LIBRARY_IMPL(hp_rms_norm, CUDA, m) {
  m.impl("rms_norm", &rms_norm_hip);
  m.impl("relu", &relu_hip);
  m.impl("relu_max0", &relu_max0_hip);
  m.impl("rms_norm_plain", &rms_norm_plain_hip);
  m.impl("rms_norm_fp8_quant", &rms_norm_fp8_hip);
  m.impl("rms_norm_fp8_quant_ub", &rms_norm_fp8_ub_hip);
  m.impl("rms_norm_fp8_static_quant", &rms_norm_fp8_static_hip);
  m.impl("rms_norm_fp8_group_quant", &rms_norm_fp8_group_hip);
  m.impl("rms_norm_out", &rms_norm_out_hip);
  m.impl("reduce_add_rms_norm", &reduce_rms_norm_hip);
  m.impl("rms_norm_mx_quant", &rms_norm_mx_hip);
  m.impl("rms_norm_backward", &rms_norm_backward_hip);
  m.impl("linear_cross_entropy", &linear_cross_entropy_hip);
  m.impl("linear_cross_entropy_backward", &linear_cross_entropy_backward_hip);
  m.impl("grad_norm", &grad_norm_hip);
  m.impl("clip_grad_norm_", &clip_grad_norm_hip_);
  m.impl("clip_grad_norm_out", &clip_grad_norm_out_hip);
}

// Shape checks only, for fake tensors / torch.compile tracing.  Meta tensors
// carry no data, so nothing is computed here.
TORCH_LIBRARY_IMPL(hp_rms_norm, Meta, m) {
  m.impl("rms_norm", &rms_norm_meta);
  m.impl("relu", &stream_meta);
  m.impl("relu_max0", &stream_meta);
  m.impl("rms_norm_plain", &rms_norm_plain_meta);
  m.impl("rms_norm_fp8_quant", &rms_norm_fp8_meta);
  m.impl("rms_norm_fp8_quant_ub", &rms_norm_fp8_ub_meta);
  m.impl("rms_norm_fp8_static_quant", &rms_norm_fp8_static_meta);
  m.impl("rms_norm_fp8_group_quant", &rms_norm_fp8_group_meta);
  m.impl("rms_norm_out", &rms_norm_out_meta);
  m.impl("reduce_add_rms_norm", &reduce_rms_norm_meta);
  m.impl("rms_norm_mx_quant", &rms_norm_mx_meta);
  m.impl("rms_norm_backward", &rms_norm_backward_meta);
  m.impl("linear_cross_entropy", &linear_cross_entropy_meta);
  m.impl("linear_cross_entropy_backward", &linear_cross_entropy_backward_meta);
  m.impl("grad_norm", &grad_norm_meta);
  m.impl("clip_grad_norm_", &clip_grad_norm_meta_);
  m.impl("clip_grad_norm_out", &clip_grad_norm_out_meta);
}
