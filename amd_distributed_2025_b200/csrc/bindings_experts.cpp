// Python calls of the operators around a GPU's experts: rows with block scales (fp8_rows.h), tokens sorted by expert
// (moe_sort.h), the experts' fp8 products (fp8_gemm.h).  Shapes and types are looked at before devices, so that a wrong call is refused without a GPU too.
#include "bindings_experts.h"

#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <unordered_set>

#include "bindings_common.h"
#include "fp8_gemm.h"
#include "fp8_rows.h"
#include "moe_sort.h"

namespace {

using namespace b200::bind;
using c10::optional;

optional<at::Tensor> optional_arg(PyObject* o) {
  if (o == Py_None) return c10::nullopt;
  return tensor_arg(o);
}
int64_t int_arg(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw py::error_already_set();
  return v;
}
bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw py::error_already_set();
  return v != 0;
}
PyObject* tuple_of(std::initializer_list<optional<at::Tensor>> items) {
  PyObject* t = PyTuple_New((Py_ssize_t)items.size());
  if (t == nullptr) throw py::error_already_set();
  Py_ssize_t i = 0;
  for (const auto& item : items) PyTuple_SET_ITEM(t, i++, wrap(item));
  return t;
}

void check_device(const at::Tensor& t, const at::Tensor& first, const char* what) {
  TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor");
  TORCH_CHECK(t.get_device() == first.get_device(), what, " must be on the device of the other tensors (", first.device().str(),
              "), not on ", t.device().str());
}

// A matrix whose rows are contiguous; the distance between them is free (0: the same row again).
at::Tensor with_rows(const at::Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }
int64_t row_stride(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// A caller's tensor has been written: what autograd has saved of it before is no longer what it was.
void changed(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

at::Tensor new_cuda(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(shape, type, like.device(), c10::nullopt);
}

bool wants_gradient(const at::Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

// (a result without a tangent would count as one whose tangent is zero)
void check_no_tangent(const at::Tensor& t, const char* what) {
  TORCH_CHECK(!t._fw_grad(0).defined(), what, " has a forward-mode tangent, and this operator has no forward derivative");
}
void check_no_gradient(const at::Tensor& t, const char* what) {
  check_no_tangent(t, what);
  TORCH_CHECK(!wants_gradient(t), what,
              " requires a gradient, and this operator has none: call it under torch.no_grad()");
}

// ------------------------------------------------------------- rows with block scales ----

// Bytes from a tensor's first element to behind its last one.
int64_t reach(const at::Tensor& t) {
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return (last + 1) * (int64_t)t.element_size();
}
// Whether two tensors cannot share memory: one ends before the other begins, or both are columns of the same wider matrix (a
// vector, or a matrix of one row, lies in one row of it).
bool apart(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return true;
  const int64_t between = (int64_t)((intptr_t)b.const_data_ptr() - (intptr_t)a.const_data_ptr());
  if (between >= reach(a) || -between >= reach(b)) return true;
  const auto width = [](const at::Tensor& t) { return t.size(-1) > 1 && t.stride(-1) != 1 ? 0 : t.size(-1) * (int64_t)t.element_size(); };
  const auto step = [](const at::Tensor& t) { return t.dim() == 2 && t.size(0) > 1 ? t.stride(0) * (int64_t)t.element_size() : 0; };
  if (a.dim() < 1 || a.dim() > 2 || b.dim() < 1 || b.dim() > 2 || width(a) == 0 || width(b) == 0) return false;
  const int64_t rows = std::max(step(a), step(b));
  if (rows == 0 || (step(a) != rows && step(a) != 0) || (step(b) != rows && step(b) != 0)) return false;
  const int64_t within = (between % rows + rows) % rows;
  return within >= width(a) && within + width(b) <= rows;
}
void check_apart(const at::Tensor& a, const at::Tensor& b, const char* what) {
  TORCH_CHECK(apart(a, b), what, " overlap in memory");
}
// Two matrices of one shape and type, of which one is written while the other is read: the very same rows are fine (a lane
// reads its columns before it writes them).
void check_apart_or_same(const at::Tensor& a, const at::Tensor& b, const char* what) {
  const bool same = a.const_data_ptr() == b.const_data_ptr() && (a.size(0) <= 1 || a.stride(0) == b.stride(0)) &&
                    (a.size(1) <= 1 || a.stride(1) == b.stride(1));
  TORCH_CHECK(same || apart(a, b), what, " overlap in memory and are not the same");
}

// (x, weight, eps, residual or None, total_out or None, normed) -> (q, scale, total or None, normed or None)
PyObject* rms_norm_fp8(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count_args(n, 6);
    const at::Tensor& x_in = tensor_arg(v[0]);
    const at::Tensor& weight_in = tensor_arg(v[1]);
    const double eps = double_arg(v[2]);
    const optional<at::Tensor> residual_in = optional_arg(v[3]);
    optional<at::Tensor> total = optional_arg(v[4]);
    const bool want_normed = bool_arg(v[5]);
    TORCH_CHECK(x_in.dim() == 2, "x must be a matrix [rows, columns]");
    const int64_t rows = x_in.size(0), cols = x_in.size(1);
    const auto type = x_in.scalar_type();
    const int code = dtype_code(type);
    TORCH_CHECK(cols >= 1 && cols <= b200::kMaxNormCols, "x must have 1 to ", num(b200::kMaxNormCols), " columns, not ", num(cols));
    TORCH_CHECK(weight_in.dim() == 1 && weight_in.size(0) == cols, "weight must be a vector of ", num(cols), " values");
    TORCH_CHECK(weight_in.scalar_type() == type || weight_in.scalar_type() == at::kFloat, "weight must have x's type or be float32");
    TORCH_CHECK(std::isfinite(eps) && eps >= 0, "eps must not be negative");
    check_no_gradient(x_in, "x");
    check_no_gradient(weight_in, "weight");
    if (residual_in) {
      TORCH_CHECK(residual_in->sizes() == x_in.sizes() && residual_in->scalar_type() == type, "residual must have x's shape and type");
      check_no_gradient(*residual_in, "residual");
    }
    TORCH_CHECK(!total || residual_in, "total_out is the sum of x and residual: there is no residual");
    if (total) {
      TORCH_CHECK(total->sizes() == x_in.sizes() && total->scalar_type() == type, "total_out must have x's shape and type");
      TORCH_CHECK((cols == 1 || total->stride(1) == 1) && (rows <= 1 || total->stride(0) >= cols),
                  "total_out must have contiguous rows that do not overlap");
      check_no_gradient(*total, "total_out");
      check_apart_or_same(*total, x_in, "total_out and x");
      check_apart_or_same(*total, *residual_in, "total_out and residual");
      check_apart(*total, weight_in, "total_out and weight");
    }
    TORCH_CHECK(x_in.is_cuda(), "x must be a CUDA tensor");
    check_device(weight_in, x_in, "weight");
    if (residual_in) check_device(*residual_in, x_in, "residual");
    if (total) check_device(*total, x_in, "total_out");
    c10::cuda::CUDAGuard guard(x_in.device());
    if (total) changed(*total);
    const at::Tensor x = with_rows(x_in), weight = weight_in.contiguous();
    at::Tensor residual;
    if (residual_in) {
      residual = with_rows(*residual_in);
      if (!total) total = new_cuda({rows, cols}, type, x);
    }
    const at::Tensor q = new_cuda({rows, cols}, at::kFloat8_e4m3fn, x);
    const at::Tensor scale = new_cuda({rows, (cols + 127) / 128}, at::kFloat, x);
    optional<at::Tensor> normed;
    if (want_normed) normed = new_cuda({rows, cols}, type, x);
    b200::RmsNormFp8Args a = {};
    a.x = x.const_data_ptr();
    a.residual = residual_in ? residual.const_data_ptr() : nullptr;
    a.weight = weight.const_data_ptr();
    a.total = total ? total->mutable_data_ptr() : nullptr;
    a.normed = normed ? normed->mutable_data_ptr() : nullptr;
    a.q = q.mutable_data_ptr();
    a.scale = scale.mutable_data_ptr<float>();
    a.rows = rows;
    a.cols = (int32_t)cols;
    a.x_stride = row_stride(x);
    a.residual_stride = residual_in ? row_stride(residual) : 0;
    a.total_stride = total ? row_stride(*total) : 0;
    a.eps = (float)eps;
    a.dtype = code;
    a.weight_dtype = dtype_code(weight.scalar_type());
    cuda_check(b200::launch_rms_norm_fp8(a, device_sms(x.get_device()), at::cuda::getCurrentCUDAStream()), "rms_norm_fp8 launch");
    return tuple_of({q, scale, total, normed});
  });
}

PyObject* silu_mul_fp8(PyObject*, PyObject* const* v, Py_ssize_t n) {  // (x) -> (q, scale)
  return guarded([&] {
    count_args(n, 1);
    const at::Tensor& x_in = tensor_arg(v[0]);
    TORCH_CHECK(x_in.dim() == 2, "x must be a matrix [rows, 2 columns]");
    TORCH_CHECK(x_in.size(1) >= 2 && x_in.size(1) % 2 == 0 && x_in.size(1) / 2 <= b200::kMaxSiluCols,
                "x must have an even number of columns: gates, then the values that they multiply");
    const int64_t rows = x_in.size(0), cols = x_in.size(1) / 2;
    const int code = dtype_code(x_in.scalar_type());
    check_no_gradient(x_in, "x");
    TORCH_CHECK(x_in.is_cuda(), "x must be a CUDA tensor");
    c10::cuda::CUDAGuard guard(x_in.device());
    const at::Tensor x = with_rows(x_in);
    const at::Tensor q = new_cuda({rows, cols}, at::kFloat8_e4m3fn, x);
    const at::Tensor scale = new_cuda({rows, (cols + 127) / 128}, at::kFloat, x);
    b200::SiluMulFp8Args a = {};
    a.x = x.const_data_ptr();
    a.q = q.mutable_data_ptr();
    a.scale = scale.mutable_data_ptr<float>();
    a.rows = rows;
    a.cols = (int32_t)cols;
    a.x_stride = row_stride(x);
    a.dtype = code;
    cuda_check(b200::launch_silu_mul_fp8(a, device_sms(x.get_device()), at::cuda::getCurrentCUDAStream()), "silu_mul_fp8 launch");
    return tuple_of({q, scale});
  });
}

// -------------------------------------------------------------- tokens sorted by expert ----

constexpr int64_t kMaxEntries = int64_t(1) << 30;

int64_t check_entries(int64_t tokens, int64_t k) {
  TORCH_CHECK(k >= 1 && k <= b200::kSortMaxTopk, "a token must have 1 to ", num(b200::kSortMaxTopk), " experts, not ", num(k));
  TORCH_CHECK(tokens <= kMaxEntries / k, "more than 2^30 (token, expert) entries");
  return tokens * k;
}


// (x, indices, num_experts, scale or None) -> (rows, rows_scale or None, offsets, row_of); None where x wants a gradient
PyObject* sort_tokens(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count_args(n, 4);
    const at::Tensor& x_in = tensor_arg(v[0]);
    check_no_tangent(x_in, "x");
    if (wants_gradient(x_in)) Py_RETURN_NONE;
    const at::Tensor& indices_in = tensor_arg(v[1]);
    const int64_t experts = int_arg(v[2]);
    const optional<at::Tensor> scale_in = optional_arg(v[3]);
    TORCH_CHECK(x_in.dim() == 2 && x_in.size(1) >= 1, "x must be a matrix [tokens, hidden]");
    const auto type = x_in.scalar_type();
    if (type != at::kFloat8_e4m3fn) dtype_code(type);
    const int64_t tokens = x_in.size(0), hidden = x_in.size(1);
    TORCH_CHECK(hidden <= INT32_MAX / 8, "hidden is too large");
    TORCH_CHECK(indices_in.dim() == 2 && indices_in.size(0) == tokens, "indices must be [tokens, experts per token]");
    TORCH_CHECK(indices_in.scalar_type() == at::kInt || indices_in.scalar_type() == at::kLong, "indices must be int32 or int64");
    const int64_t k = indices_in.size(1);
    const int64_t entries = check_entries(tokens, k);
    TORCH_CHECK(experts >= 1 && experts <= b200::kSortMaxExperts, "num_experts must be 1 to ", num(b200::kSortMaxExperts), ", not ", num(experts));
    if (scale_in) {
      TORCH_CHECK(scale_in->dim() == 2 && scale_in->size(0) == tokens && scale_in->size(1) >= 1 &&
                      scale_in->size(1) <= INT32_MAX / 8 && scale_in->scalar_type() == at::kFloat,
                  "scale must be float32 [tokens, scales of a row]");
      check_no_gradient(*scale_in, "scale");
    }
    TORCH_CHECK(x_in.is_cuda(), "x must be a CUDA tensor");
    check_device(indices_in, x_in, "indices");
    if (scale_in) check_device(*scale_in, x_in, "scale");
    c10::cuda::CUDAGuard guard(x_in.device());
    const at::Tensor x = with_rows(x_in), indices = indices_in.contiguous();
    const at::Tensor rows = new_cuda({entries, hidden}, type, x);
    const at::Tensor offsets = new_cuda({experts + 1}, at::kInt, x), row_of = new_cuda({tokens, k}, at::kInt, x);
    at::Tensor scale, work;
    optional<at::Tensor> rows_scale;
    b200::SortTokensArgs a = {};
    if (scale_in) {
      scale = with_rows(*scale_in);
      rows_scale = new_cuda({entries, scale.size(1)}, at::kFloat, x);
      a.scale = scale.const_data_ptr<float>();
      a.rows_scale = rows_scale->mutable_data_ptr<float>();
      a.scale_stride = row_stride(scale);
      a.scale_cols = (int32_t)scale.size(1);
    }
    if (const int64_t words = b200::sort_tokens_work(tokens, (int)k, (int)experts)) {
      work = new_cuda({words}, at::kInt, x);
      a.work = work.mutable_data_ptr<int32_t>();
    }
    a.x = x.const_data_ptr();
    a.indices = indices.const_data_ptr();
    a.rows = rows.mutable_data_ptr();
    a.offsets = offsets.mutable_data_ptr<int32_t>();
    a.row_of = row_of.mutable_data_ptr<int32_t>();
    a.elem_bytes = (int32_t)x.element_size();
    a.x_stride = row_stride(x) * a.elem_bytes;
    a.row_bytes = hidden * a.elem_bytes;
    a.tokens = (int32_t)tokens;
    a.k = (int32_t)k;
    a.experts = (int32_t)experts;
    a.wide_ids = indices.scalar_type() == at::kLong;
    cuda_check(b200::launch_sort_tokens(a, device_sms(x.get_device()), at::cuda::getCurrentCUDAStream()), "sort_tokens launch");
    return tuple_of({rows, rows_scale, offsets, row_of});
  });
}

void check_order(const at::Tensor& row_of, const char* what) {
  TORCH_CHECK(row_of.dim() == 2 && row_of.scalar_type() == at::kInt, what, " must be int32 [tokens, experts per token]");
}

at::Tensor weights_of(const at::Tensor& w, const at::Tensor& row_of) {
  TORCH_CHECK(w.sizes() == row_of.sizes() && w.scalar_type() == at::kFloat, "weights must be float32 [tokens, experts per token]");
  return w;
}

// (rows, row_of, weights or None) -> out; None where something wants a gradient, or weights are of another type
PyObject* unsort_tokens(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count_args(n, 3);
    const at::Tensor& rows_in = tensor_arg(v[0]);
    const at::Tensor& row_of_in = tensor_arg(v[1]);
    const optional<at::Tensor> weights_in = optional_arg(v[2]);
    check_no_tangent(rows_in, "rows");
    if (weights_in) check_no_tangent(*weights_in, "weights");
    if (wants_gradient(rows_in) || (weights_in && (wants_gradient(*weights_in) || weights_in->scalar_type() != at::kFloat)))
      Py_RETURN_NONE;
    TORCH_CHECK(rows_in.dim() == 2 && rows_in.size(1) >= 1 && rows_in.size(1) <= INT32_MAX / 8, "rows must be a matrix [rows, hidden]");
    const int code = dtype_code(rows_in.scalar_type());
    check_order(row_of_in, "row_of");
    const int64_t tokens = row_of_in.size(0), k = row_of_in.size(1), hidden = rows_in.size(1);
    TORCH_CHECK(rows_in.size(0) == check_entries(tokens, k), "rows must have a row for each of the ", num(tokens * k), " entries, not ",
                num(rows_in.size(0)));
    if (weights_in) weights_of(*weights_in, row_of_in);
    TORCH_CHECK(rows_in.is_cuda(), "rows must be a CUDA tensor");
    check_device(row_of_in, rows_in, "row_of");
    if (weights_in) check_device(*weights_in, rows_in, "weights");
    c10::cuda::CUDAGuard guard(rows_in.device());
    const at::Tensor rows = with_rows(rows_in), row_of = row_of_in.contiguous();
    at::Tensor weights;
    if (weights_in) weights = weights_in->contiguous();
    at::Tensor out = new_cuda({tokens, hidden}, rows.scalar_type(), rows);
    b200::UnsortTokensArgs a = {};
    a.rows = rows.const_data_ptr();
    a.weights = weights_in ? weights.const_data_ptr<float>() : nullptr;
    a.row_of = row_of.const_data_ptr<int32_t>();
    a.out = out.mutable_data_ptr();
    a.rows_stride = row_stride(rows) * (int64_t)rows.element_size();
    a.num_rows = rows.size(0);
    a.tokens = (int32_t)tokens;
    a.k = (int32_t)k;
    a.hidden = (int32_t)hidden;
    a.dtype = code;
    cuda_check(b200::launch_unsort_tokens(a, device_sms(rows.get_device()), at::cuda::getCurrentCUDAStream()), "unsort_tokens launch");
    return wrap(out);
  });
}

// (grad, rows, offsets, row_of, weights or None, want_rows, want_weights) -> (grad_rows or None, grad_weights or None); rows
// may be None where the weights' gradient is not wanted
PyObject* unsort_tokens_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count_args(n, 7);
    const at::Tensor& grad_in = tensor_arg(v[0]);
    const optional<at::Tensor> rows_in = optional_arg(v[1]);
    const at::Tensor& offsets_in = tensor_arg(v[2]);
    const at::Tensor& row_of_in = tensor_arg(v[3]);
    const optional<at::Tensor> weights_in = optional_arg(v[4]);
    const bool want_rows = bool_arg(v[5]), want_weights = bool_arg(v[6]) && weights_in;
    const at::Tensor& like = rows_in ? *rows_in : grad_in;
    const auto type = like.scalar_type();
    const int code = dtype_code(type);
    check_order(row_of_in, "row_of");
    TORCH_CHECK(offsets_in.dim() == 1 && offsets_in.size(0) >= 2 && offsets_in.scalar_type() == at::kInt, "offsets must be int32 [num_experts + 1]");
    const int64_t tokens = row_of_in.size(0), k = row_of_in.size(1);
    const int64_t entries = check_entries(tokens, k);
    TORCH_CHECK(like.dim() == 2 && like.size(1) >= 1 && like.size(1) <= INT32_MAX / 8 && (!rows_in || rows_in->size(0) == entries),
                "rows must have a row for each of the ", num(entries), " entries");
    TORCH_CHECK(rows_in || !want_weights, "the weights' gradient needs the rows");
    const int64_t hidden = like.size(1);
    TORCH_CHECK(grad_in.dim() == 2 && grad_in.size(0) == tokens && grad_in.size(1) == hidden && grad_in.scalar_type() == type,
                "the gradient must be [tokens, hidden] of the rows' type");
    if (weights_in) weights_of(*weights_in, row_of_in);
    check_no_tangent(grad_in, "the gradient");
    if (rows_in) check_no_tangent(*rows_in, "rows");
    if (weights_in) check_no_tangent(*weights_in, "weights");
    TORCH_CHECK(like.is_cuda(), rows_in ? "rows" : "the gradient", " must be a CUDA tensor");
    check_device(grad_in, like, "the gradient");
    check_device(offsets_in, like, "offsets");
    check_device(row_of_in, like, "row_of");
    if (weights_in) check_device(*weights_in, like, "weights");
    c10::cuda::CUDAGuard guard(like.device());
    optional<at::Tensor> grad_rows, grad_weights;
    if (want_rows) grad_rows = new_cuda({entries, hidden}, type, like);
    if (want_weights) grad_weights = new_cuda({tokens, k}, at::kFloat, like);
    if (!want_rows && !want_weights) return tuple_of({grad_rows, grad_weights});
    const at::Tensor grad = with_rows(grad_in), offsets = offsets_in.contiguous(), row_of = row_of_in.contiguous();
    at::Tensor rows, weights;
    if (want_weights) rows = with_rows(*rows_in);
    if (weights_in) weights = weights_in->contiguous();
    b200::UnsortBackwardArgs a = {};
    a.grad = grad.const_data_ptr();
    a.rows = want_weights ? rows.const_data_ptr() : nullptr;
    a.weights = weights_in ? weights.const_data_ptr<float>() : nullptr;
    a.row_of = row_of.const_data_ptr<int32_t>();
    a.end = offsets.const_data_ptr<int32_t>() + offsets.size(0) - 1;
    a.grad_rows = want_rows ? grad_rows->mutable_data_ptr() : nullptr;
    a.grad_weights = want_weights ? grad_weights->mutable_data_ptr<float>() : nullptr;
    a.grad_stride = row_stride(grad) * (int64_t)grad.element_size();
    a.rows_stride = want_weights ? row_stride(rows) * (int64_t)rows.element_size() : 0;
    a.num_rows = entries;
    a.tokens = (int32_t)tokens;
    a.k = (int32_t)k;
    a.hidden = (int32_t)hidden;
    a.dtype = code;
    cuda_check(b200::launch_unsort_tokens_backward(a, device_sms(like.get_device()), at::cuda::getCurrentCUDAStream()),
               "unsort_tokens_backward launch");
    return tuple_of({grad_rows, grad_weights});
  });
}

// ------------------------------------------------------------- the experts' products ----

// Row-major, and at an address that a tensor map takes.
at::Tensor for_copies(const at::Tensor& t) {
  const at::Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.const_data_ptr()) & 15u) == 0 ? c : c.clone();
}

// (a, b, a_scale, b_scale, offsets, c or None, timeout_ns) -> c; None where an earlier call on the device has recorded a
// failure, which the caller takes and raises (nothing is launched then).
PyObject* fp8_grouped_gemm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count_args(n, 7);
    const at::Tensor& a_in = tensor_arg(v[0]);
    const at::Tensor& b_in = tensor_arg(v[1]);
    const at::Tensor& a_scale = tensor_arg(v[2]);
    const at::Tensor& b_scale = tensor_arg(v[3]);
    const at::Tensor& offsets_in = tensor_arg(v[4]);
    optional<at::Tensor> c = optional_arg(v[5]);
    const int64_t timeout_ns = int_arg(v[6]);
    TORCH_CHECK(a_in.dim() == 2 && b_in.dim() == 3 && a_in.size(1) == b_in.size(2), "a [M, K] and b [E, N, K] must have equal K");
    TORCH_CHECK(a_in.scalar_type() == at::kFloat8_e4m3fn && b_in.scalar_type() == at::kFloat8_e4m3fn, "a and b must be float8_e4m3fn");
    const int64_t M = a_in.size(0), E = b_in.size(0), N = b_in.size(1), K = a_in.size(1);
    const int64_t kb = (K + 127) / 128, nb = (N + 127) / 128;
    TORCH_CHECK(E >= 1 && E <= b200::kGroupedMaxExperts, "b must have 1 to ", num(b200::kGroupedMaxExperts), " experts, not ", num(E));
    TORCH_CHECK(K >= 16 && K % 16 == 0, "K must be a multiple of 16");
    TORCH_CHECK(N >= 1, "N must not be 0");
    TORCH_CHECK(M <= INT32_MAX / 2 && E * N <= INT32_MAX / 2 && K <= INT32_MAX / 2, "the problem is too large");
    TORCH_CHECK(a_scale.scalar_type() == at::kFloat && a_scale.dim() == 2 && a_scale.size(0) == M && a_scale.size(1) == kb,
                "a_scale must be fp32 [M, ceil(K/128)]");
    TORCH_CHECK(b_scale.scalar_type() == at::kFloat && b_scale.dim() == 3 && b_scale.size(0) == E && b_scale.size(1) == nb &&
                    b_scale.size(2) == kb,
                "b_scale must be fp32 [E, ceil(N/128), ceil(K/128)]");
    TORCH_CHECK(offsets_in.scalar_type() == at::kInt && offsets_in.dim() == 1 && offsets_in.size(0) == E + 1, "offsets must be int32 [E + 1]");
    if (c)
      TORCH_CHECK(c->scalar_type() == at::kBFloat16 && c->dim() == 2 && c->size(0) == M && c->size(1) == N && c->is_contiguous(),
                  "c must be bf16 [M, N], row-major");
    TORCH_CHECK(timeout_ns > 0, "timeout_ms must be positive");
    check_no_gradient(a_in, "a");
    check_no_gradient(b_in, "b");
    check_no_gradient(a_scale, "a_scale");
    check_no_gradient(b_scale, "b_scale");
    if (c) {
      check_no_gradient(*c, "c");
      check_apart(*c, a_in, "c and a");
      check_apart(*c, b_in, "c and b");
      check_apart(*c, a_scale, "c and a_scale");
      check_apart(*c, b_scale, "c and b_scale");
      check_apart(*c, offsets_in, "c and offsets");
    }
    TORCH_CHECK(a_in.is_cuda(), "a must be a CUDA tensor");
    check_device(b_in, a_in, "b");
    check_device(a_scale, a_in, "a_scale");
    check_device(b_scale, a_in, "b_scale");
    check_device(offsets_in, a_in, "offsets");
    if (c) check_device(*c, a_in, "c");
    c10::cuda::CUDAGuard guard(a_in.device());
    if (fp8_status_code(a_in.get_device()) != 0) Py_RETURN_NONE;
    const bool zero_rest = !c;
    if (c) changed(*c);
    else c = new_cuda({M, N}, at::kBFloat16, a_in);
    if (M == 0) return wrap(c);
    const at::Tensor a = for_copies(a_in), b = for_copies(b_in), offsets = offsets_in.contiguous();
    b200::Fp8GroupedArgs g = {};
    g.a = a.const_data_ptr();
    g.b = b.const_data_ptr();
    g.a_scale = a_scale.const_data_ptr<float>();
    g.b_scale = b_scale.const_data_ptr<float>();
    g.offsets = offsets.const_data_ptr<int32_t>();
    g.c = c->mutable_data_ptr();
    g.M = (int)M;
    g.N = (int)N;
    g.K = (int)K;
    g.experts = (int)E;
    g.as_stride_m = a_scale.stride(0);
    g.as_stride_k = a_scale.stride(1);
    g.bs_stride_e = b_scale.stride(0);
    g.bs_stride_n = b_scale.stride(1);
    g.bs_stride_k = b_scale.stride(2);
    g.zero_rest = zero_rest;
    g.timeout_ns = (uint64_t)timeout_ns;
    g.status = fp8_status(a.get_device());
    g.sms = device_sms(a.get_device());
    cuda_check(b200::launch_fp8_grouped_gemm(g, at::cuda::getCurrentCUDAStream()), "fp8_grouped_gemm launch");
    return wrap(c);
  });
}

// While the current stream is being captured: whether a leaf behind `t` has its gradient added up on another stream, as it
// does when an eager graph of it is alive.  The captured backward pass would have to wait for that stream, which ends
// the process from inside the autograd engine.
bool adds_up_elsewhere(const at::Tensor& t) {
  if (!t.requires_grad()) return false;
  const c10::Stream here = at::cuda::getCurrentCUDAStream(t.get_device()).unwrap();
  std::vector<std::shared_ptr<torch::autograd::Node>> todo;
  std::unordered_set<torch::autograd::Node*> seen;
  const auto visit = [&](std::shared_ptr<torch::autograd::Node> node) {
    if (node && seen.insert(node.get()).second) todo.push_back(std::move(node));
  };
  if (t.grad_fn()) visit(t.grad_fn());
  else visit(torch::autograd::impl::try_get_grad_accumulator(t));
  while (!todo.empty()) {
    const auto node = todo.back();
    todo.pop_back();
    if (node->num_outputs() == 0) {  // a leaf's
      const auto stream = node->stream();
      if (stream && *stream != here) return true;
    }
    for (const auto& edge : node->next_edges()) visit(edge.function);
  }
  return false;
}

#define B200_CALL(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef kExpertCalls[] = {B200_CALL(rms_norm_fp8), B200_CALL(silu_mul_fp8), B200_CALL(sort_tokens), B200_CALL(unsort_tokens),
                              B200_CALL(unsort_tokens_backward), B200_CALL(fp8_grouped_gemm), {nullptr, nullptr, 0, nullptr}};
#undef B200_CALL

}  // namespace

void b200::bind_experts(py::module& m) {
  if (PyModule_AddFunctions(m.ptr(), kExpertCalls) != 0) throw py::error_already_set();
  m.def("adds_up_elsewhere", &adds_up_elsewhere);
  m.def("fp8_grouped_tile", &b200::fp8_grouped_tile);
  m.def("fp8_grouped_local_bytes", &b200::fp8_grouped_local_bytes);
  m.def("fp8_grouped_share", [](int tile, int experts) { return py::make_tuple(b200::fp8_grouped_smem(tile, experts), 512); });
}
