// The training operators' calls from Python: argument checks, outputs and scratch from torch's caching allocator, and the call of the
// C ABI, in one step.  A training step makes these calls for rows of any number, and for few rows they are what it costs: checked and
// allocated from Python a LayerNorm forward took 12.9 us of host time, 3 of them its launch.
//
// The library is not linked: its functions' addresses are handed over by the module that has loaded it (bind), so that both use the
// same copy of it.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <map>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/b200pair.h"

namespace py = pybind11;
using at::ScalarType;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using OptType = std::optional<ScalarType>;

namespace {

// kMaxCols: of a LayerNorm row; kMaxKept: of a checkpoint's, kMaxWidth: of a linear layer, as the library counts them
constexpr int64_t kGroup = 32, kMaxCols = 8192, kMaxKept = (int64_t(1) << 31) - 1, kMaxWidth = 1 << 24;

#define B200_BOUND(f) decltype(&b200_##f) f##_
struct {
  B200_BOUND(layer_norm_save_fwd);
  B200_BOUND(layer_norm_bwd_workspace_bytes);
  B200_BOUND(layer_norm_bwd);
  B200_BOUND(checkpoint8_fwd);
  B200_BOUND(checkpoint8_restore);
  B200_BOUND(linear_act_fwd);
  B200_BOUND(linear_act_bwd_workspace_bytes);
  B200_BOUND(linear_act_bwd);
} lib;
PyObject* g_check = nullptr;  // raises what a status code stands for

void bind(const std::map<std::string, uintptr_t>& at, py::object check) {
#define B200_BIND(f) lib.f##_ = reinterpret_cast<decltype(lib.f##_)>(at.at("b200_" #f))
  B200_BIND(layer_norm_save_fwd);
  B200_BIND(layer_norm_bwd_workspace_bytes);
  B200_BIND(layer_norm_bwd);
  B200_BIND(checkpoint8_fwd);
  B200_BIND(checkpoint8_restore);
  B200_BIND(linear_act_fwd);
  B200_BIND(linear_act_bwd_workspace_bytes);
  B200_BIND(linear_act_bwd);
  g_check = check.release().ptr();
}

void check(int status) {
  if (status == B200_OK) return;
  const py::handle raise(g_check);
  raise(status);
}

// ---------------------------------------------------------------------------
// Arguments
// ---------------------------------------------------------------------------
template <class... Args>
[[noreturn]] void refuse(const Args&... args) {
  throw py::value_error(c10::str(args...));
}
std::string kind(const Tensor& t) { return c10::str(t.scalar_type(), " ", t.sizes()); }

int code(ScalarType t, const char* what) {
  if (t == at::kFloat) return B200_DTYPE_F32;
  if (t == at::kBFloat16) return B200_DTYPE_BF16;
  if (t == at::kHalf) return B200_DTYPE_F16;
  refuse(what, " must be float32, bfloat16 or float16, got ", t);
}

// A wrapper around other tensors (DTensor) has a shape and a device but no memory, nor has a parameter whose storage was given back:
// its null pointer would read as an argument that was not given.
void in_memory(const Tensor& t) {
  if (t.is_meta() || t.numel() == 0 || (t.has_storage() && t.storage().data())) return;
  refuse("a tensor of shape ", t.sizes(), " has no memory of its own: wrappers such as DTensor are not taken, their local tensors are");
}

// Called when everything else about the arguments is right.
void on_one_device(const Tensor& first, std::initializer_list<const Tensor*> others) {
  in_memory(first);
  for (const Tensor* t : others)
    if (t) in_memory(*t);
  auto cuda = [](const Tensor& t) {
    if (!t.is_cuda()) throw std::runtime_error("bioemu2_b200 runs on CUDA tensors only (there is no CPU path)");
  };
  cuda(first);
  for (const Tensor* t : others)
    if (t) {
      cuda(*t);
      if (t->device() != first.device()) refuse("tensors on ", first.device(), " and ", t->device());
    }
}
bool has_tangent(const OptTensor& a, const OptTensor& b, const OptTensor& c, const OptTensor& d) {
  for (const OptTensor* t : {&a, &b, &c, &d})
    if (*t && (*t)->_fw_grad(0).defined()) return true;
  return false;
}

const Tensor* given(const OptTensor& t) { return t ? &*t : nullptr; }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
void* pointer(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

int64_t last(const Tensor& t) { return t.dim() ? t.size(-1) : 0; }
at::IntArrayRef leading(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }
std::vector<int64_t> with_last(at::IntArrayRef lead, int64_t n) {
  std::vector<int64_t> s(lead.begin(), lead.end());
  s.push_back(n);
  return s;
}
Tensor fresh(at::IntArrayRef sizes, ScalarType t, const Tensor& like) { return at::empty(sizes, like.options().dtype(t).requires_grad(false)); }

// A tensor as rows of `cols` neighbours, `pitch` elements apart: its own memory where its leading axes lie evenly spaced (a slice
// of wider rows), a copy otherwise.  step > 1: rows start on 16 bytes and lie a multiple of `step` elements apart.
struct Rows {
  Tensor t;
  int64_t pitch;
  void* ptr() const { return t.data_ptr(); }
};
Rows rows_of(const Tensor& t, int64_t cols, int64_t step = 1) {
  if (t.is_neg()) return {t.detach().resolve_neg().contiguous(), cols};  // a view whose memory has the other sign
  const bool starts = step == 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  if (starts && t.is_contiguous()) return {t, cols};
  if (starts && (t.size(-1) == 1 || t.stride(-1) == 1)) {
    // the axes before the last as one axis of evenly spaced rows, those of length one aside
    int64_t pitch = -1, covered = 0;
    bool even = true;
    for (int64_t d = t.dim() - 2; d >= 0 && even; --d) {
      if (t.size(d) == 1) continue;
      if (pitch < 0) pitch = t.stride(d), covered = t.stride(d) * t.size(d);
      else if (t.stride(d) == covered) covered *= t.size(d);
      else even = false;
    }
    if (pitch < 0) pitch = cols;
    if (even && pitch >= cols && pitch % step == 0) return {t, pitch};
  }
  return {t.detach().clone(at::MemoryFormat::Contiguous), cols};
}

// A parameter of `cols` values as contiguous fp32.
OptTensor parameter(const OptTensor& t, int64_t cols, const char* what) {
  if (!t) return t;
  if (t->dim() != 1 || t->size(0) != cols) refuse(what, " has shape ", t->sizes(), ", expected [", cols, "]");
  code(t->scalar_type(), what);
  return t;
}
// Contiguous, of the sign that its memory has.
Tensor plain(const Tensor& t) { return t.is_contiguous() && !t.is_neg() ? t : t.detach().resolve_neg().contiguous(); }
OptTensor as_fp32(const OptTensor& t) {
  if (!t || (t->scalar_type() == at::kFloat && t->is_contiguous() && !t->is_neg())) return t;
  return t->detach().resolve_neg().to(at::kFloat).contiguous();
}

// ---------------------------------------------------------------------------
// Checkpoints
// ---------------------------------------------------------------------------
std::tuple<Tensor, Tensor> empty_checkpoint(const Tensor& x) {
  return {fresh(x.sizes(), at::kFloat8_e4m3fn, x), fresh(with_last(leading(x), (last(x) + kGroup - 1) / kGroup), at::kByte, x)};
}

void kept_cols(const Tensor& t, const char* what) {
  if (last(t) < 1 || last(t) > kMaxKept) refuse(what, " has shape ", t.sizes(), ": rows of at least one column and at most ", kMaxKept, " are wanted");
}
void check_kept(const Tensor& values, const Tensor& exponents) {
  if (values.scalar_type() != at::kFloat8_e4m3fn || exponents.scalar_type() != at::kByte)
    refuse("a checkpoint is float8_e4m3fn with uint8 exponents, got ", values.scalar_type(), " with ", exponents.scalar_type());
  kept_cols(values, "a checkpoint");
  if (exponents.sizes() != at::IntArrayRef(with_last(leading(values), (last(values) + kGroup - 1) / kGroup)))
    refuse("exponents have shape ", exponents.sizes(), ", expected one for each ", kGroup, " of ", values.sizes());
}
Tensor dense(const Tensor& t) {  // contiguous, on 16 bytes
  return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.detach().clone(at::MemoryFormat::Contiguous);
}

std::tuple<Tensor, Tensor> checkpoint8(const Tensor& x) {
  const int type = code(x.scalar_type(), "x");
  const int64_t cols = last(x);
  kept_cols(x, "x");
  on_one_device(x, {});
  const c10::cuda::CUDAGuard guard(x.device());
  auto kept = empty_checkpoint(x);
  if (x.numel()) {
    const Rows r = rows_of(x, cols);
    check(lib.checkpoint8_fwd_(r.ptr(), r.pitch, std::get<0>(kept).data_ptr(), std::get<1>(kept).data_ptr<uint8_t>(), x.numel() / cols,
                               int(cols), type, stream_of(x)));
  }
  return kept;
}

Tensor restore8(const Tensor& values, const Tensor& exponents, ScalarType dtype) {
  check_kept(values, exponents);
  const int type = code(dtype, "restored activation");
  on_one_device(values, {&exponents});
  const c10::cuda::CUDAGuard guard(values.device());
  Tensor out = fresh(values.sizes(), dtype, values);
  if (out.numel()) {
    const Tensor v = dense(values), e = exponents.contiguous();
    check(lib.checkpoint8_restore_(v.data_ptr(), e.data_ptr<uint8_t>(), out.data_ptr(), v.numel() / last(v), int(last(v)), type, stream_of(v)));
  }
  return out;
}

// ---------------------------------------------------------------------------
// LayerNorm
// ---------------------------------------------------------------------------
int64_t norm_cols(const Tensor& x, ScalarType x_type, ScalarType y_type) {
  const int64_t cols = last(x);
  if (cols < 1 || cols > kMaxCols) refuse("layer norm takes rows of 1 to ", kMaxCols, " columns, got shape ", x.sizes());
  code(x_type, "x");
  code(y_type, "y");
  if (y_type != x_type && x_type != at::kFloat)
    refuse("an output of another type than x wants x in float32, got ", x_type, " and ", y_type);
  return cols;
}

std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor> layer_norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                                                            double eps, OptType out_type, bool keep) {
  const ScalarType y_type = out_type.value_or(x.scalar_type());
  const int64_t cols = norm_cols(x, x.scalar_type(), y_type);
  parameter(weight, cols, "weight");
  parameter(bias, cols, "bias");
  on_one_device(x, {given(weight), given(bias)});
  const c10::cuda::CUDAGuard guard(x.device());
  const OptTensor w = as_fp32(weight), b = as_fp32(bias);
  Tensor y = fresh(x.sizes(), y_type, x), mean = fresh(leading(x), at::kFloat, x), rstd = fresh(leading(x), at::kFloat, x);
  OptTensor values, exponents;
  if (keep) std::tie(values, exponents) = empty_checkpoint(x);
  if (x.numel()) {
    const Rows r = rows_of(x, cols);
    check(lib.layer_norm_save_fwd_(r.ptr(), r.pitch, static_cast<float*>(pointer(w)), static_cast<float*>(pointer(b)), y.data_ptr(),
                                   mean.data_ptr<float>(), rstd.data_ptr<float>(), pointer(values),
                                   static_cast<uint8_t*>(pointer(exponents)), x.numel() / cols, int(cols), float(eps),
                                   code(x.scalar_type(), "x"), code(y_type, "y"), stream_of(x)));
  }
  return {y, mean, rstd, values, exponents};
}

// x is the saved tensor, or with `exponents` the values of its checkpoint, of type x_type before it was kept.
std::tuple<OptTensor, OptTensor, OptTensor> layer_norm_backward(const Tensor& dy, const Tensor& x, const OptTensor& exponents, OptType kept_type,
                                                                const Tensor& mean, const Tensor& rstd, const OptTensor& weight,
                                                                std::optional<std::tuple<bool, bool, bool>> wanted, OptType grad_type) {
  const ScalarType x_type = exponents ? kept_type.value() : x.scalar_type();
  if (exponents) check_kept(x, *exponents);
  const int64_t cols = norm_cols(x, x_type, dy.scalar_type());
  if (dy.sizes() != x.sizes()) refuse("dy has shape ", dy.sizes(), ", x ", x.sizes());
  if (mean.scalar_type() != at::kFloat || rstd.scalar_type() != at::kFloat || mean.sizes() != leading(x) || rstd.sizes() != leading(x))
    refuse("mean and rstd must be float32 of shape ", leading(x), ", got ", kind(mean), " and ", kind(rstd));
  parameter(weight, cols, "weight");
  const auto needs = wanted.value_or(std::make_tuple(true, weight.has_value(), weight.has_value()));
  const ScalarType g_type = grad_type.value_or(weight ? weight->scalar_type() : at::kFloat);
  const int g_code = code(g_type, "the parameters' gradient");
  on_one_device(dy, {&x, given(exponents), &mean, &rstd, given(weight)});
  const c10::cuda::CUDAGuard guard(dy.device());
  OptTensor dx, dw, db;
  if (std::get<0>(needs)) dx = fresh(dy.sizes(), x_type, dy);
  if (std::get<1>(needs)) dw = fresh({cols}, g_type, dy);
  if (std::get<2>(needs)) db = fresh({cols}, g_type, dy);
  if (!dx && !dw && !db) return {dx, dw, db};
  const OptTensor w = as_fp32(weight);
  const Rows d = rows_of(dy, cols);
  const Rows s = exponents ? Rows{dense(x), cols} : rows_of(x, cols);
  const Tensor e = exponents ? exponents->contiguous() : Tensor();
  const Tensor m = plain(mean), r = plain(rstd);
  const int64_t rows = dy.numel() / cols;
  const size_t size = dw || db ? lib.layer_norm_bwd_workspace_bytes_(rows, int(cols)) : 0;
  const Tensor scratch = size ? fresh({int64_t(size)}, at::kByte, dy) : Tensor();
  check(lib.layer_norm_bwd_(d.ptr(), d.pitch, exponents ? nullptr : s.ptr(), s.pitch, exponents ? s.ptr() : nullptr,
                            exponents ? e.data_ptr<uint8_t>() : nullptr, m.data_ptr<float>(), r.data_ptr<float>(),
                            static_cast<float*>(pointer(w)), pointer(dx), pointer(dw), pointer(db), rows, int(cols), code(x_type, "x"),
                            code(dy.scalar_type(), "dy"), g_code, size ? scratch.data_ptr() : nullptr, size, stream_of(dy)));
  return {dx, dw, db};
}

// ---------------------------------------------------------------------------
// Linear layer
// ---------------------------------------------------------------------------
struct LinearSizes {
  int64_t k, n;
};
LinearSizes linear_sizes(int64_t width, ScalarType x_type, const Tensor& weight) {
  if ((x_type != at::kBFloat16 && x_type != at::kHalf) || weight.scalar_type() != x_type)
    refuse("x and weight must both be bfloat16 or both float16, got ", x_type, " and ", weight.scalar_type());
  if (weight.dim() != 2 || width != weight.size(1)) refuse("weight ", weight.sizes(), " does not match x of ", width, " columns");
  const int64_t n = weight.size(0), k = weight.size(1);
  if (k % 8 || n % 8 || k < 1 || n < 1 || k > kMaxWidth || n > kMaxWidth)
    refuse("in_features=", k, " and out_features=", n, " must be positive multiples of 8, at most ", kMaxWidth);
  return {k, n};
}

std::tuple<Tensor, OptTensor> linear_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias, int act, const OptTensor& residual,
                                             OptType out_type, OptType save_type) {
  const ScalarType type = x.scalar_type();
  const auto [k, n] = linear_sizes(last(x), type, weight);
  const std::vector<int64_t> shape = with_last(leading(x), n);
  const ScalarType y_type = out_type.value_or(residual ? residual->scalar_type() : type);
  if (y_type != type && y_type != at::kFloat) refuse("y is ", type, " like x or float32, got ", y_type);
  if (residual && (residual->sizes() != at::IntArrayRef(shape) || residual->scalar_type() != y_type))
    refuse("residual is ", kind(*residual), ", y ", y_type, " ", at::IntArrayRef(shape));
  if (save_type && *save_type != type && *save_type != at::kFloat)
    refuse("the value before the activation is saved as ", type, " like x or float32, not as ", *save_type);
  parameter(bias, n, "bias");
  on_one_device(x, {&weight, given(bias), given(residual)});
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = fresh(shape, y_type, x);
  OptTensor a;
  if (save_type && act) a = fresh(shape, *save_type, x);
  if (y.numel()) {
    const OptTensor b = as_fp32(bias);
    const Rows xr = rows_of(x, k, 8), wr = rows_of(weight, k, 8);
    const Rows rr = residual ? rows_of(*residual, n, 8) : Rows{Tensor(), n};
    check(lib.linear_act_fwd_(xr.ptr(), xr.pitch, wr.ptr(), wr.pitch, static_cast<float*>(pointer(b)), act, residual ? rr.ptr() : nullptr,
                              rr.pitch, y.data_ptr(), pointer(a), x.numel() / k, int(k), int(n), code(type, "x"), code(y_type, "y"),
                              code(save_type.value_or(type), "the saved value"), stream_of(x)));
  }
  return {y, a};
}

// x as in layer_norm_backward; it may be missing where dw is not wanted.
std::tuple<OptTensor, OptTensor, OptTensor> linear_backward(const Tensor& dy, const OptTensor& x, const OptTensor& exponents, OptType kept_type,
                                                            const Tensor& weight, const OptTensor& pre, int act, bool want_dx, bool want_dw,
                                                            OptType bias_type) {
  if (!x && want_dw) refuse("the weight's gradient wants x");
  if (exponents) check_kept(*x, *exponents);
  const ScalarType type = !x ? weight.scalar_type() : exponents ? kept_type.value() : x->scalar_type();
  const auto [k, n] = linear_sizes(x ? last(*x) : last(weight), type, weight);
  if (dy.dim() < 1) refuse("dy has no columns");
  const at::IntArrayRef lead = x ? leading(*x) : leading(dy);
  const std::vector<int64_t> shape = with_last(lead, n);
  if (dy.sizes() != at::IntArrayRef(shape) || (dy.scalar_type() != type && dy.scalar_type() != at::kFloat))
    refuse("dy must be ", type, " or float32 of shape ", at::IntArrayRef(shape), ", got ", kind(dy));
  if (act && (!pre || pre->sizes() != at::IntArrayRef(shape) || (pre->scalar_type() != type && pre->scalar_type() != at::kFloat)))
    refuse("pre must be ", type, " or float32 of shape ", at::IntArrayRef(shape), ", got ", pre ? kind(*pre) : "None");
  b200_linear_grad g = {};
  if (bias_type) g.db_dtype = code(*bias_type, "the bias's gradient");
  on_one_device(dy, {given(x), given(exponents), &weight, given(pre)});
  const c10::cuda::CUDAGuard guard(dy.device());
  OptTensor dx, dw, db;
  if (want_dx) dx = fresh(with_last(lead, k), type, dy);
  if (want_dw) dw = fresh({n, k}, type, dy);
  if (bias_type) db = fresh({n}, *bias_type, dy);
  if (!dx && !dw && !db) return {dx, dw, db};
  const Rows d = rows_of(dy, n, 8), wr = rows_of(weight, k, 8);
  g.dy = d.ptr(), g.dy_pitch = d.pitch, g.w = wr.ptr(), g.w_pitch = wr.pitch;
  Rows xr{Tensor(), k}, pr{Tensor(), n};
  Tensor e;
  if (exponents) {
    xr.t = dense(*x), e = exponents->contiguous();
    g.values = xr.ptr(), g.exponents = e.data_ptr<uint8_t>();
  } else if (x) {
    xr = rows_of(*x, k, 8);
    g.x = xr.ptr();
  }
  g.x_pitch = xr.pitch;
  if (act) {
    pr = rows_of(*pre, n, 8);
    g.pre = pr.ptr(), g.pre_dtype = code(pre->scalar_type(), "pre");
  }
  g.pre_pitch = pr.pitch;
  g.dx = pointer(dx), g.dw = pointer(dw), g.db = pointer(db);
  g.rows = dy.numel() / n, g.k = int(k), g.n = int(n), g.act = act, g.dtype = code(type, "x"), g.dy_dtype = code(dy.scalar_type(), "dy");
  const size_t size = lib.linear_act_bwd_workspace_bytes_(&g);
  const Tensor scratch = size ? fresh({int64_t(size)}, at::kByte, dy) : Tensor();
  check(lib.linear_act_bwd_(&g, size ? scratch.data_ptr() : nullptr, size, stream_of(dy)));
  return {dx, dw, db};
}

}  // namespace

PYBIND11_MODULE(_training, m) {
  m.doc() = "Calls of the training operators: see bioemu2_b200.training.";
  m.def("bind", &bind);
  m.def("has_tangent", &has_tangent);
  m.def("checkpoint8", &checkpoint8);
  m.def("restore8", &restore8);
  m.def("layer_norm_forward", &layer_norm_forward);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("linear_forward", &linear_forward);
  m.def("linear_backward", &linear_backward);
}
