// efficient_ops of linear layers in 8-bit floating point: quantised activations and
// weights, the norm that quantises, products of the two.  New ops with no counterpart
// in the reference; shapes and types are checked by the kernel library
// (include/mi355x_ops.h), devices and leading dims here.
#include <ATen/ATen.h>

#include "dispatch_util.h"
#include "efficient_ops.h"

namespace torch_gcu {
namespace efficient {

namespace {

void check_fp8(const char* op, std::initializer_list<std::pair<const char*, const at::Tensor*>> ts) {
  std::optional<at::Device> common;
  for (const auto& [name, t] : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(is_gcu(*t), op, ": ", name, " must be a gcu tensor");
    check_device(common, *t, op, name);
  }
}

const at::Tensor& or_undefined(const std::optional<at::Tensor>& t) {
  static const at::Tensor none;
  return t.has_value() ? *t : none;
}

mi_tensor_t desc2(const at::Tensor& t, int64_t rows, int64_t cols, int64_t ld) {
  mi_tensor_t d{};
  d.data = rows > 0 && cols > 0 ? t.data_ptr() : nullptr;
  d.dtype = (int32_t)t.scalar_type();
  d.ndim = 2;
  d.sizes[0] = rows;
  d.sizes[1] = cols;
  d.strides[0] = ld;
  d.strides[1] = 1;
  return d;
}

// [..., columns] as rows of one stride with dense columns: the tensor itself where
// its leading dims allow that, else a dense copy (kept alive here)
struct Rows {
  at::Tensor t;
  mi_tensor_t d;
  Rows(const char* op, const char* name, const at::Tensor& x) : t(x) {
    TORCH_CHECK(x.dim() >= 1, op, ": ", name, " must have at least one dim");
    int64_t rows = 1, ld = x.size(-1);
    bool uniform = x.size(-1) <= 1 || x.stride(-1) == 1;
    for (int64_t i = x.dim() - 2, outer = -1; i >= 0; --i) {
      if (x.size(i) != 1) {
        if (outer < 0) ld = x.stride(i);
        else uniform = uniform && x.stride(i) == outer;
        outer = x.stride(i) * x.size(i);
      }
      rows *= x.size(i);
    }
    if (!uniform && x.numel() > 0) {
      t = x.clone(at::MemoryFormat::Contiguous);
      ld = x.size(-1);
    }
    d = desc2(t, rows, x.size(-1), ld);
  }
};

// New codes and scales of activations with these leading dims: rows of codes begin at
// multiples of 16 bytes, which the products read as they are.
struct NewRows {
  at::Tensor codes, scales;
  mi_fp8_t d;
  NewRows(const at::Tensor& like, at::IntArrayRef sizes) {
    const auto opt = like.options().dtype(at::kByte);
    const int64_t cols = sizes.back(), pitch = (cols + 15) / 16 * 16, groups = (cols + 127) / 128;
    c10::SmallVector<int64_t, 6> shape(sizes.begin(), sizes.end()), strides(sizes.size(), 1);
    int64_t rows = 1;
    for (int64_t i = (int64_t)sizes.size() - 2; i >= 0; --i) {
      strides[i] = pitch * rows;
      rows *= sizes[i];
    }
    codes = pitch == cols ? at::empty(shape, opt) : at::empty_strided(shape, strides, opt);
    shape.back() = groups;
    scales = at::empty(shape, opt);
    d = {desc2(codes, rows, cols, pitch), desc2(scales, rows, groups, groups)};
  }
};

// Activations that a product reads.
struct ReadRows {
  Rows codes, scales;
  mi_fp8_t d;
  ReadRows(const char* op, const at::Tensor& c, const at::Tensor& s)
      : codes(op, "codes of x", c), scales(op, "scales of x", s), d{codes.d, scales.d} {
    TORCH_CHECK(c.dim() == s.dim() && c.sizes().slice(0, c.dim() - 1) == s.sizes().slice(0, s.dim() - 1),
                op, ": codes of x are ", c.sizes(), ", scales ", s.sizes());
  }
};

std::vector<int64_t> with_columns(const at::Tensor& x, int64_t n) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n;
  return shape;
}

void check_weight(const char* op, const char* name, const at::Tensor& codes, const at::Tensor& scales) {
  TORCH_CHECK(codes.dim() == 2 && scales.dim() == 2, op, ": codes and scales of ", name, " must be 2-D");
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> fp8_quantize(const at::Tensor& x) {
  check_fp8("fp8_quantize", {{"x", &x}});
  const c10::DeviceGuard g(x.device());
  const Rows r("fp8_quantize", "x", x);
  NewRows out(x, x.sizes());
  check_mi(mi_fp8_quantize(&out.d, &r.d, mi_stream(x)), "fp8_quantize");
  after_op();
  return {out.codes, out.scales};
}

std::tuple<at::Tensor, at::Tensor> fp8_quantize_weight(const at::Tensor& weight) {
  check_fp8("fp8_quantize_weight", {{"weight", &weight}});
  TORCH_CHECK(weight.dim() == 2, "fp8_quantize_weight: weight must be 2-D [N, K]");
  const c10::DeviceGuard g(weight.device());
  const Rows r("fp8_quantize_weight", "weight", weight);
  const int64_t n = weight.size(0), k = weight.size(1), pitch = (k + 15) / 16 * 16;
  const auto opt = weight.options().dtype(at::kByte);
  at::Tensor codes = at::empty_strided({n, k}, {pitch, 1}, opt);
  at::Tensor scales = at::empty({(n + 127) / 128, (k + 127) / 128}, opt);
  const mi_fp8_t out{desc(codes), desc(scales)};
  check_mi(mi_fp8_quantize_weight(&out, &r.d, mi_stream(weight)), "fp8_quantize_weight");
  after_op();
  return {codes, scales};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_fp8(const at::Tensor& x,
                                                            const std::optional<at::Tensor>& weight,
                                                            double eps,
                                                            const std::optional<at::Tensor>& residual) {
  const char* op = "rms_norm_fp8";
  const at::Tensor &w = or_undefined(weight), &res = or_undefined(residual);
  check_fp8(op, {{"x", &x}, {"weight", &w}, {"residual", &res}});
  const c10::DeviceGuard g(x.device());
  const Rows r(op, "x", x);
  TORCH_CHECK(!w.defined() || (w.dim() == 1 && w.size(0) == x.size(-1) && w.scalar_type() == x.scalar_type()),
              op, ": weight must be a vector of ", x.size(-1), " elements of x's type");
  TORCH_CHECK(!res.defined() || (res.sizes() == x.sizes() && res.scalar_type() == x.scalar_type()), op,
              ": residual must have x's shape and type");
  NewRows out(x, x.sizes());
  const at::Tensor wc = w.defined() ? w.contiguous() : w;
  const mi_tensor_t wd = desc(wc);
  at::Tensor total;
  if (res.defined()) {
    const Rows rr(op, "residual", res);
    total = at::empty(x.sizes(), x.options());
    const mi_tensor_t td = desc2(total, r.d.sizes[0], r.d.sizes[1], r.d.sizes[1]);
    check_mi(mi_rms_norm_fp8(&out.d, &td, &r.d, &rr.d, &wd, eps, mi_stream(x)), op);
  } else {
    total = at::empty({0}, x.options());
    check_mi(mi_rms_norm_fp8(&out.d, nullptr, &r.d, nullptr, &wd, eps, mi_stream(x)), op);
  }
  after_op();
  return {out.codes, out.scales, total};
}

at::Tensor fp8_linear(const at::Tensor& x, const at::Tensor& x_scales, const at::Tensor& weight,
                      const at::Tensor& weight_scales, const std::optional<at::Tensor>& bias,
                      const std::optional<at::Tensor>& residual, std::optional<at::ScalarType> dtype) {
  const char* op = "fp8_linear";
  const at::Tensor &b = or_undefined(bias), &res = or_undefined(residual);
  check_fp8(op, {{"codes of x", &x}, {"scales of x", &x_scales}, {"codes of weight", &weight},
                 {"scales of weight", &weight_scales}, {"bias", &b}, {"residual", &res}});
  check_weight(op, "weight", weight, weight_scales);
  const c10::DeviceGuard g(x.device());
  const ReadRows xr(op, x, x_scales);
  const Rows wc(op, "codes of weight", weight), ws(op, "scales of weight", weight_scales);
  const std::vector<int64_t> shape = with_columns(x, weight.size(0));
  TORCH_CHECK(!res.defined() || res.sizes() == at::IntArrayRef(shape), op, ": residual has shape ",
              res.sizes(), ", expected ", at::IntArrayRef(shape));
  TORCH_CHECK(!b.defined() || b.dim() == 1, op, ": bias must be a vector");
  const at::ScalarType type = dtype.has_value() ? *dtype : res.defined() ? res.scalar_type() : at::kBFloat16;
  at::Tensor out = at::empty(shape, x.options().dtype(type));
  const mi_tensor_t o = desc2(out, xr.d.codes.sizes[0], weight.size(0), weight.size(0));
  const mi_fp8_t w{wc.d, ws.d};
  const at::Tensor bc = b.defined() ? b.contiguous() : b;
  const mi_tensor_t bd = desc(bc);
  if (res.defined()) {
    const Rows rr(op, "residual", res);
    check_mi(mi_fp8_linear(&o, &xr.d, &w, &bd, &rr.d, mi_stream(x)), op);
  } else {
    check_mi(mi_fp8_linear(&o, &xr.d, &w, &bd, nullptr, mi_stream(x)), op);
  }
  after_op();
  return out;
}

std::tuple<at::Tensor, at::Tensor> fp8_linear_silu_mul(const at::Tensor& x, const at::Tensor& x_scales,
                                                       const at::Tensor& w_gate,
                                                       const at::Tensor& gate_scales,
                                                       const at::Tensor& w_up,
                                                       const at::Tensor& up_scales) {
  const char* op = "fp8_linear_silu_mul";
  check_fp8(op, {{"codes of x", &x}, {"scales of x", &x_scales}, {"codes of w_gate", &w_gate},
                 {"scales of w_gate", &gate_scales}, {"codes of w_up", &w_up},
                 {"scales of w_up", &up_scales}});
  check_weight(op, "w_gate", w_gate, gate_scales);
  check_weight(op, "w_up", w_up, up_scales);
  const c10::DeviceGuard g(x.device());
  const ReadRows xr(op, x, x_scales);
  const Rows gc(op, "codes of w_gate", w_gate), gs(op, "scales of w_gate", gate_scales),
      uc(op, "codes of w_up", w_up), us(op, "scales of w_up", up_scales);
  NewRows out(x, with_columns(x, w_gate.size(0)));
  const mi_fp8_t wg{gc.d, gs.d}, wu{uc.d, us.d};
  check_mi(mi_fp8_linear_silu_mul(&out.d, &xr.d, &wg, &wu, mi_stream(x)), op);
  after_op();
  return {out.codes, out.scales};
}

}  // namespace efficient
}  // namespace torch_gcu
