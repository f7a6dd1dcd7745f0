// Checks that the entry points of the 8-bit floating point linear layers share.
// They read descriptors only and run before any device call.
#include "fp8_common.h"

namespace mi {

namespace {
bool dense_columns(const mi_tensor_t& t) { return t.sizes[1] <= 1 || t.strides[1] == 1; }
bool rows_apart(const mi_tensor_t& t) { return t.sizes[0] <= 1 || t.strides[0] >= t.sizes[1]; }
}  // namespace

mi_status_t fp8_check(const char* op, const char* name, const mi_fp8_t* t, bool weight, bool written,
                      Fp8Mat* m) {
  MI_CHECK_ARG(t != nullptr, "%s: %s is NULL", op, name);
  const mi_tensor_t &c = t->codes, &s = t->scales;
  MI_RETURN_IF(validate(&c, name));
  MI_RETURN_IF(validate(&s, name));
  MI_CHECK_ARG(c.dtype == MI_U8 && c.ndim == 2, "%s: codes of %s must be uint8 [rows, columns]", op, name);
  const int64_t rows = weight ? fp8_groups(c.sizes[0]) : c.sizes[0];
  MI_CHECK_ARG(s.dtype == MI_U8 && s.ndim == 2 && s.sizes[0] == rows &&
                   s.sizes[1] == fp8_groups(c.sizes[1]),
               "%s: scales of %s must be uint8 [%lld, %lld], one for each %s", op, name,
               (long long)rows, (long long)fp8_groups(c.sizes[1]),
               weight ? "128 x 128 block" : "row's 128 columns");
  MI_CHECK_ARG(dense_columns(c) && dense_columns(s), "%s: rows of %s must be dense", op, name);
  if (written) {
    MI_CHECK_ARG(rows_apart(c) && rows_apart(s), "%s: rows of %s overlap", op, name);
    MI_RETURN_IF(fp8_check_apart(op, "codes", &c, "scales", &s));
  }
  if (c.sizes[0] > 0x7fffffff || c.sizes[1] > (1 << 30))
    MI_FAIL(MI_ERR_TOO_LARGE, "%s: %s has 2^31 rows or more, or more than 2^30 columns", op, name);
  *m = Fp8Mat{(uint8_t*)c.data, (uint8_t*)s.data, c.strides[0], s.strides[0]};
  return MI_OK;
}

mi_status_t fp8_check_wide(const char* op, const char* name, const mi_tensor_t* t, bool f32) {
  MI_RETURN_IF(validate(t, name));
  MI_CHECK_ARG(t->ndim == 2 && dense_columns(*t), "%s: %s must be [rows, columns] with dense rows", op,
               name);
  MI_CHECK_ARG(t->dtype == MI_BF16 || t->dtype == MI_F16 || (f32 && t->dtype == MI_F32),
               "%s: %s must be bfloat16%s", op, name, f32 ? ", float16 or float32" : " or float16");
  return MI_OK;
}

mi_status_t fp8_check_apart(const char* op, const char* name, const mi_tensor_t* out,
                            const char* other_name, const mi_tensor_t* other) {
  auto range = [](const mi_tensor_t& t, __int128* first, __int128* last) {
    *first = *last = (uintptr_t)t.data;
    __int128 n = dtype_size(t.dtype);
    for (int d = 0; d < t.ndim; ++d) {
      if (t.sizes[d] == 0) return false;
      n += (__int128)(t.sizes[d] - 1) * t.strides[d] * dtype_size(t.dtype);
    }
    *last += n;
    return true;
  };
  if (out == nullptr || other == nullptr || out->data == nullptr || other->data == nullptr) return MI_OK;
  __int128 a0, a1, b0, b1;
  if (!range(*out, &a0, &a1) || !range(*other, &b0, &b1) || a1 <= b0 || b1 <= a0) return MI_OK;
  // rows of one may lie between rows of the other, in one buffer of the same row stride
  const int64_t size = dtype_size(out->dtype), other_size = dtype_size(other->dtype);
  if (out->ndim == 2 && other->ndim == 2 && out->sizes[0] > 1 && other->sizes[0] > 1 &&
      out->strides[0] * size == other->strides[0] * other_size && out->strides[0] > 0) {
    const __int128 step = out->strides[0] * size, w = out->sizes[1] * size,
                   v = other->sizes[1] * other_size;
    const __int128 off = ((b0 - a0) % step + step) % step;  // where other's rows begin in out's
    if (off >= w && off + v <= step) return MI_OK;
  }
  MI_FAIL(MI_ERR_INVALID, "%s: %s shares memory with %s", op, name, other_name);
}

}  // namespace mi
