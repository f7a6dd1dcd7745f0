// efficient_ops of the 8-bit key/value cache: append, attention, accumulated
// weights and eviction over a paged pool of e4m3 codes.  New ops with no
// counterpart in the reference; argument shapes are checked by the kernel
// library (include/mi355x_ops.h), devices and what has to be copied here.
#include <ATen/ATen.h>

#include <cmath>

#include "dispatch_util.h"
#include "efficient_ops.h"

namespace torch_gcu {
namespace efficient {

namespace {

// The cache's four tensors and whatever else a call takes: gcu tensors of one
// device.  Nothing that a call writes, and no index tensor, is copied.
void check_kv8(const char* op, std::initializer_list<std::pair<const char*, const at::Tensor*>> ts) {
  std::optional<at::Device> common;
  for (const auto& [name, t] : ts) {
    TORCH_CHECK(is_gcu(*t), op, ": ", name, " must be a gcu tensor");
    check_device(common, *t, op, name);
  }
}

mi_kv8_cache_t cache_desc(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_scale,
                          const at::Tensor& v_scale) {
  return {desc(k), desc(v), desc(k_scale), desc(v_scale)};
}

// [tokens, heads, head_dim] with dense, 16-byte aligned rows
at::Tensor rows3(const char* op, const char* name, const at::Tensor& t) {
  TORCH_CHECK(t.dim() == 3, op, ": ", name, " must be [tokens, heads, head_dim]");
  const bool ok = t.stride(2) == 1 && t.stride(1) % 8 == 0 && t.stride(0) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

double scale_or_default(const std::optional<double>& scale, const at::Tensor& q) {
  return scale.has_value() ? *scale : 1.0 / std::sqrt((double)std::max<int64_t>(q.size(2), 1));
}

}  // namespace

void kv8_append(at::Tensor& k_cache, at::Tensor& v_cache, at::Tensor& k_scale, at::Tensor& v_scale,
                const at::Tensor& k, const at::Tensor& v, const at::Tensor& block_table,
                const at::Tensor& lengths, const at::Tensor& starts) {
  check_kv8("kv8_append", {{"k_cache", &k_cache}, {"v_cache", &v_cache}, {"k_scale", &k_scale},
                           {"v_scale", &v_scale}, {"k", &k}, {"v", &v},
                           {"block_table", &block_table}, {"lengths", &lengths},
                           {"starts", &starts}});
  const c10::DeviceGuard g(k_cache.device());
  const at::Tensor kr = rows3("kv8_append", "k", k), vr = rows3("kv8_append", "v", v);
  const mi_kv8_cache_t c = cache_desc(k_cache, v_cache, k_scale, v_scale);
  const mi_tensor_t kd = desc(kr), vd = desc(vr), t = desc(block_table), l = desc(lengths),
                    s = desc(starts);
  check_mi(mi_kv8_append(&c, &kd, &vd, &t, &l, &s, mi_stream(k_cache)), "kv8_append");
  after_op();
}

std::tuple<at::Tensor, at::Tensor> kv8_attention(const at::Tensor& q, const at::Tensor& k_cache,
                                                 const at::Tensor& v_cache,
                                                 const at::Tensor& k_scale,
                                                 const at::Tensor& v_scale,
                                                 const at::Tensor& block_table,
                                                 const at::Tensor& lengths,
                                                 const at::Tensor& starts,
                                                 std::optional<double> scale) {
  check_kv8("kv8_attention", {{"q", &q}, {"k_cache", &k_cache}, {"v_cache", &v_cache},
                              {"k_scale", &k_scale}, {"v_scale", &v_scale},
                              {"block_table", &block_table}, {"lengths", &lengths},
                              {"starts", &starts}});
  const c10::DeviceGuard g(q.device());
  const at::Tensor qr = rows3("kv8_attention", "q", q);
  at::Tensor out = at::empty(q.sizes(), q.options());
  at::Tensor lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  const mi_kv8_cache_t c = cache_desc(k_cache, v_cache, k_scale, v_scale);
  const mi_tensor_t o = desc(out), e = desc(lse), qd = desc(qr), t = desc(block_table),
                    l = desc(lengths), s = desc(starts);
  check_mi(mi_kv8_attention(&o, &e, &qd, &c, &t, &l, &s, scale_or_default(scale, q),
                            /*fill_rest=*/1, mi_stream(out)),
           "kv8_attention");
  after_op();
  return {out, lse};
}

void kv8_weigh_(at::Tensor& weights, const at::Tensor& q, const at::Tensor& lse,
                const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& k_scale,
                const at::Tensor& v_scale, const at::Tensor& block_table,
                const at::Tensor& lengths, const at::Tensor& starts, std::optional<double> scale) {
  check_kv8("kv8_weigh_", {{"weights", &weights}, {"q", &q}, {"lse", &lse},
                           {"k_cache", &k_cache}, {"v_cache", &v_cache}, {"k_scale", &k_scale},
                           {"v_scale", &v_scale}, {"block_table", &block_table},
                           {"lengths", &lengths}, {"starts", &starts}});
  const c10::DeviceGuard g(weights.device());
  const at::Tensor qr = rows3("kv8_weigh_", "q", q);
  const mi_kv8_cache_t c = cache_desc(k_cache, v_cache, k_scale, v_scale);
  const mi_tensor_t w = desc(weights), qd = desc(qr), e = desc(lse), t = desc(block_table),
                    l = desc(lengths), s = desc(starts);
  check_mi(mi_kv8_weigh(&w, &qd, &e, &c, &t, &l, &s, scale_or_default(scale, q),
                        mi_stream(weights)),
           "kv8_weigh_");
  after_op();
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> kv8_evict(
    at::Tensor& k_cache, at::Tensor& v_cache, at::Tensor& k_scale, at::Tensor& v_scale,
    const at::Tensor& weights, const at::Tensor& block_table, const at::Tensor& new_table,
    const at::Tensor& lengths, int64_t keep, int64_t recent, int64_t sink) {
  check_kv8("kv8_evict", {{"k_cache", &k_cache}, {"v_cache", &v_cache}, {"k_scale", &k_scale},
                          {"v_scale", &v_scale}, {"weights", &weights},
                          {"block_table", &block_table}, {"new_table", &new_table},
                          {"lengths", &lengths}});
  TORCH_CHECK(weights.dim() == 3 && keep >= 1,
              "kv8_evict: weights must be [sequences, heads, positions] and keep positive");
  const c10::DeviceGuard g(k_cache.device());
  at::Tensor kept = at::empty({weights.size(0), weights.size(1), keep}, lengths.options());
  at::Tensor left = at::empty({weights.size(0)}, lengths.options());
  at::Tensor moved = at::empty(weights.sizes(), weights.options());
  const mi_kv8_cache_t c = cache_desc(k_cache, v_cache, k_scale, v_scale);
  const mi_tensor_t w = desc(weights), t = desc(block_table), n = desc(new_table),
                    l = desc(lengths), kd = desc(kept), ld = desc(left), md = desc(moved);
  check_mi(mi_kv8_evict(&c, &w, &t, &n, &l, keep, recent, sink, &kd, &ld, &md, mi_stream(kept)),
           "kv8_evict");
  after_op();
  return {kept, left, moved};
}

}  // namespace efficient
}  // namespace torch_gcu
