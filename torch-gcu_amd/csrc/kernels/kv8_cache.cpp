// Checks that the entry points of the 8-bit key/value cache share.  They read
// descriptors only and run before any device call.
#include <utility>

#include "kv8_common.h"

namespace mi {

namespace {
// int32 vector with unit stride
mi_status_t check_ints(const char* op, const mi_tensor_t* t, const char* name, int64_t n) {
  MI_RETURN_IF(validate(t, name));
  MI_CHECK_ARG(t->dtype == MI_I32 && t->ndim == 1, "%s: %s must be an int32 vector", op, name);
  MI_CHECK_ARG(n < 0 || t->sizes[0] == n, "%s: %s has %lld entries, expected %lld", op, name,
               (long long)t->sizes[0], (long long)n);
  MI_CHECK_ARG(t->sizes[0] <= 1 || t->strides[0] == 1, "%s: %s must be dense", op, name);
  return MI_OK;
}
}  // namespace

bool kv8_apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t extent) {
  if (n0 <= 1 && n1 <= 1) return true;
  if (n0 <= 1) return s1 >= extent;
  if (n1 <= 1) return s0 >= extent;
  if (s0 < s1) {
    std::swap(n0, n1);
    std::swap(s0, s1);
  }
  return s1 >= extent && s0 >= (__int128)(n1 - 1) * s1 + extent;
}

bool kv8_disjoint(const Kv8Rows& a, const Kv8Rows& b, int64_t extent) {
  const __int128 a0 = (uintptr_t)a.data, b0 = (uintptr_t)b.data;
  auto end = [&](const Kv8Rows& x, __int128 at) {
    return at + (__int128)(x.n0 - 1) * x.s0 + (__int128)(x.n1 - 1) * x.s1 + extent;
  };
  if (a.n0 < 1 || a.n1 < 1 || b.n0 < 1 || b.n1 < 1 || end(a, a0) <= b0 || end(b, b0) <= a0)
    return true;
  // rows of one lie among those of the other: with the same strides they meet where
  // some steps of the two make up the distance, to less than a row
  if (a.n0 != b.n0 || a.n1 != b.n1 || (a.n0 > 1 && a.s0 != b.s0) || (a.n1 > 1 && a.s1 != b.s1))
    return false;
  int64_t few = a.n0, step = a.s0, many = a.n1, stride = a.s1;
  if (few > many) {
    std::swap(few, many);
    std::swap(step, stride);
  }
  for (int64_t i = 1 - few; i < few; ++i) {
    const __int128 left = b0 - a0 - (__int128)i * step;
    const __int128 near = many > 1 && stride > 0 ? left / stride : 0;
    for (__int128 j = near - 1; j <= near + 1; ++j) {
      const __int128 off = left - j * stride;
      if (j > -many && j < many && off > -extent && off < extent) return false;
    }
  }
  return true;
}

mi_status_t kv8_check_cache(const char* op, const mi_kv8_cache_t* cache, Kv8Cache* c,
                            int64_t* dim) {
  MI_CHECK_ARG(cache != nullptr, "%s: cache is NULL", op);
  const mi_tensor_t *k = &cache->k, *v = &cache->v;
  const mi_tensor_t *ks = &cache->k_scale, *vs = &cache->v_scale;
  MI_RETURN_IF(validate(k, "k_cache"));
  MI_RETURN_IF(validate(v, "v_cache"));
  MI_RETURN_IF(validate(ks, "k_scale"));
  MI_RETURN_IF(validate(vs, "v_scale"));
  const mi_tensor_t* codes[2] = {k, v};
  const mi_tensor_t* scales[2] = {ks, vs};
  for (int i = 0; i < 2; ++i) {
    const char* n = i ? "v" : "k";
    const mi_tensor_t &t = *codes[i], &s = *scales[i];
    MI_CHECK_ARG(t.dtype == MI_U8 && t.ndim == 4,
                 "%s: %s_cache must be uint8 [pages, heads, page, head_dim]", op, n);
    for (int d = 0; d < 4; ++d)
      MI_CHECK_ARG(t.sizes[d] == k->sizes[d], "%s: k_cache and v_cache have different shapes", op);
    MI_CHECK_ARG(s.dtype == MI_F32 && s.ndim == 2 && s.sizes[0] == t.sizes[0] &&
                     s.sizes[1] == t.sizes[1],
                 "%s: %s_scale must be float32 [pages, heads]", op, n);
    MI_CHECK_ARG(t.sizes[0] >= 1 && t.sizes[1] >= 1, "%s: the cache has no pages or no heads", op);
    if (t.sizes[3] != 64 && t.sizes[3] != 128)
      MI_FAIL(MI_ERR_UNSUPPORTED, "%s: head_dim %lld, 64 and 128 are supported", op,
              (long long)t.sizes[3]);
    const int64_t p = t.sizes[2];
    MI_CHECK_ARG(p >= 16 && p <= 256 && (p & (p - 1)) == 0,
                 "%s: page size %lld is not a power of two from 16 to 256", op, (long long)p);
    MI_CHECK_ARG(t.strides[3] == 1 && t.strides[2] == t.sizes[3] && t.strides[1] % 16 == 0 &&
                     t.strides[0] % 16 == 0 && (uintptr_t)t.data % 16 == 0,
                 "%s: a page's head in %s_cache must be dense and 16-byte aligned", op, n);
    // a page or head that shares memory with another would be written twice
    MI_CHECK_ARG(kv8_apart(t.sizes[0], t.strides[0], t.sizes[1], t.strides[1], p * t.sizes[3]) &&
                     kv8_apart(s.sizes[0], s.strides[0], s.sizes[1], s.strides[1], 1),
                 "%s: pages or heads of the %s cache overlap", op, n);
    MI_CHECK_ARG(t.sizes[0] <= 0x7fffffff && t.sizes[1] <= 65535, "%s: too many pages or heads", op);
  }
  c->k = (const uint8_t*)k->data;
  c->v = (const uint8_t*)v->data;
  c->k_scale = (const float*)ks->data;
  c->v_scale = (const float*)vs->data;
  c->k_sp = k->strides[0];
  c->k_sh = k->strides[1];
  c->v_sp = v->strides[0];
  c->v_sh = v->strides[1];
  c->ks_sp = ks->strides[0];
  c->ks_sh = ks->strides[1];
  c->vs_sp = vs->strides[0];
  c->vs_sh = vs->strides[1];
  c->pages = (int)k->sizes[0];
  c->heads = (int)k->sizes[1];
  c->shift = 0;
  while ((1 << c->shift) < k->sizes[2]) ++c->shift;
  *dim = k->sizes[3];
  return MI_OK;
}

mi_status_t kv8_check_written(const char* op, const Kv8Cache& c, int64_t dim) {
  const int64_t n = sizeof(float);
  const Kv8Rows k{c.k, c.pages, c.k_sp, c.heads, c.k_sh};
  const Kv8Rows v{c.v, c.pages, c.v_sp, c.heads, c.v_sh};
  const Kv8Rows ks{c.k_scale, c.pages, n * c.ks_sp, c.heads, n * c.ks_sh};
  const Kv8Rows vs{c.v_scale, c.pages, n * c.vs_sp, c.heads, n * c.vs_sh};
  MI_CHECK_ARG(kv8_disjoint(k, v, dim << c.shift) && kv8_disjoint(ks, vs, n),
               "%s: k and v of the cache are the same memory", op);
  return MI_OK;
}

mi_status_t kv8_check_queries(const char* op, const mi_tensor_t* q, const mi_tensor_t* lse,
                              int64_t dim, Kv8Args* a) {
  MI_RETURN_IF(validate(q, "q"));
  MI_RETURN_IF(validate(lse, "lse"));
  MI_CHECK_ARG((q->dtype == MI_BF16 || q->dtype == MI_F16) && q->ndim == 3,
               "%s: q must be bfloat16 or float16 [tokens, heads, head_dim]", op);
  MI_CHECK_ARG(q->sizes[2] == dim && q->sizes[1] >= 1 && q->sizes[1] % a->c.heads == 0,
               "%s: q has %lld heads of %lld, the cache %d of %lld", op, (long long)q->sizes[1],
               (long long)q->sizes[2], a->c.heads, (long long)dim);
  if (q->strides[2] != 1 || q->strides[0] % 8 != 0 || q->strides[1] % 8 != 0 ||
      (uintptr_t)q->data % 16 != 0)
    MI_FAIL(MI_ERR_UNSUPPORTED, "%s: rows of q must be dense and 16-byte aligned", op);
  MI_CHECK_ARG(lse->dtype == MI_F32 && lse->ndim == 2 && lse->sizes[0] == q->sizes[0] &&
                   lse->sizes[1] == q->sizes[1],
               "%s: lse must be float32 [tokens, heads]", op);
  a->group = (int)(q->sizes[1] / a->c.heads);
  a->q = (const uint16_t*)q->data;
  a->q_st = q->strides[0];
  a->q_sh = q->strides[1];
  a->lse = (float*)lse->data;
  a->lse_st = lse->strides[0];
  a->lse_sh = lse->strides[1];
  return MI_OK;
}

mi_status_t kv8_check_seqs(const char* op, const mi_tensor_t* table, const mi_tensor_t* lengths,
                           const mi_tensor_t* starts, int64_t tokens, Kv8Args* a) {
  MI_RETURN_IF(validate(table, "block_table"));
  MI_CHECK_ARG(table->dtype == MI_I32 && table->ndim == 2 &&
                   (table->sizes[1] <= 1 || table->strides[1] == 1),
               "%s: block_table must be int32 [sequences, pages of one] with dense rows", op);
  const int64_t seqs = table->sizes[0];
  MI_RETURN_IF(check_ints(op, lengths, "lengths", seqs));
  if (starts != nullptr) MI_RETURN_IF(check_ints(op, starts, "starts", seqs + 1));
  MI_CHECK_ARG(seqs == 0 || table->sizes[1] >= 1, "%s: block_table has no columns", op);
  if (seqs > 0xffff || (table->sizes[1] << a->c.shift) > ((int64_t)1 << 30))
    MI_FAIL(MI_ERR_TOO_LARGE, "%s: more than 65535 sequences, or of more than 2^30 positions", op);
  // items of a call are counted in 32 bits
  if (tokens * a->c.heads * a->group > ((int64_t)1 << 28))
    MI_FAIL(MI_ERR_TOO_LARGE, "%s: more than 2^28 tokens x heads", op);
  a->table = (const int*)table->data;
  a->t_sb = table->strides[0];
  a->width = (int)table->sizes[1];
  a->lengths = (const int*)lengths->data;
  a->starts = starts ? (const int*)starts->data : nullptr;
  a->seqs = (int)seqs;
  a->tokens = (int)tokens;
  return MI_OK;
}

mi_status_t kv8_check_kept(const char* op, const mi_tensor_t* kept, int64_t keep, const Kv8Args& a) {
  MI_RETURN_IF(validate(kept, "kept"));
  MI_CHECK_ARG(kept->dtype == MI_I32 && kept->ndim == 3 && kept->sizes[0] == a.seqs &&
                   kept->sizes[1] == a.c.heads && kept->sizes[2] == keep &&
                   (keep == 1 || kept->strides[2] == 1) &&
                   kv8_apart(kept->sizes[0], kept->strides[0], kept->sizes[1], kept->strides[1], keep),
               "%s: kept must be int32 [sequences, heads, keep] with dense rows of their own", op);
  return MI_OK;
}

mi_status_t kv8_check_weights(const char* op, const mi_tensor_t* w, const char* name,
                              const Kv8Args& a) {
  MI_RETURN_IF(validate(w, name));
  const int64_t cap = (int64_t)a.width << a.c.shift;
  MI_CHECK_ARG(w->dtype == MI_F32 && w->ndim == 3 && w->sizes[0] == a.seqs &&
                   w->sizes[1] == a.c.heads && w->sizes[2] >= cap &&
                   (w->sizes[2] <= 1 || w->strides[2] == 1),
               "%s: %s must be float32 [sequences, heads, at least %lld positions] with dense rows",
               op, name, (long long)cap);
  if (w->sizes[2] > 0x7fffffff) MI_FAIL(MI_ERR_TOO_LARGE, "%s: %s has too many positions", op, name);
  // rows that share memory would be added to twice
  MI_CHECK_ARG(kv8_apart(w->sizes[0], w->strides[0], w->sizes[1], w->strides[1], w->sizes[2]),
               "%s: rows of %s overlap", op, name);
  return MI_OK;
}

}  // namespace mi
