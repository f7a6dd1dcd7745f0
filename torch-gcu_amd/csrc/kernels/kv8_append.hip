// Writes new tokens' keys and values into the pages of an 8-bit cache.
//
// A block (page and k/v head) has one power-of-two scale s, the smallest with
// amax <= 448 s: e4m3 is a floating type, so a power of two loses nothing of
// its precision, and when a larger token makes the scale of a page grow, the
// codes that are there move by an exact shift of their exponents (but for
// numbers that become subnormal).  Tokens written one by one so end up as
// tokens written together.
//
// What bounds it: a prompt's bytes (16-bit tokens read, codes written), a
// decode step's chain of dependent reads (starts, table, token, scale).  One
// thread block per touched page and head owns that page's scale, so nothing
// is shared between blocks.  8 heads of 128: 11137 tokens of four sequences 17.7
// us (68 MB, 3.9 TB/s where a large copy reaches 5.0), 8 tokens of as many
// sequences 4.4 us.
//
// A token with an infinite or NaN element has NaN codes for its whole key, so
// that every query that sees it gets NaN, and 0 in place of the bad elements
// of its value: a bad value reaches the queries that see its token through
// the score, and no other (0 x NaN in a masked place would).
#include <algorithm>

#include "kv8_common.h"

namespace mi {
namespace {

struct Kv8New {
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_st, k_sh, v_st, v_sh;  // strides of a token and a head, in elements
};

template <typename T>
__device__ __forceinline__ void widen8(u32x4 p, float* x) {
  union {
    u32x4 w;
    uint16_t e[8];
  } u;
  u.w = p;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Num<T>::load(u.e[i]);
}

// U 16-byte pieces of the page's keys and as many of its values a thread, in
// registers between the maximum and the codes; NT threads, so that pages of 256
// tokens have as many in flight (11137 tokens of 8 heads of 128, us: in registers,
// and read a second time for the codes, pages of 16 18.6 / 22.0, of 64 17.7 / 18.8,
// of 256 24.2 / 37.7).
template <typename T, int D, int U, int NT>
__global__ __launch_bounds__(NT) void kv8_append_kernel(Kv8Args a, Kv8New x) {
  constexpr int CH = D / 8;  // 8-element pieces of a token's row
  __shared__ int bad[256];   // tokens of the page with a non-finite element
  __shared__ float most[2][NT / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int cap = a.width << a.c.shift, shift = a.c.shift, size = 1 << shift;
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    kv8_report_lengths(a.lengths, a.seqs, cap, a.fault);
    for (int b = threadIdx.x; b < a.seqs; b += blockDim.x) {
      const Kv8Seq s = kv8_seq(a.starts[b], a.starts[b + 1], a.lengths[b], a.tokens, cap);
      if (!s.bad && s.n > s.len) record_index_fault(a.fault, s.len - s.n, cap);
    }
  }
  int seq, nth;
  Kv8Seq s;
  const bool found = Kv8Lanes(a).find(
      blockIdx.x, [&](const Kv8Seq& x) { return kv8_touched(x, shift); }, &seq, &s, &nth);
  if (!found) return;
  const int old = s.len - s.n;  // position of the first new token
  const int index = (old >> shift) + nth;
  const int entry = a.table[seq * a.t_sb + index], page = kv8_page(entry, a.c.pages);
  if (page < 0) {
    if (threadIdx.x == 0) record_index_fault(a.fault, entry, a.c.pages);
    return;
  }
  const int lo = max(old - (index << shift), 0), hi = min(s.len - (index << shift), size);
  const int head = blockIdx.y;
  const int64_t row0 = (int64_t)s.first + (index << shift) - old;  // token of slot 0
  const uint16_t* src[2] = {x.k + row0 * x.k_st + head * x.k_sh, x.v + row0 * x.v_st + head * x.v_sh};
  const int64_t st[2] = {x.k_st, x.v_st};
  uint8_t* dst[2] = {(uint8_t*)a.c.k + page * a.c.k_sp + head * a.c.k_sh,
                     (uint8_t*)a.c.v + page * a.c.v_sp + head * a.c.v_sh};
  float* scales[2] = {(float*)a.c.k_scale + page * a.c.ks_sp + head * a.c.ks_sh,
                      (float*)a.c.v_scale + page * a.c.vs_sp + head * a.c.vs_sh};

  const int n = (hi - lo) * CH;
  u32x4 r[2][U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (NT * u < n) {
      const int i = min((int)threadIdx.x + NT * u, n - 1), slot = lo + i / CH, c = i % CH;
#pragma unroll
      for (int w = 0; w < 2; ++w) r[w][u] = *(const u32x4*)(src[w] + slot * st[w] + 8 * c);
    }
  const float was[2] = {*scales[0], *scales[1]};
  for (int i = threadIdx.x; i < size; i += NT) bad[i] = 0;
  __syncthreads();  // and every thread has read the scales
  float am[2] = {0.f, 0.f};
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (NT * u < n) {
      const int slot = lo + min((int)threadIdx.x + NT * u, n - 1) / CH;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float e[8];
        widen8<T>(r[w][u], e);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (kv8_finite(e[j])) am[w] = fmaxf(am[w], fabsf(e[j]));
          else bad[slot] = 1;  // every writer writes the same
        }
      }
    }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    am[w] = wave_fmax(am[w]);
    if (lane == 0) most[w][wave] = am[w];
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float m = most[w][0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) m = fmaxf(m, most[w][i]);
    const float before = was[w];
    // a page starts anew with its first slot, whatever scale it had
    float scale = kv8_scale_of(m);
    if (lo > 0) scale = fmaxf(scale, before);
    if (lo > 0 && scale != before) {
      const float ratio = before / scale;
      for (int i = threadIdx.x; i < lo * (D / 16); i += NT) {
        u32x4* p = (u32x4*)dst[w] + i;
        u32x4 v = *p;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = f32x4_to_fp8(fp8x4_to_f32(v[j]) * ratio);
        *p = v;
      }
    }
    const float inv = 1.0f / scale;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = threadIdx.x + NT * u, slot = lo + i / CH, c = i % CH;
      if (i >= n) continue;
      float e[8];
      widen8<T>(r[w][u], e);
      const bool nan = w == 0 && bad[slot] != 0;
      f32x4 p[2];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = kv8_finite(e[j]) ? e[j] * inv : 0.f;
        p[j >> 2][j & 3] = nan ? NAN : y;
      }
      *(u32x2*)(dst[w] + slot * D + 8 * c) = u32x2{f32x4_to_fp8(p[0]), f32x4_to_fp8(p[1])};
    }
    if (threadIdx.x == 0) *scales[w] = scale;
  }
}

}  // namespace
}  // namespace mi

extern "C" mi_status_t mi_kv8_append(const mi_kv8_cache_t* cache, const mi_tensor_t* k,
                                     const mi_tensor_t* v, const mi_tensor_t* block_table,
                                     const mi_tensor_t* lengths, const mi_tensor_t* starts,
                                     mi_stream_t stream) {
  using namespace mi;
  clear_error();
  const char* op = "kv8_append";
  Kv8Args a{};
  int64_t dim = 0;
  a.group = 1;
  MI_RETURN_IF(kv8_check_cache(op, cache, &a.c, &dim));
  MI_RETURN_IF(kv8_check_written(op, a.c, dim));
  MI_RETURN_IF(validate(k, "k"));
  MI_RETURN_IF(validate(v, "v"));
  for (const mi_tensor_t* t : {k, v}) {
    MI_CHECK_ARG(t->ndim == 3 && t->sizes[1] == a.c.heads && t->sizes[2] == dim,
                 "%s: k and v must be [tokens, heads, head_dim] of the cache's heads and head_dim",
                 op);
    MI_CHECK_ARG((t->dtype == MI_BF16 || t->dtype == MI_F16) && t->dtype == k->dtype,
                 "%s: k and v must both be bfloat16 or float16", op);
    MI_CHECK_ARG(t->sizes[0] == k->sizes[0], "%s: k and v have different numbers of tokens", op);
    if (t->strides[2] != 1 || t->strides[0] % 8 != 0 || t->strides[1] % 8 != 0 ||
        (uintptr_t)t->data % 16 != 0)
      MI_FAIL(MI_ERR_UNSUPPORTED, "%s: rows of k and v must be dense and 16-byte aligned", op);
  }
  MI_RETURN_IF(kv8_check_seqs(op, block_table, lengths, starts, k->sizes[0], &a));
  if (a.tokens == 0 || a.seqs == 0) return MI_OK;
  a.fault = index_fault_word();
  const Kv8New x{(const uint16_t*)k->data, (const uint16_t*)v->data, k->strides[0], k->strides[1],
                 v->strides[0], v->strides[1]};
  const dim3 grid((unsigned)kv8_touched_most(a.tokens, a.seqs, a.c.shift), (unsigned)a.c.heads);
  hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, a, x);
  };
  auto run = [&](auto type, auto width) {
    typedef decltype(type) T;
    constexpr int D = decltype(width)::value;
    const int64_t pieces = (int64_t)(D / 8) << a.c.shift;
    if (pieces <= 512) launch(kv8_append_kernel<T, D, 2, 256>, 256);
    else if (pieces <= 1024) launch(kv8_append_kernel<T, D, 4, 256>, 256);
    else if (pieces <= 2048) launch(kv8_append_kernel<T, D, 4, 512>, 512);
    else if constexpr (D == 128) launch(kv8_append_kernel<T, D, 4, 1024>, 1024);
  };
  const std::integral_constant<int, 128> wide;
  const std::integral_constant<int, 64> narrow;
  if (k->dtype == MI_BF16) dim == 128 ? run(BF16{}, wide) : run(BF16{}, narrow);
  else dim == 128 ? run(F16{}, wide) : run(F16{}, narrow);
  return check_launch(op);
}
