// Cuts each sequence of the 8-bit cache down to `keep` tokens per k/v head: the
// first `sink`, the last `recent`, and of the others those with the largest
// accumulated weight (ties: the lower position), in their old order, moved to
// pages of the sequence's own row of a second table.
//
// kv8_select_kernel, a block per sequence and head: the weight of rank r among
// the candidates is found by a radix selection on order-preserving integers, 8
// bits a pass; then one pass in order writes the kept positions and weights.
// kv8_move_kernel, a block per new page and head: gathers the tokens' codes,
// takes their largest magnitude, and writes them under the new page's scale.
// Scales are powers of two, so codes move by an exact shift unless they become
// subnormal under a larger scale (half a step of 2^-9 of the new scale).  What
// bounds the pair: the latency of the selection's passes for few sequences, the
// gathered bytes for many.
#include <algorithm>

#include "kv8_common.h"

namespace mi {
namespace {

struct Kv8Evict {
  const float* w;
  int64_t w_sb, w_sh;
  float* new_w;
  int64_t nw_sb, nw_sh;
  int* kept;
  int64_t k_sb, k_sh;
  int* new_lengths;
  const int* new_table;
  int64_t nt_sb;
  int size;  // positions of new_w
  int keep, recent, sink;
};

// Larger weight, larger integer; -0 as 0, NaN below everything.
__device__ __forceinline__ uint32_t rank_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int SELT = 1024;

__global__ __launch_bounds__(SELT) void kv8_select_kernel(Kv8Args a, Kv8Evict e) {
  __shared__ int hist[256];
  __shared__ int pick[2];
  __shared__ int sums[2][SELT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int head = blockIdx.x, b = blockIdx.y, cap = a.width << a.c.shift;
  const int raw = a.lengths[b];
  const int len = raw < 0 || raw > cap ? 0 : raw;
  if (len != raw && head == 0 && tid == 0) record_index_fault(a.fault, raw, (int64_t)cap + 1);
  const float* w = e.w + b * e.w_sb + head * e.w_sh;
  float* nw = e.new_w + b * e.nw_sb + head * e.nw_sh;
  int* kept = e.kept + b * e.k_sb + head * e.k_sh;
  const int left = min(len, e.keep);
  if (head == 0 && tid == 0) e.new_lengths[b] = left;
  // candidates [lo, hi), of which `want` stay
  const bool cut = len > e.keep;
  const int lo = cut ? e.sink : len, hi = cut ? len - e.recent : len;
  const int want = cut ? e.keep - e.sink - e.recent : 0;
  uint32_t prefix = 0, mask = 0;
  int ties = want;  // how many of the candidates at the threshold stay
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += SELT) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += SELT) {
        const uint32_t u = rank_of(w[i]);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (wave == 0) {
        // lane l: the four bins 255 - 4 l - 0 .. 3, from the largest down
        int h[4], sum = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += h[k] = hist[255 - 4 * lane - k];
        const int upto = wave_scan(sum);
        int above = upto - sum;
        const uint64_t hit = __ballot(upto >= ties);
        if (lane == __builtin_ctzll(hit)) {
          int k = 0;
          while (above + h[k] < ties) above += h[k++];
          pick[0] = 255 - 4 * lane - k;
          pick[1] = ties - above;
        }
      }
      __syncthreads();
      prefix |= (uint32_t)pick[0] << shift;
      mask |= 255u << shift;
      ties = pick[1];
      __syncthreads();
    }
  }
  // in order: what stays, and the first `ties` of those at the threshold
  int done = 0, tied = 0;
  for (int i0 = 0; i0 < len; i0 += SELT) {
    const int i = i0 + tid;
    const float x = i < len ? w[i] : 0.f;
    const uint32_t u = rank_of(x);
    const bool cand = i >= lo && i < hi;
    const bool tie = cand && want > 0 && u == prefix;
    const bool sure = i < len && (!cand || (want > 0 && u > prefix));
    const uint64_t mt = __ballot(tie), ms = __ballot(sure);
    if (lane == 0) {
      sums[0][wave] = __popcll(mt);
      sums[1][wave] = __popcll(ms);
    }
    __syncthreads();
    int t0 = tied, tw = 0, s_all = 0, s0 = 0;
#pragma unroll
    for (int k = 0; k < SELT / 64; ++k) {
      if (k < wave) {
        tw += sums[0][k];
        s0 += sums[1][k];
      }
      t0 += sums[0][k];
      s_all += sums[1][k];
    }
    const uint64_t under = ((uint64_t)1 << lane) - 1;
    const int tie_at = tied + tw + __popcll(mt & under);
    const bool stay = sure || (tie && tie_at < ties);
    // ties that stay before this one: all of them until `ties` are there
    const int at = done + s0 + __popcll(ms & under) + min(tie_at, ties) - min(tied, ties);
    if (stay && at < e.keep) {
      kept[at] = i;
      nw[at] = x;
    }
    done += s_all + min(t0, ties) - min(tied, ties);
    tied = t0;
    __syncthreads();
  }
  for (int i = left + tid; i < e.keep; i += SELT) kept[i] = -1;
  for (int i = left + tid; i < e.size; i += SELT) nw[i] = 0.f;
}

template <int D>
__global__ __launch_bounds__(256) void kv8_move_kernel(Kv8Args a, Kv8Evict e) {
  constexpr int CH = D / 16;  // 16-code pieces of a row
  __shared__ float most[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int index = blockIdx.x, head = blockIdx.y, b = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  const int shift = a.c.shift, size = 1 << shift, cap = a.width << shift;
  const int raw = a.lengths[b], len = raw < 0 || raw > cap ? 0 : raw;
  const int left = min(len, e.keep), n = min(left - (index << shift), size);
  if (n <= 0) return;
  const int entry = e.new_table[b * e.nt_sb + index], page = kv8_page(entry, a.c.pages);
  if (page < 0) {
    if (tid == 0) record_index_fault(a.fault, entry, a.c.pages);
    return;
  }
  const uint8_t* codes = (is_v ? a.c.v : a.c.k) + head * (is_v ? a.c.v_sh : a.c.k_sh);
  const float* scales = (is_v ? a.c.v_scale : a.c.k_scale) + head * (is_v ? a.c.vs_sh : a.c.ks_sh);
  const int64_t sp = is_v ? a.c.v_sp : a.c.k_sp, ssp = is_v ? a.c.vs_sp : a.c.ks_sp;
  const int* kept = e.kept + b * e.k_sb + head * e.k_sh + (index << shift);
  const int* table = a.table + b * a.t_sb;
  auto source = [&](int i, u32x4* v, float* scale) __attribute__((always_inline)) {
    const int pos = kv8_clamp(kept[i / CH], 0, cap - 1);
    const int from = table[pos >> shift], p = kv8_page(from, a.c.pages);
    *v = u32x4{};
    *scale = 0.f;
    if (p >= 0) {
      *v = *(const u32x4*)(codes + p * sp + (pos & (size - 1)) * D + 16 * (i % CH));
      *scale = scales[p * ssp];
    } else {
      record_index_fault(a.fault, from, a.c.pages);
    }
  };
  float am = 0.f;
  for (int i = tid; i < n * CH; i += 256) {
    u32x4 v;
    float sc;
    source(i, &v, &sc);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 x = fp8x4_to_f32(v[w]) * sc;
#pragma unroll
      for (int k = 0; k < 4; ++k) am = kv8_finite(x[k]) ? fmaxf(am, fabsf(x[k])) : am;
    }
  }
  am = wave_fmax(am);
  if (lane == 0) most[wave] = am;
  __syncthreads();
  const float scale = kv8_scale_of(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])));
  const float inv = 1.0f / scale;
  uint8_t* dst = (uint8_t*)codes + page * sp;
  for (int i = tid; i < n * CH; i += 256) {
    u32x4 v;
    float sc;
    source(i, &v, &sc);
#pragma unroll
    for (int w = 0; w < 4; ++w) v[w] = f32x4_to_fp8(fp8x4_to_f32(v[w]) * (sc * inv));
    *(u32x4*)(dst + (i / CH) * D + 16 * (i % CH)) = v;
  }
  if (tid == 0) ((float*)scales)[page * ssp] = scale;
}

}  // namespace
}  // namespace mi

extern "C" mi_status_t mi_kv8_evict(const mi_kv8_cache_t* cache, const mi_tensor_t* weights,
                                    const mi_tensor_t* block_table, const mi_tensor_t* new_table,
                                    const mi_tensor_t* lengths, int64_t keep, int64_t recent,
                                    int64_t sink, const mi_tensor_t* kept,
                                    const mi_tensor_t* new_lengths, const mi_tensor_t* new_weights,
                                    mi_stream_t stream) {
  using namespace mi;
  clear_error();
  const char* op = "kv8_evict";
  Kv8Args a{};
  Kv8Evict e{};
  int64_t dim = 0;
  a.group = 1;
  MI_RETURN_IF(kv8_check_cache(op, cache, &a.c, &dim));
  MI_RETURN_IF(kv8_check_seqs(op, block_table, lengths, nullptr, 0, &a));
  MI_RETURN_IF(kv8_check_weights(op, weights, "weights", a));
  MI_RETURN_IF(kv8_check_weights(op, new_weights, "new_weights", a));
  MI_CHECK_ARG(new_weights->sizes[2] == weights->sizes[2], "%s: weights of different lengths", op);
  MI_CHECK_ARG(keep >= 1 && recent >= 0 && sink >= 0 && recent <= keep && sink <= keep - recent,
               "%s: keep %lld, recent %lld, sink %lld: keep must be positive and hold the other two",
               op, (long long)keep, (long long)recent, (long long)sink);
  if (keep > ((int64_t)1 << 30)) MI_FAIL(MI_ERR_TOO_LARGE, "%s: keep is over 2^30", op);
  MI_RETURN_IF(validate(new_table, "new_table"));
  const int64_t pages = (keep + ((int64_t)1 << a.c.shift) - 1) >> a.c.shift;
  MI_CHECK_ARG(new_table->dtype == MI_I32 && new_table->ndim == 2 &&
                   new_table->sizes[0] == a.seqs && new_table->sizes[1] >= pages &&
                   (new_table->sizes[1] <= 1 || new_table->strides[1] == 1),
               "%s: new_table must be int32 [sequences, at least %lld pages] with dense rows", op,
               (long long)pages);
  MI_RETURN_IF(validate(kept, "kept"));
  MI_CHECK_ARG(kept->dtype == MI_I32 && kept->ndim == 3 && kept->sizes[0] == a.seqs &&
                   kept->sizes[1] == a.c.heads && kept->sizes[2] == keep &&
                   (keep == 1 || kept->strides[2] == 1) &&
                   (a.seqs <= 1 || kept->strides[0] >= keep) &&
                   (a.c.heads <= 1 || kept->strides[1] >= keep),
               "%s: kept must be int32 [sequences, heads, keep] with dense rows of their own", op);
  MI_RETURN_IF(validate(new_lengths, "new_lengths"));
  MI_CHECK_ARG(new_lengths->dtype == MI_I32 && new_lengths->ndim == 1 &&
                   new_lengths->sizes[0] == a.seqs &&
                   (a.seqs <= 1 || new_lengths->strides[0] == 1),
               "%s: new_lengths must be a dense int32 vector of the sequences", op);
  if (a.seqs > 32767) MI_FAIL(MI_ERR_TOO_LARGE, "%s: more than 32767 sequences", op);
  if (a.seqs == 0) return MI_OK;
  e.w = (const float*)weights->data;
  e.w_sb = weights->strides[0];
  e.w_sh = weights->strides[1];
  e.new_w = (float*)new_weights->data;
  e.nw_sb = new_weights->strides[0];
  e.nw_sh = new_weights->strides[1];
  e.kept = (int*)kept->data;
  e.k_sb = kept->strides[0];
  e.k_sh = kept->strides[1];
  e.new_lengths = (int*)new_lengths->data;
  e.new_table = (const int*)new_table->data;
  e.nt_sb = new_table->strides[0];
  e.size = (int)new_weights->sizes[2];
  e.keep = (int)keep;
  e.recent = (int)recent;
  e.sink = (int)sink;
  a.fault = index_fault_word();
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(kv8_select_kernel, dim3((unsigned)a.c.heads, (unsigned)a.seqs), dim3(SELT), 0,
                     s, a, e);
  MI_RETURN_IF(check_launch(op));
  const dim3 grid((unsigned)pages, (unsigned)a.c.heads, 2u * (unsigned)a.seqs);
  if (dim == 128) hipLaunchKernelGGL((kv8_move_kernel<128>), grid, dim3(256), 0, s, a, e);
  else hipLaunchKernelGGL((kv8_move_kernel<64>), grid, dim3(256), 0, s, a, e);
  return check_launch(op);
}
