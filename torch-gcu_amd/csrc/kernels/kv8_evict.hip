// Cuts each sequence of the 8-bit cache down to `keep` tokens per k/v head: the
// first `sink`, the last `recent`, and of the others those with the largest
// accumulated weight (ties: the lower position), in their old order, moved to
// pages of the sequence's own row of a second table.
//
// kv8_select_kernel, a block per sequence and head: the weight of rank r among
// the candidates is found by a radix selection on order-preserving integers, 8
// bits a pass; then one scan writes the kept positions and weights in order.
// kv8_move_kernel, a block per new page and head: gathers the tokens' codes,
// takes their largest magnitude, and writes them under the new page's scale.
// Scales are powers of two, so codes move by an exact shift unless they become
// subnormal under a larger scale (half a step of 2^-9 of the new scale).  What
// bounds the pair: the latency of the selection's passes for few sequences, the
// gathered bytes for many.  8 heads of 128: 16 sequences of 4000 to 16000 cut to
// 2000 tokens, 18 us for the selection and 24 for the moves (131 MB, 5.4 TB/s);
// 1 of 1000 cut to 250, 8.7 and 4.
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

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Larger weight, larger integer; -0 as 0, NaN below every number but above 0,
// which stands for positions that are no candidates.
__device__ __forceinline__ uint32_t rank_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 1;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int SELT = 1024;      // threads, four positions each: a chunk
constexpr int SELN = 16 * SELT;  // positions of a round: four chunks

// Up to SELN positions the candidates' ranks are made once and stay in LDS,
// longer sequences make them again in each pass.  What stays is counted per 256
// positions (a wave's four a lane), and one scan of the counts, which every wave
// makes for itself, places it.  Loops stay rolled: with few sequences the
// kernel is a chain of latencies, and the fetch of unrolled code was the longest
// of them (1 x 8 heads of 1000 positions: 16 us with the weights in registers,
// 7.5 like this).
__global__ __launch_bounds__(SELT) void kv8_select_kernel(Kv8Args a, Kv8Evict e) {
  __shared__ __align__(16) uint32_t ranks[SELN];
  __shared__ __align__(16) int hist[4][256][4];  // [pass][bin][copy]: copies ease the adds to one bin
  __shared__ int counts[64];  // sure + (ties << 16) of each 256 positions of a round
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int head = blockIdx.x, b = blockIdx.y, cap = a.width << a.c.shift;
  const int raw = ld_const(a.lengths + b);
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
  const bool held = len <= SELN;
  auto rank_at = [&](int i) __attribute__((always_inline)) {
    return i >= lo && i < hi ? rank_of(w[i]) : 0u;
  };
  auto ranks_at = [&](int i) __attribute__((always_inline)) {
    if (held) return *(const u32x4*)(ranks + i);
    return u32x4{rank_at(i), rank_at(i + 1), rank_at(i + 2), rank_at(i + 3)};
  };
  // all of a thread's loads in flight at once, and the histograms cleared meanwhile
  float x[SELN / SELT];
  if (held && want > 0) {
#pragma unroll
    for (int k = 0; k < SELN / SELT; ++k) x[k] = w[min(k * SELT + tid, len - 1)];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) ((int*)hist)[i * SELT + tid] = 0;
  if (held && want > 0) {
#pragma unroll
    for (int k = 0; k < SELN / SELT; ++k) {
      const int i = k * SELT + tid;
      if (k * SELT < len) ranks[i] = i >= lo && i < hi ? rank_of(x[k]) : 0u;
    }
  }
  __syncthreads();
  uint32_t prefix = 0, mask = 0;
  int ties = want;  // how many of the candidates at the threshold stay
  if (want > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
#pragma unroll 1
      for (int i = 4 * tid; i < len; i += 4 * SELT) {
        const u32x4 u = ranks_at(i);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if ((u[k] & mask) == prefix) atomicAdd(&hist[pass][(u[k] >> shift) & 255][lane & 3], 1);
      }
      __syncthreads();
      // lane l: the four bins 252 - 4 l + 3 .. 0, from the largest down; every
      // wave finds the bin of rank `ties` for itself (the zeros of positions
      // that are no candidates lie behind all candidates)
      int h[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const i32x4 c = *(const i32x4*)hist[pass][252 - 4 * lane + k];
        h[k] = c[0] + c[1] + c[2] + c[3];
      }
      const int sum = h[0] + h[1] + h[2] + h[3], upto = wave_scan(sum);
      const int l = __builtin_ctzll(__ballot(upto >= ties));
      int above = upto - sum, bin = 3;
#pragma unroll
      for (int k = 3; k > 0; --k) {
        if (bin == k && above + h[k] < ties) {
          above += h[k];
          bin = k - 1;
        }
      }
      prefix |= (uint32_t)__builtin_amdgcn_readlane(252 - 4 * lane + bin, l) << shift;
      mask |= 255u << shift;
      ties -= __builtin_amdgcn_readlane(above, l);
    }
  }
  // of positions i .. i + 3: bit k, it stays for sure; bit 4 + k, it is at the
  // threshold, where the first `ties` stay
  auto kinds = [&](int i) __attribute__((always_inline)) {
    if (!cut) return i + 4 <= len ? 15 : i < len ? (1 << (len - i)) - 1 : 0;
    const u32x4 u = want > 0 && i < len ? ranks_at(i) : u32x4{};
    int r = 0;
    if (want > 0 && wave_uniform(i) >= lo && wave_uniform(i) + 256 <= hi) {  // all of the wave's
#pragma unroll
      for (int k = 0; k < 4; ++k) r |= (u[k] > prefix ? 1 << k : 0) | (u[k] == prefix ? 16 << k : 0);
      return r;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool forced = i + k < lo || (i + k >= hi && i + k < len);
      r |= (forced || (u[k] > prefix && want > 0)) << k;
      r |= (want > 0 && u[k] == prefix) << (4 + k);
    }
    return r;
  };
  auto packed = [](int x) __attribute__((always_inline)) {
    return __popc(x & 15) | __popc(x >> 4) << 16;
  };
  int done = 0, tied = 0;
  for (int r0 = 0; r0 < len; r0 += SELN) {
    const int chunks = min((len - r0 + 4 * SELT - 1) / (4 * SELT), 4);
    if (tid < 64) counts[tid] = 0;
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < chunks; ++k) {
      const int own = 4 * (k * SELT + tid), x = kinds(r0 + own), scan = wave_scan(packed(x));
      *(i32x2*)(ranks + own) = i32x2{x, scan};  // in place of the lane's four ranks
      if (lane == 63) counts[k * (SELT / 64) + wave] = scan;
    }
    __syncthreads();
    const int mine = counts[lane], upto = wave_scan(mine);
    const int all = __builtin_amdgcn_readlane(upto, 63);
#pragma unroll 1
    for (int k = 0; k < chunks; ++k) {
      const int own = 4 * (k * SELT + tid), i = r0 + own;
      const i32x2 got = *(const i32x2*)(ranks + own);
      const int x = got[0], n = packed(x);
      const int before = __builtin_amdgcn_readlane(upto - mine, k * (SELT / 64) + wave) + got[1] - n;
      // ties before this position, of which those under `ties` stay
      int tie_at = tied + (int)((uint32_t)before >> 16);
      int at = done + (before & 0xffff) + min(tie_at, ties) - min(tied, ties);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool tie = x >> (4 + q) & 1;
        if ((x >> q & 1) || (tie && tie_at < ties)) {
          if (at < e.keep) {
            kept[at] = i + q;
            nw[at] = w[i + q];
          }
          ++at;
        }
        tie_at += tie;
      }
    }
    done += (all & 0xffff) + min(tied + (int)((uint32_t)all >> 16), ties) - min(tied, ties);
    tied += (int)((uint32_t)all >> 16);
    __syncthreads();
  }
  for (int i = left + tid; i < e.keep; i += SELT) kept[i] = -1;
  for (int i = left + tid; i < e.size; i += SELT) nw[i] = 0.f;
}

// U 16-byte pieces of the page a thread, in registers between the maximum and
// the rescaling.
template <int D, int U>
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
  u32x4 v[U];
  float sc[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = min(tid + 256 * u, n * CH - 1);
    const int pos = kv8_clamp(kept[i / CH], 0, cap - 1);
    const int from = table[pos >> shift], p = kv8_page(from, a.c.pages);
    if (p < 0) record_index_fault(a.fault, from, a.c.pages);
    const int64_t old = max(p, 0);
    v[u] = *(const u32x4*)(codes + old * sp + (pos & (size - 1)) * D + 16 * (i % CH));
    sc[u] = scales[old * ssp];
    if (p < 0) {  // a page that is not there: zeros, whatever the scale of the one read instead
      v[u] = u32x4{};
      sc[u] = 1.f;
    }
  }
  float am = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 x = fp8x4_to_f32(v[u][w]) * sc[u];
#pragma unroll
      for (int k = 0; k < 4; ++k) am = kv8_finite(x[k]) ? fmaxf(am, fabsf(x[k])) : am;
    }
  am = wave_fmax(am);
  if (lane == 0) most[wave] = am;
  __syncthreads();
  const float scale = kv8_scale_of(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])));
  const float inv = 1.0f / scale;
  uint8_t* dst = (uint8_t*)codes + page * sp;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = tid + 256 * u;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // one scale after the other: their product can be infinite where the code is 0
      v[u][w] = f32x4_to_fp8(fp8x4_to_f32(v[u][w]) * sc[u] * inv);
    }
    if (i < n * CH) *(u32x4*)(dst + (i / CH) * D + 16 * (i % CH)) = v[u];
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
  MI_RETURN_IF(kv8_check_written(op, a.c, dim));
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
  MI_RETURN_IF(kv8_check_kept(op, kept, keep, a));
  MI_RETURN_IF(validate(new_lengths, "new_lengths"));
  MI_CHECK_ARG(new_lengths->dtype == MI_I32 && new_lengths->ndim == 1 &&
                   new_lengths->sizes[0] == a.seqs &&
                   (a.seqs <= 1 || new_lengths->strides[0] == 1),
               "%s: new_lengths must be a dense int32 vector of the sequences", op);
  // blocks read the old ones while others write
  auto rows = [](const mi_tensor_t* t) {
    return Kv8Rows{t->data, t->sizes[0], 4 * t->strides[0], t->sizes[1], 4 * t->strides[1]};
  };
  MI_CHECK_ARG(kv8_disjoint({new_lengths->data, 1, 0, 1, 0}, {lengths->data, 1, 0, 1, 0},
                            4 * (int64_t)a.seqs) &&
                   kv8_disjoint(rows(new_weights), rows(weights), 4 * weights->sizes[2]),
               "%s: new_lengths and new_weights need memory of their own", op);
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
  auto move = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, e); };
  const int64_t pieces = (dim / 16) << a.c.shift;
  if (dim == 128) {
    if (pieces <= 256) move(kv8_move_kernel<128, 1>);
    else if (pieces <= 512) move(kv8_move_kernel<128, 2>);
    else if (pieces <= 1024) move(kv8_move_kernel<128, 4>);
    else move(kv8_move_kernel<128, 8>);
  } else {
    if (pieces <= 256) move(kv8_move_kernel<64, 1>);
    else if (pieces <= 512) move(kv8_move_kernel<64, 2>);
    else move(kv8_move_kernel<64, 4>);
  }
  return check_launch(op);
}
