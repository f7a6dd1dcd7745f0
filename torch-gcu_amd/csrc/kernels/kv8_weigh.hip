// Adds up, per cached position and k/v head, the softmax weights that a call's
// queries gave it: weights[b, hk, j] += sum over the queries i of sequence b and
// the heads of the group of exp(scale q_i k_j - lse_i), j up to the query's own
// position.  lse is what the attention call returned, so the weights need no
// second pass over the keys' maxima, and every position is owned by one lane:
// no atomics, the same sums every time.
//
// What bounds it: a decode step reads the keys' codes once; a prompt's scores
// are one matrix product.  A wave keeps 32 keys as MFMA operands and takes the
// query rows 32 at a time (S^T = K Q^T, v_mfma_f32_32x32x16); a lane adds its 16
// scores' weights over all rows of its column and the 32 columns are added at
// the end.
#include <algorithm>

#include "kv8_common.h"

namespace mi {
namespace {

struct Kv8Weights {
  float* w;
  int64_t sb, sh;
};

constexpr int WKT = 32, WRT = 32, WNW = 4;

// Parts that a sequence's keys are cut into, by its work in 32 x 32 tiles.
__device__ __forceinline__ int weigh_parts(const Kv8Seq& s, int group, int chunk) {
  const Kv8Cut c = kv8_cut(s, group, WRT, WKT);
  if (c.row_tiles == 0 || c.key_tiles == 0) return 0;
  const int64_t parts = ((int64_t)c.row_tiles * c.key_tiles + chunk - 1) / chunk;
  return (int)(parts < c.key_tiles ? parts : c.key_tiles);
}

template <typename T, int D>
__global__ __launch_bounds__(64 * WNW, 2) void kv8_weigh_kernel(Kv8Args a, Kv8Weights wt) {
  typedef typename AttnOp<T>::vec vec;
  constexpr int P = D / 32;  // 16-byte pieces of a lane's half of a key
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int cap = a.width << a.c.shift;
  if (blockIdx.x == 0) kv8_report_lengths(a.lengths, a.seqs, cap, a.fault);
  const Kv8Lanes lanes(a);
  const int chunk =
      lanes.chunk([&](const Kv8Seq& s) { return kv8_cut(s, a.group, WRT, WKT).work(); });
  int seq, place;
  Kv8Seq s;
  const bool found = lanes.find(
      blockIdx.x, [&](const Kv8Seq& x) { return a.c.heads * weigh_parts(x, a.group, chunk); }, &seq,
      &s, &place);
  if (!found) return;
  const int parts = weigh_parts(s, a.group, chunk), part = place % parts, head = place / parts;
  const Kv8Cut cut = kv8_cut(s, a.group, WRT, WKT);
  const int lo = (int)((int64_t)cut.key_tiles * part / parts);
  const int hi = (int)((int64_t)cut.key_tiles * (part + 1) / parts);
  const int group = a.group, in_page = (1 << a.c.shift) - 1;
  const int* table = a.table + seq * a.t_sb;
  float* out = wt.w + seq * wt.sb + head * wt.sh;

  for (int j = lo + wave; j < hi; j += WNW) {
    const int key0 = j * WKT;
    // the lane's key: page, codes, scale of each 16 keys
    bool ok[2];
    float sc[2];
    int64_t at[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int pos = key0 + 16 * t;
      const int entry = ld_const(table + min(pos >> a.c.shift, a.width - 1));
      const int p = kv8_page(entry, a.c.pages);
      ok[t] = pos < s.len && p >= 0;
      if (pos < s.len && p < 0 && lane == 0) record_index_fault(a.fault, entry, a.c.pages);
      const int64_t page = max(p, 0);
      at[t] = page * a.c.k_sp + (pos & in_page) * D;
      sc[t] = a.scale_log2 * ld_const(a.c.k_scale + page * a.c.ks_sp + head * a.c.ks_sh);
    }
    const uint8_t* kp =
        a.c.k + head * a.c.k_sh + (col < 16 ? at[0] : at[1]) + (col & 15) * D + 16 * half;
    vec kf[2 * P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const u32x4 x = *(const u32x4*)(kp + 32 * p);
      kf[2 * p] = fp8x8_to<T>(x[0], x[1]);
      kf[2 * p + 1] = fp8x8_to<T>(x[2], x[3]);
    }
    f32x16 sum = f32x16{};
    // rows before this one see none of the keys
    const int first = max(0, key0 - (s.len - s.n)) * group / WRT;
    for (int r0 = first * WRT; r0 < cut.rows; r0 += WRT) {
      const int row = r0 + col, rc = min(row, cut.rows - 1);
      const int64_t t = s.first + rc / group, h = head * group + rc % group;
      const int lim = row < cut.rows ? kv8_limit(s, rc / group) : 0;
      const uint16_t* q = a.q + t * a.q_st + h * a.q_sh + 16 * half;
      const float lse = a.lse[t * a.lse_st + h * a.lse_sh] * 1.4426950408889634f;
      f32x16 x = f32x16{};
#pragma unroll
      for (int p = 0; p < P; ++p) {
        x = AttnOp<T>::mma(kf[2 * p], *(const vec*)(q + 32 * p), x);
        x = AttnOp<T>::mma(kf[2 * p + 1], *(const vec*)(q + 32 * p + 8), x);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = key0 + 8 * (r >> 2) + 4 * half + (r & 3);
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], sc[r >> 3], -lse));
        sum[r] += key < lim ? e : 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float v = sum[r];
      v += dpp_f32<0xB1>(v);
      v += dpp_f32<0x4E>(v);
      v += dpp_f32<0x141>(v);
      v += dpp_f32<0x140>(v);
      v += __shfl_xor(v, 16, 64);
      const int key = key0 + 8 * (r >> 2) + 4 * half + (r & 3);
      if (col == r && key < s.len && ok[r >> 3]) out[key] += v;
    }
  }
}

}  // namespace
}  // namespace mi

extern "C" mi_status_t mi_kv8_weigh(const mi_tensor_t* weights, const mi_tensor_t* q,
                                    const mi_tensor_t* lse, const mi_kv8_cache_t* cache,
                                    const mi_tensor_t* block_table, const mi_tensor_t* lengths,
                                    const mi_tensor_t* starts, double scale, mi_stream_t stream) {
  using namespace mi;
  clear_error();
  const char* op = "kv8_weigh";
  Kv8Args a{};
  int64_t dim = 0;
  MI_RETURN_IF(kv8_check_cache(op, cache, &a.c, &dim));
  MI_RETURN_IF(kv8_check_queries(op, q, lse, dim, &a));
  MI_RETURN_IF(kv8_check_seqs(op, block_table, lengths, starts, q->sizes[0], &a));
  MI_RETURN_IF(kv8_check_weights(op, weights, "weights", a));
  MI_CHECK_ARG(std::isfinite(scale), "%s: scale is not finite", op);
  if (a.tokens == 0 || a.seqs == 0) return MI_OK;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.fault = index_fault_word();
  a.target = 8 * cu_count();
  a.least = 1;
  const Kv8Weights w{(float*)weights->data, weights->strides[0], weights->strides[1]};
  const dim3 grid((unsigned)(a.target + (int64_t)std::min(a.seqs, a.tokens) * a.c.heads));
  hipStream_t s = (hipStream_t)stream;
  const dim3 block(64 * WNW);
  if (q->dtype == MI_BF16 && dim == 128)
    hipLaunchKernelGGL((kv8_weigh_kernel<BF16, 128>), grid, block, 0, s, a, w);
  else if (q->dtype == MI_BF16)
    hipLaunchKernelGGL((kv8_weigh_kernel<BF16, 64>), grid, block, 0, s, a, w);
  else if (dim == 128)
    hipLaunchKernelGGL((kv8_weigh_kernel<F16, 128>), grid, block, 0, s, a, w);
  else
    hipLaunchKernelGGL((kv8_weigh_kernel<F16, 64>), grid, block, 0, s, a, w);
  return check_launch(op);
}
