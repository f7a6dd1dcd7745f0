// Adds up, per cached position and k/v head, the softmax weights that a call's
// queries gave it: weights[b, hk, j] += sum over the queries i of sequence b and
// the heads of the group of exp(scale q_i k_j - lse_i), j up to the query's own
// position.  lse is what the attention call returned, so the weights need no
// second pass over the keys' maxima, and every position is owned by one lane:
// no atomics, the same sums every time.
//
// What bounds it: a decode step reads the keys' codes once; a prompt's scores
// are one matrix product with an exp2 for each.
//   kv8_weigh_rows_kernel    few rows: a wave takes 32 keys and the rows 16 at a
//     time (S^T = K Q^T, v_mfma_f32_16x16x32, the key layout of the decode
//     attention), and adds the 16 columns by DPP.
//   kv8_weigh_prompt_kernel  many rows: a wave keeps 32 keys as operands
//     (32x32x16), the block's four waves share tiles of 64 rows in LDS, and a
//     lane adds its 16 keys' weights over all rows of its column before the 32
//     columns are added at the end.
// 32 query heads on 8 of 128: 8 sequences of 4000, a token each 10 us (34.9 MB, 3.5
// TB/s: no load of a wave's next codes is in flight while a tile is computed); 2 of
// 4333, 333 tokens each 40.5 us (560 TFLOP/s: an exp2 and two more vector
// instructions a score take twice the products' time, and 544 blocks are two a CU
// and three on some).
#include <algorithm>

#include "kv8_common.h"

namespace mi {
namespace {

struct Kv8Weights {
  float* w;
  int64_t sb, sh;
};

constexpr int WKT = 32, WNW = 4;  // keys of a wave, waves of a block

// The keys' tiles (of KT) of sequences with new tokens, weighed by their tiles of
// RT rows, in parts; a part is a range of tiles of one k/v head.
template <int RT, int KT>
struct WeighItem {
  Kv8Seq s;
  int seq, head, lo, hi, rows;

  static __device__ __forceinline__ int parts(const Kv8Seq& s, int group, int chunk) {
    const Kv8Cut c = kv8_cut(s, group, RT, KT);
    if (c.row_tiles == 0 || c.key_tiles == 0) return 0;
    const int64_t parts = ((int64_t)c.row_tiles * c.key_tiles + chunk - 1) / chunk;
    return (int)(parts < c.key_tiles ? parts : c.key_tiles);
  }
  __device__ __forceinline__ bool find(const Kv8Args& a) {
    const Kv8Lanes lanes(a);
    const int chunk =
        lanes.chunk([&](const Kv8Seq& x) { return kv8_cut(x, a.group, RT, KT).work(); });
    int place;
    if (!lanes.find(
            blockIdx.x, [&](const Kv8Seq& x) { return a.c.heads * parts(x, a.group, chunk); }, &seq,
            &s, &place))
      return false;
    const Kv8Cut cut = kv8_cut(s, a.group, RT, KT);
    // heads first: blocks go to the XCDs in turn, so with 8 heads each L2 holds the
    // queries of one
    const int n = parts(s, a.group, chunk), part = place / a.c.heads;
    head = place % a.c.heads;
    lo = (int)((int64_t)cut.key_tiles * part / n);
    hi = (int)((int64_t)cut.key_tiles * (part + 1) / n);
    rows = cut.rows;
    return true;
  }
};

// Pages of a wave's 32 keys from position key0 on: where the codes of each 16
// lie, their scale times the softmax scale, and whether they exist.
struct WeighKeys {
  bool ok[2];
  float sc[2];
  int64_t at[2];

  __device__ __forceinline__ WeighKeys(const Kv8Args& a, const Kv8Seq& s, int seq, int head,
                                       int key0, int D) {
    const int* table = a.table + seq * a.t_sb;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool in = key0 + 16 * t < s.len;
      const int pos = kv8_group_at(key0 + 16 * t, s.len);
      const int entry = ld_const(table + (pos >> a.c.shift));
      const int p = kv8_page(entry, a.c.pages);
      ok[t] = in && p >= 0;
      if (in && p < 0 && (threadIdx.x & 63) == 0) record_index_fault(a.fault, entry, a.c.pages);
      const int64_t page = max(p, 0);  // read instead, and nothing of it used
      at[t] = page * a.c.k_sp + head * a.c.k_sh + (pos & ((1 << a.c.shift) - 1)) * D;
      sc[t] = a.scale_log2 * ld_const(a.c.k_scale + page * a.c.ks_sp + head * a.c.ks_sh);
    }
  }
};

// The first row of a group that sees a key: that of the token at its position.
__device__ __forceinline__ int first_row(const Kv8Seq& s, int key, int group) {
  return kv8_clamp(key - (s.len - s.n), 0, s.n) * group;
}

template <typename T, int D>
__global__ __launch_bounds__(64 * WNW, 4) void kv8_weigh_rows_kernel(Kv8Args a, Kv8Weights wt) {
  typedef typename AttnOp<T>::vec vec;
  constexpr int RT = 16, KS = D / 32;
  if (blockIdx.x == 0)
    kv8_report_lengths(a.lengths, a.seqs, a.width << a.c.shift, a.fault);
  WeighItem<RT, WKT> it;
  if (!it.find(a)) return;
  const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4, group = a.group;
  const Kv8Seq s = it.s;
  const int past = s.len - s.n;
  float* out = wt.w + it.seq * wt.sb + it.head * wt.sh;
  vec qf[KS];
  float lse = 0.f;
  auto rows = [&](int r0) __attribute__((always_inline)) {
    const int rc = min(r0 + c, it.rows - 1);
    const int64_t t = s.first + rc / group, h = it.head * group + rc % group;
    const uint16_t* q = a.q + t * a.q_st + h * a.q_sh + 16 * g;
#pragma unroll
    for (int k = 0; k < KS; ++k) qf[k] = *(const vec*)(q + 64 * (k >> 1) + 8 * (k & 1));
    lse = a.lse[t * a.lse_st + h * a.lse_sh] * 1.4426950408889634f;
  };
  rows(0);
  for (int j = it.lo + wave; j < it.hi; j += WNW) {
    const int key0 = j * WKT;
    const WeighKeys keys(a, s, it.seq, it.head, key0, D);
    u32x4 x[2][D / 64];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        x[t][h] = *(const u32x4*)(a.c.k + keys.at[t] + c * D + 16 * g + 64 * h);
    // lane c = 4 t + i of each 16 will hold key 16 t + 4 g + i
    const int mine = key0 + 16 * (c >> 2 & 1) + 4 * g + (c & 3);
    const bool owner = c < 8 && mine < s.len && (c & 4 ? keys.ok[1] : keys.ok[0]);
    const float before = owner ? out[mine] : 0.f;
    vec kf[2][KS];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int k = 0; k < KS; ++k)
        kf[t][k] = fp8x8_to<T>(x[t][k >> 1][2 * (k & 1)], x[t][k >> 1][2 * (k & 1) + 1]);
    float sum[8] = {};
    // rows before these see none of the keys
    for (int r0 = max(0, key0 - past) * group / RT * RT; r0 < it.rows; r0 += RT) {
      if (it.rows > RT) rows(r0);
      const int row = r0 + c;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x4 acc = f32x4{};
#pragma unroll
        for (int k = 0; k < KS; ++k) acc = Mma16<T>::mma(kf[t][k], qf[k], acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 16 * t + 4 * g + i;
          const bool sees = row < it.rows && row >= first_row(s, key, group);
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i], keys.sc[t], -lse));
          sum[4 * t + i] += sees ? e : 0.f;
        }
      }
    }
    float got = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = sum[i];
      v += dpp_f32<0xB1>(v);
      v += dpp_f32<0x4E>(v);
      v += dpp_f32<0x141>(v);
      v += dpp_f32<0x140>(v);
      got = c == i ? v : got;
    }
    if (owner) out[mine] = before + got;
  }
}

// RS waves share 32 keys, each with its part of a tile's rows.
template <typename T, int D, int RS>
__global__ __launch_bounds__(64 * WNW, 3) void kv8_weigh_prompt_kernel(Kv8Args a, Kv8Weights wt) {
  typedef typename AttnOp<T>::vec vec;
  constexpr int RT = RS == 4 ? 128 : 64, KT = WKT * WNW / RS, P = D / 32, CH = D / 8;
  constexpr int U = RT / 32 / RS;  // a wave's halves of 32 rows
  constexpr int N = RT * CH / (64 * WNW);  // 16-byte pieces of a row tile a thread stages
  __shared__ __align__(16) uint16_t qs[3][RT * D];
  __shared__ __align__(16) float ls[3][RT];
  __shared__ __align__(16) uint16_t none[D];  // the query of a row that is none
  __shared__ float part[WNW][WKT];
  if (blockIdx.x == 0)
    kv8_report_lengths(a.lengths, a.seqs, a.width << a.c.shift, a.fault);
  WeighItem<RT, KT> it;
  if (!it.find(a)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int half = lane >> 5, col = lane & 31, group = a.group;
  const Kv8Seq s = it.s;
  if (tid < CH) *(u32x4*)(none + 8 * tid) = u32x4{};  // the loop's first barriers lie before its readers
  const int past = s.len - s.n;
  float* out = wt.w + it.seq * wt.sb + it.head * wt.sh;
  // A tile of up to RT rows is whole tokens' heads, or RT heads of one token where
  // the group has more: its rows lie at the same offsets from its first one in
  // every tile, so a lane's addresses cost one addition a tile.
  const int hp = min(group, RT), tp = RT / hp;
  struct RowTile {
    int t, g;  // first token and first head of the group
  };
  auto next = [&](RowTile& x) __attribute__((always_inline)) {
    x.g += RT;
    if (x.g >= group) x = {x.t + tp, 0};
  };
  auto count = [&](const RowTile& x) __attribute__((always_inline)) {
    return min(tp, s.n - x.t) * min(hp, group - x.g);
  };
  // It goes from global memory straight to LDS, 16 bytes a lane: this thread copies
  // a piece of rows tid / CH + n RPI, the one that belongs at place tid % CH of its
  // rows (the XOR swizzle repeats with the rows of a wave's copies).  Rows past the
  // last one read the first one.
  constexpr int RPI = 64 * WNW / CH;
  const int piece = 8 * (tid % CH ^ swz_k_of<D>(tid / CH & 31));
  const uint16_t* q_at[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int i = tid / CH + n * RPI;
    q_at[n] = a.q + (i / hp) * a.q_st + (i % hp) * a.q_sh + piece;
  }
  const bool has_l = wave < RT / 64;  // a lane each
  const float* l_at = a.lse + (tid / hp) * a.lse_st + (tid % hp) * a.lse_sh;
  // places in LDS once: a cast of the pointers in the loop costs more than the copies
  const uint32_t q_to = lds_place(qs[0]) + wave * 64 * 16, l_to = lds_place(ls[0]) + wave * 64 * 4;
  auto copy = [&](const RowTile& x, int buf) __attribute__((always_inline)) {
    const int64_t token = s.first + x.t, h = it.head * group + x.g;
    const int64_t at = token * a.q_st + h * a.q_sh;
    const int64_t l = token * a.lse_st + h * a.lse_sh;
    const uint32_t to = q_to + buf * RT * D * 2;
    const int rows = count(x);
    if (rows == RT) {
#pragma unroll
      for (int n = 0; n < N; ++n) lds_copy16_at(q_at[n] + at, to + n * 64 * WNW * 16);
      if (has_l) lds_copy4_at(l_at + l, l_to + buf * RT * 4);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n)
        lds_copy16_at((tid / CH + n * RPI < rows ? q_at[n] : a.q + piece) + at,
                      to + n * 64 * WNW * 16);
      if (has_l) lds_copy4_at((tid < rows ? l_at : a.lse) + l, l_to + buf * RT * 4);
    }
  };

  for (int j = it.lo; j < it.hi; ++j) {
    const int key0 = j * KT + wave / RS * WKT;
    const WeighKeys keys(a, s, it.seq, it.head, key0, D);
    const uint8_t* kp = a.c.k + (col < 16 ? keys.at[0] : keys.at[1]) + (col & 15) * D + 16 * half;
    vec kf[2 * P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const u32x4 x = *(const u32x4*)(kp + 32 * p);
      kf[2 * p] = fp8x8_to<T>(x[0], x[1]);
      kf[2 * p + 1] = fp8x8_to<T>(x[2], x[3]);
    }
    // the lane's own weight: one read and one write, not one for each product
    const int mine = key0 + 8 * (col >> 2) + 4 * half + (col & 3);
    const bool owner = wave % RS == 0 && col < 16 && mine < s.len &&
                       (col < 8 ? keys.ok[0] : keys.ok[1]);
    const float before = owner ? out[mine] : 0.f;
    f32x16 sum = f32x16{};
    // the block's first key is seen from its own token on, all keys of the wave by
    // the tokens from `full` on
    RowTile now = {max(0, j * KT - past) / tp * tp, 0}, ahead = now;
    const int full = key0 + WKT - 1 - past;
    __syncthreads();  // the buffers' last readers
    copy(ahead, 0);
    next(ahead);
    if (ahead.t < s.n) copy(ahead, 1);
    for (int buf = 0; now.t < s.n; next(now), buf = buf == 2 ? 0 : buf + 1) {
      // this wave's copies of the tile, with those of the next one still on the way
      if (ahead.t >= s.n) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      else if (wave < RT / 64) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N + 1) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
      __syncthreads();
      if (ahead.t < s.n) next(ahead);
      if (ahead.t < s.n) copy(ahead, buf == 0 ? 2 : buf - 1);
      if (key0 >= s.len) continue;
      const int rows = count(now);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = 32 * (wave % RS * U + u) + col;
        // a row that is none weighs nothing; its place in the tile holds another
        // row's query, and one that is not finite would be no 0 even with this lse
        const uint16_t* q = row < rows ? qs[buf] + row * D : none;
        const float lse = row < rows ? ls[buf][row] * 1.4426950408889634f : INFINITY;
        f32x16 x = f32x16{};
#pragma unroll
        for (int p = 0; p < P; ++p) {
          // d = 32 p + 16 half + 0 .. 15: pieces 4 p + 2 half and the next
          const int ch = 4 * p + 2 * half, sw = swz_k_of<D>(col);
          x = AttnOp<T>::mma(kf[2 * p], *(const vec*)(q + 8 * (ch ^ sw)), x);
          x = AttnOp<T>::mma(kf[2 * p + 1], *(const vec*)(q + 8 * ((ch + 1) ^ sw)), x);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
          x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], keys.sc[r >> 3], -lse));
        if (now.t >= full) {
#pragma unroll
          for (int r = 0; r < 16; ++r) sum[r] += x[r];
        } else {
          // how many of the lane's keys, from its first one on, the row's token sees
          const int seen = past + now.t + row / hp - (key0 + 4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r) sum[r] += 8 * (r >> 2) + (r & 3) <= seen ? x[r] : 0.f;
        }
      }
    }
    float got = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float v = sum[r];
      v += dpp_f32<0xB1>(v);
      v += dpp_f32<0x4E>(v);
      v += dpp_f32<0x141>(v);
      v += dpp_f32<0x140>(v);
      v = row_sum(v);
      got = col == r ? v : got;
    }
    if constexpr (RS > 1) {  // added in the order of the rows' parts
      if (col < 16) part[wave][16 * half + col] = got;
      __syncthreads();
      if (wave % RS == 0 && col < 16)
#pragma unroll
        for (int i = 1; i < RS; ++i) got += part[wave + i][16 * half + col];
    }
    if (owner) out[mine] = before + got;
  }
}

template <typename T, int D>
mi_status_t run_weigh(Kv8Args& a, const Kv8Weights& w, hipStream_t s) {
  const int some = std::min(a.seqs, a.tokens);
  const dim3 block(64 * WNW);
  // blocks of few rows: four a CU at once
  const bool few = (int64_t)a.tokens * a.group <= (int64_t)32 * some;
  a.plan = {4 * cu_count(), 0, 1, 4 * cu_count()};
  const dim3 grid((unsigned)(a.plan.many + some * a.c.heads));
  const int64_t keys = (int64_t)a.width << a.c.shift, tile = WKT * WNW;
  const int64_t blocks = some * a.c.heads * ((keys + tile - 1) / tile);
  if (few) hipLaunchKernelGGL((kv8_weigh_rows_kernel<T, D>), grid, block, 0, s, a, w);
  // (by the table's width, as wide as the longest sequence in these times)  A block
  // walks all rows, and where the blocks of 128 keys leave CUs idle, smaller
  // ones with waves that share the rows walk faster, at twice (four times) the
  // copies.  us, one, two and four waves to 32 keys, 32 query heads on 8 of 128: 64
  // tokens behind 500 (40 blocks of 128 keys) 9.6 / 8.9 / 8.9, 333 behind 1000 (88)
  // 25.5 / 21.3 / 29, behind 4000 (272) 28.5 / 27.4 / 67, 2 x 333 behind 4000 (544) 42
  // / 65 / 122; 5 heads on one of 64, 5 x 301 behind 721 (40) 27.5 / 21.2 / 14.4.
  else if (4 * blocks <= cu_count())
    hipLaunchKernelGGL((kv8_weigh_prompt_kernel<T, D, 4>), grid, block, 0, s, a, w);
  else if (blocks <= cu_count())
    hipLaunchKernelGGL((kv8_weigh_prompt_kernel<T, D, 2>), grid, block, 0, s, a, w);
  else
    hipLaunchKernelGGL((kv8_weigh_prompt_kernel<T, D, 1>), grid, block, 0, s, a, w);
  return check_launch("kv8_weigh");
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
  const Kv8Weights w{(float*)weights->data, weights->strides[0], weights->strides[1]};
  hipStream_t s = (hipStream_t)stream;
  if (q->dtype == MI_BF16) return dim == 128 ? run_weigh<BF16, 128>(a, w, s) : run_weigh<BF16, 64>(a, w, s);
  return dim == 128 ? run_weigh<F16, 128>(a, w, s) : run_weigh<F16, 64>(a, w, s);
}
