// Attention of a few query rows per sequence (decode steps, drafted tokens)
// over the 8-bit cache: o = softmax(scale q k^T) v over the positions up to the
// query's own, D = 64 or 128, bf16 / f16 queries.
//
// What bounds it: the codes are read once from HBM, one byte an element; the
// G query heads of a k/v head times the sequence's new tokens share the read as
// the rows of one MFMA tile (16 NB).
//
//   S^T = K Q^T   16 keys x 32 d (v_mfma_f32_16x16x32): lane (c, g) = (lane % 16,
//                 lane / 16) loads 16 codes of key c at d = 64 h + 16 g: two
//                 operands of 8, converted in registers (e4m3 is exact in both
//                 16-bit types).  Which d an operand's place means is free as
//                 long as Q's agree.
//   O^T = V^T P^T accumulator (row c, keys 4 g + i) of two S^T tiles is the P^T
//                 operand as it stands.  V^T needs 8 keys of one d per lane: the
//                 lane loads D / 16 codes of each of its 8 keys, and the bytes
//                 are turned around by v_perm before the conversion, so neither
//                 K nor V passes through LDS.
//
// The scales multiply scores (K) and weights (V) in fp32: one scalar per 16
// keys, since a page holds a multiple of 16.  P is rounded to the input type; for
// f16 as Kv8Weight says.
//
// Work: kv8_plan cuts each sequence's keys into parts so that all sequences
// together make a few blocks per CU, whatever their lengths; the device reads
// the lengths, so a captured call follows them.  A block's waves take 32-key
// tiles in turn, never wait for each other, and are merged through LDS; parts
// are merged by kv8_combine_kernel in a fixed order.  32 query heads on 8 of 128:
// 32 sequences of 4000 to 16000 118 us (648 MB, 5.5 TB/s), 8 of 4000 16 us and
// the merge's 4 (65.7 MB, 3.3 TB/s together), 1 of 301 7 us.
#include <algorithm>

#include "kv8_combine.h"

namespace mi {
namespace {

constexpr int RKT = 32;  // keys of a wave's tile

template <int D>
struct RowsTile {
  u32x4 k[2][D / 64];       // [16-key half][64-d piece]
  uint32_t v[8][D / 64];    // [key of the lane][4-d piece]
  float ks[2], vs[2];
  bool ok[2];               // the 16-key half lies in a page
};

template <typename T, int D, int NB, int NW, bool ONCE>
__device__ __forceinline__ void rows_item(const Kv8Args& a) {
  typedef typename AttnOp<T>::vec vec;
  typedef Kv8Weight<T> Wt;
  constexpr bool F = Wt::F;
  constexpr int RT = 16 * NB, KS = D / 32, DT = D / 16, W = D / 64;
  __shared__ float red[NW * NB * DT * 4 * 64];
  __shared__ float ml[NW][RT][3];

  Kv8Item it;
  if (!kv8_item<RT, RKT, false>(a, blockIdx.x, &it)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int group = a.group, rows = it.cut.rows, row0 = it.tile * RT, len = it.s.len;

  vec qf[NB][KS];
  int lim[NB];
  int64_t q_at[NB], o_at[NB], l_at[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int row = row0 + 16 * nb + c, rc = min(row, rows - 1);
    const int64_t t = it.s.first + rc / group, h = it.head * group + rc % group;
    lim[nb] = row < rows ? kv8_limit(it.s, rc / group) : 0;
    q_at[nb] = t * a.q_st + h * a.q_sh;
    o_at[nb] = t * a.o_st + h * a.o_sh;
    l_at[nb] = t * a.lse_st + h * a.lse_sh;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      qf[nb][k] = *(const vec*)(a.q + q_at[nb] + 64 * (k >> 1) + 16 * g + 8 * (k & 1));
  }
  // what the tile's first and last rows see
  const int least = kv8_limit(it.s, row0 / group);
  const int most = kv8_limit(it.s, (min(rows, row0 + RT) - 1) / group);
  const int tiles = (most + RKT - 1) / RKT;
  const int lo = (int)((int64_t)tiles * it.part / it.parts);
  const int hi = (int)((int64_t)tiles * (it.part + 1) / it.parts);

  const int shift = a.c.shift, in_page = (1 << shift) - 1;
  const int* table = a.table + it.seq * a.t_sb;
  const uint8_t* kc = a.c.k + it.head * a.c.k_sh + c * D + 16 * g;
  const uint8_t* vc = a.c.v + it.head * a.c.v_sh + 4 * g * D + W * 4 * c;
  const float* ksc = a.c.k_scale + it.head * a.c.ks_sh;
  const float* vsc = a.c.v_scale + it.head * a.c.vs_sh;
  auto entries = [&](int j, int* e) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
      e[t] = ld_const(table + min((j * RKT + 16 * t) >> shift, a.width - 1));
  };
  // codes that one block reads once are not kept in the caches
  auto code = [](const auto* p) __attribute__((always_inline)) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    else return *p;
  };
  auto load = [&](int j, const int* e, RowsTile<D>& x) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int pos = j * RKT + 16 * t;
      const int p = kv8_page(e[t], a.c.pages);
      x.ok[t] = pos < len && p >= 0;
      if (pos < len && p < 0 && lane == 0) record_index_fault(a.fault, e[t], a.c.pages);
      const int64_t page = max(p, 0);  // a page that is not there: page 0 is read, and nothing of it used
      const int off = (pos & in_page) * D;
      const uint8_t* kp = kc + page * a.c.k_sp + off;
      const uint8_t* vp = vc + page * a.c.v_sp + off;
#pragma unroll
      for (int h = 0; h < W; ++h) x.k[t][h] = code((const u32x4*)(kp + 64 * h));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (W == 2) {
          const u32x2 y = code((const u32x2*)(vp + i * D));
          x.v[4 * t + i][0] = y[0];
          x.v[4 * t + i][1] = y[1];
        } else {
          x.v[4 * t + i][0] = code((const uint32_t*)(vp + i * D));
        }
      }
      x.ks[t] = ld_const(ksc + page * a.c.ks_sp);
      x.vs[t] = ld_const(vsc + page * a.c.vs_sp);
    }
  };

  f32x4 o[NB][DT];
  float m_run[NB], l_run[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m_run[nb] = -INFINITY;
    l_run[nb] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[nb][i] = f32x4{};
  }
  float vref = 0x1p-126f;  // f16: o holds sums over it

  auto compute = [&](int j, RowsTile<D>& x) __attribute__((always_inline)) {
    const bool edge = j * RKT + RKT > least || !x.ok[0] || !x.ok[1];
    float vs[2] = {x.ok[0] ? x.vs[0] : 0.f, x.ok[1] ? x.vs[1] : 0.f};
    bool apart[2] = {false, false};
    if constexpr (F) {
      const float top = wave_uniform_f32(Wt::ref(fmaxf(vs[0], vs[1])));
      if (top > vref) {
        const float r = wave_uniform_f32(vref * __builtin_amdgcn_rcpf(top));
        vref = top;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < DT; ++i) o[nb][i] *= r;
      }
      const float inv = __builtin_amdgcn_rcpf(vref);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        vs[t] = wave_uniform_f32(vs[t] * inv);
        apart[t] = Wt::apart(vs[t]);
      }
    }
    vec kf[2][KS];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int k = 0; k < KS; ++k)
        kf[t][k] = fp8x8_to<T>(x.k[t][k >> 1][2 * (k & 1)], x.k[t][k >> 1][2 * (k & 1) + 1]);
    f32x8 p[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      f32x8 s;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x4 acc = f32x4{};
#pragma unroll
        for (int k = 0; k < KS; ++k) acc = Mma16<T>::mma(kf[t][k], qf[nb][k], acc);
        const float sc = a.scale_log2 * x.ks[t];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * t + i] = acc[i] * sc;
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = j * RKT + 16 * (i >> 2) + 4 * g + (i & 3);
          s[i] = key < lim[nb] && x.ok[i >> 2] ? s[i] : -INFINITY;
        }
      }
      float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                       fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
      mx = half_max(row_max(mx));
      mx = Wt::top(mx);
      if (mx > m_run[nb]) {
        const float corr = __builtin_amdgcn_exp2f(m_run[nb] - mx);
        m_run[nb] = mx;
        l_run[nb] *= corr;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[nb][i] *= corr;
      }
      const float m_use = Wt::offset(m_run[nb]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[nb][i] = __builtin_amdgcn_exp2f(s[i] - m_use);
        l_run[nb] += p[nb][i];
      }
    }
    // d = 4 w + 2 h and the next of the lane's 8 keys, as operands
    auto values = [&](int w, int h, vec* vf) __attribute__((always_inline)) {
      union {
        typename Fp8To<T>::pair p[4];
        vec v;
      } u[2];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        // the two bytes of keys 2 q and 2 q + 1, side by side
        const uint32_t e = __builtin_amdgcn_perm(x.v[2 * q + 1][w], x.v[2 * q][w],
                                                 h == 0 ? 0x05010400u : 0x07030602u);
        u[0].p[q] = Fp8To<T>::template cvt<false>(e);
        u[1].p[q] = Fp8To<T>::template cvt<true>(e);
      }
      vf[0] = u[0].v;
      vf[1] = u[1].v;
    };
    if (j * RKT + RKT > len || !x.ok[0] || !x.ok[1] || apart[0] || apart[1]) {
      // what lies behind the last token, or on a page that is not there, may
      // hold anything, NaN codes too: 0 x NaN must not come in
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = j * RKT + 16 * (i >> 2) + 4 * g + (i & 3);
#pragma unroll
        for (int w = 0; w < W; ++w)
          x.v[i][w] = key < len && x.ok[i >> 2] ? x.v[i][w] : 0u;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!apart[t]) continue;
        // 16 keys by themselves, the other half's weights as 0
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          f32x8 half = f32x8{};
#pragma unroll
          for (int i = 4 * t; i < 4 * t + 4; ++i) half[i] = p[nb][i];
          const vec pk = __builtin_convertvector(half, vec);
#pragma unroll
          for (int w = 0; w < W; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              vec vf[2];
              values(w, h, vf);
#pragma unroll
              for (int e = 0; e < 2; ++e)
                o[nb][4 * w + 2 * h + e] += Mma16<T>::mma(vf[e], pk, f32x4{}) * vs[t];
            }
        }
        vs[t] = 0.f;
      }
    }
    vec pk[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[nb][i] *= vs[i >> 2];
      pk[nb] = __builtin_convertvector(p[nb], vec);
    }
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        vec vf[2];
        values(w, h, vf);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            o[nb][4 * w + 2 * h + e] = Mma16<T>::mma(vf[e], pk[nb], o[nb][4 * w + 2 * h + e]);
      }
  };

  // this wave's tiles lo + wave, then every NW-th, their table entries one step
  // ahead; the other waves of the SIMD cover the loads
  int j = lo + wave;
  if (j < hi) {
    RowsTile<D> x;
    int e[2];
    entries(j, e);
    for (; j < hi; j += NW) {
      load(j, e, x);
      entries(j + NW, e);
      compute(j, x);
    }
  }

  // merge the waves: common max, scaled sums, O added in wave order
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float l = half_sum(row_sum(l_run[nb])) * Wt::UNIT;
    if (g == 0) {
      ml[wave][16 * nb + c][0] = m_run[nb];
      ml[wave][16 * nb + c][1] = l;
    }
  }
  __syncthreads();
  float M[NB], l[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    M[nb] = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M[nb] = fmaxf(M[nb], ml[w][16 * nb + c][0]);
    const float mu = M[nb] == -INFINITY ? 0.f : M[nb];
    l[nb] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w)
      l[nb] += ml[w][16 * nb + c][1] * __builtin_amdgcn_exp2f(ml[w][16 * nb + c][0] - mu);
    float own = __builtin_amdgcn_exp2f(m_run[nb] - mu);
    if constexpr (F) own *= vref * Wt::UNIT;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        red[(((wave * NB + nb) * DT + i) * 4 + r) * 64 + lane] = o[nb][i][r] * own;
  }
  __syncthreads();
  const bool whole = it.parts == 1;
  const int64_t part0 = (int64_t)blockIdx.x * RT;
  if (!whole && (int)blockIdx.x >= a.slots) return;
  // run (nb, r, i4): the four d = D / 4 g + D / 16 r + 4 i4 .. + 3 of the lane's row
  for (int run = wave; run < NB * DT; run += NW) {
    const int nb = run / DT, r = run % DT / (DT / 4), i4 = run % (DT / 4);
    f32x4 x = f32x4{};
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] += red[(((w * NB + nb) * DT + 4 * i4 + e) * 4 + r) * 64 + lane];
    const int d = D / 4 * g + D / 16 * r + 4 * i4;
    const int row = 16 * nb + c;
    const float ln = nb == 0 ? l[0] : l[NB - 1];
    if (row0 + row >= rows) continue;
    if (whole) {
      typedef typename AttnOp<T>::elem E;
      typedef E e4 __attribute__((ext_vector_type(4)));
      const float inv = ln == 0.f ? 0.f : 1.0f / ln;  // no visible key: 0
      *(e4*)(a.o + (nb == 0 ? o_at[0] : o_at[NB - 1]) + d) = __builtin_convertvector(x * inv, e4);
    } else {
      *(f32x4*)(a.part_o + (part0 + row) * D + d) = x;
    }
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int row = 16 * nb + c;
    if (wave != nb % NW || g != 0 || row0 + row >= rows) continue;
    if (whole) {
      a.lse[l_at[nb]] = l[nb] == 0.f ? -INFINITY
                                     : (M[nb] + __builtin_amdgcn_logf(l[nb])) * 0.6931471805599453f;
    } else {
      a.part_ml[(part0 + row) * 2] = M[nb];
      a.part_ml[(part0 + row) * 2 + 1] = l[nb];
    }
  }
}

template <typename T, int D, int NB, int NW, bool ONCE>
__global__ __launch_bounds__(64 * NW, 4) void kv8_rows_kernel(Kv8Args a) {
  rows_item<T, D, NB, NW, ONCE>(a);
  kv8_rest<D>(a);
}

template <typename T, int D>
mi_status_t run_rows(Kv8Args& a, hipStream_t s) {
  constexpr int NB = 1, NW = 8;
  // (The rules here and in mi_kv8_attention go by the table's width, since the host
  // does not know the lengths; the times are those of tables as wide as the longest
  // sequence.)  Two blocks of eight waves per CU, and twice as many parts where they are long
  // enough that the last ones to end count (32 sequences of 4000 to 16000: 130 ->
  // 119 us).  A part is at least a tile per wave, and short sequences stay whole,
  // since the merge is a launch of 4 us: up to 1024 positions (1 of 300: 13 -> 8
  // us), or 4096 where a row tile and head for each block fill seven eighths of
  // their rounds over the CUs (32 x 8 of 4000: 52 -> 45, of 1000 to 4000 43 -> 37,
  // 56 x 8 of 3000 69 -> 63; but 40 x 8 of 4000 62 -> 76, of 2000 38 -> 40).
  const int cus = cu_count();
  const int64_t tiles = (((int64_t)a.width << a.c.shift) + RKT - 1) / RKT;
  // if the sequences' new tokens are about as many in each
  const int64_t some = std::min(a.seqs, a.tokens), rows = (int64_t)a.tokens * a.group;
  const int64_t blocks = some > 0 ? some * ((rows / some + 16 * NB - 1) / (16 * NB)) * a.c.heads : 0;
  const int64_t rounds = (blocks + cus - 1) / cus;
  const int whole = blocks > 0 && blocks * 8 >= rounds * cus * 7 ? 16 * NW : 4 * NW;
  // each sequence's last part is half a one on the average: room for them, or a few
  // blocks start when the others end (12 x 8 of 4000: 29 -> 24 us, 16 x 8 of 4000 to
  // 8000 40 -> 35; 24 x 16 of 2000, more than the CUs: 34 -> 39)
  const int few = 2 * cus - (blocks < cus ? (int)blocks / 2 : 0);
  a.plan = {few, 64, tiles <= whole ? whole : NW, 4 * cus};
  // one row tile a sequence: its codes are read once
  if (rows <= 16 * NB * some)
    return kv8_launch<T, D, 16 * NB, RKT, false>(a, kv8_rows_kernel<T, D, NB, NW, true>, 64 * NW, s);
  return kv8_launch<T, D, 16 * NB, RKT, false>(a, kv8_rows_kernel<T, D, NB, NW, false>, 64 * NW, s);
}

}  // namespace
}  // namespace mi

extern "C" mi_status_t mi_kv8_attention(const mi_tensor_t* out, const mi_tensor_t* lse,
                                        const mi_tensor_t* q, const mi_kv8_cache_t* cache,
                                        const mi_tensor_t* block_table, const mi_tensor_t* lengths,
                                        const mi_tensor_t* starts, double scale, int32_t fill_rest,
                                        mi_stream_t stream) {
  using namespace mi;
  clear_error();
  const char* op = "kv8_attention";
  Kv8Args a{};
  int64_t dim = 0;
  MI_RETURN_IF(kv8_check_cache(op, cache, &a.c, &dim));
  MI_RETURN_IF(kv8_check_queries(op, q, lse, dim, &a));
  MI_RETURN_IF(validate(out, "out"));
  MI_CHECK_ARG(out->dtype == q->dtype && out->ndim == 3 && out->sizes[0] == q->sizes[0] &&
                   out->sizes[1] == q->sizes[1] && out->sizes[2] == dim,
               "%s: out must have q's shape and type", op);
  if (out->strides[2] != 1 || out->strides[0] % 8 != 0 || out->strides[1] % 8 != 0 ||
      (uintptr_t)out->data % 16 != 0)
    MI_FAIL(MI_ERR_UNSUPPORTED, "%s: rows of out must be dense and 16-byte aligned", op);
  MI_CHECK_ARG(kv8_apart(out->sizes[0], out->strides[0], out->sizes[1], out->strides[1], dim) &&
                   kv8_apart(lse->sizes[0], lse->strides[0], lse->sizes[1], lse->strides[1], 1),
               "%s: rows of out or lse overlap", op);
  MI_RETURN_IF(kv8_check_seqs(op, block_table, lengths, starts, q->sizes[0], &a));
  MI_CHECK_ARG(std::isfinite(scale), "%s: scale is not finite", op);
  if (a.tokens == 0) return MI_OK;
  a.o = (uint16_t*)out->data;
  a.o_st = out->strides[0];
  a.o_sh = out->strides[1];
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.fill_rest = fill_rest;
  a.fault = index_fault_word();
  hipStream_t s = (hipStream_t)stream;
  // The kernel here reads a sequence's keys once for each 16 rows, the prompt
  // kernel once for 128, but with more to do around it.  us, this and the prompt
  // kernel, 32 query heads on 8, D = 128: 8 sequences of 3000, 8 new tokens (32
  // rows) each 21 / 46, 16: 29 / 49, 24: 43 / 39; 32 of 8000, 16 tokens each 196 /
  // 200; 1 of 2000, 64 tokens 18 / 24; 1 of 16000, 24 tokens 37 / 31.
  const int64_t rows = (int64_t)a.tokens * a.group;
  if (rows > (int64_t)64 * std::min(a.seqs, a.tokens) &&
      rows * a.c.heads * ((int64_t)a.width << a.c.shift) > (int64_t)1 << 23)
    return kv8_prompt(a, dim, q->dtype == MI_F16, s);
  if (q->dtype == MI_BF16) return dim == 128 ? run_rows<BF16, 128>(a, s) : run_rows<BF16, 64>(a, s);
  return dim == 128 ? run_rows<F16, 128>(a, s) : run_rows<F16, 64>(a, s);
}
