// Attention of many query rows per sequence (pieces of prompts) over the 8-bit
// cache.
//
// What bounds it: 4 D flops per query row and key on the matrix instructions, and
// more time of exp2, maxima and sums on the vector unit, one after the other: the
// barrier of a tile keeps a SIMD's waves in the same phase.  32 query heads on 8 of
// 128: 2048 tokens behind 14000 546 us (924 TFLOP/s where a large product reaches
// 1426; matrix instructions 4.8e5 and vector ones 6.5e5 cycles a SIMD of 1.15e6),
// 2783 tokens of four sequences behind 359 to 823 82 us (527: 704 blocks on 512
// places).
//   A block takes 32 NW query rows of one k/v head (the group's heads of
// consecutive tokens), a wave 32 of them, and walks the keys in tiles of 64:
//   S^T = K Q^T, O^T = V^T P^T (v_mfma_f32_32x32x16), P^T taken from the S^T
//   accumulators as they stand.
// The codes of the next tile are loaded into registers while a tile is
// computed, converted once per block (e4m3 is exact in both 16-bit types) and
// written to the other of two LDS buffers: K by rows, V transposed, both in
// 16-byte pieces whose places are XORed so that neither the writes nor the
// fragment reads conflict.  One barrier a tile.
// A key's scale multiplies its scores inside the exponent's FMA (one scalar per
// 16 keys); a value's scale multiplies the weights, and only where it differs
// from the one that the accumulators are relative to (Kv8Weight).
#include <algorithm>

#include "kv8_combine.h"

namespace mi {
namespace {

constexpr int PKT = 64;  // keys per tile

template <int D>
__device__ __forceinline__ int swz_vt(int d) {
  return ((d >> 1) & 7) ^ ((d >> 4) & 1);
}

template <typename T, int D, int NW>
__device__ __forceinline__ void prompt_item(const Kv8Args& a) {
  typedef typename AttnOp<T>::vec vec;
  typedef Kv8Weight<T> Wt;
  constexpr int RT = 32 * NW, NT = 64 * NW;
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int VU = D / 4 * 8;              // V units: 4 d of 8 keys
  constexpr int KU = PKT * D / 16;           // K units: 16 d of a key
  constexpr int KN = NW == 8 ? KU / 256 : KU / NT;  // a thread's K units
  __shared__ __align__(16) uint16_t kt[2][PKT * D];
  __shared__ __align__(16) uint16_t vt[2][PKT * D];
  __shared__ __align__(16) float scales[2][8];  // of a tile's 16-key groups: scores', values'
  // of a tile: the largest V scale and the least that is not 0, the scale of all
  // groups or -1, and as an int, bit g: group g does not exist
  __shared__ __align__(16) float about[2][4];

  Kv8Item it;
  if (!kv8_item<RT, PKT, true>(a, blockIdx.x, &it)) return;
  it.tile = it.cut.row_tiles - 1 - it.tile;  // the farthest-seeing rows first
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int group = a.group, rows = it.cut.rows, len = it.s.len;
  const int row0 = it.tile * RT, wrow0 = row0 + 32 * wave;

  // positions that the block's rows see, and this wave's: all, and any
  const int most = kv8_limit(it.s, (min(rows, row0 + RT) - 1) / group);
  const int w_least = wrow0 < rows ? kv8_limit(it.s, wrow0 / group) : 0;
  const int w_most = wrow0 < rows ? kv8_limit(it.s, (min(rows, wrow0 + 32) - 1) / group) : 0;
  const int tiles = (most + PKT - 1) / PKT;
  const int lo = (int)((int64_t)tiles * it.part / it.parts);
  const int hi = (int)((int64_t)tiles * (it.part + 1) / it.parts);

  const float scale = fabsf(a.scale_log2);
  const int shift = a.c.shift, in_page = (1 << shift) - 1;
  const int* table = a.table + it.seq * a.t_sb;
  const uint8_t* kc = a.c.k + it.head * a.c.k_sh;
  const uint8_t* vc = a.c.v + it.head * a.c.v_sh;
  const float* ksc = a.c.k_scale + it.head * a.c.ks_sh;
  const float* vsc = a.c.v_scale + it.head * a.c.vs_sh;
  auto entry_of = [&](int pos) __attribute__((always_inline)) {
    return table[min(pos >> shift, a.width - 1)];
  };

  // this thread's units of a tile
  const bool has_v = tid < VU, has_k = NW != 8 || tid >= 256;
  const int ku = NW == 8 ? tid - 256 : tid;
  const int v_dc = tid % (D / 4), v_kg = tid / (D / 4) & 7;
  const int v_key = 16 * (v_kg >> 1) + 4 * (v_kg & 1);  // then + 1, 2, 3, 8, 9, 10, 11
  u32x4 kr[KN];
  uint32_t vr[8];
  int ke[KN], ve = 0;
  // one thread a 16-key group brings its scales: they come by the way of the
  // codes, since scalar loads return out of order and would make every wait for
  // an LDS read a wait for all of them
  int se = 0;
  float s_k = 0.f, s_v = 0.f;
  bool s_ok = true;
  int v_left = 0;  // of this thread's 8 keys those nearer than this exist
  auto entries = [&](int j) __attribute__((always_inline)) {
    if (has_k) {
#pragma unroll
      for (int n = 0; n < KN; ++n)
        ke[n] = entry_of(j * PKT + (ku + n * (NW == 8 ? 256 : NT)) / (D / 16));
    }
    if (has_v) ve = entry_of(j * PKT + v_key);
    if (tid < 4) se = entry_of(j * PKT + 16 * tid);
  };
  auto load = [&](int j) __attribute__((always_inline)) {
    const int key0 = j * PKT;
    if (has_k) {
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        const int u = ku + n * (NW == 8 ? 256 : NT);
        const int pos = key0 + u / (D / 16);
        const int64_t page = max(kv8_page(ke[n], a.c.pages), 0);
        kr[n] = *(const u32x4*)(kc + page * a.c.k_sp + (pos & in_page) * D + 16 * (u % (D / 16)));
      }
    }
    if (has_v) {
      const int pos = key0 + v_key;
      const int p = kv8_page(ve, a.c.pages);
      const uint8_t* vp = vc + max(p, 0) * a.c.v_sp + (pos & in_page) * D + 4 * v_dc;
      v_left = p < 0 ? 0 : len - pos;
#pragma unroll
      for (int i = 0; i < 8; ++i) vr[i] = *(const uint32_t*)(vp + (i < 4 ? i : i + 4) * D);
    }
    if (tid < 4) {
      const int p = kv8_page(se, a.c.pages);
      const bool in = key0 + 16 * tid < len;
      s_ok = in && p >= 0;
      if (in && p < 0) record_index_fault(a.fault, se, a.c.pages);
      s_k = ksc[max(p, 0) * a.c.ks_sp];
      s_v = vsc[max(p, 0) * a.c.vs_sp];
    }
  };
  auto store = [&](int buf) __attribute__((always_inline)) {
    if (tid < 4) {
      const float k = scale * s_k;
      // masked scores stay -inf when multiplied by it
      scales[buf][tid] = !s_ok || k < 0x1p-100f ? 0x1p-100f : k;
      const float v = s_ok ? s_v : 0.f;
      scales[buf][4 + tid] = v;
      const int gone = (int)__ballot(!s_ok);
      const bool even = __ballot(v == wave_uniform_f32(v)) == 15;
      float large = fmaxf(v, dpp_f32<0xB1>(v));
      large = fmaxf(large, dpp_f32<0x4E>(large));
      float least = v > 0.f ? v : large;
      least = fminf(least, dpp_f32<0xB1>(least));
      least = fminf(least, dpp_f32<0x4E>(least));
      if (tid == 0)
        *(f32x4*)about[buf] = f32x4{large, least, even ? v : -1.f, __builtin_bit_cast(float, gone)};
    }
    if (has_k) {
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        const int u = ku + n * (NW == 8 ? 256 : NT);
        const int key = u / (D / 16), c = 2 * (u % (D / 16)), sw = swz_k_of<D>(key);
        *(vec*)(kt[buf] + key * D + 8 * (c ^ sw)) = fp8x8_to<T>(kr[n][0], kr[n][1]);
        *(vec*)(kt[buf] + key * D + 8 * ((c + 1) ^ sw)) = fp8x8_to<T>(kr[n][2], kr[n][3]);
      }
    }
    if (has_v) {
      // behind the last token, or on a page that is not there, may lie
      // anything, NaN codes too: 0 x NaN must not come in
      if (v_left < 12) {
#pragma unroll
        for (int i = 0; i < 8; ++i) vr[i] = (i < 4 ? i : i + 4) < v_left ? vr[i] : 0u;
      }
      union {
        typename Fp8To<T>::pair p[4];
        vec v;
      } vf[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t e0 = __builtin_amdgcn_perm(vr[2 * q + 1], vr[2 * q], 0x05010400u);
        const uint32_t e1 = __builtin_amdgcn_perm(vr[2 * q + 1], vr[2 * q], 0x07030602u);
        vf[0].p[q] = Fp8To<T>::template cvt<false>(e0);
        vf[1].p[q] = Fp8To<T>::template cvt<true>(e0);
        vf[2].p[q] = Fp8To<T>::template cvt<false>(e1);
        vf[3].p[q] = Fp8To<T>::template cvt<true>(e1);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 4 * v_dc + e;
        *(vec*)(vt[buf] + d * PKT + 8 * (v_kg ^ swz_vt<D>(d))) = vf[e].v;
      }
    }
  };

  f32x16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  float vref = 0x1p-126f;  // o holds sums over it

  if (lo < hi) {
    entries(lo);
    load(lo);
  }
  const int row = wrow0 + col, rc = min(row, rows - 1);
  const int64_t tok = it.s.first + rc / group, head = it.head * group + rc % group;
  const int lim = row < rows ? kv8_limit(it.s, rc / group) : 0;
  vec qf[KS];
#pragma unroll
  for (int t = 0; t < KS; ++t) {
    qf[t] = *(const vec*)(a.q + tok * a.q_st + head * a.q_sh + 16 * t + 8 * half);
  }
  if (a.scale_log2 < 0.f) {  // scales below are positive
#pragma unroll
    for (int t = 0; t < KS; ++t) qf[t] = -qf[t];
  }
  // tile j's codes are loaded two steps before it is computed and converted one
  // step before, their table entries a step earlier still
  if (lo < hi) {
    entries(lo + 1);
    store(0);
    load(lo + 1);
    entries(lo + 2);
  }
  for (int j = lo; j < hi; ++j) {
    const int buf = (j - lo) & 1, key0 = j * PKT;
    __syncthreads();
    if (j + 1 < hi) store(buf ^ 1);
    if (j + 2 < hi) load(j + 2);
    entries(j + 3);
    if (key0 < w_most) {
      const f32x4 sc = *(const f32x4*)scales[buf], vs = *(const f32x4*)(scales[buf] + 4);
      const f32x4 ab = *(const f32x4*)about[buf];
      const float large = ab[0], least = ab[1], even = ab[2], bits = ab[3];
      const int gone = wave_uniform(__builtin_bit_cast(int, bits));
      f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const uint16_t* kp = kt[buf] + col * D + 8 * ((2 * t + half) ^ swz_k_of<D>(col));
        s[0] = AttnOp<T>::mma(*(const vec*)kp, qf[t], s[0]);
        s[1] = AttnOp<T>::mma(*(const vec*)(kp + 32 * D), qf[t], s[1]);
      }
      // fragments read 6 ahead of their products
      __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      // accumulator r of half st is key 32 st + 8 (r / 4) + 4 half + r % 4, of
      // the 16-key group 2 st + r / 8
      if (key0 + PKT > w_least || gone != 0) {
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = key0 + 32 * st + 8 * (r >> 2) + 4 * half + (r & 3);
            s[st][r] = key < lim && !(gone >> (2 * st + (r >> 3)) & 1) ? s[st][r] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float x = s[g >> 1][8 * (g & 1)];
#pragma unroll
        for (int r = 1; r < 8; ++r) x = fmaxf(x, s[g >> 1][8 * (g & 1) + r]);
        mx = fmaxf(mx, x * sc[g]);
      }
      mx = Wt::top(half_max(mx));
      const float top = wave_uniform_f32(Wt::ref(large));
      float corr = 1.f;
      if (top > vref) {
        corr = vref * __builtin_amdgcn_rcpf(top);
        vref = top;
      }
      if (mx > m_run || corr != 1.f) {
        const float grow = mx > m_run ? __builtin_amdgcn_exp2f(m_run - mx) : 1.f;
        m_run = fmaxf(m_run, mx);
        l_run *= grow;
        corr *= grow;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[i][r] *= corr;
      }
      const float m_use = Wt::offset(m_run);
      float ls[4] = {0.f, 0.f, 0.f, 0.f};
      const bool plain = wave_uniform(even == vref) != 0;
      f32x8 p[4];
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          p[g][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g >> 1][8 * (g & 1) + r], sc[g], -m_use));
          ls[r & 3] += p[g][r];
        }
      l_run += (ls[0] + ls[1]) + (ls[2] + ls[3]);
      asm volatile("" : "+v"(l_run));  // the sums stay here
      if (!plain) {
        float inv = __builtin_amdgcn_rcpf(vref);
        asm volatile("" : "+v"(inv));  // the products below stay in this branch
        f32x4 f = vs * inv;
        if (wave_uniform(Wt::apart(least * inv) || Wt::apart(large * inv))) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (!wave_uniform(Wt::apart(f[g]))) continue;
            const vec own = __builtin_convertvector(p[g], vec);  // the 16 keys by themselves
#pragma unroll
            for (int i = 0; i < DT; ++i) {
              const int d = 32 * i + col;
              const vec vf = *(const vec*)(vt[buf] + d * PKT + 8 * ((2 * g + half) ^ swz_vt<D>(d)));
              const f32x16 x = AttnOp<T>::mma(vf, own, f32x16{});
#pragma unroll
              for (int r = 0; r < 16; ++r) o[i][r] = __builtin_fmaf(x[r], f[g], o[i][r]);
              __builtin_amdgcn_sched_barrier(0);
            }
            f[g] = 0.f;
          }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) p[g] *= f[g];
      }
      vec pk[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) pk[g] = __builtin_convertvector(p[g], vec);
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          const int d = 32 * i + col;
          const vec vf = *(const vec*)(vt[buf] + d * PKT + 8 * ((2 * g + half) ^ swz_vt<D>(d)));
          o[i] = AttnOp<T>::mma(vf, pk[g], o[i]);
        }
      __builtin_amdgcn_sched_group_barrier(0x100, 8, 1);
#pragma unroll
      for (int i = 0; i < 4 * DT; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
      }
    }
  }

  const float l = half_sum(l_run) * Wt::UNIT;
  if (row >= rows) return;
  const bool whole = it.parts == 1;
  if (!whole && (int)blockIdx.x >= a.slots) return;
  const int64_t at = (int64_t)blockIdx.x * RT + 32 * wave + col;
  const float unit = vref * Wt::UNIT, f = whole ? (l == 0.f ? 0.f : unit / l) : unit;
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * i + 8 * q + 4 * half;
      const f32x4 x = f32x4{o[i][4 * q], o[i][4 * q + 1], o[i][4 * q + 2], o[i][4 * q + 3]} * f;
      if (whole) {
        typedef typename AttnOp<T>::elem E;
        typedef E e4 __attribute__((ext_vector_type(4)));
        *(e4*)(a.o + tok * a.o_st + head * a.o_sh + d) = __builtin_convertvector(x, e4);
      } else {
        *(f32x4*)(a.part_o + at * D + d) = x;
      }
    }
  if (half != 0) return;
  if (whole) {
    a.lse[tok * a.lse_st + head * a.lse_sh] =
        l == 0.f ? -INFINITY : (m_run + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
  } else {
    a.part_ml[at * 2] = m_run;
    a.part_ml[at * 2 + 1] = l;
  }
}

template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void kv8_prompt_kernel(Kv8Args a) {
  prompt_item<T, D, NW>(a);
  kv8_rest<D>(a);
}

template <typename T, int D>
mi_status_t run_prompt(Kv8Args& a, hipStream_t s) {
  const int cus = cu_count();
  const int64_t tiles = (((int64_t)a.width << a.c.shift) + PKT - 1) / PKT;
  // blocks, if the sequences' new tokens are about as many in each
  auto blocks = [&](int nw) {
    const int64_t some = std::min(a.seqs, a.tokens), rows = (int64_t)a.tokens * a.group;
    return some > 0 ? some * ((rows / some + 32 * nw - 1) / (32 * nw)) * a.c.heads : 0;
  };
  // 256 rows a block halve what is spent on conversions and loads, but one such
  // block fills a CU: taken for long sequences whose blocks fill seven eighths of
  // their rounds over the CUs.  us, 256 and 128 rows, 32 query heads on 8: 1 x 2048
  // tokens behind 14000 (256 blocks) 546 / 603, 2 x 2048 behind 14000 (512) 1042 /
  // 1154, 4 x 2048 behind 4000 (1024) 732 / 788, 3 x 1500 behind 4000 (576) 474 /
  // 465, 8 x 1024 behind nothing 137 / 125.
  const int64_t wide = blocks(8), rounds = (wide + cus - 1) / cus;
  if (tiles >= 64 && wide > 0 && wide * 8 >= rounds * cus * 7) {
    a.plan = {cus, 0x40000000, 24, cus};
    return kv8_launch<T, D, 256, PKT, true>(a, kv8_prompt_kernel<T, D, 8>, 512, s);
  }
  // (tiles of the table's width, as wide as the longest sequence in these times)  A
  // block per CU where its tiles are few: two share a CU at 2.6 us a tile of
  // each, one alone takes 1.7 to 2, and a part more costs 8 us and its partials
  // (32 sequences of 512, 32 new tokens each: 28 us uncut, 47 in halves; 1 of
  // 16128, 128 new: 89 us with a block per CU, 67 with two; 16 heads of 64, 4 x up to
  // 1024 tokens behind 1000: 47 us uncut, 67 in parts).
  a.plan = {cus, 24, blocks(4) >= cus && tiles <= 32 ? 32 : 4, 2 * cus};
  return kv8_launch<T, D, 128, PKT, true>(a, kv8_prompt_kernel<T, D, 4>, 256, s);
}

}  // namespace

mi_status_t kv8_prompt(Kv8Args& a, int64_t dim, bool f16, hipStream_t s) {
  if (f16) return dim == 128 ? run_prompt<F16, 128>(a, s) : run_prompt<F16, 64>(a, s);
  return dim == 128 ? run_prompt<BF16, 128>(a, s) : run_prompt<BF16, 64>(a, s);
}

}  // namespace mi
