// The kernel of 8-bit floating point products with few rows of activations: the
// linear layers of a decode step.
//
// The weight is read once, and what bounds it is that stream (and up to 4096 x 4096 a
// launch, the first copies' latency and the waves' join): so a block has as few weight rows
// as an instruction takes, 16, which gives many blocks, and its waves share the K instead,
// each with its own copies in flight and no barrier between first and last.  The rows of
// activations, which every block reads, come from the caches.  us a launch: M1 N4096 K4096
// 5.0 (16.8 MB, 3.4 TB/s), M24 N4096 K11008 11.4 (4.0 TB/s), a gate of M8 N11008 K4096 16.5
// (90 MB, 5.5 TB/s) and 3.5 for its codes' launch.
#pragma once

#include "fp8_gemm.h"
#include "fp8_rule.h"

namespace mi {
namespace {

// XR x 8 rows of activations (M <= 8 XR), RT tiles of 16 weight rows a block, whose NW
// waves take units of 128 of K in turn, each through a ring of D of its own: WAYS[I] of the
// rule's.
template <const Fp8Few* WAYS, int I>
struct R8Cfg {
  static constexpr Fp8Few F = WAYS[I];
  static constexpr int XR = F.xr, RT = F.rt, NW = F.nw, D = F.d;
  static constexpr int MT = (XR + 1) / 2;                 // tiles of 16 activation rows
  static constexpr int LPU = F.copies();                  // 1 KiB copies a unit
  static constexpr int UNIT = LPU * 1024, BODY = F.body();
  static_assert(D >= 2 && LPU * (D - 1) < 64, "copies in flight are counted in 6 bits");
};

// y [M][N] float32 of a gate instead of out; the weight tiles are then half gate's,
// half up's, of the same columns.
template <class C, bool GATE>
__global__ __launch_bounds__(64 * C::NW) void fp8_rows_gemm_kernel(Fp8Gemm p) {
  constexpr int XR = C::XR, RT = C::RT, NW = C::NW, D = C::D, MT = C::MT, LPU = C::LPU, UNIT = C::UNIT;
  constexpr int COLS = 16 * (GATE ? RT / 2 : RT);  // output columns of a block
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, row = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int M = p.M, N = p.N, K = p.K, KB = (K + 127) / 128, units = K / 128;
  const int n0 = blockIdx.x * COLS;
  // weight tile t of 16 rows: columns n0 + 16 (t % (RT / 2)) of gate, then of up
  auto up = [&](int t) __attribute__((always_inline)) { return GATE && t >= RT / 2; };
  auto column = [&](int t) __attribute__((always_inline)) { return n0 + 16 * (GATE ? t % (RT / 2) : t); };
  const uint8_t* wb[2] = {p.w.codes + (int64_t)n0 * p.w.ld, GATE ? p.w2.codes + (int64_t)n0 * p.w2.ld : nullptr};
  // byte offsets of a lane's 16 bytes of each copy (8 rows of 128 bytes); rows past the
  // end read the last one and feed outputs that are not stored
  uint32_t off[LPU];
#pragma unroll
  for (int q = 0; q < LPU; ++q) {
    const int r8 = lane >> 3;
    if (q < 2 * RT) {
      const int t = q / 2, r = 8 * (q & 1) + r8;
      off[q] = (uint32_t)((min(column(t) + r, N - 1) - n0) * (up(t) ? p.w2.ld : p.w.ld) + 16 * dl_swz(r, lane & 7));
    } else {
      const int r = 8 * (q - 2 * RT) + r8;
      off[q] = (uint32_t)(min(r, M - 1) * p.x.ld + 16 * dl_swz(r, lane & 7));
    }
  }
  char* ring = smem + wave * (D * UNIT);
  auto base_of = [&](int q) __attribute__((always_inline)) {
    return q < 2 * RT ? (up(q / 2) ? wb[1] : wb[0]) : p.x.codes;
  };
  // (a unit past the end is not multiplied)
  auto issue = [&](int slot, int u) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < LPU; ++q)
      lds_copy16(base_of(q) + (int64_t)min(u, units - 1) * 128, off[q], ring + slot * UNIT + q * 1024);
  };
  // The scales first, a word each, into LDS behind the ring: [8 XR][KB] of the rows, [KB] of
  // the weight's block (of both of a gate), each in whole wave copies; a block's columns
  // lie in one block of 128.
  // (Copied as the codes are: loaded to registers and stored, 0.4 to 0.8 us more.)
  int* xs = (int*)(smem + C::BODY);
  int* ws = xs + (8 * XR * KB + 63) / 64 * 64;
  int* ws2 = ws + (KB + 63) / 64 * 64;
  {
    for (int i = wave * 64; i < 8 * XR * KB; i += 64 * NW) {
      const int at = min(i + lane, 8 * XR * KB - 1), r = at / KB;
      lds_copy_byte(p.x.scales, (uint32_t)(min(r, M - 1) * (int)p.x.sld + at - r * KB), xs + i);
    }
    for (int i = wave * 64; i < KB; i += 64 * NW) {
      lds_copy_byte(p.w.scales + n0 / kFp8Group * p.w.sld, (uint32_t)min(i + lane, KB - 1), ws + i);
      if constexpr (GATE)
        lds_copy_byte(p.w2.scales + n0 / kFp8Group * p.w2.sld, (uint32_t)min(i + lane, KB - 1), ws2 + i);
    }
  }
  if (units > 0) {
#pragma unroll
    for (int s = 0; s < D - 1; ++s) issue(s, wave + s * NW);
    wait_vmcnt<(D - 1) * LPU>();
  } else {
    wait_vmcnt<0>();
  }
  __syncthreads();
  f32x4_t acc[RT][MT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4_t{};
  const int ro0 = row * 128 + 16 * dl_swz(row, lane >> 4), ro1 = row * 128 + 16 * dl_swz(row, 4 + (lane >> 4));
  auto fragment = [&](const char* t, int r0, int r1) __attribute__((always_inline)) {
    const u32x4_t lo = *(const u32x4_t*)(t + r0), hi = *(const u32x4_t*)(t + r1);
    return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  auto multiply = [&](const char* s, int kb) __attribute__((always_inline)) {
    i32x8_t fw[RT], fx[MT];
    int sw[2], sx[MT];
#pragma unroll
    for (int h = 0; h < (GATE ? 2 : 1); ++h) sw[h] = (h ? ws2 : ws)[kb];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      // (an odd number of 8 rows: the last tile's lower half again)
      const bool half = 2 * j + 1 >= XR;
      const int r = half ? row & 7 : row;
      const char* t = s + (2 * RT + 2 * j) * 1024;
      sx[j] = xs[(16 * j + r) * KB + kb];
      if (half) fx[j] = fragment(t, r * 128 + 16 * dl_swz(r, lane >> 4), r * 128 + 16 * dl_swz(r, 4 + (lane >> 4)));
      else fx[j] = fragment(t, ro0, ro1);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) fw[i] = fragment(s + 2 * i * 1024, ro0, ro1);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] = mma_fp8(fw[i], fx[j], acc[i][j], sw[up(i) ? 1 : 0], sx[j]);
  };
  int slot = 0;
  for (int u = wave; u < units; u += NW) {
    const int refill = slot == 0 ? D - 1 : slot - 1;  // its reads were waited for by the last products
    __builtin_amdgcn_sched_barrier(0);
    issue(refill, u + (D - 1) * NW);
    wait_vmcnt<(D - 1) * LPU>();
    asm volatile("" : : : "memory");
    __builtin_amdgcn_sched_barrier(0);
    multiply(ring + slot * UNIT, u);
    slot = slot + 1 == D ? 0 : slot + 1;
  }
  if (K % 128 != 0 && wave == units % NW) {
    // the last K % 128 columns, zeros behind them
    typedef u64x2_t __attribute__((aligned(1))) u64x2_u;
    wait_vmcnt<0>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < LPU; ++q) {
      const int r = (q < 2 * RT ? 8 * (q & 1) : 8 * (q - 2 * RT)) + (lane >> 3);
      const int chunk = dl_swz(r, lane & 7), k = units * 128 + 16 * chunk;
      const uint8_t* at = base_of(q) + off[q] - 16 * chunk;
      u64x2_t v;
      if (K >= 16) {
        v = shift_down(*(const u64x2_u*)(at + min(k, K - 16)), max(0, k - (K - 16)));
      } else {
        v = u64x2_t{};
        for (int e = 0; e < 16; ++e)
          if (k + e < K) v[e >> 3] |= (uint64_t)at[k + e] << (8 * (e & 7));
      }
      *(u64x2_t*)(ring + q * 1024 + lane * 16) = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    multiply(ring, units);
  }
  wait_vmcnt<0>();  // the copies of units past the end
  __syncthreads();
  f32x4_t* red = (f32x4_t*)smem;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) red[(wave * RT * MT + i * MT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  auto sum = [&](int t, int l) __attribute__((always_inline)) {
    f32x4_t s = red[t * 64 + l];
#pragma unroll
    for (int w = 1; w < NW; ++w) s += red[(w * RT * MT + t) * 64 + l];
    return s;
  };
  auto wide = [&](uint16_t v) __attribute__((always_inline)) { return p.f16 ? f16_to_f32(v) : bf16_to_f32(v); };
  constexpr int TILES = GATE ? RT / 2 * MT : RT * MT;
  for (int id = threadIdx.x; id < TILES * 64; id += 64 * NW) {
    const int t = id >> 6, l = id & 63;
    const int m = 16 * (t % MT) + (l & 15), n = n0 + 16 * (t / MT) + 4 * (l >> 4);
    f32x4_t s = sum(t, l);
    if constexpr (GATE) {
      const f32x4_t u = sum(t + TILES, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = silu_mul_f32(s[e], u[e]);
    }
    if (m >= M || n >= N) continue;
    if constexpr (GATE) {
      *(f32x4_t*)(p.part + (int64_t)m * p.ldp + n) = s;  // (ldp is a multiple of 4)
      continue;
    }
    uint16_t* dst = (uint16_t*)p.out + (int64_t)m * p.ldc + n;
    const uint16_t* res = p.res == nullptr ? nullptr : p.res + (int64_t)m * p.ldr + n;
    uint16_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float y = s[e];
      const int at = min(e, N - 1 - n);
      if (p.bias != nullptr)
        y += p.bias_dtype == MI_F32 ? ((const float*)p.bias)[n + at] : wide(((const uint16_t*)p.bias)[n + at]);
      if (res != nullptr) y += wide(res[at]);
      v[e] = p.f16 ? f32_to_f16(y) : f32_to_bf16(y);
    }
    if (n + 3 < N && (uintptr_t)dst % 8 == 0) {
      *(u16x4_t*)dst = u16x4_t{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < N) dst[e] = v[e];
    }
  }
}

}  // namespace
}  // namespace mi
