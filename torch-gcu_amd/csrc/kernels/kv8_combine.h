// Merging of the partial results of an attention call over the 8-bit cache whose
// sequences were cut along their keys.
#pragma once

#include "kv8_common.h"

namespace mi {
namespace {

// A wave per output row of a sequence that was cut: its parts' partials merged
// in order, eight at a time (their loads in flight together).  Calls in which
// nothing was cut end with the plan.
template <typename T, int D, int RT, int KT, bool LAST_FIRST>
__global__ __launch_bounds__(256) void kv8_combine_kernel(Kv8Args a) {
  constexpr int E = D / 64, U = 8;
  typedef float fe __attribute__((ext_vector_type(E)));
  const int heads = a.c.heads * a.group;
  const Kv8Lanes lanes(a);
  const int lane = lanes.lane;
  bool some = false;
  // (the attention kernel's own number: a float of the plan compiled here could
  // be rounded differently)
  const int chunk = wave_uniform(*a.chunk);
  for (int b0 = 0; b0 < a.seqs; b0 += 64) {
    const Kv8Seq s = lanes.at(b0);
    some = some || __ballot(s.n > 0 && kv8_cut(s, a.group, RT, KT).parts(chunk) > 1) != 0;
  }
  if (!some) return;
  const int64_t all = (int64_t)a.tokens * heads;
  for (int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); id < all;
       id += (int64_t)gridDim.x * 4) {
    const int t = wave_uniform((int)(id / heads)), h = wave_uniform((int)(id % heads));
    // the sequence that token t is of, and the items before it
    int64_t before = 0;
    bool found = false;
    int where = 0;
    Kv8Seq s{};
    for (int b0 = 0; b0 < a.seqs && !found; b0 += 64) {
      const Kv8Seq mine = lanes.at(b0);
      const Kv8Cut c = kv8_cut(mine, a.group, RT, KT);
      const int n = a.c.heads * c.row_tiles * c.parts(chunk), upto = wave_scan(n);
      const uint64_t hit = __ballot(t >= mine.first && t < mine.first + mine.n);
      if (hit != 0) {
        const int l = __builtin_ctzll(hit);
        found = true;
        where = l;
        s = Kv8Lanes::pick(mine, l);
        before += __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l);
      } else {
        before += __builtin_amdgcn_readlane(upto, 63);
      }
    }
    if (!found) continue;
    const Kv8Cut c = kv8_cut(s, a.group, RT, KT);
    const int parts = c.parts(chunk);
    if (parts == 1) continue;
    const int row = (t - s.first) * a.group + h % a.group;
    const int tile = LAST_FIRST ? c.row_tiles - 1 - row / RT : row / RT;
    int64_t item = before + ((int64_t)tile * a.c.heads + h / a.group) * parts;
    int64_t step = 1;  // from a part to the next
    if (LAST_FIRST && Kv8RoundItems::apply(a)) {
      const Kv8RoundItems all = Kv8RoundItems::of<RT, KT>(a, lanes.head, chunk);
      const int k = tile + __builtin_amdgcn_readlane(all.rounds.off, where);
      const int n = all.rounds.in(k) ? all.parts : 0;
      const int first = all.before(k) + __builtin_amdgcn_readlane(wave_scan(n) - n, where);
      step = a.c.heads;
      item = (int64_t)first * step + h / a.group;
    }
    if (item < 0 || item + (parts - 1) * step >= a.slots) continue;
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2* pm = (const f2*)a.part_ml + item * RT + row % RT;
    const float* po = a.part_o + (item * RT + row % RT) * D + lane * E;
    float M = -INFINITY, l = 0.f;
    fe acc = {};
    for (int p0 = 0; p0 < parts; p0 += U) {
      fe v[U];
      f2 ml[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t p = min(p0 + u, parts - 1) * step;
        v[u] = *(const fe*)(po + p * RT * D);
        ml[u] = pm[p * RT];
        if (p0 + u >= parts) ml[u] = f2{-INFINITY, 0.f};
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, ml[u][0]);
      const float mu = top == -INFINITY ? 0.f : top;
      const float before = __builtin_amdgcn_exp2f(M - mu);
      M = top;
      l *= before;
      acc *= before;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = __builtin_amdgcn_exp2f(ml[u][0] - mu);
        l += ml[u][1] * w;
        if (p0 + u < parts) acc += v[u] * w;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    typedef typename AttnOp<T>::elem Et;
    typedef Et ee __attribute__((ext_vector_type(E)));
    *(ee*)(a.o + t * a.o_st + h * a.o_sh + lane * E) = __builtin_convertvector(acc * inv, ee);
    if (lane == 0)
      a.lse[t * a.lse_st + h * a.lse_sh] =
          l == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
  }
}

// Room for the partials of a call whose parts are planned by a.plan, then the
// attention kernel and, where anything can have been cut,
// the merge.
template <typename T, int D, int RT, int KT, bool LAST_FIRST, typename K>
mi_status_t kv8_launch(Kv8Args& a, K kernel, int threads, hipStream_t s) {
  const int64_t base = kv8_row_tiles_most(a.tokens, a.seqs, a.group, RT) * a.c.heads;
  const int64_t key_tiles = (((int64_t)a.width << a.c.shift) + KT - 1) / KT;
  const int64_t parts = std::max<int64_t>((key_tiles + a.plan.least - 1) / a.plan.least, 1);
  bool cut = parts > 1;
  // (idle blocks are not free: 8 sequences of 4000 took 19 us with 512 of them,
  // 24 with 4096)
  a.slots = (int)std::max<int64_t>(std::min(base + a.plan.many, base * parts), 1);
  Workspace ws;
  if (cut) {
    const size_t rows = (size_t)a.slots * RT;
    if (ws.alloc((rows * (D + 2) + 1) * sizeof(float), s) == MI_OK) {
      a.part_o = (float*)ws.get();
      a.part_ml = a.part_o + rows * D;
      a.chunk = (int*)(a.part_ml + rows * 2);
    } else {  // whole sequences need none
      clear_error();
      cut = false;
      a.plan.least = 0x40000000;
      a.slots = (int)std::max<int64_t>(base, 1);
    }
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)a.slots), dim3(threads), 0, s, a);
  MI_RETURN_IF(check_launch("kv8_attention"));
  if (!cut) return MI_OK;
  const int64_t rows = (int64_t)a.tokens * a.c.heads * a.group;
  const unsigned grid = (unsigned)std::min<int64_t>((rows + 3) / 4, 8 * cu_count());
  hipLaunchKernelGGL((kv8_combine_kernel<T, D, RT, KT, LAST_FIRST>), dim3(grid), dim3(256), 0, s, a);
  return check_launch("kv8_attention");
}

}  // namespace
}  // namespace mi
