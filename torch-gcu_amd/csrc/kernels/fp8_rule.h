// Which kernel computes a product of 8-bit floating point.  Plain C++: the tests run it on
// the host against timings of every way.
//
// Each way's time is estimated in us, and the least is taken; what a way costs is what
// follows from its blocks:
//   tiles  rounds of `per_cu` blocks a CU, each of `steps` K steps of lo (few CUs busy) to
//          hi (one block on each) to hi2 (two on each) us, or the weight's stream (some of
//          which a gate never hides); launch, first copies and epilogue; what every
//          further round adds; and for slices of K their sums through the caches
//   few    the few-row kernel: the weight's stream, or what the busiest CU takes in (its
//          blocks' weight rows and all rows of x), and what every further round of blocks
//          adds; for a gate the launch that makes codes of y
//
// The constants are a fit to timings of these kernels on an MI355X, with weights from HBM
// and from the last-level cache: products of 433 sizes (M 1 .. 9000, N 128 .. 33000, K 128 ..
// 12000) and gates of 501.  Of 507 other sizes, by which one of five fits was chosen, the pick
// takes 0.8 % (a gate 0.3 %) longer than the fastest way on average, 18 % (20 %) at worst.  us, by
// few rows: M60 N14272 K256 3.8 in tiles and 8.6 in the few-row kernel, M32 N4096 K4096 9.8
// and 6.8; a gate of M64 N11008 K4096 in 64-row tiles 25.7 cut in two and 30.0 whole, of M512
// 52 in 256-row tiles and 65 in 128-row ones.
//
// Not built: 256 x 128 tiles (M2048 N4096 K11008 85 us, as picked 90), and two slices of 128 x
// 128 tiles (M93 N10944 K9216 33 us, as picked 39; of 122 sizes up to M 1024 they were faster
// by more than 2 % on 5).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

namespace mi {

// A tile shape: outputs of a block (of a gate half of its columns), blocks a CU counted to a
// round (a third of 64 x 128 fits, and its times tell of two), and the terms above.
struct Fp8Shape {
  int bm, bn, per_cu;
  float fixed, lo, hi, hi2, round;
  int slices[3];
};
constexpr Fp8Shape kFp8Shapes[] = {{256, 256, 1, 12.2f, 0.858f, 1.4f, 0, 9.76f, {1}},
                                   {128, 128, 2, 3.75f, 0.396f, 0.619f, 0.925f, 2.97f, {1}},
                                   {64, 128, 2, 3.24f, 0.305f, 0.564f, 0.664f, 1.73f, {1}},
                                   {64, 64, 2, 3.26f, 0.216f, 0.247f, 0.448f, 1.31f, {1, 2, 4}}};
constexpr Fp8Shape kFp8GateShapes[] = {{256, 128, 1, 10.5f, 1.04f, 1.37f, 0, 8.69f, {1}},
                                       {128, 128, 1, 5.48f, 0.673f, 0.924f, 0, 3.45f, {1}},
                                       {64, 128, 1, 3.97f, 0.514f, 0.833f, 0, 1.87f, {1, 2, 4}}};

// A few-row kernel: up to 8 xr rows of x, rt tiles of 16 weight rows a block (of a gate half
// of them the gate's), nw waves, rings of d units.
struct Fp8Few {
  int xr, rt, nw, d;
  constexpr int copies() const { return 2 * rt + xr; }  // 1 KiB copies a unit
  constexpr int ring() const { return nw * d * copies() * 1024; }
  constexpr int partial() const { return nw * rt * ((xr + 1) / 2) * 1024; }
  constexpr int body() const { return ring() > partial() ? ring() : partial(); }
  // and the scales of n groups, whole waves of them
  constexpr size_t lds(size_t n) const {
    return body() + (8 * xr * n + 63) / 64 * 256 + 2 * ((n + 63) / 64 * 256);
  }
};
constexpr Fp8Few kFp8Few[] = {{1, 1, 8, 2}, {2, 1, 4, 3}, {3, 1, 8, 2}, {4, 1, 4, 2}, {6, 1, 4, 2}, {8, 1, 4, 2}};
constexpr Fp8Few kFp8GateFew[] = {{1, 2, 4, 2}, {2, 2, 4, 2}, {4, 2, 4, 2}, {8, 2, 4, 2}};

constexpr size_t kFp8Lds = 160 * 1024;
// Blocks of up to 512 threads that a grid's first dimension holds.
constexpr int64_t kFp8Blocks = ((int64_t)1 << 23) - 1;

// A few-row kernel (index, or -1), or a tile shape and its slices of K.
struct Fp8Way {
  int few, shape, slices;
  float us;
};

// What differs between a product and a gate; times in us, rates in bytes a us.
struct Fp8Fit {
  int products;
  float stream, stream_rest;                     // and us a byte
  float slice_fixed, slice_rate;                 // and us a sum
  float few_fixed, few_rate, few_stream, few_round, few_codes;  // the last us an output
};
constexpr Fp8Fit kFp8Fit = {1, 5.19e6f, 0.f, 2.35f, 1.57e-6f, 2.61f, 76.4e3f, 5.62e6f, 1.57f, 0.f};
constexpr Fp8Fit kFp8GateFit = {2, 8.08e6f, 0.0127e-6f, 3.92f, 0.709e-6f, 4.8f, 59.7e3f, 6.99e6f, 1.07f, 6.44e-6f};

template <int SHAPES, int FEWS>
Fp8Way fp8_pick(int M, int N, int K, int cus, const Fp8Shape (&shapes)[SHAPES], const Fp8Few (&fews)[FEWS],
                const Fp8Fit& fit) {
  const int64_t groups = ((int64_t)K + 127) / 128;
  const float weight = (float)N * (float)K * (float)fit.products, outputs = (float)M * (float)N;
  Fp8Way best{-1, 0, 1, 3e38f};
  for (int i = 0; i < SHAPES; ++i) {
    const Fp8Shape& c = shapes[i];
    const int64_t across = ((int64_t)N + c.bn - 1) / c.bn, tiles = ((int64_t)M + c.bm - 1) / c.bm * across;
    if (i > 0 && tiles > kFp8Blocks) continue;
    for (int s : c.slices) {
      if (s == 0 || (s > 1 && groups < 2 * s)) break;
      const float steps = (float)((groups + s - 1) / s), per_cu = (float)c.per_cu;
      auto step = [&](float l) { return l <= 1.f ? c.lo + (c.hi - c.lo) * l : c.hi + (c.hi2 - c.hi) * (l - 1.f); };
      const float load = (float)(tiles * s) / (float)cus, full = std::floor(load / per_cu), rest = load - full * per_cu;
      const float products = full * steps * step(per_cu) + (rest > 0.f ? steps * step(rest) : 0.f);
      float us = c.fixed + std::max(products, weight / fit.stream) + weight * fit.stream_rest +
                 c.round * std::max(0.f, full - (rest > 0.f ? 0.f : 1.f));
      if (s > 1) us += fit.slice_fixed + (float)(s * fit.products) * outputs * fit.slice_rate;
      if (us < best.us) best = Fp8Way{-1, i, s, us};
    }
  }
  for (int i = 0; i < FEWS; ++i) {
    const Fp8Few& f = fews[i];
    const size_t lds = f.lds((size_t)groups);
    const int64_t columns = ((int64_t)N + 15) / 16;
    if (M > 8 * f.xr || lds > kFp8Lds || columns > kFp8Blocks) continue;
    const float blocks = (float)columns / (float)cus, per_cu = (float)(kFp8Lds / lds);
    const float full = std::floor(blocks / per_cu), rest = blocks - full * per_cu;
    const float block = (float)(16 * fit.products + (M + 7) / 8 * 8) * (float)K;
    const float busiest = (full * per_cu + (rest > 0.f ? std::max(1.f, rest) : 0.f)) * block;
    const float us = fit.few_fixed + std::max(weight / fit.few_stream, busiest / fit.few_rate) +
                     fit.few_round * (full - (rest > 0.f ? 0.f : 1.f)) + fit.few_codes * outputs;
    if (us <= best.us) best = Fp8Way{i, 0, 1, us};
    break;  // the first that holds the rows and scales
  }
  return best;
}

inline Fp8Way fp8_pick_linear(int M, int N, int K, int cus) {
  return fp8_pick(M, N, K, cus, kFp8Shapes, kFp8Few, kFp8Fit);
}
inline Fp8Way fp8_pick_gate(int M, int N, int K, int cus) {
  return fp8_pick(M, N, K, cus, kFp8GateShapes, kFp8GateFew, kFp8GateFit);
}

}  // namespace mi
