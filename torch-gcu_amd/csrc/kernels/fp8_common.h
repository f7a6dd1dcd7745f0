// Shared by the kernels of linear layers in 8-bit floating point: rows of e4m3
// codes with a power-of-two scale for each 128 columns, weights with one for each
// 128 x 128 block; a scale is its biased exponent, 2^(byte - 127), which is what the
// scaled matrix instructions take.
#pragma once

#include <algorithm>
#include <cmath>

#include "gemm_common.h"

namespace mi {

constexpr int kFp8Group = 128;

// One operand as a kernel reads (or writes) it: rows of codes and of scale bytes,
// dense along columns.
struct Fp8Mat {
  uint8_t* codes;
  uint8_t* scales;
  int64_t ld, sld;  // row strides, in bytes
};

// Any number of blocks as a grid (a dimension holds fewer than 2^32 threads); the
// kernel's block is fp8_block(), and those past the last end at once.
inline dim3 fp8_grid(int64_t blocks) {
  const int64_t x = blocks < (1 << 20) ? blocks : 1 << 20;
  return dim3((unsigned)x, ceil_div_u(blocks, x));
}

inline int64_t fp8_groups(int64_t n) { return (n + kFp8Group - 1) / kFp8Group; }

// Checks of the entry points (fp8_check.cpp); they read descriptors only.
// codes uint8 [rows, cols] and scales uint8 [rows or its blocks, column groups],
// dense along columns; written: rows of its own.
mi_status_t fp8_check(const char* op, const char* name, const mi_fp8_t* t, bool weight, bool written,
                      Fp8Mat* m);
// [rows, cols] with unit column stride, of a 16-bit type (or float32 with f32)
mi_status_t fp8_check_wide(const char* op, const char* name, const mi_tensor_t* t, bool f32);
// INVALID where an output shares memory with another tensor of the call
mi_status_t fp8_check_apart(const char* op, const char* name, const mi_tensor_t* out,
                            const char* other_name, const mi_tensor_t* other);

// y float32 [rows][ld], with 16-byte aligned rows, to codes and scales (fp8_quantize.hip)
mi_status_t fp8_quantize_f32(const float* y, int64_t ld, int64_t rows, int cols, const Fp8Mat& out,
                             hipStream_t s, const char* op);

namespace {

typedef uint32_t f8_u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int64_t fp8_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// The scale byte of a group whose largest finite magnitude has these float bits:
// the smallest power of two s >= 2^-110 with amax <= 448 s.  448 is 1.75 x 2^8, so the
// exponent is amax's less 8, and one more where its mantissa is over 1.75.  (2^-110
// keeps 1 / s and every product of it ordinary floats; the least is the 8-bit cache's.)
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax) {
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 127 - 110);
}
// 1 / s, exact
__device__ __forceinline__ float fp8_inverse(uint32_t byte) {
  return __uint_as_float((254u - byte) << 23);
}
// x, or NaN where it is infinite (0 inf is NaN): e4m3 has no infinity.
__device__ __forceinline__ float fp8_no_inf(float x) { return __builtin_fmaf(x, 0.f, x); }
// The larger of m and |x|, of m and a NaN m.
__device__ __forceinline__ float fp8_larger(float m, float x) { return __builtin_fmaxf(m, __builtin_fabsf(x)); }
// Four values times a power of two as codes, to nearest, ties to even; NaN stays NaN.  The
// caller's scale keeps the others within 448.
__device__ __forceinline__ uint32_t fp8_codes4(float a, float b, float c, float d, float inv) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, r, true);
}

// The largest over each row of 16 lanes, in all of them (of floats that are not negative:
// they order as their bits do).
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  auto step = [&](uint32_t o) __attribute__((always_inline)) { v = v > o ? v : o; };
  step((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
  step((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
  step((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));
  step((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));
  return v;
}

}  // namespace
}  // namespace mi
