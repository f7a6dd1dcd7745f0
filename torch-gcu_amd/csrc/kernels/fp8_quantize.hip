// Activations and weights to e4m3 codes with a power-of-two scale for each 128
// columns of a row, or each 128 x 128 block; and the root-mean-square norm, with the
// residual's addition before it, whose output goes straight to such codes.
//
// A scale is the smallest power of two s >= 2^-110 with amax <= 448 s: e4m3 is a
// floating type, so a power of two costs none of its precision, division by it is
// exact, and the matrix instructions multiply by it for free.
//
// What bounds them: HBM, each element read once and its code written.  A lane holds
// 8 neighbouring elements, so 16 lanes are a group and its maximum four DPP steps; a
// row stays in registers between the sum of squares, the maxima and the codes.
#include "fp8_common.h"

namespace mi {
namespace {

constexpr int NORM = 0, NORM_RES = 1;

struct RowsArgs {
  const void* x;
  const void* res;
  const void* weight;
  void* total;
  int64_t x_ld, res_ld, total_ld;  // row strides, in elements
  Fp8Mat out;
  int64_t rows;
  int cols;
  float eps;
};

// Eight neighbouring elements as they lie in memory.
template <typename T>
struct Eight {
  typedef typename Num<T>::storage St;
  static constexpr int W = sizeof(St) * 2;  // 32-bit words
  union {
    uint32_t w[W] = {};
    St e[8];
  };
  __device__ __forceinline__ float get(int i) const { return Num<T>::load(e[i]); }
  // A row's elements col .. col + 7, zeros behind its end.  Rows may begin anywhere (a
  // global load takes any address); those whose length is no multiple of 8 end with
  // single elements.
  typedef typename AnyAligned<sizeof(St)>::type vec;
  static __device__ __forceinline__ Eight load(const void* row, int col, int cols) {
    const St* p = (const St*)row;
    return cols >= 8 ? load_ragged(p, whole(p, min(col, cols - 8)), col, cols) : load_ragged(p, Eight(), col, cols);
  }
  // elements col .. col + 7, all of which are the row's
  static __device__ __forceinline__ Eight whole(const St* p, int col) {
    Eight r;
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const u32x4_t v = *((const vec*)(p + col) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v[j];
    }
    return r;
  }
  static __device__ __forceinline__ Eight load_ragged(const St* p, Eight r, int col, int cols) {
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = col < cols ? r.w[i] : 0u;
    if ((cols & 7) != 0 && col < cols && col + 8 > cols) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.e[i] = p[min(col + i, cols - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i) r.e[i] = col + i < cols ? r.e[i] : (St)0;
    }
    return r;
  }
  __device__ __forceinline__ void store(void* row, int col, int cols) const {
    St* p = (St*)row + col;
    if (col + 8 <= cols) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i)
        *((vec*)p + i) = u32x4_t{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < cols) p[i] = e[i];
    }
  }
};

// The codes of a lane's 8 values of a group that a row of 16 lanes holds, and the group's
// scale byte.
__device__ __forceinline__ f8_u32x2 codes_of(float* y, uint32_t* byte) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = fp8_no_inf(y[i]);
    most = fp8_larger(most, y[i]);
  }
  *byte = fp8_scale_byte(row16_max(__float_as_uint(most)));
  const float inv = fp8_inverse(*byte);
  return f8_u32x2{fp8_codes4(y[0], y[1], y[2], y[3], inv), fp8_codes4(y[4], y[5], y[6], y[7], inv)};
}

__device__ __forceinline__ void store_codes(uint8_t* row, int col, int cols, f8_u32x2 c) {
  typedef f8_u32x2 __attribute__((aligned(1))) vec;
  if (col + 8 <= cols) {
    *(vec*)(row + col) = c;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < cols) row[col + i] = (uint8_t)(c[i >> 2] >> (8 * (i & 3)));
  }
}

// A wave to 512 columns of a row.
template <typename T>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(RowsArgs a, int chunks) {
  typedef Eight<T> E;
  const int64_t id = fp8_block() * 4 + (threadIdx.x >> 6), row = id / chunks;
  if (row >= a.rows) return;
  const int col = (int)(id - row * chunks) * 512 + (threadIdx.x & 63) * 8;
  const E v = E::load((const typename E::St*)a.x + row * a.x_ld, col, a.cols);
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = v.get(j);
  uint32_t byte;
  const f8_u32x2 c = codes_of(y, &byte);
  store_codes(a.out.codes + row * a.out.ld, col, a.cols, c);
  if ((threadIdx.x & 15) == 0 && col < a.cols) a.out.scales[row * a.out.sld + col / kFp8Group] = (uint8_t)byte;
}

// The norm: TPR threads a row, VPL x 8 elements a thread in registers; VPL 0: rows of any
// length, read again for the codes (the total from where it was written).
template <typename T, int KIND, int TPR, int VPL>
__global__ __launch_bounds__(256) void fp8_rows_kernel(RowsArgs a) {
  typedef Eight<T> E;
  typedef typename E::St St;
  constexpr int STEP = TPR * 8, N = VPL > 0 ? VPL : 1;
  __shared__ float red[4];
  const int t = threadIdx.x % TPR;
  const int64_t row = fp8_block() * (256 / TPR) + threadIdx.x / TPR;
  if (row >= a.rows) return;
  const int cols = a.cols;
  const St* x = (const St*)a.x + row * a.x_ld;
  const St* res = KIND == NORM_RES ? (const St*)a.res + row * a.res_ld : nullptr;
  St* total = KIND == NORM_RES ? (St*)a.total + row * a.total_ld : nullptr;
  uint8_t* codes = a.out.codes + row * a.out.ld;
  uint8_t* scales = a.out.scales + row * a.out.sld;
  E v[N], r[N];
  auto load = [&](int i, int col) __attribute__((always_inline)) {
    v[i] = E::load(x, col, cols);
    if constexpr (KIND == NORM_RES) r[i] = E::load(res, col, cols);
  };
  float ss = 0.f;
  auto add_up = [&](int i, int col) __attribute__((always_inline)) {
    if constexpr (KIND == NORM_RES) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i].e[j] = Num<T>::store(v[i].get(j) + r[i].get(j));
      v[i].store(total, col, cols);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(v[i].get(j), v[i].get(j), ss);
  };
  if constexpr (VPL > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) load(i, t * 8 + i * STEP);
#pragma unroll
    for (int i = 0; i < N; ++i) add_up(i, t * 8 + i * STEP);
  } else {
    for (int c = t * 8; c < cols; c += STEP) {
      load(0, c);
      add_up(0, c);
    }
  }
  ss = wave_sum(ss);
  if constexpr (TPR == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = (red[0] + red[1]) + (red[2] + red[3]);
  }
  const float norm = 1.0f / __builtin_sqrtf(ss / (float)cols + a.eps);
  auto finish = [&](const E& s, int col) __attribute__((always_inline)) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = s.get(j) * norm;
    if (a.weight != nullptr) {
      const E w = E::load(a.weight, col, cols);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= w.get(j);
    }
    // (0 x an infinite norm is NaN: what lies behind the row's end stays 0)
    if (col >= cols) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = 0.f;
    } else if ((cols & 7) != 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = col + j < cols ? y[j] : 0.f;
    }
    uint32_t byte;
    const f8_u32x2 c = codes_of(y, &byte);
    store_codes(codes, col, cols, c);
    if ((t & 15) == 0 && col < cols) scales[col / kFp8Group] = (uint8_t)byte;
  };
  if constexpr (VPL > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) finish(v[i], t * 8 + i * STEP);
  } else {
    // whole rows of 16 lanes take part in a group's maximum
    for (int c = t * 8; c / kFp8Group * kFp8Group < cols; c += STEP)
      finish(E::load(KIND == NORM_RES ? total : x, c, cols), c);
  }
}

// A block of 512 threads to a 128 x 128 block of the weight, 4 rows a thread: bf16 11008 x
// 4096 23.7 us (135 MB, 5.7 TB/s, a part of it from the last-level cache), f32 1000 x 1500 4.9
// (in 256 threads, with loads behind conditions, 31 and 12.8).
template <typename T>
__global__ __launch_bounds__(512) void fp8_weight_kernel(const void* w, int64_t ld, int64_t rows, int cols,
                                                         Fp8Mat out) {
  typedef Eight<T> E;
  typedef typename E::St St;
  constexpr int R = 4, NW = 8;
  __shared__ uint32_t red[NW];
  const int col = blockIdx.x * kFp8Group + (threadIdx.x & 15) * 8;
  const int64_t row0 = (int64_t)blockIdx.y * kFp8Group + (threadIdx.x >> 4);
  // (rows past the end read the last one again, which is in the block)
  const St* p[R];
#pragma unroll
  for (int i = 0; i < R; ++i) p[i] = (const St*)w + min(row0 + 32 * i, rows - 1) * ld;
  E v[R];
  if ((cols & 7) == 0 || (int)(blockIdx.x + 1) * kFp8Group <= cols) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = E::whole(p[i], min(col, cols - 8));
    if (col >= cols)
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] = E();
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = E::load(p[i], col, cols);
  }
  float y[R][8], mine = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y[i][j] = fp8_no_inf(v[i].get(j));
      mine = fp8_larger(mine, y[i][j]);
    }
  uint32_t most = row16_max(__float_as_uint(mine));
  most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
  most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
  __syncthreads();
  most = red[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) most = max(most, red[i]);
  const uint32_t byte = fp8_scale_byte(most);
  const float inv = fp8_inverse(byte);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const f8_u32x2 c = {fp8_codes4(y[i][0], y[i][1], y[i][2], y[i][3], inv),
                        fp8_codes4(y[i][4], y[i][5], y[i][6], y[i][7], inv)};
    if (row0 + 32 * i < rows) store_codes(out.codes + (row0 + 32 * i) * out.ld, col, cols, c);
  }
  if (threadIdx.x == 0) out.scales[blockIdx.y * out.sld + blockIdx.x] = (uint8_t)byte;
}

// A wave to 512 columns: f16 rows of 11008 out of 22016, 6011 of them, 37.4 us (198 MB, 5.3
// TB/s), with 2048 columns a wave 10 % more, with a block to a row 39 %; bf16 8192 x 4096 with
// these 15 % more and 8 % less; one row of 4096 2.0 us, 7 % more with either.
template <typename T>
mi_status_t launch_quantize(const RowsArgs& a, hipStream_t s, const char* op) {
  const int64_t chunks = (a.cols + 511) / 512;
  const int64_t blocks = (a.rows * chunks + 3) / 4;
  if (blocks > (int64_t)65535 << 20) MI_FAIL(MI_ERR_TOO_LARGE, "%s: too many elements", op);
  hipLaunchKernelGGL((fp8_quantize_kernel<T>), fp8_grid(blocks), dim3(256), 0, s, a, (int)chunks);
  return check_launch(op);
}

// Up to 1024 columns a wave holds a row, above a block; rows over 8192 are read again for
// the codes.  us, with the residual: bf16 8192 x 1024 13.3 (with a block a row 16.4), 8192 x
// 4096 46.4 (235 MB, 5.1 TB/s; with a wave a row 65), 8 x 4096 4.3 (9.6), 4096 x 11008 84
// (107 with the row held).
template <typename T, int KIND>
mi_status_t launch_norm(const RowsArgs& a, hipStream_t s, const char* op) {
  auto go = [&](auto tpr, auto vpl) {
    constexpr int TPR = decltype(tpr)::value;
    hipLaunchKernelGGL((fp8_rows_kernel<T, KIND, TPR, decltype(vpl)::value>),
                       fp8_grid((a.rows + 256 / TPR - 1) / (256 / TPR)), dim3(256), 0, s, a);
    return check_launch(op);
  };
  const std::integral_constant<int, 64> wave;
  const std::integral_constant<int, 256> block;
  const std::integral_constant<int, 0> any;
  const std::integral_constant<int, 1> one;
  const std::integral_constant<int, 2> two;
  const std::integral_constant<int, 4> four;
  if (a.cols <= 512) return go(wave, one);
  if (a.cols <= 1024) return go(wave, two);
  if (a.cols <= 2048) return go(block, one);
  if (a.cols <= 4096) return go(block, two);
  if (a.cols <= 8192) return go(block, four);
  return go(block, any);
}

template <int KIND>
mi_status_t run_norm(const RowsArgs& a, int dtype, hipStream_t s, const char* op) {
  if (dtype == MI_BF16) return launch_norm<BF16, KIND>(a, s, op);
  if (dtype == MI_F16) return launch_norm<F16, KIND>(a, s, op);
  return launch_norm<float, KIND>(a, s, op);
}

mi_status_t check_shape(const char* op, const mi_fp8_t* out, const mi_tensor_t* x, const char* name) {
  MI_CHECK_ARG(out->codes.sizes[0] == x->sizes[0] && out->codes.sizes[1] == x->sizes[1],
               "%s: codes are [%lld, %lld], %s [%lld, %lld]", op, (long long)out->codes.sizes[0],
               (long long)out->codes.sizes[1], name, (long long)x->sizes[0], (long long)x->sizes[1]);
  return MI_OK;
}

mi_status_t check_outputs_apart(const char* op, const mi_fp8_t* out, const char* name,
                                const mi_tensor_t* t) {
  MI_RETURN_IF(fp8_check_apart(op, "codes", &out->codes, name, t));
  return fp8_check_apart(op, "scales", &out->scales, name, t);
}

}  // namespace

mi_status_t fp8_quantize_f32(const float* y, int64_t ld, int64_t rows, int cols, const Fp8Mat& out,
                             hipStream_t s, const char* op) {
  RowsArgs a{};
  a.x = y;
  a.x_ld = ld;
  a.rows = rows;
  a.cols = cols;
  a.out = out;
  return launch_quantize<float>(a, s, op);
}

}  // namespace mi

using namespace mi;

extern "C" {

mi_status_t mi_fp8_quantize(const mi_fp8_t* out, const mi_tensor_t* x, mi_stream_t stream) {
  clear_error();
  const char* op = "fp8_quantize";
  RowsArgs a{};
  MI_RETURN_IF(fp8_check(op, "out", out, false, true, &a.out));
  MI_RETURN_IF(fp8_check_wide(op, "x", x, true));
  MI_RETURN_IF(check_shape(op, out, x, "x"));
  MI_RETURN_IF(check_outputs_apart(op, out, "x", x));
  if (numel(*x) == 0) return MI_OK;
  a.x = x->data;
  a.x_ld = x->strides[0];
  a.rows = x->sizes[0];
  a.cols = (int)x->sizes[1];
  hipStream_t s = (hipStream_t)stream;
  if (x->dtype == MI_BF16) return launch_quantize<BF16>(a, s, op);
  return x->dtype == MI_F16 ? launch_quantize<F16>(a, s, op) : launch_quantize<float>(a, s, op);
}

mi_status_t mi_fp8_quantize_weight(const mi_fp8_t* out, const mi_tensor_t* weight, mi_stream_t stream) {
  clear_error();
  const char* op = "fp8_quantize_weight";
  Fp8Mat m;
  MI_RETURN_IF(fp8_check(op, "out", out, true, true, &m));
  MI_RETURN_IF(fp8_check_wide(op, "weight", weight, true));
  MI_RETURN_IF(check_shape(op, out, weight, "weight"));
  MI_RETURN_IF(check_outputs_apart(op, out, "weight", weight));
  if (numel(*weight) == 0) return MI_OK;
  const int64_t rows = weight->sizes[0], cols = weight->sizes[1], ld = weight->strides[0];
  if (fp8_groups(rows) > 65535 || fp8_groups(cols) >= (1 << 23))
    MI_FAIL(MI_ERR_TOO_LARGE, "%s: more than 65535 x 128 rows, or 2^30 - 127 columns", op);
  const dim3 grid((unsigned)fp8_groups(cols), (unsigned)fp8_groups(rows));
  auto go = [&](auto type) {
    hipLaunchKernelGGL((fp8_weight_kernel<decltype(type)>), grid, dim3(512), 0, (hipStream_t)stream,
                       weight->data, ld, rows, (int)cols, m);
    return check_launch(op);
  };
  return weight->dtype == MI_BF16 ? go(BF16{}) : weight->dtype == MI_F16 ? go(F16{}) : go(0.f);
}

mi_status_t mi_rms_norm_fp8(const mi_fp8_t* out, const mi_tensor_t* total, const mi_tensor_t* x,
                            const mi_tensor_t* residual, const mi_tensor_t* weight, double eps,
                            mi_stream_t stream) {
  clear_error();
  const char* op = "rms_norm_fp8";
  RowsArgs a{};
  MI_RETURN_IF(fp8_check(op, "out", out, false, true, &a.out));
  MI_RETURN_IF(fp8_check_wide(op, "x", x, true));
  MI_RETURN_IF(check_shape(op, out, x, "x"));
  MI_RETURN_IF(check_outputs_apart(op, out, "x", x));
  const bool has_res = residual != nullptr && residual->data != nullptr;
  const bool has_w = weight != nullptr && weight->data != nullptr;
  if (has_res) {
    MI_CHECK_ARG(total != nullptr, "%s: total is NULL", op);
    const mi_tensor_t* ts[2] = {residual, total};
    const char* names[2] = {"residual", "total"};
    for (int i = 0; i < 2; ++i) {
      MI_RETURN_IF(fp8_check_wide(op, names[i], ts[i], true));
      MI_CHECK_ARG(ts[i]->dtype == x->dtype && ts[i]->sizes[0] == x->sizes[0] &&
                       ts[i]->sizes[1] == x->sizes[1],
                   "%s: %s must have x's shape and type", op, names[i]);
    }
    for (int i = 0; i < 2; ++i) {
      MI_RETURN_IF(check_outputs_apart(op, out, names[i], ts[i]));
      // total may be the same tensor as an input: a thread reads what it writes
      const mi_tensor_t* in = i == 0 ? x : residual;
      if (!(in->data == total->data && (in->sizes[0] <= 1 || in->strides[0] == total->strides[0])))
        MI_RETURN_IF(fp8_check_apart(op, "total", total, i == 0 ? "x" : "residual", in));
    }
    MI_CHECK_ARG(total->sizes[0] <= 1 || total->strides[0] >= total->sizes[1], "%s: rows of total overlap",
                 op);
    a.res = residual->data;
    a.res_ld = residual->strides[0];
    a.total = total->data;
    a.total_ld = total->strides[0];
  }
  if (has_w) {
    MI_RETURN_IF(validate(weight, "weight"));
    MI_CHECK_ARG(weight->ndim == 1 && weight->sizes[0] == x->sizes[1] && weight->dtype == x->dtype &&
                     (weight->sizes[0] <= 1 || weight->strides[0] == 1),
                 "%s: weight must be a dense vector of x's type and columns", op);
    MI_RETURN_IF(check_outputs_apart(op, out, "weight", weight));
    if (has_res) MI_RETURN_IF(fp8_check_apart(op, "total", total, "weight", weight));
    a.weight = weight->data;
  }
  if (has_res) {
    MI_RETURN_IF(fp8_check_apart(op, "total", total, "codes", &out->codes));
    MI_RETURN_IF(fp8_check_apart(op, "total", total, "scales", &out->scales));
  }
  if (numel(*x) == 0) return MI_OK;
  a.x = x->data;
  a.x_ld = x->strides[0];
  a.rows = x->sizes[0];
  a.cols = (int)x->sizes[1];
  a.eps = (float)eps;
  return has_res ? run_norm<NORM_RES>(a, x->dtype, (hipStream_t)stream, op)
                 : run_norm<NORM>(a, x->dtype, (hipStream_t)stream, op);
}

}  // extern "C"
