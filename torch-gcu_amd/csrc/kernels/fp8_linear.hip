// Products of activations and a weight in 8-bit floating point, and the gate and up
// products of a feed-forward layer with silu(gate) up as codes again.
#include "fp8_rows.h"

namespace mi {
namespace {

typedef F8Cfg<2, 2, 128, 128, 2> F256;  // 256 x 256 (a gate's 128 gate and 128 up columns)
typedef F8Cfg<2, 2, 64, 64, 2> F128;
typedef F8Cfg<2, 2, 32, 64, 2> F64x128;
typedef F8Cfg<2, 2, 32, 32, 4> F64;
typedef F8Cfg<2, 4, 64, 64, 2> G128;    // a gate's 128 x (128 and 128)
typedef F8Cfg<2, 4, 32, 64, 2> G64;

// out = the slices' sums in order (+ bias) (+ residual), 4 columns a thread
__global__ __launch_bounds__(256) void fp8_combine_kernel(Fp8Gemm p, int S) {
  const int64_t runs = p.ldp / 4, idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = idx / runs;
  const int n = (int)(idx - m * runs) * 4;
  if (m >= p.M) return;
  const float* src = p.part + m * p.ldp + n;
  f32x4_t s = *(const f32x4_t*)src;
#pragma unroll 4
  for (int i = 1; i < S; ++i) s += *(const f32x4_t*)(src + i * (p.M * p.ldp));
  auto wide = [&](uint16_t v) __attribute__((always_inline)) { return p.f16 ? f16_to_f32(v) : bf16_to_f32(v); };
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= p.N) break;
    float y = s[e];
    if (p.bias != nullptr)
      y += p.bias_dtype == MI_F32 ? ((const float*)p.bias)[n + e] : wide(((const uint16_t*)p.bias)[n + e]);
    if (p.res != nullptr) y += wide(p.res[m * p.ldr + n + e]);
    ((uint16_t*)p.out)[m * p.ldc + n + e] = p.f16 ? f32_to_f16(y) : f32_to_bf16(y);
  }
}

// silu(gate) up of the slices' sums, and its codes: 32 lanes a group of 128 columns
__global__ __launch_bounds__(256) void fp8_gate_combine_kernel(Fp8Gemm p, int S) {
  const int groups = (p.N + kFp8Group - 1) / kFp8Group;
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t m = id / groups;
  const int group = (int)(id - m * groups), n = group * kFp8Group + 4 * (threadIdx.x & 31);
  const bool live = m < p.M;
  float y[4] = {}, mine = 0.f;
  if (live && n < p.N) {
    const int64_t slice = p.M * p.ldp;
    const float* src = p.part + m * p.ldp + n;
    f32x4_t g = *(const f32x4_t*)src, u = *(const f32x4_t*)(src + S * slice);
#pragma unroll 4
    for (int i = 1; i < S; ++i) {
      g += *(const f32x4_t*)(src + i * slice);
      u += *(const f32x4_t*)(src + (S + i) * slice);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) y[e] = gate_of(g[e], u[e], &mine);
  }
  uint32_t most = row16_max(__float_as_uint(mine));
  most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
  if (!live) return;
  const uint32_t byte = fp8_scale_byte(most);
  const uint32_t c = fp8_codes4(y[0], y[1], y[2], y[3], fp8_inverse(byte));
  uint8_t* dst = p.codes.codes + m * p.codes.ld + n;
  if (n + 3 < p.N && (uintptr_t)dst % 4 == 0) {
    *(uint32_t*)dst = c;
  } else {
    for (int e = 0; e < 4 && n + e < p.N; ++e) dst[e] = (uint8_t)(c >> (8 * e));
  }
  if ((threadIdx.x & 31) == 0) p.codes.scales[m * p.codes.sld + group] = (uint8_t)byte;
}

mi_status_t launch_combine(const Fp8Gemm& q, bool gate, int S, hipStream_t s, const char* op) {
  if (gate)
    hipLaunchKernelGGL(fp8_gate_combine_kernel, dim3(ceil_div_u(q.M * fp8_groups(q.N), 8)), dim3(256), 0, s, q, S);
  else
    hipLaunchKernelGGL(fp8_combine_kernel, dim3(ceil_div_u(q.M * (q.ldp / 4), 256)), dim3(256), 0, s, q, S);
  return check_launch(op);
}

// A grid's first dimension holds fewer than 2^32 threads.
mi_status_t check_grid(int64_t blocks, int threads, const char* op) {
  if (blocks * threads >= (int64_t)1 << 32) MI_FAIL(MI_ERR_TOO_LARGE, "%s: too many outputs", op);
  return MI_OK;
}

template <class C, int EPI>
mi_status_t launch_tiles(Fp8Gemm q, int S, hipStream_t s, const char* op) {
  static const bool attr = [] {
    (void)hipFuncSetAttribute((const void*)fp8_gemm_kernel<C, EPI>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)C::LDS_BYTES);
    return true;
  }();
  (void)attr;
  constexpr int BN = EPI == F8_GATE || EPI == F8_GATE_PART ? C::BN / 2 : C::BN;
  q.tiles_m = (q.M + C::BM - 1) / C::BM;
  q.tiles_n = (q.N + BN - 1) / BN;
  MI_RETURN_IF(check_grid((int64_t)q.tiles_m * q.tiles_n, C::NT, op));
  hipLaunchKernelGGL((fp8_gemm_kernel<C, EPI>), dim3((unsigned)(q.tiles_m * q.tiles_n), (unsigned)S),
                     dim3(C::NT), C::LDS_BYTES, s, q);
  return check_launch(op);
}

template <class C, bool GATE>
mi_status_t launch(const Fp8Gemm& q, hipStream_t s, const char* op) {
  return launch_tiles<C, GATE ? F8_GATE : F8_OUT>(q, 1, s, op);
}

// One launch, or S slices of K and their sum.
template <class C, bool GATE>
mi_status_t launch_slices(Fp8Gemm q, int S, hipStream_t s, const char* op) {
  Workspace ws;
  q.ldp = ((int64_t)q.N + 3) / 4 * 4;
  if (S > 1 && ws.alloc((size_t)(GATE ? 2 : 1) * S * q.M * q.ldp * sizeof(float), s) != MI_OK) {
    clear_error();  // the whole K in one block needs no workspace
    S = 1;
  }
  if (S <= 1) return launch<C, GATE>(q, s, op);
  q.part = (float*)ws.get();
  MI_RETURN_IF((launch_tiles<C, GATE ? F8_GATE_PART : F8_PART>(q, S, s, op)));
  return launch_combine(q, GATE, S, s, op);
}

// Few rows of activations: one launch, or for a gate its y in float32 and then the codes.
template <class C, bool GATE>
mi_status_t launch_few(Fp8Gemm q, hipStream_t s, const char* op) {
  static const bool attr = [] {
    (void)hipFuncSetAttribute((const void*)fp8_rows_gemm_kernel<C, GATE>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    return true;
  }();
  (void)attr;
  constexpr int COLS = 16 * (GATE ? C::RT / 2 : C::RT);
  MI_RETURN_IF(check_grid(((int64_t)q.N + COLS - 1) / COLS, 64 * C::NW, op));
  Workspace ws;
  if (GATE) {
    q.ldp = ((int64_t)q.N + 3) / 4 * 4;
    MI_RETURN_IF(ws.alloc((size_t)(q.M * q.ldp) * sizeof(float), s));
    q.part = (float*)ws.get();
  }
  hipLaunchKernelGGL((fp8_rows_gemm_kernel<C, GATE>), dim3(ceil_div_u(q.N, COLS)), dim3(64 * C::NW),
                     C::F.lds((size_t)fp8_groups(q.K)), s, q);
  MI_RETURN_IF(check_launch(op));
  return GATE ? fp8_quantize_f32(q.part, q.ldp, q.M, q.N, q.codes, s, op) : MI_OK;
}

template <class C, bool GATE>
constexpr bool is_shape(const Fp8Shape& s) {
  return s.bm == C::BM && s.bn == (GATE ? C::BN / 2 : C::BN) &&
         (s.per_cu == (int)(kFp8Lds / C::LDS_BYTES) || (s.per_cu == 2 && C::LDS_BYTES * 2 <= kFp8Lds));
}
static_assert(is_shape<F256, false>(kFp8Shapes[0]) && is_shape<F128, false>(kFp8Shapes[1]) &&
                  is_shape<F64x128, false>(kFp8Shapes[2]) && is_shape<F64, false>(kFp8Shapes[3]) &&
                  is_shape<F256, true>(kFp8GateShapes[0]) && is_shape<G128, true>(kFp8GateShapes[1]) &&
                  is_shape<G64, true>(kFp8GateShapes[2]),
              "the rule's shapes are the kernels', with no more blocks a CU than its LDS holds");

// Up to 16 rows: no more columns than a few-row kernel's grid holds, whichever way is taken.
mi_status_t check_columns(const Fp8Gemm& q, const Fp8Few& f, const char* op) {
  return q.M <= 16 ? check_grid(((int64_t)q.N + 15) / 16, 64 * f.nw, op) : MI_OK;
}

template <int I = 0>
mi_status_t run_few(int i, const Fp8Gemm& q, hipStream_t s, const char* op) {
  if constexpr (I < (int)(sizeof(kFp8Few) / sizeof(kFp8Few[0])))
    return i == I ? launch_few<R8Cfg<kFp8Few, I>, false>(q, s, op) : run_few<I + 1>(i, q, s, op);
  MI_FAIL(MI_ERR_INVALID, "%s: no such kernel", op);
}
template <int I = 0>
mi_status_t run_gate_few(int i, const Fp8Gemm& q, hipStream_t s, const char* op) {
  if constexpr (I < (int)(sizeof(kFp8GateFew) / sizeof(kFp8GateFew[0])))
    return i == I ? launch_few<R8Cfg<kFp8GateFew, I>, true>(q, s, op) : run_gate_few<I + 1>(i, q, s, op);
  MI_FAIL(MI_ERR_INVALID, "%s: no such kernel", op);
}

mi_status_t run_linear(const Fp8Gemm& q, hipStream_t s, const char* op) {
  MI_RETURN_IF(check_columns(q, kFp8Few[0], op));
  const Fp8Way c = fp8_pick_linear(q.M, q.N, q.K, cu_count());
  if (c.few >= 0) return run_few(c.few, q, s, op);
  switch (c.shape) {
    case 0: return launch<F256, false>(q, s, op);
    case 1: return launch<F128, false>(q, s, op);
    case 2: return launch<F64x128, false>(q, s, op);
    default: return launch_slices<F64, false>(q, c.slices, s, op);
  }
}

mi_status_t run_gate(const Fp8Gemm& q, hipStream_t s, const char* op) {
  MI_RETURN_IF(check_columns(q, kFp8GateFew[0], op));
  const Fp8Way c = fp8_pick_gate(q.M, q.N, q.K, cu_count());
  if (c.few >= 0) return run_gate_few(c.few, q, s, op);
  switch (c.shape) {
    case 0: return launch<F256, true>(q, s, op);
    case 1: return launch<G128, true>(q, s, op);
    default: return launch_slices<G64, true>(q, c.slices, s, op);
  }
}

// Offsets inside a block's 256 rows are 32-bit byte counts.
constexpr int64_t kFarRows = 1 << 22;

// Rows of 16-byte aligned codes, and scales whose rows are near: the operand itself, or
// copies in workspace.
mi_status_t aligned_rows(const mi_fp8_t* t, Fp8Mat* m, Workspace* ws, hipStream_t s) {
  const int64_t rows = t->codes.sizes[0], cols = t->codes.sizes[1];
  if (t->scales.sizes[0] <= 1) {
    m->sld = 0;
  } else if (m->sld >= kFarRows) {
    mi_tensor_t to = t->scales;
    to.strides[0] = to.sizes[1];
    to.strides[1] = 1;
    MI_RETURN_IF(ws[1].alloc((size_t)(to.sizes[0] * to.sizes[1]), s));
    to.data = ws[1].get();
    MI_RETURN_IF(mi_copy(&to, &t->scales, (mi_stream_t)s));
    m->scales = (uint8_t*)to.data;
    m->sld = to.sizes[1];
  }
  if ((uintptr_t)m->codes % 16 == 0 && ((m->ld % 16 == 0 && m->ld < kFarRows) || rows <= 1)) {
    if (rows <= 1) m->ld = 0;
    return MI_OK;
  }
  const int64_t ld = (cols + 15) / 16 * 16;
  MI_RETURN_IF(ws->alloc((size_t)(rows * ld), s));
  mi_tensor_t to = t->codes;
  to.data = ws->get();
  to.strides[0] = ld;
  to.strides[1] = 1;
  MI_RETURN_IF(mi_copy(&to, &t->codes, (mi_stream_t)s));
  m->codes = (uint8_t*)ws->get();
  m->ld = ld;
  return MI_OK;
}

mi_status_t check_product(const char* op, const mi_fp8_t* x, const mi_fp8_t* w, const char* name,
                          Fp8Gemm* q) {
  MI_CHECK_ARG(x->codes.sizes[1] == w->codes.sizes[1], "%s: x has %lld columns, %s %lld", op,
               (long long)x->codes.sizes[1], name, (long long)w->codes.sizes[1]);
  q->M = (int)x->codes.sizes[0];
  q->N = (int)w->codes.sizes[0];
  q->K = (int)x->codes.sizes[1];
  // (tiles are at least 64 x 64, and counted in 31 bits)
  const int64_t tiles = (((int64_t)q->M + 63) / 64) * (((int64_t)q->N + 63) / 64);
  if (q->K > kFarRows - 16 || tiles > 0x7fffffff || q->M > 0x7fff0000 || q->N > 0x7fff0000)
    MI_FAIL(MI_ERR_TOO_LARGE, "%s: more than 2^22 - 16 columns, or too many outputs", op);
  return MI_OK;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

mi_status_t mi_fp8_linear(const mi_tensor_t* out, const mi_fp8_t* x, const mi_fp8_t* weight,
                          const mi_tensor_t* bias, const mi_tensor_t* residual, mi_stream_t stream) {
  clear_error();
  const char* op = "fp8_linear";
  hipStream_t s = (hipStream_t)stream;
  Fp8Gemm q{};
  MI_RETURN_IF(fp8_check(op, "x", x, false, false, &q.x));
  MI_RETURN_IF(fp8_check(op, "weight", weight, true, false, &q.w));
  MI_RETURN_IF(check_product(op, x, weight, "weight", &q));
  MI_RETURN_IF(fp8_check_wide(op, "out", out, false));
  MI_CHECK_ARG(out->sizes[0] == q.M && out->sizes[1] == q.N, "%s: out is [%lld, %lld], expected [%d, %d]",
               op, (long long)out->sizes[0], (long long)out->sizes[1], q.M, q.N);
  MI_CHECK_ARG(q.M <= 1 || out->strides[0] >= q.N, "%s: rows of out overlap", op);
  for (const mi_fp8_t* t : {x, weight}) {
    MI_RETURN_IF(fp8_check_apart(op, "out", out, "codes", &t->codes));
    MI_RETURN_IF(fp8_check_apart(op, "out", out, "scales", &t->scales));
  }
  if (bias != nullptr && bias->data != nullptr) {
    MI_RETURN_IF(validate(bias, "bias"));
    MI_CHECK_ARG(bias->ndim == 1 && bias->sizes[0] == q.N && (q.N <= 1 || bias->strides[0] == 1) &&
                     (bias->dtype == out->dtype || bias->dtype == MI_F32),
                 "%s: bias must be a dense vector of %d, of out's type or float32", op, q.N);
    MI_RETURN_IF(fp8_check_apart(op, "out", out, "bias", bias));
    q.bias = bias->data;
    q.bias_dtype = bias->dtype;
  }
  if (residual != nullptr && residual->data != nullptr) {
    MI_RETURN_IF(fp8_check_wide(op, "residual", residual, false));
    MI_CHECK_ARG(residual->dtype == out->dtype && residual->sizes[0] == q.M && residual->sizes[1] == q.N,
                 "%s: residual must have out's shape and type", op);
    // an element is read by the thread that writes it
    if (!(residual->data == out->data && (q.M <= 1 || residual->strides[0] == out->strides[0])))
      MI_RETURN_IF(fp8_check_apart(op, "out", out, "residual", residual));
    q.res = (const uint16_t*)residual->data;
    q.ldr = residual->strides[0];
  }
  if (q.M == 0 || q.N == 0) return MI_OK;
  q.out = out->data;
  q.ldc = out->strides[0];
  q.f16 = out->dtype == MI_F16;
  Workspace wx[2], ww[2];
  MI_RETURN_IF(aligned_rows(x, &q.x, wx, s));
  MI_RETURN_IF(aligned_rows(weight, &q.w, ww, s));
  return run_linear(q, s, op);
}

mi_status_t mi_fp8_linear_silu_mul(const mi_fp8_t* out, const mi_fp8_t* x, const mi_fp8_t* w_gate,
                                   const mi_fp8_t* w_up, mi_stream_t stream) {
  clear_error();
  const char* op = "fp8_linear_silu_mul";
  hipStream_t s = (hipStream_t)stream;
  Fp8Gemm q{};
  MI_RETURN_IF(fp8_check(op, "x", x, false, false, &q.x));
  MI_RETURN_IF(fp8_check(op, "w_gate", w_gate, true, false, &q.w));
  MI_RETURN_IF(fp8_check(op, "w_up", w_up, true, false, &q.w2));
  MI_RETURN_IF(fp8_check(op, "out", out, false, true, &q.codes));
  MI_RETURN_IF(check_product(op, x, w_gate, "w_gate", &q));
  MI_CHECK_ARG(w_up->codes.sizes[0] == q.N && w_up->codes.sizes[1] == q.K,
               "%s: w_gate and w_up have different shapes", op);
  MI_CHECK_ARG(out->codes.sizes[0] == q.M && out->codes.sizes[1] == q.N,
               "%s: codes are [%lld, %lld], expected [%d, %d]", op, (long long)out->codes.sizes[0],
               (long long)out->codes.sizes[1], q.M, q.N);
  for (const mi_fp8_t* t : {x, w_gate, w_up})
    for (const mi_tensor_t* mine : {&out->codes, &out->scales}) {
      MI_RETURN_IF(fp8_check_apart(op, "out", mine, "codes", &t->codes));
      MI_RETURN_IF(fp8_check_apart(op, "out", mine, "scales", &t->scales));
    }
  if (q.M == 0 || q.N == 0) return MI_OK;
  Workspace wx[2], wg[2], wu[2];
  MI_RETURN_IF(aligned_rows(x, &q.x, wx, s));
  MI_RETURN_IF(aligned_rows(w_gate, &q.w, wg, s));
  MI_RETURN_IF(aligned_rows(w_up, &q.w2, wu, s));
  return run_gate(q, s, op);
}

}  // extern "C"
