// The tile kernel of 8-bit floating point products, by block shapes (fp8_linear.hip
// chooses one).
//
// out[m][n] = sum over k of x[m][k] w[n][k], an element being code 2^(scale byte - 127).
// One matrix instruction multiplies 128 of K and its scales with them, so a group of 128
// columns with one scale is one instruction's K, and nothing is left to do for scales but
// to hand their bytes over.  The instruction adds 8 neighbours of K at a time with 13 bits
// below the largest of them, and those sums in fp32: 1.5e-5 of a sum of normal numbers, a
// thirteenth of an f16 output's rounding, and next to e4m3's own 2^-4 an element of no
// account; so outputs are 16 bits or codes, and float32 ones are not offered.  The 8-bit
// instructions without scales add so too; the 16-bit ones, which codes would have to be
// widened for, keep 23 bits (5e-9) at less than half the rate (this library's product of 16
// bits takes 558 us for M8192 N4096 K11008).
//
// A block copies K steps of 128 of its rows of x and w straight to an LDS ring (swizzled,
// so that fragments are read without conflicts), and its waves multiply from there.
//
// What bounds it: of 256 x 256 tiles the matrix unit under the card's power limit.  M8192
// N4096 K11008 with a residual takes 264 us (2.8 PFLOP/s): a step 2380 to 2560 cycles where
// its products need 2048, at 1.9 to 2.0 GHz (2.4 with operands of zeros), and 10 us a tile
// of first copies and epilogue, which nothing overlaps (one block a CU fills registers and
// LDS).  Four waves of 128 x 128 outputs read a third less from LDS than eight of 64 x 128,
// which were 5 % slower.  (Were every copy a hit of its XCD's cache, another 5 % less; copies made
// ahead into that cache, of lines or of single bytes, were slower.)  Of the smaller tiles
// the copies to LDS: M777 N4096 K4096 by 224 tiles of 128 x 128, whose weight the last-level
// cache holds, 235 MB in its 19 us at 18 to 20 TB/s (1.37 PFLOP/s).  Where the weight comes
// from HBM it is rather their latency: M355 N7616 K10880 has 180 such tiles, 32 to 64 KiB in
// flight on each of as many CUs, and copies 500 MB in its 48 us (11 TB/s).
#pragma once

#include "fp8_common.h"
#include "gemm_dl.h"

namespace mi {

struct Fp8Gemm {
  Fp8Mat x, w, w2;     // activations [M][K], weight [N][K]; w2: the up weight of a gate
  void* out;           // [M][ldc] bf16 or f16
  int64_t ldc;
  const void* bias;
  int bias_dtype;
  const uint16_t* res;
  int64_t ldr;
  Fp8Mat codes;        // a gate's output
  float* part;         // [2 of a gate][slices][M][ldp] sums of K slices
  int64_t ldp;
  int M, N, K;
  int f16;             // out, residual and 16-bit bias are f16
  int tiles_m, tiles_n;
};

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

// acc += a b^T over 128 of K: lane l holds 32 bytes of row l % 16 of each operand
// (the same 32 of the 128 in both) and ends up with rows 4 (l / 16) + 0 .. 3 of
// column l % 16.  A scale multiplies a lane's 32 products; here the four lanes of a
// row give the same one.  (Format 0 is e4m3.)
__device__ __forceinline__ f32x4_t mma_fp8(i32x8_t a, i32x8_t b, f32x4_t c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// A byte a lane, from a wave-uniform base and a 32-bit offset of its own, to a 32-bit
// word a lane at lds on (the counterpart of lds_copy16).
__device__ __forceinline__ void lds_copy_byte(const uint8_t* base, uint32_t off, void* lds) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds);
  const uint64_t b = (uint64_t)base;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)b);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
  const uint64_t sb = ((uint64_t)hi << 32) | lo;
  uint64_t at;  // (as in lds_copy16)
  asm volatile("s_mov_b64 %0, %2\n\tglobal_load_lds_ubyte %1, %0" : "=&s"(at) : "v"(off), "s"(sb), "{m0}"(m0)
               : "memory");
}

// silu(g) u, NaN where it is not finite, and the largest magnitude so far
__device__ __forceinline__ float gate_of(float g, float u, float* most) {
  const float y = fp8_no_inf(silu_mul_f32(g, u));
  *most = fp8_larger(*most, y);
  return y;
}

constexpr int F8_OUT = 0, F8_PART = 1, F8_GATE = 2, F8_GATE_PART = 3;

// WM x WN waves of TM x TN outputs each, K steps of 128 through a ring of STAGES.
template <int WM_, int WN_, int TM_, int TN_, int STAGES_>
struct F8Cfg {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, STAGES = STAGES_;
  static constexpr int NW = WM * WN, NT = 64 * NW, BM = WM * TM, BN = WN * TN;
  static constexpr int FM = TM / 16, FN = TN / 16;
  static constexpr int RB = FN < 8 ? 2 : 4;  // weight fragments held
  // 1 KiB wave copies a step: the activations' and of the weight the rows of each wave's
  // first RB fragments, then the others'
  static constexpr int NQA = BM / 8 / NW, NQB = BN / 8 / NW, NQL = NQB * RB / FN;
  static constexpr int LPW = NQA + NQB;
  // one wave a SIMD, whose registers hold the next step's activations too
  static constexpr bool PAIRS = TM * TN > 64 * 128;
  static constexpr int TA = BM * 128, TB = BN * 128, STAGE = TA + TB;
  // scales of KS K steps at a time, a word each, two of such sets in turn: 64 / KS rows a
  // wave copy, then the weight's blocks (KS 8, or 4 where the LDS has no room for those)
  static constexpr int KS = STAGES * STAGE + 2 * (BM * 32 + 512) <= 160 * 1024 ? 8 : 4;
  static constexpr int NQS = (BM * KS / 64 + NW - 1) / NW, SET = BM * KS * 4 + 512, SCALES = STAGES * STAGE;
  static constexpr int HC = TN < 64 ? TN : 64, EP = HC + 4;  // columns of an epilogue pass
  static constexpr int CP = 128 + 16;                         // a gate's staged code rows
  static constexpr size_t cmax(size_t a, size_t b) { return a > b ? a : b; }
  static constexpr size_t LDS_BYTES =
      cmax((size_t)SCALES + 2 * SET, cmax((size_t)NW * TM * EP * 4, (size_t)BM * CP + (size_t)WN * BM * 4));
  static_assert(LDS_BYTES <= 160 * 1024 && NQA >= 1 && NQB >= 1 && FN % RB == 0 && NQL * FN == NQB * RB &&
                    (STAGES - 1) * LPW < 64, "shape");
  static_assert(!PAIRS || (FM == 8 && FN == 8 && NQA == 8 && NQB == 8 && STAGES == 2), "the order of its step");
  // a set of scales is written while the one before it is still read
  static_assert(KS >= STAGES, "sets");
};

template <class C, int EPI>
__global__ __launch_bounds__(C::NT, C::PAIRS ? 1 : 2) void fp8_gemm_kernel(Fp8Gemm p) {
  constexpr int WN = C::WN, TM = C::TM, TN = C::TN, BM = C::BM, BN = C::BN, FM = C::FM, FN = C::FN;
  constexpr int RB = C::RB, NQA = C::NQA, NQB = C::NQB, NQL = C::NQL, LPW = C::LPW, STAGES = C::STAGES;
  constexpr int KS = C::KS, NQS = C::NQS, SET = C::SET, SC = BM * KS / 64;
  constexpr int TA = C::TA, STAGE = C::STAGE, GROUP_M = 8;
  constexpr bool PAIRS = C::PAIRS;
  constexpr bool GATE = EPI == F8_GATE || EPI == F8_GATE_PART;
  constexpr bool SPLIT = EPI == F8_PART || EPI == F8_GATE_PART;
  static_assert(EPI != F8_GATE || BN == 256, "a block holds whole groups of a gate's output");
  extern __shared__ __align__(16) char smem[];
  // XCD-aware tile order (blocks go round the 8 XCDs in turn), then groups of
  // GROUP_M row panels, so the tiles an XCD runs together share panels
  int tm, tn;
  {
    const int total = p.tiles_m * p.tiles_n, xcd = blockIdx.x % 8;
    const int id = xcd * (total / 8) + min(xcd, total % 8) + blockIdx.x / 8;
    const int group = id / (GROUP_M * p.tiles_n), first = group * GROUP_M;
    const int size = min(p.tiles_m - first, GROUP_M), in_group = id - group * GROUP_M * p.tiles_n;
    tm = first + in_group % size;
    tn = in_group / size;
  }
  const int M = p.M, N = p.N, K = p.K;
  const int m0 = tm * BM, n0 = tn * (GATE ? BN / 2 : BN);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int KT = K / 128, k_first = 0;
  if constexpr (SPLIT) {
    const int S = gridDim.y, s = blockIdx.y, base = KT / S, rem = KT % S;
    k_first = s * base + min(s, rem);
    KT = base + (s < rem ? 1 : 0);
  }
  // The weight row of row r of the B tile.  A gate's wave holds TN / 2 columns of
  // the gate and the same of up, so a lane has both products of an output.
  auto b_row = [&](int r) __attribute__((always_inline)) {
    return GATE ? n0 + r / TN * (TN / 2) + r % (TN / 2) : n0 + r;
  };
  auto b_up = [&](int r) __attribute__((always_inline)) { return GATE && r % TN >= TN / 2; };
  const uint8_t* A = p.x.codes + (int64_t)m0 * p.x.ld;
  const uint8_t* B[2] = {p.w.codes + (int64_t)n0 * p.w.ld, GATE ? p.w2.codes + (int64_t)n0 * p.w2.ld : nullptr};
  // byte offsets of a lane's 16 bytes of each copy (8 rows of 128 bytes), which fit 32
  // bits; rows past the matrix read its last one and feed outputs that are not stored.
  // LDS chunk c of row r holds the row's chunk dl_swz(r, c).
  uint32_t ao[NQA], bo[NQB];
  // the 8 rows of the B tile that copy q of the wave takes (q < NQL: of first fragments)
  auto b_copy = [&](int q) __attribute__((always_inline)) {
    if (PAIRS) return wave * NQB + q;
    const bool lo = q < NQL;
    const int i = lo ? wave * NQL + q : wave * (NQB - NQL) + q - NQL, per = 2 * (lo ? RB : FN - RB);
    return i / per * (TN / 8) + (lo ? 0 : 2 * RB) + i % per;
  };
#pragma unroll
  for (int q = 0; q < NQA; ++q) {
    const int r = (wave * NQA + q) * 8 + lane / 8;
    ao[q] = (uint32_t)((min(m0 + r, M - 1) - m0) * p.x.ld + 16 * dl_swz(r, lane % 8));
  }
#pragma unroll
  for (int q = 0; q < NQB; ++q) {
    const int r = b_copy(q) * 8 + lane / 8;
    bo[q] = (uint32_t)((min(b_row(r), N - 1) - n0) * (b_up(r) ? p.w2.ld : p.w.ld) + 16 * dl_swz(r, lane % 8));
  }
  // The scales of set `set` (of the whole K): lane l of a copy takes that of row l / KS (of
  // the weight's block l / KS) at the set's K step l % KS.  (A copy so takes 8 bytes of 8
  // rows: a step's bytes of 64 rows, each in a cache line of its own, made M8192 N4096
  // K11008 10 % slower.)  The offsets are made anew each time: kept, they cost registers
  // that the main loop has not.
  const int KB = (K + 127) / 128;
  const uint8_t* xs = p.x.scales + (int64_t)m0 * p.x.sld;
  constexpr int NBLK = GATE ? 1 : (BN + 127) / 128;  // blocks of one weight in a tile
  const uint8_t* ws = p.w.scales + (int64_t)(n0 / kFp8Group) * p.w.sld;
  auto issue_scales = [&](int set) __attribute__((always_inline)) {
    char* s = smem + C::SCALES + (set & 1) * SET;
    int l = lane;
    asm volatile("" : "+v"(l));
    const int k = min(set * KS + l % KS, KB - 1);
#pragma unroll
    for (int q = 0; q < NQS; ++q) {
      const int c = (wave * NQS + q) % SC;
      lds_copy_byte(xs, (uint32_t)(min(c * (64 / KS) + l / KS, M - 1 - m0) * (int)p.x.sld + k), s + c * 256);
    }
    if (wave == C::NW - 1) {
      const int last = (N - 1) / kFp8Group - n0 / kFp8Group;
      lds_copy_byte(ws, (uint32_t)(min(l / KS % NBLK, last) * (int)p.w.sld + k), s + BM * KS * 4);
    }
    if (GATE && wave == C::NW - 2)
      lds_copy_byte(p.w2.scales + (int64_t)(n0 / kFp8Group) * p.w2.sld, (uint32_t)k, s + BM * KS * 4 + 256);
  };
  // copy q of K step kt (of this slice) into stage st
  auto issue_one = [&](int st, int kt, int q) __attribute__((always_inline)) {
    char* s = smem + st * STAGE;
    const int64_t k = (int64_t)(k_first + kt) * 128;
    if (q < NQA) {
      lds_copy16(A + k, ao[q], s + (wave * NQA + q) * 1024);
    } else {
      const int c = b_copy(q - NQA);
      lds_copy16((b_up(c * 8) ? B[1] : B[0]) + k, bo[q - NQA], s + TA + c * 1024);
    }
  };
  auto issue = [&](int st, int kt, int copies) __attribute__((always_inline)) {
    if (kt == 0 || (k_first + kt) % KS == 0) issue_scales((k_first + kt) / KS);
#pragma unroll
    for (int q = 0; q < copies; ++q) issue_one(st, kt, q);
  };
  // fragments: lane l reads row l % 16, chunks l / 16 (half 0) and 4 + l / 16
  const int row = lane & 15;
  const int ro[2] = {row * 128 + 16 * dl_swz(row, lane >> 4), row * 128 + 16 * dl_swz(row, 4 + (lane >> 4))};
  auto whole_of = [](const u32x4_t* v) __attribute__((always_inline)) {
    const u32x4_t lo = v[0], hi = v[1];
    return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  // acc[j][i]: outputs m = 16 i + l % 16, n = 16 j + 4 (l / 16) + 0 .. 3 of the wave's
  f32x4_t acc[FN][FM];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[j][i] = f32x4_t{};
  u32x4_t af[PAIRS ? 2 : 1][FM][2], bf[RB][2];
  int sa[FM], sb[2], sa_next[FM], sb_next[2];
  auto read_a = [&](int set, int st, int i, int h) __attribute__((always_inline)) {
    af[set][i][h] = *(const u32x4_t*)(smem + st * STAGE + (wm * TM + 16 * i) * 128 + ro[h]);
  };
  auto read_b = [&](int st, int j, int h) __attribute__((always_inline)) {
    bf[j % RB][h] = *(const u32x4_t*)(smem + st * STAGE + TA + (wn * TN + 16 * j) * 128 + ro[h]);
  };
  auto read_scales = [&](int kt) __attribute__((always_inline)) {
    const int k = k_first + kt;
    const int* s = (const int*)(smem + C::SCALES + (k / KS & 1) * SET) + k % KS;
#pragma unroll
    for (int i = 0; i < FM; ++i) sa_next[i] = s[(wm * TM + 16 * i + row) * KS];
#pragma unroll
    for (int h = 0; h < (GATE ? 2 : 1); ++h) sb_next[h] = s[BM * KS + (GATE ? 64 * h : wn * TN / 128 * KS)];
  };
  auto take_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[i] = sa_next[i];
    sb[0] = sb_next[0];
    if constexpr (GATE) sb[1] = sb_next[1];
  };
  auto mfma_one = [&](int set, int j, int i) __attribute__((always_inline)) {
    acc[j][i] =
        mma_fp8(whole_of(bf[j % RB]), whole_of(af[set][i]), acc[j][i], sb[GATE && j >= FN / 2 ? 1 : 0], sa[i]);
  };
  auto first_reads = [&](int st) __attribute__((always_inline)) {
    read_scales(0);
#pragma unroll
    for (int j = 0; j < RB - 1; ++j) read_b(st, j, 0), read_b(st, j, 1);
#pragma unroll
    for (int i = 0; i < FM; ++i) read_a(0, st, i, 0), read_a(0, st, i, 1);
    take_scales();
  };
  // One K step over stage st, a row of MFMAs (one weight fragment) at a time.  The weight
  // fragment RB - 1 rows on is read at each row's start, the activations' of the next
  // step during the last row, each behind its last use.  So the activations' part of a
  // stage and the rows of the first RB fragments have been read by row 1, the other rows
  // by row JB, from where the reads are the next step's.  Both refill as soon as they
  // have been read (a barrier tells), which keeps STAGES - 1 steps' copies in flight over
  // each wait: with one barrier a step, at row JB, that was STAGES - 2, and two stages
  // waited out a copy's whole latency every step.
  constexpr int JB = FN - RB + 1, NLO = NQA + NQL;  // copies behind the first barrier
  static_assert(JB > 1 || NQL == NQB, "one barrier where every fragment is read by row 1");
  constexpr int SLO = (JB > 1 ? JB - 1 : FN - 1) * FM, PLO = (NLO + SLO - 1) / SLO;
  constexpr int SHI = (FN - JB) * FM, PHI = (LPW - NLO + SHI - 1) / SHI;
  constexpr int AHEAD = (JB > 1 ? STAGES - 1 : STAGES - 2) * LPW;
  auto step = [&](int st, int kt, auto issue_c, auto next_c) __attribute__((always_inline)) {
    constexpr bool ISSUE = decltype(issue_c)::value, NEXT = decltype(next_c)::value;
    const int nst = st + 1 == STAGES ? 0 : st + 1;
    // (Here and not between the rows: the compiler sinks products that stand before a
    // branch to behind it.  A set's copies count as none in the waits, which are so a
    // little early.)
    if (ISSUE && (k_first + kt + STAGES) % KS == 0) issue_scales((k_first + kt + STAGES) / KS);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      if ((j == 1 && JB > 1) || (j == JB && NEXT)) {
        if (ISSUE) wait_vmcnt<AHEAD>();
        else wait_vmcnt<0>();
        __syncthreads();
        if (j == JB) read_scales(kt + 1);
      }
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        if (i == 0 || i == FM / 2) {
          if (j + RB - 1 < FN) read_b(st, j + RB - 1, i > 0);
          else if (NEXT) read_b(nst, j + RB - 1 - FN, i > 0);
        }
        mfma_one(0, j, i);
        if (j == FN - 1 && NEXT) read_a(0, nst, i, 0), read_a(0, nst, i, 1);
        if (ISSUE && j >= 1 && (j < JB || JB == 1))
#pragma unroll
          for (int u = 0; u < PLO; ++u) {
            const int q = ((j - 1) * FM + i) * PLO + u;
            if (q < NLO) issue_one(st, kt + STAGES, q);
          }
        if (ISSUE && j >= JB && JB > 1)
#pragma unroll
          for (int u = 0; u < PHI; ++u) {
            const int q = NLO + ((j - JB) * FM + i) * PHI + u;
            if (q < LPW) issue_one(st, kt + STAGES, q);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (NEXT) take_scales();
  };

  // One K step of PAIRS, with its activations in set NOW of the fragments: 64 products, and
  // between them, one at most, the halves of fragments and the copies that later steps
  // need.  (Two reads at a time cost 6 % of the cycles: one wave issues them all, and waits
  // where LDS is behind.)  The next step's activations are read in rows 1 to 4.  At row 5 a
  // barrier lets the stage's weight refill, and what holds the next step's activations in
  // the step after: 6 of the weight's copies come at once, the other 2 and those of the
  // activations in the next step.  So each copy has half a step or more until the barrier
  // that waits for it.
  auto pair_step = [&](auto set_c, int st, int kt, auto issue_c, auto next_c) __attribute__((always_inline)) {
    constexpr int NOW = decltype(set_c)::value;
    constexpr bool ISSUE = decltype(issue_c)::value, NEXT = decltype(next_c)::value;
    const int nst = 1 - st;
    if (ISSUE && (kt + 2) % KS == 0) issue_scales((kt + 2) / KS);
#pragma unroll
    for (int n = 0; n < FN * FM; ++n) {
      const int j = n / FM, i = n % FM;
      if (NEXT && (n == FM || n == 5 * FM)) {
        if (ISSUE) wait_vmcnt<8>();  // behind row 1's are the weight's 8, behind row 5's the activations'
        else wait_vmcnt<0>();
        __syncthreads();
        if (n > FM) read_scales(kt + 1);
      }
      if (i % 4 == 0) {
        if (j + RB - 1 < FN) read_b(st, j + RB - 1, i / 4);
        else if (NEXT) read_b(nst, j + RB - 1 - FN, i / 4);
      }
      if (NEXT && j >= 1 && j < 5 && n % 2 == 1) read_a(1 - NOW, nst, n / 4 - 2, n / 2 % 2);
      mfma_one(NOW, j, i);
      if (n % 4 == 2) {
        if (n < FM && NEXT) issue_one(nst, kt + 1, NQA + 6 + n / 4);
        if (j >= 1 && j < 5 && ISSUE) issue_one(st, kt + 2, n / 4 - 2);
        if (j >= 5 && ISSUE) issue_one(st, kt + 2, NQA + n / 4 - 10);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (NEXT) take_scales();
  };

  // Pairs of steps take an even number: an odd last one goes first and by itself, through
  // the last stage, as do the last K % 128 columns with zeros behind them.
  const int odd = PAIRS ? KT & 1 : 0;
  KT -= odd;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < KT) issue(s, s, LPW);
  auto alone = [&](bool tail) __attribute__((always_inline)) {
    const int kt0 = tail ? K / 128 : KT;
    if (!tail) {
#pragma unroll
      for (int q = 0; q < LPW; ++q) issue_one(STAGES - 1, KT, q);
      wait_vmcnt<0>();
    } else {
      typedef u64x2_t __attribute__((aligned(1))) u64x2_u;
      char* t = smem + (STAGES - 1) * STAGE;
#pragma unroll
      for (int q = 0; q < NQA + NQB; ++q) {
        const int c = q < NQA ? wave * NQA + q : b_copy(q - NQA), r = c * 8 + lane / 8;
        const int chunk = dl_swz(r, lane % 8), k = kt0 * 128 + 16 * chunk;
        const uint8_t* base = q < NQA ? A + ao[q] : (b_up(c * 8) ? B[1] : B[0]) + bo[q - NQA];
        base -= 16 * chunk;  // the row's start
        u64x2_t v;
        if (K >= 16) {
          v = shift_down(*(const u64x2_u*)(base + min(k, K - 16)), max(0, k - (K - 16)));
        } else {
          v = u64x2_t{};
          for (int e = 0; e < 16; ++e)
            if (k + e < K) v[e >> 3] |= (uint64_t)base[k + e] << (8 * (e & 7));
        }
        *(u64x2_t*)(t + (q < NQA ? 0 : TA) + c * 1024 + lane * 16) = v;
      }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
      sa[i] = p.x.scales[(int64_t)min(m0 + wm * TM + 16 * i + row, M - 1) * p.x.sld + kt0];
    const int64_t block = min(n0 + (GATE ? 0 : wn * TN), N - 1) / kFp8Group;
    sb[0] = p.w.scales[block * p.w.sld + kt0];
    if constexpr (GATE) sb[1] = p.w2.scales[block * p.w2.sld + kt0];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FM; ++i) read_a(0, STAGES - 1, i, 0), read_a(0, STAGES - 1, i, 1);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      read_b(STAGES - 1, j, 0), read_b(STAGES - 1, j, 1);
#pragma unroll
      for (int i = 0; i < FM; ++i) mfma_one(0, j, i);
    }
    __syncthreads();
  };
  const bool tail = K % 128 != 0 && (!SPLIT || blockIdx.y + 1 == gridDim.y);
  if constexpr (PAIRS) {
#pragma unroll 1
    for (int t = 1 - odd; t < (tail ? 2 : 1); ++t) alone(t != 0);
  } else {
    if (tail) alone(true);
  }
  constexpr int FIRST = PAIRS ? LPW - 2 : LPW;  // (the step before's copies of the last stage)
  if (STAGES - 1 < KT) issue(STAGES - 1, STAGES - 1, FIRST);
  if (KT > 0) {
    if (STAGES <= KT) wait_vmcnt<(STAGES - 2) * LPW + FIRST>();
    else wait_vmcnt<0>();
    __syncthreads();
    first_reads(0);
    int st = 0, kt = 0;
    auto next = [&]() __attribute__((always_inline)) { st = st + 1 == STAGES ? 0 : st + 1; };
    const std::true_type yes;
    const std::false_type no;
    if constexpr (PAIRS) {
      const std::integral_constant<int, 0> one;
      const std::integral_constant<int, 1> two;
      for (; kt < KT - 2; kt += 2) pair_step(one, 0, kt, yes, yes), pair_step(two, 1, kt + 1, yes, yes);
      pair_step(one, 0, kt, no, yes), pair_step(two, 1, kt + 1, no, no);
    } else {
      for (; kt < KT - STAGES; ++kt, next()) step(st, kt, yes, yes);
      for (; kt < KT - 1; ++kt, next()) step(st, kt, no, yes);
      step(st, kt, no, no);
    }
  }

  const int mw = m0 + wm * TM;
  if constexpr (SPLIT) {
    // (ldp is a multiple of 4, so a run that starts inside the row fits)
    const int64_t set = (int64_t)gridDim.y * M * p.ldp;
    float* part = p.part + (int64_t)blockIdx.y * M * p.ldp;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = wn * TN + 16 * j, n = b_row(r) + 4 * (lane >> 4), m = mw + 16 * i + row;
        if (m < M && n < N) *(f32x4_t*)(part + (b_up(r) ? set : 0) + (int64_t)m * p.ldp + n) = acc[j][i];
      }
    return;
  }
  __syncthreads();  // every wave is done with the stages
  if constexpr (EPI == F8_GATE) {
    uint32_t* most = (uint32_t*)(smem + BM * C::CP);  // [WN][BM]
    float mine[FM] = {};
#pragma unroll
    for (int j = 0; j < FN / 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (columns past the end take no part in a maximum)
        const bool there = n0 + wn * (TN / 2) + 16 * j + 4 * (lane >> 4) + e < N;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const float u = there ? acc[j + FN / 2][i][e] : 0.f, g = there ? acc[j][i][e] : 0.f;
          acc[j][i][e] = gate_of(g, u, &mine[i]);
        }
      }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      uint32_t mx = __float_as_uint(mine[i]);
      mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, 64));
      mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, 64));
      if (lane < 16) most[wn * BM + wm * TM + 16 * i + row] = mx;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int r = wm * TM + 16 * i + row;
      uint32_t mx = most[r];
#pragma unroll
      for (int w = 1; w < WN; ++w) mx = max(mx, most[w * BM + r]);
      const uint32_t byte = fp8_scale_byte(mx);
      const float inv = fp8_inverse(byte);
#pragma unroll
      for (int j = 0; j < FN / 2; ++j)
        *(uint32_t*)(smem + r * C::CP + wn * (TN / 2) + 16 * j + 4 * (lane >> 4)) =
            fp8_codes4(acc[j][i][0], acc[j][i][1], acc[j][i][2], acc[j][i][3], inv);
      if (wn == 0 && lane < 16 && m0 + r < M)
        p.codes.scales[(int64_t)(m0 + r) * p.codes.sld + tn] = (uint8_t)byte;
    }
    __syncthreads();
    const bool vec = p.codes.ld % 16 == 0 && (uintptr_t)p.codes.codes % 16 == 0;
    for (int id = threadIdx.x; id < BM * 8; id += C::NT) {
      const int r = id >> 3, c = (id & 7) * 16, n = n0 + c;
      if (m0 + r >= M || n >= N) continue;
      const u32x4_t v = *(const u32x4_t*)(smem + r * C::CP + c);
      uint8_t* dst = p.codes.codes + (int64_t)(m0 + r) * p.codes.ld + n;
      if (vec && n + 15 < N) {
        *(u32x4_t*)dst = v;
      } else {
        for (int e = 0; e < 16 && n + e < N; ++e) dst[e] = (uint8_t)(v[e >> 2] >> (8 * (e & 3)));
      }
    }
    return;
  }
  // out = acc (+ bias) (+ residual), rounded once: HC columns of the wave's tile at a
  // time through LDS, for whole row segments.  Where all of the tile's columns exist and
  // rows are aligned, nothing stands behind a condition: a pass's residual is asked for at
  // once, before its products go to LDS, and rows past the end are the wave's last one
  // again, read before it is first written.  (A tile's epilogue of 14 us with a residual
  // so became 8; with a condition at each store 9.)
  constexpr int HC = C::HC, EP = C::EP, LPR = HC / 8, RPI = 64 / LPR, NI = TM / RPI, NB = NI < 4 ? NI : 4;
  float* es = (float*)smem + wave * TM * EP;
  typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
  uint16_t* out = (uint16_t*)p.out;
  const bool vec_out = p.ldc % 8 == 0 && (uintptr_t)out % 16 == 0;
  const bool vec_res = p.ldr % 8 == 0 && (uintptr_t)p.res % 16 == 0;
  if (mw >= M) return;
  const int last = M - 1 - mw;
  const bool whole = vec_out && (p.res == nullptr || vec_res) && n0 + BN <= N;
  auto finish = [&](auto half_c) __attribute__((always_inline)) {
    constexpr bool HALF = decltype(half_c)::value;
    auto wide = [](uint16_t v) __attribute__((always_inline)) { return HALF ? f16_to_f32(v) : bf16_to_f32(v); };
    auto narrow = [](float y) __attribute__((always_inline)) { return HALF ? f32_to_f16(y) : f32_to_bf16(y); };
#pragma unroll
    for (int h = 0; h < TN / HC; ++h) {
      const int c = (lane % LPR) * 8, n = n0 + wn * TN + h * HC + c;
      u16x8_t res[NI];
      if (whole && p.res != nullptr) {
#pragma unroll
        for (int it = 0; it < NI; ++it)
          res[it] = *(const u16x8_t*)(p.res + (int64_t)(mw + min(it * RPI + lane / LPR, last)) * p.ldr + n);
      } else {
#pragma unroll
        for (int it = 0; it < NI; ++it) res[it] = (u16x8_t)(uint16_t)0x8000;  // y + -0 is y
      }
      float bias[8] = {};
      if (p.bias != nullptr)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = min(n + e, N - 1);
          bias[e] = p.bias_dtype == MI_F32 ? ((const float*)p.bias)[at] : wide(((const uint16_t*)p.bias)[at]);
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < HC / 16; ++j)
#pragma unroll
        for (int i = 0; i < FM; ++i)
          *(f32x4_t*)(es + (16 * i + row) * EP + 16 * j + 4 * (lane >> 4)) = acc[h * (HC / 16) + j][i];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      if (whole) {
#pragma unroll
        for (int b = 0; b < NI; b += NB) {
          f32x4_t y[NB][2];
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u)
              y[i][u] = *(const f32x4_t*)(es + min((b + i) * RPI + lane / LPR, last) * EP + c + 4 * u);
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            u16x8_t v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = narrow(y[i][e >> 2][e & 3] + bias[e] + wide(res[b + i][e]));
            *(u16x8_t*)(out + (int64_t)(mw + min((b + i) * RPI + lane / LPR, last)) * p.ldc + n) = v;
          }
        }
        continue;
      }
#pragma unroll 1
      for (int it = 0; it < NI; ++it) {
        const int r = it * RPI + lane / LPR, m = mw + r;
        if (m >= M || n >= N) continue;
        const uint16_t* src = p.res == nullptr ? nullptr : p.res + (int64_t)m * p.ldr + n;
        uint16_t* dst = out + (int64_t)m * p.ldc + n;
        const bool all = n + 7 < N;
        u16x8_t v = (u16x8_t)(uint16_t)0x8000;
        if (src != nullptr && vec_res && all) {
          v = *(const u16x8_t*)src;
        } else if (src != nullptr) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = src[min(e, N - 1 - n)];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = narrow(es[r * EP + c + e] + bias[e] + wide(v[e]));
        if (vec_out && all) {
          *(u16x8_t*)dst = v;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < N) dst[e] = v[e];
        }
      }
    }
  };
  if (p.f16) finish(std::true_type{});
  else finish(std::false_type{});
}

}  // namespace
}  // namespace mi
