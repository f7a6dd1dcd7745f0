// Shared by the kernels of the 8-bit key/value cache: arguments, the cut of a
// call over blocks, and conversions between e4m3 codes and wider types.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_common.h"
#include "kv8_index.h"

namespace mi {

struct Kv8Cache {
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  int64_t k_sp, k_sh, v_sp, v_sh;      // strides of a page and a head, in bytes
  int64_t ks_sp, ks_sh, vs_sp, vs_sh;  // the scales', in elements
  int pages, heads, shift;             // page size = 1 << shift
};

struct Kv8Args {
  Kv8Cache c;
  const int* table;
  int64_t t_sb;     // table row stride
  int width;        // table entries per sequence
  const int* lengths;
  const int* starts;
  int seqs, tokens, group;
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* o;
  int64_t o_st, o_sh;
  float* lse;
  int64_t lse_st, lse_sh;
  float scale_log2;  // softmax scale * log2(e)
  int fill_rest;     // rows of no sequence: zeros (0: left as they were)
  Kv8Plan plan;
  int slots;         // partials there is room for
  float* part_o;     // [slots][rows of a tile][D], not normalised
  float* part_ml;    // [slots][rows of a tile][2]: max (log2 units), sum
  int* chunk;        // key tiles of a part, as the attention kernel cut them, for the merge
  IndexFault* fault;
};

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Fp8To;
template <>
struct Fp8To<BF16> {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  template <bool HI>
  static __device__ __forceinline__ pair cvt(uint32_t v) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, HI);
  }
};
template <>
struct Fp8To<F16> {
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
  template <bool HI>
  static __device__ __forceinline__ pair cvt(uint32_t v) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.0f, HI);
  }
};

// Eight e4m3 codes as an MFMA operand of eight 16-bit numbers (exact: both
// types hold every e4m3 number).
template <typename T>
__device__ __forceinline__ typename AttnOp<T>::vec fp8x8_to(uint32_t lo, uint32_t hi) {
  union {
    typename Fp8To<T>::pair p[4];
    typename AttnOp<T>::vec v;
  } u;
  u.p[0] = Fp8To<T>::template cvt<false>(lo);
  u.p[1] = Fp8To<T>::template cvt<true>(lo);
  u.p[2] = Fp8To<T>::template cvt<false>(hi);
  u.p[3] = Fp8To<T>::template cvt<true>(hi);
  return u.v;
}

// 16 x 16 tiles, 32 deep: lane l holds row (column) l % 16 at depth 8 (l / 16)
// + 0 .. 7 of its operands, and rows 4 (l / 16) + 0 .. 3 of column l % 16 of the
// result.
template <typename T>
struct Mma16;
template <>
struct Mma16<BF16> {
  static __device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma16<F16> {
  static __device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// How softmax weights become 16-bit operands that lose no more than a rounding to
// the type does, whatever scales the values have.  Sums over keys are relative to
// the largest V scale met (up to MOST, so that fp32 holds them beside the smallest
// one), and a weight may be multiplied by its V scale over that before it is rounded,
// while the quotient leaves the type's range as it is.  Where it does not, the 16
// keys' product has an accumulator of its own that is multiplied in fp32: a page of
// large values that a row does not see, or gives no weight, so costs the other
// weights nothing.
//   f16: a weight is e = 2^(score - m), with m the running maximum rounded up to a
// whole number, so at most 1; it is kept as 2^15 e (with m whole the subtraction in
// the exponent stays exact), which takes the least f16 of 2^-25 to 2^-40, and the
// quotient may take those 15 bits again.
//   bf16 has fp32's range: quotients down to 2^-60 leave weights from 2^-66 on whole.
template <typename T>
struct Kv8Weight {
  static constexpr bool F = std::is_same<T, F16>::value;
  static constexpr float BITS = F ? 15.f : 0.f, UNIT = F ? 0x1p-15f : 1.f;
  static constexpr float MOST = F ? 0x1p8f : 0x1p60f, LEAST = F ? UNIT : 0x1p-60f;
  // the running maximum for a new largest score (base 2), and what is subtracted
  static __device__ __forceinline__ float top(float mx) { return F ? ceilf(mx) : mx; }
  static __device__ __forceinline__ float offset(float m) {
    return m == -INFINITY ? 0.f : F ? m - BITS : m;
  }
  static __device__ __forceinline__ float ref(float scale) { return fminf(scale, MOST); }
  // (f16: just over 1 may be a quotient's rounding, and 2^15 x 1.5 still is a number)
  static __device__ __forceinline__ bool apart(float f) {
    return (F && f > 1.5f) || (f < LEAST && f > 0.f);
  }
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
// Four codes to floats and back (to nearest, ties to even; the caller has
// scaled to |x| <= 448, NaN becomes the NaN code).
__device__ __forceinline__ f32x4 fp8x4_to_f32(uint32_t v) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(v, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
  return f32x4{a[0], a[1], b[0], b[1]};
}
__device__ __forceinline__ uint32_t f32x4_to_fp8(f32x4 x) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], r, true);
}

__device__ __forceinline__ bool kv8_finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// Wave-uniform reads of memory that the kernel does not write: through the
// scalar cache's loads, whatever stores the compiler sees elsewhere.
template <typename V>
__device__ __forceinline__ V ld_const(const V* p) {
  return *(const __attribute__((address_space(4))) V*)p;
}

// A value that is the same in all lanes, told to the compiler: what is derived
// from it stays in scalar registers, and branches on it are scalar.
__device__ __forceinline__ int wave_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ float wave_uniform_f32(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}

// The larger (the sum) of a lane's value and that of the lane 32 (16) from it, by
// lane swaps instead of a round through LDS.
template <bool SUM>
__device__ __forceinline__ float over_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t u0 = r[0], u1 = r[1];  // (a bit cast of a vector's element takes element 0)
  const float a = __builtin_bit_cast(float, u0), b = __builtin_bit_cast(float, u1);
  return SUM ? a + b : fmaxf(a, b);
}
template <bool SUM>
__device__ __forceinline__ float over_rows(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t u0 = r[0], u1 = r[1];  // (a bit cast of a vector's element takes element 0)
  const float a = __builtin_bit_cast(float, u0), b = __builtin_bit_cast(float, u1);
  return SUM ? a + b : fmaxf(a, b);
}
__device__ __forceinline__ float half_max(float x) { return over_halves<false>(x); }
__device__ __forceinline__ float half_sum(float x) { return over_halves<true>(x); }
__device__ __forceinline__ float row_max(float x) { return over_rows<false>(x); }
__device__ __forceinline__ float row_sum(float x) { return over_rows<true>(x); }

// lds_copy16 from an address of each lane's own to m0 (of lds_place) and on.
__device__ __forceinline__ uint32_t lds_place(void* lds) {
  return wave_uniform((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds);
}
__device__ __forceinline__ void lds_copy16_at(const void* p, uint32_t m0) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "{m0}"(m0) : "memory");
}

// The same, 4 bytes a lane.
__device__ __forceinline__ void lds_copy4_at(const void* p, uint32_t m0) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(p), "{m0}"(m0) : "memory");
}

// Inclusive sums (or maxima of numbers that are not negative) over the lanes, by
// DPP within rows of 16 and two row broadcasts.
template <bool MAX, int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int v) {
  const int x = __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
  return MAX ? max(v, x) : v + x;
}
template <bool MAX = false>
__device__ __forceinline__ int wave_scan(int v) {
  v = scan_step<MAX, 0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v = scan_step<MAX, 0x112, 0xF>(v);
  v = scan_step<MAX, 0x114, 0xF>(v);
  v = scan_step<MAX, 0x118, 0xF>(v);
  v = scan_step<MAX, 0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  return scan_step<MAX, 0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}

// The call's sequences, a lane each, 64 at a time; the first 64 stay in
// registers, so that a call of up to 64 reads its index tensors once.
struct Kv8Lanes {
  const Kv8Args& a;
  int lane, cap;
  Kv8Seq head;

  __device__ __forceinline__ explicit Kv8Lanes(const Kv8Args& args)
      : a(args), lane(threadIdx.x & 63), cap(args.width << args.c.shift) {
    head = load(lane);
  }
  __device__ __forceinline__ Kv8Seq load(int b) const {
    if (b >= a.seqs) return Kv8Seq{0, 0, 0, false};
    return kv8_seq(a.starts[b], a.starts[b + 1], a.lengths[b], a.tokens, cap);
  }
  __device__ __forceinline__ Kv8Seq at(int b0) const { return b0 == 0 ? head : load(b0 + lane); }
  static __device__ __forceinline__ Kv8Seq pick(const Kv8Seq& s, int l) {
    return {__builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.n, l),
            __builtin_amdgcn_readlane(s.len, l), __builtin_amdgcn_readlane((int)s.bad, l) != 0};
  }
  // Key tiles per part, from all sequences' work; the same in every wave.
  template <typename F>
  __device__ __forceinline__ int chunk(F work) const {
    float sum = work(head);
    for (int b0 = 64; b0 < a.seqs; b0 += 64) sum += work(load(b0 + lane));
    return wave_uniform(a.plan.chunk(wave_sum(sum) * a.c.heads));
  }
  // The sequence that item `item` belongs to, counted by count(s) per sequence
  // in order, and its place in it; false if there are fewer items.  Every lane
  // gets the same answer.
  template <typename F>
  __device__ __forceinline__ bool find(int item, F count, int* seq, Kv8Seq* s, int* place) const {
    int64_t before = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += 64) {
      const Kv8Seq mine = at(b0);
      const int n = count(mine), upto = wave_scan(n);
      const uint64_t hit = __ballot(before + upto > item);
      if (hit != 0) {
        const int l = __builtin_ctzll(hit), m = __builtin_amdgcn_readlane(n, l);
        *seq = wave_uniform(b0 + l);
        *s = pick(mine, l);
        *place = wave_uniform((int)(item - before) - (__builtin_amdgcn_readlane(upto, l) - m));
        return *place >= 0 && *place < m;  // always, unless starts that overlap overflowed the sums
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
  }
};

__device__ __forceinline__ int wave_last(int x) { return __builtin_amdgcn_readlane(x, 63); }

// The items of Kv8Rounds: a wave's lanes hold a sequence each.
struct Kv8RoundItems {
  Kv8Rounds rounds;
  int parts, end;  // parts of the lane's sequence; one past the last round, of all

  template <int RT, int KT>
  static __device__ __forceinline__ Kv8RoundItems of(const Kv8Args& a, const Kv8Seq& s, int chunk) {
    const Kv8Cut c = kv8_cut(s, a.group, RT, KT);
    const int longest = wave_last(wave_scan<true>(c.row_tiles > 0 ? s.len : 0));
    const Kv8Rounds r(s, c, longest, a.group, RT);
    const int end = wave_last(wave_scan<true>(r.tiles > 0 ? r.off + r.tiles : 0));
    return {r, c.row_tiles > 0 ? c.parts(chunk) : 0, end};
  }
  // (a single sequence's items are in that order anyway)
  static __device__ __forceinline__ bool apply(const Kv8Args& a) {
    return a.seqs > 1 && a.seqs <= 64;
  }
  // items of a head in rounds 0 .. k - 1, of all sequences
  __device__ __forceinline__ int before(int k) const {
    return wave_last(wave_scan(rounds.before(k) * parts));
  }
};

// One block's share of a call over query rows and keys: row tile `tile` of k/v
// head `head` of sequence `seq`, part `part` of its `parts` of keys.
struct Kv8Item {
  Kv8Seq s;
  Kv8Cut cut;
  int seq, head, tile, part, parts;
};

// FARTHEST: in the order of Kv8Rounds, with tiles counted from the sequence's end:
// blocks start in the order of their items, and what starts last should be short
// (32 query heads on 8 of 128: 4 x up to 1024 tokens behind up to 1000 86 -> 82 us,
// 32 x up to 64 behind up to 1800 70 -> 62; finding the item takes 1 us more, which
// calls without a second round of blocks lose: 4 x up to 512 behind up to 1500, 16
// heads on 4 of 64, 42 -> 44).
template <int RT, int KT, bool FARTHEST>
__device__ __forceinline__ bool kv8_item(const Kv8Args& a, int item, Kv8Item* it) {
  const Kv8Lanes lanes(a);
  const int chunk =
      lanes.chunk([&](const Kv8Seq& s) { return kv8_cut(s, a.group, RT, KT).work(); });
  if (item == 0 && a.chunk != nullptr && threadIdx.x == 0) *a.chunk = chunk;
  int place;
  if (FARTHEST && Kv8RoundItems::apply(a)) {
    const Kv8RoundItems all = Kv8RoundItems::of<RT, KT>(a, lanes.head, chunk);
    const int want = item / a.c.heads;  // items of a round hold every head
    int lo = 0, hi = all.end;           // the round: before(lo) <= want < before(lo + 1)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (all.before(mid) <= want) lo = mid;
      else hi = mid;
    }
    const int n = all.rounds.in(lo) ? all.parts : 0, upto = wave_scan(n);
    const int rest = want - all.before(lo);
    const uint64_t hit = __ballot(upto > rest);
    if (rest < 0 || hit == 0) return false;
    const int l = __builtin_ctzll(hit);
    it->seq = wave_uniform(l);
    it->s = Kv8Lanes::pick(lanes.head, l);
    it->cut = kv8_cut(it->s, a.group, RT, KT);
    it->parts = __builtin_amdgcn_readlane(all.parts, l);
    it->part = rest - (__builtin_amdgcn_readlane(upto, l) - it->parts);
    it->head = item % a.c.heads;
    it->tile = lo - __builtin_amdgcn_readlane(all.rounds.off, l);
    return true;
  }
  const bool found = lanes.find(
      item,
      [&](const Kv8Seq& s) {
        const Kv8Cut c = kv8_cut(s, a.group, RT, KT);
        return a.c.heads * c.row_tiles * c.parts(chunk);
      },
      &it->seq, &it->s, &place);
  if (!found) return false;
  it->cut = kv8_cut(it->s, a.group, RT, KT);
  it->parts = it->cut.parts(chunk);
  it->part = place % it->parts;
  it->head = place / it->parts % a.c.heads;
  it->tile = place / it->parts / a.c.heads;
  return true;
}

// What no item covers: rows of no sequence, and sequences whose length is out
// of range, which are reported (they count as empty).
__device__ __forceinline__ void kv8_report_lengths(const int* lengths, int seqs, int cap,
                                                   IndexFault* fault) {
  for (int b = threadIdx.x; b < seqs; b += blockDim.x) {
    const int n = lengths[b];
    if (n < 0 || n > cap) record_index_fault(fault, n, (int64_t)cap + 1);
  }
}

template <int D>
__device__ __forceinline__ void kv8_rest(const Kv8Args& a) {
  if (blockIdx.x == 0) kv8_report_lengths(a.lengths, a.seqs, a.width << a.c.shift, a.fault);
  if (!a.fill_rest) return;
  const int lo = kv8_clamp(a.starts[0], 0, a.tokens);
  const int hi = kv8_clamp(a.starts[a.seqs], lo, a.tokens);
  const int rest = a.tokens - (hi - lo), heads = a.c.heads * a.group;
  for (int i = blockIdx.x; i < rest; i += gridDim.x) {
    const int64_t t = i < lo ? i : i - lo + hi;
    for (int x = threadIdx.x; x < heads * (D / 8); x += blockDim.x)
      *(u32x4*)(a.o + t * a.o_st + (x / (D / 8)) * a.o_sh + x % (D / 8) * 8) = u32x4{};
    for (int h = threadIdx.x; h < heads; h += blockDim.x)
      a.lse[t * a.lse_st + h * a.lse_sh] = -INFINITY;
  }
}

}  // namespace

// Host side (kv8_cache.cpp): the cache's own checks, and the tensors that say
// which sequences a call is about.
// Whether rows of `extent` elements, n0 x n1 of them at strides s0 and s1, lie one
// after the other with either index as the outer one.
bool kv8_apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t extent);
mi_status_t kv8_check_cache(const char* op, const mi_kv8_cache_t* cache, Kv8Cache* c, int64_t* dim);
// Rows of `extent` bytes at two strides, in bytes, and whether no row of one tensor
// shares memory with one of another.  They may lie among each other where their
// strides are the same (k and v by turns in one pool).
struct Kv8Rows {
  const void* data;
  int64_t n0, s0, n1, s1;
};
bool kv8_disjoint(const Kv8Rows& a, const Kv8Rows& b, int64_t extent);
// for calls that write it
mi_status_t kv8_check_written(const char* op, const Kv8Cache& c, int64_t dim);
mi_status_t kv8_check_queries(const char* op, const mi_tensor_t* q, const mi_tensor_t* lse,
                              int64_t dim, Kv8Args* a);
mi_status_t kv8_check_seqs(const char* op, const mi_tensor_t* table, const mi_tensor_t* lengths,
                           const mi_tensor_t* starts, int64_t tokens, Kv8Args* a);
// int32 [sequences, heads, keep], dense rows
mi_status_t kv8_check_kept(const char* op, const mi_tensor_t* kept, int64_t keep, const Kv8Args& a);
// Attention of many query rows per sequence (kv8_prompt.hip).
mi_status_t kv8_prompt(Kv8Args& a, int64_t dim, bool f16, hipStream_t s);
// float32 [sequences, heads, at least the table's positions], dense rows
mi_status_t kv8_check_weights(const char* op, const mi_tensor_t* w, const char* name,
                              const Kv8Args& a);

}  // namespace mi
