// The tiled product on the matrix pipe: BM x BN tiles, fp32 sums in 32 x 32 matrix instructions, operands copied straight
// from memory into two LDS stages of 128 bytes of the reduction (whole cache lines of a K-contiguous row: with four stages of
// 64 bytes every line was fetched twice).
//
// Bound by the matrix pipe and its power (large products) or by HBM (long thin ones).  A stage is computed in two halves.
// The fragments of a half lie in registers already while the next half's are read from LDS, and the stage after next is
// requested as soon as every wave has read the second half of this one: the matrix instructions wait for neither, and a
// stage costs one barrier.  (Four to six stages under way, for grids of one workgroup a CU, change nothing: 1024 x 1024 x 2048
// fp16 12.0 us with two, 12.1 with three, 12.9 with six.  Nor do four waves of 128 x 128 with a third fewer LDS reads, products
// without bias, activation and residual: 8192^3 e4m3 463 us against 416, 8192 x 4096 x 16,384 bf16 944 against 878: one wave a
// SIMD leaves the pipe idle at each barrier.)
//
// Measured, best of a case's launches on normal operands: 8192 x 4096 x 16,384 bf16 0.91 ms bare (1.21 PFLOP/s; the library's
// product 0.71), 0.95 with bias and gelu, 1.00 where the slopes are kept too, 0.88 dx and 0.93 dw (1.25, 1.18; the library's 0.80 and
// 0.92); 8192^3 e4m3 0.42 ms bare (2.6 PFLOP/s; the library 0.36), 0.48 with bias and residual, 0.78 for an fp32 result;
// 8192 x 2048 x 2048 fp32 0.31 ms; 169,343 x 128 x 256 fp32 0.150 ms forward (2.9 TB/s with z), 0.090 dx, 0.073 dw.
#pragma once

#include <type_traits>

#include "bf16x6.h"
#include "linear_act.h"

namespace dgcn {
namespace {

typedef int i8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef uint32_t u8v __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s4v lds_s4;

__device__ __forceinline__ u4v half0(u8v r) { return __builtin_shufflevector(r, r, 0, 1, 2, 3); }
__device__ __forceinline__ u4v half1(u8v r) { return __builtin_shufflevector(r, r, 4, 5, 6, 7); }

// What a wave does with the fragments of a stage: a raw fragment is two 16-byte units of an operand row (lane l: row l & 31,
// h = l >> 5) of a half stage's 64 bytes, prep() makes of it what the matrix instructions take, mul() adds one tile's products.
template <class T> struct TileIn;

template <class T>
struct TileIn16 {                                          // units h and 2 + h: k = 8 h .. of each 16 of the 32
  static constexpr int ES = 2;
  struct Frag { u4v r[2]; };
  static __device__ __forceinline__ Frag prep(u8v r) { return Frag{{half0(r), half1(r)}}; }
  static __device__ __forceinline__ f32x16 one(u4v a, u4v b, f32x16 c) {
    if constexpr (__is_same(T, __bf16)) {
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
  }
  static __device__ __forceinline__ void mul(const Frag (&b)[2], const Frag& a, f32x16 (&c)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int t = 0; t < 2; ++t) c[t] = one(b[t].r[s], a.r[s], c[t]);
    }
  }
};
template <> struct TileIn<__bf16> : TileIn16<__bf16> {};
template <> struct TileIn<_Float16> : TileIn16<_Float16> {};

// fp32 (units 2 h and 2 h + 1: k = 8 h .. 8 h + 7 of the 16): three bf16 parts that add up to the value bit for bit,
// and the six products of parts down to 2^-16 of the largest (bf16x6.h: off by at most 3 2^-24 |a b|)
template <> struct TileIn<float> {
  static constexpr int ES = 4;
  struct Frag { u4v h, m, l; };
  static __device__ __forceinline__ Frag prep(u8v r) {
    i4v h, m, l;
    eg_split3(__builtin_bit_cast(f4v, half0(r)), __builtin_bit_cast(f4v, half1(r)), h, m, l);
    return Frag{__builtin_bit_cast(u4v, h), __builtin_bit_cast(u4v, m), __builtin_bit_cast(u4v, l)};
  }
  static __device__ __forceinline__ void mul(const Frag (&b)[2], const Frag& a, f32x16 (&c)[2]) {
    typedef TileIn16<__bf16> P;
#pragma unroll
    for (int t = 0; t < 2; ++t) c[t] = P::one(b[t].m, a.m, c[t]);
#pragma unroll
    for (int t = 0; t < 2; ++t) c[t] = P::one(b[t].l, a.h, c[t]);
#pragma unroll
    for (int t = 0; t < 2; ++t) c[t] = P::one(b[t].h, a.l, c[t]);
#pragma unroll
    for (int t = 0; t < 2; ++t) c[t] = P::one(b[t].m, a.h, c[t]);
#pragma unroll
    for (int t = 0; t < 2; ++t) c[t] = P::one(b[t].h, a.m, c[t]);
#pragma unroll
    for (int t = 0; t < 2; ++t) c[t] = P::one(b[t].h, a.h, c[t]);
  }
};

// Infinities and NaN have no three parts (inf - inf): an fp32 operand that is not finite leaves NaN in every sum that it is
// part of.  Such a sum is an infinity or NaN, whatever its finite terms are, so it is found again from what its operands are
// alone: their signs, zeros, infinities and NaN as bf16 values (a finite number is +-1), one product each.  The sums that are
// NaN take it where it is not finite (where it is, the sum left fp32 on its way).  Straight from memory, at a tenth of the rate
// (8192 x 2048 x 2048, all NaN: 3.8 ms against 0.31): finite rows pay for the look at the sums alone, which does not show.
__device__ __forceinline__ u4v f32_kinds(const float (&v)[8]) {
  float k[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = fabsf(v[e]);
    k[e] = v[e] != v[e] ? __builtin_nanf("") : copysignf(a == 0.f || a == __builtin_inff() ? a : 1.f, v[e]);
  }
  return u4v{eg_pack_hi16(k[0], k[1]), eg_pack_hi16(k[2], k[3]), eg_pack_hi16(k[4], k[5]), eg_pack_hi16(k[6], k[7])};
}
template <class V>
__device__ __forceinline__ bool any_nan(const V& v) {
  bool nan = false;
#pragma unroll
  for (unsigned e = 0; e < sizeof(V) / 4; ++e) nan = nan || v[e] != v[e];
  return __any(nan);
}
template <class V>
__device__ __forceinline__ void take_kinds(V& c, const V& kinds) {
#pragma unroll
  for (unsigned e = 0; e < sizeof(V) / 4; ++e) c[e] = c[e] != c[e] && !(fabsf(kinds[e]) < __builtin_inff()) ? kinds[e] : c[e];
}

// eight values from k on (0 from `end` on) of line r of an operand of layout T
template <int T>
__device__ __forceinline__ u4v kinds_at(const void* x, int64_t ld, int64_t r, int64_t k, int64_t end) {
  const float* p = static_cast<const float*>(x) + (T == 0 ? r * ld + k : k * ld + r);
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = k + e < end ? p[e * (T == 0 ? 1 : ld)] : 0.f;
  return f32_kinds(v);
}

// e4m3 for a 16-bit result (units 2 h and 2 h + 1: 32 of the 64 values): one instruction at twice the 16-bit rate, its
// block scales held at 2^0.  It aligns the products of eight neighbouring k to the largest one's exponent and drops what lies
// more than 13 bits below it (measured, bit by bit), so a sum is off by up to 7 2^-13 of the largest product of each eight:
// 6e-5 of the result's root mean square over normal rows, an order below a bf16 half step and under half of an fp16 one.
template <> struct TileIn<uint8_t> {
  static constexpr int ES = 1;
  typedef i8v Frag;
  static __device__ __forceinline__ Frag prep(u8v r) { return __builtin_bit_cast(i8v, r); }
  static __device__ __forceinline__ void mul(const Frag (&b)[2], const Frag& a, f32x16 (&c)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) c[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[t], a, c[t], 0, 0, 0, 127, 0, 127);
  }
};

// e4m3 for an fp32 result: every e4m3 value is an fp16 value; their products are exact and their sum is fp32
struct WideE4m3 {};
__device__ __forceinline__ u4v widen_e4m3(uint32_t lo, uint32_t hi) {
  return u4v{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true))};
}
template <> struct TileIn<WideE4m3> {
  static constexpr int ES = 1;
  struct Frag { u4v r[4]; };
  static __device__ __forceinline__ Frag prep(u8v r) {
    return Frag{{widen_e4m3(r[0], r[1]), widen_e4m3(r[2], r[3]), widen_e4m3(r[4], r[5]), widen_e4m3(r[6], r[7])}};
  }
  static __device__ __forceinline__ void mul(const Frag (&b)[2], const Frag& a, f32x16 (&c)[2]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
#pragma unroll
      for (int t = 0; t < 2; ++t) c[t] = TileIn16<_Float16>::one(b[t].r[s], a.r[s], c[t]);
    }
  }
};

constexpr unsigned kRsrcFlags = 0x00027000;               // raw 32-bit buffer; a load behind its end gives zeros
constexpr unsigned kBehind = 0x80000000u;                 // an offset behind any buffer here (at most 2^31 bytes)

// Which chunk (16 bytes) of an operand tile a 16-byte unit of an LDS stage holds.
//   K-contiguous, R rows of 128 bytes: unit u of row r holds the row's chunk u ^ (bits 3, 2, 1 of r)
//   K-strided, k-rows of R values: unit u of k-row k holds chunk u ^ 4 (k & 3) in 16 bits, u ^ 8 (bit 3 of k) in 32
// In all, lanes that read together fall on different banks.
template <int T, int R, int ES>
__device__ __forceinline__ unsigned tile_offset(int inst, int lane, int64_t ld) {
  if constexpr (T == 0) {
    const int row = inst * 8 + (lane >> 3);
    return static_cast<unsigned>(row * ld * ES) + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  } else {
    constexpr int UNITS = R * ES / 16;
    const int k = inst * (64 / UNITS) + lane / UNITS;
    const int f = ES == 2 ? 4 * (k & 3) : 8 * ((k >> 3) & 1);
    return static_cast<unsigned>(k * ld * ES) + (((lane % UNITS) ^ f) << 4);
  }
}

// Bytes from the first to behind the last value of an operand tile whose stage holds k of the reduction, in whole dwords: the
// range check of a buffer is by dword, and the dword that holds the last value is there as long as rows start on dwords.
template <int T, int ES>
__device__ __forceinline__ int tile_bytes(int64_t ld, int64_t lines, int k) {
  return static_cast<int>((((T == 0 ? (lines - 1) * ld + k : (k - 1) * ld + lines) * ES) + 3) & ~int64_t{3});
}

// A raw buffer of `bytes` bytes at p, as its four scalar words
__device__ __forceinline__ i4v tile_buffer(const char* p, int bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  return i4v{uni(static_cast<int>(at)), uni(static_cast<int>(at >> 32) & 0xffff), uni(bytes), static_cast<int>(kRsrcFlags)};
}

// 16 bytes a lane from a buffer to LDS, `to` + 16 lane.  Written out because the compiler, which cannot tell which LDS bytes a
// transposing read takes, waits for every copy before each of them (measured on dw of 16384 x 4096 x 8192: 1.14 ms against 0.9);
// the kernel counts its copies itself (meet).  Nothing is returned in registers; the waits that the instruction needs behind
// writes of m0 and of its scalar operands are in the text.
__device__ __forceinline__ void copy16(i4v buffer, unsigned off, unsigned to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(buffer), "s"(uni(static_cast<int>(to))) : "memory", "m0");
}

template <int N>
__device__ __forceinline__ void copy_whole(const char* p, int bytes, const unsigned (&off)[N], unsigned to) {
  const i4v r = tile_buffer(p, bytes);
#pragma unroll
  for (int c = 0; c < N; ++c) copy16(r, off[c], to + c * 1024);
}

// any stage, k values of the reduction in it (none: zeros everywhere, and p is not read)
template <int T, int N, int ES>
__device__ __forceinline__ void copy_part(const char* p, int64_t ld, int64_t lines, int k, const unsigned (&off)[N], int wave,
                                          int lane, unsigned to) {
  const i4v r = tile_buffer(p, k > 0 ? tile_bytes<T, ES>(ld, lines, k) : 0);
#pragma unroll
  for (int c = 0; c < N; ++c) {
    unsigned o = off[c];
    if (T == 0) {
      // byte of the row that this lane's chunk starts at
      const unsigned at = o - static_cast<unsigned>(((wave * N + c) * 8 + (lane >> 3)) * ld * ES);
      o = at < static_cast<unsigned>(k * ES) ? o : kBehind;
    }
    copy16(r, o, to + c * 1024);
  }
}

// T: operand type, O: output type, TA / TB: layouts; a wave owns 32 TM rows x 64 channels, a workgroup WM x WN waves
template <class T, class O, int TA, int TB, int TM, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 2) void tile_kernel(const MatParams P) {
  constexpr int ES = TileIn<T>::ES;
  constexpr int BM = WM * TM * 32, BN = WN * 64, BK = 128 / ES, WAVES = WM * WN;
  constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  constexpr int IA = BM / 8 / WAVES, IB = BN / 8 / WAVES;               // copies a wave makes per stage
  static_assert(IA * 8 * WAVES == BM && IB * 8 * WAVES == BN, "a stage's copies divide over the waves");
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = lane_id(), wave = uni(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int i = lane & 31, h = lane >> 5;

  // workgroup -> tile: consecutive tiles on one XCD (hardware deals workgroups to the XCDs in turn), in groups of eight
  // tile rows, so that what an XCD works on at a time shares its operand panels in that XCD's L2
  const int tm_n = static_cast<int>((P.M + BM - 1) / BM), tn_n = static_cast<int>((P.N + BN - 1) / BN);
  int id = blockIdx.x;
  {
    const int total = tm_n * tn_n, xcd = id % kNumXCD, loc = id / kNumXCD, base = total / kNumXCD, extra = total % kNumXCD;
    id = xcd * base + (xcd < extra ? xcd : extra) + loc;
  }
  const int group = id / (8 * tn_n), first = group * 8, high = tm_n - first < 8 ? tm_n - first : 8;
  const int64_t m0 = static_cast<int64_t>(first + id % (8 * tn_n) % high) * BM;
  const int64_t n0 = static_cast<int64_t>(id % (8 * tn_n) / high) * BN;

  // this workgroup's part of the reduction
  const int steps_all = static_cast<int>((P.K + BK - 1) / BK);
  const int split = blockIdx.y;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps_all) * split / P.splits);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps_all) * (split + 1) / P.splits);

  unsigned offa[IA], offb[IB];
#pragma unroll
  for (int c = 0; c < IA; ++c) offa[c] = tile_offset<TA, BM, ES>(wave * IA + c, lane, P.lda);
#pragma unroll
  for (int c = 0; c < IB; ++c) offb[c] = tile_offset<TB, BN, ES>(wave * IB + c, lane, P.ldb);
  const int64_t rows_a = P.M - m0 < BM ? P.M - m0 : BM, rows_b = P.N - n0 < BN ? P.N - n0 : BN;

  // copy(place) requests the next stage into one of the two places.  Rows and k-rows behind the matrix lie behind the buffer's
  // end and read as zeros; so do, by an offset of kBehind, the chunks of a K-contiguous row behind K (what follows K in the
  // chunk that it ends in is cut from the fragments, see clip), and all of a stage behind the last one, which is requested all the same so
  // that a wave always has the same number of copies under way.   Columns of a K-strided operand behind M or N read what is
  // there: their sums are not stored.
  const int64_t step_a = (TA == 0 ? BK : BK * P.lda) * ES, step_b = (TB == 0 ? BK : BK * P.ldb) * ES;
  const char* pa = static_cast<const char*>(P.a) + (TA == 0 ? m0 * P.lda : m0) * ES + s0 * step_a;
  const char* pb = static_cast<const char*>(P.b) + (TB == 0 ? n0 * P.ldb : n0) * ES + s0 * step_b;
  int todo = s1 - s0;                                                   // stages not yet requested, and the last one's part of BK
  const int last_k = s1 < steps_all ? BK : static_cast<int>(P.K - static_cast<int64_t>(steps_all - 1) * BK);
  typedef std::integral_constant<int, TA> LA;
  typedef std::integral_constant<int, TB> LB;
  const int whole_a = tile_bytes<TA, ES>(P.lda, rows_a, BK), whole_b = tile_bytes<TB, ES>(P.ldb, rows_b, BK);
  const unsigned lds_at = static_cast<unsigned>(reinterpret_cast<uintptr_t>((lds_void*)lds));
  auto copy = [&](auto whole, int place) {                              // whole: the stage is known to be a full one
    const unsigned ta = lds_at + place * STAGE + wave * IA * 1024, tb = lds_at + place * STAGE + A_BYTES + wave * IB * 1024;
    if constexpr (decltype(whole)::value) {
      copy_whole<IA>(pa, whole_a, offa, ta);
      copy_whole<IB>(pb, whole_b, offb, tb);
    } else {
      const int k = todo > 1 ? BK : todo == 1 ? last_k : 0;
      copy_part<TA, IA, ES>(pa, P.lda, rows_a, k, offa, wave, lane, ta);
      copy_part<TB, IB, ES>(pb, P.ldb, rows_b, k, offb, wave, lane, tb);
    }
    pa += step_a;
    pb += step_b;
    todo -= 1;
  };

  // Raw fragment of 32 operand rows (or columns) from `line` on, of one half of the stage
  const int sw = (i >> 1) & 7;
  const int at0 = ((ES == 2 ? h : 2 * h) ^ sw) << 4, at1 = ((ES == 2 ? 2 + h : 2 * h + 1) ^ sw) << 4;
  const int kk = (lane >> 2) & 3, pc = lane & 3, g16 = (lane >> 4) & 1;  // K-strided, 16 bits: the lane fetches four columns of k-row 8 h + kk
  auto read = [&](auto layout, const char* base, int line, int rows, int half) -> u8v {
    constexpr int L = decltype(layout)::value;
    if constexpr (L == 0) {
      const char* p = base + (line + i) * 128;
      return __builtin_shufflevector(*reinterpret_cast<const u4v*>(p + (at0 ^ (64 * half))), *reinterpret_cast<const u4v*>(p + (at1 ^ (64 * half))),
                                     0, 1, 2, 3, 4, 5, 6, 7);
    } else if constexpr (ES == 2) {
      const char* p = base + (8 * h + kk) * rows * 2 + ((line * 2 + g16 * 32 + pc * 8) ^ (kk << 6));
      u4v out[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + (32 * half + 16 * s) * rows * 2));
        const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + (32 * half + 16 * s + 4) * rows * 2));
        out[s] = __builtin_bit_cast(u4v, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
      return __builtin_shufflevector(out[0], out[1], 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const char* p = base + (16 * half + 8 * h) * rows * 4 + (((line + i) * 4) ^ (h << 7));
      u8v out;
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = *reinterpret_cast<const uint32_t*>(p + e * rows * 4);
      return out;
    }
  };
  auto read_a = [&](int place, int half, int t) { return read(LA{}, lds + place * STAGE, (wm * TM + t) * 32, BM, half); };
  auto read_b = [&](int place, int half, int t) { return read(LB{}, lds + place * STAGE + A_BYTES, wn * 64 + 32 * t, BN, half); };
  f32x16 acc[TM][2];
#pragma unroll
  for (int t = 0; t < TM; ++t) {
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[t][0][e] = acc[t][1][e] = 0.f;
  }
  // All but the newest `copies` of this wave's copies have landed and its LDS reads are done; then everyone's.
  auto meet = [&](auto copies) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(copies)::value) : "memory");
  };
  // the values of a half's raw fragment of a K-contiguous operand that lie behind K, cleared (both operands': what is there
  // may be infinite or NaN)
  const int last_bytes = last_k * ES;
  auto clip = [&](auto layout, int half, u8v r) {
    if constexpr (decltype(layout)::value == 0) {
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const int n = last_bytes - 64 * half - (ES == 2 ? (w < 4 ? 16 * h : 32 + 16 * h) + 4 * (w & 3) : 32 * h + 4 * w);
        r[w] &= n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
      }
    }
    return r;
  };
  // A half: its fragments lie in fa and b.  Each row tile's products are followed by the read of the same tile of the next
  // half.  Before the second half's reads, of the next stage, the waves meet -- behind the first products, so that the
  // barrier finds the matrix pipe busy -- and behind them the stage after next is requested into the place of this one.
  // whole: that stage is a full one; cut: this stage is the one that K ends in, inside a chunk.
  u8v fa[TM], b0[2], b1[2];
  auto turn = [&](auto half, auto whole, auto cut, int place, const u8v (&b)[2], u8v (&b_next)[2]) {
    constexpr int H = decltype(half)::value;
    const int from = place ^ H;
    constexpr bool CUT = decltype(cut)::value;
    const typename TileIn<T>::Frag fb[2] = {TileIn<T>::prep(CUT ? clip(LB{}, H, b[0]) : b[0]), TileIn<T>::prep(CUT ? clip(LB{}, H, b[1]) : b[1])};
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      TileIn<T>::mul(fb, TileIn<T>::prep(CUT ? clip(LA{}, H, fa[t]) : fa[t]), acc[t]);
      if (t == 0) {
        if constexpr (H == 1) {
          __builtin_amdgcn_sched_barrier(0);
          meet(std::integral_constant<int, 0>{});
        }
        b_next[0] = read_b(from, H ^ 1, 0);
        b_next[1] = read_b(from, H ^ 1, 1);
      }
      fa[t] = read_a(from, H ^ 1, t);
      if (H == 1 && t == (TM > 1 ? 1 : 0)) copy(whole, place);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  typedef std::integral_constant<int, 0> H0;
  typedef std::integral_constant<int, 1> H1;

  copy(std::false_type{}, 0);
  copy(std::false_type{}, 1);
  meet(std::integral_constant<int, IA + IB>{});
  b0[0] = read_b(0, 0, 0);
  b0[1] = read_b(0, 0, 1);
#pragma unroll
  for (int t = 0; t < TM; ++t) fa[t] = read_a(0, 0, t);
  int place = 0, step = s0;
  const int ends = ((TA == 0 || TB == 0) && s1 == steps_all && last_bytes % 16 != 0) ? s1 - 1 : s1;
  typedef std::true_type Yes;
  typedef std::false_type No;
  for (; todo > 1; ++step, place ^= 1) {                                // full stages ahead: no selection in the loop
    turn(H0{}, Yes{}, No{}, place, b0, b1);
    turn(H1{}, Yes{}, No{}, place, b1, b0);
  }
  for (; step < ends; ++step, place ^= 1) {
    turn(H0{}, No{}, No{}, place, b0, b1);
    turn(H1{}, No{}, No{}, place, b1, b0);
  }
  if (step < s1) {
    turn(H0{}, No{}, Yes{}, place, b0, b1);
    turn(H1{}, No{}, Yes{}, place, b1, b0);
  }

  if constexpr (std::is_same<T, float>::value) {                        // see f32_kinds
    const int64_t k0 = static_cast<int64_t>(s0) * BK, k1 = static_cast<int64_t>(s1) * BK < P.K ? static_cast<int64_t>(s1) * BK : P.K;
#pragma unroll
    for (int t = 0; t < 2 * TM; ++t) {
      f32x16& c = acc[t >> 1][t & 1];
      if (!any_nan(c)) continue;
      const int64_t m = m0 + (wm * TM + (t >> 1)) * 32 + i, n = n0 + wn * 64 + 32 * (t & 1) + i;
      bool stored = false;                                              // (what lies behind the matrix may be NaN and does not count)
#pragma unroll
      for (int e = 0; e < 16; ++e) stored = stored || (c[e] != c[e] && m < P.M && n - i + 8 * (e >> 2) + 4 * h + (e & 3) < P.N);
      if (!__any(stored)) continue;
      f32x16 kinds = {};
#pragma unroll 1
      for (int64_t k = k0 + 8 * h; k - 8 * h < k1; k += 16) {
        kinds = TileIn<__bf16>::one(kinds_at<TB>(P.b, P.ldb, n < P.N ? n : P.N - 1, k, k1), kinds_at<TA>(P.a, P.lda, m < P.M ? m : P.M - 1, k, k1), kinds);
      }
      take_kinds(c, kinds);
    }
  }

  // Epilogue, through LDS (when all copies have landed and nobody reads operands any more): a wave writes its sums as rows of
  // 64 channels, up to 64 rows at a time, and takes them back eight rows by eight channels a lane, so that a store fills
  // whole lines and the code is one rolled loop.  Lane (i, h) holds row i of each 32 and, of a tile's 32 channels, 8 g + 4 h ..
  // + 3 in the sums 4 g .. 4 g + 3.  16-byte unit u of row r lies at u ^ (r & 15).  A wave reads only what it wrote.
  constexpr int PASS = TM < 2 ? TM : 2;
  meet(std::integral_constant<int, 0>{});
  char* mine = lds + wave * (PASS * 32 * 256);
  const int64_t mw = m0 + wm * TM * 32, n = n0 + wn * 64 + 8 * (lane & 7);
  const bool inside = n < P.N;
  float scale[8], bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    scale[e] = (ES == 1 && n + e < P.N) ? P.b_scale[n + e] : 1.f;
    bias[e] = 0.f;
  }
  if (P.bias && inside) load_param_run<O, 8>(P.bias, P.bias_f32, static_cast<int>(n), static_cast<int>(P.N), bias);
  constexpr int AHEAD = 4;                                              // residual rows requested together: their latency is a tile's epilogue otherwise
#pragma unroll
  for (int p = 0; p < TM / PASS; ++p) {
#pragma unroll
    for (int t = 0; t < PASS; ++t) {
#pragma unroll
      for (int u = 0; u < 16; u += 2) {                                 // unit 8 tile + 2 g + h
        const f32x16& c = acc[p * PASS + t][u >> 3];
        const int g = (u >> 1) & 3;
        *reinterpret_cast<f32x4*>(mine + (t * 32 + i) * 256 + (((u + h) ^ (i & 15)) << 4)) = f32x4{c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]};
      }
    }
#pragma unroll 1
    for (int r0 = 0; r0 < PASS * 32; r0 += 8 * AHEAD) {
      const int64_t m_first = mw + p * PASS * 32 + r0 + (lane >> 3);
      float res[AHEAD][8];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int64_t m = m_first + 8 * k;
        if (P.splits == 1 && inside && m < P.M) mat_residual<O, 8>(P, m, static_cast<int>(n), res[k]);
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int r = r0 + 8 * k + (lane >> 3), u = 2 * (lane & 7);
        const int64_t m = m_first + 8 * k;
        const f32x4 lo = *reinterpret_cast<const f32x4*>(mine + r * 256 + ((u ^ (r & 15)) << 4));
        const f32x4 hi = *reinterpret_cast<const f32x4*>(mine + r * 256 + (((u + 1) ^ (r & 15)) << 4));
        if (m < P.M && inside) {
          const float as = ES == 1 ? P.a_scale[m] : 1.f;
          float v[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = ES == 1 ? lo[e] * (as * scale[e]) : lo[e];
            v[4 + e] = ES == 1 ? hi[e] * (as * scale[4 + e]) : hi[e];
          }
          if (P.splits > 1) {
            store_chunk(P.part + (static_cast<int64_t>(split) * P.M + m) * P.N, n, P.N, v);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += bias[e];
            mat_finish<O, 8>(P, m, static_cast<int>(n), v, res[k]);
          }
        }
      }
    }
  }
}

template <class T, class O, int TA, int TB, int TM, int WM, int WN>
int tile_launch(const MatParams& P, hipStream_t s) {
  constexpr int BM = WM * TM * 32, BN = WN * 64;
  constexpr int LDS = 2 * (BM + BN) * 128;
  const int64_t tiles = ((P.M + BM - 1) / BM) * ((P.N + BN - 1) / BN);
  // 32-bit offsets inside a tile's lines, 31-bit tile count
  const int64_t far = 4 * 256 * (P.lda > P.ldb ? P.lda : P.ldb);
  if (tiles > 0x7fffffff || far + 2 * 128 * 256 > 0x7fffffff || P.splits < 1 || P.splits > 65535) return DGCN_E_SHAPE;
  if constexpr (LDS > 64 * 1024) {                                      // (a call costs as much host time as a small launch)
    const void* fn = reinterpret_cast<const void*>(tile_kernel<T, O, TA, TB, TM, WM, WN>);
    const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return static_cast<int>(e);
  }
  hipLaunchKernelGGL((tile_kernel<T, O, TA, TB, TM, WM, WN>), dim3(static_cast<unsigned>(tiles), P.splits), dim3(WM * WN * 64), LDS, s, P);
  return launch_status();
}

template <class T, class O, int TA, int TB>
int tile_size(const MatParams& P, int tile, hipStream_t s) {
  if (tile == 0) return tile_launch<T, O, TA, TB, 4, 2, 4>(P, s);
  if (tile == 1) return tile_launch<T, O, TA, TB, 2, 2, 2>(P, s);
  if constexpr (TA == 0) {
    if (tile == 2) return tile_launch<T, O, TA, TB, 1, 2, 2>(P, s);
  }
  return DGCN_E_MODE;
}

template <class T>
int tile_layout(const MatParams& P, int ta, int tb, int tile, hipStream_t s) {
  if (ta == 0 && tb == 0) return tile_size<T, T, 0, 0>(P, tile, s);
  if (ta == 0 && tb == 1) return tile_size<T, T, 0, 1>(P, tile, s);
  if (ta == 1 && tb == 1) return tile_size<T, T, 1, 1>(P, tile, s);
  return DGCN_E_MODE;
}

}  // namespace
}  // namespace dgcn
