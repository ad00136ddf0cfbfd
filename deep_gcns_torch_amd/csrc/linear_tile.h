// The tiled product on the matrix pipe: BM x BN tiles, 128 bytes of the reduction a step, operands copied straight from
// memory into LDS (two buffers), 16 x 16 matrix instructions, fp32 sums.
#pragma once

#include <type_traits>

#include "bf16x6.h"
#include "linear_act.h"

namespace dgcn {
namespace {

typedef int i8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s4v lds_s4;

// What a wave does with the fragments of one step (128 bytes of the reduction): a raw fragment is two 16-byte units of an
// operand row; prep() makes of it what the matrix instructions take, mul() adds four channel fragments' products.
template <class T> struct MatIn;

template <class T>
struct MatIn16 {
  static constexpr int ES = 2;
  struct Frag { u4v r[2]; };
  static __device__ __forceinline__ Frag prep(const u4v (&r)[2]) { return Frag{{r[0], r[1]}}; }
  static __device__ __forceinline__ f32x4 one(u4v a, u4v b, f32x4 c) {
    if constexpr (__is_same(T, __bf16)) {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
  }
  static __device__ __forceinline__ void mul(const Frag (&b)[4], const Frag& a, f32x4 (&c)[4]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int t = 0; t < 4; ++t) c[t] = one(b[t].r[s], a.r[s], c[t]);
    }
  }
  static __device__ __forceinline__ void one_tile(const Frag& b, const Frag& a, f32x4& c) {
    c = one(b.r[1], a.r[1], one(b.r[0], a.r[0], c));
  }
};
template <> struct MatIn<__bf16> : MatIn16<__bf16> {};
template <> struct MatIn<_Float16> : MatIn16<_Float16> {};

// fp32: three bf16 parts that add up to the value bit for bit, and the six products of parts down to 2^-16 of the largest
// (bf16x6.h: off by at most 3 2^-24 |a b|), at six times the cost of a bf16 product and a sixteenth of an fp32 one's
template <> struct MatIn<float> {
  static constexpr int ES = 4;
  struct Frag { i4v h, m, l; };
  static __device__ __forceinline__ Frag prep(const u4v (&r)[2]) {
    Frag f;
    eg_split3(__builtin_bit_cast(f4v, r[0]), __builtin_bit_cast(f4v, r[1]), f.h, f.m, f.l);
    return f;
  }
  static __device__ __forceinline__ void mul(const Frag (&b)[4], const Frag& a, f32x4 (&c)[4]) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = eg_mfma_bf16(b[t].m, a.m, c[t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = eg_mfma_bf16(b[t].l, a.h, c[t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = eg_mfma_bf16(b[t].h, a.l, c[t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = eg_mfma_bf16(b[t].m, a.h, c[t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = eg_mfma_bf16(b[t].h, a.m, c[t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = eg_mfma_bf16(b[t].h, a.h, c[t]);
  }
  static __device__ __forceinline__ void one_tile(const Frag& b, const Frag& a, f32x4& c) {
    c = eg_mfma_bf16(b.h, a.l, eg_mfma_bf16(b.l, a.h, eg_mfma_bf16(b.m, a.m, c)));
    c = eg_mfma_bf16(b.h, a.h, eg_mfma_bf16(b.h, a.m, eg_mfma_bf16(b.m, a.h, c)));
  }
};

// e4m3 for a 16-bit result: one instruction of K = 128 at twice the 16-bit rate, its block scales held at 2^0.  It aligns
// the products of eight neighbouring k to the largest one's exponent and drops what lies more than 13 bits below it
// (measured, bit by bit), so a sum is off by up to 7 2^-13 of the largest product of each eight: 6e-5 of the result's
// root mean square over normal rows, an order below a bf16 half step and under half of an fp16 one.
template <> struct MatIn<uint8_t> {
  static constexpr int ES = 1;
  typedef i8v Frag;
  static __device__ __forceinline__ Frag prep(const u4v (&r)[2]) {
    return __builtin_bit_cast(i8v, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
  static __device__ __forceinline__ void mul(const Frag (&b)[4], const Frag& a, f32x4 (&c)[4]) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[t], a, c[t], 0, 0, 0, 127, 0, 127);
  }
  static __device__ __forceinline__ void one_tile(const Frag& b, const Frag& a, f32x4& c) {
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, 0, 127, 0, 127);
  }
};
// e4m3 for an fp32 result: every e4m3 value is an fp16 value; their products are exact and their sum is fp32
struct WideE4m3 {};
template <> struct MatIn<WideE4m3> {
  static constexpr int ES = 1;
  struct Frag { u4v r[4]; };
  static __device__ __forceinline__ u4v widen(uint32_t lo, uint32_t hi) {
    return u4v{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true))};
  }
  static __device__ __forceinline__ Frag prep(const u4v (&r)[2]) {
    return Frag{{widen(r[0][0], r[0][1]), widen(r[0][2], r[0][3]), widen(r[1][0], r[1][1]), widen(r[1][2], r[1][3])}};
  }
  static __device__ __forceinline__ void mul(const Frag (&b)[4], const Frag& a, f32x4 (&c)[4]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
#pragma unroll
      for (int t = 0; t < 4; ++t) c[t] = MatIn16<_Float16>::one(b[t].r[s], a.r[s], c[t]);
    }
  }
  static __device__ __forceinline__ void one_tile(const Frag& b, const Frag& a, f32x4& c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = MatIn16<_Float16>::one(b.r[s], a.r[s], c);
  }
};

constexpr unsigned kRsrcFlags = 0x00027000;               // raw 32-bit buffer; a load behind its end gives zeros
constexpr unsigned kBehind = 0x80000000u;                 // an offset behind any buffer here (at most 2^31 bytes)

// Which rows / columns of an operand tile a 16-byte unit of LDS holds.
//   K-contiguous, R rows of 128 bytes: unit u of row r holds the row's chunk u ^ (r & 7)
//   K-strided, k-rows of R values: unit u of k-row k holds chunk u ^ 2 ((k & 3) | bit 3 of k << 2) in 16 bits,
//     u ^ 4 (bits 4, 3 of k) in 32
// In all, lanes that read together fall on different banks.
template <int T, int R, int ES>
__device__ __forceinline__ unsigned tile_offset(int inst, int lane, int64_t ld) {
  if constexpr (T == 0) {
    const int row = inst * 8 + (lane >> 3);
    return static_cast<unsigned>(row * ld * ES) + (((lane & 7) ^ (row & 7)) << 4);
  } else {
    constexpr int UNITS = R * ES / 16;
    const int k = inst * (64 / UNITS) + lane / UNITS;
    const int f = ES == 2 ? 2 * ((k & 3) | ((k >> 3) & 1) << 2) : 4 * ((k >> 3) & 3);
    return static_cast<unsigned>(k * ld * ES) + (((lane % UNITS) ^ f) << 4);
  }
}

// T: operand type, O: output type, TA / TB: layouts; a wave owns 16 TM rows x 64 channels, a workgroup WM x WN waves
template <class T, class O, int TA, int TB, int TM, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 2) void tile_kernel(const MatParams P) {
  constexpr int ES = MatIn<T>::ES;
  constexpr int BM = WM * TM * 16, BN = WN * 64, BK = 128 / ES, WAVES = WM * WN;
  constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  constexpr int IA = BM / 8 / WAVES, IB = BN / 8 / WAVES;               // copies a wave makes per step
  static_assert(IA * 8 * WAVES == BM && IB * 8 * WAVES == BN, "a step's copies divide over the waves");
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = lane_id(), wave = uni(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int i = lane & 15, q = lane >> 4;

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

  // Rows and k-rows behind the matrix lie behind the buffer's end and read as zeros; so do, by an offset of kBehind, the
  // chunks of a K-contiguous row behind K (a chunk that K ends in is the operand's zero padding from there).  Columns of a
  // K-strided operand behind M or N read what is there: their sums are not stored.
  constexpr int CH = 16 / ES;                                           // values in 16 bytes
  auto copy = [&](int step, int buf) {
    const int64_t k0 = static_cast<int64_t>(step) * BK;
    const int64_t left = P.K - k0 < BK ? P.K - k0 : BK;
    char* dst = lds + buf * STAGE;
    auto one = [&](auto layout, auto count, const void* base, int64_t ld, int64_t line0, int64_t lines, const unsigned* off, char* to) {
      constexpr int L = decltype(layout)::value, n = decltype(count)::value;
      const char* p = static_cast<const char*>(base) + (L == 0 ? line0 * ld + k0 : k0 * ld + line0) * ES;
      const int64_t bytes = (L == 0 ? (lines - 1) * ld + (left + CH - 1) / CH * CH : (left - 1) * ld + (lines + CH - 1) / CH * CH) * ES;
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, static_cast<int>(bytes), kRsrcFlags);
      if (L == 0 && left < BK) {
#pragma unroll
        for (int c = 0; c < n; ++c) {
          // byte of the row that this lane's chunk starts at
          const unsigned at = off[c] - static_cast<unsigned>(((wave * n + c) * 8 + (lane >> 3)) * ld * ES);
          __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(to + c * 1024), 16, at < left * ES ? off[c] : kBehind, 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int c = 0; c < n; ++c) __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(to + c * 1024), 16, off[c], 0, 0, 0);
      }
    };
    one(std::integral_constant<int, TA>{}, std::integral_constant<int, IA>{}, P.a, P.lda, m0, rows_a, offa, dst + wave * IA * 1024);
    one(std::integral_constant<int, TB>{}, std::integral_constant<int, IB>{}, P.b, P.ldb, n0, rows_b, offb, dst + A_BYTES + wave * IB * 1024);
  };

  f32x4 acc[TM][4];
#pragma unroll
  for (int tm = 0; tm < TM; ++tm) {
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[tm][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Raw fragment of 16 operand rows (or columns), row i on lane (i, q).  One byte a value: chunks q and q + 4 of the row's
  // eight; two: likewise, k = 8 q .. of each half; four: chunks 2 q and 2 q + 1, k = 8 q .. 8 q + 7.
  const int at0 = ((ES == 4 ? 2 * q : q) ^ (i & 7)) << 4, at1 = at0 ^ (ES == 4 ? 16 : 64);
  const int kk = i >> 2, pc = i & 3;                                    // K-strided, 16 bits: the lane fetches four columns of k-row 8 q + kk
  const int f2 = (kk | (q & 1) << 2) << 5;
  auto read = [&](auto layout, const char* base, int line, int rows, u4v (&out)[2]) {
    constexpr int L = decltype(layout)::value;
    if constexpr (L == 0) {
      const char* p = base + (line + i) * 128;
      out[0] = *reinterpret_cast<const u4v*>(p + at0);
      out[1] = *reinterpret_cast<const u4v*>(p + at1);
    } else if constexpr (ES == 2) {
      const char* p = base + (8 * q + kk) * rows * 2 + ((line * 2 + ((pc >> 1) << 4)) ^ f2) + (pc & 1) * 8;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + (32 * s) * rows * 2));
        const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + (32 * s + 4) * rows * 2));
        out[s] = __builtin_bit_cast(u4v, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    } else {
      const char* p = base + 8 * q * rows * 4 + (((line + i) * 4) ^ (q << 6));
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e >> 2][e & 3] = *reinterpret_cast<const uint32_t*>(p + e * rows * 4);
    }
  };

  if (s0 < s1) copy(s0, 0);
  for (int step = s0; step < s1; ++step) {
    const int buf = (step - s0) & 1;
    __builtin_amdgcn_s_waitcnt(0x0f70);                                // vmcnt(0): this wave's copies have landed
    __syncthreads();                                                   // everyone's have; nobody still reads the other buffer
    if (step + 1 < s1) copy(step + 1, buf ^ 1);
    const char* sa = lds + buf * STAGE;
    const char* sb = sa + A_BYTES;
    typename MatIn<T>::Frag fb[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      u4v raw[2];
      read(std::integral_constant<int, TB>{}, sb, wn * 64 + 16 * t, BN, raw);
      fb[t] = MatIn<T>::prep(raw);
    }
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) {
      u4v raw[2];
      read(std::integral_constant<int, TA>{}, sa, wm * TM * 16 + tm * 16, BM, raw);
      MatIn<T>::mul(fb, MatIn<T>::prep(raw), acc[tm]);
    }
  }

  // Epilogue, through LDS (the operand buffers are free): a wave writes its sums as rows of 64 channels, up to 64 rows at a
  // time, and takes them back eight rows by eight channels a lane, so that a store fills whole lines and the code is one
  // rolled loop.  Lane (i, q) holds row i of each 16 and, of fragment t, matrix rows 4 q .. 4 q + 3.  16-byte unit u of row
  // r lies at u ^ (r & 15).  A wave reads only what it wrote.
  constexpr int PASS = TM < 4 ? TM : 4;
  __syncthreads();
  char* mine = lds + wave * (PASS * 16 * 256);
  const int64_t mw = m0 + wm * TM * 16, n = n0 + wn * 64 + 8 * (lane & 7);
  float bs[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) bs[e] = (ES == 1 && n + e < P.N) ? P.b_scale[n + e] : 1.f;
#pragma unroll
  for (int p = 0; p < TM / PASS; ++p) {
#pragma unroll
    for (int tm = 0; tm < PASS; ++tm) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        *reinterpret_cast<f32x4*>(mine + (tm * 16 + i) * 256 + (((4 * t + q) ^ i) << 4)) = acc[p * PASS + tm][t];
      }
    }
#pragma unroll 1
    for (int r0 = 0; r0 < PASS * 16; r0 += 8) {
      const int r = r0 + (lane >> 3), u = 2 * (lane & 7);
      const int64_t m = mw + p * PASS * 16 + r;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(mine + r * 256 + ((u ^ (r & 15)) << 4));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(mine + r * 256 + (((u + 1) ^ (r & 15)) << 4));
      if (m < P.M && n < P.N) {
        const float as = ES == 1 ? P.a_scale[m] : 1.f;
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = ES == 1 ? lo[e] * (as * bs[e]) : lo[e];
          v[4 + e] = ES == 1 ? hi[e] * (as * bs[4 + e]) : hi[e];
        }
        if (P.splits > 1) {
          store_chunk(P.part + (static_cast<int64_t>(split) * P.M + m) * P.N, n, P.N, v);
        } else {
          mat_epilogue<O, 8>(P, m, n, v);
        }
      }
    }
  }
}

template <class T, class O, int TA, int TB, int TM, int WM, int WN>
int tile_launch(const MatParams& P, hipStream_t s) {
  constexpr int BM = WM * TM * 16, BN = WN * 64;
  constexpr int LDS = 2 * (BM + BN) * 128;
  const int64_t tiles = ((P.M + BM - 1) / BM) * ((P.N + BN - 1) / BN);
  // 32-bit offsets inside a tile's lines, 31-bit tile count
  const int64_t far = 4 * 256 * (P.lda > P.ldb ? P.lda : P.ldb);
  if (tiles > 0x7fffffff || far + 2 * 128 * 256 > 0x7fffffff || P.splits < 1 || P.splits > 65535) return DGCN_E_SHAPE;
  const void* fn = reinterpret_cast<const void*>(tile_kernel<T, O, TA, TB, TM, WM, WN>);
  const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (e != hipSuccess) return static_cast<int>(e);
  hipLaunchKernelGGL((tile_kernel<T, O, TA, TB, TM, WM, WN>), dim3(static_cast<unsigned>(tiles), P.splits), dim3(WM * WN * 64), LDS, s, P);
  return launch_status();
}

template <class T, class O, int TA, int TB>
int tile_size(const MatParams& P, int tile, hipStream_t s) {
  if (tile == 0) return tile_launch<T, O, TA, TB, 8, 2, 4>(P, s);
  if (tile == 1) return tile_launch<T, O, TA, TB, 4, 2, 2>(P, s);
  if constexpr (TA == 0) {
    if (tile == 2) return tile_launch<T, O, TA, TB, 2, 2, 2>(P, s);
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
