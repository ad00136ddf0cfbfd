// Element types, eight-element chunks and activations shared by the node-wise MLP kernels (rms_norm.hip,
// linear_act.hip).  Everything is computed in fp32; a 16-bit value is rounded once, to nearest even, where it is stored.
#pragma once

#include "dgcn_common.h"

namespace dgcn {

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Vector accesses at the element's own alignment: the device runs in unaligned-access mode, a global dwordx4 may start
// at any byte.  Rows of odd length or stride take the same wide loads as aligned ones.
typedef u4v u4v_any2 __attribute__((aligned(2)));
typedef u4v u4v_any4 __attribute__((aligned(4)));
typedef u2v u2v_any2 __attribute__((aligned(2)));
typedef u2v u2v_any1 __attribute__((aligned(1)));

template <class T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };
template <class T> struct Vec4;
template <> struct Vec4<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(4))); };
template <> struct Vec4<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(4))); };

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = __builtin_bit_cast(f32x4, *reinterpret_cast<const u4v_any4*>(p));
    const f32x4 b = __builtin_bit_cast(f32x4, *reinterpret_cast<const u4v_any4*>(p + 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
  } else {
    const auto a = __builtin_bit_cast(typename Vec8<T>::type, *reinterpret_cast<const u4v_any2*>(p));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(a[e]);
  }
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<u4v_any4*>(p) = __builtin_bit_cast(u4v, f32x4{v[0], v[1], v[2], v[3]});
    *reinterpret_cast<u4v_any4*>(p + 4) = __builtin_bit_cast(u4v, f32x4{v[4], v[5], v[6], v[7]});
  } else {
    typename Vec8<T>::type a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = static_cast<T>(v[e]);
    *reinterpret_cast<u4v_any2*>(p) = __builtin_bit_cast(u4v, a);
  }
}

template <class T>
__device__ __forceinline__ void load4(const T* p, float* v) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = __builtin_bit_cast(f32x4, *reinterpret_cast<const u4v_any4*>(p));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e];
  } else {
    const auto a = __builtin_bit_cast(typename Vec4<T>::type, *reinterpret_cast<const u2v_any2*>(p));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(a[e]);
  }
}

template <class T>
__device__ __forceinline__ void store4(T* p, const float* v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<u4v_any4*>(p) = __builtin_bit_cast(u4v, f32x4{v[0], v[1], v[2], v[3]});
  } else {
    typename Vec4<T>::type a;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = static_cast<T>(v[e]);
    *reinterpret_cast<u2v_any2*>(p) = __builtin_bit_cast(u2v, a);
  }
}

// elements [start, start + CNT) of a row of n, CNT = 4 or 8 (behind the end: reads as `fill`, is not written)
template <class T, int CNT>
__device__ __forceinline__ void load_run(const T* row, int start, int n, float (&v)[CNT], float fill = 0.f) {
  if (start + CNT <= n) {
    if constexpr (CNT == 8) load8(row + start, v); else load4(row + start, v);
  } else {
#pragma unroll
    for (int e = 0; e < CNT; ++e) v[e] = start + e < n ? static_cast<float>(row[start + e]) : fill;
  }
}

template <class T, int CNT>
__device__ __forceinline__ void store_run(T* row, int start, int n, const float (&v)[CNT]) {
  if (start + CNT <= n) {
    if constexpr (CNT == 8) store8(row + start, v); else store4(row + start, v);
  } else {
#pragma unroll
    for (int e = 0; e < CNT; ++e) {
      if (start + e < n) row[start + e] = static_cast<T>(v[e]);
    }
  }
}

template <class T>
__device__ __forceinline__ void load_chunk(const T* row, int start, int n, float (&v)[8], float fill = 0.f) {
  load_run<T, 8>(row, start, n, v, fill);
}
template <class T>
__device__ __forceinline__ void store_chunk(T* row, int start, int n, const float (&v)[8]) {
  store_run<T, 8>(row, start, n, v);
}

template <class T, int CNT>
__device__ __forceinline__ void load_param_run(const void* p, bool f32, int start, int n, float (&v)[CNT]) {
  if (f32) {
    load_run<float, CNT>(static_cast<const float*>(p), start, n, v);
  } else {
    load_run<T, CNT>(static_cast<const T*>(p), start, n, v);
  }
}

// parameters (weight, bias) come in the rows' type or in fp32
template <class T>
__device__ __forceinline__ void load_param_chunk(const void* p, bool f32, int start, int n, float (&v)[8], float none) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = none;
  } else if (f32) {
    load_chunk(static_cast<const float*>(p), start, n, v, none);
  } else {
    load_chunk(static_cast<const T*>(p), start, n, v, none);
  }
}

// four fp32 values -> four e4m3 bytes, to nearest even (|v| <= 448 up to rounding; anything not finite -> NaN, 0x7f)
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}

// ---- activations: act(z) and act'(z), in fp32 ----
// EXACT (the fp32 type): libm's exp and the longer fit below.  Otherwise the hardware's 2^x, off by |z| 2^-24, its reciprocal,
// and the shorter fit: all far below a 16-bit half step (bf16 2^-9, fp16 2^-12 of a value in [1, 2)).
template <bool EXACT>
__device__ __forceinline__ float act_exp(float x) { return EXACT ? expf(x) : fast_exp(x); }
template <bool EXACT>
__device__ __forceinline__ float act_inv(float x) { return EXACT ? 1.f / x : __builtin_amdgcn_rcpf(x); }

// Phi(z) and, in `bell`, exp(-z^2 / 2).  Both sides come from erfc(|z| / sqrt 2), so that nothing cancels for z < 0:
// erfc(x) = exp(-x^2) t P(t), t = 1 / (1 + p x), P fitted to the least relative error over 0 <= x <= 10 (degree eight, p = 0.5:
// 4e-8, with fp32's own rounding 7e-8 on average) or 14 (degree five, p = 0.45: 1e-5).  libm's erfc is several times as many
// instructions, and a 256 x 256 tile evaluates 65,536 of them.
template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float z, float& bell) {
  constexpr float kFit[9] = {0.282086422f, 0.282375231f, 0.243104417f, 0.202683901f, -0.0266177002f, 0.278054163f, -0.487187249f, 0.284568217f, -0.0590674445f};
  constexpr float kShort[6] = {0.25396813f, 0.251702589f, 0.248475618f, 0.0894637792f, 0.292237032f, -0.135856623f};
  bell = act_exp<EXACT>(-0.5f * z * z);
  const float t = act_inv<EXACT>(fmaf((EXACT ? 0.5f : 0.45f) * 0.70710678118654752f, fabsf(z), 1.f));
  float p = EXACT ? kFit[8] : kShort[5];
#pragma unroll
  for (int k = EXACT ? 7 : 4; k >= 0; --k) p = fmaf(p, t, EXACT ? kFit[k] : kShort[k < 6 ? k : 5]);
  const float tail = (0.5f * p * t) * bell;                            // Phi(-|z|)
  return z < 0.f ? tail : 1.f - tail;
}

// act(z), and act'(z) in `d` (unused: dropped by the compiler)
template <bool EXACT>
__device__ __forceinline__ float act_both(float z, int act, float slope, float& d) {
  switch (act) {
    case DGCN_ACT_RELU:                                                 // (NaN stays NaN)
      d = z > 0.f ? 1.f : z != z ? z : 0.f;
      return z < 0.f ? 0.f : z;
    case DGCN_ACT_LEAKY_RELU:
      d = z > 0.f ? 1.f : slope;
      return z > 0.f ? z : slope * z;
    case DGCN_ACT_GELU: {
      float bell;
      const float cdf = normal_cdf<EXACT>(z, bell);
      d = fmaf(z * 0.39894228040143268f, bell, cdf);
      return z * cdf;
    }
    case DGCN_ACT_SILU: {
      const float s = act_inv<EXACT>(1.f + act_exp<EXACT>(-z));
      const float y = z * s;
      d = fmaf(y, 1.f - s, s);
      return y;
    }
    default: d = 1.f; return z;
  }
}

template <bool EXACT>
__device__ __forceinline__ float act_slope(float z, int act, float slope) {
  float d;
  act_both<EXACT>(z, act, slope, d);
  return d;
}

// ---- what the backward of an activation in 16 bits keeps: act'(z) as a 16-bit code ----
// Codes up to kGateTail are fixed point, code = (act' + 1/4) 2^15: gelu's and silu's slopes lie in (-0.13, 1.13) and come back
// within 2^-16, an eighth of a bf16 half step of slopes near 1.  (z in 16 bits would be off by half a step of z in act': measured,
// 1.5 times the error of the bias gradient.)  Where a unit is saturated the slope is negative and small, and 2^-16 is too much of it
// (3 % of gelu's at z = -4, all of it at -5): slopes from -2^-6 to -2^-45 take the codes that no fixed-point slope has, as
// floating point with nine bits behind the leading one, within 2^-10 of themselves; what is smaller (gelu from z = -8.1, silu from
// -34.7) is 0.  relu and leakyrelu keep z > 0 as a slope of 1 or 0.  Code 0 is NaN (what the conversion makes of one).
constexpr uint32_t kGateTail = 45568;                      // 39 binades of 512 codes up to 65535; below it slopes up to 1.14
constexpr uint32_t kGateLow = 0x20000 + (82 << 9);         // the top 18 bits of -2^-45

__device__ __forceinline__ uint32_t gate_encode(float d) {
  uint32_t c;
  asm("v_cvt_u32_f32 %0, %1" : "=v"(c) : "v"(fmaf(d, 32768.f, 8192.5f)));
  return c;
}

__device__ __forceinline__ uint32_t gate_encode_tail(float d) {
  const uint32_t u = ((__float_as_uint(d) + 0x2000u) >> 14) - kGateLow;
  return u <= 0xffffu - kGateTail ? u + kGateTail : gate_encode(d);
}

__device__ __forceinline__ float gate_decode(uint32_t code, int act, float slope) {
  const float d = fmaf(static_cast<float>(code), 1.f / 32768.f, -0.25f);
  if (code == 0u) return __builtin_nanf("");
  if (code >= kGateTail) return __uint_as_float((code - kGateTail + kGateLow) << 14);
  return act == DGCN_ACT_LEAKY_RELU && code == 8192u ? slope : d;
}

// a run of values under one (uniform) activation: the branch is outside the run
template <bool EXACT, int CNT>
__device__ __forceinline__ void act_run(float (&v)[CNT], int act, float slope) {
  float d;
  switch (act) {
#define DGCN_ACT_CASE(A) case A: { _Pragma("unroll") for (int e = 0; e < CNT; ++e) v[e] = act_both<EXACT>(v[e], A, slope, d); break; }
    DGCN_ACT_CASE(DGCN_ACT_RELU)
    DGCN_ACT_CASE(DGCN_ACT_LEAKY_RELU)
    DGCN_ACT_CASE(DGCN_ACT_GELU)
    DGCN_ACT_CASE(DGCN_ACT_SILU)
#undef DGCN_ACT_CASE
    default: break;
  }
}

// the same in 16 bits, and the gate codes
template <int CNT>
__device__ __forceinline__ void act_gate_run(float (&v)[CNT], uint32_t (&c)[CNT], int act, float slope) {
  float d;
  switch (act) {
#define DGCN_ACT_CASE(A, ENCODE) case A: { _Pragma("unroll") for (int e = 0; e < CNT; ++e) { v[e] = act_both<false>(v[e], A, slope, d); c[e] = ENCODE(d); } break; }
    case DGCN_ACT_LEAKY_RELU: {
#pragma unroll
      for (int e = 0; e < CNT; ++e) {
        act_both<false>(v[e], DGCN_ACT_RELU, slope, d);
        c[e] = gate_encode(d);
        v[e] = act_both<false>(v[e], DGCN_ACT_LEAKY_RELU, slope, d);
      }
      break;
    }
    DGCN_ACT_CASE(DGCN_ACT_RELU, gate_encode)
    DGCN_ACT_CASE(DGCN_ACT_GELU, gate_encode_tail)
    DGCN_ACT_CASE(DGCN_ACT_SILU, gate_encode_tail)
#undef DGCN_ACT_CASE
    default: break;
  }
}

template <int CNT>
__device__ __forceinline__ void store_gates(uint16_t* row, int start, int n, const uint32_t (&c)[CNT]) {
  if (start + CNT <= n) {
    if constexpr (CNT == 8) {
      *reinterpret_cast<u4v_any2*>(row + start) = u4v{c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | c[7] << 16};
    } else {
      *reinterpret_cast<u2v_any2*>(row + start) = u2v{c[0] | c[1] << 16, c[2] | c[3] << 16};
    }
  } else {
#pragma unroll
    for (int e = 0; e < CNT; ++e) {
      if (start + e < n) row[start + e] = static_cast<uint16_t>(c[e]);
    }
  }
}

// act'(z) of eight values of a row, from what the forward kept
template <class T>
__device__ __forceinline__ void load_slopes(const void* kept, int64_t row_at, int start, int n, int act, float slope, float (&d)[8]) {
  if constexpr (sizeof(T) == 4) {
    load_chunk(static_cast<const float*>(kept) + row_at, start, n, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = act_slope<true>(d[e], act, slope);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(kept) + row_at;
    if (start + 8 <= n) {
      const u4v v = *reinterpret_cast<const u4v_any2*>(p + start);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = gate_decode((v[e >> 1] >> (16 * (e & 1))) & 0xffffu, act, slope);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = start + e < n ? gate_decode(p[start + e], act, slope) : 0.f;
    }
  }
}

}  // namespace dgcn
