// The product of a few rows (kSmallRows at most) with a weight: what a model answers with one token or one node at a time.
//
// Bound by reading the weight once (2 rows flop a byte in 16 bits).  A workgroup owns 16 channels and all of K, its eight
// waves take the 128-byte steps of the reduction in turn, straight from memory into matrix fragments (no LDS: nothing of
// the weight is used twice), UNROLL steps requested ahead; the waves' sums meet in LDS in wave order.  Loads may start at
// any byte, so odd strides and lengths need no copy of the weight.
#pragma once

#include "linear_tile.h"

namespace dgcn {
namespace {

// The types' fragments of a step (128 bytes of the reduction) for 16 x 16 matrix instructions; see TileIn
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
  static __device__ __forceinline__ void one_tile(const Frag& b, const Frag& a, f32x4& c) {
    c = one(b.r[1], a.r[1], one(b.r[0], a.r[0], c));
  }
};
template <> struct MatIn<__bf16> : MatIn16<__bf16> {};
template <> struct MatIn<_Float16> : MatIn16<_Float16> {};

template <> struct MatIn<float> {
  static constexpr int ES = 4;
  struct Frag { i4v h, m, l; };
  static __device__ __forceinline__ Frag prep(const u4v (&r)[2]) {
    Frag f;
    eg_split3(__builtin_bit_cast(f4v, r[0]), __builtin_bit_cast(f4v, r[1]), f.h, f.m, f.l);
    return f;
  }
  static __device__ __forceinline__ void one_tile(const Frag& b, const Frag& a, f32x4& c) {
    c = eg_mfma_bf16(b.h, a.l, eg_mfma_bf16(b.l, a.h, eg_mfma_bf16(b.m, a.m, c)));
    c = eg_mfma_bf16(b.h, a.h, eg_mfma_bf16(b.h, a.m, eg_mfma_bf16(b.m, a.h, c)));
  }
};

template <> struct MatIn<uint8_t> {
  static constexpr int ES = 1;
  typedef i8v Frag;
  static __device__ __forceinline__ Frag prep(const u4v (&r)[2]) {
    return __builtin_bit_cast(i8v, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
  static __device__ __forceinline__ void one_tile(const Frag& b, const Frag& a, f32x4& c) {
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, 0, 127, 0, 127);
  }
};
template <> struct MatIn<WideE4m3> {
  static constexpr int ES = 1;
  struct Frag { u4v r[4]; };
  static __device__ __forceinline__ Frag prep(const u4v (&r)[2]) {
    return Frag{{widen_e4m3(r[0][0], r[0][1]), widen_e4m3(r[0][2], r[0][3]), widen_e4m3(r[1][0], r[1][1]), widen_e4m3(r[1][2], r[1][3])}};
  }
  static __device__ __forceinline__ void one_tile(const Frag& b, const Frag& a, f32x4& c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = MatIn16<_Float16>::one(b.r[s], a.r[s], c);
  }
};

typedef u4v u4v_any1 __attribute__((aligned(1)));

// 16 bytes at `at` of a row of `bytes`; behind its end zeros
__device__ __forceinline__ u4v row_unit(const char* row, int64_t at, int64_t bytes) {
  if (at + 16 <= bytes) return *reinterpret_cast<const u4v_any1*>(row + at);
  u4v v = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    if (at + e < bytes) v[e >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[at + e])) << (8 * (e & 3));
  }
  return v;
}

constexpr int kSmallWaves = 8;

// MT: tiles of 16 rows
template <class T, class O, int MT>
__global__ __launch_bounds__(kSmallWaves * 64) void small_kernel(const MatParams P) {
  constexpr int ES = MatIn<T>::ES, UNROLL = MT == 1 ? 4 : 2;
  __shared__ f32x4 red[kSmallWaves][MT][64];
  const int lane = lane_id(), wave = uni(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16, bytes = P.K * ES;
  const int64_t nrow = n0 + i < P.N ? n0 + i : P.N - 1;
  const char* wrow = static_cast<const char*>(P.b) + nrow * P.ldb * ES;
  const char* xrow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = 16 * t + i < P.M ? 16 * t + i : P.M - 1;
    xrow[t] = static_cast<const char*>(P.a) + m * P.lda * ES;
  }
  const int at0 = (ES == 4 ? 2 * q : q) * 16, at1 = at0 + (ES == 4 ? 16 : 64);
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto add = [&](const u4v (&rw)[2], const u4v (&rx)[MT][2]) {
    const typename MatIn<T>::Frag w = MatIn<T>::prep(rw);
#pragma unroll
    for (int t = 0; t < MT; ++t) MatIn<T>::one_tile(w, MatIn<T>::prep(rx[t]), acc[t]);
  };
  const int64_t whole = bytes / 128;                       // steps that end inside every row
  int64_t s = wave;
  for (; s + (UNROLL - 1) * kSmallWaves < whole; s += UNROLL * kSmallWaves) {
    u4v rw[UNROLL][2], rx[UNROLL][MT][2];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t at = (s + u * kSmallWaves) * 128;
      rw[u][0] = *reinterpret_cast<const u4v_any1*>(wrow + at + at0);
      rw[u][1] = *reinterpret_cast<const u4v_any1*>(wrow + at + at1);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        rx[u][t][0] = *reinterpret_cast<const u4v_any1*>(xrow[t] + at + at0);
        rx[u][t][1] = *reinterpret_cast<const u4v_any1*>(xrow[t] + at + at1);
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) add(rw[u], rx[u]);
  }
  for (; s * 128 < bytes; s += kSmallWaves) {
    const int64_t at = s * 128;
    u4v rw[2] = {row_unit(wrow, at + at0, bytes), row_unit(wrow, at + at1, bytes)}, rx[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      rx[t][0] = row_unit(xrow[t], at + at0, bytes);
      rx[t][1] = row_unit(xrow[t], at + at1, bytes);
    }
    add(rw, rx);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  // lane (i, q) of tile t: row 16 t + i, channels 4 q .. 4 q + 3
  if (wave < MT) {
    f32x4 sum = red[0][wave][lane];
#pragma unroll
    for (int w = 1; w < kSmallWaves; ++w) sum += red[w][wave][lane];
    const int64_t m = 16 * wave + i, n = n0 + 4 * q;
    if (m < P.M && n < P.N) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = ES == 1 ? sum[e] * (P.a_scale[m] * (n + e < P.N ? P.b_scale[n + e] : 0.f)) : sum[e];
      mat_epilogue<O, 4>(P, m, n, v);
    }
  }
}

template <class T, class O, int MT>
int small_go(const MatParams& P, hipStream_t s) {
  hipLaunchKernelGGL((small_kernel<T, O, MT>), dim3(static_cast<unsigned>((P.N + 15) / 16)), dim3(kSmallWaves * 64), 0, s, P);
  return launch_status();
}

template <class T, class O>
int small_launch(const MatParams& P, hipStream_t s) {
  if (P.M <= 16) return small_go<T, O, 1>(P, s);
  if (P.M <= 32) return small_go<T, O, 2>(P, s);
  return P.M <= 64 ? small_go<T, O, 4>(P, s) : DGCN_E_SHAPE;
}

}  // namespace
}  // namespace dgcn
