// The product of a few rows (16; 32 whose rows do not start on dwords) with a weight: what a model answers with one token or one node at a time.
//
// Bound by reading the weight once (2 rows flop a byte in 16 bits).  A workgroup owns 16 channels and all of K, its eight or
// sixteen waves take the 128-byte steps of the reduction in turn, straight from memory into matrix fragments (no LDS: nothing of
// the weight is used twice), UNROLL steps requested ahead; the waves' sums meet in LDS in wave order.  Rows may start at any
// byte, so odd strides and lengths need no copy of the weight.  Measured: 4096 x 4096 bf16, one row 7.8 us (4.3 TB/s),
// the same over 24 weights in turn, which no cache holds; 16,384 x 4096 e4m3, 16 rows 14.4 us (4.7 TB/s), over 12 weights in
// turn 17.6 (3.8 TB/s); 4096 x 4096 fp32, one row 17.2 us (3.9 TB/s), over 12 weights in turn 18.0.
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

// e4m3: exact products, summed in fp32 (the 8-bit instruction would cut them, see TileIn<uint8_t>; here the pipe has time:
// 16,384 x 4096, 16 rows, 14.9 us with either)
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

// A row that the kernel reads 16 bytes at a time.  Loads may start at any byte, but off a dword they take more than twice
// as long (14,057 e4m3 channels, 5,121 rows of weight: 60 us against 29): SHIFT reads the five dwords that hold the 16 bytes,
// which lie in the same allocation as the bytes do, and takes them together by a byte shift.
template <bool SHIFT>
struct Row {
  const char* p;
  uint32_t by;
  __device__ __forceinline__ explicit Row(const char* row) : p(row), by(0) {
    if constexpr (SHIFT) {
      by = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 3u);
      p = row - by;
    }
  }
  __device__ __forceinline__ u4v at(int64_t a) const {
    if constexpr (!SHIFT) return *reinterpret_cast<const u4v_any4*>(p + a);
    const u4v v = *reinterpret_cast<const u4v_any4*>(p + a);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p + a + (by ? 16 : 12));
    return u4v{__builtin_amdgcn_alignbyte(v[1], v[0], by), __builtin_amdgcn_alignbyte(v[2], v[1], by),
               __builtin_amdgcn_alignbyte(v[3], v[2], by), __builtin_amdgcn_alignbyte(w, v[3], by)};
  }
  // at(a) of a row of `bytes`, zeros behind its end
  __device__ __forceinline__ u4v end(int64_t a, int64_t bytes) const {
    if (a + 16 <= bytes) return at(a);
    u4v v = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if (a + e < bytes) v[e >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(p[a + by + e])) << (8 * (e & 3));
    }
    return v;
  }
};

// MT: tiles of 16 rows, NT: tiles of 16 channels a workgroup owns
template <class T, class O, int MT, int NT, int WAVES, bool SHIFT>
__global__ __launch_bounds__(WAVES * 64) void small_kernel(const MatParams P) {
  constexpr int ES = MatIn<T>::ES, UNROLL = MT * NT == 1 ? 4 : 2;
  __shared__ f32x4 red[WAVES][MT * NT][64];
  const int lane = lane_id(), wave = uni(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT), bytes = P.K * ES;
  auto row_of = [&](const void* x, int64_t r, int64_t n, int64_t ld) { return static_cast<const char*>(x) + (r < n ? r : n - 1) * ld * ES; };
  const Row<SHIFT> w0(row_of(P.b, n0 + i, P.N, P.ldb)), w1(row_of(P.b, n0 + 16 * (NT - 1) + i, P.N, P.ldb));
  const Row<SHIFT> x0(row_of(P.a, i, P.M, P.lda)), x1(row_of(P.a, 16 * (MT - 1) + i, P.M, P.lda));
  const int at0 = (ES == 4 ? 2 * q : q) * 16, at1 = at0 + (ES == 4 ? 16 : 64);
  f32x4 acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto w_row = [&](int u) -> const Row<SHIFT>& { return u ? w1 : w0; };
  auto x_row = [&](int t) -> const Row<SHIFT>& { return t ? x1 : x0; };
  auto add = [&](const u4v (&rw)[NT][2], const u4v (&rx)[MT][2]) {
    typename MatIn<T>::Frag w[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) w[u] = MatIn<T>::prep(rw[u]);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const typename MatIn<T>::Frag x = MatIn<T>::prep(rx[t]);
#pragma unroll
      for (int u = 0; u < NT; ++u) MatIn<T>::one_tile(w[u], x, acc[t][u]);
    }
  };
  const int64_t whole = bytes / 128;                       // steps that end inside every row
  int64_t s = wave;
  for (; s + (UNROLL - 1) * WAVES < whole; s += UNROLL * WAVES) {
    u4v rw[UNROLL][NT][2], rx[UNROLL][MT][2];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int64_t at = (s + k * WAVES) * 128;
#pragma unroll
      for (int u = 0; u < NT; ++u) { rw[k][u][0] = w_row(u).at(at + at0); rw[k][u][1] = w_row(u).at(at + at1); }
#pragma unroll
      for (int t = 0; t < MT; ++t) { rx[k][t][0] = x_row(t).at(at + at0); rx[k][t][1] = x_row(t).at(at + at1); }
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) add(rw[k], rx[k]);
  }
  for (; s * 128 < bytes; s += WAVES) {
    const int64_t at = s * 128;
    u4v rw[NT][2], rx[MT][2];
#pragma unroll
    for (int u = 0; u < NT; ++u) { rw[u][0] = w_row(u).end(at + at0, bytes); rw[u][1] = w_row(u).end(at + at1, bytes); }
#pragma unroll
    for (int t = 0; t < MT; ++t) { rx[t][0] = x_row(t).end(at + at0, bytes); rx[t][1] = x_row(t).end(at + at1, bytes); }
    add(rw, rx);
  }
  if constexpr (std::is_same<T, float>::value) {           // see f32_kinds
#pragma unroll
    for (int t = 0; t < MT * NT; ++t) {
      f32x4& c = acc[t / NT][t % NT];
      if (!any_nan(c)) continue;
      auto of = [&](const Row<SHIFT>& row, int64_t at) {
        const f32x4 lo = __builtin_bit_cast(f32x4, row.end(at + at0, bytes)), hi = __builtin_bit_cast(f32x4, row.end(at + at1, bytes));
        const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        return f32_kinds(v);
      };
      f32x4 kinds = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int64_t at = 128 * wave; at < bytes; at += 128 * WAVES) kinds = MatIn16<__bf16>::one(of(w_row(t % NT), at), of(x_row(t / NT), at), kinds);
      take_kinds(c, kinds);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int u = 0; u < NT; ++u) red[wave][t * NT + u][lane] = acc[t][u];
  }
  __syncthreads();
  // lane (i, q) of tile (t, u): row 16 t + i, channels 16 u + 4 q .. + 3
  if (wave < MT * NT) {
    f32x4 sum = red[0][wave][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += red[w][wave][lane];
    const int64_t m = 16 * (wave / NT) + i, n = n0 + 16 * (wave % NT) + 4 * q;
    if (m < P.M && n < P.N) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = ES == 1 ? sum[e] * (P.a_scale[m] * (n + e < P.N ? P.b_scale[n + e] : 0.f)) : sum[e];
      mat_epilogue<O, 4>(P, m, n, v);
    }
  }
}

template <class T, class O, int MT, int NT, int WAVES>
int small_go(const MatParams& P, bool shift, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((P.N + 16 * NT - 1) / (16 * NT)));
  if constexpr (MatIn<T>::ES < 4) {
    if (shift) {
      hipLaunchKernelGGL((small_kernel<T, O, MT, NT, WAVES, true>), grid, dim3(WAVES * 64), 0, s, P);
      return launch_status();
    }
  }
  hipLaunchKernelGGL((small_kernel<T, O, MT, NT, WAVES, false>), grid, dim3(WAVES * 64), 0, s, P);
  return launch_status();
}

// Sixteen waves where the channels give at most one workgroup a CU and each wave still has four steps (4096 x 4096 bf16: one
// row 7.9 us against 9.4 with eight, 16 rows 10.0 against 10.3); 32 channels a workgroup for e4m3 where they give every CU one
// (16,384 x 4096, 16 rows: 14.4 us against 17.8, one row 13.4 against 16.1; 8192 x 8192, which gives each just one: 19.9
// against 16.9; in 16 bits it is slower, 35.5 against 34.1).
template <class T, class O>
int small_launch(const MatParams& P, hipStream_t s) {
  constexpr int ES = MatIn<T>::ES;
  const uintptr_t off = reinterpret_cast<uintptr_t>(P.a) | reinterpret_cast<uintptr_t>(P.b) | static_cast<uintptr_t>(P.lda * ES) | static_cast<uintptr_t>(P.ldb * ES);
  const bool shift = (off & 3) != 0;
  if (P.M > 32) return DGCN_E_SHAPE;
  if (P.M > 16) return small_go<T, O, 2, 1, 8>(P, shift, s);
  if constexpr (ES == 1) {
    if (P.N >= 32 * static_cast<int64_t>(num_cus())) return small_go<T, O, 1, 2, 8>(P, shift, s);
  }
  if (P.N <= 16 * static_cast<int64_t>(num_cus()) && P.K * ES >= 64 * 128) return small_go<T, O, 1, 1, 16>(P, shift, s);
  return small_go<T, O, 1, 1, 8>(P, shift, s);
}

}  // namespace
}  // namespace dgcn
