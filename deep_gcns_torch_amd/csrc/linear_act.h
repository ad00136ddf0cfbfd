// What the product kernels share: the description of one product, and the epilogue of a run of consecutive channels.
#pragma once

#include "mlp_common.h"

namespace dgcn {

// Y(m, n) = epilogue( sum_k A(m, k) B(n, k) ).  An operand is K-contiguous, X(r, k) = x[r * ld + k] (t = 0: rows of a
// Linear's input or weight), or K-strided, X(r, k) = x[k * ld + r] (t = 1: the weight under dx, both operands under dw).
struct MatParams {
  const void* a;
  int64_t lda;
  const void* b;
  int64_t ldb;
  const float* a_scale; // [M] or null
  const float* b_scale; // [N] or null
  const void* bias;     // [N] or null, in the output's type or fp32
  int32_t bias_f32;
  int32_t act;
  float slope;
  int32_t splits;       // > 1: the reduction in that many parts, fp32 partial sums part[split][M][N] instead of an epilogue
  float* part;
  const void* res;      // [M, N] row stride ldr, or null
  int64_t ldr;
  void* z;              // [M, N] contiguous, or null: what the backward keeps (fp32: z; 16 bits: gate codes, mlp_common.h)
  void* y;              // [M, N] contiguous
  int64_t M, N, K;
};

// What the backward keeps, the activation, the residual r and the store of the channels n .. n + CNT - 1 of row m (v: the
// scaled sums with their bias)
template <class O, int CNT>
__device__ __forceinline__ void mat_finish(const MatParams& P, int64_t m, int n, float (&v)[CNT], const float (&r)[CNT]) {
  constexpr bool EXACT = sizeof(O) == 4;
  const int N = static_cast<int>(P.N);
  const int64_t at = m * P.N;
  if constexpr (EXACT) {
    if (P.z) store_run<O, CNT>(static_cast<O*>(P.z) + at, n, N, v);
    act_run<EXACT, CNT>(v, P.act, P.slope);
  } else if (P.z) {
    uint32_t c[CNT];
    act_gate_run<CNT>(v, c, P.act, P.slope);
    store_gates<CNT>(static_cast<uint16_t*>(P.z) + at, n, N, c);
  } else {
    act_run<EXACT, CNT>(v, P.act, P.slope);
  }
#pragma unroll
  for (int e = 0; e < CNT; ++e) v[e] += r[e];
  store_run<O, CNT>(static_cast<O*>(P.y) + at, n, N, v);
}

template <class O, int CNT>
__device__ __forceinline__ void mat_residual(const MatParams& P, int64_t m, int n, float (&r)[CNT]) {
  if (P.res) {
    load_run<O, CNT>(static_cast<const O*>(P.res) + m * P.ldr, n, static_cast<int>(P.N), r);
  } else {
#pragma unroll
    for (int e = 0; e < CNT; ++e) r[e] = 0.f;
  }
}

// all of an epilogue for one run of channels
template <class O, int CNT>
__device__ __forceinline__ void mat_epilogue(const MatParams& P, int64_t m, int64_t n, float (&v)[CNT]) {
  float r[CNT];
  mat_residual<O, CNT>(P, m, static_cast<int>(n), r);
  if (P.bias) {
    float b[CNT];
    load_param_run<O, CNT>(P.bias, P.bias_f32, static_cast<int>(n), static_cast<int>(P.N), b);
#pragma unroll
    for (int e = 0; e < CNT; ++e) v[e] += b[e];
  }
  mat_finish<O, CNT>(P, m, static_cast<int>(n), v, r);
}

// The tiled product (linear_tile_*.hip), by operand type; the operands' rows (k-rows) start on dwords.
// tile: 0 = 256 x 256, 1 = 128 x 128, 2 = 64 x 128 (K-contiguous A only)
int mat_tile_f32(const MatParams& P, int ta, int tb, int tile, hipStream_t s);
int mat_tile_bf16(const MatParams& P, int ta, int tb, int tile, hipStream_t s);
int mat_tile_f16(const MatParams& P, int ta, int tb, int tile, hipStream_t s);
int mat_tile_e4m3(const MatParams& P, int out_type, int tile, hipStream_t s);

// The product of a few K-contiguous rows, at most 32 (linear_small.h): operands at any byte
int mat_small_f32(const MatParams& P, hipStream_t s);
int mat_small_bf16(const MatParams& P, hipStream_t s);
int mat_small_f16(const MatParams& P, hipStream_t s);
int mat_small_e4m3(const MatParams& P, int out_type, hipStream_t s);

}  // namespace dgcn
