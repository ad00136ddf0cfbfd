// The product of node rows with a weight, with the bias, the activation and the residual in its epilogue, in 32, 16 and
// 8 bits, and the products of its backward.
//
//   z = s_x s_w (x w^T) + b        y = act(z) + r              (s_x, s_w: the scales of e4m3 rows, else 1)
//   dz = g act'(z)     gb = sum over rows of dz     gx = dz w     gw = dz^T x     gr = g
//
// Every sum is held in fp32.  z is kept for the backward rounded to the rows' type (half a step of z in act'(z)), and dz
// is rounded to it before the two products, which take the rows' type on the matrix pipe.

#include "mlp_common.h"

namespace dgcn {
namespace {

struct MatParams {
  const void* a;        // A(m, k) at a + m * am + k * ak
  int64_t am, ak;
  const void* b;        // B(n, k) at b + n * bn + k * bk
  int64_t bn, bk;
  const float* a_scale; // [M] or null
  const float* b_scale; // [N] or null
  const void* bias;     // [N] or null, in the output's type or fp32
  int32_t bias_f32;
  int32_t act;
  float slope;
  const void* res;      // [M, N] row stride ldr, or null
  int64_t ldr;
  void* z;              // [M, N] contiguous, or null
  void* y;              // [M, N] contiguous
  int64_t M, N, K;
};

__device__ __forceinline__ float elem(const uint8_t* p, int64_t i) {
  return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(p[i]), 0);
}
template <class T>
__device__ __forceinline__ float elem(const T* p, int64_t i) { return static_cast<float>(p[i]); }

// The plain form of all three products: 64 x 64 tiles, fp32 operands in LDS, 4 x 4 sums a thread.
template <class T, class O>
__global__ __launch_bounds__(256) void mat_simple_kernel(const MatParams P) {
  constexpr int BM = 64, BN = 64, BK = 16;
  __shared__ float As[BK][BM + 4], Bs[BK][BN + 4];
  const T* A = static_cast<const T*>(P.a);
  const T* B = static_cast<const T*>(P.b);
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * BM, n0 = static_cast<int64_t>(blockIdx.y) * BN;
  const int tm = threadIdx.x & 15, tn = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < P.K; k0 += BK) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int idx = threadIdx.x + i * 256;
      // consecutive threads along the axis that is contiguous
      const int ka = P.ak == 1 ? idx % BK : idx / BM, ma = P.ak == 1 ? idx / BK : idx % BM;
      const int kb = P.bk == 1 ? idx % BK : idx / BN, nb = P.bk == 1 ? idx / BK : idx % BN;
      As[ka][ma] = (m0 + ma < P.M && k0 + ka < P.K) ? elem(A, (m0 + ma) * P.am + (k0 + ka) * P.ak) : 0.f;
      Bs[kb][nb] = (n0 + nb < P.N && k0 + kb < P.K) ? elem(B, (n0 + nb) * P.bn + (k0 + kb) * P.bk) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BK; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { a[i] = As[k][tm * 4 + i]; b[i] = Bs[k][tn * 4 + i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + tm * 4 + i;
    if (m >= P.M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tn * 4 + j;
      if (n >= P.N) continue;
      float z = acc[i][j];
      if (P.a_scale) z *= P.a_scale[m];
      if (P.b_scale) z *= P.b_scale[n];
      if (P.bias) z += load_param<O>(P.bias, P.bias_f32, n);
      if (P.z) static_cast<O*>(P.z)[m * P.N + n] = static_cast<O>(z);
      float y = act_fwd<sizeof(O) == 4>(z, P.act, P.slope);
      if (P.res) y += static_cast<float>(static_cast<const O*>(P.res)[m * P.ldr + n]);
      static_cast<O*>(P.y)[m * P.N + n] = static_cast<O>(y);
    }
  }
}

template <class T, class O>
int mat_launch(const MatParams& P, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((P.M + 63) / 64), static_cast<unsigned>((P.N + 63) / 64));
  hipLaunchKernelGGL((mat_simple_kernel<T, O>), grid, dim3(256), 0, s, P);
  return launch_status();
}

int mat_same(const MatParams& P, int dtype, hipStream_t s) {
  switch (dtype) {
    case DGCN_T_F32: return mat_launch<float, float>(P, s);
    case DGCN_T_BF16: return mat_launch<__bf16, __bf16>(P, s);
    case DGCN_T_F16: return mat_launch<_Float16, _Float16>(P, s);
    default: return DGCN_E_MODE;
  }
}

// dz = g act'(z), and the column sums of dz over a slab of rows: CL lanes (eight channels each) across, 256 / CL rows at
// a time; a workgroup takes the rows blockIdx.y * slab .. and leaves one partial sum per channel
template <class T>
__global__ __launch_bounds__(256) void gate_kernel(const T* __restrict__ g, int64_t ldg, const T* __restrict__ z, int act,
                                                   float slope, T* __restrict__ dz, float* __restrict__ part,
                                                   int64_t rows, int N, int cl, int64_t slab) {
  __shared__ float red[256 * 8];
  const int lane = threadIdx.x % cl, slot = threadIdx.x / cl, slots = 256 / cl;
  const int at = (blockIdx.x * cl + lane) * 8;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * slab;
  const int64_t r1 = r0 + slab < rows ? r0 + slab : rows;
  float sum[8] = {};
  if (at < N) {
    for (int64_t r = r0 + slot; r < r1; r += slots) {
      float d[8];
      load_chunk(g + r * ldg, at, N, d);
      if (act != DGCN_ACT_NONE) {
        float zz[8];
        load_chunk(z + r * N, at, N, zz);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] *= act_slope<sizeof(T) == 4>(zz[e], act, slope);
        store_chunk(dz + r * N, at, N, d);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += d[e];
    }
  }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[(slot * cl + lane) * 8 + e] = sum[e];
  __syncthreads();
  for (int c = threadIdx.x; c < cl * 8; c += 256) {
    const int64_t col = static_cast<int64_t>(blockIdx.x) * cl * 8 + c;
    if (col < N) {
      float t = 0.f;
      for (int sl = 0; sl < slots; ++sl) t += red[sl * cl * 8 + c];
      part[static_cast<int64_t>(blockIdx.y) * N + col] = t;
    }
  }
}

struct GateShape {
  int cl;
  unsigned gx, gy;
  int64_t slab;
};

inline GateShape gate_shape(int64_t rows, int N) {
  GateShape S;
  const int chunks = (N + 7) / 8;
  S.cl = 1;
  while (S.cl < 64 && S.cl < chunks) S.cl <<= 1;
  S.gx = static_cast<unsigned>((chunks + S.cl - 1) / S.cl);
  // about eight workgroups a CU, at least 8 row steps each
  int64_t want = 8 * static_cast<int64_t>(num_cus()) / S.gx;
  const int64_t step = 256 / S.cl, most = (rows + 8 * step - 1) / (8 * step);
  if (want > most) want = most;
  if (want < 1) want = 1;
  S.slab = (rows + want - 1) / want;
  S.gy = static_cast<unsigned>((rows + S.slab - 1) / S.slab);
  return S;
}

inline bool known_act(int act) { return act >= DGCN_ACT_NONE && act <= DGCN_ACT_SILU; }
inline bool sizes_ok(int64_t rows, int32_t K, int32_t N) {
  return rows >= 0 && rows < (int64_t{1} << 36) && K >= 1 && N >= 1 && K <= (1 << 20) && N <= (1 << 20);
}

}  // namespace
}  // namespace dgcn

using namespace dgcn;

extern "C" int dgcn_linear_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const float* x_scale,
                               const float* w_scale, const void* bias, int32_t bias_f32, const void* res, int64_t ldr,
                               int32_t act, float slope, int32_t in_type, int32_t out_type, void* z, void* y, int64_t rows,
                               int32_t K, int32_t N, void* stream) {
  if (!x || !w || !y || (in_type == DGCN_T_E4M3 && (!x_scale || !w_scale))) return DGCN_E_NULL;
  if (!sizes_ok(rows, K, N) || ldx < 0 || ldw < 0 || (res && ldr < 0)) return DGCN_E_SHAPE;
  if (!known_act(act) || (in_type != DGCN_T_E4M3 && in_type != out_type)) return DGCN_E_MODE;
  if (rows == 0) return DGCN_OK;
  MatParams P = {x, ldx, 1, w, ldw, 1, x_scale, w_scale, bias, bias_f32, act, slope, res, ldr, z, y, rows, N, K};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (in_type != DGCN_T_E4M3) {
    P.a_scale = P.b_scale = nullptr;
    return mat_same(P, in_type, s);
  }
  switch (out_type) {
    case DGCN_T_F32: return mat_launch<uint8_t, float>(P, s);
    case DGCN_T_BF16: return mat_launch<uint8_t, __bf16>(P, s);
    case DGCN_T_F16: return mat_launch<uint8_t, _Float16>(P, s);
    default: return DGCN_E_MODE;
  }
}

extern "C" int32_t dgcn_linear_gate_num_partials(int64_t rows, int32_t N) {
  if (rows <= 0 || N < 1) return 0;
  return static_cast<int32_t>(gate_shape(rows, N).gy);
}

extern "C" int dgcn_linear_gate(const void* g, int64_t ldg, const void* z, int32_t act, float slope, int32_t dtype,
                                void* dz, float* db_part, int64_t rows, int32_t N, void* stream) {
  if (!g || (act != DGCN_ACT_NONE && (!z || !dz))) return DGCN_E_NULL;
  if (!sizes_ok(rows, 1, N) || ldg < 0) return DGCN_E_SHAPE;
  if (!known_act(act)) return DGCN_E_MODE;
  if (rows == 0) return DGCN_OK;
  const GateShape S = gate_shape(rows, N);
  const dim3 grid(S.gx, S.gy);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case DGCN_T_F32:
      hipLaunchKernelGGL(gate_kernel<float>, grid, dim3(256), 0, s, static_cast<const float*>(g), ldg,
                         static_cast<const float*>(z), act, slope, static_cast<float*>(dz), db_part, rows, N, S.cl, S.slab);
      break;
    case DGCN_T_BF16:
      hipLaunchKernelGGL(gate_kernel<__bf16>, grid, dim3(256), 0, s, static_cast<const __bf16*>(g), ldg,
                         static_cast<const __bf16*>(z), act, slope, static_cast<__bf16*>(dz), db_part, rows, N, S.cl, S.slab);
      break;
    case DGCN_T_F16:
      hipLaunchKernelGGL(gate_kernel<_Float16>, grid, dim3(256), 0, s, static_cast<const _Float16*>(g), ldg,
                         static_cast<const _Float16*>(z), act, slope, static_cast<_Float16*>(dz), db_part, rows, N, S.cl, S.slab);
      break;
    default: return DGCN_E_MODE;
  }
  return launch_status();
}

extern "C" int dgcn_linear_dx(const void* dz, int64_t lddz, const void* w, int64_t ldw, int32_t dtype, void* dx,
                              int64_t rows, int32_t K, int32_t N, void* stream) {
  if (!dz || !w || !dx) return DGCN_E_NULL;
  if (!sizes_ok(rows, K, N) || lddz < 0 || ldw < 0) return DGCN_E_SHAPE;
  if (rows == 0) return DGCN_OK;
  const MatParams P = {dz, lddz, 1, w, 1, ldw, nullptr, nullptr, nullptr, 0, DGCN_ACT_NONE, 0.f, nullptr, 0, nullptr, dx, rows, K, N};
  return mat_same(P, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int dgcn_linear_dw(const void* dz, int64_t lddz, const void* x, int64_t ldx, int32_t dtype, void* dw,
                              int64_t rows, int32_t K, int32_t N, void* stream) {
  if (!dz || !x || !dw) return DGCN_E_NULL;
  if (!sizes_ok(rows, K, N) || lddz < 0 || ldx < 0) return DGCN_E_SHAPE;
  const MatParams P = {dz, 1, lddz, x, 1, ldx, nullptr, nullptr, nullptr, 0, DGCN_ACT_NONE, 0.f, nullptr, 0, nullptr, dw, N, K, rows};
  return mat_same(P, dtype, static_cast<hipStream_t>(stream));
}
