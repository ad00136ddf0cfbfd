// The product of node rows with a weight, with the bias, the activation and the residual in its epilogue, in 32, 16 and
// 8 bits, and the products of its backward.
//
//   z = s_x s_w (x w^T) + b        y = act(z) + r              (s_x, s_w: the scales of e4m3 rows, else 1)
//   dz = g act'(z)     gb = sum over rows of dz     gx = dz w     gw = dz^T x     gr = g
//
// Every sum is held in fp32.  For the backward the forward keeps z in fp32, or act'(z) in 16-bit fixed point where the rows
// have 16 bits (mlp_common.h); dz is rounded to the rows' type before the two products, which take that on the matrix pipe.

#include "linear_act.h"

namespace dgcn {
namespace {

// the epilogue of a product whose reduction was split: the partial sums are added in split order
template <class O>
__global__ __launch_bounds__(256) void split_join_kernel(const MatParams P) {
  const int64_t per = (P.N + 3) / 4, total = P.M * per;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; it < total; it += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t m = it / per, n = (it - m * per) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const float* p = P.part + m * P.N + n;
    for (int s = 0; s < P.splits; ++s, p += P.M * P.N) {
      float t[4];
      if (n + 4 <= P.N) {
        load4(p, t);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = n + j < P.N ? p[j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += t[j];
    }
    mat_epilogue<O, 4>(P, m, n, v);
  }
}

struct MatPlan {
  int tile;
  int splits;
};

// Tile and split by the cost of the alternatives, in cycles of a CU: a workgroup's step takes what its matrix instructions and LDS
// traffic take (`work`, times the workgroups a CU holds), and at least the latency of the copies behind it; a split
// writes and reads fp32 partial sums and launches once more.
inline MatPlan mat_plan(int64_t M, int64_t N, int64_t K, int type, int ta) {
  struct { int bm, bn, held; double work; } tiles[3] = {{256, 256, 1, 3000.}, {128, 128, 2, 900.}, {64, 128, 3, 600.}};
  const int64_t bk = type == DGCN_T_E4M3 ? 128 : type == DGCN_T_F32 ? 32 : 64, steps = (K + bk - 1) / bk;
  const double cus = num_cus();
  MatPlan best = {0, 1};
  double least = 1e300;
  for (int t = 0; t < (ta ? 2 : 3); ++t) {
    const double wgs1 = static_cast<double>((M + tiles[t].bm - 1) / tiles[t].bm) * ((N + tiles[t].bn - 1) / tiles[t].bn);
    for (int sp = 1; sp <= 512 && sp <= steps; sp *= 2) {
      const double wgs = wgs1 * sp, per_cu = ceil(wgs / cus);
      const double held = per_cu < tiles[t].held ? per_cu : tiles[t].held;
      const double step = held * tiles[t].work > 2000. ? held * tiles[t].work : 2000.;
      double c = ceil(per_cu / tiles[t].held) * ((steps + sp - 1) / sp * step + 4000.);
      if (sp > 1) c += 8. * M * N * sp / 2000. + 10000.;
      if (c < least) { least = c; best = {t, sp}; }
    }
  }
  return best;
}

inline size_t plan_bytes(const MatPlan& p, int64_t M, int64_t N) {
  return p.splits > 1 ? static_cast<size_t>(p.splits) * M * N * sizeof(float) : 0;
}

template <class O>
int split_join(const MatParams& P, hipStream_t s) {
  int64_t wgs = (P.M * ((P.N + 3) / 4) + 255) / 256;
  if (wgs > 16 * num_cus()) wgs = 16 * num_cus();
  hipLaunchKernelGGL((split_join_kernel<O>), dim3(static_cast<unsigned>(wgs)), dim3(256), 0, s, P);
  return launch_status();
}

inline bool aligned16(const void* p, int64_t ld, int es) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * es % 16 == 0; }

int mat_run(MatParams P, int ta, int tb, int in_type, int out_type, void* ws, size_t ws_bytes, hipStream_t s) {
  if (ta == 0 && tb == 0 && P.M <= kSmallRows) {
    switch (in_type) {
      case DGCN_T_F32: return mat_small_f32(P, s);
      case DGCN_T_BF16: return mat_small_bf16(P, s);
      case DGCN_T_F16: return mat_small_f16(P, s);
      default: return mat_small_e4m3(P, out_type, s);
    }
  }
  const MatPlan plan = mat_plan(P.M, P.N, P.K, in_type, ta);
  const int es = in_type == DGCN_T_E4M3 ? 1 : in_type == DGCN_T_F32 ? 4 : 2;
  if (!aligned16(P.a, P.lda, es) || !aligned16(P.b, P.ldb, es)) return DGCN_E_ALIGN;
  if (plan.splits > 1 && (ws_bytes < plan_bytes(plan, P.M, P.N) || !ws)) return DGCN_E_WORKSPACE;
  P.splits = plan.splits;
  P.part = static_cast<float*>(ws);
  int rc = DGCN_E_MODE;
  switch (in_type) {
    case DGCN_T_F32: rc = mat_tile_f32(P, ta, tb, plan.tile, s); break;
    case DGCN_T_BF16: rc = mat_tile_bf16(P, ta, tb, plan.tile, s); break;
    case DGCN_T_F16: rc = mat_tile_f16(P, ta, tb, plan.tile, s); break;
    case DGCN_T_E4M3: rc = mat_tile_e4m3(P, out_type, plan.tile, s); break;
    default: break;
  }
  if (rc != DGCN_OK || plan.splits == 1) return rc;
  switch (out_type) {
    case DGCN_T_F32: return split_join<float>(P, s);
    case DGCN_T_BF16: return split_join<__bf16>(P, s);
    default: return split_join<_Float16>(P, s);
  }
}

// dz = g act'(z), and the column sums of dz over a slab of rows: CL lanes (eight channels each) across, 256 / CL rows at
// a time; a workgroup takes the rows blockIdx.y * slab .. and leaves one partial sum per channel
template <class T>
__global__ __launch_bounds__(256) void gate_kernel(const T* __restrict__ g, int64_t ldg, const void* __restrict__ z, int act,
                                                   float slope, T* __restrict__ dz, int64_t lddz, float* __restrict__ part,
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
      if (dz) {
        if (act != DGCN_ACT_NONE) {
          float sl[8];
          load_slopes<T>(z, r * N, at, N, act, slope, sl);
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] *= sl[e];
        }
        store_chunk(dz + r * lddz, at, static_cast<int>(lddz), d);     // (d is 0 behind N)
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

// rows of C bytes -> rows of ldo bytes (ldo a multiple of 16, less than 16 more than C), zeros behind; 16 bytes a thread
__global__ __launch_bounds__(256) void pad_rows_kernel(const uint8_t* __restrict__ x, int64_t ldx, uint8_t* __restrict__ out,
                                                       int64_t ldo, int64_t rows, int64_t C) {
  typedef u4v u4v_any1 __attribute__((aligned(1)));
  const int64_t per = ldo / 16, total = rows * per;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; it < total; it += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = it / per, at = (it - r * per) * 16;
    const uint8_t* p = x + r * ldx + at;
    u4v v = {0, 0, 0, 0};
    if (at + 16 <= C) {
      v = *reinterpret_cast<const u4v_any1*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (at + e < C) v[e >> 2] |= static_cast<uint32_t>(p[e]) << (8 * (e & 3));
      }
    }
    *reinterpret_cast<u4v*>(out + r * ldo + at) = v;
  }
}

inline bool known_act(int act) { return act >= DGCN_ACT_NONE && act <= DGCN_ACT_SILU; }
inline bool sizes_ok(int64_t rows, int32_t K, int32_t N) {
  return rows >= 0 && rows < (int64_t{1} << 36) && K >= 1 && N >= 1 && K <= (1 << 20) && N <= (1 << 20);
}

}  // namespace
}  // namespace dgcn

using namespace dgcn;

extern "C" int32_t dgcn_linear_small_rows(void) { return kSmallRows; }

extern "C" size_t dgcn_linear_workspace(int32_t product, int64_t rows, int32_t K, int32_t N, int32_t in_type) {
  if (rows <= 0 || K < 1 || N < 1) return 0;
  switch (product) {
    case 0: return rows <= kSmallRows ? 0 : plan_bytes(mat_plan(rows, N, K, in_type, 0), rows, N);
    case 1: return plan_bytes(mat_plan(rows, K, N, in_type, 0), rows, K);
    case 2: return plan_bytes(mat_plan(N, K, rows, in_type, 1), N, K);
    default: return 0;
  }
}

extern "C" int dgcn_linear_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const float* x_scale,
                               const float* w_scale, const void* bias, int32_t bias_f32, const void* res, int64_t ldr,
                               int32_t act, float slope, int32_t in_type, int32_t out_type, void* z, void* y, int64_t rows,
                               int32_t K, int32_t N, void* ws, size_t ws_bytes, void* stream) {
  if (!x || !w || !y || (in_type == DGCN_T_E4M3 && (!x_scale || !w_scale))) return DGCN_E_NULL;
  if (!sizes_ok(rows, K, N) || ldx < 0 || ldw < 0 || (res && ldr < 0)) return DGCN_E_SHAPE;
  if (!known_act(act) || out_type < DGCN_T_F32 || out_type > DGCN_T_F16 || (in_type != DGCN_T_E4M3 && in_type != out_type)) return DGCN_E_MODE;
  if (rows == 0) return DGCN_OK;
  const bool scaled = in_type == DGCN_T_E4M3;
  const MatParams P = {x, ldx, w, ldw, scaled ? x_scale : nullptr, scaled ? w_scale : nullptr, bias, bias_f32, act, slope, 1,
                       nullptr, res, ldr, z, y, rows, N, K};
  return mat_run(P, 0, 0, in_type, out_type, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int32_t dgcn_linear_gate_num_partials(int64_t rows, int32_t N) {
  if (rows <= 0 || N < 1) return 0;
  return static_cast<int32_t>(gate_shape(rows, N).gy);
}

extern "C" int dgcn_linear_gate(const void* g, int64_t ldg, const void* z, int32_t act, float slope, int32_t dtype,
                                void* dz, int64_t lddz, float* db_part, int64_t rows, int32_t N, void* stream) {
  if (!g || (act != DGCN_ACT_NONE && (!z || !dz))) return DGCN_E_NULL;
  if (!sizes_ok(rows, 1, N) || ldg < 0 || (dz && (lddz < N || lddz > (N + 7) / 8 * 8))) return DGCN_E_SHAPE;
  if (!known_act(act)) return DGCN_E_MODE;
  if (rows == 0) return DGCN_OK;
  const GateShape S = gate_shape(rows, N);
  const dim3 grid(S.gx, S.gy);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case DGCN_T_F32:
      hipLaunchKernelGGL(gate_kernel<float>, grid, dim3(256), 0, s, static_cast<const float*>(g), ldg,
                         z, act, slope, static_cast<float*>(dz), lddz, db_part, rows, N, S.cl, S.slab);
      break;
    case DGCN_T_BF16:
      hipLaunchKernelGGL(gate_kernel<__bf16>, grid, dim3(256), 0, s, static_cast<const __bf16*>(g), ldg,
                         z, act, slope, static_cast<__bf16*>(dz), lddz, db_part, rows, N, S.cl, S.slab);
      break;
    case DGCN_T_F16:
      hipLaunchKernelGGL(gate_kernel<_Float16>, grid, dim3(256), 0, s, static_cast<const _Float16*>(g), ldg,
                         z, act, slope, static_cast<_Float16*>(dz), lddz, db_part, rows, N, S.cl, S.slab);
      break;
    default: return DGCN_E_MODE;
  }
  return launch_status();
}

extern "C" int dgcn_linear_dx(const void* dz, int64_t lddz, const void* w, int64_t ldw, int32_t dtype, void* dx,
                              int64_t rows, int32_t K, int32_t N, void* ws, size_t ws_bytes, void* stream) {
  if (!dz || !w || !dx) return DGCN_E_NULL;
  if (!sizes_ok(rows, K, N) || lddz < 0 || ldw < 0) return DGCN_E_SHAPE;
  if (dtype < DGCN_T_F32 || dtype > DGCN_T_F16) return DGCN_E_MODE;
  if (rows == 0) return DGCN_OK;
  const MatParams P = {dz, lddz, w, ldw, nullptr, nullptr, nullptr, 0, DGCN_ACT_NONE, 0.f, 1, nullptr, nullptr, 0, nullptr, dx, rows, K, N};
  return mat_run(P, 0, 1, dtype, dtype, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int dgcn_linear_dw(const void* dz, int64_t lddz, const void* x, int64_t ldx, int32_t dtype, void* dw,
                              int64_t rows, int32_t K, int32_t N, void* ws, size_t ws_bytes, void* stream) {
  if (!dz || !x || !dw) return DGCN_E_NULL;
  if (!sizes_ok(rows, K, N) || rows == 0 || lddz < 0 || ldx < 0) return DGCN_E_SHAPE;
  if (dtype < DGCN_T_F32 || dtype > DGCN_T_F16) return DGCN_E_MODE;
  const MatParams P = {dz, lddz, x, ldx, nullptr, nullptr, nullptr, 0, DGCN_ACT_NONE, 0.f, 1, nullptr, nullptr, 0, nullptr, dw, N, K, rows};
  return mat_run(P, 1, 1, dtype, dtype, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int dgcn_pad_rows(const void* x, int64_t ldx, void* out, int64_t ldo, int64_t rows, int64_t bytes, void* stream) {
  if (!x || !out) return DGCN_E_NULL;
  if (rows < 0 || bytes < 1 || ldx < 0 || ldo != (bytes + 15) / 16 * 16) return DGCN_E_SHAPE;
  if (reinterpret_cast<uintptr_t>(out) & 15) return DGCN_E_ALIGN;
  if (rows == 0) return DGCN_OK;
  int64_t wgs = (rows * (ldo / 16) + 255) / 256;
  if (wgs > 32 * num_cus()) wgs = 32 * num_cus();
  hipLaunchKernelGGL(pad_rows_kernel, dim3(static_cast<unsigned>(wgs)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint8_t*>(x), ldx, static_cast<uint8_t*>(out), ldo, rows, bytes);
  return launch_status();
}
