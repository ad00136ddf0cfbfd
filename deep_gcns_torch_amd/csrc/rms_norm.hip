// Root-mean-square norm over node rows, with the residual's addition in front and, for a layer in 8 bits, the rounding
// to e4m3 rows behind it; its backward; and the rounding alone.
//
//   h = x [+ r]      y = h * rstd * w      rstd = (mean(h^2) + eps)^(-1/2)
//   gx = gr = rstd * (w g - xh * mean(w g xh)) + g_h      gw = sum over rows of g xh      xh = h * rstd
//   e4m3: scale = max|y| / 448 over the row's finite values (1 where there is none but zeros), q = e4m3(y / scale)
//
// What bounds it: HBM.  A row is read once into registers (eight elements a chunk, NV chunks a lane, one to sixteen
// waves or a part of a wave a row), the sum of squares is joined by shuffles (and LDS between waves), and everything
// that depends on the row is written from the same registers.  The statistics use the fp32 sum x + r, of which h is the
// rounding to the rows' type; the backward adds x and r again (the stored h instead is one row less to read and to keep,
// 16,384 x 4096 bf16 114 us against 145, but half a step of it is off in every term of the weight's gradient: bf16 2.3e-3 of its
// norm against 1.7e-3 that its own rounding costs).  The weight's gradient stays in registers over all rows of a workgroup and leaves as one
// partial per workgroup, summed in a fixed order by a second launch: no atomics, the same bits every time.
//
// Measured (a copy of 1 GiB reaches 5.1 TB/s; what fits the 256 MB of memory-side cache goes faster): 16,384 x 4096 bf16 with
// residual 84 us forward (6.4 TB/s over x, r, h, y) and 145 us backward (4.6 over g, g_h, x, r, gx); 169,343 x 128 fp32 28 and
// 48 us (6.2 and 5.5); to e4m3 rows 8192 x 8192 bf16 with residual 116 us (4.0), the rounding alone of 8192 x 16,384 95 us (4.2).

#include "mlp_common.h"

namespace dgcn {
namespace {

constexpr float kE4m3Inv = 1.f / 448.f;      // max|y| times this, as torch divides by a number on the device: the same bits
constexpr int kRmsMaxC = 32768;

struct RmsParams {
  const void* x;
  int64_t ldx;
  const void* res;
  int64_t ldr;
  const void* w;      // [C] or null
  int32_t w_f32;
  int32_t C;
  float eps;
  int64_t rows;
  void* y;            // [rows, C] contiguous
  void* h;            // [rows, C] contiguous or null
  uint8_t* q;         // e4m3 [rows, C] contiguous
  float* scale;       // [rows]
  float* rstd;        // [rows] or null
};

template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 1; o < (LPR < kWave ? LPR : kWave); o <<= 1) v += __shfl_xor(v, o);
  if constexpr (LPR > kWave) {
    if (lane_id() == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < LPR / kWave; ++i) v += red[i];
  }
  return v;
}

template <int LPR>
__device__ __forceinline__ float row_max(float v, float* red) {
#pragma unroll
  for (int o = 1; o < (LPR < kWave ? LPR : kWave); o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  if constexpr (LPR > kWave) {
    if (lane_id() == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < LPR / kWave; ++i) v = fmaxf(v, red[i]);
  }
  return v;
}

// LPR lanes a row (a workgroup of 256 holds 256 / LPR rows; LPR > 64: one row a workgroup of LPR), NV chunks of eight a lane
template <class T, int LPR, int NV, bool NORM, bool Q8>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void rms_fwd_kernel(const RmsParams P) {
  constexpr int THREADS = LPR > 256 ? LPR : 256;
  constexpr int RPB = THREADS / LPR;
  __shared__ float red[2][2][16];              // [sum | max][row parity]: a slot is written again two rows later
  const int lane = threadIdx.x % LPR;
  const int C = P.C;
  const T* X = static_cast<const T*>(P.x);
  const T* R = static_cast<const T*>(P.res);
  int par = 0;
  // the loop is uniform over a workgroup where it holds barriers (one row a workgroup)
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / LPR; row < P.rows;
       row += static_cast<int64_t>(gridDim.x) * RPB, par ^= 1) {
    float v[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (lane + i * LPR) * 8;
      if (at < C) {
        load_chunk(X + row * P.ldx, at, C, v[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
      }
    }
    if (NORM && R) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = (lane + i * LPR) * 8;
        if (at < C) {
          float r[8];
          load_chunk(R + row * P.ldr, at, C, r);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] += r[e];
        }
      }
    }
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[i][e], v[i][e], ss);
      }
      ss = row_sum<LPR>(ss, red[0][par]);
      const float rstd = 1.f / sqrtf(ss / static_cast<float>(C) + P.eps);
      if (P.rstd && lane == 0) P.rstd[row] = rstd;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = (lane + i * LPR) * 8;
        if (at < C) {
          if (P.h) store_chunk(static_cast<T*>(P.h) + row * C, at, C, v[i]);
          float w[8];
          load_param_chunk<T>(P.w, P.w_f32, at, C, w, 1.f);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * rstd * w[e];
          if constexpr (!Q8) store_chunk(static_cast<T*>(P.y) + row * C, at, C, v[i]);
        }
      }
    }
    if constexpr (Q8) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = fabsf(v[i][e]);
          top = fmaxf(top, a < __builtin_inff() ? a : 0.f);
        }
      }
      top = row_max<LPR>(top, red[1][par]);
      const float scale = top > 0.f ? fmaxf(top * kE4m3Inv, 1.17549435e-38f) : 1.f;
      if (lane == 0) P.scale[row] = scale;
      // The quotient to its last bit, so that a value between two e4m3 numbers goes where y / scale goes: the product with the
      // rounded reciprocal, and its remainder's part once more (y / scale itself is some ten instructions a value: 8192 x 16,384
      // bf16 107 us).  Small scales are lifted first, by a power of two, so that no remainder underflows.
      const float lift = scale < 0x1p-64f ? 0x1p64f : 1.f, by = scale * lift, inv = 1.f / by;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = (lane + i * LPR) * 8;
        if (at < C) {
          float t[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = v[i][e] * lift, b = a * inv, r = fmaf(-b, by, a);
            t[e] = fabsf(v[i][e]) < __builtin_inff() ? fmaf(r, inv, b) : __builtin_nanf("");
          }
          const u2v b = {pack_e4m3(t[0], t[1], t[2], t[3]), pack_e4m3(t[4], t[5], t[6], t[7])};
          uint8_t* q = P.q + row * C + at;
          if (at + 8 <= C) {
            *reinterpret_cast<u2v_any1*>(q) = b;
          } else {
            for (int e = 0; at + e < C; ++e) q[e] = static_cast<uint8_t>(b[e >> 2] >> (8 * (e & 3)));
          }
        }
      }
    }
  }
}

struct RmsBwdParams {
  const void* g;      // gradient of y, or null
  int64_t ldg;
  const void* gh;     // gradient of h, or null
  int64_t ldgh;
  const void* x;
  int64_t ldx;
  const void* res;    // h = x + res in fp32, or null: h = x
  int64_t ldr;
  const void* w;
  int32_t w_f32;
  int32_t C;
  const float* rstd;
  int64_t rows;
  void* dx;           // [rows, C] contiguous or null
  float* dw_part;     // [gridDim.x][C] or null
};

template <class T, int LPR, int NV>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void rms_bwd_kernel(const RmsBwdParams P) {
  constexpr int THREADS = LPR > 256 ? LPR : 256;
  constexpr int RPB = THREADS / LPR;
  __shared__ float red[2][16];
  __shared__ float dws[LPR < 256 ? THREADS * 8 * NV : 1];
  const int lane = threadIdx.x % LPR;
  const int C = P.C;
  float dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  }
  int par = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / LPR; row < P.rows;
       row += static_cast<int64_t>(gridDim.x) * RPB, par ^= 1) {
    float g[NV][8], h[NV][8];
    const float rstd = P.rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (lane + i * LPR) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) { g[i][e] = 0.f; h[i][e] = 0.f; }
      if (at < C) {
        load_chunk(static_cast<const T*>(P.x) + row * P.ldx, at, C, h[i]);
        load_chunk(static_cast<const T*>(P.g) + row * P.ldg, at, C, g[i]);
      }
    }
    if (P.res) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = (lane + i * LPR) * 8;
        if (at < C) {
          float r[8];
          load_chunk(static_cast<const T*>(P.res) + row * P.ldr, at, C, r);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[i][e] += r[e];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (lane + i * LPR) * 8;
      if (at < C) {
        float w[8];
        load_param_chunk<T>(P.w, P.w_f32, at, C, w, 1.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          h[i][e] *= rstd;
          dw[i][e] = fmaf(g[i][e], h[i][e], dw[i][e]);
          g[i][e] *= w[e];
          dot = fmaf(g[i][e], h[i][e], dot);
        }
      }
    }
    if (!P.dx) continue;                     // (uniform)
    dot = row_sum<LPR>(dot, red[par]) / static_cast<float>(C);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (lane + i * LPR) * 8;
      if (at < C) {
        float d[8], gh[8];
        if (P.gh) {
          load_chunk(static_cast<const T*>(P.gh) + row * P.ldgh, at, C, gh);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) gh[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = fmaf(rstd, g[i][e] - h[i][e] * dot, gh[e]);
        store_chunk(static_cast<T*>(P.dx) + row * C, at, C, d);
      }
    }
  }
  if (!P.dw_part) return;
  float* out = P.dw_part + static_cast<int64_t>(blockIdx.x) * C;
  if constexpr (LPR >= 256) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (lane + i * LPR) * 8;
      if (at < C) store_chunk(out, at, C, dw[i]);
    }
  } else {
    // the workgroup's row slots meet in LDS, in slot order
    float* mine = dws + (threadIdx.x / LPR) * (LPR * NV * 8);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) mine[(lane + i * LPR) * 8 + e] = dw[i][e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += THREADS) {
      float t = 0.f;
      for (int s = 0; s < RPB; ++s) t += dws[s * (LPR * NV * 8) + c];
      out[c] = t;
    }
  }
}

// out[c] = sum over p of parts[p][c], in the parameter's type: 32 columns a workgroup, 32 segments of the partials, four loads
// under way each (eight segments: 24 us for 2048 x 256)
constexpr int kSumSegs = 32;
template <class O>
__global__ __launch_bounds__(32 * kSumSegs) void param_sum_kernel(const float* __restrict__ parts, int nparts, int64_t width,
                                                                  O* __restrict__ out) {
  __shared__ float red[kSumSegs][32];
  const int c = threadIdx.x & 31, seg = threadIdx.x >> 5;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + c;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (col < width) {
    int p = seg;
    for (; p + 3 * kSumSegs < nparts; p += 4 * kSumSegs) {
#pragma unroll
      for (int u = 0; u < 4; ++u) a[u] += parts[static_cast<int64_t>(p + u * kSumSegs) * width + col];
    }
    for (; p < nparts; p += kSumSegs) a[0] += parts[static_cast<int64_t>(p) * width + col];
  }
  red[seg][c] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  if (seg == 0 && col < width) {
    float t = 0.f;
#pragma unroll
    for (int s = 0; s < kSumSegs; ++s) t += red[s][c];
    out[col] = static_cast<O>(t);
  }
}

// rows a workgroup holds for C channels (the launch tables below use the same split)
inline int rms_rows_per_wg(int C) {
  const int chunks = (C + 7) / 8;
  if (chunks > 128) return 1;
  int lpr = 2;
  while (lpr < 64 && lpr < chunks) lpr <<= 1;
  return 256 / lpr;
}

inline int64_t rms_bwd_grid(int64_t rows, int C) {
  const int64_t wgs = (rows + rms_rows_per_wg(C) - 1) / rms_rows_per_wg(C);
  const int64_t cap = 2 * static_cast<int64_t>(num_cus());
  return wgs < cap ? wgs : cap;
}

template <class T, int LPR, int NV>
struct RmsFwd {
  template <bool NORM, bool Q8>
  static int go(const RmsParams& P, hipStream_t s) {
    constexpr int THREADS = LPR > 256 ? LPR : 256;
    int64_t wgs = (P.rows + THREADS / LPR - 1) / (THREADS / LPR);
    if (wgs > (1 << 20)) wgs = 1 << 20;
    hipLaunchKernelGGL((rms_fwd_kernel<T, LPR, NV, NORM, Q8>), dim3(static_cast<unsigned>(wgs)), dim3(THREADS), 0, s, P);
    return launch_status();
  }
};

template <class T, bool NORM, bool Q8>
int rms_fwd(const RmsParams& P, hipStream_t s) {
  const int chunks = (P.C + 7) / 8;
  if (chunks <= 2) return RmsFwd<T, 2, 1>::template go<NORM, Q8>(P, s);
  if (chunks <= 4) return RmsFwd<T, 4, 1>::template go<NORM, Q8>(P, s);
  if (chunks <= 8) return RmsFwd<T, 8, 1>::template go<NORM, Q8>(P, s);
  if (chunks <= 16) return RmsFwd<T, 16, 1>::template go<NORM, Q8>(P, s);
  if (chunks <= 32) return RmsFwd<T, 32, 1>::template go<NORM, Q8>(P, s);
  if (chunks <= 64) return RmsFwd<T, 64, 1>::template go<NORM, Q8>(P, s);
  if (chunks <= 128) return RmsFwd<T, 64, 2>::template go<NORM, Q8>(P, s);
  if (chunks <= 256) return RmsFwd<T, 256, 1>::template go<NORM, Q8>(P, s);
  if (chunks <= 512) return RmsFwd<T, 512, 1>::template go<NORM, Q8>(P, s);
  // one barrier a row: more waves with less each (8192 x 8192 bf16 98 us against 111); two: the other way (112 against 129);
  // none of a norm, from 8193 channels on: half the waves (8192 x 16,384 94 us; 90 against 102 before values were divided to the
  // last bit)
  if (chunks <= 1024) return Q8 ? RmsFwd<T, 512, 2>::template go<NORM, Q8>(P, s) : RmsFwd<T, 1024, 1>::template go<NORM, Q8>(P, s);
  if (chunks <= 2048) return NORM ? RmsFwd<T, 1024, 2>::template go<NORM, Q8>(P, s) : RmsFwd<T, 512, 4>::template go<NORM, Q8>(P, s);
  return RmsFwd<T, 1024, 4>::template go<NORM, Q8>(P, s);
}

template <class T, int LPR, int NV>
int rms_bwd_go(const RmsBwdParams& P, hipStream_t s) {
  constexpr int THREADS = LPR > 256 ? LPR : 256;
  hipLaunchKernelGGL((rms_bwd_kernel<T, LPR, NV>), dim3(static_cast<unsigned>(rms_bwd_grid(P.rows, P.C))), dim3(THREADS),
                     0, s, P);
  return launch_status();
}

template <class T>
int rms_bwd(const RmsBwdParams& P, hipStream_t s) {
  const int chunks = (P.C + 7) / 8;
  if (chunks <= 2) return rms_bwd_go<T, 2, 1>(P, s);
  if (chunks <= 4) return rms_bwd_go<T, 4, 1>(P, s);
  if (chunks <= 8) return rms_bwd_go<T, 8, 1>(P, s);
  if (chunks <= 16) return rms_bwd_go<T, 16, 1>(P, s);
  if (chunks <= 32) return rms_bwd_go<T, 32, 1>(P, s);
  if (chunks <= 64) return rms_bwd_go<T, 64, 1>(P, s);
  if (chunks <= 128) return rms_bwd_go<T, 64, 2>(P, s);
  if (chunks <= 256) return rms_bwd_go<T, 256, 1>(P, s);
  if (chunks <= 512) return rms_bwd_go<T, 512, 1>(P, s);
  if (chunks <= 1024) return rms_bwd_go<T, 512, 2>(P, s);
  if (chunks <= 2048) return rms_bwd_go<T, 1024, 2>(P, s);
  return rms_bwd_go<T, 1024, 4>(P, s);
}

}  // namespace
}  // namespace dgcn

using namespace dgcn;

extern "C" int dgcn_rms_norm_fwd(const void* x, int64_t ldx, const void* res, int64_t ldr, const void* w, int32_t w_f32,
                                 float eps, int32_t dtype, void* y, void* h, uint8_t* q, float* scale, float* rstd,
                                 int64_t rows, int32_t C, void* stream) {
  if (!x || (!y && !q) || (q && !scale)) return DGCN_E_NULL;
  if (y && q) return DGCN_E_MODE;
  if (rows < 0 || C < 1 || C > kRmsMaxC || ldx < 0 || (res && ldr < 0)) return DGCN_E_SHAPE;
  if (rows == 0) return DGCN_OK;
  const RmsParams P = {x, ldx, res, ldr, w, w_f32, C, eps, rows, y, h, q, scale, rstd};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case DGCN_T_F32: return q ? rms_fwd<float, true, true>(P, s) : rms_fwd<float, true, false>(P, s);
    case DGCN_T_BF16: return q ? rms_fwd<__bf16, true, true>(P, s) : rms_fwd<__bf16, true, false>(P, s);
    case DGCN_T_F16: return q ? rms_fwd<_Float16, true, true>(P, s) : rms_fwd<_Float16, true, false>(P, s);
    default: return DGCN_E_MODE;
  }
}

extern "C" int dgcn_quantize_rows_e4m3(const void* x, int64_t ldx, int32_t dtype, uint8_t* q, float* scale, int64_t rows,
                                       int32_t C, void* stream) {
  if (!x || !q || !scale) return DGCN_E_NULL;
  if (rows < 0 || C < 1 || C > kRmsMaxC || ldx < 0) return DGCN_E_SHAPE;
  if (rows == 0) return DGCN_OK;
  const RmsParams P = {x, ldx, nullptr, 0, nullptr, 0, C, 0.f, rows, nullptr, nullptr, q, scale, nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case DGCN_T_F32: return rms_fwd<float, false, true>(P, s);
    case DGCN_T_BF16: return rms_fwd<__bf16, false, true>(P, s);
    case DGCN_T_F16: return rms_fwd<_Float16, false, true>(P, s);
    default: return DGCN_E_MODE;
  }
}

extern "C" int32_t dgcn_rms_norm_num_partials(int64_t rows, int32_t C) {
  if (rows <= 0 || C < 1 || C > kRmsMaxC) return 0;
  return static_cast<int32_t>(rms_bwd_grid(rows, C));
}

extern "C" int dgcn_param_sum(const float* parts, int32_t nparts, int64_t width, int32_t dtype, void* out, void* stream) {
  if (!out || (!parts && nparts > 0)) return DGCN_E_NULL;
  if (nparts < 0 || width < 0) return DGCN_E_SHAPE;
  if (width == 0) return DGCN_OK;
  const dim3 grid(static_cast<unsigned>((width + 31) / 32));
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case DGCN_T_F32: hipLaunchKernelGGL(param_sum_kernel<float>, grid, dim3(32 * kSumSegs), 0, s, parts, nparts, width, static_cast<float*>(out)); break;
    case DGCN_T_BF16: hipLaunchKernelGGL(param_sum_kernel<__bf16>, grid, dim3(32 * kSumSegs), 0, s, parts, nparts, width, static_cast<__bf16*>(out)); break;
    case DGCN_T_F16: hipLaunchKernelGGL(param_sum_kernel<_Float16>, grid, dim3(32 * kSumSegs), 0, s, parts, nparts, width, static_cast<_Float16*>(out)); break;
    default: return DGCN_E_MODE;
  }
  return launch_status();
}

extern "C" int dgcn_rms_norm_sum_bwd(const void* g, int64_t ldg, const void* gh, int64_t ldgh, const void* x, int64_t ldx,
                                     const void* res, int64_t ldr, const void* w, int32_t w_f32, const float* rstd,
                                     int32_t dtype, void* dx, void* dw, float* dw_part, int64_t rows, int32_t C, void* stream) {
  if (!g || !x || !rstd || (!dx && !dw) || (dw && !dw_part)) return DGCN_E_NULL;
  if (rows < 1 || C < 1 || C > kRmsMaxC || ldg < 0 || ldx < 0 || (gh && ldgh < 0) || (res && ldr < 0)) return DGCN_E_SHAPE;
  const RmsBwdParams P = {g, ldg, gh, ldgh, x, ldx, res, ldr, w, w_f32, C, rstd, rows, dx, dw ? dw_part : nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  int rc = DGCN_E_MODE;
  switch (dtype) {
    case DGCN_T_F32: rc = rms_bwd<float>(P, s); break;
    case DGCN_T_BF16: rc = rms_bwd<__bf16>(P, s); break;
    case DGCN_T_F16: rc = rms_bwd<_Float16>(P, s); break;
    default: break;
  }
  if (rc != DGCN_OK || !dw) return rc;
  return dgcn_param_sum(dw_part, static_cast<int32_t>(rms_bwd_grid(rows, C)), C, w_f32 ? DGCN_T_F32 : dtype, dw, stream);
}

extern "C" int dgcn_rms_norm_bwd(const void* g, int64_t ldg, const void* gh, int64_t ldgh, const void* h, int64_t ldh,
                                 const void* w, int32_t w_f32, const float* rstd, int32_t dtype, void* dx, void* dw,
                                 float* dw_part, int64_t rows, int32_t C, void* stream) {
  return dgcn_rms_norm_sum_bwd(g, ldg, gh, ldgh, h, ldh, nullptr, 0, w, w_f32, rstd, dtype, dx, dw, dw_part, rows, C, stream);
}
