// The product of node rows with a weight, with the bias, the activation and the residual in its epilogue, in 32, 16 and
// 8 bits, and the products of its backward.
//
//   z = s_x s_w (x w^T) + b        y = act(z) + r              (s_x, s_w: the scales of e4m3 rows, else 1)
//   dz = g act'(z)     gb = sum over rows of dz     gx = dz w     gw = dz^T x     gr = g
//
// Every sum is held in fp32.  For the backward the forward keeps z in fp32, or act'(z) as a 16-bit code where the rows have
// 16 bits (mlp_common.h); dz is rounded to the rows' type before the two products: the matrix pipe takes
// operands of one 16-bit type, and dz in two parts would be twice its work (8192 x 4096 x 16,384 bf16: some 1.8 ms more of 2.95).  The
// rounding costs dx and dw as much as their own (bf16 2.3e-3 of their norms in all, 1.7e-3 without it); where there is no
// activation, or relu, dz has none.  The bias gradient sums dz before it.

#include "linear_act.h"

namespace dgcn {
namespace {

// The epilogue of a product whose reduction was split: four channels an item, 256 / segs items a workgroup; `segs` threads of
// an item add every segs-th partial sum and meet in LDS, in a fixed order.  (One thread an item, which a 256 x 128 result with
// 128 partial sums was until then, took 71 us: 128 loads one behind the other on 32 workgroups.)
template <class O>
__global__ __launch_bounds__(256) void split_join_kernel(const MatParams P, int segs) {
  __shared__ f32x4 red[256];
  const int items = 256 / segs, mine = threadIdx.x % items, seg = threadIdx.x / items;
  const int64_t per = (P.N + 3) / 4, total = P.M * per, it = static_cast<int64_t>(blockIdx.x) * items + mine;
  const int64_t m = it / per, n = (it - m * per) * 4, size = P.M * P.N;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (it < total) {
    const float* p = P.part + m * P.N + n;
    const bool whole = n + 4 <= P.N;
    auto load = [&](int s) {
      float t[4];
      if (whole) {
        load4(p + s * size, t);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = n + j < P.N ? p[s * size + j] : 0.f;
      }
      return f32x4{t[0], t[1], t[2], t[3]};
    };
    int s = seg;
    for (; s + 3 * segs < P.splits; s += 4 * segs) {
      const f32x4 a = load(s), b = load(s + segs), c = load(s + 2 * segs), d = load(s + 3 * segs);
      sum += (a + b) + (c + d);
    }
    for (; s < P.splits; s += segs) sum += load(s);
  }
  red[threadIdx.x] = sum;
  __syncthreads();
  if (seg == 0 && it < total) {
    for (int g = 1; g < segs; ++g) sum += red[g * items + mine];
    float v[4] = {sum[0], sum[1], sum[2], sum[3]};
    mat_epilogue<O, 4>(P, m, n, v);
  }
}

struct MatPlan {
  int tile;
  int splits;
};

// Tile and split by what the alternatives cost, in us.  A CU's workgroups take `work` for each step (128 bytes of the
// reduction) of each of them, and a step takes at least `lag` however few they are; a round of workgroups ends in an epilogue;
// a split writes and reads fp32 partial sums (from the caches: 8 TB/s) and launches once more.  The constants are fits to
// measured times, bf16 and fp16 | e4m3 | fp32: 4096^3 (bf16) takes 117 / 156 / 210 us by tiles of 256 / 128 / 64 rows,
// 1024 x 4096 x 4096 55 (split by four) / 48 / 43, 66,880 x 294 x 192 41 / 30 / 29, 512 x 512 x 40,000 51 / 47 / -- split by 32 / 16.
struct TileCost {
  int bm, bn, held;      // rows, channels, workgroups a CU holds
  double work, lag, end;
};
constexpr TileCost kCost16[3] = {{256, 256, 1, 1.55, 1.55, 8.}, {128, 128, 2, 0.55, 0.65, 4.}, {64, 128, 3, 0.30, 0.50, 3.}};
constexpr TileCost kCost32[3] = {{256, 256, 1, 5.0, 5.0, 12.}, {128, 128, 2, 1.4, 1.6, 5.}, {64, 128, 3, 0.8, 1.0, 4.}};

inline MatPlan mat_plan(int64_t M, int64_t N, int64_t K, int type, int ta) {
  const TileCost* cost = type == DGCN_T_F32 ? kCost32 : kCost16;
  const int64_t bk = type == DGCN_T_E4M3 ? 128 : type == DGCN_T_F32 ? 32 : 64, steps = (K + bk - 1) / bk;
  const double cus = num_cus();
  MatPlan best = {0, 1};
  double least = 1e300;
  for (int t = 0; t < (ta ? 2 : 3); ++t) {
    const double tiles = static_cast<double>((M + cost[t].bm - 1) / cost[t].bm) * ((N + cost[t].bn - 1) / cost[t].bn);
    for (int sp = 1; sp <= 512 && sp <= steps; sp *= 2) {
      const double per_cu = ceil(tiles * sp / cus), rounds = ceil(per_cu / cost[t].held);
      const double each = static_cast<double>((steps + sp - 1) / sp), busy = per_cu * cost[t].work, lag = rounds * cost[t].lag;
      double us = each * (busy > lag ? busy : lag) + rounds * cost[t].end;
      if (sp > 1) us += 3. + 1e-6 * M * N * sp;
      if (us < least) { least = us; best = {t, sp}; }
    }
  }
  return best;
}

template <class O>
int split_join(const MatParams& P, hipStream_t s) {
  const int64_t total = P.M * ((P.N + 3) / 4);
  int segs = 1;
  while (segs < 32 && segs * 4 <= P.splits && total * segs < 128 * static_cast<int64_t>(num_cus())) segs *= 2;
  const int64_t wgs = (total + 256 / segs - 1) / (256 / segs);
  if (wgs > 0x7fffffff) return DGCN_E_SHAPE;
  hipLaunchKernelGGL((split_join_kernel<O>), dim3(static_cast<unsigned>(wgs)), dim3(256), 0, s, P, segs);
  return launch_status();
}

// dz = g act'(z), and the column sums of dz over a slab of rows: CL lanes (eight channels each) across, 256 / CL rows at
// a time; a workgroup takes the rows blockIdx.y * slab .. and leaves one partial sum per channel
// (one slab: the bias gradient itself).  HBM: 8192 x 16,384 bf16
// 167 us, 169,343 x 256 fp32 109 us, both 4.8 TB/s.
template <class T>
__global__ __launch_bounds__(256) void gate_kernel(const T* __restrict__ g, int64_t ldg, const void* __restrict__ z, int act,
                                                   float slope, T* __restrict__ dz, int64_t lddz, float* __restrict__ part,
                                                   void* __restrict__ db, int db_f32, int64_t rows, int N, int cl, int64_t slab) {
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
  if (!db) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[(slot * cl + lane) * 8 + e] = sum[e];
  __syncthreads();
  for (int c = threadIdx.x; c < cl * 8; c += 256) {
    const int64_t col = static_cast<int64_t>(blockIdx.x) * cl * 8 + c;
    if (col < N) {
      float t = 0.f;
      for (int sl = 0; sl < slots; ++sl) t += red[sl * cl * 8 + c];
      if (gridDim.y > 1) {
        part[static_cast<int64_t>(blockIdx.y) * N + col] = t;
      } else if (db_f32) {
        static_cast<float*>(db)[col] = t;
      } else {
        static_cast<T*>(db)[col] = static_cast<T>(t);
      }
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
  // about four workgroups a CU, at least 8 row steps each
  int64_t want = 4 * static_cast<int64_t>(num_cus()) / S.gx;
  const int64_t step = 256 / S.cl, most = (rows + 8 * step - 1) / (8 * step);
  if (want > most) want = most;
  if (want < 1) want = 1;
  S.slab = (rows + want - 1) / want;
  S.gy = static_cast<unsigned>((rows + S.slab - 1) / S.slab);
  return S;
}

// rows of C bytes -> rows of ldo bytes (ldo a multiple of 16, less than 16 more than C), zeros behind; 16 bytes a thread, one
// or two matrices a launch (a launch costs as much as a copy of 2 MB: fp16 1021 x 1013 and 2047 x 1013 take 6 us, in two launches 9)
struct PadJob {
  const uint8_t* x;
  int64_t ldx;
  uint8_t* out;
  int64_t ldo, rows, C;
  unsigned wgs;
};
struct PadJobs {
  PadJob job[2];
  int n;
};

__global__ __launch_bounds__(256) void pad_rows_kernel(const PadJobs jobs) {
  typedef u4v u4v_any1 __attribute__((aligned(1)));
  const bool second = blockIdx.x >= jobs.job[0].wgs;
  const PadJob& J = jobs.job[second];
  const int64_t per = J.ldo / 16, total = J.rows * per;
  for (int64_t it = static_cast<int64_t>(blockIdx.x - (second ? jobs.job[0].wgs : 0)) * 256 + threadIdx.x; it < total; it += static_cast<int64_t>(J.wgs) * 256) {
    // (a 64-bit division is as long as the rest)
    const int64_t r = total <= 0xffffffff ? static_cast<uint32_t>(it) / static_cast<uint32_t>(per) : it / per, at = (it - r * per) * 16;
    const uint8_t* p = J.x + r * J.ldx + at;
    u4v v = {0, 0, 0, 0};
    if (at + 16 <= J.C) {
      v = *reinterpret_cast<const u4v_any1*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (at + e < J.C) v[e >> 2] |= static_cast<uint32_t>(p[e]) << (8 * (e & 3));
      }
    }
    *reinterpret_cast<u4v*>(J.out + r * J.ldo + at) = v;
  }
}

inline bool known_act(int act) { return act >= DGCN_ACT_NONE && act <= DGCN_ACT_SILU; }
inline bool sizes_ok(int64_t rows, int32_t K, int32_t N) {
  return rows >= 0 && rows < (int64_t{1} << 36) && K >= 1 && N >= 1 && K <= (1 << 20) && N <= (1 << 20);
}

inline int type_bytes(int type) { return type == DGCN_T_F32 ? 4 : type == DGCN_T_E4M3 ? 1 : 2; }
inline int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// Memory of one call, handed out front to back in 256-byte steps (base null: only counted)
struct Arena {
  char* base;
  size_t used, size;
  void* take(size_t bytes) {
    char* p = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
  bool full() const { return used > size; }
};

// Rows off dwords are copied rather than read in place: a tile that takes them through registers, dwords and byte shifts, runs
// fp16 1021 x 1013 x 2047 in 24.7 us against 25.8, but 4096 x 4095 x 4096 in 250 against 148 (it wins where a few rows meet a large
// weight: 33 x 8191 x 8192 40 against 91; up to 32 rows the small kernel reads in place).
// An operand as the tiled kernel takes it: rows that start on dwords, and, where they are the k-rows of a K-strided operand
// (span: their C values), that do not repeat or overlap -- the k-rows behind the last one have to lie behind the buffer's end
struct Operand {
  const void* p;
  int64_t ld;
};

constexpr int64_t kFarStride = int64_t{1} << 20;           // strides from here on leave the tile's 32-bit offsets

inline bool operand_ready(const void* p, int64_t ld, int es, int64_t span) {
  return ld >= span && (reinterpret_cast<uintptr_t>(p) & 3) == 0 && ld * es % 4 == 0 && ld <= kFarStride;
}

// p's rows as an operand; where they are not ready, the copy that makes them so is added to the jobs (at most two)
Operand operand(const void* p, int64_t ld, int64_t rows, int64_t C, bool strided, int es, Arena& ws, PadJobs* jobs) {
  if (operand_ready(p, ld, es, strided ? C : 0)) return {p, ld};
  const int64_t ldo = round16(C * es);
  int64_t wgs = (rows * (ldo / 16) + 255) / 256;
  if (wgs > 32 * num_cus()) wgs = 32 * num_cus();
  uint8_t* to = static_cast<uint8_t*>(ws.take(rows * ldo));
  jobs->job[jobs->n++] = {static_cast<const uint8_t*>(p), ld * es, to, ldo, rows, C * es, static_cast<unsigned>(wgs)};
  return {to, ldo / es};
}

int pad_launch(const PadJobs& jobs, const Arena& ws, hipStream_t s) {
  if (ws.full()) return DGCN_E_WORKSPACE;
  if (jobs.n == 0) return DGCN_OK;
  hipLaunchKernelGGL(pad_rows_kernel, dim3(jobs.job[0].wgs + (jobs.n > 1 ? jobs.job[1].wgs : 0)), dim3(256), 0, s, jobs);
  return launch_status();
}

// One product; launch false: only its workspace is counted
int mat_run(MatParams P, int ta, int tb, int in_type, int out_type, Arena& ws, bool launch, hipStream_t s) {
  const MatPlan plan = mat_plan(P.M, P.N, P.K, in_type, ta);
  P.splits = plan.splits;
  if (plan.splits > 1) P.part = static_cast<float*>(ws.take(static_cast<size_t>(plan.splits) * P.M * P.N * sizeof(float)));
  if (!launch) return DGCN_OK;
  if (ws.full()) return DGCN_E_WORKSPACE;
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

int small_run(const MatParams& P, int in_type, int out_type, hipStream_t s) {
  switch (in_type) {
    case DGCN_T_F32: return mat_small_f32(P, s);
    case DGCN_T_BF16: return mat_small_bf16(P, s);
    case DGCN_T_F16: return mat_small_f16(P, s);
    default: return mat_small_e4m3(P, out_type, s);
  }
}

int linear_forward(MatParams P, int in_type, int out_type, Arena& ws, bool launch, hipStream_t s) {
  const int es = type_bytes(in_type);
  // Few rows go straight from memory.  From 17 on the tile is faster (32 rows x 16,384 x 4096 bf16: 31 us against 50, 1024 x 8192
  // 13 against 25, 4096 x 4096 16 against 14), but not by as much as a copy of a weight whose rows start off dwords costs.
  const bool ready = operand_ready(P.a, P.lda, es, 0) && operand_ready(P.b, P.ldb, es, 0);
  // Nor do few channels with a long K, whose workgroups leave most CUs idle: 256 x 16,384 bf16 takes 20 - 30 us against 9 split
  // over the tile's workgroups, 1024 x 8192 12 - 17 against 11, 512 x 4096 7 - 9 against 8.
  const bool narrow = P.N < 8 * static_cast<int64_t>(num_cus()) && P.K * es >= 16384;
  if (P.M <= (ready ? 16 : 32) && !(ready && narrow)) return launch ? small_run(P, in_type, out_type, s) : DGCN_OK;
  PadJobs pads = {};
  const Operand a = operand(P.a, P.lda, P.M, P.K, false, es, ws, &pads), b = operand(P.b, P.ldb, P.N, P.K, false, es, ws, &pads);
  if (launch) {
    const int rc = pad_launch(pads, ws, s);
    if (rc != DGCN_OK) return rc;
  }
  P.a = a.p; P.lda = a.ld; P.b = b.p; P.ldb = b.ld;
  return mat_run(P, 0, 0, in_type, out_type, ws, launch, s);
}

struct BwdArgs {
  const void* g;
  int64_t ldg;
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  const void* z;
  int act;
  float slope;
  int type;
  void *dx, *dw, *db;
  int db_f32;
  int64_t rows;
  int K, N;
};

inline MatParams plain_product(Operand a, Operand b, void* y, int64_t M, int64_t N, int64_t K) {
  MatParams P = {};
  P.a = a.p; P.lda = a.ld; P.b = b.p; P.ldb = b.ld;
  P.act = DGCN_ACT_NONE; P.splits = 1; P.y = y; P.M = M; P.N = N; P.K = K;
  return P;
}

template <class T>
int gate_launch(const BwdArgs& A, const GateShape& S, void* dz, int64_t lddz, float* part, hipStream_t s) {
  hipLaunchKernelGGL(gate_kernel<T>, dim3(S.gx, S.gy), dim3(256), 0, s, static_cast<const T*>(A.g), A.ldg, A.z, A.act, A.slope,
                     static_cast<T*>(dz), lddz, part, A.db, A.db_f32, A.rows, A.N, S.cl, S.slab);
  return launch_status();
}

int linear_backward(const BwdArgs& A, Arena& ws, bool launch, hipStream_t s) {
  const int es = type_bytes(A.type);
  const bool products = A.dx || A.dw, ready = operand_ready(A.g, A.ldg, es, A.dw ? A.N : 0);
  Operand dz = {A.g, A.ldg}, w = {}, x = {};
  int rc = DGCN_OK;
  if (A.act != DGCN_ACT_NONE || A.db || (products && !ready)) {
    const GateShape S = gate_shape(A.rows, A.N);
    void* to = nullptr;
    if (A.act != DGCN_ACT_NONE || (products && !ready)) {
      const int64_t ld = round16(static_cast<int64_t>(A.N) * es) / es;
      to = ws.take(A.rows * ld * es);
      dz = {to, ld};
    }
    float* part = A.db && S.gy > 1 ? static_cast<float*>(ws.take(static_cast<size_t>(S.gy) * A.N * sizeof(float))) : nullptr;
    if (launch) {
      if (ws.full()) return DGCN_E_WORKSPACE;
      switch (A.type) {
        case DGCN_T_F32: rc = gate_launch<float>(A, S, to, dz.ld, part, s); break;
        case DGCN_T_BF16: rc = gate_launch<__bf16>(A, S, to, dz.ld, part, s); break;
        default: rc = gate_launch<_Float16>(A, S, to, dz.ld, part, s); break;
      }
      if (rc == DGCN_OK && part) rc = dgcn_param_sum(part, S.gy, A.N, A.db_f32 ? DGCN_T_F32 : A.type, A.db, s);
      if (rc != DGCN_OK) return rc;
    }
  }
  PadJobs pads = {};
  if (A.dx) w = operand(A.w, A.ldw, A.N, A.K, true, es, ws, &pads);
  if (A.dw) x = operand(A.x, A.ldx, A.rows, A.K, true, es, ws, &pads);
  if (launch) rc = pad_launch(pads, ws, s);
  if (A.dx && rc == DGCN_OK) rc = mat_run(plain_product(dz, w, A.dx, A.rows, A.K, A.N), 0, 1, A.type, A.type, ws, launch, s);
  if (A.dw && rc == DGCN_OK) rc = mat_run(plain_product(dz, x, A.dw, A.N, A.K, A.rows), 1, 1, A.type, A.type, ws, launch, s);
  return rc;
}

}  // namespace
}  // namespace dgcn

using namespace dgcn;

extern "C" size_t dgcn_linear_workspace(const void* x, int64_t ldx, const void* w, int64_t ldw, int32_t in_type, int64_t rows,
                                        int32_t K, int32_t N) {
  if (!sizes_ok(rows, K, N) || rows == 0 || in_type < DGCN_T_F32 || in_type > DGCN_T_E4M3) return 0;
  MatParams P = {};
  P.a = x; P.lda = ldx; P.b = w; P.ldb = ldw; P.M = rows; P.N = N; P.K = K;
  Arena ws = {nullptr, 0, 0};
  linear_forward(P, in_type, in_type, ws, false, nullptr);
  return ws.used;
}

extern "C" int dgcn_linear_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const float* x_scale,
                               const float* w_scale, const void* bias, int32_t bias_f32, const void* res, int64_t ldr,
                               int32_t act, float slope, int32_t in_type, int32_t out_type, void* z, void* y, int64_t rows,
                               int32_t K, int32_t N, void* ws, size_t ws_bytes, void* stream) {
  if (!x || !w || !y || (in_type == DGCN_T_E4M3 && (!x_scale || !w_scale))) return DGCN_E_NULL;
  if (!sizes_ok(rows, K, N) || ldx < 0 || ldw < 0 || (res && ldr < 0)) return DGCN_E_SHAPE;
  if (!known_act(act) || out_type < DGCN_T_F32 || out_type > DGCN_T_F16 || (in_type != DGCN_T_E4M3 && in_type != out_type)) return DGCN_E_MODE;
  if (reinterpret_cast<uintptr_t>(ws) & 15) return DGCN_E_ALIGN;
  if (rows == 0) return DGCN_OK;
  const bool scaled = in_type == DGCN_T_E4M3;
  const MatParams P = {x, ldx, w, ldw, scaled ? x_scale : nullptr, scaled ? w_scale : nullptr, bias, bias_f32, act, slope, 1,
                       nullptr, res, ldr, z, y, rows, N, K};
  Arena arena = {static_cast<char*>(ws), 0, ws ? ws_bytes : 0};
  return linear_forward(P, in_type, out_type, arena, true, static_cast<hipStream_t>(stream));
}

extern "C" size_t dgcn_linear_bwd_workspace(const void* g, int64_t ldg, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                            int32_t act, int32_t dtype, int32_t want, int64_t rows, int32_t K, int32_t N) {
  if (!sizes_ok(rows, K, N) || rows == 0 || dtype < DGCN_T_F32 || dtype > DGCN_T_F16) return 0;
  char any;
  const BwdArgs A = {g, ldg, x, ldx, w, ldw, nullptr, act, 0.f, dtype, want & 1 ? &any : nullptr, want & 2 ? &any : nullptr,
                     want & 4 ? &any : nullptr, 0, rows, K, N};
  Arena ws = {nullptr, 0, 0};
  linear_backward(A, ws, false, nullptr);
  return ws.used;
}

extern "C" int dgcn_linear_bwd(const void* g, int64_t ldg, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* z,
                               int32_t act, float slope, int32_t dtype, void* dx, void* dw, void* db, int32_t db_f32,
                               int64_t rows, int32_t K, int32_t N, void* ws, size_t ws_bytes, void* stream) {
  if (!g || (dw && !x) || (dx && !w) || (act != DGCN_ACT_NONE && !z)) return DGCN_E_NULL;
  if (!sizes_ok(rows, K, N) || rows == 0 || ldg < 0 || ldx < 0 || ldw < 0) return DGCN_E_SHAPE;
  if (!known_act(act) || dtype < DGCN_T_F32 || dtype > DGCN_T_F16) return DGCN_E_MODE;
  if (reinterpret_cast<uintptr_t>(ws) & 15) return DGCN_E_ALIGN;
  if (!dx && !dw && !db) return DGCN_OK;
  const BwdArgs A = {g, ldg, x, ldx, w, ldw, z, act, slope, dtype, dx, dw, db, db_f32, rows, K, N};
  Arena arena = {static_cast<char*>(ws), 0, ws ? ws_bytes : 0};
  return linear_backward(A, arena, true, static_cast<hipStream_t>(stream));
}
