// Layer norm of each head's columns with a SiLU gate, for gfx950:
//   z = (x - mean_h) rstd_h,  f = z w + b,  y = f * SiLU(u)   (y = f without a gate)
// over the head_dim columns of every (row, head); heads = 1 is the layer norm of a row.
// With D = dL/dy SiLU(u) (or dL/dy):
//   dw = sum_rows D z,  db = sum_rows D,  dx = rstd (D w - mean_h(D w) - z mean_h(D w z)),
//   du = dL/dy f SiLU'(u).
//
// Bound: memory -- x, u, y once forward; dy, x, u, dx, du once backward.  Nothing is
// saved between the two: the backward has x in registers anyway and takes mean and rstd
// from it again, which is cheaper than a statistics buffer's traffic.  25728 rows of 8 heads
// of 64, bf16, gated: forward 16.6 us (79 MB, 4.8 TB/s), backward 30 us (132 MB, 4.4 TB/s)
// and 5 us for the sums of its 1024 row blocks.
//
// Layout: LPG lanes (a power of two, at most a wave) hold one head's columns as VPL
// vectors each, so a head's sums are log2(LPG) lane exchanges and no LDS.  A thread keeps
// its head and columns over the rows it walks: the weight gradients stay in its registers
// until the end, are added over the workgroup's rows in LDS and over the workgroups by a
// second kernel, both in a fixed order (no atomics: the same bits every run).
#include "grk_vec.h"

namespace grk {

constexpr int kHnThreads = 256;
constexpr int kHnFwdBlocks = 2048;     // workgroups of a forward at most: a full card, each walking its rows
constexpr int kHnBwdBlocks = 1024;     // row blocks of a backward at most: 4 workgroups on each CU
constexpr int kHnMaxDim = 2048;

struct HNParams {
  const void* x; int64_t ldx;
  const void* gate; int64_t ldg;
  const float* weight; const float* bias;   // either may be NULL (1 / 0)
  float eps;
  int64_t rows; int heads, dim;
  int head_tile, rows_per_iter;             // heads and rows of a workgroup's tile
  int vec_affine;                           // weight and bias start on 16 bytes
  void* y; int64_t ldy;
  // backward
  const void* dy; int64_t lddy;
  void* dx; int64_t lddx;
  void* dgate; int64_t lddg;
  float* partial;                           // [gridDim.x, 2, heads * dim], or NULL
};

template <int LPG>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = LPG / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// SiLU and its derivative.  fp32 rows take expf (within an ulp or two); the 16-bit types
// round away far more than the hardware exponential's 2^-21.
template <typename T>
__device__ __forceinline__ float sigmoid_of(float u) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-u));
  else return sigmoid_fast(u);
}

// A thread's place: its head, its first row and whether it has one.
struct HNPlace {
  int head, lane, row;
  bool on;
};
template <int LPG>
__device__ __forceinline__ HNPlace hn_place(const HNParams& p) {
  HNPlace t;
  const int g = threadIdx.x / LPG;
  t.lane = threadIdx.x % LPG;
  t.row = g / p.head_tile;
  t.head = blockIdx.y * p.head_tile + g % p.head_tile;
  t.on = t.row < p.rows_per_iter && t.head < p.heads;
  return t;
}

template <typename T, int V, int LPG, int VPL>
__device__ __forceinline__ void hn_load(const void* base, int64_t row, int64_t ld, int head, int dim, int lane,
                                        float* f) {
  const T* src = reinterpret_cast<const T*>(base) + row * ld + (int64_t)head * dim;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int c = (lane + LPG * j) * V;
    if (c < dim) {
      vload<T, V>(src + c, f + j * V);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[j * V + e] = 0.f;
    }
  }
}

template <typename T, int V, int LPG, int VPL>
__device__ __forceinline__ void hn_store(void* base, int64_t row, int64_t ld, int head, int dim, int lane,
                                         const float* f) {
  T* dst = reinterpret_cast<T*>(base) + row * ld + (int64_t)head * dim;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int c = (lane + LPG * j) * V;
    if (c < dim) vstore<T, V>(dst + c, f + j * V);
  }
}

// x -> z in place; returns rstd.  Mean first, then the centred squares (rows whose mean is
// large beside their spread keep their digits); columns past dim stay 0.
template <int V, int LPG, int VPL>
__device__ __forceinline__ float hn_normalise(float* x, int dim, int lane, float eps) {
  const float inv = 1.f / (float)dim;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < V * VPL; ++i) s += x[i];
  const float mean = group_sum<LPG>(s) * inv;
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < VPL; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = (lane + LPG * j) * V < dim ? x[j * V + e] - mean : 0.f;
      x[j * V + e] = d;
      q += d * d;
    }
  const float rstd = 1.f / sqrtf(group_sum<LPG>(q) * inv + eps);
#pragma unroll
  for (int i = 0; i < V * VPL; ++i) x[i] *= rstd;
  return rstd;
}

template <int V, int LPG, int VPL>
__device__ __forceinline__ void hn_affine(const float* src, bool vec, int head, int dim, int lane, float none,
                                          float* f) {
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int c = (lane + LPG * j) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) f[j * V + e] = none;
    if (!src || c >= dim) continue;
    const float* s = src + (int64_t)head * dim + c;
    if (V >= 4 && vec) {
#pragma unroll
      for (int e = 0; e + 3 < V; e += 4) vload<float, 4>(s + e, f + j * V + e);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[j * V + e] = s[e];
    }
  }
}

template <typename T, int V, int LPG, int VPL>
__global__ void __launch_bounds__(kHnThreads) k_hn_fwd(HNParams p) {
  constexpr int E = V * VPL;
  const HNPlace t = hn_place<LPG>(p);
  if (!t.on) return;   // whole groups of LPG lanes leave together
  float w[E], b[E];
  hn_affine<V, LPG, VPL>(p.weight, p.vec_affine, t.head, p.dim, t.lane, 1.f, w);
  hn_affine<V, LPG, VPL>(p.bias, p.vec_affine, t.head, p.dim, t.lane, 0.f, b);
  for (int64_t row = (int64_t)blockIdx.x * p.rows_per_iter + t.row; row < p.rows;
       row += (int64_t)gridDim.x * p.rows_per_iter) {
    float z[E], u[E];
    hn_load<T, V, LPG, VPL>(p.x, row, p.ldx, t.head, p.dim, t.lane, z);
    if (p.gate) hn_load<T, V, LPG, VPL>(p.gate, row, p.ldg, t.head, p.dim, t.lane, u);
    hn_normalise<V, LPG, VPL>(z, p.dim, t.lane, p.eps);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      z[i] = z[i] * w[i] + b[i];
      if (p.gate) z[i] *= u[i] * sigmoid_of<T>(u[i]);
    }
    hn_store<T, V, LPG, VPL>(p.y, row, p.ldy, t.head, p.dim, t.lane, z);
  }
}

template <typename T, int V, int LPG, int VPL>
__global__ void __launch_bounds__(kHnThreads) k_hn_bwd(HNParams p) {
  constexpr int E = V * VPL;
  __shared__ float red[2][kHnThreads * V];
  const HNPlace t = hn_place<LPG>(p);
  float w[E], b[E], dw[E], db[E];
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = db[i] = 0.f;
  if (t.on) {
    hn_affine<V, LPG, VPL>(p.weight, p.vec_affine, t.head, p.dim, t.lane, 1.f, w);
    hn_affine<V, LPG, VPL>(p.bias, p.vec_affine, t.head, p.dim, t.lane, 0.f, b);
    const float inv = 1.f / (float)p.dim;
    for (int64_t row = (int64_t)blockIdx.x * p.rows_per_iter + t.row; row < p.rows;
         row += (int64_t)gridDim.x * p.rows_per_iter) {
      float z[E], u[E], d[E];
      hn_load<T, V, LPG, VPL>(p.x, row, p.ldx, t.head, p.dim, t.lane, z);
      hn_load<T, V, LPG, VPL>(p.dy, row, p.lddy, t.head, p.dim, t.lane, d);
      if (p.gate) hn_load<T, V, LPG, VPL>(p.gate, row, p.ldg, t.head, p.dim, t.lane, u);
      const float rstd = hn_normalise<V, LPG, VPL>(z, p.dim, t.lane, p.eps);
      if (p.gate) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float sg = sigmoid_of<T>(u[i]), g = d[i];
          d[i] = g * (u[i] * sg);
          u[i] = g * (z[i] * w[i] + b[i]) * (sg * (1.f + u[i] * (1.f - sg)));
        }
        hn_store<T, V, LPG, VPL>(p.dgate, row, p.lddg, t.head, p.dim, t.lane, u);
      }
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        dw[i] += d[i] * z[i];
        db[i] += d[i];
        d[i] *= w[i];
        s1 += d[i];
        s2 += d[i] * z[i];
      }
      s1 = group_sum<LPG>(s1) * inv;
      s2 = group_sum<LPG>(s2) * inv;
#pragma unroll
      for (int i = 0; i < E; ++i) d[i] = rstd * (d[i] - s1 - z[i] * s2);
      hn_store<T, V, LPG, VPL>(p.dx, row, p.lddx, t.head, p.dim, t.lane, d);
    }
  }
  if (!p.partial) return;
  // the workgroup's rows, added in row order (threads of one head and lane are
  // head_tile * LPG apart)
  const int step = p.head_tile * LPG;
  const int64_t cols = (int64_t)p.heads * p.dim;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) {
      red[0][threadIdx.x * V + e] = dw[j * V + e];
      red[1][threadIdx.x * V + e] = db[j * V + e];
    }
    __syncthreads();
    const int c = (t.lane + LPG * j) * V;
    if (t.on && t.row == 0 && c < p.dim) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float a = 0.f, s = 0.f;
        for (int r = 0; r < p.rows_per_iter; ++r) {
          a += red[0][(threadIdx.x + r * step) * V + e];
          s += red[1][(threadIdx.x + r * step) * V + e];
        }
        float* dst = p.partial + (int64_t)blockIdx.x * 2 * cols + (int64_t)t.head * p.dim + c + e;
        dst[0] = a;
        dst[cols] = s;
      }
    }
  }
}

// out[i] = sum over the row blocks' partials: 16 threads a column, each every 16th block
// in order, their sums in order.
constexpr int kHnColGroups = 16;
__global__ void __launch_bounds__(64 * kHnColGroups) k_hn_colsum(const float* partial, int nblocks, int64_t cols,
                                                                  float* dw, float* db) {
  __shared__ float part[kHnColGroups][64];
  const int cl = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + cl;
  float s = 0.f;
  if (i < 2 * cols) {
#pragma unroll 8
    for (int b = g; b < nblocks; b += kHnColGroups) s += partial[(int64_t)b * 2 * cols + i];
  }
  part[g][cl] = s;
  __syncthreads();
  if (g == 0 && i < 2 * cols) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < kHnColGroups; ++j) t += part[j][cl];
    if (i < cols) { if (dw) dw[i] = t; }
    else if (db) db[i - cols] = t;
  }
}

// The lanes and vectors of a head: whole 16-byte vectors where rows and width allow,
// else single elements; the fewest lanes (a power of two) that hold it, at most a wave.
struct HNShape { int v, lpg, vpl; };
static HNShape hn_shape(int dim, int dtype, bool vec) {
  HNShape s;
  s.v = vec ? 16 / (int)dtype_size(dtype) : 1;
  const int n = (dim + s.v - 1) / s.v;
  s.lpg = 1;
  if (!vec) s.lpg = n <= 16 ? 16 : 64;
  while (s.lpg < n && s.lpg < 64) s.lpg *= 2;
  const int need = (n + s.lpg - 1) / s.lpg;
  s.vpl = 1;
  while (s.vpl < need) s.vpl *= 2;
  if (!vec && s.vpl > 1) s.vpl = s.vpl <= 4 ? 4 : 32;
  return s;
}

static void hn_tile(const HNShape& s, HNParams& p) {
  p.vec_affine = ((uintptr_t)p.weight | (uintptr_t)p.bias) % 16 == 0;
  const int groups = kHnThreads / s.lpg;
  p.head_tile = p.heads < groups ? p.heads : groups;
  p.rows_per_iter = groups / p.head_tile;
}

// Row blocks of a backward: each writes its partial weight gradients, so few rows take one
// workgroup a CU and no more until each has 4 turns.  Both kernels with 128, 256 and 512 blocks
// at least: 2000 rows of 1000, fp32, 16.6, 14.2 and 16.6 us, 4099 rows 20.3, 20.4 and 19.2; 2000
// rows of 8 heads of 64, bf16, 11.2, 9.8 and 11.9.
static int hn_bwd_blocks(int64_t rows, int rows_per_iter) {
  const int64_t turns = (rows + rows_per_iter - 1) / rows_per_iter;
  int64_t b = turns / 4;
  if (b > kHnBwdBlocks) b = kHnBwdBlocks;
  if (b < 256) b = turns < 256 ? turns : 256;
  return (int)b;
}

template <typename T, int V, int LPG, int VPL>
static void hn_launch(const HNParams& p, bool bwd, unsigned gx, hipStream_t s) {
  const dim3 grid(gx, (p.heads + p.head_tile - 1) / p.head_tile);
  if (bwd) k_hn_bwd<T, V, LPG, VPL><<<grid, kHnThreads, 0, s>>>(p);
  else k_hn_fwd<T, V, LPG, VPL><<<grid, kHnThreads, 0, s>>>(p);
}

template <typename T>
static int hn_run(const HNParams& p, const HNShape& c, bool bwd, unsigned gx, hipStream_t s) {
  constexpr int VE = vec_elems<T>();
#define HN_CASE(V, LPG, VPL) \
  if (c.v == V && c.lpg == LPG && c.vpl == VPL) return hn_launch<T, V, LPG, VPL>(p, bwd, gx, s), GRK_OK
  HN_CASE(VE, 1, 1); HN_CASE(VE, 2, 1); HN_CASE(VE, 4, 1); HN_CASE(VE, 8, 1); HN_CASE(VE, 16, 1);
  HN_CASE(VE, 32, 1); HN_CASE(VE, 64, 1); HN_CASE(VE, 64, 2); HN_CASE(VE, 64, 4);
  if constexpr (VE == 4) { HN_CASE(VE, 64, 8); }
  HN_CASE(1, 16, 1); HN_CASE(1, 64, 1); HN_CASE(1, 64, 4); HN_CASE(1, 64, 32);
#undef HN_CASE
  set_error("head_norm: no kernel for head_dim %d", p.dim);
  return GRK_EUNSUPPORTED;
}

static int hn_check(const HNParams& p, int dtype) {
  GRK_CHECK_ARG(known_dtype(dtype), "dtype must be fp32, bf16 or fp16");
  GRK_CHECK_ARG(p.rows >= 0 && p.heads > 0 && p.heads <= 65535, "rows >= 0 and heads in [1, 65535] required");
  GRK_CHECK_ARG(p.dim > 0 && p.dim <= kHnMaxDim, "head_dim must be in [1, %d]", kHnMaxDim);
  GRK_CHECK_ARG(p.eps >= 0.f, "eps must not be negative");
  return GRK_OK;
}

static int hn_rows_ok(const void* q, int64_t ld, const HNParams& p, const char* name) {
  GRK_CHECK_ARG(q, "%s required", name);
  GRK_CHECK_ARG(p.rows == 1 ? ld >= 0 : ld >= (int64_t)p.heads * p.dim, "%s: row stride below heads * head_dim", name);
  return GRK_OK;
}

}  // namespace grk

using namespace grk;

extern "C" int grk_head_norm_fwd(const void* x, int64_t ldx, const void* gate, int64_t ldg, const float* weight,
                                 const float* bias, float eps, int64_t rows, int heads, int head_dim, int dtype,
                                 void* y, int64_t ldy, void* stream) {
  clear_error();
  HNParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.ldx = ldx; p.gate = gate; p.ldg = ldg; p.weight = weight; p.bias = bias; p.eps = eps;
  p.rows = rows; p.heads = heads; p.dim = head_dim; p.y = y; p.ldy = ldy;
  int rc = hn_check(p, dtype);
  if (rc || rows == 0) return rc;
  if ((rc = hn_rows_ok(x, ldx, p, "x")) || (rc = hn_rows_ok(y, ldy, p, "y"))) return rc;
  if (gate && (rc = hn_rows_ok(gate, ldg, p, "gate"))) return rc;
  const bool vec = vec_rows(x, ldx, dtype) && vec_rows(y, ldy, dtype) && (!gate || vec_rows(gate, ldg, dtype)) &&
                   head_dim * (int)dtype_size(dtype) % 16 == 0;
  const HNShape c = hn_shape(head_dim, dtype, vec);
  hn_tile(c, p);
  const int64_t iters = (rows + p.rows_per_iter - 1) / p.rows_per_iter;
  const int gy = (heads + p.head_tile - 1) / p.head_tile;
  const int64_t most = gy < kHnFwdBlocks ? kHnFwdBlocks / gy : 1;
  const unsigned gx = (unsigned)(iters < most ? iters : most);
  rc = for_dtype(dtype, [&](auto t) { return hn_run<decltype(t)>(p, c, false, gx, (hipStream_t)stream); });
  if (rc) return rc;
  GRK_LAUNCH_CHECK();
  return GRK_OK;
}

extern "C" size_t grk_head_norm_bwd_workspace(int64_t rows, int heads, int head_dim) {
  if (rows <= 0 || heads <= 0 || head_dim <= 0) return 0;
  // a workgroup walks one row at a time at least: no fewer blocks than any launch takes
  return (size_t)hn_bwd_blocks(rows, 1) * 2 * (size_t)heads * head_dim * sizeof(float);
}

extern "C" int grk_head_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* gate,
                                 int64_t ldg, const float* weight, const float* bias, float eps, int64_t rows,
                                 int heads, int head_dim, int dtype, void* dx, int64_t lddx, void* dgate,
                                 int64_t lddg, float* dweight, float* dbias, void* ws, size_t ws_bytes,
                                 void* stream) {
  clear_error();
  HNParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.ldx = ldx; p.gate = gate; p.ldg = ldg; p.weight = weight; p.bias = bias; p.eps = eps;
  p.rows = rows; p.heads = heads; p.dim = head_dim;
  p.dy = dy; p.lddy = lddy; p.dx = dx; p.lddx = lddx; p.dgate = dgate; p.lddg = lddg;
  int rc = hn_check(p, dtype);
  if (rc) return rc;
  hipStream_t s = (hipStream_t)stream;
  const int64_t cols = (int64_t)heads * head_dim;
  if (rows == 0) {
    if (dweight) GRK_CHECK_HIP(zero_async(dweight, cols * sizeof(float), s));
    if (dbias) GRK_CHECK_HIP(zero_async(dbias, cols * sizeof(float), s));
    return GRK_OK;
  }
  if ((rc = hn_rows_ok(dy, lddy, p, "dy")) || (rc = hn_rows_ok(x, ldx, p, "x")) ||
      (rc = hn_rows_ok(dx, lddx, p, "dx")))
    return rc;
  if (gate && ((rc = hn_rows_ok(gate, ldg, p, "gate")) || (rc = hn_rows_ok(dgate, lddg, p, "dgate")))) return rc;
  if (dweight || dbias) {
    GRK_CHECK_ARG(ws && ws_bytes >= grk_head_norm_bwd_workspace(rows, heads, head_dim), "workspace too small");
    p.partial = (float*)ws;
  }
  const bool vec = vec_rows(x, ldx, dtype) && vec_rows(dy, lddy, dtype) && vec_rows(dx, lddx, dtype) &&
                   (!gate || (vec_rows(gate, ldg, dtype) && vec_rows(dgate, lddg, dtype))) &&
                   head_dim * (int)dtype_size(dtype) % 16 == 0;
  const HNShape c = hn_shape(head_dim, dtype, vec);
  hn_tile(c, p);
  const int nb = hn_bwd_blocks(rows, p.rows_per_iter);
  rc = for_dtype(dtype, [&](auto t) { return hn_run<decltype(t)>(p, c, true, (unsigned)nb, s); });
  if (rc) return rc;
  GRK_LAUNCH_CHECK();
  if (p.partial) {
    k_hn_colsum<<<(unsigned)((2 * cols + 63) / 64), 64 * kHnColGroups, 0, s>>>(p.partial, nb, cols, dweight, dbias);
    GRK_LAUNCH_CHECK();
  }
  return GRK_OK;
}
