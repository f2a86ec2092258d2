// Rotary positions for gfx950.  In each head the first 2r columns hold r pairs
// (x_i, x_j): (i, i + r) in the half layout, (2i, 2i + 1) interleaved.  A row at
// position p turns pair i by p * freq_i:
//   y_i = s (cos x_i - sin x_j),  y_j = s (cos x_j + sin x_i),
// the other columns pass.  The gradient is the same pass with -sin (the turn's
// transpose is the turn back), so it needs neither x nor y.
//
// Bound: memory -- every element is read and written once for 3 operations.  The
// angles are what could cost more: sine and cosine of one (row, i) serve every head of
// the row, so a workgroup computes those of its rows once into LDS and then streams
// the rows in 16-byte vectors (25728 rows of 16 heads of 64, bf16, 105 MB: 23.7 us, 4.4 TB/s;
// 32771 rows of 8 heads of 80, fp32, 168 MB: 27.4 us, 6.1 TB/s, part of it from the cache).
#include "grk_vec.h"

namespace grk {

constexpr int kRotThreads = 256;
constexpr int kRotAngles = 1024;   // (cos, sin) pairs of a workgroup's rows: 8 KB of LDS

struct RotParams {
  const void* x; int64_t ldx;
  void* y; int64_t ldy;
  const void* pos; int pos64;
  const double* freqs;
  int64_t rows;
  int heads, head_dim, r, interleaved;
  float scale, sign;
  int rows_per_block;
};

// One pair turned by w = (cos, sin); the fma is written out so that every path (layouts,
// vectors or single columns) gives the same bits.
__device__ __forceinline__ void turn(float& a, float& b, float2 w) {
  const float x = a, y = b;
  a = fmaf(x, w.x, -(y * w.y));
  b = fmaf(y, w.x, x * w.y);
}

// The angle is reduced in 64 bits: at position 10^6 an fp32 product p * freq is off by
// up to 0.03 rad, the fp64 one by 10^-10.  What is left, a fraction of a turn, is an
// fp32 argument of sincospi (2^-25 of half a turn).
template <typename T, int V, bool PAST>
__global__ void __launch_bounds__(kRotThreads) k_rotary(RotParams p) {
  __shared__ float2 cs[kRotAngles];
  const int64_t row0 = (int64_t)blockIdx.x * p.rows_per_block;
  const int nrows = (int)(p.rows - row0 < p.rows_per_block ? p.rows - row0 : p.rows_per_block);
  for (int a = threadIdx.x; a < nrows * p.r; a += kRotThreads) {
    const int row = a / p.r, i = a - row * p.r;
    const double pos = p.pos64 ? (double)reinterpret_cast<const int64_t*>(p.pos)[row0 + row]
                               : (double)reinterpret_cast<const int32_t*>(p.pos)[row0 + row];
    const double turns = pos * p.freqs[i] * 0.15915494309189533577;   // 1 / (2 pi)
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[a] = make_float2(c * p.scale, s * p.scale * p.sign);
  }
  __syncthreads();
  // units of a head: with the half layout r / V turned pairs of vectors (columns c and
  // c + r), then the vectors that pass; interleaved every vector by itself
  const int turned = p.interleaved ? 0 : p.r / V;
  const int units = p.interleaved ? p.head_dim / V : turned + (p.head_dim - 2 * p.r) / V;
  const int per_row = units * p.heads;
  for (int n = threadIdx.x; n < nrows * per_row; n += kRotThreads) {
    const int row = n / per_row, rest = n - row * per_row;
    const int h = rest / units, u = rest - h * units;
    const T* x = reinterpret_cast<const T*>(p.x) + (row0 + row) * p.ldx + (int64_t)h * p.head_dim;
    T* y = reinterpret_cast<T*>(p.y) + (row0 + row) * p.ldy + (int64_t)h * p.head_dim;
    const float2* t = cs + row * p.r;
    if (u < turned) {
      float xa[V], xb[V];
      vload<T, V>(x + u * V, xa);
      vload<T, V>(x + p.r + u * V, xb);
#pragma unroll
      for (int e = 0; e < V; ++e) turn(xa[e], xb[e], t[u * V + e]);
      vstore<T, V, PAST>(y + u * V, xa);
      vstore<T, V, PAST>(y + p.r + u * V, xb);
    } else if (!p.interleaved) {
      const int c = 2 * p.r + (u - turned) * V;
      float v[V];
      vload<T, V>(x + c, v);
      vstore<T, V, PAST>(y + c, v);
    } else {
      static_assert(V == 1 || V % 2 == 0, "");
      const int c = u * V;
      if constexpr (V == 1) {   // one column of a pair: the unit of its even column writes both
        if (c < 2 * p.r) {
          if (!(c & 1)) {
            float a = to_f32(x[c]), b = to_f32(x[c + 1]);
            turn(a, b, t[c >> 1]);
            y[c] = from_f32<T>(a);
            y[c + 1] = from_f32<T>(b);
          }
        } else {
          y[c] = x[c];
        }
      } else {
        float v[V];
        vload<T, V>(x + c, v);
#pragma unroll
        for (int e = 0; e < V; e += 2)
          if (c + e < 2 * p.r) turn(v[e], v[e + 1], t[(c + e) >> 1]);
        vstore<T, V, PAST>(y + c, v);
      }
    }
  }
}

}  // namespace grk

using namespace grk;

extern "C" int grk_rotary(const void* x, int64_t ldx, void* y, int64_t ldy, int dtype, const void* positions,
                          int itype, const double* freqs, int64_t rows, int heads, int head_dim, int rotary_dim,
                          int interleaved, float scale, int inverse, void* stream) {
  clear_error();
  GRK_CHECK_ARG(known_dtype(dtype), "dtype must be fp32, bf16 or fp16");
  GRK_CHECK_ARG(itype == GRK_I32 || itype == GRK_I64, "positions must be int32 or int64");
  GRK_CHECK_ARG(rows >= 0 && heads > 0 && head_dim > 0 && (int64_t)heads * head_dim <= (1 << 20),
                "rows >= 0, heads > 0, head_dim > 0 and heads * head_dim <= 2^20");
  GRK_CHECK_ARG(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim && rotary_dim <= 2 * kRotAngles,
                "rotary_dim must be even, in [2, min(head_dim, %d)]", 2 * kRotAngles);
  if (rows == 0) return GRK_OK;
  const int64_t cols = (int64_t)heads * head_dim;
  GRK_CHECK_ARG(x && y && positions && freqs, "x / y / positions / freqs required");
  GRK_CHECK_ARG((rows == 1 || (ldx >= cols && ldy >= cols)) && ldx >= 0 && ldy >= 0,
                "row strides must be at least heads * head_dim");
  GRK_CHECK_ARG(x != y || ldx == ldy, "in place: x and y must have one row stride");
  RotParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.ldx = ldx; p.y = y; p.ldy = ldy; p.pos = positions; p.pos64 = itype == GRK_I64; p.freqs = freqs;
  p.rows = rows; p.heads = heads; p.head_dim = head_dim; p.r = rotary_dim / 2; p.interleaved = interleaved != 0;
  p.scale = scale; p.sign = inverse ? -1.f : 1.f;
  const int ve = 16 / (int)dtype_size(dtype);
  // whole vectors: the rows, the heads in them and, in the half layout, both halves
  const bool vec = vec_rows(x, ldx, dtype) && vec_rows(y, ldy, dtype) && head_dim % ve == 0 &&
                   (p.interleaved || p.r % ve == 0);
  // An output of a quarter of the 256 MB cache or more passes it by and leaves it to what was
  // there, the input among it (32771 rows of 8 heads of 80, fp32, 84 MB: 39.7 -> 27.4 us);
  // smaller ones stay for their reader (25728 rows of 16 heads of 64, bf16, 53 MB: 23.4 us,
  // past the cache 25.2).  Heads of 64, three inputs and outputs in turn, stored to the cache
  // and past it: bf16 32 MB 12.5 and 13.6 us, 64 MB 29.2 and 25.4, 128 MB 52.9 and 51.2; fp32 12.1
  // and 12.3, 26.6 and 22.0, 50.3 and 48.7.  48 MB gain too (22.2 and 19.3), unless the same
  // buffers come again (17.2 and 19.3).
  const bool past = rows * cols * (int64_t)dtype_size(dtype) >= (64 << 20);
  // rows of a workgroup: enough that it streams 32 KB, few enough that the grid holds
  // 1024 workgroups (4 on each CU) and their angles fit the LDS table
  int64_t rpb = 32768 / (cols * (int64_t)dtype_size(dtype));
  if (rpb > rows / 1024) rpb = rows / 1024;
  if (rpb > kRotAngles / p.r) rpb = kRotAngles / p.r;
  if (rpb < 1) rpb = 1;
  p.rows_per_block = (int)rpb;
  const int64_t grid = (rows + rpb - 1) / rpb;
  GRK_CHECK_ARG(grid < (1 << 24), "too many rows");
  hipStream_t s = (hipStream_t)stream;
  const int rc = for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (vec && past) k_rotary<T, vec_elems<T>(), true><<<(unsigned)grid, kRotThreads, 0, s>>>(p);
    else if (vec) k_rotary<T, vec_elems<T>(), false><<<(unsigned)grid, kRotThreads, 0, s>>>(p);
    else k_rotary<T, 1, false><<<(unsigned)grid, kRotThreads, 0, s>>>(p);
    return 0;
  });
  (void)rc;
  GRK_LAUNCH_CHECK();
  return GRK_OK;
}
