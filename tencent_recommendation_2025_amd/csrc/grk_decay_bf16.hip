// Decayed linear attention of bf16 rows on the bf16 matrix instruction, for gfx950 (the
// formulas: grk_decay.h; heads and rows made of 16-byte vectors).
//
// A workgroup walks a segment in chunks of 64 steps; each wave owns NE tiles of 16 columns
// of the state and of the output.  v_mfma_f32_16x16x32_bf16: lane
// l = 16 g + c holds A[c][8 g + s] and B[8 g + s][c], s < 8, and D[4 g + i][c], i < 4 -- A
// and B fragments are laid out alike, so exchanging them transposes D.  What is stored
// comes out transposed on purpose: P^T = K Q^T and O^T = V^T P^T + S^T Q^T leave 4
// neighbouring columns of one row in a lane (8-byte stores).  The state tile
// S = K^T V leaves rows 4 g + i of column c in a lane: two tiles are the fragment of S^T
// if the contraction takes its 32 d in the order (4 g + i, 16 + 4 g + i), so Q is read
// from LDS in that order (two 8-byte reads) and the state never leaves its registers.
//
// Per chunk and wave (DP = 64): P^T 6 MFMA (lower tiles only), O^T 8 + 6, S 8: 28, a
// quarter of the time the chunk's 32 KB take from HBM on one CU of 256, so the kernel is
// bound by memory and by what hides its latency: the next chunk is loaded to registers
// while this one is computed, and 4 workgroups share a CU.
#include "grk_decay.h"
#include "grk_mfma.h"

namespace grk {

// Powers of g in LDS: pw[n] = g^n for 0 <= n <= 64 and 0 for -16 < n < 0 (above the diagonal).
constexpr int kDecayPowers = 16 + kDecayChunk + 1;

template <int DP> constexpr size_t decay_lds_bf16(bool state_only) {
  return (size_t)(state_only ? 2 : 3) * kDecayChunk * DP * 2 + (state_only ? 0 : kDecayChunk * kDecayChunk * 2) +
         kDecayChunk * 4 + (kDecayPowers + 3) / 4 * 16;
}

__device__ __forceinline__ void mfma32(bf16x8 a, bf16x8 b, f32x4& c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  mfma_keep(c, a, b);
}

// Fragment of M^T: element s of lane (c, g) = M[row0 + 8 g + s][col0 + c].  A 16-lane group
// of the transposing read takes 4 rows of 16 columns, lane i of it the row i / 4 from
// column 4 (i % 4) on, and receives column i of the 4 rows.
template <int HD>
__device__ __forceinline__ bf16x8 lds_col8(const char* base, int row0, int col0, int lane) {
  const int i = lane & 15, row = row0 + 8 * (lane >> 4) + (i >> 2), col = col0 + 4 * (i & 3);
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + lds_off<HD>(row, col)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + lds_off<HD>(row + 4, col)));
  const bf16x4 l = __builtin_bit_cast(bf16x4, lo), h = __builtin_bit_cast(bf16x4, hi);
  return bf16x8{l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
}

// Fragment of the rows in the state's order: M[row][col0 + 4 g + s], M[row][col0 + 16 + 4 g + s].
template <int HD>
__device__ __forceinline__ bf16x8 lds_row_pair(const char* base, int row, int col0, int g) {
  const uint2 a = *reinterpret_cast<const uint2*>(base + lds_off<HD>(row, col0 + 4 * g));
  const uint2 b = *reinterpret_cast<const uint2*>(base + lds_off<HD>(row, col0 + 16 + 4 * g));
  return __builtin_bit_cast(bf16x8, make_uint4(a.x, a.y, b.x, b.y));
}

__device__ __forceinline__ bf16x8 pack8(const float* f) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (__bf16)f[i];
  return r;
}

// Rows of a chunk on their way from memory: thread t holds columns [8 (t % (DP / 8)), + 8) of
// row t / (DP / 8) and of every R-th after it, R = threads / (DP / 8).  Masked steps are loaded too (their row exists) and zeroed by
// selection, so the loads do not wait for the mask.
template <int DP, int NTH>
struct DecayRows {
  static constexpr int R = NTH / (DP / 8), N = kDecayChunk / R;
  int64_t row[N];
  bool live[N];
  __device__ __forceinline__ void at(const DecayParams& p, const DecayPlace& w, int rev, int64_t base, int t0) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int t = t0 + (int)threadIdx.x / (DP / 8) + R * k;
      const int pos = rev ? p.seq_len - 1 - t : w.start + t;
      const int64_t r = base + pos;
      live[k] = t < w.t1 && r >= 0 && r < p.capacity;
      row[k] = live[k] ? r : 0;
      if (p.key_valid && live[k]) live[k] = p.key_valid[(int64_t)w.b * p.seq_len + pos] != 0;
    }
  }
  __device__ __forceinline__ void load(uint4* f, const void* src, int64_t ld, int64_t col) const {
#pragma unroll
    for (int k = 0; k < N; ++k)
      f[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16_t*>(src) + row[k] * ld + col);
  }
  __device__ __forceinline__ void store(const uint4* f, char* dst, bool has) const {
#pragma unroll
    for (int k = 0; k < N; ++k)
      *reinterpret_cast<uint4*>(dst + lds_off<DP>((int)threadIdx.x / (DP / 8) + R * k, (int)threadIdx.x % (DP / 8) * 8)) =
          live[k] && has ? f[k] : make_uint4(0u, 0u, 0u, 0u);
  }
};

// NS: bf16 parts of g^(n-1-j) v_j in the state's sum.  1 where the state only feeds bf16
// outputs (it is rounded to bf16 as their operand anyway); 3 (all 24 bits of the fp32
// value) where it is returned in fp32.
template <int DP, int NE, int NS, bool STATE>
__global__ void __launch_bounds__(DP * 4 / NE, NE == 1 ? 4 : 2) k_decay_bf16(DecayParams p) {
  constexpr int C = kDecayChunk, NT = DP / 16, KS = DP / 32, NW = NT / NE, NTH = NW * 64;
  using Rows = DecayRows<DP, NTH>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char* sb = lds;
  char* sc = sb + C * DP * 2;
  char* sa = sc + C * DP * 2;
  char* sp = sa + (STATE ? 0 : C * DP * 2);
  float* pw = reinterpret_cast<float*>(sp + (STATE ? 0 : C * C * 2)) + 16;
  int* slive = reinterpret_cast<int*>(pw - 16 + (kDecayPowers + 3) / 4 * 4);
  const DecayPlace w = decay_place(p);
  if (!w.on) return;
  const DecayRole r = p.role[w.role];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t bh = (int64_t)w.b * p.heads + w.h, hcol = (int64_t)w.h * p.head_dim;
  const int64_t base = p.row_base ? p.row_base[w.b] : (int64_t)w.b * p.seq_len;
  const int ccol = (int)threadIdx.x % (DP / 8) * 8;      // this thread's columns when rows are moved
  const bool has = ccol < p.head_dim;
  const int64_t mcol = hcol + (has ? ccol : 0);
  f32x4 st[NE][NT];
  float* frag = p.ws + (((int64_t)w.role * p.batch * p.heads + bh) * p.nseg + w.seg) * DP * DP;
  bool some = STATE || (p.nseg > 1 ? w.seg > 0 || p.state_in : p.state_in != nullptr);   // the state is not all 0
#pragma unroll
  for (int x = 0; x < NE; ++x) {
    const int et = NE * wave + x;   // the wave's column tiles
#pragma unroll
    for (int dt = 0; dt < NT; ++dt) {
      st[x][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (!STATE && p.nseg > 1) {
        st[x][dt] = *reinterpret_cast<const f32x4*>(frag + ((dt * NT + et) * 64 + lane) * 4);
      } else if (!STATE && p.state_in) {
        const float f = decay_pow(w.lg, w.start);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 16 * dt + 4 * g + i, e = 16 * et + c;
          if (d < p.head_dim && e < p.head_dim) st[x][dt][i] = f * p.state_in[(bh * p.head_dim + d) * p.head_dim + e];
        }
      }
    }
  }
  Rows rows;
  uint4 fa[Rows::N], fb[Rows::N], fc[Rows::N];
  if (w.t0 < w.t1) {
    rows.at(p, w, r.rev, base, w.t0);
    rows.load(fb, r.b, r.ldb, mcol);
    rows.load(fc, r.c, r.ldc, mcol);
    if (!STATE) rows.load(fa, r.a, r.lda, mcol);
  }
  for (int n = threadIdx.x; n < kDecayPowers; n += NTH) pw[n - 16] = n < 16 ? 0.f : decay_pow(w.lg, n - 16);
  if constexpr (!STATE) {
    for (int n = threadIdx.x; n < C * C / 8; n += NTH) reinterpret_cast<uint4*>(sp)[n] = make_uint4(0u, 0u, 0u, 0u);
    decay_zero_rows<bf16_t>(p, w, r);
  }
  for (int t0 = w.t0; t0 < w.t1; t0 += C) {
    const int n = w.t1 - t0 < C ? w.t1 - t0 : C;
    const bool last = t0 + C >= w.t1;
    __syncthreads();
    rows.store(fb, sb, has);
    rows.store(fc, sc, has);
    if constexpr (!STATE) {
      rows.store(fa, sa, has);
      if (ccol == 0) {
#pragma unroll
        for (int k = 0; k < Rows::N; ++k) slive[(int)threadIdx.x / (DP / 8) + Rows::R * k] = rows.live[k];
      }
    }
    __syncthreads();
    if (!last) {
      rows.at(p, w, r.rev, base, t0 + C);
      rows.load(fb, r.b, r.ldb, mcol);
      rows.load(fc, r.c, r.ldc, mcol);
      if (!STATE) rows.load(fa, r.a, r.lda, mcol);
    }
    if constexpr (!STATE) {
      // P^T, lower tiles; the tiles above the diagonal that a 32-deep step reads stay 0
      for (int tile = wave; tile < 10; tile += NW) {
        const int it = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, jt = tile - it * (it + 1) / 2;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          mfma32(lds_row8<DP>(sb, 16 * jt + c, 32 * ks + 8 * g), lds_row8<DP>(sa, 16 * it + c, 32 * ks + 8 * g), x);
        const float* lag = pw + 16 * (it - jt) + c - 4 * g;
        bf16x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (__bf16)(x[i] * lag[-i]);
        *reinterpret_cast<bf16x4*>(sp + lds_off<C>(16 * it + c, 16 * jt + 4 * g)) = y;
      }
      __syncthreads();
    }
    bf16x8 vf[NE][2];
#pragma unroll
    for (int x = 0; x < NE; ++x)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) vf[x][ks] = lds_col8<DP>(sc, 32 * ks, 16 * (NE * wave + x), lane);
    if constexpr (!STATE) {
      bf16x8 sf[NE][KS];
#pragma unroll
      for (int x = 0; x < NE; ++x)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const f32x4 a = st[x][2 * ks], b = st[x][2 * ks + 1];
          const float f[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
          sf[x][ks] = pack8(f);
        }
#pragma unroll
      for (int it = 0; it < C / 16; ++it) {
        f32x4 o[NE];
#pragma unroll
        for (int x = 0; x < NE; ++x) o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (some) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const bf16x8 q = lds_row_pair<DP>(sa, 16 * it + c, 32 * ks, g);
#pragma unroll
            for (int x = 0; x < NE; ++x) mfma32(sf[x][ks], q, o[x]);
          }
#pragma unroll
          for (int x = 0; x < NE; ++x) o[x] *= pw[16 * it + c + 1];
        }
#pragma unroll
        for (int ks = 0; ks <= it / 2; ++ks) {
          const bf16x8 y = lds_row8<C>(sp, 16 * it + c, 32 * ks + 8 * g);
#pragma unroll
          for (int x = 0; x < NE; ++x) mfma32(vf[x][ks], y, o[x]);
        }
        const int t = 16 * it + c;
        const int64_t row = base + (r.rev ? p.seq_len - 1 - (t0 + t) : w.start + t0 + t);
        if (t < n && row >= 0 && row < p.capacity) {
          const bool live = slive[t];
#pragma unroll
          for (int x = 0; x < NE; ++x) {
            const int e = 16 * (NE * wave + x) + 4 * g;
            bf16x4 y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = (__bf16)(live ? p.scale * o[x][i] : 0.f);
            if (e < p.head_dim)
              *reinterpret_cast<bf16x4*>(reinterpret_cast<bf16_t*>(r.out) + row * r.ldo + hcol + e) = y;
          }
        }
      }
    }
    if (!STATE && last && !(p.nseg == 1 && p.state_out)) break;   // nothing reads the state any more
    some = true;
    const float gn = pw[n];
#pragma unroll
    for (int x = 0; x < NE; ++x)
#pragma unroll
      for (int dt = 0; dt < NT; ++dt) st[x][dt] *= gn;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      bf16x8 part[NE][NS];
#pragma unroll
      for (int x = 0; x < NE; ++x) {
        float f[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const int j = 32 * ks + 8 * g + s;
          f[s] = (float)vf[x][ks][s] * (j < n ? pw[n - 1 - j] : 0.f);
        }
#pragma unroll
        for (int q = 0; q < NS; ++q) {
          part[x][q] = pack8(f);
#pragma unroll
          for (int s = 0; s < 8; ++s) f[s] -= (float)part[x][q][s];
        }
      }
#pragma unroll
      for (int dt = 0; dt < NT; ++dt) {
        const bf16x8 k = lds_col8<DP>(sb, 32 * ks, 16 * dt, lane);
#pragma unroll
        for (int x = 0; x < NE; ++x)
#pragma unroll
          for (int q = NS - 1; q >= 0; --q) mfma32(k, part[x][q], st[x][dt]);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < NE; ++x)
#pragma unroll
    for (int dt = 0; dt < NT; ++dt) {
      const int et = NE * wave + x;
      if (STATE) {
        *reinterpret_cast<f32x4*>(frag + ((dt * NT + et) * 64 + lane) * 4) = st[x][dt];
      } else if (p.nseg == 1 && p.state_out) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 16 * dt + 4 * g + i, e = 16 * et + c;
          if (d < p.head_dim && e < p.head_dim) p.state_out[(bh * p.head_dim + d) * p.head_dim + e] = st[x][dt][i];
        }
      }
    }
}

template <int DP, int NE>
static int decay_bf16_run(const DecayParams& p, hipStream_t s) {
  const int64_t groups = (int64_t)p.batch * p.heads * p.nseg;
  const unsigned grid = (unsigned)((groups + 7) / 8 * 8 * p.roles);
  if (p.nseg > 1) {
    constexpr size_t lds = decay_lds_bf16<DP>(true);
    if (p.state_out) {
      GRK_CHECK_HIP(ensure_dynamic_lds((const void*)k_decay_bf16<DP, NE, 3, true>, lds));
      k_decay_bf16<DP, NE, 3, true><<<grid, DP * 4 / NE, lds, s>>>(p);
    } else {
      GRK_CHECK_HIP(ensure_dynamic_lds((const void*)k_decay_bf16<DP, NE, 1, true>, lds));
      k_decay_bf16<DP, NE, 1, true><<<grid, DP * 4 / NE, lds, s>>>(p);
    }
    GRK_LAUNCH_CHECK();
    const int rc = decay_scan_launch(p, DP, s);
    if (rc) return rc;
  }
  constexpr size_t lds = decay_lds_bf16<DP>(false);
  if (p.nseg == 1 && p.state_out) {
    GRK_CHECK_HIP(ensure_dynamic_lds((const void*)k_decay_bf16<DP, NE, 3, false>, lds));
    k_decay_bf16<DP, NE, 3, false><<<grid, DP * 4 / NE, lds, s>>>(p);
  } else {
    GRK_CHECK_HIP(ensure_dynamic_lds((const void*)k_decay_bf16<DP, NE, 1, false>, lds));
    k_decay_bf16<DP, NE, 1, false><<<grid, DP * 4 / NE, lds, s>>>(p);
  }
  GRK_LAUNCH_CHECK();
  return GRK_OK;
}

// Whole 16-byte vectors: rows, strides and heads start on them (8 bytes for the output).
bool decay_bf16_takes(const DecayParams& p) {
  bool ok = p.head_dim % 8 == 0;
  for (int i = 0; i < p.roles; ++i) {
    const DecayRole& r = p.role[i];
    ok = ok && ((uintptr_t)r.a | (uintptr_t)r.b | (uintptr_t)r.c) % 16 == 0 && (r.lda | r.ldb | r.ldc) % 8 == 0 &&
         (uintptr_t)r.out % 8 == 0 && r.ldo % 4 == 0;
  }
  return ok;
}

int decay_bf16_launch(const DecayParams& p, hipStream_t s) {
  if (p.head_dim <= 32) return decay_bf16_run<32, 1>(p, s);
  if (p.head_dim <= 64) return decay_bf16_run<64, 1>(p, s);
  return decay_bf16_run<128, 2>(p, s);
}

}  // namespace grk
