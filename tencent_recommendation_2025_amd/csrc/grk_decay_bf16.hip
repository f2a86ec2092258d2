// Decayed linear attention of bf16 rows on the bf16 matrix instruction, for gfx950 (the
// formulas: grk_decay.h; heads and rows made of 16-byte vectors).
//
// A workgroup walks a segment in chunks of C steps with EW columns of the state (and of the
// output); each wave owns NE tiles of 16 of them.  v_mfma_f32_16x16x32_bf16: lane
// l = 16 g + c holds A[c][8 g + s] and B[8 g + s][c], s < 8, and D[4 g + i][c], i < 4 -- A
// and B fragments are laid out alike, so exchanging them transposes D.  What is stored
// comes out transposed on purpose: P^T = K Q^T and O^T = V^T P^T + S^T Q^T leave 4
// neighbouring columns of one row in a lane (8-byte stores).  The state tile
// S = K^T V leaves rows 4 g + i of column c in a lane: two tiles are the fragment of S^T
// if the contraction takes its 32 d in the order (4 g + i, 16 + 4 g + i), so Q is read
// from LDS in that order (two 8-byte reads) and the state never leaves its registers.
//
// Bound: heads of 64, memory's latency -- a wave takes some 20 MFMA, 190 VALU operations and
// 26 LDS accesses for 32 steps, half of the time that their 16 KB take from HBM on one CU
// of 256; what is left is the wait of a chunk's two barriers, which the next chunk's loads
// (to registers, while this one is computed) and 4 to 5 waves a SIMD cover in part.  128
// sequences of up to 201 events (16 K packed rows) of 8 heads of 64: forward 17.6 us (66
// MB, 3.8 TB/s), gradients 35.9 us (116 MB, 3.2 TB/s).  Heads of 128: LDS, read for every
// operand of 4 products a chunk.  8 x 4096 events of 4 heads: 39 us and gradients 89 us
// after 40 and 44 us for the segment states.
//
// LDS rows are 16 bytes longer than the head: 16 rows' 16-byte pieces fall on all 64 banks
// at once, every address is a lane's base plus a constant, and a transposing read that
// takes every second row (4 rows 8 banks apart) has no conflicts either.  So the
// contraction over a chunk's steps takes each 8 of them in the order 0 2 4 6 1 3 5 7 ("slots"):
// P and the weights of the state's sum are laid down in that order.
#include <type_traits>

#include "grk_decay.h"
#include "grk_mfma.h"

namespace grk {

// Tables in LDS: scale g^n for 0 <= n <= C, 0 for -16 < n < 0 (above the diagonal); the
// state's weights g^(C - 1 - j) by slot; one word a step that holds an event.
template <int C> constexpr int decay_powers() { return 16 + C + 4; }

template <int DP> constexpr int decay_stride() { return DP * 2 + 16; }   // bytes of an LDS row

template <int DP, int EW, int C> constexpr size_t decay_lds_bf16(bool state_only) {
  return (size_t)C * ((state_only ? 1 : 2) * decay_stride<DP>() + decay_stride<EW>()) +
         (state_only ? 0 : C * decay_stride<C>()) + (decay_powers<C>() + 2 * C) * 4;
}

__device__ __forceinline__ void mfma32(bf16x8 a, bf16x8 b, f32x4& c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  mfma_keep(c, a, b);
}

__device__ __forceinline__ bf16x8 lds_b128(const char* p) {
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(p));
}

// Fragment of M^T in slot order from a lane's base (decay_col_base): rows 8 g + 0 2 4 6 and
// + 1 3 5 7 of column c.  A 16-lane group of the transposing read takes 4 rows of 16
// columns, lane i of it row i / 4 from column 4 (i % 4) on, and receives column i.
template <int ST>
__device__ __forceinline__ int decay_col_base(int lane) {
  const int i = lane & 15;
  return (8 * (lane >> 4) + 2 * (i >> 2)) * ST + 8 * (i & 3);
}
template <int ST>
__device__ __forceinline__ bf16x8 lds_col8s(const char* p) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + ST));
  const bf16x4 l = __builtin_bit_cast(bf16x4, lo), h = __builtin_bit_cast(bf16x4, hi);
  return bf16x8{l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
}

// Fragment of a row in the state's order: columns 4 g + s and 16 + 4 g + s from p = column 4 g.
__device__ __forceinline__ bf16x8 lds_row_pair(const char* p) {
  const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + 32);
  return __builtin_bit_cast(bf16x8, make_uint4(a.x, a.y, b.x, b.y));
}

__device__ __forceinline__ bf16x8 pack8(const float* f) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (__bf16)f[i];
  return r;
}

// The row of the chunk that DP / 8 threads hold first: 16 neighbouring lanes write one row
// of 128 columns, or rows 8 (4) apart whose 16-byte pieces fall on different banks.
template <int DP>
__device__ __forceinline__ int decay_first_row() {
  const int q = (int)threadIdx.x / (DP / 8);
  if constexpr (DP == 128) return q;
  if constexpr (DP == 64) return (q & 1) * 8 + (q >> 1 & 7) + (q & ~15);
  return (q & 3) * 4 + (q >> 2 & 3) + (q & ~15);
}

// Rows of a chunk on their way from memory: thread t holds columns [8 (t % (DP / 8)), + 8) of
// its first row and of every R-th after it, R = threads / (DP / 8).  The chunk's lowest
// row is a uniform pointer, a lane's offset from it 32 bits (the host admits row strides
// below 2^24 elements).  Masked steps are loaded too (their row exists) and zeroed by
// selection when they are laid down: nothing waits for the mask before that (3 x 8191
// events, 8 heads of 64, a mask: 25.4 us -> 24.2).
template <int DP, int NTH, int C>
struct DecayRows {
  static constexpr int R = NTH / (DP / 8), N = C / R;
  static_assert(N * R == C, "whole turns");
  unsigned at[N];    // the row's place above the chunk's lowest
  bool inside[N];    // the step is one of the chunk's
  unsigned mask[N];  // its byte of key_valid, as it comes from memory
  int64_t low;       // the chunk's lowest row
  __device__ __forceinline__ void chunk(const DecayParams& p, const DecayPlace& w, int rev, int64_t base, bool masked,
                                        int t0) {
    const int n = w.t1 - t0 < C ? w.t1 - t0 : C;
    const int pos0 = rev ? p.seq_len - t0 - n : w.start + t0;
    low = base + pos0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int t = decay_first_row<DP>() + R * k, s = t < n ? t : n - 1;
      at[k] = rev ? n - 1 - s : s;
      inside[k] = t < n;
      mask[k] = 1;
    }
    if (masked) {
      const uint8_t* q = p.key_valid + (int64_t)w.b * p.seq_len + pos0;
#pragma unroll
      for (int k = 0; k < N; ++k) mask[k] = q[at[k]];
    }
  }
  __device__ __forceinline__ bool live(int k) const { return inside[k] && mask[k] != 0; }   // it holds an event
  __device__ __forceinline__ void load(uint4* f, const void* src, int64_t ld, int64_t col, int ccol) const {
    const char* q = reinterpret_cast<const char*>(src) + (low * ld + col) * 2;
#pragma unroll
    for (int k = 0; k < N; ++k)
      f[k] = *reinterpret_cast<const uint4*>(q + (at[k] * (unsigned)ld + (unsigned)ccol) * 2u);
  }
  __device__ __forceinline__ void store(const uint4* f, char* dst, bool has) const {
#pragma unroll
    for (int k = 0; k < N; ++k)
      *reinterpret_cast<uint4*>(dst + (decay_first_row<DP>() + R * k) * decay_stride<DP>() +
                                (int)threadIdx.x % (DP / 8) * 16) = live(k) && has ? f[k] : make_uint4(0u, 0u, 0u, 0u);
  }
};

// c + 0 * each element.
__device__ __forceinline__ float times_zero(bf16x8 v, float c) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 zero = {(__bf16)0.f, (__bf16)0.f};
#pragma unroll
  for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[i], v[i + 1]}, zero, c, false);
  return c;
}

// P V of a chunk with infinities or NaNs in V: a matrix product takes every step's V_j to
// every row, as 0 * V_j to the rows before j.  So they leave the fragments here, and are
// added to the outputs of the rows i >= j, one by one.  (Looking for them and selecting P
// instead of multiplying it by 0 costs 2 to 3 % of the kernel where there are none.)
template <int NE, int CK>
__device__ __forceinline__ void decay_odd_steps(bf16x8 (&vf)[NE][CK], f32x4 (&o)[2 * CK][NE], const char* sp, int lane) {
  constexpr int PS = decay_stride<32 * CK>();
  asm volatile("" : "+v"(lane));   // (else its addresses are kept in registers through every chunk)
  const int g = lane >> 4, c = lane & 15;
#pragma unroll
  for (int x = 0; x < NE; ++x)
    for (;;) {
      int at = -1;   // one of the lanes' 8 CK slots that has any
      float f = 0.f;
#pragma unroll
      for (int k = 0; k < 8 * CK; ++k) {
        const float y = (float)vf[x][k / 8][k % 8];
        if (__any(!decay_finite(y))) { at = k; f = y; }
      }
      if (at < 0) break;
#pragma unroll
      for (int k = 0; k < 8 * CK; ++k)
        if (k == at && !decay_finite(f)) vf[x][k / 8][k % 8] = (__bf16)0.f;
      for (uint64_t m = __ballot(!decay_finite(f)); m; m &= m - 1) {
        const int l = __builtin_ctzll(m), q = at & 7, col = l & 15;
        const int slot = (at & ~7) * 4 + 8 * (l >> 4) + q, j = slot - q + (q < 4 ? 2 * q : 2 * q - 7);
        const float v = __shfl(f, l);
#pragma unroll
        for (int it = 0; it < 2 * CK; ++it) {
          const float y = (float)*reinterpret_cast<const __bf16*>(sp + (16 * it + c) * PS + 2 * slot) * v;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (4 * g + k == col && 16 * it + c >= j) o[it][x][k] += y;
        }
      }
    }
}

// NS: bf16 parts of g^(n-1-j) v_j in the state's sum: 2 (16 bits; the state is rounded to
// bf16 only as an operand of the output) or, where the state is returned in fp32, 3 (all 24
// bits).  One part would cost 2 % (heads of 64) to 10 % (128) less time and put a third
// rounding of 2^-9 into every output: its distance from the exact one, normwise, was 0.0025
// with it, 0.0023 without, and 0.0017 for fp32 products rounded once.
// Waves a SIMD: 5 with heads of up to 64 (96 registers; gradients of 128 sequences of up to 201
// events, 8 heads of 64: 36 us, with 4 waves 37.5).
template <int DP, int EW, int NE, int C, int NS, bool STATE>
__global__ void __launch_bounds__(EW * 4 / NE, NE == 2 ? 2 : DP <= 64 ? 5 : 4) k_decay_bf16(DecayParams p) {
  constexpr int CK = C / 32, NT = DP / 16, KS = DP / 32, NW = EW / 16 / NE, NTH = NW * 64;
  constexpr int ST = decay_stride<DP>(), SE = decay_stride<EW>(), PS = decay_stride<C>();
  using Rows = DecayRows<DP, NTH, C>;    // of a and b
  using Cols = DecayRows<EW, NTH, C>;    // of c
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char* sb = lds;
  char* sc = sb + C * ST;
  char* sa = sc + C * SE;
  char* sp = sa + (STATE ? 0 : C * ST);
  float* pw = reinterpret_cast<float*>(sp + (STATE ? 0 : C * PS)) + 16;
  float* wv = pw - 16 + decay_powers<C>();
  int* slive = reinterpret_cast<int*>(wv + C);
  DecayPlace w = decay_place(p, DP / EW);
  if (!w.on || (STATE && !decay_state_used(p, w))) return;
  const DecayRole r = p.role[w.role];
  const int64_t bh = (int64_t)w.b * p.heads + w.h, hcol = (int64_t)w.h * p.head_dim;
  const int64_t base = w.base;
  if (base + w.start < 0 || base + p.seq_len > p.capacity) w.t1 = w.t0;   // rows that do not exist: no step
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  // (a range that grk_seq_ranges calls contiguous leaves nothing to mask)
  const bool masked = p.key_valid && !(p.seq_range && p.seq_range[3 * (int64_t)w.b + 1] == 1);
  const int rcol = (int)threadIdx.x % (DP / 8) * 8, ecol = w.part * EW + (int)threadIdx.x % (EW / 8) * 8;
  const bool has = rcol < p.head_dim, ehas = ecol < p.head_dim;   // this thread's columns when rows are moved
  const int et0 = w.part * (EW / 16) + NE * wave;                 // the wave's first column tile
  f32x4 st[NE][NT];
  float* frag = p.ws + (((int64_t)(w.role < 2 ? w.role : 1) * p.batch * p.heads + bh) * p.nseg + w.seg) * DP * DP;
  bool some = STATE || (p.nseg > 1 ? w.seg > 0 || p.state_in : p.state_in != nullptr);   // the state is not all 0
#pragma unroll
  for (int x = 0; x < NE; ++x) {
    const int et = et0 + x;
#pragma unroll
    for (int dt = 0; dt < NT; ++dt) {
      st[x][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (!STATE && p.nseg > 1) {
        if (w.role < 2) {
          st[x][dt] = *reinterpret_cast<const f32x4*>(frag + ((dt * NT + et) * 64 + lane) * 4);
        } else {   // the transpose of role 1's state, element by element
#pragma unroll
          for (int i = 0; i < 4; ++i) st[x][dt][i] = frag[((et * NT + dt) * 64 + (c >> 2) * 16 + 4 * g + i) * 4 + (c & 3)];
        }
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
  Cols cols;
  uint4 fa[Rows::N], fb[Rows::N], fc[Cols::N];
  auto fetch = [&](int t0) {
    rows.chunk(p, w, r.rev, base, masked, t0);
    rows.load(fb, r.b, r.ldb, hcol, has ? rcol : 0);
    if (!STATE) rows.load(fa, r.a, r.lda, hcol, has ? rcol : 0);
    if constexpr (EW == DP) {
      cols = rows;
    } else {
      cols.chunk(p, w, r.rev, base, masked, t0);
    }
    cols.load(fc, r.c, r.ldc, hcol, ehas ? ecol : 0);
  };
  if (w.t0 < w.t1) fetch(w.t0);
  if (!STATE)
    for (int n = threadIdx.x; n <= 16 + C; n += NTH) pw[n - 16] = n < 16 ? 0.f : p.scale * decay_pow(w.lg, n - 16);
  auto weights = [&](int n) {   // of a chunk of n steps, by slot
    for (int k = threadIdx.x; k < C; k += NTH) {
      const int q = k & 7, j = k - q + (q < 4 ? 2 * q : 2 * q - 7);
      wv[k] = j < n ? decay_pow(w.lg, n - 1 - j) : 0.f;
    }
  };
  weights(C);
  const float gc = decay_pow(w.lg, C);
  if constexpr (!STATE) {
    for (int n = threadIdx.x; n < C * PS / 16; n += NTH) reinterpret_cast<uint4*>(sp)[n] = make_uint4(0u, 0u, 0u, 0u);
    if (w.part == 0) decay_zero_rows<bf16_t>(p, w, r);
  }
  // The state's loads are waited for here, by a use that is none: left to its first use in the
  // loop, every chunk would wait there for the next chunk's rows as well (18.5 us, not 17.3).
#pragma unroll
  for (int x = 0; x < NE; ++x)
#pragma unroll
    for (int dt = 0; dt < NT; ++dt) asm volatile("" : "+v"(st[x][dt]));
  const int row_b = c * ST + 16 * g, col_b = decay_col_base<ST>(lane);   // this lane's LDS bases
  // A chunk: its rows to LDS | P, what the output takes from the state, the state's step |
  // the output.  Two barriers: behind the second one only P is read, so the next chunk's
  // rows may be laid down at once.
  for (int t0 = w.t0; t0 < w.t1; t0 += C) {
    const int n = w.t1 - t0 < C ? w.t1 - t0 : C;
    const bool last = t0 + C >= w.t1;
    rows.store(fb, sb, has);
    cols.store(fc, sc, ehas);
    if constexpr (!STATE) {
      rows.store(fa, sa, has);
      if (rcol == 0) {
#pragma unroll
        for (int k = 0; k < Rows::N; ++k) slive[decay_first_row<DP>() + Rows::R * k] = rows.live(k);
      }
    }
    const int64_t low = rows.low;
    __syncthreads();
    if (!last) fetch(t0 + C);
    if constexpr (!STATE) {
      // P^T, lower tiles; the tiles above the diagonal that a 32-deep step reads stay 0
      for (int tile = wave; tile < C / 16 * (C / 16 + 1) / 2; tile += NW) {
        const int it = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, jt = tile - it * (it + 1) / 2;
        const char* q = sa + 16 * it * ST + row_b;
        const char* k = sb + 16 * jt * ST + row_b;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) mfma32(lds_b128(k + 64 * ks), lds_b128(q + 64 * ks), x);
        const float* lag = pw + 16 * (it - jt) + c - 4 * g;
        x *= f32x4{lag[0], lag[-1], lag[-2], lag[-3]};
        const int ahead = 16 * (it - jt) + c - 4 * g;   // steps from j = 4 g to i
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ahead < i ? 0.f : x[i];   // (no product by 0: K_j may hold a NaN)
        const bf16x4 y = {(__bf16)x[0], (__bf16)x[2], (__bf16)x[1], (__bf16)x[3]};
        const uint2 z = __builtin_bit_cast(uint2, y);   // steps 0 2 | 1 3 of four
        char* dst = sp + (16 * it + c) * PS + (2 * jt + (g >> 1)) * 16 + 4 * (g & 1);
        *reinterpret_cast<unsigned*>(dst) = z.x;
        *reinterpret_cast<unsigned*>(dst + 8) = z.y;
      }
    }
    bf16x8 vf[NE][CK];
#pragma unroll
    for (int x = 0; x < NE; ++x)
#pragma unroll
      for (int ks = 0; ks < CK; ++ks) vf[x][ks] = lds_col8s<SE>(sc + decay_col_base<SE>(lane) + 32 * ks * SE + 32 * (NE * wave + x));
    f32x4 o[C / 16][NE];
    bool live[C / 16];
    if constexpr (!STATE) {
#pragma unroll
      for (int it = 0; it < C / 16; ++it) {
        live[it] = slive[16 * it + c];
      }
      if (some) {
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
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const bf16x8 q = lds_row_pair(sa + c * ST + 8 * g + 16 * it * ST + 64 * ks);
#pragma unroll
            for (int x = 0; x < NE; ++x) {
              if (ks == 0) o[it][x] = f32x4{0.f, 0.f, 0.f, 0.f};
              mfma32(sf[x][ks], q, o[it][x]);
            }
          }
          const float rise = pw[16 * it + c + 1];
#pragma unroll
          for (int x = 0; x < NE; ++x) o[it][x] *= rise;
        }
      } else {
#pragma unroll
        for (int it = 0; it < C / 16; ++it)
#pragma unroll
          for (int x = 0; x < NE; ++x) o[it][x] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
    if (STATE || !last || (p.nseg == 1 && p.state_out)) {   // (nothing reads the state behind the last chunk else)
      some = true;
      float gn = gc;
      if (n < C) {   // the last chunk only
        weights(n);
        __syncthreads();
        gn = decay_pow(w.lg, n);
      }
#pragma unroll
      for (int x = 0; x < NE; ++x)
#pragma unroll
        for (int dt = 0; dt < NT; ++dt) st[x][dt] *= gn;
#pragma unroll
      for (int ks = 0; ks < CK; ++ks) {
        bf16x8 part[NE][NS];
        const f32x4 w0 = *reinterpret_cast<const f32x4*>(wv + 32 * ks + 8 * g);
        const f32x4 w1 = *reinterpret_cast<const f32x4*>(wv + 32 * ks + 8 * g + 4);
#pragma unroll
        for (int x = 0; x < NE; ++x) {
          float f[8];
#pragma unroll
          for (int s = 0; s < 8; ++s) f[s] = (float)vf[x][ks][s] * (s < 4 ? w0[s & 3] : w1[s & 3]);
#pragma unroll
          for (int q = 0; q < NS; ++q) {
            uint4 y = __builtin_bit_cast(uint4, pack8(f));
            asm("" : "+v"(y.x), "+v"(y.y), "+v"(y.z), "+v"(y.w));   // (else the compiler rounds each again to subtract it)
            part[x][q] = __builtin_bit_cast(bf16x8, y);
            const unsigned u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int s = 0; s < 8; ++s) f[s] -= __uint_as_float(s & 1 ? u[s / 2] & 0xffff0000u : u[s / 2] << 16);
          }
        }
#pragma unroll
        for (int dt = 0; dt < NT; ++dt) {
          const bf16x8 k = lds_col8s<ST>(sb + col_b + 32 * ks * ST + 32 * dt);
#pragma unroll
          for (int q = NS - 1; q >= 0; --q)
#pragma unroll
            for (int x = 0; x < NE; ++x) mfma32(k, part[x][q], st[x][dt]);
        }
      }
    }
    bool odd = false;   // an infinity or a NaN in the wave's V: 0 times it is a NaN
    if constexpr (!STATE) {
      float z = 0.f;
#pragma unroll
      for (int x = 0; x < NE; ++x)
#pragma unroll
        for (int ks = 0; ks < CK; ++ks) z = times_zero(vf[x][ks], z);
      odd = __any(z != 0.f);
    }
    __syncthreads();
    if constexpr (!STATE) {
      if (__builtin_expect(odd, 0)) decay_odd_steps<NE, CK>(vf, o, sp, lane);
      char* out = reinterpret_cast<char*>(r.out) + (low * r.ldo + hcol) * 2;
#pragma unroll
      for (int it = 0; it < C / 16; ++it) {
#pragma unroll
        for (int ks = 0; ks <= it / 2; ++ks) {
          const bf16x8 y = lds_b128(sp + c * PS + 16 * g + 16 * it * PS + 64 * ks);
#pragma unroll
          for (int x = 0; x < NE; ++x) mfma32(vf[x][ks], y, o[it][x]);
        }
        const int t = 16 * it + c;
        if (t < n) {
          const unsigned at = (unsigned)(r.rev ? n - 1 - t : t) * (unsigned)r.ldo;
#pragma unroll
          for (int x = 0; x < NE; ++x) {
            const int e = 16 * (et0 + x) + 4 * g;
            const f32x4 v = o[it][x];
            const bf16x4 y = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
            const uint2 z = live[it] ? __builtin_bit_cast(uint2, y) : make_uint2(0u, 0u);
            if (e < p.head_dim) *reinterpret_cast<uint2*>(out + (at + (unsigned)e) * 2u) = z;
          }
        }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < NE; ++x)
#pragma unroll
    for (int dt = 0; dt < NT; ++dt) {
      const int et = et0 + x;
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

// Segment states are those of roles 0 and 1: role 2 (K, Q, dO) sums q dO^T where role 1
// (V, dO, Q) sums dO q^T.
template <int DP, int NE, int MC>
static int decay_bf16_run(const DecayParams& p, hipStream_t s) {
  const int64_t groups = ((int64_t)p.batch * p.heads * p.nseg + 7) / 8 * 8;
  auto launch = [&](auto ew, auto ne, auto ns, auto state, const DecayParams& q) -> int {
    constexpr int EW = decltype(ew)::value, E = decltype(ne)::value, NS = decltype(ns)::value;
    constexpr int C = decltype(state)::value ? kDecayChunk : MC;
    constexpr bool STATE = decltype(state)::value;
    constexpr size_t lds = decay_lds_bf16<DP, EW, C>(STATE);
    GRK_CHECK_HIP(ensure_dynamic_lds((const void*)k_decay_bf16<DP, EW, E, C, NS, STATE>, lds));
    const unsigned grid = (unsigned)(groups * (DP / EW) * q.roles);
    k_decay_bf16<DP, EW, E, C, NS, STATE><<<grid, EW * 4 / E, lds, s>>>(q);
    GRK_LAUNCH_CHECK();
    return GRK_OK;
  };
  typedef std::integral_constant<int, 1> one;
  typedef std::integral_constant<int, 2> two;
  typedef std::integral_constant<int, 3> three;
  typedef std::integral_constant<int, DP> whole;
  typedef std::integral_constant<int, NE> ne;
  typedef std::integral_constant<int, (DP < 64 ? DP : 64)> half;   // (of a head of 128)
  if (p.nseg > 1) {
    DecayParams q = p;
    q.roles = p.roles < 2 ? p.roles : 2;
    int rc = p.state_out ? launch(half{}, one{}, three{}, std::true_type{}, q)
                         : launch(half{}, one{}, two{}, std::true_type{}, q);
    if (rc || (rc = decay_scan_launch(q, DP, s))) return rc;
    return launch(whole{}, ne{}, two{}, std::false_type{}, p);
  }
  return p.state_out ? launch(whole{}, ne{}, three{}, std::false_type{}, p)
                     : launch(whole{}, ne{}, two{}, std::false_type{}, p);
}

// Whole 16-byte vectors: rows, strides and heads start on them (8 bytes for the output);
// 64 rows' offsets fit 32 bits.
bool decay_bf16_takes(const DecayParams& p) {
  bool ok = p.head_dim % 8 == 0;
  for (int i = 0; i < p.roles; ++i) {
    const DecayRole& r = p.role[i];
    ok = ok && ((uintptr_t)r.a | (uintptr_t)r.b | (uintptr_t)r.c) % 16 == 0 && (r.lda | r.ldb | r.ldc) % 8 == 0 &&
         (uintptr_t)r.out % 8 == 0 && r.ldo % 4 == 0 && (r.lda | r.ldb | r.ldc | r.ldo) < (1 << 24);
  }
  return ok;
}

// Chunks of 32 steps for heads of up to 64 columns (128 sequences of up to 201 events,
// 8 heads of 64: forward 19.6 us, with 64 steps 22.0), of 64 steps above (8 x 4096 events, 4
// heads of 128: gradients 91 us, with 32 steps and one tile a wave 95).  Two column tiles a
// wave halve what the waves read from LDS: taken where that bounds them, at 128 columns (the
// same 91 us, one tile 104); at 64 more waves hide more latency (the former's forward 17.3
// us, two tiles 19.2; its gradients 36 us with either).
int decay_bf16_launch(const DecayParams& p, hipStream_t s) {
  if (p.head_dim <= 32) return decay_bf16_run<32, 1, 32>(p, s);
  if (p.head_dim <= 64) return decay_bf16_run<64, 1, 32>(p, s);
  return decay_bf16_run<128, 2, 64>(p, s);
}

}  // namespace grk
