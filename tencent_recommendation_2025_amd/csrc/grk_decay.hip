// Decayed linear attention for gfx950 (the formulas: grk_decay.h): the general kernel --
// fp32, bf16 or fp16 rows, any head_dim up to 128 -- on the fp32 matrix instruction, the
// segments' scan and the single-step kernel.
#include <type_traits>

#include "grk_decay.h"

namespace grk {

// grk_sort.hip
size_t sort_pairs_workspace(int64_t n);
int sort_pairs(unsigned* k0, unsigned long long* v0, unsigned* k1, unsigned long long* v1, int64_t n, int end_bit,
               void* ws, unsigned** kres, unsigned long long** vres, hipStream_t s, bool hist0_ready);

// ---------------------------------------------------------- general kernel --
// One workgroup walks a segment in chunks of 32 steps; wave w owns columns [16 w, 16 w + 16)
// of the state and of the output (head_dim padded to DP with zeros: DP / 16 waves), its
// 16-row tiles of the state in registers.  v_mfma_f32_16x16x4_f32: lane l = 16 g + c holds
// A[c][g], B[g][c] and D[4 g + i][c], i < 4 -- A and B alike, so exchanging them transposes
// D.  The four k of a 16-deep step are taken as 4 g + s (s = 0..3) instead of 4 s + g: then
// register s of a state tile S = K^T V is the operand of step s in O^T = S^T Q^T + V^T P^T,
// and the row-major operands are 16-byte LDS reads.  P^T and O^T come out with 4
// neighbouring columns of one row in a lane (vector stores).
//
// Bound: the fp32 matrix instruction (1/16 of bf16's rate): of a 64-wide head a step takes
// 16 K operations of the state and 6 K of its chunk -- 32 steps, not 64, keep the latter
// small and leave LDS for 5 workgroups a CU.  (33 x 101 events of 2 heads of 32 in fp32: 12 us
// forward, 12 us the gradients -- 66 and 198 workgroups of 4 chunks each, latency.  Rows
// enough for the card keep the instruction half busy: 80 x 204 events of 8 heads of 64, fp32 48
// us forward and 113 us the gradients, fp16 45 and 108.)
constexpr int kF32Chunk = 32;
constexpr int kF32Pad = 4;   // floats after each LDS row: rows 4 apart fall 16 banks apart

template <int DP> constexpr size_t decay_lds_f32(bool state_only) {
  return (size_t)((state_only ? 2 : 3) * kF32Chunk * (DP + kF32Pad) + (state_only ? 0 : kF32Chunk * (kF32Chunk + kF32Pad)) +
                  16 + kF32Chunk + 4 + 2 * kF32Chunk) * 4;
}

// 4 elements of a row (or one, V = 1) as they lie in memory.
template <typename T, int V> struct DecayRaw;
template <> struct DecayRaw<float, 4> { typedef uint4 type; };
template <> struct DecayRaw<bf16_t, 4> { typedef uint2 type; };
template <> struct DecayRaw<f16_t, 4> { typedef uint2 type; };
template <typename T> struct DecayRaw<T, 1> { typedef T type; };

// A thread's part of a chunk on its way from memory: V columns of N rows.
template <typename T, int V, int DP>
struct DecayRowsF32 {
  typedef typename DecayRaw<T, V>::type raw;
  static constexpr int NTH = DP * 4, U = DP / V, R = NTH / U, N = kF32Chunk / R;
  int64_t row[N];    // -1: no step there
  bool inside[N];    // (whether there is: kept longer than row)
  unsigned mask[N];  // its byte of key_valid, as it comes from memory (looked at when the row is laid down)
  __device__ __forceinline__ void chunk(const DecayParams& p, const DecayPlace& w, int rev, int t0) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      row[k] = decay_row(p, w, rev, t0 + (int)threadIdx.x / U + R * k);
      inside[k] = row[k] >= 0;
      mask[k] = 1;
    }
    if (p.key_valid) {
      const uint8_t* q = p.key_valid + (int64_t)w.b * p.seq_len;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        int t = t0 + (int)threadIdx.x / U + R * k;
        t = t < w.t1 ? t : w.t1 - 1;
        mask[k] = q[rev ? p.seq_len - 1 - t : w.start + t];
      }
    }
  }
  __device__ __forceinline__ bool live(int k) const { return inside[k] && mask[k] != 0; }   // it holds an event
  __device__ __forceinline__ void load(raw* f, const void* src, int64_t ld, int64_t hcol, int head_dim) const {
    const int c = (int)threadIdx.x % U * V;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      f[k] = raw{};
      if (row[k] >= 0 && c < head_dim)
        f[k] = *reinterpret_cast<const raw*>(reinterpret_cast<const T*>(src) + row[k] * ld + hcol + c);
    }
  }
  __device__ __forceinline__ void store(const raw* f, float* dst) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const raw z = live(k) ? f[k] : raw{};
      T t[V];
      __builtin_memcpy(t, &z, sizeof(raw));
      float* d = dst + ((int)threadIdx.x / U + R * k) * (DP + kF32Pad) + (int)threadIdx.x % U * V;
      if constexpr (V == 4) *reinterpret_cast<float4*>(d) = make_float4(to_f32(t[0]), to_f32(t[1]), to_f32(t[2]), to_f32(t[3]));
      else *d = to_f32(t[0]);
    }
  }
};

// c += A B over 16 of the contraction: step s takes element s of both.
__device__ __forceinline__ void mfma16(f32x4 a, f32x4 b, f32x4& c) {
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
  mfma_keep(c, a, b);
}

// P V of a chunk with infinities or NaNs in V (grk_decay_bf16.hip): they leave the operand,
// and are added to the outputs of the rows i >= j, one by one.
template <int PT>
__device__ __forceinline__ void decay_odd_steps(f32x4 (&v)[2], f32x4 (&o)[2], const float* sp, int lane) {
  asm volatile("" : "+v"(lane));   // (its addresses are not kept through the chunks)
  const int g = lane >> 4, c = lane & 15;
#pragma unroll
  for (int at = 0; at < 8; ++at) {
    const float f = v[at / 4][at % 4];
    if (!decay_finite(f)) v[at / 4][at % 4] = 0.f;
    for (uint64_t m = __ballot(!decay_finite(f)); m; m &= m - 1) {
      const int l = __builtin_ctzll(m), j = 16 * (at / 4) + 4 * (l >> 4) + at % 4, col = l & 15;
      const float x = __shfl(f, l);
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        const float y = sp[(16 * it + c) * PT + j] * x;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (4 * g + k == col && 16 * it + c >= j) o[it][k] += y;
      }
    }
  }
}

template <typename T, int V, int DP, bool STATE>
__global__ void __launch_bounds__(DP * 4, 4) k_decay_f32(DecayParams p) {
  constexpr int C = kF32Chunk, ST = DP + kF32Pad, PT = C + kF32Pad, NT = DP / 16, NTH = DP * 4;
  using Rows = DecayRowsF32<T, V, DP>;
  extern __shared__ __attribute__((aligned(16))) float sm[];
  float* sb = sm;
  float* sc = sb + C * ST;
  float* sa = sc + C * ST;
  float* sp = sa + (STATE ? 0 : C * ST);
  float* pw = sp + (STATE ? 0 : C * PT) + 16;   // scale g^n, 0 <= n <= C; 0 for -16 < n < 0
  float* wv = pw - 16 + 16 + C + 4;             // g^(n-1-j): the weight of step j in the state
  int* slive = reinterpret_cast<int*>(wv + C);  // the step holds an event
  const DecayPlace w = decay_place(p);
  if (!w.on || (STATE && !decay_state_used(p, w))) return;
  const DecayRole r = p.role[w.role];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t bh = (int64_t)w.b * p.heads + w.h, hcol = (int64_t)w.h * p.head_dim;
  const int col = 16 * wave + c;   // the state column of this lane
  f32x4 st[NT];
  float* frag = p.ws + (((int64_t)w.role * p.batch * p.heads + bh) * p.nseg + w.seg) * DP * DP;
  bool some = STATE || (p.nseg > 1 ? w.seg > 0 || p.state_in : p.state_in != nullptr);   // the state is not all 0
#pragma unroll
  for (int dt = 0; dt < NT; ++dt) {
    st[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!STATE && p.nseg > 1) {
      st[dt] = *reinterpret_cast<const f32x4*>(frag + ((dt * NT + wave) * 64 + lane) * 4);
    } else if (!STATE && p.state_in) {
      const float f = decay_pow(w.lg, w.start);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 16 * dt + 4 * g + i;
        if (d < p.head_dim && col < p.head_dim)
          st[dt][i] = f * p.state_in[(bh * p.head_dim + d) * p.head_dim + col];
      }
    }
  }
  Rows rows;
  typename Rows::raw fa[Rows::N], fb[Rows::N], fc[Rows::N];
  if (w.t0 < w.t1) {
    rows.chunk(p, w, r.rev, w.t0);
    rows.load(fb, r.b, r.ldb, hcol, p.head_dim);
    rows.load(fc, r.c, r.ldc, hcol, p.head_dim);
    if (!STATE) rows.load(fa, r.a, r.lda, hcol, p.head_dim);
  }
  if (!STATE) {
    for (int n = threadIdx.x; n <= 16 + C; n += NTH) pw[n - 16] = n < 16 ? 0.f : p.scale * decay_pow(w.lg, n - 16);
    decay_zero_rows<T>(p, w, r);
  }
  auto weights = [&](int n) {
    for (int j = threadIdx.x; j < C; j += NTH) wv[j] = j < n ? decay_pow(w.lg, n - 1 - j) : 0.f;
  };
  weights(C);
  const float gc = decay_pow(w.lg, C);
  // (the state's loads are waited for before the loop: grk_decay_bf16.hip)
#pragma unroll
  for (int dt = 0; dt < NT; ++dt) asm volatile("" : "+v"(st[dt]));
  // A chunk: its rows to LDS | P, what the output takes from the state, the state's step |
  // the output.  Behind the second barrier only P (and V, kept in registers) is read.
  for (int t0 = w.t0; t0 < w.t1; t0 += C) {
    const int n = w.t1 - t0 < C ? w.t1 - t0 : C;
    const bool last = t0 + C >= w.t1;
    rows.store(fb, sb);
    rows.store(fc, sc);
    if constexpr (!STATE) {
      rows.store(fa, sa);
      if ((int)threadIdx.x % Rows::U == 0) {
#pragma unroll
        for (int k = 0; k < Rows::N; ++k) slive[(int)threadIdx.x / Rows::U + Rows::R * k] = rows.live(k);
      }
    }
    __syncthreads();
    if (!last) {
      rows.chunk(p, w, r.rev, t0 + C);
      rows.load(fb, r.b, r.ldb, hcol, p.head_dim);
      rows.load(fc, r.c, r.ldc, hcol, p.head_dim);
      if (!STATE) rows.load(fa, r.a, r.lda, hcol, p.head_dim);
    }
    if constexpr (!STATE) {
      for (int tile = wave; tile < 3; tile += NT) {   // P^T, tiles (0, 0), (1, 0), (1, 1)
        const int it = tile > 0, jt = tile > 1;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int dt = 0; dt < NT; ++dt)
          mfma16(*reinterpret_cast<const f32x4*>(sb + (16 * jt + c) * ST + 16 * dt + 4 * g),
                 *reinterpret_cast<const f32x4*>(sa + (16 * it + c) * ST + 16 * dt + 4 * g), x);
        const float* lag = pw + 16 * (it - jt) + c - 4 * g;
        x *= f32x4{lag[0], lag[-1], lag[-2], lag[-3]};
        const int ahead = 16 * (it - jt) + c - 4 * g;   // steps from j = 4 g to i
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ahead < i ? 0.f : x[i];   // (no product by 0: K_j may hold a NaN)
        *reinterpret_cast<f32x4*>(sp + (16 * it + c) * PT + 16 * jt + 4 * g) = x;
      }
    }
    f32x4 v[2];   // V[16 jt + 4 g + s][col]
#pragma unroll
    for (int jt = 0; jt < 2; ++jt) {
      const float* q = sc + (16 * jt + 4 * g) * ST + col;
      v[jt] = f32x4{q[0], q[ST], q[2 * ST], q[3 * ST]};
    }
    f32x4 o[2];
    bool live[2];
    if constexpr (!STATE) {
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        live[it] = slive[16 * it + c];
        o[it] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (some) {
#pragma unroll
          for (int dt = 0; dt < NT; ++dt)
            mfma16(st[dt], *reinterpret_cast<const f32x4*>(sa + (16 * it + c) * ST + 16 * dt + 4 * g), o[it]);
          o[it] *= pw[16 * it + c + 1];
        }
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
      for (int dt = 0; dt < NT; ++dt) st[dt] *= gn;
#pragma unroll
      for (int jt = 0; jt < 2; ++jt) {
        const f32x4 y = v[jt] * *reinterpret_cast<const f32x4*>(wv + 16 * jt + 4 * g);
#pragma unroll
        for (int dt = 0; dt < NT; ++dt) {
          const float* k = sb + (16 * jt + 4 * g) * ST + 16 * dt + c;
          mfma16(f32x4{k[0], k[ST], k[2 * ST], k[3 * ST]}, y, st[dt]);
        }
      }
    }
    const f32x4 sum = v[0] + v[1];   // not finite where an element is not (or the sum overflows)
    const bool odd = !STATE && __any(!decay_finite((sum[0] + sum[1]) + (sum[2] + sum[3])));
    __syncthreads();
    if constexpr (!STATE) {
      if (__builtin_expect(odd, 0)) decay_odd_steps<PT>(v, o, sp, lane);
#pragma unroll
      for (int it = 0; it < 2; ++it) {
#pragma unroll
        for (int jt = 0; jt <= it; ++jt)
          mfma16(v[jt], *reinterpret_cast<const f32x4*>(sp + (16 * it + c) * PT + 16 * jt + 4 * g), o[it]);
        const int64_t row = decay_row(p, w, r.rev, t0 + 16 * it + c);
        const int e = 16 * wave + 4 * g;
        if (row >= 0 && e < p.head_dim) {
          T* dst = reinterpret_cast<T*>(r.out) + row * r.ldo + hcol + e;
          T y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = from_f32<T>(live[it] ? o[it][i] : 0.f);
          if constexpr (V == 4) {
            typename Rows::raw z;
            __builtin_memcpy(&z, y, sizeof(z));
            *reinterpret_cast<typename Rows::raw*>(dst) = z;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (e + i < p.head_dim) dst[i] = y[i];
          }
        }
      }
    }
  }
  if (STATE) {
#pragma unroll
    for (int dt = 0; dt < NT; ++dt)
      *reinterpret_cast<f32x4*>(frag + ((dt * NT + wave) * 64 + lane) * 4) = st[dt];
  } else if (p.nseg == 1 && p.state_out) {
#pragma unroll
    for (int dt = 0; dt < NT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 16 * dt + 4 * g + i;
        if (d < p.head_dim && col < p.head_dim)
          p.state_out[(bh * p.head_dim + d) * p.head_dim + col] = st[dt][i];
      }
  }
}

// The segments' own states -> the state before each segment (and behind the last one):
// run <- g^len run + own, W elements of the state to a thread.  Few states are bound by the
// latency of their loads: one element a thread, the loads of U segments (8, 16 or 32, as
// there are) in flight at once (24 states of 64 x 64, 26 segments: 7.7 us; 4 elements and
// 8 loads 8.8).  Many are bound by memory: 4 elements, 8 loads (32 states of 128 x 128, 16
// segments: 7.5 us; one element 14.3).
template <int DP, int W, int U>
__global__ void __launch_bounds__(256) k_decay_scan(DecayParams p) {
  constexpr int NT = DP / 16, N = DP * DP / W;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;   // (role, b, h, elements in fragment order)
  const int f = (int)(i % N) * W;
  const int64_t rbh = i / N;
  if (rbh >= (int64_t)p.roles * p.batch * p.heads) return;
  const int64_t bh = rbh % ((int64_t)p.batch * p.heads);
  const int b = (int)(bh / p.heads), h = (int)(bh % p.heads);
  const int lane = f >> 2 & 63, tile = f >> 8, wave = tile & (NT - 1), dt = tile / NT;
  const int e = 16 * wave + (lane & 15), d0 = 16 * dt + 4 * (lane >> 4) + (f & 3);
  int start = p.seq_range ? p.seq_range[3 * (int64_t)b] : 0;
  start = start < 0 ? 0 : (start > p.seq_len ? p.seq_len : start);
  const int len = p.seq_len - start;
  const float lg = decay_log(p.log_decay[h]), gs = decay_pow(lg, p.seg_len);
  typedef float vec __attribute__((ext_vector_type(W)));
  vec run = 0.f;
  auto outside = [&](int k) { return (bh * p.head_dim + d0 + k) * p.head_dim + e; };   // in state_in / state_out
  auto has = [&](int k) { return d0 + k < p.head_dim && e < p.head_dim; };
  if (p.state_in) {
    const float g0 = decay_pow(lg, start);
#pragma unroll
    for (int k = 0; k < W; ++k)
      if (has(k)) run[k] = g0 * p.state_in[outside(k)];
  }
  vec* own = reinterpret_cast<vec*>(p.ws + rbh * p.nseg * DP * DP + f);
  for (int s0 = 0; s0 < p.nseg; s0 += U) {
    vec x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u < p.nseg ? s0 + u : p.nseg - 1;
      x[u] = own[(int64_t)s * N];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u, left = len - s * p.seg_len;   // steps from this segment on
      if (s < p.nseg) {
        own[(int64_t)s * N] = run;
        run = run * (left >= p.seg_len ? gs : decay_pow(lg, left < 0 ? 0 : left)) + x[u];
      }
    }
  }
  if (p.state_out) {
#pragma unroll
    for (int k = 0; k < W; ++k)
      if (has(k)) p.state_out[outside(k)] = run[k];
  }
}

// -------------------------------------------------------------- single step --
// One workgroup per (event, head): S <- g S + k v^T in place, o = scale q S.  The state
// is read and written once, in rows of `lanes` threads of V columns; a thread keeps its
// columns, so o is a sum over the thread rows in LDS.  Bound: memory, 8 head_dim^2 bytes
// of state per (event, head), with heads of 64 and more; narrow ones leave threads without a
// row (heads of 16: 192 of 256) and are bound by the workgroups' number.  States of 240 MB, read
// and written, part of them in the cache: heads of 128 49 us, 64 41, 32 62, 16 276.
constexpr int kStepThreads = 256;
// Events up to which every workgroup looks for its slot's others itself (a call of 8 heads of 64:
// 256 events 14.5 us, with links 17.5; 1024 events 54 and 55.5).
constexpr int kStepInline = 256;
// Events up to which every pair is compared (one launch); more are sorted by slot (8 launches).
// A call of 8192 events of one 16-wide head: 49 us with the pairs, 53 sorted; 12000: 79 and 63;
// 4096: 25 and 43.
constexpr int kStepPairs = 8192;

struct StepParams {
  const void* q; int64_t ldq;
  const void* k; int64_t ldk;
  const void* v; int64_t ldv;
  const float* log_decay;
  float* state; int64_t num_slots;
  const void* slots; int slots64;
  int differ;                    // no two events have one slot
  int64_t n;
  int heads, hd;
  float scale;
  int32_t* err;
  void* out; int64_t ldo;
  int32_t* links;                // [n, 2]: has an earlier event of its slot, the next one (or -1); or NULL
};

__device__ __forceinline__ int64_t step_slot(const StepParams& p, int64_t i) {
  if (!p.slots) return i;
  return p.slots64 ? reinterpret_cast<const int64_t*>(p.slots)[i]
                   : (int64_t)reinterpret_cast<const int32_t*>(p.slots)[i];
}

// Events of one slot are consecutive events of that user: the first one's workgroup
// takes them all, in order.  links[i] = (an earlier event has this slot, the next event
// that has it), by comparing every pair: 32 threads an event, a part of the others each.
constexpr int kLinkShare = 32;
__global__ void __launch_bounds__(kStepThreads) k_step_links(StepParams p) {
  __shared__ int64_t tile[kStepThreads];
  const int64_t i = (int64_t)blockIdx.x * (kStepThreads / kLinkShare) + threadIdx.x / kLinkShare;
  const int64_t mine = i < p.n ? step_slot(p, i) : -1;
  int before = 0;
  int next = 0x7fffffff;
  for (int64_t j0 = 0; j0 < p.n; j0 += kStepThreads) {
    __syncthreads();
    tile[threadIdx.x] = j0 + threadIdx.x < p.n ? step_slot(p, j0 + threadIdx.x) : -2;
    __syncthreads();
#pragma unroll 8
    for (int t = threadIdx.x % kLinkShare; t < kStepThreads; t += kLinkShare) {
      const int j = (int)j0 + t;
      const bool same = tile[t] == mine;
      before |= same && j < i;
      next = same && j > i && j < next ? j : next;
    }
  }
#pragma unroll
  for (int off = kLinkShare / 2; off > 0; off >>= 1) {
    before |= __shfl_xor(before, off);
    const int o = __shfl_xor(next, off);
    next = o < next ? o : next;
  }
  if (i < p.n && threadIdx.x % kLinkShare == 0) {
    p.links[2 * i] = before;
    p.links[2 * i + 1] = next == 0x7fffffff ? -1 : next;
  }
}

// The same links of many events, in linear time: their indices stably sorted by slot, each
// one's neighbours compared.  A key is 32 bits of the slot from `shift` on (a pool of 2^32
// states or more takes two sorts, the low bits first); slots outside the pool lie behind
// all others, so that they part no slot's events.  order: the events' indices so far, or NULL.
__global__ void __launch_bounds__(kStepThreads) k_step_keys(StepParams p, const unsigned long long* order, int shift,
                                                            unsigned* keys, unsigned long long* index) {
  const int64_t j = (int64_t)blockIdx.x * kStepThreads + threadIdx.x;
  if (j >= p.n) return;
  const int64_t i = order ? (int64_t)order[j] : j;
  int64_t s = step_slot(p, i);
  if (s < 0 || s > p.num_slots) s = p.num_slots;
  keys[j] = (unsigned)((uint64_t)s >> shift);
  index[j] = (unsigned long long)i;
}

__global__ void __launch_bounds__(kStepThreads) k_step_sorted_links(StepParams p, const unsigned long long* order) {
  const int64_t j = (int64_t)blockIdx.x * kStepThreads + threadIdx.x;
  if (j >= p.n) return;
  const int64_t i = (int64_t)order[j], slot = step_slot(p, i);
  p.links[2 * i] = j > 0 && step_slot(p, (int64_t)order[j - 1]) == slot;
  int next = -1;
  if (j + 1 < p.n && step_slot(p, (int64_t)order[j + 1]) == slot) next = (int)order[j + 1];
  p.links[2 * i + 1] = next;
}

// The states pass the caches by: each is touched once a call, and a pool is larger than they
// are (1024 events of 8 heads of 64, 268 MB: 57.3 -> 52.3 us, 5.1 TB/s, the rate of a large
// copy; fetching rows ahead of their turn, 4 to a thread, made it 64).
template <int V>
__device__ __forceinline__ void state_load(const float* p, float* s) {
  if constexpr (V == 4) {
    const f32x4 x = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = x[i];
  } else {
    s[0] = __builtin_nontemporal_load(p);
  }
}
template <int V>
__device__ __forceinline__ void state_store(float* p, const float* s) {
  if constexpr (V == 4) __builtin_nontemporal_store(f32x4{s[0], s[1], s[2], s[3]}, reinterpret_cast<f32x4*>(p));
  else __builtin_nontemporal_store(s[0], p);
}

template <typename T, int V>
__global__ void __launch_bounds__(kStepThreads) k_decay_step(StepParams p) {
  __shared__ float sq[128], sk[128], sv[128], red[kStepThreads * V];
  __shared__ int found[2];
  const int64_t i0 = blockIdx.x / p.heads;
  const int h = (int)(blockIdx.x % p.heads), hd = p.hd;
  const int lanes = hd / V, rows = kStepThreads / lanes;
  const int lr = threadIdx.x / lanes, e = threadIdx.x % lanes * V;
  const bool on = lr < rows;
  const int64_t slot = step_slot(p, i0);
  if (slot < 0 || slot >= p.num_slots) {
    if (slot >= 0 && p.err && threadIdx.x == 0) *p.err = 1;
    for (int c = threadIdx.x; c < hd; c += kStepThreads)
      reinterpret_cast<T*>(p.out)[i0 * p.ldo + (int64_t)h * hd + c] = from_f32<T>(0.f);
    return;
  }
  const float g = expf(decay_log(p.log_decay[h]));
  float* S = p.state + (slot * p.heads + h) * hd * hd;
  for (int64_t i = i0; i >= 0;) {
    // the slot's other events
    int64_t next = -1;
    if (p.slots && !p.differ) {
      if (p.links) {
        if (i == i0 && p.links[2 * i]) return;
        next = p.links[2 * i + 1];
      } else {
        if (threadIdx.x == 0) { found[0] = 0; found[1] = 0x7fffffff; }
        __syncthreads();
        for (int64_t j = threadIdx.x; j < p.n; j += kStepThreads)
          if (j != i && step_slot(p, j) == slot) {
            if (j < i) found[0] = 1;
            else atomicMin(&found[1], (int)j);
          }
        __syncthreads();
        const int first = found[0], nx = found[1];
        __syncthreads();
        if (i == i0 && first) return;
        next = nx == 0x7fffffff ? -1 : nx;
      }
    }
    const int64_t at = (int64_t)h * hd;
    for (int c = threadIdx.x; c < hd; c += kStepThreads) {
      sq[c] = to_f32(reinterpret_cast<const T*>(p.q)[i * p.ldq + at + c]);
      sk[c] = to_f32(reinterpret_cast<const T*>(p.k)[i * p.ldk + at + c]);
      sv[c] = to_f32(reinterpret_cast<const T*>(p.v)[i * p.ldv + at + c]);
    }
    __syncthreads();
    float o[V], v[V];
#pragma unroll
    for (int x = 0; x < V; ++x) { o[x] = 0.f; v[x] = on ? sv[e + x] : 0.f; }
    if (on)
#pragma unroll 4
      for (int d = lr; d < hd; d += rows) {
        float s[V];
        state_load<V>(S + d * hd + e, s);
        const float kd = sk[d], qd = sq[d];
#pragma unroll
        for (int x = 0; x < V; ++x) {
          s[x] = g * s[x] + kd * v[x];
          o[x] += qd * s[x];
        }
        state_store<V>(S + d * hd + e, s);
      }
#pragma unroll
    for (int x = 0; x < V; ++x)
      if (on) red[lr * hd + e + x] = o[x];
    __syncthreads();
    for (int c = threadIdx.x; c < hd; c += kStepThreads) {
      float t = 0.f;
      for (int r = 0; r < rows; ++r) t += red[r * hd + c];
      reinterpret_cast<T*>(p.out)[i * p.ldo + at + c] = from_f32<T>(p.scale * t);
    }
    __syncthreads();
    i = next;
  }
}

// ------------------------------------------------------------------ launch --
int decay_scan_launch(const DecayParams& p, int dp, hipStream_t s) {
  const int64_t n = (int64_t)p.roles * p.batch * p.heads * dp * dp;
  auto run = [&](auto w) {
    constexpr int DP = decltype(w)::value;
    const unsigned one = (unsigned)((n + 255) / 256), four = (unsigned)((n / 4 + 255) / 256);
    if (n >= 1 << 18) k_decay_scan<DP, 4, 8><<<four, 256, 0, s>>>(p);
    else if (p.nseg <= 8) k_decay_scan<DP, 1, 8><<<one, 256, 0, s>>>(p);
    else if (p.nseg <= 16) k_decay_scan<DP, 1, 16><<<one, 256, 0, s>>>(p);
    else k_decay_scan<DP, 1, 32><<<one, 256, 0, s>>>(p);
  };
  if (dp == 16) run(std::integral_constant<int, 16>{});
  else if (dp == 32) run(std::integral_constant<int, 32>{});
  else if (dp == 64) run(std::integral_constant<int, 64>{});
  else run(std::integral_constant<int, 128>{});
  GRK_LAUNCH_CHECK();
  return GRK_OK;
}

static int decay_dp(int hd) { return hd <= 16 ? 16 : hd <= 32 ? 32 : hd <= 64 ? 64 : 128; }

// Segments: a workgroup walks a sequence alone where the (sequence, head) pairs already
// fill half the workgroups that run at once (4 a CU; 2 with heads wider than 64); else the
// sequence is cut into as many segments as fill them, of at least 4 chunks.  (A cut costs a
// second read of two operands and the traffic of its states: one round of longer
// segments beat two of shorter ones.)
static void decay_segments(DecayParams& p) {
  const int64_t units = (int64_t)p.roles * p.batch * p.heads, slots = p.head_dim > 64 ? 512 : 1024;
  int64_t nseg = 2 * units >= slots ? 1 : slots / (units > 0 ? units : 1);
  const int64_t most = p.seq_len / (4 * kDecayChunk);
  if (nseg > most) nseg = most;
  if (nseg < 1) nseg = 1;
  const int64_t chunks = (p.seq_len + kDecayChunk - 1) / kDecayChunk;
  const int64_t per = (chunks + nseg - 1) / nseg;
  p.seg_len = (int)((per < 1 ? 1 : per) * kDecayChunk);
  p.nseg = (int)((chunks + per - 1) / (per < 1 ? 1 : per));
  if (p.nseg < 1) p.nseg = 1;
}

static size_t decay_ws(const DecayParams& p) {
  if (p.nseg <= 1) return 0;
  // (the bf16 kernels pad the narrowest heads to 32 columns)
  const size_t dp = p.head_dim <= 16 ? 32 : decay_dp(p.head_dim);
  return (size_t)p.roles * p.batch * p.heads * p.nseg * dp * dp * sizeof(float);
}

static int decay_check(const grk_decay_args* a) {
  GRK_CHECK_ARG(a, "args required");
  GRK_CHECK_ARG(known_dtype(a->dtype), "dtype must be fp32, bf16 or fp16");
  GRK_CHECK_ARG(a->batch >= 0 && a->heads > 0 && a->seq_len >= 0, "batch >= 0, heads > 0 and seq_len >= 0 required");
  if (a->head_dim < 1 || a->head_dim > 128) {
    set_error("head_dim must be in [1, 128]");
    return GRK_EUNSUPPORTED;
  }
  GRK_CHECK_ARG(a->batch > 0 || !a->row_base || a->capacity == 0, "packed rows without a sequence: capacity must be 0");
  GRK_CHECK_ARG((int64_t)a->batch * a->heads < (1 << 21) && a->seq_len < (1 << 30),
                "batch * heads must be below 2^21 and seq_len below 2^30");
  return GRK_OK;
}

static int decay_rows_ok(const void* q, int64_t ld, const grk_decay_args* a, int64_t capacity, const char* name) {
  GRK_CHECK_ARG(q, "%s required", name);
  GRK_CHECK_ARG(capacity == 1 ? ld >= 0 : ld >= (int64_t)a->heads * a->head_dim,
                "%s: row stride below heads * head_dim", name);
  return GRK_OK;
}

static void decay_params(const grk_decay_args* a, DecayParams& p) {
  memset(&p, 0, sizeof(p));
  p.batch = a->batch; p.heads = a->heads; p.seq_len = a->seq_len; p.head_dim = a->head_dim; p.scale = a->scale;
  p.log_decay = a->log_decay; p.key_valid = a->key_valid; p.seq_range = a->seq_range;
  p.row_base = a->row_base; p.num_rows = a->num_rows;
  p.capacity = a->row_base ? a->capacity : (int64_t)a->batch * a->seq_len;
}

template <typename T, int V, int DP>
static int decay_run(const DecayParams& p, hipStream_t s) {
  const int64_t groups = (int64_t)p.batch * p.heads * p.nseg;
  const unsigned grid = (unsigned)((groups + 7) / 8 * 8 * p.roles);
  if (p.nseg > 1) {
    constexpr size_t lds = decay_lds_f32<DP>(true);
    GRK_CHECK_HIP(ensure_dynamic_lds((const void*)k_decay_f32<T, V, DP, true>, lds));
    k_decay_f32<T, V, DP, true><<<grid, DP * 4, lds, s>>>(p);
    GRK_LAUNCH_CHECK();
    const int rc = decay_scan_launch(p, DP, s);
    if (rc) return rc;
  }
  constexpr size_t lds = decay_lds_f32<DP>(false);
  GRK_CHECK_HIP(ensure_dynamic_lds((const void*)k_decay_f32<T, V, DP, false>, lds));
  k_decay_f32<T, V, DP, false><<<grid, DP * 4, lds, s>>>(p);
  GRK_LAUNCH_CHECK();
  return GRK_OK;
}

static int decay_launch(const DecayParams& p, int dtype, hipStream_t s) {
  if (dtype == GRK_BF16 && decay_bf16_takes(p)) return decay_bf16_launch(p, s);
  // 8- or 16-byte accesses of 4 columns: rows and heads start on them
  bool vec = p.head_dim % 4 == 0;
  const size_t b4 = 4 * dtype_size(dtype);
  for (int r = 0; r < p.roles; ++r) {
    const DecayRole& x = p.role[r];
    vec = vec && ((uintptr_t)x.a | (uintptr_t)x.b | (uintptr_t)x.c | (uintptr_t)x.out) % b4 == 0 &&
          (x.lda | x.ldb | x.ldc | x.ldo) % 4 == 0;
  }
  return for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    switch (decay_dp(p.head_dim)) {
      case 16: return vec ? decay_run<T, 4, 16>(p, s) : decay_run<T, 1, 16>(p, s);
      case 32: return vec ? decay_run<T, 4, 32>(p, s) : decay_run<T, 1, 32>(p, s);
      case 64: return vec ? decay_run<T, 4, 64>(p, s) : decay_run<T, 1, 64>(p, s);
      default: return vec ? decay_run<T, 4, 128>(p, s) : decay_run<T, 1, 128>(p, s);
    }
  });
}

}  // namespace grk

using namespace grk;

extern "C" size_t grk_decay_attn_workspace(const grk_decay_args* a, int backward) {
  clear_error();
  if (decay_check(a)) return 0;
  DecayParams p;
  decay_params(a, p);
  p.roles = backward ? 3 : 1;
  decay_segments(p);
  return decay_ws(p);
}

extern "C" int grk_decay_attn_fwd(const grk_decay_args* a, const float* state_in, float* state_out, void* out,
                                  int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  int rc = decay_check(a);
  if (rc) return rc;
  if (a->batch == 0) return GRK_OK;
  DecayParams p;
  decay_params(a, p);
  if (p.capacity == 0 && !state_out) return GRK_OK;
  GRK_CHECK_ARG(a->log_decay, "log_decay required");
  GRK_CHECK_ARG(!a->row_base || (a->seq_range && a->capacity >= 0), "row_base needs seq_range and capacity >= 0");
  if (p.capacity > 0 &&
      ((rc = decay_rows_ok(a->q, a->ldq, a, p.capacity, "q")) || (rc = decay_rows_ok(a->k, a->ldk, a, p.capacity, "k")) ||
       (rc = decay_rows_ok(a->v, a->ldv, a, p.capacity, "v")) || (rc = decay_rows_ok(out, ldo, a, p.capacity, "out"))))
    return rc;
  p.roles = 1;
  p.role[0] = DecayRole{a->q, a->ldq, a->k, a->ldk, a->v, a->ldv, out, ldo, 0};
  p.state_in = state_in; p.state_out = state_out;
  decay_segments(p);
  GRK_CHECK_ARG(decay_ws(p) == 0 || (ws && ws_bytes >= decay_ws(p)), "workspace too small");
  p.ws = (float*)ws;
  return decay_launch(p, a->dtype, (hipStream_t)stream);
}

extern "C" int grk_decay_attn_bwd(const grk_decay_args* a, const void* dout, int64_t lddo, void* dq, int64_t lddq,
                                  void* dk, int64_t lddk, void* dv, int64_t lddv, void* ws, size_t ws_bytes,
                                  void* stream) {
  clear_error();
  int rc = decay_check(a);
  if (rc) return rc;
  DecayParams p;
  decay_params(a, p);
  if (a->batch == 0 || p.capacity == 0) return GRK_OK;
  GRK_CHECK_ARG(a->log_decay, "log_decay required");
  GRK_CHECK_ARG(!a->row_base || a->seq_range, "row_base needs seq_range");
  if ((rc = decay_rows_ok(a->q, a->ldq, a, p.capacity, "q")) || (rc = decay_rows_ok(a->k, a->ldk, a, p.capacity, "k")) ||
      (rc = decay_rows_ok(a->v, a->ldv, a, p.capacity, "v")) || (rc = decay_rows_ok(dout, lddo, a, p.capacity, "dout")) ||
      (rc = decay_rows_ok(dq, lddq, a, p.capacity, "dq")) || (rc = decay_rows_ok(dk, lddk, a, p.capacity, "dk")) ||
      (rc = decay_rows_ok(dv, lddv, a, p.capacity, "dv")))
    return rc;
  p.roles = 3;
  p.role[0] = DecayRole{dout, lddo, a->v, a->ldv, a->k, a->ldk, dq, lddq, 0};
  p.role[1] = DecayRole{a->v, a->ldv, dout, lddo, a->q, a->ldq, dk, lddk, 1};
  p.role[2] = DecayRole{a->k, a->ldk, a->q, a->ldq, dout, lddo, dv, lddv, 1};
  decay_segments(p);
  GRK_CHECK_ARG(decay_ws(p) == 0 || (ws && ws_bytes >= decay_ws(p)), "workspace too small");
  p.ws = (float*)ws;
  return decay_launch(p, a->dtype, (hipStream_t)stream);
}

// Behind the links, where the events are sorted: two buffers of indices, two of keys, the sort's own.
extern "C" size_t grk_decay_attn_step_workspace(int64_t n, int has_slots) {
  if (!has_slots || n <= kStepInline) return 0;
  return (size_t)n * 8 + (n > kStepPairs ? (size_t)n * 24 + sort_pairs_workspace(n) : 0);
}

static int step_sort_links(const StepParams& p, hipStream_t s) {
  unsigned long long* va = (unsigned long long*)(p.links + 2 * p.n);
  unsigned long long* vb = va + p.n;
  unsigned* ka = (unsigned*)(vb + p.n);
  unsigned* kb = ka + p.n;
  void* ws = kb + p.n;
  const unsigned grid = (unsigned)((p.n + kStepThreads - 1) / kStepThreads);
  const unsigned long long* order = nullptr;
  for (int shift = 0; shift < 64 && (shift == 0 || p.num_slots >> shift); shift += 32) {
    const unsigned top = p.num_slots >> shift > 0xffffffffll ? 0xffffffffu : (unsigned)(p.num_slots >> shift);
    int bits = 1;
    while (bits < 32 && top >> bits) ++bits;
    unsigned* keys;
    unsigned long long* sorted;
    unsigned long long* from = order == va ? vb : va;   // the indices so far are not overwritten
    unsigned long long* other = from == va ? vb : va;
    k_step_keys<<<grid, kStepThreads, 0, s>>>(p, order, shift, ka, from);
    GRK_LAUNCH_CHECK();
    const int rc = sort_pairs(ka, from, kb, other, p.n, bits, ws, &keys, &sorted, s, false);
    if (rc) return rc;
    order = sorted;
  }
  k_step_sorted_links<<<grid, kStepThreads, 0, s>>>(p, order);
  GRK_LAUNCH_CHECK();
  return GRK_OK;
}

extern "C" int grk_decay_attn_step(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                   int dtype, const float* log_decay, int64_t n, int heads, int head_dim, float scale,
                                   float* state, int64_t num_slots, const void* slots, int itype, int32_t* err_flag,
                                   void* out, int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  const bool differ = itype & GRK_SLOTS_DIFFER;
  itype &= ~GRK_SLOTS_DIFFER;
  GRK_CHECK_ARG(known_dtype(dtype), "dtype must be fp32, bf16 or fp16");
  GRK_CHECK_ARG(itype == GRK_I32 || itype == GRK_I64, "slots must be int32 or int64");
  GRK_CHECK_ARG(n >= 0 && heads > 0 && num_slots >= 0 && n < (1 << 24) &&
                n * heads < (1 << 24), "n >= 0, heads > 0, num_slots >= 0 and n * heads < 2^24 required");
  if (head_dim < 1 || head_dim > 128) {
    set_error("head_dim must be in [1, 128]");
    return GRK_EUNSUPPORTED;
  }
  if (n == 0) return GRK_OK;
  const int64_t cols = (int64_t)heads * head_dim;
  GRK_CHECK_ARG(q && k && v && log_decay && out && (state || num_slots == 0), "q / k / v / log_decay / state / out required");
  GRK_CHECK_ARG(n == 1 || (ldq >= cols && ldk >= cols && ldv >= cols && ldo >= cols),
                "row strides must be at least heads * head_dim");
  GRK_CHECK_ARG(slots || num_slots >= n, "without slots event i takes state i: num_slots must be at least n");
  const size_t need = grk_decay_attn_step_workspace(n, slots && !differ);
  GRK_CHECK_ARG(need == 0 || (ws && ws_bytes >= need), "workspace too small");
  GRK_CHECK_ARG(need == 0 || (uintptr_t)ws % 8 == 0, "workspace must be aligned to 8 bytes");
  StepParams p;
  memset(&p, 0, sizeof(p));
  p.q = q; p.ldq = ldq; p.k = k; p.ldk = ldk; p.v = v; p.ldv = ldv; p.log_decay = log_decay; p.state = state;
  p.num_slots = num_slots; p.slots = slots; p.slots64 = itype == GRK_I64; p.differ = differ; p.n = n;
  p.heads = heads; p.hd = head_dim; p.scale = scale; p.err = err_flag; p.out = out; p.ldo = ldo; p.links = need ? (int32_t*)ws : nullptr;
  hipStream_t s = (hipStream_t)stream;
  if (need && n > kStepPairs) {
    const int rc = step_sort_links(p, s);
    if (rc) return rc;
  } else if (need) {
    constexpr int per = kStepThreads / kLinkShare;
    k_step_links<<<(unsigned)((n + per - 1) / per), kStepThreads, 0, s>>>(p);
    GRK_LAUNCH_CHECK();
  }
  const unsigned grid = (unsigned)(n * heads);
  const bool vec = head_dim % 4 == 0 && (uintptr_t)state % 16 == 0;
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (vec) k_decay_step<T, 4><<<grid, kStepThreads, 0, s>>>(p);
    else k_decay_step<T, 1><<<grid, kStepThreads, 0, s>>>(p);
    return 0;
  });
  GRK_LAUNCH_CHECK();
  return GRK_OK;
}
