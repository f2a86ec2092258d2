// Shared pieces of the decayed linear attention kernels (gfx950).
//
//   S_t = g S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   g = exp(log_decay[h])
//
// In chunks of steps this is three products per chunk (i, j: steps of the chunk,
// n: its length, S: the state before it):
//   P_ij = [j <= i] g^(i-j) q_i . k_j,   o_i = scale (sum_j P_ij v_j + g^(i+1) q_i S),
//   S   <- g^n S + sum_j g^(n-1-j) k_j v_j^T.
// No power of g has a negative exponent, so decays near 0 (log_decay -inf: g = 0) neither
// overflow nor divide.
//
// The gradients are the same recurrence on other operands:
//   dq = f(dO, V, K);  dk = f(V, dO, Q) and dv = f(K, Q, dO) run from the last step back.
// A role is one such pass: (a, b, c) in the places of (q, k, v), and a direction.
#pragma once
#include "grk_vec.h"

namespace grk {

constexpr int kDecayChunk = 64;

struct DecayRole {
  const void* a; int64_t lda;
  const void* b; int64_t ldb;
  const void* c; int64_t ldc;
  void* out; int64_t ldo;
  int rev;
};

struct DecayParams {
  DecayRole role[3];
  int roles;
  int batch, heads, seq_len, head_dim;
  float scale;
  const float* log_decay;
  const uint8_t* key_valid;
  const int32_t* seq_range;
  const int64_t* row_base; const int64_t* num_rows;
  int64_t capacity;                // rows of every operand
  int nseg, seg_len;               // segments of a sequence, steps of one (whole chunks)
  const float* state_in; float* state_out;   // [batch, heads, head_dim, head_dim]
  float* ws;                       // segment states [role][batch, heads][segment][DP * DP], fragment order
};

// min(log g, 0); NaN stays (fminf would make it 0).
__device__ __forceinline__ float decay_log(float lg) { return lg > 0.f ? 0.f : lg; }

// One workgroup's pass: a role, a (sequence, head) and a segment of it.
struct DecayPlace {
  int b, h, seg, role, part;       // part: its columns of the state and the output, where they are shared out
  int64_t base;                    // row of position 0
  int start, len;                  // first position of the sequence, its steps
  int t0, t1;                      // steps of the segment
  float lg;                        // log g <= 0
  bool on;
};

// Workgroups of the roles and parts of one (sequence, head, segment) read the same rows: their
// indices differ by multiples of 8, so one XCD's L2 serves them (workgroups go round the
// 8 XCDs in order).
__device__ __forceinline__ DecayPlace decay_place(const DecayParams& p, int parts = 1) {
  DecayPlace w;
  const int64_t gid = blockIdx.x;
  const int same = p.roles * parts, k = (int)((gid / 8) % same);
  w.role = k % p.roles;
  w.part = k / p.roles;
  const int64_t u = gid / (8 * same) * 8 + gid % 8;
  w.on = u < (int64_t)p.batch * p.heads * p.nseg;
  const int64_t bh = w.on ? u / p.nseg : 0;
  w.seg = (int)(u - bh * p.nseg);
  w.b = (int)(bh / p.heads);
  w.h = (int)(bh - (int64_t)w.b * p.heads);
  if (p.seq_range) {   // the longest sequences first: 128 of 50 to 201 events, forward 19.8 -> 18.4 us
    const int by_length = p.seq_range[3 * (int64_t)w.b + 2];
    if ((unsigned)by_length < (unsigned)p.batch) w.b = by_length;
  }
  w.base = p.row_base ? p.row_base[w.b] : (int64_t)w.b * p.seq_len;
  int s = p.seq_range ? p.seq_range[3 * (int64_t)w.b] : 0;
  w.start = s < 0 ? 0 : (s > p.seq_len ? p.seq_len : s);
  w.len = p.seq_len - w.start;
  w.t0 = w.seg * p.seg_len;
  w.t1 = w.t0 + p.seg_len < w.len ? w.t0 + p.seg_len : w.len;
  w.lg = decay_log(p.log_decay[w.h]);
  return w;
}

// Whether a later segment, or state_out, takes this one's sums (the workspace of the others is
// never written, and the scan's sums with it are never used).
__device__ __forceinline__ bool decay_state_used(const DecayParams& p, const DecayPlace& w) {
  return p.state_out || w.t0 + p.seg_len < w.len;
}

// g^n for n >= 0 (g^0 = 1 also for g = 0).
__device__ __forceinline__ float decay_pow(float lg, int n) { return n == 0 ? 1.f : expf(lg * (float)n); }

__device__ __forceinline__ bool decay_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Row of step t, masked or not, or -1 past the segment (or where no row exists).
__device__ __forceinline__ int64_t decay_row(const DecayParams& p, const DecayPlace& w, int rev, int t) {
  if (t >= w.t1) return -1;
  const int pos = rev ? p.seq_len - 1 - t : w.start + t;
  const int64_t row = w.base + pos;
  return row >= 0 && row < p.capacity ? row : -1;
}

// Rows of the output that no step writes: a padded sequence's rows before its start, and
// the rows behind the last sequence of packed rows.  Spread over the segments' workgroups.
template <typename T>
__device__ __forceinline__ void decay_zero_rows(const DecayParams& p, const DecayPlace& w, const DecayRole& r) {
  int64_t first, last, step;
  if (p.row_base) {
    if (!p.num_rows) return;
    const int64_t n = *p.num_rows;
    first = (n < 0 ? 0 : n) + (int64_t)w.b * p.nseg + w.seg;
    last = p.capacity;
    step = (int64_t)p.batch * p.nseg;
  } else {
    first = (int64_t)w.b * p.seq_len + w.seg;
    last = (int64_t)w.b * p.seq_len + w.start;
    step = p.nseg;
  }
  for (int64_t row = first; row < last; row += step)
    for (int c = threadIdx.x; c < p.head_dim; c += blockDim.x)
      reinterpret_cast<T*>(r.out)[row * r.ldo + (int64_t)w.h * p.head_dim + c] = from_f32<T>(0.f);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

// Keeps an MFMA's sources alive past it, so that its result never takes their registers
// (the 16x16 forms' results are not tied to srcC by the compiler; make's overlap check
// rejects such code).  The statement holds no instruction: nothing reads the result early.
template <typename A, typename B>
__device__ __forceinline__ void mfma_keep(f32x4& acc, const A& a, const B& b) {
  asm("" : "+v"(acc) : "v"(a), "v"(b));
}

// host: the bf16 kernels (grk_decay_bf16.hip)
bool decay_bf16_takes(const DecayParams& p);
int decay_bf16_launch(const DecayParams& p, hipStream_t s);
// the segments' scan (grk_decay.hip), for states padded to dp
int decay_scan_launch(const DecayParams& p, int dp, hipStream_t s);

}  // namespace grk
