// linear_common.cuh — what the kernels of linear attention with a decay per head share: one operator with roles, the
// geometry of sequences and segments, and the state slots of a pool.
//
// With lam = exp(min(log_decay, 0)) per state (kv head), every product of the forward and the backward is the same
// operator over tokens, in one direction or the other:
//     out_i = w_intra sum_j lam^|i-j| (a_i . b_j) c_j + w_inter lam^n_i X^T a_i      (j <= i, or j >= i reversed)
//     X'    = lam^C X + w_up sum_j lam^m_j b_j c_j^T                                   over a chunk of C tokens
// where X is the state that enters the chunk; i counts from the chunk's start:
//     forward  : n_i = i + 1,     m_j = C - 1 - j,   w_intra = w_inter = scale, w_up = 1
//     reversed : n_i = C - 1 - i, m_j = j + 1,       w_intra = w_up = scale,    w_inter = 1
//   out   a   b   c   state X       direction
//   o     q   k   v   S             forward
//   dq    dO  v   k   S^T           forward
//   dk    v   dO  q   R^T           reversed
//   dv    k   q   dO  R             reversed
// A sequence is cut into segments of seg_len tokens.  Where there is more than one, the segments' own sums are formed
// side by side (state kernel), joined in order by a small kernel, and each segment's outputs then start from its own state.
#pragma once
#include "fa_common.cuh"

namespace fa {

constexpr int LIN_ERR_SLOT = 1;     // a slot outside the pool, or named twice
constexpr int LIN_ERR_WAIT = 2;     // a pipeline wait gave up
constexpr int LIN_NONE = -1;

struct LinSeqs {
  const int* cu;
  const float* log_decay;
  long long total;
  int batch, S, nhk, seg_len, nseg;
  int slots;             // segments of all sequences (lin_slots): the states' workspace is [slots][nhk][da dc]
};

// Segments have slots: nseg for each dense sequence, and for packed ones, whatever their lengths, floor(total / seg_len) + batch, the first of
// sequence z being floor(row0 / seg_len) + z (floor(x + y) + 1 >= floor(x) + ceil(y), so they do not meet); one sequence alone needs no
// more than it has (32 empty blocks among 160 left the others on crowded SMs: 170 us, not 142).  nseg 1: one segment a sequence, of
// any length.
inline long long lin_slots(bool packed, long long total, int batch, int seg_len, int nseg) {
  return nseg == 1 ? batch : packed ? (batch == 1 ? (total + seg_len - 1) / seg_len : total / seg_len + batch) : (long long)batch * nseg;
}

// the states that sequences start from and leave
struct LinPool {
  const float* in;
  float* out;
  const int* index;
  const int* seen;
  long long slots;
};

struct LinRole {
  const void *a, *b, *c;
  void* out;
  FaStrides sa, sb, sc, so;
  int na, nb;            // heads of a (and out), and of b and c, that belong to one state; one of them is 1
  int da, dc;            // dims of a and b, of c and out
  int transposed;        // X[i][j] is stored at [j][i]
  float w_intra, w_inter, w_up;
  float x_in = 1.f;      // the tensor-core kernel holds the state times this, and w_inter and w_up with it
};

struct LinSpan {
  long long row0;        // first row (packed rows), or 0
  int len;               // tokens of the sequence
};

__host__ __device__ __forceinline__ LinSpan lin_span(const LinSeqs& q, int z) {
  LinSpan s{0, q.S};
  if (q.cu) {
    const long long lo = min(max((long long)q.cu[z], 0ll), q.total);
    const long long hi = min(max((long long)q.cu[z + 1], lo), q.total);
    s.row0 = lo;
    s.len = (int)(hi - lo);
  }
  return s;
}
__host__ __device__ __forceinline__ long long lin_first_slot(const LinSeqs& q, int z, long long row0) {
  return q.nseg == 1 ? z : q.cu ? row0 / q.seg_len + z : (long long)z * q.nseg;
}
// an empty sequence has none, and its first slot may be the one past the last
__host__ __device__ __forceinline__ int lin_segments(const LinSeqs& q, int len) {
  return len <= 0 ? 0 : q.nseg == 1 ? 1 : (int)(((long long)len + q.seg_len - 1) / q.seg_len);
}
// the sequence of a slot and its tokens [t0, t1); t0 == t1 where the slot has none
__host__ __device__ __forceinline__ LinSpan lin_segment(const LinSeqs& q, int slot, int& z, int& t0, int& t1) {
  z = q.nseg == 1 ? slot : slot / q.nseg;
  if (q.nseg > 1 && q.cu) {
    int hi = q.batch;                      // the last sequence whose first slot is not past this one
    z = 0;
    while (hi - z > 1) {
      const int mid = (z + hi) / 2;
      if (lin_first_slot(q, mid, min(max((long long)q.cu[mid], 0ll), q.total)) <= slot) z = mid;
      else hi = mid;
    }
  }
  const LinSpan s = lin_span(q, z);
  const long long n = slot - lin_first_slot(q, z, s.row0);
  t0 = q.nseg == 1 ? 0 : (int)min(max(n, 0ll) * q.seg_len, (long long)s.len);
  t1 = q.nseg == 1 ? s.len : n < 0 ? t0 : (int)min((long long)t0 + q.seg_len, (long long)s.len);
  return s;
}
__device__ __forceinline__ float lin_log2_decay(const float* log_decay, int h) {
  const float g = log_decay[h];
  return (g > 0.f ? 0.f : g < -1e30f ? -1e30f : g) * FA_LOG2E;     // -infinity would give NaN at a power of 0; a NaN stays one
}
// lam^n from log2(lam): accurate exp2 (tables of a chunk, a few values a thread)
__device__ __forceinline__ float lin_power(float g2, int n) { return exp2f(g2 * (float)n); }

// Slot of sequence z in the pool, or LIN_NONE: padding, outside the pool, or named by an earlier sequence too (the
// earlier one has it).  All threads of the block call it.
__device__ __forceinline__ int lin_slot(const LinPool& p, int z, int nthreads, int* error) {
  if (!p.index) return z;
  const int s = p.index[z];
  if (s < 0) return LIN_NONE;
  int bad = s >= p.slots;
  for (int i = threadIdx.x; i < z; i += nthreads) bad |= p.index[i] == s;
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0) atomicOr(error, LIN_ERR_SLOT);
  return bad ? LIN_NONE : s;
}

// Packed rows that belong to no sequence are 0: each of `parts` blocks of a head writes its share.
template <typename T>
__device__ void lin_zero_outside(const LinSeqs& q, const LinRole& r, int h0, int part, int parts, int nthreads) {
  if (!q.cu) return;
  T* out = (T*)r.out;
  const LinSpan end = lin_span(q, q.batch - 1);
  const long long first = lin_span(q, 0).row0, last = end.row0 + end.len;
  for (int side = 0; side < 2; ++side) {
    const long long r0 = side ? last : 0, r1 = side ? q.total : first;
    for (long long row = r0 + part; row < r1; row += parts)
      for (int e = threadIdx.x; e < r.na * r.dc; e += nthreads)
        out[row * r.so.s + (long long)(h0 + e / r.dc) * r.so.h + e % r.dc] = Elem<T>::from_f(0.f);
  }
}

// kernel families (host).  ws: the states that segments start from, joined already; null = one segment that starts from the
// pool and leaves its last state there.
int lin_simt_states(const LinSeqs& q, const LinRole& r, bool reversed, float* ws, int dtype, cudaStream_t st);
int lin_simt_main(const LinSeqs& q, const LinRole& r, bool reversed, const float* ws, const LinPool& pool, int dtype, cudaStream_t st);
int lin_tc_states(const LinSeqs& q, const LinRole& r, bool reversed, float* ws, int dtype, cudaStream_t st, bool* taken);
int lin_tc_main(const LinSeqs& q, const LinRole& r, bool reversed, const float* ws, const LinPool& pool, int dtype, cudaStream_t st,
                bool* taken);
bool lin_tc_takes(const LinSeqs& q, const LinRole& r, int dtype);
int lin_device_error(int clear);
int lin_tc_device_error(int clear);
}  // namespace fa
