// kvcache.cu — writing to and reading back from paged caches (fa_kv_append_launch,
// fa_kv_gather_launch of fable_attn.h): new K/V rows are rotated and stored behind each
// sequence's cached tokens, as they are or in 8 bits with a scale for each block of slots and
// head; ranges of the caches come back as packed rows.
//
// All three are bound by the bytes they move.  The unit of work is 16 elements of a row as two groups of 8: for a
// rotated piece in NeoX order the groups are the two halves of 8 pairs, otherwise they are neighbours, so that
// a thread rotates what it loads.  Rows whose addresses or rotary size (no multiple of 16) do not allow 16-byte groups, and
// 8-bit pages of less than 16 slots, take the scalar kernels: 67k rows of 8 x 96 with 24 dims rotated 400 us against 81 with 32
// (fp16 caches), with blocks of 64 to int8 907 against 189 us (and read back); blocks of 8 in pages of 8 slots 1046 us, in pages of 16
// 213 us (8 x 128).
#include <algorithm>
#include <type_traits>
#include "fa_launch.h"
#include "kv8_common.cuh"

namespace {

using namespace fa_kv;

__device__ int g_kv_error = 0;
__device__ __forceinline__ void record(int bit) { atomicOr(&g_kv_error, bit); }

struct Turn {   // rotation of k
  const float *cos, *sin;
  int dim, rows, interleaved;
};

// element d of a row at table row `pos` (pos < 0: as it is): every product and the sum rounded in fp32
template <typename T>
__device__ __forceinline__ float turned(const T* x, int d, const Turn& r, int pos) {
  const float a = Elem<T>::to_f(x[d]);
  if (pos < 0 || d >= r.dim) return a;
  const int half = r.dim / 2;
  const bool low = r.interleaved ? !(d & 1) : d < half;
  const int j = r.interleaved ? d / 2 : d % half;
  const float b = Elem<T>::to_f(x[r.interleaved ? d ^ 1 : low ? d + half : d - half]);
  const float c = r.cos[(long long)pos * half + j], s = r.sin[(long long)pos * half + j];
  return low ? __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)) : __fadd_rn(__fmul_rn(a, c), __fmul_rn(b, s));
}

// table row of token i of sequence z, -1 for none
__device__ __forceinline__ int turn_pos(const FaKvAppendParams& p, int z, int i, bool is_k) {
  if (!is_k || !p.cos) return -1;
  const int pos = (p.rot_pos ? p.rot_pos[z] : p.ctx_len[z]) + i;
  if (pos >= 0 && pos < p.rot_seqlen_ro) return pos;
  record(ERR_ROTARY);
  return -1;
}

// one warp per (new row, head, K or V): caches of the inputs' kind
template <typename T, typename C>
__global__ void __launch_bounds__(128) append_kernel(const FaKvAppendParams p, const Pages pg) {
  pdl_wait();
  pdl_trigger();
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / 32, items = p.total * p.heads * 2;
  if (w >= items) return;
  const bool is_k = w % 2 == 0;
  const int h = (int)(w / 2 % p.heads);
  const long long row = w / 2 / p.heads;
  const RowMap rm{p.cu_new, p.tokens, p.batch};
  const int z = rm.seq_of_row(row), i = (int)(row - rm.first(z)), pos = p.ctx_len[z] + i;
  if (i < 0 || i >= rm.count(z, p.total)) return;   // a row of no sequence
  const long long blk = pg.of(z, pos);
  if (blk < 0) {
    record(ERR_PAGE);
    return;
  }
  const Turn r{p.cos, p.sin, p.rot_dim, p.rot_seqlen_ro, p.rot_interleaved};
  const int tp = turn_pos(p, z, i, is_k);
  const T* x = is_k ? (const T*)p.k + row * p.k_row + h * p.k_head : (const T*)p.v + row * p.v_row + h * p.v_head;
  C* out = (C*)(is_k ? p.Kc : p.Vc) + ((blk * p.page + (pos & (p.page - 1))) * p.heads + h) * p.dim;
  for (int d = threadIdx.x % 32; d < p.dim; d += 32) out[d] = Elem<C>::from_f(turned(x, d, r, tp));
}

// one warp per (scale block of a sequence, head, K or V)
template <typename T, typename Q>
__global__ void __launch_bounds__(128) append8_kernel(const FaKvAppendParams p, const Pages pg, const long long slots) {
  pdl_wait();
  pdl_trigger();
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  if (w >= slots * p.heads * 2) return;
  const int lane = threadIdx.x % 32;
  const bool is_k = w % 2 == 0;
  const int h = (int)(w / 2 % p.heads), SB = p.block, gs = log2_of(SB);
  const long long slot = w / 2 / p.heads;
  const RowMap rm{p.cu_new, p.tokens, p.batch};
  const int z = rm.seq_of_slot(slot, gs), n = rm.count(z, p.total), ctx = p.ctx_len[z];
  if (ctx < 0) {
    record(ERR_PAGE);
    return;
  }
  const int b0 = (int)((ctx >> gs) + slot - ((rm.first(z) >> gs) + 2 * z)) << gs;   // first position of the block
  const int a = max(ctx, b0), e = min(ctx + n, b0 + SB);
  if (a >= e) return;
  const long long blk = pg.of(z, b0);
  if (blk < 0) {
    record(ERR_PAGE);
    return;
  }
  const Turn r{p.cos, p.sin, p.rot_dim, p.rot_seqlen_ro, p.rot_interleaved};
  const long long in_page = b0 & (p.page - 1);
  typename Q::T* out = (typename Q::T*)(is_k ? p.Kc : p.Vc) + ((blk * p.page + in_page) * p.heads + h) * p.dim;
  const long long step = (long long)p.heads * p.dim;
  float* sc = (is_k ? p.Ks : p.Vs) + (blk * p.heads + h) * (p.page >> gs) + (in_page >> gs);
  auto row_of = [&](int pos) {
    const long long row = rm.first(z) + pos - ctx;
    return is_k ? (const T*)p.k + row * p.k_row + h * p.k_head : (const T*)p.v + row * p.v_row + h * p.v_head;
  };
  float most = 0.f;
  bool fine = true;
  for (int pos = a; pos < e; ++pos) {
    const int tp = turn_pos(p, z, pos - ctx, is_k);
    for (int d = lane; d < p.dim; d += 32) {
      const float x = fabsf(turned(row_of(pos), d, r, tp));
      fine &= x <= 3.402823466e38f;
      most = fmaxf(most, x);
    }
  }
  for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
  fine = __all_sync(~0u, fine);
  const float old = a > b0 ? *sc : 0.f;
  float s = fmaxf(__fmul_rn(most, 1.f / Q::QMAX), MIN_SCALE);
  if (old > s) s = old;
  const bool again = s > old && a > b0;
  if (!fine || isnan(old)) s = __int_as_float(0x7fc00000);
  const float inv = __frcp_rn(s);
  for (int pos = a; pos < e; ++pos) {
    const int tp = turn_pos(p, z, pos - ctx, is_k);
    for (int d = lane; d < p.dim; d += 32)
      out[(pos - b0) * step + d] = isnan(s) ? Q::from_f(0.f) : Q::from_f(__fmul_rn(turned(row_of(pos), d, r, tp), inv));
  }
  if (again && !isnan(s)) {
    const float ratio = __fdiv_rn(old, s);
    for (int pos = b0; pos < a; ++pos)
      for (int d = lane; d < p.dim; d += 32) {
        typename Q::T& c = out[(pos - b0) * step + d];
        c = Q::from_f(__fmul_rn(Q::to_f(c), ratio));
      }
  }
  __syncwarp();
  if (lane == 0) *sc = s;
}

// ---------------------------------------------------------------- groups of 8 elements
template <typename T>
struct Raw8 { uint4 u[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* x) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = __ldg(reinterpret_cast<const uint4*>(x) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ void to_float8(const Raw8<T>& r, float* v) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Elem<T>::to_f(e[i]);
}
template <typename T>
__device__ __forceinline__ void store_raw(T* x, const Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(x)[i] = r.u[i];
}
template <typename T>
__device__ __forceinline__ void store8(T* x, const float* v) {
  Raw8<T> r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = Elem<T>::from_f(v[i]);
  store_raw(x, r);
}
// Groups of unit u of a row: rotated NeoX pieces pair group 8 u with the one rot_dim / 2 further, all others their neighbour.
__device__ __forceinline__ void groups_of(int u, const Turn& r, bool is_k, int& d1, int& d2) {
  if (is_k && r.cos && !r.interleaved && 16 * u < r.dim) {
    d1 = 8 * u;
    d2 = d1 + r.dim / 2;
  } else {
    d1 = 16 * u;
    d2 = d1 + 8;
  }
}
__device__ __forceinline__ void turn2(float& x, float& y, float c, float s) {   // every product and the sum rounded in fp32
  const float lo = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s)), hi = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
  x = lo;
  y = hi;
}
// rotates a unit's groups v[0, 8) and v[8, 16) by table row tp
__device__ __forceinline__ void turn16(float* v, int u, const Turn& r, int tp) {
  const long long at = (long long)tp * (r.dim / 2) + 8 * u;
  const float4* ct = reinterpret_cast<const float4*>(r.cos + at);
  const float4* st = reinterpret_cast<const float4*>(r.sin + at);
  const float4 c0 = __ldg(ct), c1 = __ldg(ct + 1), s0 = __ldg(st), s1 = __ldg(st + 1);
  const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
  if (r.interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn2(v[2 * i], v[2 * i + 1], c[i], s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn2(v[i], v[8 + i], c[i], s[i]);
  }
}

// ---------------------------------------------------------------- append, caches of the inputs' type
// A CTA takes `rows` new rows of K or of V; where each goes stands in shared memory before its threads walk the rows' units.
// 67k fp16 rows of 8 x 128, rotated: 105 us, 5.4 TB/s (the floor is 89 us; a warp a row and head, element by element: 400 us).
// Left over is the latency of a CTA's own chain: sequence, page, rows.
constexpr int AT = 256, MAX_ROWS = 16;
template <typename T>
__global__ void __launch_bounds__(AT) append_vec_kernel(const FaKvAppendParams p, const Pages pg, const int rows, const Div per_row,
                                                        const Div per_head) {
  __shared__ long long s_slot[MAX_ROWS];   // cache row, -1: none
  __shared__ int s_turn[MAX_ROWS];
  pdl_wait();
  pdl_trigger();
  const long long row0 = (long long)blockIdx.x * rows;
  if (threadIdx.x < rows) {
    const long long row = row0 + threadIdx.x;
    const RowMap rm{p.cu_new, p.tokens, p.batch};
    long long slot = -1;
    int tp = -1;
    if (row < p.total) {
      const int z = rm.seq_of_row(row), i = (int)(row - rm.first(z)), pos = p.ctx_len[z] + i;
      if (i >= 0 && i < rm.count(z, p.total)) {   // else a row of no sequence
        const int blk = pg.of(z, pos);
        if (blk < 0) record(ERR_PAGE);
        else {
          slot = (long long)blk * p.page + (pos & (p.page - 1));
          tp = turn_pos(p, z, i, true);
        }
      }
    }
    s_slot[threadIdx.x] = slot;
    s_turn[threadIdx.x] = tp;
  }
  __syncthreads();
  const Turn r{p.cos, p.sin, p.rot_dim, p.rot_seqlen_ro, p.rot_interleaved};
  const bool is_k = blockIdx.y == 0;
  const T* const src = (const T*)(is_k ? p.k : p.v);
  T* const cache = (T*)(is_k ? p.Kc : p.Vc);
  const long long row_step = is_k ? p.k_row : p.v_row, head_step = is_k ? p.k_head : p.v_head;
#pragma unroll 4
  for (int e = threadIdx.x; e < rows * (int)per_row.d; e += AT) {
    const int i = per_row.of(e), w = e - i * per_row.d, h = per_head.of(w), u = w - h * per_head.d;
    const long long slot = s_slot[i];
    if (slot < 0) continue;
    const T* x = src + (row0 + i) * row_step + h * head_step;
    T* out = cache + (slot * p.heads + h) * p.dim;
    int d1, d2;
    groups_of(u, r, is_k, d1, d2);
    const Raw8<T> a = load8(x + d1), b = load8(x + d2);
    if (is_k && s_turn[i] >= 0 && 16 * u < r.dim) {
      float v[16];
      to_float8(a, v);
      to_float8(b, v + 8);
      turn16(v, u, r, s_turn[i]);
      store8(out + d1, v);
      store8(out + d2, v + 8);
    } else {
      store_raw(out + d1, a);
      store_raw(out + d2, b);
    }
  }
}

// ---------------------------------------------------------------- append, 8 bits
// codes of 8 values times inv, as 8 bytes
template <typename Q>
__device__ __forceinline__ uint2 codes8(const float* v, float inv) {
  uint2 out;
  uint32_t* o = &out.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* x = v + 4 * i;
    if constexpr (std::is_same<Q, I8>::value) {
      // 1.5 * 2^23 + y rounds y to a whole number, whose low byte is the code (|y| <= 127 after rounding)
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn(x[j], inv), 12582912.f));
      o[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[0], inv), __fmul_rn(x[1], inv)), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[2], inv), __fmul_rn(x[3], inv)), __NV_SATFINITE, __NV_E4M3);
      o[i] = lo | (hi << 16);
    }
  }
  return out;
}
template <typename Q>
__device__ __forceinline__ void values8(uint2 c, float* v) {
  const typename Q::T* e = reinterpret_cast<const typename Q::T*>(&c);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Q::to_f(e[i]);
}
// the larger; NaN where either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// A warp holds 16 positions (an aligned group, within one page) of one head of K or V in registers: LP lanes a row, each one
// unit, 32 / LP rows a pass.  The largest magnitude of a scale block comes from the row's lanes, then from the rows of the
// block: lanes, passes and, where a block has more than 16 slots, the block's warps.  One read of the new rows, one write of the
// codes; earlier codes of the first block are touched only where its scale grew.  The warps of a CTA take the heads of the
// same rows, which share their cos / sin rows in L1.  BIG: a block has 16 slots or more, so a warp has one scale.
// 67k bf16 rows of 8 x 128 to e4m3, rotated: 131 us, 3.1 TB/s (106 us unrotated; the floor is 64 us; element by element: 1.5 ms).
// Bound by the latency of warps that live for one group: a warp has 16 rows of loads under way, an SM 16 warps of 127
// registers, DRAM is at 36 %.  Keeping rows as loaded and rotating them twice for fewer registers: 158 us; several heads a
// warp: 193 us.
template <typename T, typename Q, int LP, bool BIG>
__global__ void __launch_bounds__(512, 1) append8_vec_kernel(const FaKvAppendParams p, const Pages pg, const long long slots) {
  constexpr int RPP = 32 / LP, PASS = 16 / RPP;
  constexpr bool KEEP = LP <= 8;                      // values stay in registers; rows of more than 128 are read again (from L1)
  constexpr int NB = BIG ? 1 : PASS;                  // scales of a thread
  __shared__ float s_most[16];
  pdl_wait();
  pdl_trigger();
  const int SB = p.block, bs = log2_of(SB), gs = BIG ? bs : 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ws = BIG ? bs - 4 : 0, in_block = warp & ((1 << ws) - 1);   // warps of a block; this one's place
  const int units = (int)(blockDim.x >> 5) >> ws;     // (slot, K or V, head) items of a CTA
  const unsigned item = blockIdx.x * units + (warp >> ws);
  const int h = (int)(item % (unsigned)p.heads);
  const bool is_k = ((item / (unsigned)p.heads) & 1) == 0;
  const long long slot = item / (unsigned)p.heads / 2;
  const RowMap rm{p.cu_new, p.tokens, p.batch};
  // ---- positions [c0, c0 + 16) of this warp; new tokens are [n0, n1)
  int z = 0, n0 = 0, n1 = 0, c0 = 0;
  long long row0 = 0;                                 // row of position 0, so to say
  if (slot < slots) {
    z = rm.seq_of_slot(slot, gs);
    n0 = p.ctx_len[z];
    if (n0 < 0) {
      record(ERR_PAGE);
      n0 = 0;
    } else {
      const long long first = rm.first(z);
      c0 = (int)(((n0 >> gs) + slot - ((first >> gs) + 2 * z)) << gs) + 16 * in_block;
      n1 = n0 + rm.count(z, p.total);
      row0 = first - n0;
    }
  }
  const int block0 = c0 & ~(SB - 1);                  // first position of the block (of the warp's first block)
  // new tokens in the warp's blocks (a sequence that has none may name pages that another one is appending to)
  bool any = n0 < n1 && block0 < n1 && max(c0 + 16, block0 + SB) > n0;
  const int blk = any ? pg.of(z, c0) : -1;
  if (any && blk < 0) record(ERR_PAGE);
  any = blk >= 0;

  const Turn r{p.cos, p.sin, p.rot_dim, p.rot_seqlen_ro, p.rot_interleaved};
  const int u = lane % LP, rp = lane / LP;            // unit; row of a pass
  const bool mine = any && u < p.dim / 16;
  int d1, d2;
  groups_of(u, r, is_k, d1, d2);
  const long long row_step = is_k ? p.k_row : p.v_row;
  const T* const src = (const T*)(is_k ? p.k : p.v) + (row0 + c0 + rp) * row_step + h * (is_k ? p.k_head : p.v_head);
  const bool turn = is_k && p.cos && 16 * u < r.dim;
  const int tp0 = turn && mine ? (p.rot_pos ? p.rot_pos[z] - n0 : 0) + c0 + rp : 0;   // table row of the first pass
  auto fresh = [&](int i) { const int pos = c0 + i * RPP + rp; return mine && pos >= n0 && pos < n1; };
  auto finish = [&](const Raw8<T>& a, const Raw8<T>& b, int i, float* v) {
    to_float8(a, v);
    to_float8(b, v + 8);
    if (turn) {
      const int tp = tp0 + i * RPP;
      if (tp >= 0 && tp < r.rows) turn16(v, u, r, tp);
      else record(ERR_ROTARY);
    }
  };
  float x[KEEP ? PASS : 1][16], most[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) most[i] = 0.f;
  if constexpr (KEEP) {
    Raw8<T> a[PASS], b[PASS];                         // all loads first
#pragma unroll
    for (int i = 0; i < PASS; ++i)
      if (fresh(i)) {
        a[i] = load8(src + i * RPP * row_step + d1);
        b[i] = load8(src + i * RPP * row_step + d2);
      }
#pragma unroll
    for (int i = 0; i < PASS; ++i)
      if (fresh(i)) {
        finish(a[i], b[i], i, x[i]);
        float& m = most[BIG ? 0 : i];
#pragma unroll
        for (int j = 0; j < 16; ++j) m = max_nan(m, fabsf(x[i][j]));
      }
  } else {
#pragma unroll
    for (int i = 0; i < PASS; ++i)
      if (fresh(i)) {
        finish(load8(src + i * RPP * row_step + d1), load8(src + i * RPP * row_step + d2), i, x[0]);
        float& m = most[BIG ? 0 : i];
#pragma unroll
        for (int j = 0; j < 16; ++j) m = max_nan(m, fabsf(x[0][j]));
      }
  }
  // ---- the blocks' largest: lanes of a row, rows of a pass, passes, warps
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
      if (BIG || o < LP * SB) most[i] = max_nan(most[i], __shfl_xor_sync(~0u, most[i], o));
  if constexpr (!BIG) {
#pragma unroll
    for (int o = 1; o < PASS; o <<= 1)
      if (o * RPP < SB) {
#pragma unroll
        for (int i = 0; i < PASS; ++i)
          if (!(i & o)) most[i] = most[i | o] = max_nan(most[i], most[i | o]);
      }
  } else if (ws) {
    if (lane == 0) s_most[warp] = most[0];
    __syncthreads();
    for (int w = 0; w < 1 << ws; ++w) most[0] = max_nan(most[0], s_most[(warp & ~((1 << ws) - 1)) + w]);
  }
  // ---- scales
  const int in_page = c0 & (p.page - 1);
  float* const sc = (is_k ? p.Ks : p.Vs) + ((long long)max(blk, 0) * p.heads + h) * (p.page >> bs);
  float s[NB], old[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int pos = c0 + i * RPP + rp, first = BIG ? block0 : pos & ~(SB - 1);
    const bool touched = any && first < n1 && first + SB > n0;
    old[i] = touched && first < n0 ? sc[(first & (p.page - 1)) >> bs] : 0.f;   // the block holds earlier tokens
    s[i] = fmaxf(fmaxf(__fmul_rn(most[i], 1.f / Q::QMAX), MIN_SCALE), old[i]);
    if (!(most[i] <= 3.402823466e38f) || isnan(old[i])) s[i] = __int_as_float(0x7fc00000);
    if (!touched) s[i] = -1.f;
  }
  // ---- codes
  const long long step = (long long)p.heads * p.dim;
  typename Q::T* const out = (typename Q::T*)(is_k ? p.Kc : p.Vc) + ((long long)max(blk, 0) * p.page + in_page + rp) * step + (long long)h * p.dim;
#pragma unroll
  for (int i = 0; i < PASS; ++i) {
    const int pos = c0 + i * RPP + rp;
    const float si = s[BIG ? 0 : i], was = old[BIG ? 0 : i];
    typename Q::T* const o = out + i * RPP * step;
    if (fresh(i)) {
      uint2 c1 = make_uint2(0, 0), c2 = c1;
      if (!isnan(si)) {
        const float inv = __frcp_rn(si);
        float* const v = x[KEEP ? i : 0];
        if constexpr (!KEEP) finish(load8(src + i * RPP * row_step + d1), load8(src + i * RPP * row_step + d2), i, v);
        c1 = codes8<Q>(v, inv);
        c2 = codes8<Q>(v + 8, inv);
      }
      *reinterpret_cast<uint2*>(o + d1) = c1;
      *reinterpret_cast<uint2*>(o + d2) = c2;
    } else if (mine && pos < n0 && was > 0.f && si > was) {   // earlier token: onto the scale that grew (never where it is NaN)
      const float ratio = __fdiv_rn(was, si);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint2* const at = reinterpret_cast<uint2*>(o + 16 * u + 8 * j);
        float v[8];
        values8<Q>(*at, v);
        *at = codes8<Q>(v, ratio);
      }
    }
  }
  // every reader of the old scale is done before the new one is written
  if (BIG && ws) __syncthreads();
  else __syncwarp();
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int pos = c0 + i * RPP + rp;
    if (s[i] == -1.f || (BIG ? lane != 0 || c0 != block0 : u != 0 || (pos & (SB - 1)) != 0)) continue;
    sc[(pos & (p.page - 1)) >> bs] = s[i];
  }
}

// ---------------------------------------------------------------- gather
// A CTA takes `rows` rows of K or of V; a thread makes 32 bytes of the output at a time (16 or 8 elements).
// 393k e4m3 rows of 8 x 128 to bf16: 365 us, 6.6 TB/s; what a copy of as many bytes takes (element by element: 4.2 ms).
constexpr int GT = 256;
struct __align__(32) Out32 { uint32_t u[8]; };
__device__ __forceinline__ void store32(void* o, const Out32& v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o), "r"(v.u[0]), "r"(v.u[1]), "r"(v.u[2]),
               "r"(v.u[3]), "r"(v.u[4]), "r"(v.u[5]), "r"(v.u[6]), "r"(v.u[7]) : "memory");
}
// values of 4 codes in a word, times s
template <typename Q>
__device__ __forceinline__ void values4(uint32_t w, float s, float* v) {
  if constexpr (std::is_same<Q, I8>::value) {
    const uint32_t x = w ^ 0x80808080u;   // c + 128 as the low byte of 2^23 + (c + 128)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(x, 0x4B000000u, 0x7440 + i)), 8388736.f), s);
  } else {
    uint32_t a, b;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(a), "=r"(b) : "r"(w));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a)), g = __half22float2(*reinterpret_cast<const __half2*>(&b));
    v[0] = __fmul_rn(f.x, s); v[1] = __fmul_rn(f.y, s); v[2] = __fmul_rn(g.x, s); v[3] = __fmul_rn(g.y, s);
  }
}
template <typename T, typename C, bool SCALED>
__global__ void __launch_bounds__(GT) gather_kernel(const FaKvGatherParams p, const Pages pg, const int rows, const Div per_row,
                                                    const Div per_head) {
  __shared__ long long s_slot[MAX_ROWS], s_scale[MAX_ROWS];   // cache row; scale of its head 0
  constexpr int N = 32 / sizeof(T);
  pdl_wait();
  pdl_trigger();
  const long long row0 = (long long)blockIdx.x * rows;
  const int bs = SCALED ? log2_of(p.block) : 0, per_page = p.page >> bs;
  if (threadIdx.x < rows) {
    const long long row = row0 + threadIdx.x;
    const RowMap rm{p.cu_k, 0, p.batch};
    long long slot = -1, sc = 0;
    if (row < p.total) {
      const int z = rm.seq_of_row(row), i = (int)(row - rm.first(z));
      if (i >= 0 && i < rm.count(z, p.total)) {   // else a row of no sequence
        const int pos = i + (p.starts ? p.starts[z] : 0), blk = pg.of(z, pos);
        if (blk < 0) record(ERR_PAGE);
        else {
          const int in_page = pos & (p.page - 1);
          slot = (long long)blk * p.page + in_page;
          sc = (long long)blk * p.heads * per_page + (in_page >> bs);
        }
      }
    }
    s_slot[threadIdx.x] = slot;
    s_scale[threadIdx.x] = sc;
  }
  __syncthreads();
  const int n = (int)min((long long)rows, p.total - row0) * per_row.d;
  const bool is_v = blockIdx.y;
  const void* const cache = is_v ? p.Vc : p.Kc;
  const float* const scales = is_v ? p.Vs : p.Ks;
  T* const out = (T*)(is_v ? p.v : p.k) + row0 * p.heads * p.dim;
#pragma unroll 4
  for (int e = threadIdx.x; e < n; e += GT) {
    const int i = per_row.of(e), w = e - i * per_row.d;
    const long long slot = s_slot[i], at = slot * p.heads * p.dim + w * N;
    Out32 o = {};
    T* const t = reinterpret_cast<T*>(&o);
    if (slot >= 0) {
      if constexpr (std::is_same<T, C>::value) {
        const uint4* x = reinterpret_cast<const uint4*>((const C*)cache + at);
        reinterpret_cast<uint4*>(&o)[0] = __ldg(x);
        reinterpret_cast<uint4*>(&o)[1] = __ldg(x + 1);
      } else {
        float v[N];
        if constexpr (SCALED) {
          const float s = __ldg(scales + s_scale[i] + per_head.of(w) * per_page);
          uint32_t c[N / 4];
          if constexpr (N == 16) *reinterpret_cast<uint4*>(c) = __ldg(reinterpret_cast<const uint4*>((const unsigned char*)cache + at));
          else *reinterpret_cast<uint2*>(c) = __ldg(reinterpret_cast<const uint2*>((const unsigned char*)cache + at));
#pragma unroll
          for (int j = 0; j < N / 4; ++j) values4<C>(c[j], s, v + 4 * j);
        } else {
#pragma unroll
          for (int j = 0; j < N; j += 8) to_float8(load8((const C*)cache + at + j), v + j);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) t[j] = Elem<T>::from_f(v[j]);
      }
    }
    store32(out + (long long)e * N, o);
  }
}

// rows of a CTA: as many as leave every SM two CTAs.  A call of few rows spreads over the SMs, one of many finds its rows'
// pages once for 16.
int rows_of_cta(long long total, int most) {
  int r = most;
  while (r > 1 && (total + r - 1) / r < 2 * fa::num_sms()) r /= 2;
  return r;
}

template <typename P>
bool cache_ok(const P& p, const char* who) {
  if (!(p.page > 0 && (p.page & (p.page - 1)) == 0 && p.max_blocks > 0 && p.num_blocks > 0)) {
    fa::set_error("%s: page=%d must be a power of two, max_blocks=%d and num_blocks=%lld positive", who, p.page,
                  p.max_blocks, p.num_blocks);
    return false;
  }
  if (!(p.batch >= 0 && p.heads > 0 && p.heads <= 256)) {
    fa::set_error("%s: batch=%d heads=%d (up to 256)", who, p.batch, p.heads);
    return false;
  }
  const bool scaled = p.code == FA_CODE_I8 || p.code == FA_CODE_E4M3;
  if (!scaled && p.code != FA_DTYPE_F16 && p.code != FA_DTYPE_BF16 && p.code != FA_DTYPE_F32) {
    fa::set_error("%s: cache element code %d", who, p.code);
    return false;
  }
  if (scaled != (p.Ks != nullptr) || scaled != (p.Vs != nullptr)) {
    fa::set_error("%s: Ks and Vs go with int8 and e4m3 caches, and only with them", who);
    return false;
  }
  if (scaled && !(p.block > 0 && (p.block & (p.block - 1)) == 0 && p.block <= p.page && p.block <= 256)) {
    fa::set_error("%s: block=%d must be a power of two, at most page=%d and 256", who, p.block, p.page);
    return false;
  }
  return true;
}
bool float_code(int c) { return c == FA_DTYPE_F16 || c == FA_DTYPE_BF16 || c == FA_DTYPE_F32; }
bool dim_ok(int d, const char* who) {
  if (d > 0 && d % 16 == 0 && d <= 256) return true;
  fa::set_error("%s: dim=%d must be a multiple of 16 up to 256", who, d);
  return false;
}
template <typename P>
Pages pages_of(const P& p) {
  return Pages{p.block_table, log2_of(p.page), p.max_blocks, p.num_blocks};
}

template <typename T, typename Q>
cudaError_t append8(const FaKvAppendParams& p, const Pages& pg, bool vec, cudaStream_t st) {
  if (!vec || p.page < 16) {
    const long long slots = p.total / p.block + 2ll * p.batch, warps = slots * p.heads * 2;
    return fa::launch_pdl(append8_kernel<T, Q>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, st, p, pg, slots);
  }
  const int group = std::max(p.block, 16), wpb = group / 16, warps = std::max(4, wpb), units = warps / wpb;
  const long long slots = p.total / group + 2ll * p.batch, items = slots * p.heads * 2;
  const dim3 grid((unsigned)((items + units - 1) / units)), block(32 * warps);
  const auto go = [&](auto kernel) { return fa::launch_pdl(kernel, grid, block, 0, st, p, pg, slots); };
  const bool big = p.block >= 16;
  if (p.dim <= 32) return big ? go(append8_vec_kernel<T, Q, 2, true>) : go(append8_vec_kernel<T, Q, 2, false>);
  if (p.dim <= 64) return big ? go(append8_vec_kernel<T, Q, 4, true>) : go(append8_vec_kernel<T, Q, 4, false>);
  if (p.dim <= 128) return big ? go(append8_vec_kernel<T, Q, 8, true>) : go(append8_vec_kernel<T, Q, 8, false>);
  return big ? go(append8_vec_kernel<T, Q, 16, true>) : go(append8_vec_kernel<T, Q, 16, false>);
}

template <typename T>
int append(const FaKvAppendParams& p, cudaStream_t st) {
  const Pages pg = pages_of(p);
  // groups of 8 elements start on 16-byte boundaries and a rotary unit is whole
  constexpr int U = 16 / sizeof(T);
  const bool vec = (((uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.Kc | (uintptr_t)p.Vc) % 16 == 0) && p.k_row % U == 0 &&
                   p.k_head % U == 0 && p.v_row % U == 0 && p.v_head % U == 0 &&
                   (!p.cos || (p.rot_dim % 16 == 0 && ((uintptr_t)p.cos | (uintptr_t)p.sin) % 16 == 0));
  cudaError_t e;
  if (p.code == FA_CODE_I8) {
    e = append8<T, I8>(p, pg, vec, st);
  } else if (p.code == FA_CODE_E4M3) {
    e = append8<T, E4M3>(p, pg, vec, st);
  } else if (vec) {
    const int rows = rows_of_cta(p.total * 2, MAX_ROWS);
    e = fa::launch_pdl(append_vec_kernel<T>, dim3((unsigned)((p.total + rows - 1) / rows), 2), dim3(AT), 0, st, p, pg, rows,
                       Div(p.heads * p.dim / 16), Div(p.dim / 16));
  } else {
    e = fa::launch_pdl(append_kernel<T, T>, dim3((unsigned)((p.total * p.heads * 2 + 3) / 4)), dim3(128), 0, st, p, pg);
  }
  fa::count_launch();
  return fa::cuda_status(e, "kv append launch");
}

template <typename T>
int gather(const FaKvGatherParams& p, cudaStream_t st) {
  const Pages pg = pages_of(p);
  const int rows = rows_of_cta(p.total * 2, MAX_ROWS);
  const dim3 grid((unsigned)((p.total + rows - 1) / rows), 2), block(GT);
  constexpr int N = 32 / sizeof(T);
  const Div per_row(p.heads * p.dim / N), per_head(p.dim / N);
  const auto go = [&](auto kernel) { return fa::launch_pdl(kernel, grid, block, 0, st, p, pg, rows, per_row, per_head); };
  const cudaError_t e = p.code == FA_CODE_I8      ? go(gather_kernel<T, I8, true>)
                        : p.code == FA_CODE_E4M3  ? go(gather_kernel<T, E4M3, true>)
                        : p.code == FA_DTYPE_F16  ? go(gather_kernel<T, __half, false>)
                        : p.code == FA_DTYPE_BF16 ? go(gather_kernel<T, __nv_bfloat16, false>)
                                                  : go(gather_kernel<T, float, false>);
  fa::count_launch();
  return fa::cuda_status(e, "kv gather launch");
}

}  // namespace

namespace fa {
int kv_device_error(int clear) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_kv_error, sizeof(int));
  if (clear && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_kv_error, &zero, sizeof(int));
  }
  return v;
}
}  // namespace fa

extern "C" FA_API int fa_kv_append_launch(const FaKvAppendParams* pp, int dtype, void* stream) {
  FA_ABI_GUARD(pp, FaKvAppendParams);
  const FaKvAppendParams& p = *pp;
  FA_CHECK_ARG(float_code(dtype), "kv append: dtype code %d", dtype);
  FA_CHECK_ARG(p.k && p.v && p.Kc && p.Vc && p.block_table && p.ctx_len,
               "kv append: k, v, Kc, Vc, block_table, ctx_len must be non-null");
  if (!cache_ok(p, "kv append")) return FA_ERR_INVALID;
  FA_CHECK_ARG(!float_code(p.code) || p.code == dtype, "kv append: a 16/32-bit cache has the new rows' type");
  if (!dim_ok(p.dim, "kv append")) return FA_ERR_UNSUPPORTED;
  FA_CHECK_ARG(p.total >= 0 && (p.cu_new || p.total == (long long)p.batch * p.tokens),
               "kv append: total=%lld rows, batch=%d tokens=%d", p.total, p.batch, p.tokens);
  if (p.cos)
    FA_CHECK_ARG(p.sin && p.rot_dim > 0 && p.rot_dim % 2 == 0 && p.rot_dim <= p.dim && p.rot_seqlen_ro > 0,
                 "kv append: rotary needs sin, an even rot_dim=%d in (0, dim], rot_seqlen_ro=%d > 0", p.rot_dim,
                 p.rot_seqlen_ro);
  if (p.total == 0) return FA_OK;
  FA_CHECK_ARG(p.batch > 0, "kv append: %lld rows of no sequence", p.total);
  if ((p.total + 2ll * p.batch) * p.heads >= 1ll << 30) {
    fa::set_error("kv append: %lld rows of %d heads are more than one call takes", p.total, p.heads);
    return FA_ERR_SIZE;
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == FA_DTYPE_F16) return append<__half>(p, st);
  if (dtype == FA_DTYPE_BF16) return append<__nv_bfloat16>(p, st);
  return append<float>(p, st);
}

extern "C" FA_API int fa_kv_gather_launch(const FaKvGatherParams* pp, int dtype, void* stream) {
  FA_ABI_GUARD(pp, FaKvGatherParams);
  const FaKvGatherParams& p = *pp;
  FA_CHECK_ARG(float_code(dtype), "kv gather: dtype code %d", dtype);
  FA_CHECK_ARG(p.k && p.v && p.Kc && p.Vc && p.block_table && p.cu_k,
               "kv gather: k, v, Kc, Vc, block_table, cu_k must be non-null");
  if (!cache_ok(p, "kv gather")) return FA_ERR_INVALID;
  if (!dim_ok(p.dim, "kv gather")) return FA_ERR_UNSUPPORTED;
  FA_CHECK_ARG(p.total >= 0, "kv gather: total=%lld", p.total);
  if (p.total == 0) return FA_OK;
  FA_CHECK_ARG(p.batch > 0, "kv gather: %lld rows of no sequence", p.total);
  if (p.total * p.heads >= 1ll << 31) {
    fa::set_error("kv gather: %lld rows of %d heads are more than one call takes", p.total, p.heads);
    return FA_ERR_SIZE;
  }
  FA_CHECK_ARG(((uintptr_t)p.Kc | (uintptr_t)p.Vc) % 16 == 0 && ((uintptr_t)p.k | (uintptr_t)p.v) % 32 == 0,
               "kv gather: Kc and Vc must be 16-byte, k and v 32-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == FA_DTYPE_F16) return gather<__half>(p, st);
  if (dtype == FA_DTYPE_BF16) return gather<__nv_bfloat16>(p, st);
  return gather<float>(p, st);
}
