// kvcache.cu — writing to and reading back from paged caches (fa_kv_append_launch,
// fa_kv_gather_launch of fable_attn.h): new K/V rows are rotated and stored behind each
// sequence's cached tokens, as they are or in 8 bits with a scale for each block of slots and
// head; ranges of the caches come back as packed rows.
//
// All three are bound by the bytes they move.  The unit of work is 16 elements of a row as two groups of 8: for a
// rotated piece in NeoX order the groups are the two halves of 8 pairs, otherwise they are neighbours, so that
// a thread rotates what it loads.  Rows whose addresses or rotary size do not allow 16-byte groups take the
// scalar kernels.
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
  if (i < 0 || i >= rm.count(z)) return;   // a row of no sequence
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
  const int z = rm.seq_of_slot(slot, gs), n = rm.count(z), ctx = p.ctx_len[z];
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
__device__ __forceinline__ void store8(T* x, const float* v) {
  Raw8<T> r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = Elem<T>::from_f(v[i]);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(x)[i] = r.u[i];
}

// Groups of unit u of a row: rotated NeoX pieces pair group 8 u with the one rot_dim / 2 further, all others their neighbour.
__device__ __forceinline__ void groups_of(int u, const Turn& r, bool turn, int& d1, int& d2) {
  if (turn && !r.interleaved && 16 * u < r.dim) {
    d1 = 8 * u;
    d2 = d1 + r.dim / 2;
  } else {
    d1 = 16 * u;
    d2 = d1 + 8;
  }
}
// rotates a unit's groups a, b by table row tp: every product and the sum rounded in fp32
__device__ __forceinline__ void turn8(float* a, float* b, int u, const Turn& r, int tp) {
  const int half = r.dim / 2;
  const float4* ct = reinterpret_cast<const float4*>(r.cos + (long long)tp * half + 8 * u);
  const float4* st = reinterpret_cast<const float4*>(r.sin + (long long)tp * half + 8 * u);
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 x = __ldg(ct + i), y = __ldg(st + i);
    c[4 * i] = x.x; c[4 * i + 1] = x.y; c[4 * i + 2] = x.z; c[4 * i + 3] = x.w;
    s[4 * i] = y.x; s[4 * i + 1] = y.y; s[4 * i + 2] = y.z; s[4 * i + 3] = y.w;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float& x = r.interleaved ? (i < 4 ? a[2 * i] : b[2 * i - 8]) : a[i];
    float& y = r.interleaved ? (i < 4 ? a[2 * i + 1] : b[2 * i - 7]) : b[i];
    const float lo = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i])), hi = __fadd_rn(__fmul_rn(y, c[i]), __fmul_rn(x, s[i]));
    x = lo;
    y = hi;
  }
}

// ---------------------------------------------------------------- append, caches of the inputs' type
// A CTA takes `rows` new rows; where each goes stands in shared memory before its threads walk the units of their K and V.
constexpr int AT = 256, MAX_ROWS = 16;
template <typename T>
__global__ void __launch_bounds__(AT) append_vec_kernel(const FaKvAppendParams p, const Pages pg, const int rows) {
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
      if (i >= 0 && i < rm.count(z)) {   // else a row of no sequence
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
  const int per_head = p.dim / 16, per_row = 2 * p.heads * per_head;   // K's units, then V's
#pragma unroll 4
  for (int e = threadIdx.x; e < rows * per_row; e += AT) {
    const int i = e / per_row, w = e % per_row, hu = w % (p.heads * per_head), h = hu / per_head, u = hu % per_head;
    const bool is_k = w < p.heads * per_head;
    const long long slot = s_slot[i], row = row0 + i;
    if (slot < 0) continue;
    const T* x = is_k ? (const T*)p.k + row * p.k_row + h * p.k_head : (const T*)p.v + row * p.v_row + h * p.v_head;
    T* out = (T*)(is_k ? p.Kc : p.Vc) + (slot * p.heads + h) * p.dim;
    const int tp = is_k ? s_turn[i] : -1;
    int d1, d2;
    groups_of(u, r, tp >= 0, d1, d2);
    float a[8], b[8];
    to_float8(load8(x + d1), a);
    to_float8(load8(x + d2), b);
    if (tp >= 0 && 16 * u < r.dim) turn8(a, b, u, r, tp);
    store8(out + d1, a);
    store8(out + d2, b);
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

// A warp holds 16 positions (an aligned group) of one head of K or V in registers: LP lanes a row, each one unit, 32 / LP
// rows a pass.  The largest magnitude of a scale block comes from the row's lanes, then from the rows of the block: lanes, passes and,
// where a block has more than 16 slots, the block's warps.  One read of the new rows, one write of the codes; earlier codes of the
// first block are touched only where its scale grew.  The warps of a CTA take the heads of the same rows, which share
// their cos / sin rows in L1.
template <typename T, typename Q, int LP>
__global__ void __launch_bounds__(512, 1) append8_vec_kernel(const FaKvAppendParams p, const Pages pg, const long long slots) {
  constexpr int RPP = 32 / LP, PASS = 16 / RPP;
  constexpr bool KEEP = LP <= 8;                      // values stay in registers; rows of more than 128 are read again (from L1)
  __shared__ float s_most[16];
  pdl_wait();
  pdl_trigger();
  const int SB = p.block, wpb = SB > 16 ? SB / 16 : 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int units = (blockDim.x >> 5) / wpb;          // (slot, K or V, head) items of a CTA
  const long long item = (long long)blockIdx.x * units + warp / wpb;
  const int h = (int)(item % p.heads), gs = log2_of(max(SB, 16));
  const bool is_k = (item / p.heads) % 2 == 0;
  const long long slot = item / p.heads / 2;
  const RowMap rm{p.cu_new, p.tokens, p.batch};
  // ---- positions [c0, c0 + 16) of this warp; new tokens are [n0, n1)
  int z = 0, ctx = 0, n0 = 0, n1 = 0, c0 = 0;
  if (slot < slots) {
    z = rm.seq_of_slot(slot, gs);
    ctx = p.ctx_len[z];
    if (ctx < 0) record(ERR_PAGE);
    else {
      const long long i = slot - ((rm.first(z) >> gs) + 2 * z);
      c0 = (int)((((ctx >> gs) + i) << gs) + 16 * (warp % wpb));
      n0 = ctx;
      n1 = ctx + rm.count(z);
    }
  }
  const bool any = n1 > n0 && c0 < n1 && c0 + 16 > n0;   // new tokens among them
  const Turn r{p.cos, p.sin, p.rot_dim, p.rot_seqlen_ro, p.rot_interleaved};
  const int u = lane % LP, per_head = p.dim / 16;
  const bool mine = u < per_head;
  const int blk0 = p.page >= 16 && n1 > n0 ? pg.of(z, c0) : -1;
  auto page_of = [&](int pos) { return p.page >= 16 ? blk0 : pg.of(z, pos); };
  // this lane's unit of the new token at pos, rotated; d1, d2: where its groups lie
  auto load = [&](int pos, int& d1, int& d2, float* x) {
    const long long row = rm.first(z) + pos - ctx;
    const T* src = is_k ? (const T*)p.k + row * p.k_row + h * p.k_head : (const T*)p.v + row * p.v_row + h * p.v_head;
    const int tp = turn_pos(p, z, pos - ctx, is_k);
    groups_of(u, r, tp >= 0, d1, d2);
    to_float8(load8(src + d1), x);
    to_float8(load8(src + d2), x + 8);
    if (tp >= 0 && 16 * u < r.dim) turn8(x, x + 8, u, r, tp);
  };
  int d1[PASS], d2[PASS];
  float x[KEEP ? PASS : 1][16];
  float most[PASS];
  bool fresh[PASS];
#pragma unroll
  for (int i = 0; i < PASS; ++i) {
    const int pos = c0 + i * RPP + lane / LP;
    fresh[i] = any && pos >= n0 && pos < n1;
    most[i] = 0.f;
    d1[i] = d2[i] = 0;
    if (fresh[i] && page_of(pos) < 0) {
      record(ERR_PAGE);
      fresh[i] = false;
    }
    if (fresh[i] && mine) {
      float* const v = x[KEEP ? i : 0];
      load(pos, d1[i], d2[i], v);
#pragma unroll
      for (int j = 0; j < 16; ++j) most[i] = max_nan(most[i], fabsf(v[j]));
    }
  }
  // ---- the blocks' largest: lanes of a row, rows of a pass, passes, warps
#pragma unroll
  for (int i = 0; i < PASS; ++i) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
      if (o < LP * SB) most[i] = max_nan(most[i], __shfl_xor_sync(~0u, most[i], o));
  }
#pragma unroll
  for (int o = 1; o < PASS; o <<= 1)
    if (o * RPP < SB) {
#pragma unroll
      for (int i = 0; i < PASS; ++i)
        if (!(i & o)) most[i] = most[i | o] = max_nan(most[i], most[i | o]);
    }
  if (wpb > 1) {
    if (lane == 0) s_most[warp] = most[0];
    __syncthreads();
    float a = 0.f;
    for (int w = 0; w < wpb; ++w) a = max_nan(a, s_most[warp / wpb * wpb + w]);
#pragma unroll
    for (int i = 0; i < PASS; ++i) most[i] = a;
  }
  // ---- scales, codes
  const long long step = (long long)p.heads * p.dim;
  float* const scales = is_k ? p.Ks : p.Vs;
  typename Q::T* const cache = (typename Q::T*)(is_k ? p.Kc : p.Vc);
  const int bs = log2_of(SB);
  float news[PASS];
  int where[PASS];                                    // index of the block's scale within its page and head
#pragma unroll
  for (int i = 0; i < PASS; ++i) {
    const int pos = c0 + i * RPP + lane / LP, first = pos & ~(SB - 1);   // of its block
    const bool touched = n1 > n0 && first < n1 && first + SB > n0;
    const int blk = touched ? page_of(pos) : -1;
    where[i] = (pos & (p.page - 1)) >> bs;
    news[i] = 0.f;
    if (blk < 0) continue;
    float* const sc = scales + ((long long)blk * p.heads + h) * (p.page >> bs) + where[i];
    const bool kept = first < n0;                     // the block holds earlier tokens
    const float old = kept ? *sc : 0.f;
    float s = fmaxf(__fmul_rn(most[i], 1.f / Q::QMAX), MIN_SCALE);
    if (old > s) s = old;
    if (!(most[i] <= 3.402823466e38f) || isnan(old)) s = __int_as_float(0x7fc00000);
    news[i] = s;
    typename Q::T* const out = cache + ((long long)blk * p.page + (pos & (p.page - 1))) * step + (long long)h * p.dim;
    if (mine && fresh[i]) {
      if (isnan(s)) {
        *reinterpret_cast<uint2*>(out + d1[i]) = *reinterpret_cast<uint2*>(out + d2[i]) = make_uint2(0, 0);
      } else {
        const float inv = __frcp_rn(s);
        float* const v = x[KEEP ? i : 0];
        if constexpr (!KEEP) load(pos, d1[i], d2[i], v);
        *reinterpret_cast<uint2*>(out + d1[i]) = codes8<Q>(v, inv);
        *reinterpret_cast<uint2*>(out + d2[i]) = codes8<Q>(v + 8, inv);
      }
    } else if (mine && kept && pos < n0 && s > old) { // earlier token: onto the scale that grew (never where s is NaN)
      const float ratio = __fdiv_rn(old, s);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint2* const at = reinterpret_cast<uint2*>(out + 16 * u + 8 * j);
        float v[8];
        values8<Q>(*at, v);
        *at = codes8<Q>(v, ratio);
      }
    }
  }
  // every reader of the old scale is done before the new one is written
  if (wpb > 1) __syncthreads();
  else __syncwarp();
#pragma unroll
  for (int i = 0; i < PASS; ++i) {
    const int pos = c0 + i * RPP + lane / LP;
    if (news[i] != 0.f && u == 0 && (pos & (SB - 1)) == 0)
      scales[((long long)page_of(pos) * p.heads + h) * (p.page >> bs) + where[i]] = news[i];
  }
}

// ---------------------------------------------------------------- gather
// A CTA takes `rows` rows; a thread makes 16 bytes of the output at a time (8 or 4 elements), K's and then V's.
constexpr int GT = 256;
template <typename T, typename C, bool SCALED>
__global__ void __launch_bounds__(GT) gather_kernel(const FaKvGatherParams p, const Pages pg, const int rows) {
  __shared__ long long s_slot[MAX_ROWS], s_scale[MAX_ROWS];   // cache row; scale of its head 0
  constexpr int N = 16 / sizeof(T);
  pdl_wait();
  pdl_trigger();
  const long long row0 = (long long)blockIdx.x * rows;
  const int per_page = SCALED ? p.page / p.block : 1;
  if (threadIdx.x < rows) {
    const long long row = row0 + threadIdx.x;
    const RowMap rm{p.cu_k, 0, p.batch};
    long long slot = -1, sc = 0;
    if (row < p.total) {
      const int z = rm.seq_of_row(row), i = (int)(row - rm.first(z));
      if (i >= 0 && i < rm.count(z)) {   // else a row of no sequence
        const int pos = i + (p.starts ? p.starts[z] : 0), blk = pg.of(z, pos);
        if (blk < 0) record(ERR_PAGE);
        else {
          const int in_page = pos & (p.page - 1);
          slot = (long long)blk * p.page + in_page;
          sc = (long long)blk * p.heads * per_page + (SCALED ? in_page / p.block : 0);
        }
      }
    }
    s_slot[threadIdx.x] = slot;
    s_scale[threadIdx.x] = sc;
  }
  __syncthreads();
  const int per_row = p.heads * p.dim / N, live = (int)min((long long)rows, p.total - row0);
  const bool is_v = blockIdx.y;
  const void* const cache = is_v ? p.Vc : p.Kc;
  const float* const scales = is_v ? p.Vs : p.Ks;
  T* const out = (T*)(is_v ? p.v : p.k) + row0 * p.heads * p.dim;
#pragma unroll 4
  for (int e = threadIdx.x; e < live * per_row; e += GT) {
    const int i = e / per_row, w = e - i * per_row;
    const long long slot = s_slot[i];
    uint4 u = make_uint4(0, 0, 0, 0);
    T* const o = reinterpret_cast<T*>(&u);
    if (slot >= 0) {
      const long long at = slot * p.heads * p.dim + (long long)w * N;
      if constexpr (SCALED) {
        const float s = __ldg(scales + s_scale[i] + w * N / p.dim * per_page);
        typename C::T c[N];
        if constexpr (N == 8) *reinterpret_cast<uint2*>(c) = __ldg(reinterpret_cast<const uint2*>((const unsigned char*)cache + at));
        else *reinterpret_cast<uint32_t*>(c) = __ldg(reinterpret_cast<const uint32_t*>((const unsigned char*)cache + at));
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = Elem<T>::from_f(C::to_f(c[j]) * s);
      } else if constexpr (std::is_same<T, C>::value) {
        u = __ldg(reinterpret_cast<const uint4*>((const C*)cache + at));
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = Elem<T>::from_f(Elem<C>::to_f(((const C*)cache)[at + j]));
      }
    }
    *reinterpret_cast<uint4*>(out + (long long)e * N) = u;
  }
}

// rows of a CTA: as many as leave every SM two CTAs
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
  if (!(p.batch >= 0 && p.heads > 0)) {
    fa::set_error("%s: batch=%d heads=%d", who, p.batch, p.heads);
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
  if (!vec) {
    const long long slots = p.total / p.block + 2ll * p.batch, warps = slots * p.heads * 2;
    return fa::launch_pdl(append8_kernel<T, Q>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, st, p, pg, slots);
  }
  const int group = std::max(p.block, 16), wpb = group / 16, warps = std::max(4, wpb), units = warps / wpb;
  const long long slots = p.total / group + 2ll * p.batch, items = slots * p.heads * 2;
  const dim3 grid((unsigned)((items + units - 1) / units)), block(32 * warps);
  if (p.dim <= 32) return fa::launch_pdl(append8_vec_kernel<T, Q, 2>, grid, block, 0, st, p, pg, slots);
  if (p.dim <= 64) return fa::launch_pdl(append8_vec_kernel<T, Q, 4>, grid, block, 0, st, p, pg, slots);
  if (p.dim <= 128) return fa::launch_pdl(append8_vec_kernel<T, Q, 8>, grid, block, 0, st, p, pg, slots);
  return fa::launch_pdl(append8_vec_kernel<T, Q, 16>, grid, block, 0, st, p, pg, slots);
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
    const int rows = rows_of_cta(p.total, MAX_ROWS);
    e = fa::launch_pdl(append_vec_kernel<T>, dim3((unsigned)((p.total + rows - 1) / rows)), dim3(AT), 0, st, p, pg, rows);
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
  cudaError_t e;
  if (p.code == FA_CODE_I8) e = fa::launch_pdl(gather_kernel<T, I8, true>, grid, block, 0, st, p, pg, rows);
  else if (p.code == FA_CODE_E4M3) e = fa::launch_pdl(gather_kernel<T, E4M3, true>, grid, block, 0, st, p, pg, rows);
  else if (p.code == FA_DTYPE_F16) e = fa::launch_pdl(gather_kernel<T, __half, false>, grid, block, 0, st, p, pg, rows);
  else if (p.code == FA_DTYPE_BF16) e = fa::launch_pdl(gather_kernel<T, __nv_bfloat16, false>, grid, block, 0, st, p, pg, rows);
  else e = fa::launch_pdl(gather_kernel<T, float, false>, grid, block, 0, st, p, pg, rows);
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
  if (p.total == 0 || p.batch == 0) return FA_OK;
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
  FA_CHECK_ARG(((uintptr_t)p.Kc | (uintptr_t)p.Vc | (uintptr_t)p.k | (uintptr_t)p.v) % 16 == 0,
               "kv gather: Kc, Vc, k and v must be 16-byte aligned");
  if (p.total == 0 || p.batch == 0) return FA_OK;
  if (p.total * p.heads >= 1ll << 31) {
    fa::set_error("kv gather: %lld rows of %d heads are more than one call takes", p.total, p.heads);
    return FA_ERR_SIZE;
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == FA_DTYPE_F16) return gather<__half>(p, st);
  if (dtype == FA_DTYPE_BF16) return gather<__nv_bfloat16>(p, st);
  return gather<float>(p, st);
}
