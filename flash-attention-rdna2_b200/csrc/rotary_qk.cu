// rotary_qk.cu — rotary of q and k at each token's own position, from frequencies instead of tables.
//
// theta = position * inv_freq.  The frequency is held as a fraction of a turn in units of 2^-64, so that the 64-bit product
// with the position wraps by itself at whole turns: no range reduction is left.  inv_freq / (2 pi) is formed in twice fp64's
// bits (a product and its rest, 1 / (2 pi) as two numbers), so that the unit is all that is rounded: the angle is off by
// 2^-64 of a turn for each position, 2^-33 of one at 2^31.  The quadrant comes off in the integers too, and sincospi sees at
// most an eighth of a turn.
//
// Bound by memory: every element of q and k is read and written once.  A block takes `TOK` tokens: its threads form the
// tokens' cos / sin once, in shared memory, and then walk all heads of q and k by 16-byte units, so that the 64-bit product and the
// sine cost one evaluation per token and pair instead of one per head.  Blocks of 4 tokens where that still gives
// every SM several blocks, else of 1 (a decode step has few tokens, and its time is latency).
#include <algorithm>
#include "fa_common.cuh"
#include "fa_launch.h"

namespace {

constexpr int THREADS = 256, MAX_PAIRS = 128;

template <typename T>
__device__ __forceinline__ void turn(const T& a, const T& b, float2 e, T& oa, T& ob) {
  const float x = Elem<T>::to_f(a), y = Elem<T>::to_f(b);
  oa = Elem<T>::from_f(x * e.x - y * e.y);
  ob = Elem<T>::from_f(y * e.x + x * e.y);
}

// radians as a fraction of a turn in units of 2^-64
__device__ __forceinline__ unsigned long long turns_of(double radians) {
  constexpr double INV_2PI = 0.15915494309189535, INV_2PI_REST = -9.839338337591243e-18;      // their sum is 1 / (2 pi) to 2^-110
  constexpr double UNITS = 18446744073709551616.0;
  const double turns = radians * INV_2PI, rest = fma(radians, INV_2PI, -turns) + radians * INV_2PI_REST;
  const double part = turns - trunc(turns);      // exact
  const unsigned long long most = __double2ull_rn(fabs(part) * UNITS);
  return (part < 0 ? 0 - most : most) + (unsigned long long)__double2ll_rn(rest * UNITS);
}

template <typename T, int U> struct alignas(U * sizeof(T) == 16 ? 16 : sizeof(T)) Unit { T e[U]; };

// U: elements of a 16-byte unit, or 1 (2 where the pairs are neighbours) for rows that do not lie on 16 bytes: those are read
// and written element by element
template <typename T, int U, bool INTER, int TOK>
__global__ void __launch_bounds__(THREADS, 5) rotary_qk_kernel(const FaRotaryQkParams p, const long long tokens) {
  __shared__ __align__(16) float2 sce[TOK][MAX_PAIRS];
  __shared__ long long off[TOK][4];        // the tokens' rows in q, k and the outputs
  const int half = p.rot_dim / 2;
  const long long first = (long long)blockIdx.x * TOK;
  const int nt = (int)min((long long)TOK, tokens - first);
  if (threadIdx.x < nt) {
    const long long row = first + threadIdx.x, z = row / p.seqlen, s = row - z * p.seqlen;
    off[threadIdx.x][0] = z * p.sQ.b + s * p.sQ.s;
    off[threadIdx.x][1] = z * p.sK.b + s * p.sK.s;
    off[threadIdx.x][2] = z * p.sQo.b + s * p.sQo.s;
    off[threadIdx.x][3] = z * p.sKo.b + s * p.sKo.s;
  }
  for (int e = threadIdx.x; e < nt * half; e += THREADS) {
    const int t = e / half, i = e - t * half;
    const long long row = first + t;
    long long pos;
    if (p.positions) {
      pos = p.pos_bytes == 8 ? ((const long long*)p.positions)[row] : ((const int*)p.positions)[row];
    } else {
      const long long z = row / p.seqlen;
      pos = row - z * p.seqlen + p.offset;
      if (p.offsets) pos += p.pos_bytes == FA_ROTARY_OFFSETS_64 ? ((const long long*)p.offsets)[z] : p.offsets[z];
    }
    const unsigned long long angle = (unsigned long long)pos * turns_of(p.inv_freq[i]);
    const unsigned int hi = (unsigned int)((angle + 0x80000000ull) >> 32);     // to nearest: opposite positions turn alike
    const unsigned int quarter = (hi + 0x20000000u) >> 30;
    float s, c;
    sincospif((float)(int)(hi - (quarter << 30)) * (1.f / 2147483648.f), &s, &c);
    if (quarter & 1) {
      const float x = c;
      c = -s;
      s = x;
    }
    if (quarter & 2) {
      c = -c;
      s = -s;
    }
    if (!isfinite(p.inv_freq[i])) c = s = __int_as_float(0x7fffffff);      // shows, and in its own pair alone
    sce[t][i] = make_float2(p.factor * c, (p.inverse ? -p.factor : p.factor) * s);
  }
  __syncthreads();
  const int heads = p.heads_q + p.heads_k;
  using V = Unit<T, U>;
  const auto rows = [&](int t, int h, const T*& x, T*& o) {
    const bool is_q = h < p.heads_q;
    const int hh = is_q ? h : h - p.heads_q;
    x = (const T*)(is_q ? p.q : p.k) + off[t][is_q ? 0 : 1] + hh * (is_q ? p.sQ.h : p.sK.h);
    o = (T*)(is_q ? p.q_out : p.k_out) + off[t][is_q ? 2 : 3] + hh * (is_q ? p.sQo.h : p.sKo.h);
    return is_q;
  };
  // A thread keeps its unit w of the head and steps over heads and tokens without a division; FLY units are in flight at a time
  constexpr int FLY = 2;
  {
    const int turning = INTER ? p.rot_dim / U : half / U;      // units of a head that turn
    const int side = max(1, THREADS / turning), mine = threadIdx.x / turning;      // heads at a time
    for (int w = threadIdx.x - mine * turning; w < turning && mine < side; w += THREADS) {
      int t = mine / heads, h = mine - t * heads;
      while (t < nt) {
        V a[FLY], b[FLY];
        T* to[FLY];
        const float2* ce[FLY];
#pragma unroll
        for (int k = 0; k < FLY; ++k) {
          to[k] = nullptr;
          if (t >= nt) break;
          const T* x;
          rows(t, h, x, to[k]);
          x += w * U;
          to[k] += w * U;
          ce[k] = sce[t] + (INTER ? w * U / 2 : w * U);
          a[k] = *reinterpret_cast<const V*>(x);
          if constexpr (!INTER) b[k] = *reinterpret_cast<const V*>(x + half);
          for (h += side; h >= heads; h -= heads) ++t;
        }
#pragma unroll
        for (int k = 0; k < FLY; ++k) {
          if (!to[k]) break;
          if constexpr (INTER) {
            V r;
#pragma unroll
            for (int i = 0; i < U; i += 2) turn<T>(a[k].e[i], a[k].e[i + 1], ce[k][i / 2], r.e[i], r.e[i + 1]);
            *reinterpret_cast<V*>(to[k]) = r;
          } else {
            V ra, rb;
#pragma unroll
            for (int i = 0; i < U; ++i) turn<T>(a[k].e[i], b[k].e[i], ce[k][i], ra.e[i], rb.e[i]);
            *reinterpret_cast<V*>(to[k]) = ra;
            *reinterpret_cast<V*>(to[k] + half) = rb;
          }
        }
      }
    }
  }
  // the dims past rot_dim, where q or k do not stay in place
  const bool copy_q = p.q_out != p.q, copy_k = p.k_out != p.k;
  if (!copy_q && !copy_k) return;
  constexpr int C = U * sizeof(T) == 16 ? U : 1;      // elements of a copied unit
  using W = Unit<T, C>;
  const int copied = (p.dim - p.rot_dim) / C, all = nt * heads * copied;
  for (int e0 = threadIdx.x; e0 < all; e0 += FLY * THREADS) {
    W a[FLY];
    T* to[FLY];
#pragma unroll
    for (int k = 0; k < FLY; ++k) {
      const int e = e0 + k * THREADS;
      to[k] = nullptr;
      if (e >= all) break;
      const int ht = e / copied, w = e - ht * copied, t = ht / heads;
      const T* x;
      T* o;
      if (!(rows(t, ht - t * heads, x, o) ? copy_q : copy_k)) continue;
      to[k] = o + p.rot_dim + w * C;
      a[k] = *reinterpret_cast<const W*>(x + p.rot_dim + w * C);
    }
#pragma unroll
    for (int k = 0; k < FLY; ++k)
      if (e0 + k * THREADS < all && to[k]) *reinterpret_cast<W*>(to[k]) = a[k];
  }
}

template <typename T, int U, bool INTER>
int go(const FaRotaryQkParams& p, cudaStream_t st) {
  const long long tokens = (long long)p.batch * p.seqlen;
  if (tokens >= 8ll * fa::num_sms()) {
    FA_CHECK_ARG((tokens + 3) / 4 < (1ll << 31), "rotary of q and k: %lld tokens", tokens);
    rotary_qk_kernel<T, U, INTER, 4><<<(int)((tokens + 3) / 4), THREADS, 0, st>>>(p, tokens);
  } else {
    rotary_qk_kernel<T, U, INTER, 1><<<(int)tokens, THREADS, 0, st>>>(p, tokens);
  }
  fa::count_launch();
  return fa::cuda_status(cudaGetLastError(), "rotary (q and k) launch");
}

template <typename T>
int run(const FaRotaryQkParams& p, cudaStream_t st) {
  constexpr int U = 16 / sizeof(T);
  const auto on = [&](const void* x, const FaStrides& s) {
    return (uintptr_t)x % 16 == 0 && (p.batch == 1 || s.b % U == 0) && (p.seqlen == 1 || s.s % U == 0) && s.h % U == 0;
  };
  const bool vec = p.dim % U == 0 && p.rot_dim % (p.interleaved ? U : 2 * U) == 0 && on(p.q, p.sQ) && on(p.q_out, p.sQo) &&
                   (!p.k || (on(p.k, p.sK) && on(p.k_out, p.sKo)));
  if (p.interleaved) return vec ? go<T, U, true>(p, st) : go<T, 2, true>(p, st);
  return vec ? go<T, U, false>(p, st) : go<T, 1, false>(p, st);
}

}  // namespace

extern "C" FA_API int fa_rotary_qk_launch(const FaRotaryQkParams* pp, int dtype, void* stream) {
  FA_ABI_GUARD(pp, FaRotaryQkParams);
  FaRotaryQkParams p = *pp;
  FA_CHECK_ARG(dtype >= FA_DTYPE_F16 && dtype <= FA_DTYPE_F32, "rotary of q and k: dtype code %d", dtype);
  FA_CHECK_ARG(p.q && p.q_out && p.inv_freq && !p.k == !p.k_out, "rotary of q and k: q, q_out, inv_freq must be non-null, k goes with k_out");
  FA_CHECK_ARG(p.batch >= 0 && p.seqlen >= 0 && p.heads_q > 0 && p.dim > 0 && (!p.k || p.heads_k > 0),
               "rotary of q and k: batch=%d seqlen=%d heads %d / %d dim=%d", p.batch, p.seqlen, p.heads_q, p.heads_k, p.dim);
  FA_CHECK_ARG(p.rot_dim > 0 && p.rot_dim % 2 == 0 && p.rot_dim <= p.dim && p.rot_dim <= 2 * MAX_PAIRS,
               "rotary of q and k: rot_dim=%d must be even, at most dim=%d and at most %d", p.rot_dim, p.dim, 2 * MAX_PAIRS);
  FA_CHECK_ARG(!p.positions || p.pos_bytes == 4 || p.pos_bytes == 8, "rotary of q and k: positions of %d bytes", p.pos_bytes);
  if (!p.k) p.heads_k = 0;
  if (p.batch == 0 || p.seqlen == 0) return FA_OK;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == FA_DTYPE_F16) return run<__half>(p, st);
  if (dtype == FA_DTYPE_BF16) return run<__nv_bfloat16>(p, st);
  return run<float>(p, st);
}
