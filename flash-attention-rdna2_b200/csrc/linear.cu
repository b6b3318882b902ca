// linear.cu — linear attention with a decay per head: the recurrent kernel for few tokens, the CUDA-core kernels that take
// every type and head dim, the kernel that joins segments, and the entry points.
#include <algorithm>
#include "linear_common.cuh"
#include "fa_launch.h"

namespace {

using namespace fa;

__device__ int g_lin_error = 0;

// =====================================================================================
// Recurrent kernel: S_t = lam S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t, token by token.
// Bound by reading and writing the state once: 8 dk dv bytes a sequence and head.  A block holds 32 columns of one state
// (a 128-byte line of each row) in registers, so that a state of 128 columns gives four blocks and small batches still spread;
// all its loads are issued before anything else is looked at, the other sequences' slots among them.
// =====================================================================================
constexpr int STEP_THREADS = 128, STEP_COLS = 32, STEP_BATCH = 4;

// ROWS = rows of the state a thread holds: dk <= 16 * ROWS; G = query heads of a group that are summed together
template <typename T, int ROWS, int G>
__global__ void __launch_bounds__(STEP_THREADS, ROWS > 8 ? 3 : 6)
    lin_step_kernel(const LinSeqs q, const LinRole r, const LinPool pool, const int blocks_v) {
  __shared__ __align__(16) float sk[STEP_BATCH][256], sq[STEP_BATCH][G][256], sv[STEP_BATCH][STEP_COLS], sred[STEP_BATCH][4][G][STEP_COLS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int vb = blockIdx.x % blocks_v, hz = blockIdx.x / blocks_v, h = hz % q.nhk, z = hz / q.nhk;
  const int named = pool.index ? pool.index[z] : z;
  const bool old = pool.in && !(pool.seen && pool.seen[z] <= 0);
  const LinSpan span = lin_span(q, z);
  const float lam = exp2f(lin_log2_decay(q.log_decay, h));
  const int col = vb * STEP_COLS + (tid & 7) * 4, row0 = tid >> 3;
  const bool mine = col < r.dc, inside = named >= 0 && (!pool.index || named < pool.slots);
  const long long at = ((long long)named * q.nhk + h) * r.da * r.dc + col;
  float4 x[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = row0 + 16 * i;
    x[i] = old && mine && inside && row < r.da ? __ldcs(reinterpret_cast<const float4*>(pool.in + at + (long long)row * r.dc))
                                               : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const T* a = (const T*)r.a + (q.cu ? 0 : z * r.sa.b) + span.row0 * r.sa.s + (long long)h * r.na * r.sa.h;
  const T* b = (const T*)r.b + (q.cu ? 0 : z * r.sb.b) + span.row0 * r.sb.s + (long long)h * r.sb.h;
  const T* c = (const T*)r.c + (q.cu ? 0 : z * r.sc.b) + span.row0 * r.sc.s + (long long)h * r.sc.h;
  T* out = (T*)r.out + (q.cu ? 0 : z * r.so.b) + span.row0 * r.so.s + (long long)h * r.na * r.so.h;
  if (vb == 0) lin_zero_outside<T>(q, r, h * r.na, z, q.batch, STEP_THREADS);
  if (lin_slot(pool, z, STEP_THREADS, &g_lin_error) < 0) {
    for (long long e = tid; e < (long long)span.len * r.na * STEP_COLS; e += STEP_THREADS) {
      const int cc = vb * STEP_COLS + (int)(e % STEP_COLS), g = (int)(e / STEP_COLS % r.na), t = (int)(e / STEP_COLS / r.na);
      if (cc < r.dc) out[t * r.so.s + g * r.so.h + cc] = Elem<T>::from_f(0.f);
    }
    return;
  }
  // Tokens in batches: their rows come in together, and their sums are joined together (one by one a token cost 5 us, most of it
  // waiting).  Groups of more than G query heads take one token at a time.
  const int batch = r.na <= G ? STEP_BATCH : 1;
  for (int t0 = 0; t0 < span.len; t0 += batch) {
    const int nt = min(batch, span.len - t0);
    for (int g0 = 0; g0 < r.na; g0 += G) {
      const int ng = min(G, r.na - g0);
      if (t0 > 0 || g0 > 0) __syncthreads();
      if (g0 == 0 && tid < nt * STEP_COLS) {
        const int cc = vb * STEP_COLS + tid % STEP_COLS;
        sv[tid / STEP_COLS][tid % STEP_COLS] = cc < r.dc ? Elem<T>::to_f(c[(t0 + tid / STEP_COLS) * r.sc.s + cc]) : 0.f;
      }
      // All rows of the batch in flight at once.  Dims past dk and heads past the group's are 0, so that the products below run
      // without a test: with one at each step a token of four heads took 4.5 us.
      for (int e = tid; e < 16 * ROWS; e += STEP_THREADS) {
        const bool real = e < r.da;
        T gk[STEP_BATCH], gq[STEP_BATCH][G];
#pragma unroll
        for (int tt = 0; tt < STEP_BATCH; ++tt) {
          gk[tt] = Elem<T>::from_f(0.f);
          if (g0 == 0 && real && tt < nt) gk[tt] = b[(t0 + tt) * r.sb.s + e];
#pragma unroll
          for (int g = 0; g < G; ++g) {
            gq[tt][g] = Elem<T>::from_f(0.f);
            if (real && tt < nt && g < ng) gq[tt][g] = a[(t0 + tt) * r.sa.s + (g0 + g) * r.sa.h + e];
          }
        }
#pragma unroll
        for (int tt = 0; tt < STEP_BATCH; ++tt) {
          if (g0 == 0) sk[tt][e] = Elem<T>::to_f(gk[tt]);
#pragma unroll
          for (int g = 0; g < G; ++g) sq[tt][g][e] = Elem<T>::to_f(gq[tt][g]);
        }
      }
      __syncthreads();
      for (int tt = 0; tt < nt; ++tt) {
        const float4 v = *reinterpret_cast<const float4*>(&sv[tt][(tid & 7) * 4]);
        float4 o[G];
#pragma unroll
        for (int g = 0; g < G; ++g) o[g] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (g0 == 0) {
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            const float k = sk[tt][row0 + 16 * i];
            x[i].x = fmaf(lam, x[i].x, k * v.x);
            x[i].y = fmaf(lam, x[i].y, k * v.y);
            x[i].z = fmaf(lam, x[i].z, k * v.z);
            x[i].w = fmaf(lam, x[i].w, k * v.w);
          }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const float w = sq[tt][g][row0 + 16 * i];
            o[g].x = fmaf(w, x[i].x, o[g].x);
            o[g].y = fmaf(w, x[i].y, o[g].y);
            o[g].z = fmaf(w, x[i].z, o[g].z);
            o[g].w = fmaf(w, x[i].w, o[g].w);
          }
        // the state is on its way back before the sums are joined
        if (t0 + tt == span.len - 1 && g0 + G >= r.na && pool.out && mine) {
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            const int row = row0 + 16 * i;
            if (row < r.da) __stcs(reinterpret_cast<float4*>(pool.out + at + (long long)row * r.dc), x[i]);
          }
        }
        // lanes of one column group differ in bits 3 and 4; then the four warps
#pragma unroll
        for (int m = 8; m <= 16; m *= 2)
#pragma unroll
          for (int g = 0; g < G; ++g) {
            o[g].x += __shfl_xor_sync(0xffffffffu, o[g].x, m);
            o[g].y += __shfl_xor_sync(0xffffffffu, o[g].y, m);
            o[g].z += __shfl_xor_sync(0xffffffffu, o[g].z, m);
            o[g].w += __shfl_xor_sync(0xffffffffu, o[g].w, m);
          }
        if (lane < 8) {
#pragma unroll
          for (int g = 0; g < G; ++g) *reinterpret_cast<float4*>(&sred[tt][warp][g][lane * 4]) = o[g];
        }
      }
      __syncthreads();
      for (int e = tid; e < nt * G * STEP_COLS; e += STEP_THREADS) {
        const int cc = e % STEP_COLS, g = e / STEP_COLS % G, tt = e / STEP_COLS / G;
        if (g < ng && vb * STEP_COLS + cc < r.dc)
          out[(t0 + tt) * r.so.s + (g0 + g) * r.so.h + vb * STEP_COLS + cc] =
              Elem<T>::from_f(r.w_inter * (sred[tt][0][g][cc] + sred[tt][1][g][cc] + sred[tt][2][g][cc] + sred[tt][3][g][cc]));
      }
    }
  }
  if (span.len > 0 || !pool.out || !mine) return;      // without tokens the state is passed on
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = row0 + 16 * i;
    if (row < r.da) *reinterpret_cast<float4*>(pool.out + at + (long long)row * r.dc) = x[i];
  }
}

// =====================================================================================
// CUDA-core chunked kernel: every type, dims up to 256, any strides.  A block walks one segment of one state in chunks of
// SC tokens, for 64 of the c dim's columns, all in fp32: the state, the chunk's rows and the pair products in shared memory.
// The dims of a and b go by in slices of 64: a slice adds to the pair products and to a X, then its rows of X are brought up
// to date; so the rows take the same room for every dim, and two blocks fit on an SM up to dims of 128.
// Bound by shared memory's reads: a thread's tile is SC/16 rows by 4 columns, read four elements at a time (rows padded to an odd
// number of 16-byte units, so that the lanes of a quarter warp meet different banks).  With 64 tokens eight 16-byte reads feed
// 64 multiply-adds, with 32 tokens six feed 32; pairs that the order masks are neither multiplied nor read, and two adjacent
// elements go through one packed multiply-add.  fp32, 4 x 4096 tokens, 16 heads of 64: 430 us, 15 TFLOP/s (with 2 x 4 outputs
// a thread and whole rows of a and b in shared memory it was 809).
// =====================================================================================
constexpr int SCOL = 64, SDIM = 64, SLD = SDIM + 4, SIMT_THREADS = 256;
constexpr int SIMT_WIDE = 160;      // dims of a up to which an SM holds two blocks of 64-token chunks (110 KB)

template <int SC>
__host__ __device__ constexpr int simt_smem_floats(int da) { return 2 * SC * SLD + SC * SCOL + da * SCOL + SC * (SC + 4) + SC + 4; }

__device__ __forceinline__ float2 twice(float w) { return make_float2(w, w); }
struct Quad { float2 lo, hi; };      // four columns
__device__ __forceinline__ Quad quad(const float* s) {
  const float4 v = *reinterpret_cast<const float4*>(s);
  return Quad{make_float2(v.x, v.y), make_float2(v.z, v.w)};
}
__device__ __forceinline__ void axpy(float2 w, const Quad& v, Quad& s) {
  s.lo = __ffma2_rn(w, v.lo, s.lo);
  s.hi = __ffma2_rn(w, v.hi, s.hi);
}
// s[u] += p[u][0..3] rows 0..3 of v (row stride SCOL)
template <int R>
__device__ __forceinline__ void rows_by_four(const float* p, int ld, const float* v, Quad (&s)[R]) {
  const Quad v0 = quad(v), v1 = quad(v + SCOL), v2 = quad(v + 2 * SCOL), v3 = quad(v + 3 * SCOL);
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const float4 w = *reinterpret_cast<const float4*>(p + u * ld);
    axpy(twice(w.x), v0, s[u]);
    axpy(twice(w.y), v1, s[u]);
    axpy(twice(w.z), v2, s[u]);
    axpy(twice(w.w), v3, s[u]);
  }
}

template <typename T> struct __align__(4 * sizeof(T)) Four { T x[4]; };

// rows [0, n) of 64 columns, of which the first `real` exist (the rest, and the rows up to SC, are 0)
template <typename T, int SC>
__device__ __forceinline__ void simt_rows(float* to, int ld, const T* from, long long step, int real, int n, bool wide) {
#pragma unroll 4
  for (int e = threadIdx.x; e < SC * 16; e += SIMT_THREADS) {
    const int j = e >> 4, i = (e & 15) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (j < n && i < real) {
      const T* s = from + j * step + i;
      Four<T> w;
      if (wide) w = *reinterpret_cast<const Four<T>*>(s);
      else w = Four<T>{{s[0], s[1], s[2], s[3]}};
      x = make_float4(Elem<T>::to_f(w.x[0]), Elem<T>::to_f(w.x[1]), Elem<T>::to_f(w.x[2]), Elem<T>::to_f(w.x[3]));
    }
    *reinterpret_cast<float4*>(to + j * ld + i) = x;
  }
}
__device__ __forceinline__ void copy16(float* to, const float* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy16_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// f(element of X in shared memory, place in the state, whether it exists) for every four elements that lie together in the state: of
// a row of X, or (`across`, stored transposed) of a column, where a warp takes 8 columns by 4 units so that both sides go by 32 bytes or more
template <typename F, typename G>
__device__ __forceinline__ void simt_state(const LinRole& r, int c0, F along, G across, float* sx) {
  const int n4 = r.da / 4;
#pragma unroll 4
  for (int e = threadIdx.x; e < r.da * (SCOL / 4); e += SIMT_THREADS) {
    if (r.transposed) {
      const int i = e / 8 % n4 * 4, j = e / 8 / n4 * 8 + (e & 7);
      across(sx + i * SCOL + j, (long long)(c0 + j) * r.da + i, c0 + j < r.dc);
    } else {
      const int i = e / (SCOL / 4), j = e % (SCOL / 4) * 4;
      along(sx + i * SCOL + j, (long long)i * r.dc + c0 + j, c0 + j < r.dc);
    }
  }
}
// four elements at a time: base and strides on their boundary
template <typename T>
__device__ __forceinline__ bool simt_wide(const void* p, const FaStrides& s) {
  return ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0 && ((s.b | s.s | s.h) & 3) == 0;
}

template <typename T, int SC, bool REV, bool STATES>
__global__ void __launch_bounds__(SIMT_THREADS, SC == 32 ? 3 : 2)
    lin_simt_kernel(const LinSeqs q, const LinRole r, const float* ws, float* ws_out, const LinPool pool, const int blocks_c) {
  extern __shared__ __align__(16) float sm[];
  constexpr int R = SC / 16, SPLD = SC + 4;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  float* sa = sm;                           // [SC][SLD]
  float* sb = sa + SC * SLD;
  float* sc = sb + SC * SLD;                // [SC][SCOL]
  float* sx = sc + SC * SCOL;               // [da][SCOL]
  float* sp = sx + r.da * SCOL;             // [SC][SPLD]
  float* lam = sp + SC * SPLD;              // lam^n, n <= SC
  const int cb = blockIdx.x % blocks_c;
  const int h = blockIdx.x / blocks_c % q.nhk, seg = blockIdx.x / blocks_c / q.nhk;
  const int c0 = cb * SCOL;
  if (!STATES && cb == 0) lin_zero_outside<T>(q, r, h * r.na, seg, q.slots, SIMT_THREADS);
  int z, t0, t1;
  const LinSpan span = lin_segment(q, seg, z, t0, t1);
  if (t1 <= t0 && (STATES || ws)) return;
  const int slot = STATES ? z : lin_slot(pool, z, SIMT_THREADS, &g_lin_error);
  T* out = (T*)r.out + (q.cu ? 0 : z * r.so.b) + span.row0 * r.so.s + (long long)h * r.na * r.so.h;
  const T* a = (const T*)r.a + (q.cu ? 0 : z * r.sa.b) + span.row0 * r.sa.s + (long long)h * r.na * r.sa.h;
  const T* b = (const T*)r.b + (q.cu ? 0 : z * r.sb.b) + span.row0 * r.sb.s + (long long)h * r.nb * r.sb.h;
  const T* c = (const T*)r.c + (q.cu ? 0 : z * r.sc.b) + span.row0 * r.sc.s + (long long)h * r.nb * r.sc.h;
  if (!STATES && slot < 0) {
    for (int g = 0; g < r.na; ++g)
      for (long long e = tid; e < (long long)(t1 - t0) * SCOL; e += SIMT_THREADS)
        if (c0 + e % SCOL < r.dc) out[(t0 + e / SCOL) * r.so.s + g * r.so.h + c0 + e % SCOL] = Elem<T>::from_f(0.f);
    return;
  }
  const float g2 = lin_log2_decay(q.log_decay, h);
  for (int e = tid; e <= SC; e += SIMT_THREADS) lam[e] = lin_power(g2, e);
  // the state that enters the segment
  const long long per = (long long)r.da * r.dc, segs = (long long)seg * q.nhk + h;
  const float* x0 = nullptr;
  if (!STATES) {
    if (ws) x0 = ws + segs * per;
    else if (pool.in && !(pool.seen && pool.seen[z] <= 0)) x0 = pool.in + ((long long)slot * q.nhk + h) * per;
  }
  simt_state(r, c0, [&](float* to, long long from, bool real) {
    if (real && x0) copy16(to, x0 + from);      // in flight while the first rows are loaded
    else *reinterpret_cast<float4*>(to) = make_float4(0.f, 0.f, 0.f, 0.f);
  }, [&](float* to, long long from, bool real) {
    const float4 x = real && x0 ? *reinterpret_cast<const float4*>(x0 + from) : make_float4(0.f, 0.f, 0.f, 0.f);
    to[0] = x.x, to[SCOL] = x.y, to[2 * SCOL] = x.z, to[3 * SCOL] = x.w;
  }, sx);
  float* x1 = nullptr;
  if (STATES) x1 = ws_out + segs * per;
  else if (!ws && pool.out) x1 = pool.out + ((long long)slot * q.nhk + h) * per;
  const bool wide_a = simt_wide<T>(r.a, r.sa), wide_b = simt_wide<T>(r.b, r.sb), wide_c = simt_wide<T>(r.c, r.sc),
             wide_o = simt_wide<T>(r.out, r.so);
  const int chunks = (t1 - t0 + SC - 1) / SC, groups = STATES ? r.nb : max(r.na, r.nb), slices = (r.da + SDIM - 1) / SDIM;
  const int diagonal = R * ty / 16;         // the 16 columns of P that hold this thread's rows (one for the whole warp)
  for (int m = 0; m < chunks; ++m) {
    const int at = t0 + (REV ? chunks - 1 - m : m) * SC, cn = min(SC, t1 - at);
    Quad o[R];
    for (int g = 0; g < groups; ++g) {
      const bool new_a = g == 0 || r.na > 1, new_b = g == 0 || r.nb > 1, last_a = r.na > 1 || g == groups - 1,
                 last_b = r.nb > 1 || g == groups - 1;
      float2 p[R][R] = {};
      if (!STATES && new_a) {
#pragma unroll
        for (int u = 0; u < R; ++u) o[u] = Quad{};
      }
      for (int s = 0; s < slices; ++s) {
        const int d0 = s * SDIM, width = min(SDIM, r.da - d0);
        __syncthreads();
        if (!STATES && (new_a || slices > 1))
          simt_rows<T, SC>(sa, SLD, a + at * r.sa.s + (r.na > 1 ? g : 0) * r.sa.h + d0, r.sa.s, width, cn, wide_a);
        if (new_b || slices > 1) simt_rows<T, SC>(sb, SLD, b + at * r.sb.s + (r.nb > 1 ? g : 0) * r.sb.h + d0, r.sb.s, width, cn, wide_b);
        if (new_b && s == 0) simt_rows<T, SC>(sc, SCOL, c + at * r.sc.s + (r.nb > 1 ? g : 0) * r.sc.h + c0, r.sc.s, r.dc - c0, cn, wide_c);
        copy16_wait();
        __syncthreads();
        if constexpr (!STATES) {
          const float *ar = sa + R * ty * SLD, *br = sb + tx * SLD;
          for (int i = 0; i < width; i += 4) {
            Quad x[R];
#pragma unroll
            for (int u = 0; u < R; ++u) x[u] = quad(ar + u * SLD + i);
#pragma unroll
            for (int w = 0; w < R; ++w) {
              if (REV ? w < diagonal : w > diagonal) continue;
              const Quad y = quad(br + 16 * w * SLD + i);
#pragma unroll
              for (int u = 0; u < R; ++u) p[u][w] = __ffma2_rn(x[u].hi, y.hi, __ffma2_rn(x[u].lo, y.lo, p[u][w]));
            }
          }
          if (new_a)
            for (int i = 0; i < width; i += 4) rows_by_four<R>(ar + i, SLD, sx + (d0 + i) * SCOL + tx * 4, o);
          __syncthreads();
        }
        // this slice's rows of X: their old values have been used by every reader of the chunk (the last chunk's are kept only if asked for)
        if (last_b && (x1 || m < chunks - 1) && 4 * ty < width) {
          const float keep = r.nb > 1 && g > 0 ? 1.f : lam[cn];
          Quad x[4] = {};
#pragma unroll 4
          for (int j = 0; j < cn; ++j) {
            const float4 w4 = *reinterpret_cast<const float4*>(sb + j * SLD + 4 * ty);
            Quad v = quad(sc + j * SCOL + tx * 4);
            const float2 w = twice(lam[REV ? j + 1 : cn - 1 - j]);
            v.lo = __fmul2_rn(v.lo, w);
            v.hi = __fmul2_rn(v.hi, w);
            axpy(twice(w4.x), v, x[0]);
            axpy(twice(w4.y), v, x[1]);
            axpy(twice(w4.z), v, x[2]);
            axpy(twice(w4.w), v, x[3]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float4& to = *reinterpret_cast<float4*>(sx + (d0 + 4 * ty + k) * SCOL + tx * 4);
            to = make_float4(fmaf(r.w_up, x[k].lo.x, keep * to.x), fmaf(r.w_up, x[k].lo.y, keep * to.y),
                             fmaf(r.w_up, x[k].hi.x, keep * to.z), fmaf(r.w_up, x[k].hi.y, keep * to.w));
          }
        }
      }
      if constexpr (!STATES) {
#pragma unroll
        for (int u = 0; u < R; ++u) {
          const int i = R * ty + u;
          if (new_a) {
            const int steps = REV ? cn - 1 - i : i + 1;
            const float2 w = twice(i < cn ? r.w_inter * lam[max(steps, 0)] : 0.f);
            o[u].lo = __fmul2_rn(o[u].lo, w);
            o[u].hi = __fmul2_rn(o[u].hi, w);
          }
#pragma unroll
          for (int w = 0; w < R; ++w) {
            const int j = tx + 16 * w, gap = REV ? j - i : i - j;
            sp[i * SPLD + j] = gap >= 0 && i < cn && j < cn ? r.w_intra * (p[u][w].x + p[u][w].y) * lam[gap] : 0.f;
          }
        }
        __syncwarp();      // a warp reads its own rows of P only
        const int j1 = REV ? cn : min(cn, R * (ty + 1));      // rows past the sequence are 0
        for (int j = REV ? R * ty & ~3 : 0; j < j1; j += 4) rows_by_four<R>(sp + R * ty * SPLD + j, SPLD, sc + j * SCOL + tx * 4, o);
        if (last_a && c0 + tx * 4 < r.dc) {
#pragma unroll
          for (int u = 0; u < R; ++u) {
            const int i = R * ty + u;
            if (i >= cn) continue;
            T* to = out + (at + i) * r.so.s + (r.na > 1 ? g : 0) * r.so.h + c0 + tx * 4;
            const Four<T> y{{Elem<T>::from_f(o[u].lo.x), Elem<T>::from_f(o[u].lo.y), Elem<T>::from_f(o[u].hi.x), Elem<T>::from_f(o[u].hi.y)}};
            if (wide_o) *reinterpret_cast<Four<T>*>(to) = y;
            else to[0] = y.x[0], to[1] = y.x[1], to[2] = y.x[2], to[3] = y.x[3];
          }
        }
      }
    }
  }
  if (!x1) return;
  copy16_wait();
  __syncthreads();
  simt_state(r, c0, [&](const float* from, long long to, bool real) {
    if (real) *reinterpret_cast<float4*>(x1 + to) = *reinterpret_cast<const float4*>(from);
  }, [&](const float* from, long long to, bool real) {
    if (real) *reinterpret_cast<float4*>(x1 + to) = make_float4(from[0], from[SCOL], from[2 * SCOL], from[3 * SCOL]);
  }, sx);
}

// =====================================================================================
// Joining segments: ws[n] holds what segment n adds from a state of 0; it becomes the state that enters the segment, and
// the state past the last one goes to the pool.  A sequence without tokens has no segment: its state goes through untouched.
// One thread a float4 of the state; the next segment's load is in flight while the running state is scaled.
// =====================================================================================
template <bool REV>
__global__ void __launch_bounds__(256) lin_join_kernel(const LinSeqs q, float* ws, const LinPool pool, const int per4) {
  const int z = blockIdx.x / q.nhk, h = blockIdx.x % q.nhk;
  const int slot = lin_slot(pool, z, 256, &g_lin_error);
  const int e = blockIdx.y * 256 + threadIdx.x;
  if (slot < 0 || e >= per4) return;
  const LinSpan span = lin_span(q, z);
  const float g2 = lin_log2_decay(q.log_decay, h);
  const int real = lin_segments(q, span.len);
  const long long step = (long long)q.nhk * per4;      // from one segment's state to the next
  float4* w = reinterpret_cast<float4*>(ws) + lin_first_slot(q, z, span.row0) * step + (long long)h * per4 + e;
  const long long at = ((long long)slot * q.nhk + h) * per4 + e;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (pool.in && !(pool.seen && pool.seen[z] <= 0)) x = reinterpret_cast<const float4*>(pool.in)[at];
  const auto seg = [&](int m) { return REV ? real - 1 - m : m; };
  float4 u = real > 0 ? w[seg(0) * step] : make_float4(0.f, 0.f, 0.f, 0.f);
  for (int m = 0; m < real; ++m) {
    const int n = seg(m);
    float4 next = u;
    if (m + 1 < real) next = w[seg(m + 1) * step];
    w[n * step] = x;
    const float keep = lin_power(g2, n == real - 1 ? span.len - n * q.seg_len : q.seg_len);
    x.x = fmaf(keep, x.x, u.x); x.y = fmaf(keep, x.y, u.y); x.z = fmaf(keep, x.z, u.z); x.w = fmaf(keep, x.w, u.w);
    u = next;
  }
  if (pool.out) reinterpret_cast<float4*>(pool.out)[at] = x;
}

// chunks of 64 tokens, or of 32 where segments are no longer than that or two blocks of 64 do not fit on an SM (fa_linear_plan has the times)
template <typename T, int SC>
int simt_go(const LinSeqs& q, const LinRole& r, bool rev, bool states, const float* ws, float* ws_out, const LinPool& pool,
            cudaStream_t st) {
  const int blocks_c = (r.dc + SCOL - 1) / SCOL;
  const long long grid = (long long)q.slots * q.nhk * blocks_c;
  FA_CHECK_ARG(grid < (1ll << 31) && (long long)q.batch * q.nhk < (1ll << 31), "linear attention: %lld blocks", grid);
  const auto go = [&](auto kernel, unsigned long long* done) -> int {
    if (int rc = ensure_smem((const void*)kernel, simt_smem_floats<SC>(256) * 4, done)) return rc;
    kernel<<<(int)grid, SIMT_THREADS, simt_smem_floats<SC>(r.da) * 4, st>>>(q, r, ws, ws_out, pool, blocks_c);
    count_launch();
    return cuda_status(cudaGetLastError(), "linear attention launch");
  };
  static unsigned long long done[4] = {};
  if (states) return rev ? go(lin_simt_kernel<T, SC, true, true>, done) : go(lin_simt_kernel<T, SC, false, true>, done + 1);
  return rev ? go(lin_simt_kernel<T, SC, true, false>, done + 2) : go(lin_simt_kernel<T, SC, false, false>, done + 3);
}
template <typename T>
int simt_launch(const LinSeqs& q, const LinRole& r, bool rev, bool states, const float* ws, float* ws_out, const LinPool& pool,
                cudaStream_t st) {
  return q.seg_len <= 32 || r.da > SIMT_WIDE ? simt_go<T, 32>(q, r, rev, states, ws, ws_out, pool, st) : simt_go<T, 64>(q, r, rev, states, ws, ws_out, pool, st);
}

template <typename T>
int step_launch(const LinSeqs& q, const LinRole& r, const LinPool& pool, cudaStream_t st) {
  const int blocks_v = (r.dc + STEP_COLS - 1) / STEP_COLS;
  const long long grid = (long long)q.batch * q.nhk * blocks_v;
  FA_CHECK_ARG(grid < (1ll << 31), "linear attention: %lld blocks", grid);
  const auto go = [&](auto one, auto four) {
    if (r.na == 1) one<<<(int)grid, STEP_THREADS, 0, st>>>(q, r, pool, blocks_v);
    else four<<<(int)grid, STEP_THREADS, 0, st>>>(q, r, pool, blocks_v);
  };
  if (r.da <= 64) go(lin_step_kernel<T, 4, 1>, lin_step_kernel<T, 4, 4>);
  else if (r.da <= 128) go(lin_step_kernel<T, 8, 1>, lin_step_kernel<T, 8, 4>);
  else go(lin_step_kernel<T, 16, 1>, lin_step_kernel<T, 16, 4>);
  count_launch();
  return cuda_status(cudaGetLastError(), "linear attention (recurrent) launch");
}

int join(const LinSeqs& q, bool rev, float* ws, const LinPool& pool, int per, cudaStream_t st) {
  const dim3 grid(q.batch * q.nhk, (per / 4 + 255) / 256);
  if (rev) lin_join_kernel<true><<<grid, 256, 0, st>>>(q, ws, pool, per / 4);
  else lin_join_kernel<false><<<grid, 256, 0, st>>>(q, ws, pool, per / 4);
  count_launch();
  return cuda_status(cudaGetLastError(), "linear attention (join) launch");
}

// 16 bits on the CUDA cores take nine times as long: FABLE_ATTN_REQUIRE_TC refuses them
int allow_cuda_cores(const LinSeqs& q, const LinRole& r, int dtype) {
  if (dtype == FA_DTYPE_F32 || !(q.cu ? q.total > 0 : q.S > 0) || !require_tc()) return FA_OK;
  set_error("linear attention: FABLE_ATTN_REQUIRE_TC is set and the tensor-core kernels do not take this request (dims %d and %d, "
            "alignment or strides, or the build's register count)", r.da, r.dc);
  return FA_ERR_UNSUPPORTED;
}
int states(const LinSeqs& q, const LinRole& r, bool rev, float* ws, int dtype, cudaStream_t st) {
  bool taken = false;
  if (int rc = lin_tc_states(q, r, rev, ws, dtype, st, &taken)) return rc;
  if (taken) return FA_OK;
  if (int rc = allow_cuda_cores(q, r, dtype)) return rc;
  return lin_simt_states(q, r, rev, ws, dtype, st);
}
int main_pass(const LinSeqs& q, const LinRole& r, bool rev, const float* ws, const LinPool& pool, int dtype, cudaStream_t st) {
  bool taken = false;
  if (int rc = lin_tc_main(q, r, rev, ws, pool, dtype, st, &taken)) return rc;
  if (taken) return FA_OK;
  if (int rc = allow_cuda_cores(q, r, dtype)) return rc;
  return lin_simt_main(q, r, rev, ws, pool, dtype, st);
}
// The tensor-core kernels' last state comes from the states kernel (whose sums keep fp32's bits), so one segment goes
// through it too where a last state is asked for.
bool through_states(const LinSeqs& q, const LinRole& r, const float* out, int dtype) {
  return q.nseg > 1 || (out && lin_tc_takes(q, r, dtype));
}

bool dims_ok(int dk, int dv) { return dk > 0 && dv > 0 && dk <= 256 && dv <= 256 && dk % 8 == 0 && dv % 8 == 0; }
bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

}  // namespace

namespace fa {
int lin_simt_states(const LinSeqs& q, const LinRole& r, bool rev, float* ws, int dtype, cudaStream_t st) {
  const LinPool none{};
  if (dtype == FA_DTYPE_F16) return simt_launch<__half>(q, r, rev, true, nullptr, ws, none, st);
  if (dtype == FA_DTYPE_BF16) return simt_launch<__nv_bfloat16>(q, r, rev, true, nullptr, ws, none, st);
  return simt_launch<float>(q, r, rev, true, nullptr, ws, none, st);
}
int lin_simt_main(const LinSeqs& q, const LinRole& r, bool rev, const float* ws, const LinPool& pool, int dtype, cudaStream_t st) {
  if (dtype == FA_DTYPE_F16) return simt_launch<__half>(q, r, rev, false, ws, nullptr, pool, st);
  if (dtype == FA_DTYPE_BF16) return simt_launch<__nv_bfloat16>(q, r, rev, false, ws, nullptr, pool, st);
  return simt_launch<float>(q, r, rev, false, ws, nullptr, pool, st);
}
int lin_device_error(int clear) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_lin_error, sizeof(int));
  if (clear && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_lin_error, &zero, sizeof(int));
  }
  return v | lin_tc_device_error(clear);
}
}  // namespace fa

// floats of the workspace, 0 where none is needed
static long long workspace(long long total, int batch, int seg_len, int nseg, long long nhk, int dk, int dv, bool tc) {
  return nseg > 1 || tc ? fa::lin_slots(total > 0, total, batch, seg_len, nseg) * nhk * dk * dv : 0;
}

extern "C" FA_API long long fa_linear_plan(int batch, int S, long long total, int NH, int gqa, int dk, int dv, int dtype, int* seg_len,
                                           int* nseg) {
  if (seg_len) *seg_len = 128;
  if (nseg) *nseg = 1;
  if (!seg_len || !nseg || batch <= 0 || S <= 0 || gqa <= 0 || NH < gqa || !dims_ok(dk, dv)) return 0;
  const long long states = (long long)batch * (NH / gqa);
  const long long tokens = total > 0 && total < (long long)batch * S ? std::max(1ll, total / batch) : S;
  const bool tc = dtype != FA_DTYPE_F32 && dk <= 128 && dv <= 128;
  const long long chunks = (tokens + 127) / 128, sms = num_sms();
  long long best = 1, unit = 128;
  if (tc) {
    // Blocks run one to an SM.  In units of one head's chunk in the output kernel (3 us): a chunk costs its query heads and 0.4 for the
    // state, a block 2.5 to start, and the states kernel, which more than one segment needs, 0.5 a chunk and 1.5 to start, with
    // 2 for it and the join.  Blocks of one length run in waves; where lengths differ they fill in, and the longest is what is left over.
    const double heads = gqa, per_chunk = heads + 0.4;
    double least = 1e30;
    for (long long n = 1; n <= std::min((S + 127ll) / 128, 1024ll); ++n) {
      const double walk = (double)(((S + 127ll) / 128 + n - 1) / n);
      const bool ragged = tokens < S;
      double cost;
      if (ragged) {
        const double blocks = (double)states * ((double)chunks / walk + 0.5) / (double)sms;
        cost = blocks * 2.5 + (double)(states * chunks) / (double)sms * (per_chunk + (n > 1 ? 0.5 : 0.0)) + walk * per_chunk * 0.5;
      } else {
        const double waves = (double)((states * n + sms - 1) / sms);
        cost = waves * (walk * (per_chunk + (n > 1 ? 0.5 : 0.0)) + (n > 1 ? 4.0 : 2.5)) + (n > 1 ? 2.0 : 0.0);
      }
      if (cost < least) least = cost, best = n;
      if (walk <= 1.0) break;
    }
    unit = 128;
    const long long whole = (S + 127ll) / 128;
    *seg_len = (int)std::min((whole + best - 1) / best * 128, 1ll << 30);
    *nseg = (int)((S + (long long)*seg_len - 1) / *seg_len);
    return workspace(total, batch, *seg_len, *nseg, NH / gqa, dk, dv, true);
  } else {
    // Segments of one chunk of 32 tokens while two blocks an SM can take them all (each costs a state written and read again, and its
    // keys and values read twice): fp32, 8 heads of 64, 512 tokens in 19 us, against 23 with chunks of 64.  Past that chunks of 64, in as
    // many segments as run at once: 2048 tokens 35 against 40 us, 4 x 4096 tokens of 16 heads 430 against 543.
    // Dims of more than 160 keep to chunks of 32 (with 64 an SM holds one block: 2085 against 1564 us for 4096 tokens of
    // 16 heads of 256), and to four blocks an SM, two waves of them.
    const long long blocks = std::max(1ll, states * ((dv + 63) / 64)), small = (tokens + 31) / 32;
    const bool large = std::max(dk, dv) > SIMT_WIDE;
    unit = large || small <= 2 * sms / blocks ? 32 : 64;
    best = std::max(1ll, std::min((tokens + unit - 1) / unit, (large ? 4 : 2) * sms / blocks));
  }
  const long long units = (tokens + unit - 1) / unit;
  long long len = (units + best - 1) / best * unit;
  if (len >= S) len = (S + unit - 1ll) / unit * unit;
  *seg_len = (int)std::min(len, 1ll << 30);
  *nseg = (int)((S + (long long)*seg_len - 1) / *seg_len);
  return workspace(total, batch, *seg_len, *nseg, NH / gqa, dk, dv, false);
}

extern "C" FA_API int fa_linear_launch(const FaLinearParams* pp, int dtype, void* stream) {
  FA_ABI_GUARD(pp, FaLinearParams);
  const FaLinearParams& p = *pp;
  cudaStream_t st = (cudaStream_t)stream;
  FA_CHECK_ARG(dtype >= FA_DTYPE_F16 && dtype <= FA_DTYPE_F32, "linear attention: dtype code %d", dtype);
  const bool rows = p.cu ? p.total > 0 : (long long)p.batch * p.S > 0;
  FA_CHECK_ARG(p.log_decay && (!rows || (p.q && p.k && p.v && p.o)), "linear attention: q, k, v, o, log_decay must be non-null");
  FA_CHECK_ARG(p.batch >= 0 && p.S >= 0 && p.NH > 0 && p.gqa > 0 && p.NH % p.gqa == 0 && p.total >= 0,
               "linear attention: batch=%d S=%d NH=%d gqa=%d total=%lld", p.batch, p.S, p.NH, p.gqa, p.total);
  FA_CHECK_ARG(dims_ok(p.dk, p.dv), "linear attention: dk=%d and dv=%d must be multiples of 8 up to 256", p.dk, p.dv);
  FA_CHECK_ARG(aligned16(p.state_in) && aligned16(p.state_out) && aligned16(p.states), "linear attention: states must lie on 16 bytes");
  FA_CHECK_ARG(p.slots >= 0 && (p.state_index || !(p.state_in || p.state_out) || p.slots >= p.batch),
               "linear attention: %lld slots for %d sequences", p.slots, p.batch);
  FA_CHECK_ARG(!p.cu || p.batch > 0 || p.total == 0, "linear attention: %lld packed rows of no sequence", p.total);
  if (p.batch == 0) return FA_OK;
  const bool step = !p.keep_states && p.S <= FA_LINEAR_STEP_TOKENS;
  LinSeqs q{p.cu, p.log_decay, p.total, p.batch, p.S, p.NH / p.gqa, 0, 1, p.batch};
  if (!step) {
    q.seg_len = p.seg_len;
    q.nseg = p.nseg;
    FA_CHECK_ARG(p.seg_len > 0 && p.nseg > 0 && (long long)p.seg_len * p.nseg >= p.S, "linear attention: %d segments of %d tokens for S=%d",
                 p.nseg, p.seg_len, p.S);
    const long long slots = lin_slots(p.cu != nullptr, p.total, p.batch, p.seg_len, p.nseg);
    FA_CHECK_ARG(slots < (1ll << 31), "linear attention: %lld segments", slots);
    q.slots = (int)slots;
    FA_CHECK_ARG(p.nseg == 1 || p.states, "linear attention: %d segments need the workspace `states`", p.nseg);
  }
  const LinPool pool{p.state_in, p.state_out, p.state_index, p.seen, p.state_index ? p.slots : p.batch};
  const LinRole r{p.q, p.k, p.v, p.o, p.sQ, p.sK, p.sV, p.sO, p.gqa, 1, p.dk, p.dv, 0, p.scale, p.scale, 1.f};
  if (step) {
    if (dtype == FA_DTYPE_F16) return step_launch<__half>(q, r, pool, st);
    if (dtype == FA_DTYPE_BF16) return step_launch<__nv_bfloat16>(q, r, pool, st);
    return step_launch<float>(q, r, pool, st);
  }
  const bool joined = through_states(q, r, p.state_out, dtype);
  FA_CHECK_ARG(!joined || p.states, "linear attention: the workspace `states` is missing");
  if (joined) {
    if (int rc = states(q, r, false, p.states, dtype, st)) return rc;
    if (int rc = join(q, false, p.states, pool, p.dk * p.dv, st)) return rc;
  }
  return main_pass(q, r, false, joined ? p.states : nullptr, pool, dtype, st);
}

extern "C" FA_API int fa_linear_backward_launch(const FaLinearBwdParams* pp, int dtype, void* stream) {
  FA_ABI_GUARD(pp, FaLinearBwdParams);
  const FaLinearBwdParams& p = *pp;
  cudaStream_t st = (cudaStream_t)stream;
  FA_CHECK_ARG(dtype >= FA_DTYPE_F16 && dtype <= FA_DTYPE_F32, "linear attention backward: dtype code %d", dtype);
  const bool rows = p.cu ? p.total > 0 : (long long)p.batch * p.S > 0;
  FA_CHECK_ARG(p.log_decay && (!rows || (p.q && p.k && p.v && p.dO && p.dQ && p.dK && p.dV)),
               "linear attention backward: q, k, v, dO, dQ, dK, dV, log_decay must be non-null");
  FA_CHECK_ARG(p.batch >= 0 && p.S >= 0 && p.NH > 0 && p.gqa > 0 && p.NH % p.gqa == 0 && p.total >= 0,
               "linear attention backward: batch=%d S=%d NH=%d gqa=%d total=%lld", p.batch, p.S, p.NH, p.gqa, p.total);
  FA_CHECK_ARG(dims_ok(p.dk, p.dv), "linear attention backward: dk=%d and dv=%d must be multiples of 8 up to 256", p.dk, p.dv);
  FA_CHECK_ARG(aligned16(p.initial) && aligned16(p.dfinal) && aligned16(p.dinitial) && aligned16(p.states) && aligned16(p.work),
               "linear attention backward: states must lie on 16 bytes");
  FA_CHECK_ARG(!p.cu || p.batch > 0 || p.total == 0, "linear attention backward: %lld packed rows of no sequence", p.total);
  if (p.batch == 0) return FA_OK;
  FA_CHECK_ARG(p.seg_len > 0 && p.nseg > 0 && (long long)p.seg_len * p.nseg >= p.S,
               "linear attention backward: %d segments of %d tokens for S=%d", p.nseg, p.seg_len, p.S);
  FA_CHECK_ARG(p.nseg == 1 || (p.states && p.work), "linear attention backward: %d segments need `states` and `work`", p.nseg);
  const long long slots = lin_slots(p.cu != nullptr, p.total, p.batch, p.seg_len, p.nseg);
  FA_CHECK_ARG(slots < (1ll << 31), "linear attention backward: %lld segments", slots);
  const LinSeqs q{p.cu, p.log_decay, p.total, p.batch, p.S, p.NH / p.gqa, p.seg_len, p.nseg, (int)slots};
  const float s = p.scale;
  const LinRole dq{p.dO, p.v, p.k, p.dQ, p.sdO, p.sV, p.sK, p.sdQ, p.gqa, 1, p.dv, p.dk, 1, s, s, 1.f};
  const LinRole dk{p.v, p.dO, p.q, p.dK, p.sV, p.sdO, p.sQ, p.sdK, 1, p.gqa, p.dv, p.dk, 1, s, 1.f, s};
  const LinRole dv{p.k, p.q, p.dO, p.dV, p.sK, p.sQ, p.sdO, p.sdV, 1, p.gqa, p.dk, p.dv, 0, s, 1.f, s};
  const LinPool forward{p.initial, nullptr, nullptr, nullptr, p.batch};
  const LinPool back{p.dfinal, p.dinitial, nullptr, nullptr, p.batch}, back_only{p.dfinal, nullptr, nullptr, nullptr, p.batch};
  const bool joined = through_states(q, dv, p.dinitial, dtype);
  FA_CHECK_ARG(!joined || p.work, "linear attention backward: the workspace `work` is missing");
  if (joined) {
    if (int rc = states(q, dv, true, p.work, dtype, st)) return rc;
    if (int rc = join(q, true, p.work, back, p.dk * p.dv, st)) return rc;
  }
  const float* from = joined ? p.work : nullptr;
  if (int rc = main_pass(q, dq, false, q.nseg > 1 ? p.states : nullptr, forward, dtype, st)) return rc;
  if (int rc = main_pass(q, dk, true, from, back_only, dtype, st)) return rc;
  return main_pass(q, dv, true, from, joined ? back_only : back, dtype, st);
}
