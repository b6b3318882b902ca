// linear_sm100.cu — linear attention with a decay per head on the Blackwell tensor cores (tcgen05 + TMEM + TMA), fp16 and bf16,
// head dims up to 128 (tiles of 64 or 128 columns, the columns past the real dims zero-filled by the TMA).
//
// Chunks of 128 tokens.  In the terms of linear_common.cuh, per chunk that the state X enters:
//     P  = a b^T               (SS)    scaled by lam^|i-j| and masked on the way back into TMEM, as hi + lo 16-bit operands
//     O  = a X                 (SS)    X from shared memory as hi + lo, its rows' factor w_inter lam^n_i applied in fp32 in the epilogue
//     O  = P c                 (TS)
//     X  = lam^C X + (w lam^m b)^T c   (TS)   X stays in TMEM in fp32; the decayed rows b~ are read from the tile column by column
//                                             (a thread is a dim), so that they are the transposed A operand in TMEM
// With SWAP, c takes b's part in the state: X^T = lam^C X^T + (w lam^m c)^T b.  dk runs so: then q is the operand that is
// decayed and rounded, and dO, which may be tiny (fp16 gradients), enters every product as it is.
//
// Operands of 16 bits: what is computed (P, X, b~) enters as hi + lo, which leaves 2^-16 (bf16) or 2^-22 (fp16) of a term; the result's own rounding is
// 2^-9 or 2^-12, and one 16-bit number each would add as much again.  fp16 has no range to spare: rows of P are brought
// to a largest value of about 2^10 by a power of 2 each, and X by one for the tile, taken back in the epilogue; the decayed rows are
// left as they are: where they fall below 2^-14 their steps are 2^-24, which is fp16's own step for such inputs.
//
// Warp roles (320 threads): warps 0-7 elementwise, two to a TMEM lane quadrant (w and w + 4 share 32 lanes, w / 4 takes half
// of the columns or tokens), warp 8 TMA, warp 9 MMA.  The elementwise warps take the decayed rows of item t, the epilogue of
// item t - 1, then the state, the pair products and a X of item t, so that each waits for an MMA that has had another step's
// time.  Every wait is bounded.
#include <cudaTypedefs.h>
#include "linear_common.cuh"
#include "fa_launch.h"
#include "sm100_ptx.cuh"

namespace {

using namespace sm100;
using namespace fa;

constexpr int C = 128;               // tokens of a chunk
constexpr int NTHREADS = 320, NELEM = 256, WARP_TMA = 8, WARP_MMA = 9;
__device__ int g_lin_tc_error = 0;
__device__ __forceinline__ void record_error(int code) { atomicOr(&g_lin_tc_error, code); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  } else {
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// what is left of a pair once it is rounded to 16 bits (exact)
template <bool BF16>
__device__ __forceinline__ float2 rest2(float2 d, uint32_t hi) {
  return __ffma2_rn(unpack2<BF16>(hi), make_float2(-1.f, -1.f), d);
}
// a pair as hi + lo 16-bit pairs
template <bool BF16>
__device__ __forceinline__ void split2(float2 d, uint32_t& hi, uint32_t& lo) {
  hi = pack2<BF16>(d.x, d.y);
  const float2 l = rest2<BF16>(d, hi);
  lo = pack2<BF16>(l.x, l.y);
}

// Four 8 x 8 blocks of 16-bit elements, transposed: a thread gets of each block the dim lane / 4 of tokens 2 (lane % 4) and + 1
__device__ __forceinline__ void ldsm_t4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 TMEM lanes x 8 columns: thread T's r[2 n + e] goes to lane 8 e + T / 4, column 4 n + T % 4, which is where ldsm_t4 of
// 16 dims x 16 tokens leaves token pairs
__device__ __forceinline__ void tmem_st_16x8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
               ::"l"((uint64_t)map), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// The decayed rows of a chunk, transposed for the A operand in TMEM: a warp takes 32 dims and 64 tokens (half hf).  Its thread
// reads pairs of tokens 64 hf + 16 s + 8 m + 2 (lane % 4) (+ 1), whose factors w[2 s + m] stay in registers from chunk to
// chunk.  Element by element from shared memory this took 6000 cycles a chunk, and half of the kernel's time.
template <bool REV>
__device__ __forceinline__ void row_factors(float2* w, const float* lam, float times, int hf, int lane, int cn) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = 64 * hf + 8 * i + 2 * (lane & 3);
    w[i].x = j < cn ? times * lam[REV ? j + 1 : cn - 1 - j] : 0.f;
    w[i].y = j + 1 < cn ? times * lam[REV ? j + 2 : cn - 2 - j] : 0.f;
  }
}
template <bool BF16, int TERMS>
__device__ __forceinline__ void decay_rows(uint32_t tile, uint32_t bt, const float2* w, int qd, int hf, int lane, int cn) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {          // 16 dims each
    const int unit = 4 * (qd & 1) + 2 * half + ((lane >> 3) & 1), token = 64 * hf + 8 * (lane >> 4) + (lane & 7);
    const uint32_t from = tile + (qd >> 1) * C * 128 + token * 128 + ((unit ^ (lane & 7)) << 4);
    const uint32_t to = bt + ((uint32_t)(16 * half) << 16) + 32 * hf;
#pragma unroll
    for (int s = 0; s < 4; ++s) {                 // 16 tokens each
      uint32_t r[4], o[3][4];
      ldsm_t4(from + s * 16 * 128, r);
#pragma unroll
      for (int i = 0; i < 4; ++i) {               // blocks: dims 0-7 and 8-15 of the first 8 tokens, then of the next 8
        if (cn < C) {                             // rows past the sequence may hold anything: a factor of 0 is not enough
          const int j = 64 * hf + 16 * s + 8 * (i >> 1) + 2 * (lane & 3);
          r[i] &= (j < cn ? 0xffffu : 0u) | (j + 1 < cn ? 0xffff0000u : 0u);
        }
        float2 x = __fmul2_rn(unpack2<BF16>(r[i]), w[2 * s + (i >> 1)]);
#pragma unroll
        for (int u = 0; u < TERMS; ++u) {
          o[u][i] = pack2<BF16>(x.x, x.y);
          if (u + 1 < TERMS) x = rest2<BF16>(x, o[u][i]);
        }
      }
#pragma unroll
      for (int u = 0; u < TERMS; ++u) tmem_st_16x8(to + 64 * u + 8 * s, o[u]);
    }
  }
}

// descriptors of a [rows][D] tile stored as D / 64 chunks of rows x 128 bytes (128-byte swizzle)
__device__ __forceinline__ uint64_t desc_k(uint32_t tile) { return sdesc_sw128(tile, 16, 1024); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, int rows) { return sdesc_sw128(tile, rows * 128, 1024); }
// 16 steps along the contracted dim, in 16-byte units
__device__ __forceinline__ uint32_t step_k(int kk, int rows) { return (uint32_t)(((kk / 4) * rows * 128 + (kk % 4) * 32) >> 4); }

__device__ __forceinline__ void bar_elem() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void bar_pair(int quadrant) { asm volatile("bar.sync %0, 64;" ::"r"(2 + quadrant) : "memory"); }

// power of 2 that brings a largest value of `top` to [2^10, 2^11); 1 for 0 and for what is not finite
__device__ __forceinline__ float scale_to(uint32_t top_bits) {
  const int e = (int)(top_bits >> 23);
  if (e == 0 || e == 255) return 1.f;
  return __uint_as_float((uint32_t)min(max(127 + 10 - (e - 127), 1), 254) << 23);
}

// rows [r0, 128) of a tile of `chunks` x 128 rows x 128 bytes to 0 (the calling warp)
__device__ __forceinline__ void zero_rows(uint8_t* tile, int chunks, int r0, int lane) {
  for (int c = 0; c < chunks; ++c)
    for (int e = r0 * 8 + lane; e < C * 8; e += 32) *reinterpret_cast<uint4*>(tile + c * C * 128 + e * 16) = make_uint4(0, 0, 0, 0);
}

// =====================================================================================
// outputs
// =====================================================================================
template <int D>
struct Cfg {
  static constexpr int NCH = D / 64;
  static constexpr int TILE = C * D * 2;            // a, b or c
  static constexpr int XT = D * D * 2;              // X hi or lo
  static constexpr int NA = D == 128 ? 1 : 2, NB = D == 128 ? 1 : 2, NC = 2;
  static constexpr int OFF_X = 0, OFF_A = 2 * XT, OFF_B = OFF_A + NA * TILE, OFF_C = OFF_B + NB * TILE;
  static constexpr int OFF_O = OFF_C + NC * TILE;   // outputs on their way: a box of 32 rows x D / 2 columns for each warp
  static constexpr int OFF_BAR = OFF_O + TILE;
  static constexpr int OFF_LAM = OFF_BAR + 256;     // lam^n, n = 0 .. 128
  static constexpr int OFF_MAX = OFF_LAM + 132 * 4; // [2] largest |X|, then [2][128] largest |P| of half a row (fp16)
  static constexpr int SMEM = OFF_MAX + 16 + 2 * C * 4 + 1024;
  static constexpr uint32_t P_COL = 0, BT_COL = 128, X_COL = 256, O_COL = 256 + D;
  static_assert(SMEM <= 232448, "shared memory per CTA");
};
struct Bz {
  static constexpr int A_FULL = 0, A_EMPTY = 16, B_FULL = 32, B_EMPTY = 48, C_FULL = 64, C_EMPTY = 80, P_FULL = 96, P_READY = 104,
                       PV_DONE = 112, XS_READY = 120, BT_READY = 128, X_DONE = 136, OI_FULL = 144, OI_READ = 152, O_READ = 160,
                       DRAIN = 168, TMEM_ADDR = 176;
};

template <int D, bool BF16, bool REV, bool SWAP>
__global__ void __launch_bounds__(NTHREADS, 1)
    lin_tc_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap tc,
                  const __grid_constant__ CUtensorMap to, const LinSeqs q, const LinRole r, const float* ws, const LinPool pool) {
  using K = Cfg<D>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = blockIdx.x % q.nseg, h = blockIdx.x / q.nseg % q.nhk, z = blockIdx.x / q.nseg / q.nhk;
  lin_zero_outside<T>(q, r, z, h * r.na, n, q.nseg, NTHREADS);
  const LinSpan span = lin_span(q, z);
  int t0, t1;
  lin_segment(q, span.len, n, t0, t1);
  if (t1 <= t0) return;
  const int slot = lin_slot(pool, z, NTHREADS, &g_lin_tc_error);
  T* out = (T*)r.out + (q.cu ? 0 : z * r.so.b) + (span.row0 + t0) * r.so.s + (long long)h * r.na * r.so.h;
  if (slot < 0) {
    for (int g = 0; g < r.na; ++g)
      for (long long e = tid; e < (long long)(t1 - t0) * r.dc; e += NTHREADS)
        out[e / r.dc * r.so.s + g * r.so.h + e % r.dc] = Elem<T>::from_f(0.f);
    return;
  }
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t bar = sbase + K::OFF_BAR;
  float* lam = reinterpret_cast<float*>(sgen + K::OFF_LAM);
  uint32_t* xmax = reinterpret_cast<uint32_t*>(sgen + K::OFF_MAX);
  uint32_t* pmax = xmax + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sgen + K::OFF_BAR + Bz::TMEM_ADDR);
  const int chunks = (t1 - t0 + C - 1) / C, groups = max(r.na, r.nb), items = chunks * groups;
  const float g2 = lin_log2_decay(q.log_decay, h);

  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar + Bz::A_FULL + 8 * s, 1);
      mbar_init(bar + Bz::A_EMPTY + 8 * s, 1);
      mbar_init(bar + Bz::B_FULL + 8 * s, 1);
      mbar_init(bar + Bz::B_EMPTY + 8 * s, 1);
      mbar_init(bar + Bz::C_FULL + 8 * s, 1);
      mbar_init(bar + Bz::C_EMPTY + 8 * s, 1);
    }
    mbar_init(bar + Bz::P_FULL, 1);
    mbar_init(bar + Bz::P_READY, NELEM);
    mbar_init(bar + Bz::PV_DONE, 1);
    mbar_init(bar + Bz::XS_READY, NELEM);
    mbar_init(bar + Bz::BT_READY, NELEM);
    mbar_init(bar + Bz::X_DONE, 1);
    mbar_init(bar + Bz::OI_FULL, 1);
    mbar_init(bar + Bz::OI_READ, NELEM);
    mbar_init(bar + Bz::O_READ, NELEM);
    mbar_init(bar + Bz::DRAIN, 1);
    xmax[0] = xmax[1] = 0;
    fence_barrier_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  if (tid <= C) lam[tid] = lin_power(g2, tid);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // item t: chunk t / groups (from the end where reversed), head t % groups of the side that has several
  const auto chunk_at = [&](int t) { return (REV ? chunks - 1 - t / groups : t / groups) * C; };

  if (warp == WARP_TMA) {
    if (lane == 0) {
      int na = 0, nb = 0, nc = 0;
      bool ok = true;
      const int z4 = q.cu ? 0 : z;
      for (int t = 0; ok && t < items; ++t) {
        const int g = t % groups, row = (int)span.row0 + t0 + chunk_at(t);
        if (g == 0 || r.na > 1) {
          const int s = na % K::NA;
          if (na >= K::NA && !mbar_wait(bar + Bz::A_EMPTY + 8 * s, ((na / K::NA) - 1) & 1)) { ok = false; break; }
          mbar_expect_tx(bar + Bz::A_FULL + 8 * s, K::TILE);
          for (int c = 0; c < K::NCH; ++c)
            tma_load_4d(sbase + K::OFF_A + s * K::TILE + c * C * 128, &ta, c * 64, row, h * r.na + (r.na > 1 ? g : 0), z4, bar + Bz::A_FULL + 8 * s);
          ++na;
        }
        if (g == 0 || r.nb > 1) {
          const int s = nb % K::NB, hh = h * r.nb + (r.nb > 1 ? g : 0);
          if (nb >= K::NB && !mbar_wait(bar + Bz::B_EMPTY + 8 * s, ((nb / K::NB) - 1) & 1)) { ok = false; break; }
          mbar_expect_tx(bar + Bz::B_FULL + 8 * s, K::TILE);
          for (int c = 0; c < K::NCH; ++c)
            tma_load_4d(sbase + K::OFF_B + s * K::TILE + c * C * 128, &tb, c * 64, row, hh, z4, bar + Bz::B_FULL + 8 * s);
          ++nb;
          const int s2 = nc % K::NC;
          if (nc >= K::NC && !mbar_wait(bar + Bz::C_EMPTY + 8 * s2, ((nc / K::NC) - 1) & 1)) { ok = false; break; }
          mbar_expect_tx(bar + Bz::C_FULL + 8 * s2, K::TILE);
          for (int c = 0; c < K::NCH; ++c)
            tma_load_4d(sbase + K::OFF_C + s2 * K::TILE + c * C * 128, &tc, c * 64, row, hh, z4, bar + Bz::C_FULL + 8 * s2);
          ++nc;
        }
      }
      if (!ok) record_error(LIN_ERR_WAIT);
      // copies must have landed before the block leaves
      for (int i = max(0, na - K::NA); i < na; ++i) mbar_wait(bar + Bz::A_FULL + 8 * (i % K::NA), (i / K::NA) & 1);
      for (int i = max(0, nb - K::NB); i < nb; ++i) mbar_wait(bar + Bz::B_FULL + 8 * (i % K::NB), (i / K::NB) & 1);
      for (int i = max(0, nc - K::NC); i < nc; ++i) mbar_wait(bar + Bz::C_FULL + 8 * (i % K::NC), (i / K::NC) & 1);
    }
    __syncwarp();
  } else if (warp == WARP_MMA) {
    constexpr uint32_t ID_P = idesc_f16(BF16 ? 1 : 0, C, C, 0, 0);
    constexpr uint32_t ID_T = idesc_f16(BF16 ? 1 : 0, C, D, 0, 1);                       // B along its rows
    constexpr uint32_t ID_I = idesc_f16(BF16 ? 1 : 0, C, D, 0, SWAP ? 0 : 1);            // O = a X: X [da][dc], or (SWAP) [dc][da]
    int ca = -1, cb = -1, cc = -1, nx = 0, nbt = 0, noi = 0;    // tiles taken, and steps signalled so far
    bool ok = true;
    for (int t = 0; ok && t < items; ++t) {
      const int g = t % groups;
      const bool first = g == 0, last = g == groups - 1, end = t / groups == chunks - 1;
      const bool do_b = (first || r.nb > 1) && !end, do_i = first || r.na > 1;
      const int cn = min(C, t1 - t0 - chunk_at(t));
      // P = a b^T
      if (first || r.na > 1) {
        ++ca;
        ok = ok && mbar_wait_warp(bar + Bz::A_FULL + 8 * (ca % K::NA), (ca / K::NA) & 1);
      }
      if (first || r.nb > 1) {
        ++cb;
        ++cc;
        ok = ok && mbar_wait_warp(bar + Bz::B_FULL + 8 * (cb % K::NB), (cb / K::NB) & 1);
        if (SWAP && cn < C && q.cu) {
          zero_rows(sgen + K::OFF_B + (cb % K::NB) * K::TILE, K::NCH, cn, lane);
          fence_proxy_async_smem();
          __syncwarp();
        }
      }
      if (t > 0) ok = ok && mbar_wait_warp(bar + Bz::PV_DONE, (t - 1) & 1);
      if (!ok) break;
      const uint32_t at = sbase + K::OFF_A + (ca % K::NA) * K::TILE, bt = sbase + K::OFF_B + (cb % K::NB) * K::TILE,
                     ct = sbase + K::OFF_C + (cc % K::NC) * K::TILE;
      tc_fence_after();
      if (lane == 0) {
        const uint64_t da = desc_k(at), db = desc_k(bt);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          mma_ss(tmem + K::P_COL, desc_add(da, step_k(kk, C)), desc_add(db, step_k(kk, C)), ID_P, kk > 0);
        mma_commit(bar + Bz::P_FULL);
      }
      __syncwarp();
      if (first || r.nb > 1) {
        ok = mbar_wait_warp(bar + Bz::C_FULL + 8 * (cc % K::NC), (cc / K::NC) & 1);
        if (ok && cn < C && q.cu) {
          zero_rows(sgen + K::OFF_C + (cc % K::NC) * K::TILE, K::NCH, cn, lane);
          fence_proxy_async_smem();
          __syncwarp();
        }
      }
      if (first) {
        ok = ok && mbar_wait_warp(bar + Bz::XS_READY, nx & 1);
        ++nx;
      }
      // X += (decayed rows)^T (rows)
      if (do_b) {
        ok = ok && mbar_wait_warp(bar + Bz::BT_READY, nbt & 1);
        ++nbt;
        tc_fence_after();
        if (ok && lane == 0) {
          const uint64_t d = desc_mn(SWAP ? bt : ct, C);
#pragma unroll
          for (int kk = 0; kk < C / 16; ++kk) {
            mma_ts(tmem + K::X_COL, tmem + K::BT_COL + 8 * kk, desc_add(d, kk * 128), ID_T, 1u);
            mma_ts(tmem + K::X_COL, tmem + K::BT_COL + 64 + 8 * kk, desc_add(d, kk * 128), ID_T, 1u);
          }
          mma_commit(bar + Bz::X_DONE);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (lane == 0 && (last || r.nb > 1)) mma_commit(bar + Bz::B_EMPTY + 8 * (cb % K::NB));
      // O = a X
      if (do_i) {
        if (t > 0) ok = mbar_wait_warp(bar + Bz::O_READ, (t - 1) & 1);
        tc_fence_after();
        if (ok && lane == 0) {
          const uint64_t da = desc_k(at);
          const uint64_t xh = SWAP ? desc_k(sbase + K::OFF_X) : desc_mn(sbase + K::OFF_X, D);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t s = SWAP ? step_k(kk, D) : (uint32_t)(kk * 128);
            mma_ss(tmem + K::O_COL, desc_add(da, step_k(kk, C)), desc_add(xh, s), ID_I, kk > 0);
            mma_ss(tmem + K::O_COL, desc_add(da, step_k(kk, C)), desc_add(xh, s + (K::XT >> 4)), ID_I, 1u);
          }
          mma_commit(bar + Bz::OI_FULL);
        }
        __syncwarp();
      }
      if (lane == 0 && (last || r.na > 1)) mma_commit(bar + Bz::A_EMPTY + 8 * (ca % K::NA));
      // O = P c, over what the elementwise warps have taken of a X or of the item before
      ok = ok && mbar_wait_warp(bar + Bz::P_READY, t & 1);
      if (do_i) {
        ok = ok && mbar_wait_warp(bar + Bz::OI_READ, noi & 1);
        ++noi;
      }
      if (!ok) break;
      tc_fence_after();
      if (lane == 0) {
        const uint64_t d = desc_mn(ct, C);
#pragma unroll
        for (int kk = 0; kk < C / 16; ++kk) {
          const uint32_t p = tmem + K::P_COL + 32 * (kk / 2) + 8 * (kk % 2);
          mma_ts(tmem + K::O_COL, p, desc_add(d, kk * 128), ID_T, kk > 0);
          mma_ts(tmem + K::O_COL, p + 16, desc_add(d, kk * 128), ID_T, 1u);
        }
        mma_commit(bar + Bz::PV_DONE);
        if (last || r.nb > 1) mma_commit(bar + Bz::C_EMPTY + 8 * (cc % K::NC));
      }
      __syncwarp();
    }
    if (!ok) record_error(LIN_ERR_WAIT);
    if (lane == 0) mma_commit(bar + Bz::DRAIN);
    __syncwarp();
    if (!mbar_wait_warp(bar + Bz::DRAIN, 0)) record_error(LIN_ERR_WAIT);
  } else {
    // ------------------------------------------------------------ elementwise
    const int qd = warp & 3, hf = warp >> 2, row = qd * 32 + lane;
    const uint32_t la = tmem + ((uint32_t)(qd * 32) << 16);
    constexpr int HD = D / 2;                       // state or output columns of a thread
    const int xl = SWAP ? r.dc : r.da, xn = SWAP ? r.da : r.dc;   // real rows (lanes) and columns of X
    const long long per = (long long)r.da * r.dc;
    const float* x0 = nullptr;
    if (ws) x0 = ws + (((long long)z * q.nhk + h) * q.nseg + n) * per;
    else if (pool.in && !(pool.seen && pool.seen[z] <= 0)) x0 = pool.in + ((long long)slot * q.nhk + h) * per;
    float acc[HD];                    // this thread's part of an output row: a X first, then P c of each item
    float p_inv = 1.f, x_inv = 1.f;
    bool ok = true;                   // false once a wait has given up: the warp goes on without waiting (the named barriers stay matched)
    int nx = 0, nbt = 0, noi = 0, cbw = -1;
    const auto wait = [&](int which, int phase) {
      ok = ok && mbar_wait_warp(bar + which, phase & 1);
      __syncwarp();
      tc_fence_after();
    };
    const uint32_t obox = K::OFF_O + warp * 32 * HD * 2;
    const auto epilogue = [&](int t) {
      const int at = chunk_at(t), cn = min(C, t1 - t0 - at), g = r.na > 1 ? t % groups : 0;
#pragma unroll
      for (int c0 = 0; c0 < HD; c0 += 32) {
        float o[32];
        tmem_ld32(la + K::O_COL + hf * HD + c0, o);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[c0 + i] = fmaf(o[i], p_inv, acc[c0 + i]);
      }
      tc_fence_before();
      mbar_arrive(bar + Bz::O_READ);
      if ((r.na == 1 && t % groups != groups - 1) || hf * HD >= r.dc) return;
      // 32 whole rows go out as one box; rows next to another sequence's one by one
      const bool whole = qd * 32 + 32 <= cn;
      T* orow = out + (long long)(at + row) * r.so.s + g * r.so.h + hf * HD;
      if (whole) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
      }
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const uint4 w = make_uint4(pack2<BF16>(acc[8 * i], acc[8 * i + 1]), pack2<BF16>(acc[8 * i + 2], acc[8 * i + 3]),
                                   pack2<BF16>(acc[8 * i + 4], acc[8 * i + 5]), pack2<BF16>(acc[8 * i + 6], acc[8 * i + 7]));
        if (whole)      // 128-byte or 64-byte swizzle
          *reinterpret_cast<uint4*>(sgen + obox + lane * HD * 2 + ((i ^ (HD == 64 ? lane & 7 : (lane >> 1) & 3)) << 4)) = w;
        else if (row < cn && hf * HD + 8 * i < r.dc)
          *reinterpret_cast<uint4*>(orow + 8 * i) = w;
      }
      if (whole) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tma_store_4d(&to, sbase + obox, hf * HD, (int)span.row0 + t0 + at + qd * 32, h * r.na + g, q.cu ? 0 : z);
      }
    };
    float2 w_rows[8];
    int w_cn = 0;
    // Factors of the pair products: a block of 32 rows x 32 columns beside the diagonal takes lam^(rows from its near edge) times
    // lam^(columns from it), both at most 1, so that nothing overflows however fast the decay
    float u_blk[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int j0 = hf * 64 + 32 * b;
      u_blk[b] = lam[REV ? max(j0 - row, 0) : max(row - j0 - 31, 0)];
    }
    for (int t = 0; t < items; ++t) {
      const int g = t % groups;
      const bool first = g == 0, end = t / groups == chunks - 1;
      const bool do_b = (first || r.nb > 1) && !end, do_i = first || r.na > 1;
      const int cn = min(C, t1 - t0 - chunk_at(t));
      // ---- decayed rows, transposed
      if (first || r.nb > 1) ++cbw;
      if (do_b) {
        if (cn != w_cn) {
          row_factors<REV>(w_rows, lam, r.w_up, hf, lane, cn);
          w_cn = cn;
        }
        const int stages = SWAP ? K::NC : K::NB, s = cbw % stages;
        wait((SWAP ? Bz::C_FULL : Bz::B_FULL) + 8 * s, cbw / stages);
        if (nbt > 0) wait(Bz::X_DONE, nbt - 1);
        if (qd * 32 < D)
          decay_rows<BF16, 2>(sbase + (SWAP ? K::OFF_C : K::OFF_B) + s * K::TILE, la + K::BT_COL, w_rows, qd, hf, lane, cn);
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(bar + Bz::BT_READY);
        ++nbt;
      }
      // ---- epilogue of the item before
      if (t > 0) {
        wait(Bz::PV_DONE, t - 1);
        epilogue(t - 1);
      }
      // ---- the state: hi + lo to shared memory, lam^C X back to TMEM
      if (first) {
        float x[HD];
        if (t > 0) {
          wait(Bz::X_DONE, nbt - 1 - (do_b ? 1 : 0));      // every update before this chunk's has landed
          if (qd * 32 < D) {
#pragma unroll
            for (int c0 = 0; c0 < HD; c0 += 32) tmem_ld32(la + K::X_COL + hf * HD + c0, x + c0);
            tc_wait_ld();
          }
        } else {
#pragma unroll
          for (int i = 0; i < HD; ++i) {
            const int col = hf * HD + i;
            const int ii = SWAP ? col : row, jj = SWAP ? row : col;
            x[i] = x0 && row < xl && col < xn ? x0[r.transposed ? (long long)jj * r.da + ii : (long long)ii * r.dc + jj] : 0.f;
          }
        }
        float xs = 1.f;
        if constexpr (!BF16) {
          float top = 0.f;
          if (qd * 32 < D) {
#pragma unroll
            for (int i = 0; i < HD; ++i) top = fmaxf(top, fabsf(x[i]));
          }
          const uint32_t all = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
          if (lane == 0) atomicMax(&xmax[nx & 1], all);
          bar_elem();
          xs = scale_to(xmax[nx & 1]);
          if (tid == 0) xmax[(nx + 1) & 1] = 0;
          x_inv = 1.f / xs;
        }
        const float keep = lam[cn];
        if (qd * 32 < D) {
          uint8_t* xr = sgen + K::OFF_X + row * 128;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) split2<BF16>(__fmul2_rn(make_float2(x[8 * i + 2 * k], x[8 * i + 2 * k + 1]), make_float2(xs, xs)), hi[k], lo[k]);
            const int col = hf * HD + 8 * i;
            uint8_t* to_x = xr + (col / 64) * D * 128 + ((((col % 64) / 8) ^ (row & 7)) << 4);
            *reinterpret_cast<uint4*>(to_x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(to_x + K::XT) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
#pragma unroll
          for (int i = 0; i < HD; ++i) x[i] *= keep;
#pragma unroll
          for (int c0 = 0; c0 < HD; c0 += 32) tmem_st32(la + K::X_COL + hf * HD + c0, reinterpret_cast<const uint32_t*>(x + c0));
        }
        tc_wait_st();
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(bar + Bz::XS_READY);
        ++nx;
      }
      // ---- pair products: decay, mask, back to TMEM as hi + lo
      wait(Bz::P_FULL, t);
      {
        float2 p[2][16];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int j0 = hf * 64 + 32 * b, side = REV ? j0 / 32 - qd : qd - j0 / 32;      // 0 on the diagonal, below 0 where nothing is seen
          if (side < 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) p[b][i] = make_float2(0.f, 0.f);
            continue;
          }
          tmem_ld32(la + K::P_COL + j0, reinterpret_cast<float*>(p[b]));
          tc_wait_ld();
          if (side > 0) {
            const float2 u = make_float2(u_blk[b], u_blk[b]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {      // columns from the near edge: lam^(31 - j), or lam^j reversed
              const float2 w = REV ? make_float2(lam[2 * i], lam[2 * i + 1]) : make_float2(lam[31 - 2 * i], lam[30 - 2 * i]);
              p[b][i] = __fmul2_rn(p[b][i], __fmul2_rn(u, w));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int gap = REV ? 2 * i - lane : lane - 2 * i, next = REV ? gap + 1 : gap - 1;
              p[b][i].x = gap >= 0 ? p[b][i].x * lam[max(gap, 0)] : 0.f;
              p[b][i].y = next >= 0 ? p[b][i].y * lam[max(next, 0)] : 0.f;
            }
          }
          if (REV && cn < C) {                  // forward, a row sees no token past its own
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (j0 + 2 * i >= cn) p[b][i].x = 0.f;
              if (j0 + 2 * i + 1 >= cn) p[b][i].y = 0.f;
            }
          }
        }
        float ps = 1.f;
        if constexpr (!BF16) {
          float top = 0.f;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(fabsf(p[b][i].x), fabsf(p[b][i].y)));
          pmax[hf * C + row] = __float_as_uint(top);
          bar_pair(qd);
          ps = scale_to(max(__float_as_uint(top), pmax[(hf ^ 1) * C + row]));
          bar_pair(qd);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) split2<BF16>(BF16 ? p[b][i] : __fmul2_rn(p[b][i], make_float2(ps, ps)), w[i], w[16 + i]);
          tmem_st32(la + K::P_COL + hf * 64 + 32 * b, w);
        }
        p_inv = r.w_intra / ps;
      }
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(bar + Bz::P_READY);
      // ---- a X
      if (do_i) {
        wait(Bz::OI_FULL, noi);
        ++noi;
        const float mul = r.w_inter * lam[REV ? max(cn - 1 - row, 0) : min(row + 1, C)] * x_inv;
#pragma unroll
        for (int c0 = 0; c0 < HD; c0 += 32) tmem_ld32(la + K::O_COL + hf * HD + c0, acc + c0);
        tc_wait_ld();
        tc_fence_before();
        mbar_arrive(bar + Bz::OI_READ);
#pragma unroll
        for (int i = 0; i < HD; ++i) acc[i] *= mul;
      }
    }
    wait(Bz::PV_DONE, items - 1);
    epilogue(items - 1);
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
    if (!ok) record_error(LIN_ERR_WAIT);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// =====================================================================================
// states: what a segment adds to the state, X = sum_j (lam^m_j b_j)^T c_j with powers up to the segment's own end, so that
// nothing is scaled on the way.  The result is a state that a caller may keep, in fp32, so the decayed rows enter as three bf16 numbers
// (2^-24 of a term) or two fp16 ones (2^-22).  The tensor cores truncate each accumulation; so every item is summed from 0, its small
// terms first (only the eight steps of the largest one then cut at the sum's full size), and items are added in registers, to nearest.
// One accumulator over a whole segment had left 2e-6 of the state.  Bound by reading b and c once.
// =====================================================================================
template <int D, bool BF16>
struct StCfg {
  static constexpr int NCH = D / 64, TILE = C * D * 2, NS = D == 128 ? 3 : 4, TERMS = BF16 ? 3 : 2;
  static constexpr int OFF_T = 0, OFF_BAR = NS * 2 * TILE, OFF_LAM = OFF_BAR + 128;
  static constexpr int SMEM = OFF_LAM + 132 * 4 + 1024;
  static constexpr uint32_t X_COL = 0, BT_COL = 128, BT_COLS = 192;      // two buffers of decayed rows
  static_assert(SMEM <= 232448, "shared memory per CTA");
};
struct StBz {
  static constexpr int FULL = 0, EMPTY = 32, BT_READY = 64, DONE = 80, X_READ = 88, DRAIN = 96, TMEM_ADDR = 104;
};

template <int D, bool BF16, bool REV>
__global__ void __launch_bounds__(NTHREADS, 1)
    lin_tc_states_kernel(const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap tc, const LinSeqs q, const LinRole r,
                         float* ws) {
  using K = StCfg<D, BF16>;
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = blockIdx.x % q.nseg, h = blockIdx.x / q.nseg % q.nhk, z = blockIdx.x / q.nseg / q.nhk;
  const LinSpan span = lin_span(q, z);
  int t0, t1;
  lin_segment(q, span.len, n, t0, t1);
  if (t1 <= t0) return;
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t bar = sbase + K::OFF_BAR;
  float* lam = reinterpret_cast<float*>(sgen + K::OFF_LAM);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sgen + K::OFF_BAR + StBz::TMEM_ADDR);
  const int chunks = (t1 - t0 + C - 1) / C, items = chunks * r.nb;
  const float g2 = lin_log2_decay(q.log_decay, h);
  if (tid == 0) {
    for (int s = 0; s < K::NS; ++s) {
      mbar_init(bar + StBz::FULL + 8 * s, 1);
      mbar_init(bar + StBz::EMPTY + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) mbar_init(bar + StBz::BT_READY + 8 * s, NELEM);
    mbar_init(bar + StBz::DONE, 1);
    mbar_init(bar + StBz::X_READ, NELEM);
    mbar_init(bar + StBz::DRAIN, 1);
    fence_barrier_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  if (tid <= C) lam[tid] = lin_power(g2, tid);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const auto tile = [&](int i) { return K::OFF_T + (i % K::NS) * 2 * K::TILE; };      // b, then c

  if (warp == WARP_TMA) {
    if (lane == 0) {
      bool ok = true;
      int i = 0;
      for (; i < items; ++i) {
        const int s = i % K::NS, row = (int)span.row0 + t0 + i / r.nb * C, hh = h * r.nb + i % r.nb, z4 = q.cu ? 0 : z;
        if (i >= K::NS && !mbar_wait(bar + StBz::EMPTY + 8 * s, ((i / K::NS) - 1) & 1)) { ok = false; break; }
        mbar_expect_tx(bar + StBz::FULL + 8 * s, 2 * K::TILE);
        for (int c = 0; c < K::NCH; ++c) {
          tma_load_4d(sbase + tile(i) + c * C * 128, &tb, c * 64, row, hh, z4, bar + StBz::FULL + 8 * s);
          tma_load_4d(sbase + tile(i) + K::TILE + c * C * 128, &tc, c * 64, row, hh, z4, bar + StBz::FULL + 8 * s);
        }
      }
      if (!ok) record_error(LIN_ERR_WAIT);
      for (int k = max(0, i - K::NS); k < i; ++k) mbar_wait(bar + StBz::FULL + 8 * (k % K::NS), (k / K::NS) & 1);
    }
    __syncwarp();
  } else if (warp == WARP_MMA) {
    constexpr uint32_t ID = idesc_f16(BF16 ? 1 : 0, C, D, 0, 1);
    bool ok = true;
    for (int i = 0; ok && i < items; ++i) {
      const int s = i % K::NS, cn = min(C, t1 - t0 - i / r.nb * C);
      ok = mbar_wait_warp(bar + StBz::FULL + 8 * s, (i / K::NS) & 1);
      if (ok && cn < C && q.cu) {
        zero_rows(sgen + tile(i) + K::TILE, K::NCH, cn, lane);
        fence_proxy_async_smem();
        __syncwarp();
      }
      ok = ok && mbar_wait_warp(bar + StBz::BT_READY + 8 * (i & 1), (i >> 1) & 1);
      if (i > 0) ok = ok && mbar_wait_warp(bar + StBz::X_READ, (i - 1) & 1);
      tc_fence_after();
      if (ok && lane == 0) {
        const uint64_t d = desc_mn(sbase + tile(i) + K::TILE, C);
        const uint32_t bt = tmem + K::BT_COL + (i & 1) * K::BT_COLS;
#pragma unroll
        for (int w = K::TERMS - 1; w >= 0; --w)
#pragma unroll
          for (int kk = 0; kk < C / 16; ++kk)
            mma_ts(tmem + K::X_COL, bt + 64 * w + 8 * kk, desc_add(d, kk * 128), ID, kk > 0 || w < K::TERMS - 1);
        mma_commit(bar + StBz::EMPTY + 8 * s);
        mma_commit(bar + StBz::DONE);
      }
      __syncwarp();
    }
    if (!ok) record_error(LIN_ERR_WAIT);
    if (lane == 0) mma_commit(bar + StBz::DRAIN);
    __syncwarp();
    if (!mbar_wait_warp(bar + StBz::DRAIN, 0)) record_error(LIN_ERR_WAIT);
  } else {
    const int qd = warp & 3, hf = warp >> 2, row = qd * 32 + lane;
    const uint32_t la = tmem + ((uint32_t)(qd * 32) << 16);
    bool ok = true;
    float acc[D / 2];
#pragma unroll
    for (int i = 0; i < D / 2; ++i) acc[i] = 0.f;
    const auto add = [&](int i) {      // item i's sum
      ok = ok && mbar_wait_warp(bar + StBz::DONE, i & 1);
      __syncwarp();
      tc_fence_after();
#pragma unroll
      for (int c0 = 0; c0 < D / 2; c0 += 32) {
        float v[32];
        tmem_ld32(la + K::X_COL + hf * (D / 2) + c0, v);
        tc_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k) acc[c0 + k] += v[k];
      }
      tc_fence_before();
      mbar_arrive(bar + StBz::X_READ);
    };
    float2 w_rows[8];
    int w_cn = 0;
    for (int i = 0; i < items; ++i) {
      // the buffer of decayed rows is free: item i - 2 was added up
      const int at = i / r.nb * C, cn = min(C, t1 - t0 - at);
      ok = ok && mbar_wait_warp(bar + StBz::FULL + 8 * (i % K::NS), (i / K::NS) & 1);
      __syncwarp();
      if (cn != w_cn) {
        row_factors<REV>(w_rows, lam, 1.f, hf, lane, cn);
        w_cn = cn;
      }
      const float far = lin_power(g2, REV ? at : t1 - t0 - at - cn);
      float2 w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = __fmul2_rn(w_rows[k], make_float2(far, far));
      if (qd * 32 < D) decay_rows<BF16, K::TERMS>(sbase + tile(i), la + K::BT_COL + (i & 1) * K::BT_COLS, w, qd, hf, lane, cn);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(bar + StBz::BT_READY + 8 * (i & 1));
      if (i > 0) add(i - 1);
    }
    add(items - 1);
    float* x = ws + (((long long)z * q.nhk + h) * q.nseg + n) * r.da * r.dc + (long long)row * r.dc;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const int col = hf * (D / 2) + 4 * i;
      if (row < r.da && col < r.dc)
        *reinterpret_cast<float4*>(x + col) = make_float4(r.w_up * acc[4 * i], r.w_up * acc[4 * i + 1], r.w_up * acc[4 * i + 2], r.w_up * acc[4 * i + 3]);
    }
    if (!ok) record_error(LIN_ERR_WAIT);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- host side
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &res) != cudaSuccess || res != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return (PFN_cuTensorMapEncodeTiled_v12000)ptr;
  }();
  return fn;
}

// boxes of `cols` columns (64, or 32) x `box_rows` rows over [batch][heads][rows][dim]; false where the layout does not allow it
bool map4(CUtensorMap* m, const void* base, bool bf16, int dim, long long rows, long long heads, long long batch, const FaStrides& st,
          int cols = 64, int box_rows = C) {
  const auto enc = encode_fn();
  if (!enc || (uintptr_t)base % 16) return false;
  // a stride that no second entry uses says nothing: any that is allowed will do
  const long long ss = rows > 1 ? st.s : (dim + 7) / 8 * 8, sh = heads > 1 ? st.h : (dim + 7) / 8 * 8, sb = batch > 1 ? st.b : (dim + 7) / 8 * 8;
  const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batch};
  const cuuint64_t strides[3] = {(cuuint64_t)ss * 2, (cuuint64_t)sh * 2, (cuuint64_t)sb * 2};
  for (int i = 0; i < 3; ++i)
    if (strides[i] == 0 || strides[i] % 16 || strides[i] >= (1ull << 40)) return false;
  const cuuint32_t box[4] = {(cuuint32_t)cols, (cuuint32_t)box_rows, 1, 1}, estr[4] = {1, 1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool takes(const LinSeqs& q, const LinRole& r, int dtype) {
  return dtype != FA_DTYPE_F32 && r.da <= 128 && r.dc <= 128 && (q.cu ? q.total > 0 : q.S > 0) && q.total < (1ll << 31) - 256;
}

template <typename Kernel, typename... Args>
int launch(Kernel kernel, int smem, unsigned long long* done, const LinSeqs& q, cudaStream_t st, const Args&... args) {
  const long long grid = (long long)q.batch * q.nhk * q.nseg;
  FA_CHECK_ARG(grid < (1ll << 31), "linear attention: %lld blocks", grid);
  if (int rc = ensure_smem((const void*)kernel, smem, done)) return rc;
  kernel<<<(int)grid, NTHREADS, smem, st>>>(args...);
  count_launch();
  return cuda_status(cudaGetLastError(), "linear attention (tensor cores) launch");
}

template <int D, bool BF16>
int run_main(const LinSeqs& q, const LinRole& r, bool rev, const float* ws, const LinPool& pool, cudaStream_t st, const CUtensorMap* m) {
  static unsigned long long done[3] = {};
  // dk: the output is along the state's rows as it is stored
  if (rev && r.transposed) return launch(lin_tc_kernel<D, BF16, true, true>, Cfg<D>::SMEM, done, q, st, m[0], m[1], m[2], m[3], q, r, ws, pool);
  if (rev) return launch(lin_tc_kernel<D, BF16, true, false>, Cfg<D>::SMEM, done + 1, q, st, m[0], m[1], m[2], m[3], q, r, ws, pool);
  return launch(lin_tc_kernel<D, BF16, false, false>, Cfg<D>::SMEM, done + 2, q, st, m[0], m[1], m[2], m[3], q, r, ws, pool);
}
template <int D, bool BF16>
int run_states(const LinSeqs& q, const LinRole& r, bool rev, float* ws, cudaStream_t st, const CUtensorMap* m) {
  static unsigned long long done[2] = {};
  using K = StCfg<D, BF16>;
  if (rev) return launch(lin_tc_states_kernel<D, BF16, true>, K::SMEM, done, q, st, m[0], m[1], q, r, ws);
  return launch(lin_tc_states_kernel<D, BF16, false>, K::SMEM, done + 1, q, st, m[0], m[1], q, r, ws);
}
}  // namespace

namespace fa {
bool lin_tc_takes(const LinSeqs& q, const LinRole& r, int dtype) { return takes(q, r, dtype); }

int lin_tc_main(const LinSeqs& q, const LinRole& r, bool rev, const float* ws, const LinPool& pool, int dtype, cudaStream_t st, bool* taken) {
  *taken = false;
  if (!takes(q, r, dtype) || (pool.out && !ws)) return FA_OK;
  const bool bf16 = dtype == FA_DTYPE_BF16;
  const long long rows = q.cu ? q.total : q.S, zs = q.cu ? 1 : q.batch;
  const bool small = r.da <= 64 && r.dc <= 64;
  CUtensorMap m[4];
  if (!map4(m, r.a, bf16, r.da, rows, (long long)q.nhk * r.na, zs, r.sa) || !map4(m + 1, r.b, bf16, r.da, rows, (long long)q.nhk * r.nb, zs, r.sb) ||
      !map4(m + 2, r.c, bf16, r.dc, rows, (long long)q.nhk * r.nb, zs, r.sc) ||
      !map4(m + 3, r.out, bf16, r.dc, rows, (long long)q.nhk * r.na, zs, r.so, small ? 32 : 64, 32))
    return FA_OK;
  *taken = true;
  if (bf16) return small ? run_main<64, true>(q, r, rev, ws, pool, st, m) : run_main<128, true>(q, r, rev, ws, pool, st, m);
  return small ? run_main<64, false>(q, r, rev, ws, pool, st, m) : run_main<128, false>(q, r, rev, ws, pool, st, m);
}

int lin_tc_states(const LinSeqs& q, const LinRole& r, bool rev, float* ws, int dtype, cudaStream_t st, bool* taken) {
  *taken = false;
  if (!takes(q, r, dtype)) return FA_OK;
  const bool bf16 = dtype == FA_DTYPE_BF16;
  const long long rows = q.cu ? q.total : q.S, zs = q.cu ? 1 : q.batch;
  CUtensorMap m[2];
  if (!map4(m, r.b, bf16, r.da, rows, (long long)q.nhk * r.nb, zs, r.sb) || !map4(m + 1, r.c, bf16, r.dc, rows, (long long)q.nhk * r.nb, zs, r.sc))
    return FA_OK;
  *taken = true;
  const bool small = r.da <= 64 && r.dc <= 64;
  if (bf16) return small ? run_states<64, true>(q, r, rev, ws, st, m) : run_states<128, true>(q, r, rev, ws, st, m);
  return small ? run_states<64, false>(q, r, rev, ws, st, m) : run_states<128, false>(q, r, rev, ws, st, m);
}

int lin_tc_device_error(int clear) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_lin_tc_error, sizeof(int));
  if (clear && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_lin_tc_error, &zero, sizeof(int));
  }
  return v;
}
}  // namespace fa
