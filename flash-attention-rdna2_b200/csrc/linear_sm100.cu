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
// left as they are: where they fall below 2^-14 their steps are 2^-24, which is fp16's own step for such inputs.  A scale that they carry
// (w_up of the reversed passes) is brought to (1/2, 1] by a power of 2 that X is held in: a scale of 64 would take inputs of 1024 past
// fp16's range, and one of 2^-14 leave them ten bits.
//
// Warp roles (640 threads, five warpgroups):
//   0-7    outputs: pair products on their way back to TMEM, a X, epilogue; two warps to a TMEM lane quadrant (w % 4), half of the columns each
//   8-15   state: X to shared memory and lam^C X back to TMEM, decayed rows; two warps to a quadrant likewise (four warps for each of the
//          two steps took longer)
//   16     TMA
//   17-19  MMAs: P = a b^T and O = P c; O = a X; X += ..  One thread alone issues an MMA in 85 to 110 cycles and the pipe takes 64, and
//          none of the three waits for what only another needs
// What a chunk needs is a chain of short steps, each a TMEM or shared memory latency long, and not their instructions: one
// set of warps that took all steps in turn needed 10000 cycles a chunk, issuing every third cycle.  Outputs of item t and the state
// of the next chunk depend on each other through the MMAs alone, so two sets run them side by side.  Registers follow the need (setmaxnreg): the epilogue holds 64 columns.  Every wait is bounded.
#include <cudaTypedefs.h>
#include <algorithm>
#include <cmath>
#include "linear_common.cuh"
#include "fa_launch.h"
#include "sm100_ptx.cuh"

namespace {

using namespace sm100;
using namespace fa;

constexpr int C = 128;               // tokens of a chunk
constexpr int NTHREADS = 640, NOUT = 256, NSTATE = 256, WARP_TMA = 16, WARP_MMA = 17, WARP_MMA2 = 18, WARP_MMA3 = 19;
// registers a thread: launched with REGS; 2 x 136 + 2 x 80 + 48 = 5 x 96
constexpr int REGS = 96;
__device__ __forceinline__ void regs_out() { asm volatile("setmaxnreg.inc.sync.aligned.u32 136;"); }
__device__ __forceinline__ void regs_state() { asm volatile("setmaxnreg.dec.sync.aligned.u32 80;"); }
__device__ __forceinline__ void regs_few() { asm volatile("setmaxnreg.dec.sync.aligned.u32 48;"); }
constexpr int NTHREADS_ST = 576, NELEM_ST = 512;      // the states kernel: 16 elementwise warps
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

// The decayed rows of a chunk, transposed for the A operand in TMEM: a warp takes 32 dims and 16 N tokens from `first` on.  Its thread
// reads pairs of tokens first + 16 s + 8 m + 2 (lane % 4) (+ 1), whose factors w[2 s + m] stay in registers from chunk to
// chunk.  Element by element from shared memory this took 6000 cycles a chunk.
template <bool REV, int N>
__device__ __forceinline__ void row_factors(float2* w, const float* lam, float times, int first, int lane, int cn) {
#pragma unroll
  for (int i = 0; i < 2 * N; ++i) {
    const int j = first + 8 * i + 2 * (lane & 3);
    w[i].x = j < cn ? times * lam[REV ? j + 1 : cn - 1 - j] : 0.f;
    w[i].y = j + 1 < cn ? times * lam[REV ? j + 2 : cn - 2 - j] : 0.f;
  }
}
// With LO_SHIFT the second term is stored 2^LO_SHIFT times as large.
template <bool BF16, int TERMS, int N, int LO_SHIFT = 0>
__device__ __forceinline__ void decay_rows(uint32_t tile, uint32_t bt, const float2* w, int qd, int first, int lane, int cn) {
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {          // 16 dims each
    const int unit = 4 * (qd & 1) + 2 * half + ((lane >> 3) & 1), token = first + 8 * (lane >> 4) + (lane & 7);
    const uint32_t from = tile + (qd >> 1) * C * 128 + token * 128 + ((unit ^ (lane & 7)) << 4);
    const uint32_t to = bt + ((uint32_t)(16 * half) << 16) + first / 2;
    uint32_t r[N][4];
#pragma unroll
    for (int s = 0; s < N; ++s) ldsm_t4(from + s * 16 * 128, r[s]);
#pragma unroll
    for (int s = 0; s < N; ++s) {                 // 16 tokens each
      uint32_t o[3][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {               // blocks: dims 0-7 and 8-15 of the first 8 tokens, then of the next 8
        if (cn < C) {                             // rows past the sequence may hold anything: a factor of 0 is not enough
          const int j = first + 16 * s + 8 * (i >> 1) + 2 * (lane & 3);
          r[s][i] &= (j < cn ? 0xffffu : 0u) | (j + 1 < cn ? 0xffff0000u : 0u);
        }
        float2 x = __fmul2_rn(unpack2<BF16>(r[s][i]), w[2 * s + (i >> 1)]);
#pragma unroll
        for (int u = 0; u < TERMS; ++u) {
          o[u][i] = pack2<BF16>(x.x, x.y);
          if (u + 1 < TERMS) x = rest2<BF16>(x, o[u][i]);
          if (LO_SHIFT && u == 0) x = __fmul2_rn(x, make_float2(float(1 << LO_SHIFT), float(1 << LO_SHIFT)));
        }
      }
#pragma unroll
      for (int u = 0; u < TERMS; ++u) tmem_st_16x8(to + 64 * u + 8 * s, o[u]);
    }
  }
}

// N = 16 or 32 fp32 columns of this thread's lane
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, float2* v) {
  if constexpr (N == 32) tmem_ld32(taddr, reinterpret_cast<float*>(v));
  else tmem_ld16(taddr, reinterpret_cast<float*>(v));
  tc_wait_ld();
}
template <int N>
__device__ __forceinline__ void tmem_store(uint32_t taddr, const float2* v) {
  if constexpr (N == 32) tmem_st32(taddr, reinterpret_cast<const uint32_t*>(v));
  else tmem_st16(taddr, reinterpret_cast<const uint32_t*>(v));
}

// descriptors of a [rows][D] tile stored as D / 64 chunks of rows x 128 bytes (128-byte swizzle)
__device__ __forceinline__ uint64_t desc_k(uint32_t tile) { return sdesc_sw128(tile, 16, 1024); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, int rows) { return sdesc_sw128(tile, rows * 128, 1024); }

// Bounded warp-uniform wait, in few instructions: the kernel has some thirty of them, and what bounded it was the fetching of
// instructions (a quarter of all stalls) while its steps were unrolled in full.  Gives up after 8e9 cycles, about 4 s.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const long long from = clock64();
  while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
    if (__any_sync(0xffffffffu, clock64() - from > 8000000000ll)) return false;
  return true;
}

__device__ __forceinline__ void bar_state() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void bar_quadrant(int quadrant) { asm volatile("bar.sync %0, 64;" ::"r"(2 + quadrant) : "memory"); }

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
template <int D, bool SWAP>
struct Cfg {
  static constexpr int NCH = D / 64;
  static constexpr int TILE = C * D * 2;            // a, b or c
  static constexpr int XT = D * D * 2;              // X hi or lo
  // two buffers for the rows that the state warps run ahead with; the others are free again before they are missed
  static constexpr int NA = D == 128 ? 1 : 2, NB = D == 128 && SWAP ? 1 : 2, NC = D == 128 && !SWAP ? 1 : 2;
  static constexpr int OFF_X = 0, OFF_A = 2 * XT, OFF_B = OFF_A + NA * TILE, OFF_C = OFF_B + NB * TILE;
  static constexpr int OFF_O = OFF_C + NC * TILE;   // outputs on their way: a box of 32 rows x D / 2 columns for each output warp
  static constexpr int OFF_BAR = OFF_O + TILE;
  static constexpr int OFF_LAM = OFF_BAR + 224;     // lam^n, n = 0 .. 128
  static constexpr int OFF_LAMC = OFF_LAM + 528;    // of a block's 32 columns: lam^(31 - j), or lam^j reversed
  static constexpr int OFF_MAX = OFF_LAMC + 128;    // fp16: [3] largest |X|, then [2][128] largest |P| of half a row
  static constexpr int SMEM = OFF_MAX + 16 + 2 * C * 4 + 1024;
  static constexpr uint32_t P_COL = 0, BT_COL = 128, X_COL = 256, O_COL = 256 + D;
  static_assert(SMEM <= 232448, "shared memory per CTA");
};
struct Bz {
  static constexpr int A_FULL = 0, A_EMPTY = 16, B_FULL = 32, B_EMPTY = 48, C_FULL = 64, C_EMPTY = 80, P_FULL = 96, P_READY = 104,
                       PV_DONE = 112, XS_READY = 120, BT_READY = 128, X_DONE = 136, OI_FULL = 144, OI_READ = 152, O_READ = 160,
                       DRAIN = 168, X_READ = 192, TMEM_ADDR = 200;
};

// MULTI: b and c have several heads (nb > 1)
template <int D, bool BF16, bool REV, bool SWAP, bool MULTI>
__global__ void __launch_bounds__(NTHREADS, 1)
    lin_tc_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap tc,
                  const __grid_constant__ CUtensorMap to, const LinSeqs q, const LinRole r, const float* ws, const LinPool pool) {
  using K = Cfg<D, SWAP>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x % q.nhk, seg = blockIdx.x / q.nhk;
  lin_zero_outside<T>(q, r, h * r.na, seg, q.slots, NTHREADS);
  int z, t0, t1;
  const LinSpan span = lin_segment(q, seg, z, t0, t1);
  if (t1 <= t0) return;
  const int slot = lin_slot(pool, z, NTHREADS, &g_lin_tc_error);
  const int tokens = t1 - t0, row_first = (int)span.row0 + t0, z4 = q.cu ? 0 : z;      // rows of the maps
  if (slot < 0) {
    T* out = (T*)r.out + z4 * r.so.b + row_first * r.so.s + (long long)h * r.na * r.so.h;
    for (int g = 0; g < r.na; ++g)
      for (long long e = tid; e < (long long)tokens * r.dc; e += NTHREADS)
        out[e / r.dc * r.so.s + g * r.so.h + e % r.dc] = Elem<T>::from_f(0.f);
    return;
  }
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t bar = sbase + K::OFF_BAR;
  float* lam = reinterpret_cast<float*>(sgen + K::OFF_LAM);
  float* lamc = reinterpret_cast<float*>(sgen + K::OFF_LAMC);
  uint32_t* xmax = reinterpret_cast<uint32_t*>(sgen + K::OFF_MAX);
  uint32_t* pmax = xmax + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sgen + K::OFF_BAR + Bz::TMEM_ADDR);
  const int chunks = (tokens + C - 1) / C, groups = max(r.na, r.nb), items = chunks * groups;
  const float g2 = lin_log2_decay(q.log_decay, h);

  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar + Bz::A_FULL + 8 * s, 1);
      mbar_init(bar + Bz::A_EMPTY + 8 * s, 2);      // both MMA warps
      mbar_init(bar + Bz::B_FULL + 8 * s, 1);
      mbar_init(bar + Bz::B_EMPTY + 8 * s, 2);
      mbar_init(bar + Bz::C_FULL + 8 * s, 1);
      mbar_init(bar + Bz::C_EMPTY + 8 * s, 2);
      mbar_init(bar + Bz::DRAIN + 8 * s, 1);
    }
    mbar_init(bar + Bz::P_FULL, 1);
    mbar_init(bar + Bz::P_READY, NOUT);
    mbar_init(bar + Bz::PV_DONE, 1);
    mbar_init(bar + Bz::XS_READY, NSTATE);
    mbar_init(bar + Bz::BT_READY, NSTATE);
    mbar_init(bar + Bz::X_DONE, 1);
    mbar_init(bar + Bz::X_READ, 1);
    mbar_init(bar + Bz::DRAIN + 16, 1);
    mbar_init(bar + Bz::OI_FULL, 1);
    mbar_init(bar + Bz::OI_READ, NOUT);
    mbar_init(bar + Bz::O_READ, NOUT);
    xmax[0] = xmax[1] = xmax[2] = 0;
    fence_barrier_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  if (tid <= C) lam[tid] = lin_power(g2, tid);
  if (tid < 32) lamc[tid] = lin_power(g2, REV ? tid : 31 - tid);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;        // all 512 columns are this block's
  if (tid == 0 && *tmem_slot != tmem) record_error(LIN_ERR_WAIT);

  // item t = ck * groups + g: chunk ck (from the end where reversed), head g of the side that has several
  const auto chunk_at = [&](int ck) { return (REV ? chunks - 1 - ck : ck) * C; };

  if (warp >= WARP_TMA) {
    regs_few();
    if (warp == WARP_TMA && lane == 0) {
      int na = 0, nb = 0, nc = 0;
      bool ok = true;
      for (int ck = 0, g = 0; ok && ck < chunks; ++g == groups ? g = 0, ++ck : 0) {
        const int row = row_first + chunk_at(ck);
        const auto load = [&](const CUtensorMap* map, int full, int empty, int off, int stages, int& i, int head) {
          const int s = i % stages;
          if (i >= stages) ok = ok && mbar_wait(bar + empty + 8 * s, ((i / stages) - 1) & 1);
          if (!ok) return;
          mbar_expect_tx(bar + full + 8 * s, K::TILE);
          for (int c = 0; c < K::NCH; ++c) tma_load_4d(sbase + off + s * K::TILE + c * C * 128, map, c * 64, row, head, z4, bar + full + 8 * s);
          ++i;
        };
        // the rows for the state first (two buffers), a next (free after a X), last what the end of an item reads
        const bool new_b = g == 0 || r.nb > 1;
        const int hb = h * r.nb + (r.nb > 1 ? g : 0);
        if (new_b && SWAP) load(&tc, Bz::C_FULL, Bz::C_EMPTY, K::OFF_C, K::NC, nc, hb);
        if (new_b && !SWAP) load(&tb, Bz::B_FULL, Bz::B_EMPTY, K::OFF_B, K::NB, nb, hb);
        if (g == 0 || r.na > 1) load(&ta, Bz::A_FULL, Bz::A_EMPTY, K::OFF_A, K::NA, na, h * r.na + (r.na > 1 ? g : 0));
        if (new_b && SWAP) load(&tb, Bz::B_FULL, Bz::B_EMPTY, K::OFF_B, K::NB, nb, hb);
        if (new_b && !SWAP) load(&tc, Bz::C_FULL, Bz::C_EMPTY, K::OFF_C, K::NC, nc, hb);
      }
      if (!ok) record_error(LIN_ERR_WAIT);
      // copies must have landed before the block leaves
      for (int i = max(0, na - K::NA); i < na; ++i) mbar_wait(bar + Bz::A_FULL + 8 * (i % K::NA), (i / K::NA) & 1);
      for (int i = max(0, nb - K::NB); i < nb; ++i) mbar_wait(bar + Bz::B_FULL + 8 * (i % K::NB), (i / K::NB) & 1);
      for (int i = max(0, nc - K::NC); i < nc; ++i) mbar_wait(bar + Bz::C_FULL + 8 * (i % K::NC), (i / K::NC) & 1);
    }
    constexpr uint32_t ID_P = idesc_f16(BF16 ? 1 : 0, C, C, 0, 0);
    constexpr uint32_t ID_T = idesc_f16(BF16 ? 1 : 0, C, D, 0, 1);                       // B along its rows
    constexpr uint32_t ID_I = idesc_f16(BF16 ? 1 : 0, C, D, 0, SWAP ? 0 : 1);            // O = a X: X [da][dc], or (SWAP) [dc][da]
    const uint32_t st = sbase;
    bool ok = true;
    if (warp == WARP_MMA) {
      // ------------------------------------------------------------ P = a b^T, O = P c
      int ca = -1, cb = -1, noi = 0;
      for (int t = 0, ck = 0, g = 0; ok && t < items; ++t, ++g == groups ? g = 0, ++ck : 0) {
        const bool first = g == 0, last = g == groups - 1, new_b = first || r.nb > 1, do_i = first || r.na > 1;
        const int cn = min(C, tokens - chunk_at(ck));
        cb += new_b ? 1 : 0;
        ca += do_i ? 1 : 0;
        const uint32_t at = st + K::OFF_A + (ca % K::NA) * K::TILE, bt = st + K::OFF_B + (cb % K::NB) * K::TILE,
                       ct = st + K::OFF_C + (cb % K::NC) * K::TILE;
        if (new_b) ok = wait_warp(bar + Bz::B_FULL + 8 * (cb % K::NB), (cb / K::NB) & 1);
        if (do_i) ok = ok && wait_warp(bar + Bz::A_FULL + 8 * (ca % K::NA), (ca / K::NA) & 1);
        if (t > 0) ok = ok && wait_warp(bar + Bz::PV_DONE, (t - 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint64_t da = desc_k(at), db = desc_k(bt);
#pragma unroll
          for (int k0 = 0; k0 < K::NCH; ++k0)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint32_t s = k0 * (C * 128 >> 4) + kk * 2;
              mma_ss(tmem + K::P_COL, desc_add(da, s), desc_add(db, s), ID_P, k0 + kk > 0);
            }
          mma_commit(bar + Bz::P_FULL);
          if (last || r.na > 1) mma_commit(bar + Bz::A_EMPTY + 8 * (ca % K::NA));
          if (last || r.nb > 1) mma_commit(bar + Bz::B_EMPTY + 8 * (cb % K::NB));
        }
        __syncwarp();
        if (new_b) {
          ok = wait_warp(bar + Bz::C_FULL + 8 * (cb % K::NC), (cb / K::NC) & 1);
          if (ok && cn < C && q.cu) {
            zero_rows(sgen + K::OFF_C + (cb % K::NC) * K::TILE, K::NCH, cn, lane);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        // over what the output warps have taken of a X or of the item before
        ok = ok && wait_warp(bar + Bz::P_READY, t & 1);
        if (do_i) {
          ok = ok && wait_warp(bar + Bz::OI_READ, noi & 1);
          ++noi;
        }
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint64_t d = desc_mn(ct, C);
#pragma unroll
          for (int k0 = 0; k0 < C / 16; k0 += 4)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint32_t p = tmem + K::P_COL + 16 * (k0 + kk);      // 16 tokens: 8 columns hi, 8 lo
              mma_ts(tmem + K::O_COL, p, desc_add(d, (k0 + kk) * 128), ID_T, k0 + kk > 0);
              mma_ts(tmem + K::O_COL, p + 8, desc_add(d, (k0 + kk) * 128), ID_T, 1u);
            }
          mma_commit(bar + Bz::PV_DONE);
          if (last || r.nb > 1) mma_commit(bar + Bz::C_EMPTY + 8 * (cb % K::NC));
        }
        __syncwarp();
      }
    } else if (warp == WARP_MMA2) {
      // ------------------------------------------------------------ O = a X
      int ca = -1, nx = 0, nor = 0;
      for (int t = 0, ck = 0, g = 0; ok && t < items; ++t, ++g == groups ? g = 0, ++ck : 0) {
        const bool first = g == 0, last = g == groups - 1, do_i = first || r.na > 1;
        if (first) {
          ok = wait_warp(bar + Bz::XS_READY, nx & 1);
          ++nx;
        }
        if (do_i) {
          ++ca;
          const uint32_t at = st + K::OFF_A + (ca % K::NA) * K::TILE;
          if (t > 0) {      // once the epilogue has taken the item before
            ok = ok && wait_warp(bar + Bz::O_READ, nor & 1);
            ++nor;
          }
          ok = ok && wait_warp(bar + Bz::A_FULL + 8 * (ca % K::NA), (ca / K::NA) & 1);
          // P goes first through the pipe: its readers have more to do.  (With several heads of b this may return a phase early,
          // which changes the order and nothing else.)
          ok = ok && wait_warp(bar + Bz::P_FULL, t & 1);
          tc_fence_after();
          if (ok && lane == 0) {
            const uint64_t da = desc_k(at), xh = SWAP ? desc_k(st + K::OFF_X) : desc_mn(st + K::OFF_X, D);
#pragma unroll 1
            for (int k0 = 0; k0 < K::NCH; ++k0)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {
                const uint32_t s = k0 * (C * 128 >> 4) + kk * 2, sx = SWAP ? k0 * (D * 128 >> 4) + kk * 2 : (4 * k0 + kk) * 128;
                mma_ss(tmem + K::O_COL, desc_add(da, s), desc_add(xh, sx), ID_I, k0 + kk > 0);
                mma_ss(tmem + K::O_COL, desc_add(da, s), desc_add(xh, sx + (K::XT >> 4)), ID_I, 1u);
              }
            mma_commit(bar + Bz::OI_FULL);
            if (r.na == 1 || last) mma_commit(bar + Bz::X_READ);
          }
          __syncwarp();
        }
        if (ok && lane == 0 && (last || r.na > 1)) mma_commit(bar + Bz::A_EMPTY + 8 * (ca % K::NA));
      }
    } else if (warp == WARP_MMA3) {
      // ------------------------------------------------------------ X += (decayed rows)^T (rows)
      int cb = -1, nx = 0, nbt = 0;
      for (int t = 0, ck = 0, g = 0; ok && t < items; ++t, ++g == groups ? g = 0, ++ck : 0) {
        const bool first = g == 0, last = g == groups - 1, end = ck == chunks - 1;
        const bool new_b = first || r.nb > 1, do_b = new_b && !end;
        const int cn = min(C, tokens - chunk_at(ck));
        cb += new_b ? 1 : 0;
        const uint32_t bt = st + K::OFF_B + (cb % K::NB) * K::TILE, ct = st + K::OFF_C + (cb % K::NC) * K::TILE;
        if (first && !end) {
          ok = wait_warp(bar + Bz::XS_READY, nx & 1);
          ++nx;
        }
        if (do_b) {
          ok = ok && wait_warp(bar + Bz::BT_READY, nbt & 1);
          ++nbt;
        }
        // The state warps have read b (SWAP: it is still to be multiplied).  No buffer is given back before its tile has been
        // seen to land, even where this warp has nothing to read: it would run ahead and give back the one before.
        if (new_b && (SWAP || !do_b)) ok = ok && wait_warp(bar + Bz::B_FULL + 8 * (cb % K::NB), (cb / K::NB) & 1);
        if (!SWAP && ok && lane == 0 && (last || r.nb > 1)) mbar_arrive(bar + Bz::B_EMPTY + 8 * (cb % K::NB));
        if (new_b && (!SWAP || !do_b)) ok = ok && wait_warp(bar + Bz::C_FULL + 8 * (cb % K::NC), (cb / K::NC) & 1);
        if (do_b) {
          // (SWAP: P = a b^T may read b's rows before or after this; nothing is taken from its columns past the sequence)
          if (ok && cn < C && q.cu) {
            zero_rows(sgen + (SWAP ? K::OFF_B + (cb % K::NB) * K::TILE : K::OFF_C + (cb % K::NC) * K::TILE), K::NCH, cn, lane);
            fence_proxy_async_smem();
            __syncwarp();
          }
          tc_fence_after();
          if (ok && lane == 0) {
            const uint64_t d = desc_mn(SWAP ? bt : ct, C);
#pragma unroll 1
            for (int k0 = 0; k0 < C / 16; k0 += 4)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {
                const uint32_t b = tmem + K::BT_COL + 8 * (k0 + kk);
                mma_ts(tmem + K::X_COL, b, desc_add(d, (k0 + kk) * 128), ID_T, 1u);
                mma_ts(tmem + K::X_COL, b + 64, desc_add(d, (k0 + kk) * 128), ID_T, 1u);
              }
            mma_commit(bar + Bz::X_DONE);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (lane == 0 && (last || r.nb > 1)) {      // read here, or by the state warps, whose rows have been waited for
          if (SWAP) mma_commit(bar + Bz::B_EMPTY + 8 * (cb % K::NB));
          mma_commit(bar + Bz::C_EMPTY + 8 * (cb % K::NC));
        }
      }
    }
    if (!ok) record_error(LIN_ERR_WAIT);
    if (warp >= WARP_MMA) {
      const uint32_t drain = bar + Bz::DRAIN + 8 * (warp - WARP_MMA);
      if (lane == 0) mma_commit(drain);
      __syncwarp();
      if (!wait_warp(drain, 0)) record_error(LIN_ERR_WAIT);
    }
    __syncwarp();
  } else {
    const int qd = warp & 3, hf = (warp >> 2) & 1, row = qd * 32 + lane;
    const uint32_t la = tmem + ((uint32_t)(qd * 32) << 16);
    constexpr int HD = D / 2;                       // state or output columns of a thread
    bool ok = true;                   // false once a wait has given up: the warp goes on without waiting (the named barriers stay matched)
    const auto wait = [&](int which, int phase) {
      ok = ok && wait_warp(bar + which, phase & 1);
      __syncwarp();
      tc_fence_after();
    };
    if (warp >= 8) {
      // ---------------------------------------------------------- state
      regs_state();
      const int xl = SWAP ? r.dc : r.da, xn = SWAP ? r.da : r.dc;   // real rows (lanes) and columns of X
      const float* x0 = nullptr;
      if (ws) x0 = ws + ((long long)seg * q.nhk + h) * r.da * r.dc;
      else if (pool.in && !(pool.seen && pool.seen[z] <= 0)) x0 = pool.in + ((long long)slot * q.nhk + h) * r.da * r.dc;
      int nx = 0, nbt = 0, cbw = -1, w_cn = 0;
      float2 w_rows[8];
      // X as it enters the segment.  Stored along its lanes it is read by whole lines; stored along its columns, a lane's row would be
      // a line of its own in every load (20000 cycles of them), so it comes in by rows through the shared memory of X.
      if (!r.transposed || SWAP) {
        float4* stage = reinterpret_cast<float4*>(sgen + K::OFF_X);      // [D][D / 4], units swapped by row
#pragma unroll 8
        for (int e = tid - 256; e < D * D / 4; e += NSTATE) {
          const int lane_x = e / (D / 4), col = e % (D / 4) * 4;
          float4 x = x0 && lane_x < xl && col < xn ? *reinterpret_cast<const float4*>(x0 + (long long)lane_x * xn + col) : make_float4(0.f, 0.f, 0.f, 0.f);
          if constexpr (!BF16 && REV) x.x *= r.x_in, x.y *= r.x_in, x.z *= r.x_in, x.w *= r.x_in;
          stage[lane_x * (D / 4) + ((col / 4) ^ (lane_x & 7))] = x;
        }
        bar_state();
        if (qd * 32 < D) {
#pragma unroll 1
          for (int c0 = hf * HD; c0 < hf * HD + HD; c0 += 16) {
            float2 x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              reinterpret_cast<float4*>(x)[i] = stage[row * (D / 4) + ((c0 / 4 + i) ^ (row & 7))];
            tmem_store<16>(la + K::X_COL + c0, x);
          }
        }
        bar_state();
      } else if (qd * 32 < D) {
#pragma unroll 1
        for (int c0 = hf * HD; c0 < hf * HD + HD; c0 += 16) {
          float2 x[8];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            reinterpret_cast<float*>(x)[i] = x0 && row < xl && c0 + i < xn ? x0[(long long)(c0 + i) * xl + row] : 0.f;
          tmem_store<16>(la + K::X_COL + c0, x);
        }
      }
      tc_wait_st();
      for (int t = 0, ck = 0, g = 0; t < items; ++t, ++g == groups ? g = 0, ++ck : 0) {
        const bool first = g == 0, end = ck == chunks - 1;
        const bool do_b = (first || r.nb > 1) && !end;
        const int cn = min(C, tokens - chunk_at(ck));
        // the last a X, which reads X in shared memory, and the last update of X, which reads the decayed rows
        if (t > 0 && first) wait(Bz::X_READ, ck - 1);
        if (nbt > 0 && (first || do_b)) wait(Bz::X_DONE, nbt - 1);
        // X: hi + lo to shared memory, lam^C X back to TMEM
        if (first) {
          float xs = 1.f;
          if constexpr (!BF16) {
            float top = 0.f;
            if (qd * 32 < D) {
#pragma unroll 1
              for (int c0 = 0; c0 < HD; c0 += 32) {
                float2 x[16];
                tmem_load<32>(la + K::X_COL + hf * HD + c0, x);
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
              }
            }
            const uint32_t all = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
            if (lane == 0) atomicMax(&xmax[nx], all);
            bar_state();
            xs = scale_to(xmax[nx]);
            nx = nx == 2 ? 0 : nx + 1;
            if (tid == 256) xmax[nx] = 0;     // three slots: the output warps may still read the one before
          }
          const float keep = lam[cn];
          if (qd * 32 < D) {
#pragma unroll 1
            for (int col = hf * HD; col < hf * HD + HD; col += 16) {
              float2 x[8];
              tmem_load<16>(la + K::X_COL + col, x);
              uint32_t hi[8], lo[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                split2<BF16>(BF16 ? x[i] : __fmul2_rn(x[i], make_float2(xs, xs)), hi[i], lo[i]);
                x[i] = __fmul2_rn(x[i], make_float2(keep, keep));
              }
              tmem_store<16>(la + K::X_COL + col, x);
              uint8_t* xr = sgen + K::OFF_X + (col / 64) * D * 128 + row * 128;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint8_t* to_x = xr + ((((col % 64) / 8 + i) ^ (row & 7)) << 4);
                *reinterpret_cast<uint4*>(to_x) = make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
                *reinterpret_cast<uint4*>(to_x + K::XT) = make_uint4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
              }
            }
          }
          tc_wait_st();
          fence_proxy_async_smem();
          tc_fence_before();
          mbar_arrive(bar + Bz::XS_READY);
        }
        // decayed rows, transposed
        if (first || r.nb > 1) ++cbw;
        if (do_b) {
          if (cn != w_cn) {
            row_factors<REV, 4>(w_rows, lam, r.w_up, 64 * hf, lane, cn);
            w_cn = cn;
          }
          const int stages = SWAP ? K::NC : K::NB, s = cbw % stages;
          wait((SWAP ? Bz::C_FULL : Bz::B_FULL) + 8 * s, cbw / stages);
          if (qd * 32 < D)
            decay_rows<BF16, 2, 4>(sbase + (SWAP ? K::OFF_C : K::OFF_B) + s * K::TILE, la + K::BT_COL, w_rows, qd, 64 * hf, lane, cn);
          tc_wait_st();
          tc_fence_before();
          mbar_arrive(bar + Bz::BT_READY);
          ++nbt;
        }
      }
    } else {
      // ---------------------------------------------------------- outputs
      regs_out();
      float2 acc[HD / 2];               // this thread's part of an output row: a X first, then P c of each item
      float p_inv = 1.f, x_inv = 1.f;
      int nx = 0, noi = 0, at = 0, cn = 0, head = 0;
      bool write = false;
      const uint32_t obox = K::OFF_O + warp * 32 * HD * 2;
      for (int t = 0, ck = 0, g = 0;; ++t, ++g == groups ? g = 0, ++ck : 0) {
        if (t > 0) {
          // epilogue of the item before
          wait(Bz::PV_DONE, t - 1);
#pragma unroll
          for (int c0 = 0; c0 < HD; c0 += 32) {
            float2 o[16];
            tmem_load<32>(la + K::O_COL + hf * HD + c0, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[c0 / 2 + i] = __ffma2_rn(o[i], make_float2(p_inv, p_inv), acc[c0 / 2 + i]);
          }
          tc_fence_before();
          if (write) mbar_arrive(bar + Bz::O_READ);      // a X comes next (else P c, which waits for the pair products)
          if (write && hf * HD < r.dc) {
            // 32 whole rows go out as one box; rows next to another sequence's one by one
            const bool whole = qd * 32 + 32 <= cn;
            uint8_t* to_row = sgen + obox + lane * HD * 2;
            int swizzle = HD == 64 ? lane & 7 : (lane >> 1) & 3, units = HD / 8;      // 128-byte or 64-byte swizzle
            if (whole) {
              if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
              __syncwarp();
            } else {
              to_row = reinterpret_cast<uint8_t*>((T*)r.out + z4 * r.so.b + (long long)(row_first + at + row) * r.so.s + (long long)(h * r.na + head) * r.so.h + hf * HD);
              swizzle = 0;
              units = row < cn ? min(units, (r.dc - hf * HD) / 8) : 0;
            }
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
              if (i < units)
                *reinterpret_cast<uint4*>(to_row + ((i ^ swizzle) << 4)) =
                    make_uint4(pack2<BF16>(acc[4 * i].x, acc[4 * i].y), pack2<BF16>(acc[4 * i + 1].x, acc[4 * i + 1].y),
                               pack2<BF16>(acc[4 * i + 2].x, acc[4 * i + 2].y), pack2<BF16>(acc[4 * i + 3].x, acc[4 * i + 3].y));
            if (whole) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) tma_store_4d(&to, sbase + obox, hf * HD, row_first + at + qd * 32, h * r.na + head, z4);
            }
          }
        }
        if (t == items) break;
        const bool first = g == 0, do_i = !MULTI || first;
        at = chunk_at(ck);
        cn = min(C, tokens - at);
        head = r.na > 1 ? g : 0;
        write = r.na > 1 || g == groups - 1;
        // Pair products: decay, mask, back to TMEM as hi + lo, in pieces of W columns (acc takes the registers where it lives on from
        // head to head).  A block of 32 x 32 beside the diagonal's takes lam^(rows from its near edge) times lam^(columns from it), both at
        // most 1, so that nothing overflows however fast the decay
        constexpr int W = MULTI ? 16 : 32;
        wait(Bz::P_FULL, t);
        float ps = 1.f;
        if constexpr (!BF16) {
          // The products before decay bound the row (factors are at most 1), those that the row sees: past the sequence's end the
          // columns are of other sequences, and may be as large as they like.
          float top = 0.f;
#pragma unroll 1
          for (int j0 = hf * 64; j0 < hf * 64 + 64; j0 += W) {
            if (REV ? j0 / 32 < qd : j0 / 32 > qd) continue;
            float2 p[W / 2];
            tmem_load<W>(la + K::P_COL + j0, p);
            if (REV && cn < C) {
#pragma unroll
              for (int i = 0; i < W / 2; ++i) {
                if (j0 + 2 * i >= cn) p[i].x = 0.f;
                if (j0 + 2 * i + 1 >= cn) p[i].y = 0.f;
              }
            }
            if (j0 / 32 == qd) {
              const int own = row - j0;
#pragma unroll
              for (int i = 0; i < W / 2; ++i) {
                if (REV ? 2 * i >= own : 2 * i <= own) top = fmaxf(top, fabsf(p[i].x));
                if (REV ? 2 * i + 1 >= own : 2 * i + 1 <= own) top = fmaxf(top, fabsf(p[i].y));
              }
            } else {
#pragma unroll
              for (int i = 0; i < W / 2; ++i) top = fmaxf(top, fmaxf(fabsf(p[i].x), fabsf(p[i].y)));
            }
          }
          uint32_t* most = pmax + row;
          most[hf * C] = __float_as_uint(top);      // the item before was read before its P c, which this P waited for
          bar_quadrant(qd);
          ps = scale_to(max(most[0], most[C]));
        }
        p_inv = r.w_intra / ps;
#pragma unroll 1
        for (int j0 = hf * 64; j0 < hf * 64 + 64; j0 += W) {
          const int edge = j0 & ~31, side = REV ? edge / 32 - qd : qd - edge / 32;
          float2 p[W / 2];
          if (side < 0) {
#pragma unroll
            for (int i = 0; i < W / 2; ++i) p[i] = make_float2(0.f, 0.f);
          } else {
            tmem_load<W>(la + K::P_COL + j0, p);
            if (side > 0) {
              const float4* w = reinterpret_cast<const float4*>(lamc + (j0 - edge));
              const float blk = lam[REV ? edge - row : row - edge - 31] * ps;
#pragma unroll
              for (int i = 0; i < W / 4; ++i) {
                const float4 f = w[i];
                p[2 * i] = __fmul2_rn(p[2 * i], __fmul2_rn(make_float2(blk, blk), make_float2(f.x, f.y)));
                p[2 * i + 1] = __fmul2_rn(p[2 * i + 1], __fmul2_rn(make_float2(blk, blk), make_float2(f.z, f.w)));
              }
            } else {
              // On the diagonal, in pieces of 8 columns: lam^(gap to the piece's far edge), which may be up to lam^-7, times the table's, and what
              // lies on the other side is masked.  Where lam^-7 could overflow, exp2 of each gap (1200 cycles a block, not 600).
              // fp16's row scale (2^10 and more where products are near 1 or smaller) goes to the factors as long as lam^-7 times it is in range
              // for every row of the warp; exp2 of a gap that counts is at most 1
              const float from = (float)(REV ? j0 - row : row - j0);      // gap of the piece's first column
              if (BF16 ? g2 > -17.f : __all_sync(0xffffffffu, ex2(-7.f * g2) * ps < 0x1p126f)) {
#pragma unroll
                for (int s = 0; s < W / 8; ++s) {
                  const float edge_gap = REV ? from + 8 * s : from - 8 * s - 7, u = ex2(g2 * edge_gap) * ps;
                  const float4 w0 = *reinterpret_cast<const float4*>(lamc + (REV ? 0 : 24)), w1 = *reinterpret_cast<const float4*>(lamc + (REV ? 4 : 28));
                  p[4 * s] = __fmul2_rn(p[4 * s], __fmul2_rn(make_float2(u, u), make_float2(w0.x, w0.y)));
                  p[4 * s + 1] = __fmul2_rn(p[4 * s + 1], __fmul2_rn(make_float2(u, u), make_float2(w0.z, w0.w)));
                  p[4 * s + 2] = __fmul2_rn(p[4 * s + 2], __fmul2_rn(make_float2(u, u), make_float2(w1.x, w1.y)));
                  p[4 * s + 3] = __fmul2_rn(p[4 * s + 3], __fmul2_rn(make_float2(u, u), make_float2(w1.z, w1.w)));
                }
                const int gap = REV ? j0 - row : row - j0;
#pragma unroll
                for (int i = 0; i < W / 2; ++i) {
                  if (REV ? gap + 2 * i < 0 : gap < 2 * i) p[i].x = 0.f;
                  if (REV ? gap + 2 * i + 1 < 0 : gap < 2 * i + 1) p[i].y = 0.f;
                }
              } else {
#pragma unroll
                for (int i = 0; i < W / 2; ++i) {
                  const float gap = REV ? from + 2 * i : from - 2 * i, next = REV ? gap + 1.f : gap - 1.f;
                  p[i].x = gap >= 0.f ? p[i].x * (ex2(g2 * gap) * ps) : 0.f;
                  p[i].y = next >= 0.f ? p[i].y * (ex2(g2 * next) * ps) : 0.f;
                }
              }
            }
            if (REV && cn < C) {                  // forward, a row sees no token past its own
#pragma unroll
              for (int i = 0; i < W / 2; ++i) {
                if (j0 + 2 * i >= cn) p[i].x = 0.f;
                if (j0 + 2 * i + 1 >= cn) p[i].y = 0.f;
              }
            }
          }
#pragma unroll
          for (int c0 = 0; c0 < W / 2; c0 += 8) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) split2<BF16>(p[c0 + i], w[i], w[8 + i]);
            tmem_st16(la + K::P_COL + j0 + 2 * c0, w);
          }
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(bar + Bz::P_READY);
        // a X
        if (do_i) {
          wait(Bz::OI_FULL, noi);
          ++noi;
          if constexpr (!BF16) {
            if (first) {
              x_inv = 1.f / scale_to(xmax[nx]);
              nx = nx == 2 ? 0 : nx + 1;
            }
          }
          const float mul = r.w_inter * lam[REV ? max(cn - 1 - row, 0) : min(row + 1, C)] * x_inv;
#pragma unroll
          for (int c0 = 0; c0 < HD; c0 += 32) tmem_load<32>(la + K::O_COL + hf * HD + c0, acc + c0 / 2);
          tc_fence_before();
          mbar_arrive(bar + Bz::OI_READ);
#pragma unroll
          for (int i = 0; i < HD / 2; ++i) acc[i] = __fmul2_rn(acc[i], make_float2(mul, mul));
        }
      }
      if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      __syncwarp();
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

// =====================================================================================
// states: what a segment adds to the state, X = sum_j (lam^m_j b_j)^T c_j with powers up to the segment's own end, so that
// nothing is scaled on the way.  The result is a state that a caller may keep, in fp32, so the decayed rows enter as three bf16 numbers
// (2^-24 of a term) or two fp16 ones (2^-22).  fp16's smallest step is 2^-24, which fast decays meet; so the second fp16 number is what
// the first left over times 2^11 (at most half a step of the first: it cannot overflow), and its sum is scaled back by the first
// MMA on top of it.  The tensor cores truncate each accumulation; so every item is summed from 0, its small
// terms first (only the eight steps of the largest one then cut at the sum's full size), and items are added in registers, to nearest.
// One accumulator over a whole segment had left 2e-6 of the state.  Bound by reading b and c once.
// =====================================================================================
template <int D, bool BF16>
struct StCfg {
  static constexpr int NCH = D / 64, TILE = C * D * 2, NS = D == 128 ? 3 : 4, TERMS = BF16 ? 3 : 2, LO_SHIFT = BF16 ? 0 : 11;
  static constexpr int OFF_T = 0, OFF_BAR = NS * 2 * TILE, OFF_LAM = OFF_BAR + 128;
  static constexpr int SMEM = OFF_LAM + 132 * 4 + 1024;
  static constexpr uint32_t X_COL = 0, BT_COL = 128, BT_COLS = 192;      // two buffers of decayed rows
  static_assert(SMEM <= 232448, "shared memory per CTA");
};
struct StBz {
  static constexpr int FULL = 0, EMPTY = 32, BT_READY = 64, DONE = 80, X_READ = 88, DRAIN = 96, TMEM_ADDR = 104;
};

template <int D, bool BF16, bool REV>
__global__ void __launch_bounds__(NTHREADS_ST, 1)
    lin_tc_states_kernel(const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap tc, const LinSeqs q, const LinRole r,
                         float* ws) {
  using K = StCfg<D, BF16>;
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x % q.nhk, seg = blockIdx.x / q.nhk;
  int z, t0, t1;
  const LinSpan span = lin_segment(q, seg, z, t0, t1);
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
    for (int s = 0; s < 2; ++s) mbar_init(bar + StBz::BT_READY + 8 * s, NELEM_ST);
    mbar_init(bar + StBz::DONE, 1);
    mbar_init(bar + StBz::X_READ, NELEM_ST);
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
          for (int kk = 0; kk < C / 16; ++kk) {
            if (K::LO_SHIFT && w == 0 && kk == 0) mma_ts_onto<K::LO_SHIFT>(tmem + K::X_COL, bt, d, ID);
            else mma_ts(tmem + K::X_COL, bt + 64 * w + 8 * kk, desc_add(d, kk * 128), ID, kk > 0 || w < K::TERMS - 1);
          }
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
    const int qd = warp & 3, qr = warp >> 2, row = qd * 32 + lane;
    const uint32_t la = tmem + ((uint32_t)(qd * 32) << 16);
    constexpr int HD = D / 4;
    bool ok = true;
    float2 acc[HD / 2];
#pragma unroll
    for (int i = 0; i < HD / 2; ++i) acc[i] = make_float2(0.f, 0.f);
    const auto add = [&](int i) {      // item i's sum
      ok = ok && mbar_wait_warp(bar + StBz::DONE, i & 1);
      __syncwarp();
      tc_fence_after();
      float2 v[HD / 2];
      tmem_load<HD>(la + K::X_COL + qr * HD, v);
      tc_fence_before();
      mbar_arrive(bar + StBz::X_READ);
#pragma unroll
      for (int k = 0; k < HD / 2; ++k) acc[k] = __fadd2_rn(acc[k], v[k]);
    };
    float2 w_rows[4];
    int w_cn = 0;
    for (int i = 0; i < items; ++i) {
      // the buffer of decayed rows is free: item i - 2 was added up
      const int at = i / r.nb * C, cn = min(C, t1 - t0 - at);
      ok = ok && mbar_wait_warp(bar + StBz::FULL + 8 * (i % K::NS), (i / K::NS) & 1);
      __syncwarp();
      if (cn != w_cn) {
        row_factors<REV, 2>(w_rows, lam, 1.f, 32 * qr, lane, cn);
        w_cn = cn;
      }
      const float far = lin_power(g2, REV ? at : t1 - t0 - at - cn);
      float2 w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = __fmul2_rn(w_rows[k], make_float2(far, far));
      if (qd * 32 < D) decay_rows<BF16, K::TERMS, 2, K::LO_SHIFT>(sbase + tile(i), la + K::BT_COL + (i & 1) * K::BT_COLS, w, qd, 32 * qr, lane, cn);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(bar + StBz::BT_READY + 8 * (i & 1));
      if (i > 0) add(i - 1);
    }
    add(items - 1);
    float* x = ws + ((long long)seg * q.nhk + h) * r.da * r.dc + (long long)row * r.dc;
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) {
      const int col = qr * HD + 4 * i;
      if (row < r.da && col < r.dc)
        *reinterpret_cast<float4*>(x + col) = make_float4(r.w_up * acc[2 * i].x, r.w_up * acc[2 * i].y, r.w_up * acc[2 * i + 1].x, r.w_up * acc[2 * i + 1].y);
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

// boxes of `cols` columns (64 or 32) x `box_rows` rows over [batch][heads][rows][dim]; false where the layout does not allow it
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
  return encode_map([&] {
    return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box,
               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }) == CUDA_SUCCESS;
}

// fp16: the role with X in units of the power of 2 next above |w_up| (up to 2^64 either way: gradients of scales past that leave
// fp16 themselves)
LinRole in_units(LinRole r) {
  int e = 0;
  if (r.w_up != 0.f && std::isfinite(r.w_up) && fabsf(frexpf(r.w_up, &e)) == 0.5f) --e;
  const int u = std::min(std::max(e, -64), 64);
  r.x_in = ldexpf(1.f, -u);
  r.w_up *= r.x_in;
  r.w_inter *= ldexpf(1.f, u);
  return r;
}

bool takes(const LinSeqs& q, const LinRole& r, int dtype) {
  return dtype != FA_DTYPE_F32 && r.da <= 128 && r.dc <= 128 && (q.cu ? q.total > 0 : q.S > 0) && q.total < (1ll << 31) - 256;
}

// The register split of lin_tc_kernel waits for good unless the block starts with REGS a thread: looked up once for each kernel.  Another
// count, of another compiler, leaves the request to the CUDA cores (FABLE_ATTN_REQUIRE_TC refuses it).
template <typename Kernel>
bool regs_fit(Kernel kernel) {
  cudaFuncAttributes a;
  return cudaFuncGetAttributes(&a, (const void*)kernel) == cudaSuccess && a.numRegs == REGS;
}

template <typename Kernel, typename... Args>
int launch(Kernel kernel, int threads, int smem, unsigned long long* done, const LinSeqs& q, cudaStream_t st, const Args&... args) {
  const long long grid = (long long)q.slots * q.nhk;
  FA_CHECK_ARG(grid < (1ll << 31), "linear attention: %lld blocks", grid);
  if (int rc = ensure_smem((const void*)kernel, smem, done)) return rc;
  kernel<<<(int)grid, threads, smem, st>>>(args...);
  count_launch();
  return cuda_status(cudaGetLastError(), "linear attention (tensor cores) launch");
}

template <int D, bool BF16, bool REV, bool SWAP, bool MULTI>
int run_one(const LinSeqs& q, const LinRole& r, const float* ws, const LinPool& pool, cudaStream_t st, const CUtensorMap* m, bool* taken) {
  static unsigned long long done = 0;
  static const bool fits = regs_fit(lin_tc_kernel<D, BF16, REV, SWAP, MULTI>);
  if (!fits) return FA_OK;
  *taken = true;
  return launch(lin_tc_kernel<D, BF16, REV, SWAP, MULTI>, NTHREADS, Cfg<D, SWAP>::SMEM, &done, q, st, m[0], m[1], m[2], m[3], q, r, ws, pool);
}
template <int D, bool BF16>
int run_main(const LinSeqs& q, const LinRole& r, bool rev, const float* ws, const LinPool& pool, cudaStream_t st, const CUtensorMap* m, bool* taken) {
  // dk: the output is along the state's rows as it is stored
  if (!rev) return run_one<D, BF16, false, false, false>(q, r, ws, pool, st, m, taken);
  if (r.nb > 1)
    return r.transposed ? run_one<D, BF16, true, true, true>(q, r, ws, pool, st, m, taken)
                        : run_one<D, BF16, true, false, true>(q, r, ws, pool, st, m, taken);
  return r.transposed ? run_one<D, BF16, true, true, false>(q, r, ws, pool, st, m, taken)
                      : run_one<D, BF16, true, false, false>(q, r, ws, pool, st, m, taken);
}
template <int D, bool BF16>
int run_states(const LinSeqs& q, const LinRole& r, bool rev, float* ws, cudaStream_t st, const CUtensorMap* m) {
  static unsigned long long done[2] = {};
  using K = StCfg<D, BF16>;
  if (rev) return launch(lin_tc_states_kernel<D, BF16, true>, NTHREADS_ST, K::SMEM, done, q, st, m[0], m[1], q, r, ws);
  return launch(lin_tc_states_kernel<D, BF16, false>, NTHREADS_ST, K::SMEM, done + 1, q, st, m[0], m[1], q, r, ws);
}
}  // namespace

namespace fa {
bool lin_tc_takes(const LinSeqs& q, const LinRole& r, int dtype) { return takes(q, r, dtype); }

int lin_tc_main(const LinSeqs& q, const LinRole& role, bool rev, const float* ws, const LinPool& pool, int dtype, cudaStream_t st, bool* taken) {
  *taken = false;
  if (!takes(q, role, dtype) || (pool.out && !ws)) return FA_OK;
  const bool bf16 = dtype == FA_DTYPE_BF16;
  const LinRole r = bf16 ? role : in_units(role);
  const long long rows = q.cu ? q.total : q.S, zs = q.cu ? 1 : q.batch;
  const bool small = r.da <= 64 && r.dc <= 64;
  CUtensorMap m[4];
  if (!map4(m, r.a, bf16, r.da, rows, (long long)q.nhk * r.na, zs, r.sa) || !map4(m + 1, r.b, bf16, r.da, rows, (long long)q.nhk * r.nb, zs, r.sb) ||
      !map4(m + 2, r.c, bf16, r.dc, rows, (long long)q.nhk * r.nb, zs, r.sc) ||
      !map4(m + 3, r.out, bf16, r.dc, rows, (long long)q.nhk * r.na, zs, r.so, small ? 32 : 64, 32))
    return FA_OK;
  if (bf16) return small ? run_main<64, true>(q, r, rev, ws, pool, st, m, taken) : run_main<128, true>(q, r, rev, ws, pool, st, m, taken);
  return small ? run_main<64, false>(q, r, rev, ws, pool, st, m, taken) : run_main<128, false>(q, r, rev, ws, pool, st, m, taken);
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
