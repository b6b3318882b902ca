// decode8.cu — attention of new tokens over a paged cache held in 8 bits (fa_decode8_launch of
// fable_attn.h).
//
// One pass over the cache with a running maximum and sum.  For a key j with codes c_j, d_j and block
// scales ks_j, vs_j, and in base 2:  x_j = scale log2(e) ks_j (q . c_j),  o = sum 2^(x_j - m) vs_j d_j / sum 2^(x_j - m).
// The value scale joins the weight, w_j = 2^(x_j - m) vs_j u, where u is a power of two of the row's own that keeps the
// largest weight that still counts in fp16's range, whatever the scales (for V values up to 2^100, that sums stay finite): it
// falls where a weight would leave that range, and rises as m does.  The tensor cores take V codes (exact in
// fp16) and weights (fp16 high and low part, 22 bits) as they are, and dividing by u at the end is exact.
//
// The floor is the bytes of the cache.  What is read goes through registers to mma.sync (m16n8k16, fp16
// operands, fp32 sums): with 8 query rows the tensor pipe has twice the time that the bytes need, and the conversion of codes
// has to pass through registers anyway (a tcgen05 form with the converted operands in tensor and shared memory: 343 against
// 189 us at the time).  A strip is 32 (or 16) positions of one kv head.  Its K rows are the B operand of
// S = Q K^T, its V rows that of O += W V.  The order of an mma's k index and of its n columns is free as long as both operands
// agree, so each thread's operands are whole 16-byte pieces of cache rows (g = lane / 4, t = lane % 4):
//   K  row at(g) (+ 8), pieces t + 4 i;      V  rows at(2 t), at(2 t + 1) (+ 8), piece g,
// and S leaves the tensor cores in the layout in which W enters them.  Each warp has a ring of strips of its own, which
// its lane 0 fills by TMA (a box of its rows x 128 bytes each for K and V) behind an mbarrier a stage: no barrier
// between warps.  The 128-byte swizzle puts piece i of row r at i ^ (r & 7); with at(c) = c for even
// columns and c ^ 4 for odd ones, the eight lanes of a shared-memory phase touch eight different pieces in both reads.
//
// Rows of a warp are (new token, query head) pairs of one kv head.  8 rows: the upper 8 rows of the
// m16 tile carry the low parts of q and of w, so that both have 22 bits for nothing.  16 rows: a second mma.
// int8 K rows need no conversion: q becomes integers of 24 bits, relative to the row's largest, whose three bytes are the
// rows of integer mma (m16n8k32) with the codes as they are, and whose sums are exact.
//
// Work split: the strips of all sequences (times the row tiles of each) form one line, cut into equal
// ranges, one for each warp of a kv head; the warps of a CTA take the heads of one range, so that the heads' rows,
// adjacent in memory, are read together.  A warp's range is cut at sequence ends; a piece that is a whole sequence
// writes its output, others leave (m, l, o) in one of the warp's two slots, and a merge kernel joins the slots of each
// cut sequence in order (no atomics: same bits on every call).
//
// Measured, both kernels, replayed as a graph: 16 x 16-32k tokens, 8 kv heads, headdim 128, one token of 32 heads (806 MB): int8
// 166 us (4.8 TB/s), e4m3 163 us (4.9 TB/s), and 170 to 179 us either in a long loop, which the card's power limit slows; with 16
// heads a kv head 252 and 253 us; 48 x 1-9k e4m3 108 us (4.6 TB/s); one int8 document of 131k 73 us (3.7 TB/s); 24 windows
// of 4k with 1-4 tokens each, int8, softcap, 88 us; 1 x 611 12.5 us.  What bounds it: an SM holds 8 warps of 240 registers, whose
// conversions, mma and softmax (135 us by themselves when the first case took 181) and copies (141 us) overlap only in part.
#include <cudaTypedefs.h>
#include <algorithm>
#include <type_traits>
#include "fa_launch.h"
#include "kv8_common.cuh"
#include "sm100_ptx.cuh"

namespace {

using namespace fa_kv;
using sm100::ex2;

__device__ int g_dec8_error = 0;
__device__ __forceinline__ void record(int bit) { atomicOr(&g_dec8_error, bit); }

#define UNLIKELY(x) __builtin_expect(!!(x), 0)
constexpr int ERR_WAIT = 32768;    // a copy's wait gave up
constexpr float NONE = -1e30f;     // maximum of a part that saw nothing
constexpr float LAZY = 8.f;        // a score may exceed the running maximum by 8 (base 2) before it is moved
constexpr int LIFT = 6;            // weights are brought to [2^6, 2^7) ...
constexpr float MOST = 16384.f;    // ... when one exceeds 2^14: fp16 then reaches 2^-30 of the largest

template <int W, int RT>
struct Cfg {
  // Positions of a strip, warps of a CTA, CTAs of an SM, stages: what 64 K registers and 227 KB of shared memory hold.
  // Strips of 32 with 8 warps an SM against strips of 16 with 12: 160 and 181 us (16 x 16-32k e4m3), 108 and 134 us (48 x 1-9k
  // e4m3), 12.5 and 12.3 us (1 x 611).
  static constexpr int ST = RT == 8 && W <= 128 ? 32 : 16;
  static constexpr int NW = 4;
  static constexpr int CTAS = W == 64 && RT == 8 ? 4 : 2;
  static constexpr int STAGES = RT == 8 ? 2 : W == 128 ? 3 : 4;
  static constexpr int JT = ST / 8;                                        // n tiles of S
  static constexpr int KS = W / 16;                                        // k steps of S
  static constexpr int ROW = W == 64 ? 64 : 128;                           // bytes of a box row
  static constexpr int PANELS = W / ROW;                                   // boxes of a row
  static constexpr int HALF_B = ST * W;                                    // K or V of a strip
  static constexpr int STAGE_B = 2 * HALF_B;
  static constexpr int Q_B = KS * 512 * (RT / 8);                          // q operands
  static constexpr int RING_B = STAGES * STAGE_B;
  static constexpr int SCALE_B = ST * 8;                                   // scales of a strip: ST of K, ST of V
  static constexpr int WARP_B = RING_B + Q_B + STAGES * SCALE_B;
  static constexpr int SMEM = NW * WARP_B + 1024;                          // + what aligns the rings to 1 KB
  static_assert(SMEM * CTAS <= 227 * 1024, "shared memory of an SM");
  static constexpr int SLOT = RT * (W + 2);                                // floats of a slot: m[RT], l[RT], o[RT][W]
};

__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ int exponent(float x) { return max(((__float_as_int(x) >> 23) & 255) - 127, -120); }
template <int N>
__device__ __forceinline__ float max_of(const float (&v)[N]) {
  float a = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) a = fmaxf(a, v[i]);
  return a;
}
// m raised to the largest of it and a row's values in each of its four threads; returns it
template <int N>
__device__ __forceinline__ float raise(float& m, const float (&v)[N]) {
  float a = max_of(v);
  a = fmaxf(a, __shfl_xor_sync(~0u, a, 1));
  a = fmaxf(a, __shfl_xor_sync(~0u, a, 2));
  return m = fmaxf(a, m);
}
template <int NT, int RT>
__device__ __forceinline__ void scale_rows(float (*o)[4], int r, float f) {
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    o[i][2 * r] *= f;
    o[i][2 * r + 1] *= f;
    if constexpr (RT == 8) { o[i][2] *= f; o[i][3] *= f; }
  }
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh to a few units of its own last place (a score far below the softcap keeps its bits, which 1 - 2 / (e^2x + 1) would take from
// it), NaN where x is.  Below 1 the fifth convergent of Lambert's continued fraction x / (1 + x^2 / (3 + x^2 / (5 + ...))), which
// is 6e-8 off at 1 and less below; above, (e^2x - 1) / (e^2x + 1), with an exponent that keeps the power finite.
__device__ __forceinline__ float tanh_rel(float x) {
  const float y = x * x;
  float e = 2.f * FA_LOG2E * x;
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(e) : "f"(64.f));
  e = ex2(e);
  const bool small = fabsf(x) < 1.f;
  return __fdividef(small ? x * fmaf(y, y + 105.f, 945.f) : e - 1.f, small ? fmaf(y, fmaf(y, 15.f, 420.f), 945.f) : e + 1.f);
}
// 16 bytes to shared memory, zeros where not valid; 4 bytes
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// position of column c of an n tile among the tile's 8
__device__ __forceinline__ int col_pos(int c) { return (c & 1) ? c ^ 4 : c; }
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// int8 K: q (signed or unsigned bytes) times codes, 32 dims, exact sums
template <bool SIGNED>
__device__ __forceinline__ void mma8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (SIGNED)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// byte i of four words
__device__ __forceinline__ uint32_t bytes_of(const int* n, int i) {
  const int sel = i | (4 + i) << 4;
  return __byte_perm(__byte_perm(n[0], n[1], sel), __byte_perm(n[2], n[3], sel), 0x5410);
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// (a, b) as fp16 high parts and what is left of them
__device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = pack(a - f.x, b - f.y);
}

// Codes as pairs of fp16 (exact).  int8: c + 128 as the low byte of 1024 + (c + 128), less 1152.
template <typename Q>
struct Conv;
template <>
struct Conv<I8> {
  static __device__ __forceinline__ uint32_t half_pair(uint32_t x, uint32_t sel) {   // bytes of x ^ 0x80808080
    const uint32_t u = __byte_perm(x, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // bytes i of two words -> (a_i, b_i)
  static __device__ __forceinline__ void across(uint32_t a, uint32_t b, uint32_t* p) {
    const uint32_t x = __byte_perm(a, b, 0x5140) ^ 0x80808080u, y = __byte_perm(a, b, 0x7362) ^ 0x80808080u;
    p[0] = half_pair(x, 0x4140); p[1] = half_pair(x, 0x4342);
    p[2] = half_pair(y, 0x4140); p[3] = half_pair(y, 0x4342);
  }
};
template <>
struct Conv<E4M3> {
  // 4 bytes of one word -> (0, 1), (2, 3)
  static __device__ __forceinline__ void along(uint32_t w, uint32_t& p0, uint32_t& p1) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(p0), "=r"(p1) : "r"(w));
  }
  static __device__ __forceinline__ void across(uint32_t a, uint32_t b, uint32_t* p) {
    along(__byte_perm(a, b, 0x5140), p[0], p[1]);
    along(__byte_perm(a, b, 0x7362), p[2], p[3]);
  }
};

// ---------------------------------------------------------------- geometry
struct Seq {
  int n, L, lo;           // new tokens, cached tokens, first key that any of them sees
  int s0, strips, tiles;  // first strip, strips (at least one, so that somebody writes the rows), row tiles
  long long first;        // its first row
};

template <int RT, int ST>
__device__ __forceinline__ Seq seq_of(const FaDec8Params& p, const Pages& pg, int z) {
  Seq s;
  const RowMap rm{p.cu_q, p.tokens, p.batch};
  s.first = rm.first(z);
  s.n = rm.count(z, p.total);
  s.L = max(p.ctx_len[z], 0);
  const long long cap = (long long)p.max_blocks << pg.shift;
  if (s.L > cap) {
    record(ERR_PAGE);
    s.L = (int)cap;
  }
  const int pos0 = p.ctx_len[z] - s.n;
  s.lo = p.leftpad ? max(p.leftpad[z], 0) : 0;
  if (p.win_left >= 0) s.lo = max(s.lo, pos0 - p.win_left);
  s.s0 = s.lo / ST;
  s.strips = max(1, (s.L + ST - 1) / ST - s.s0);
  s.tiles = (int)(((long long)s.n * p.gqa + RT - 1) / RT);
  return s;
}

// 16 elements of a row from d on
template <typename T>
__device__ __forceinline__ void load16(const T* x, int d, bool vec, float* v) {
  if (vec) {
    constexpr int U = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16; i += U) {
      union { uint4 u; T e[U]; } b;
      b.u = *reinterpret_cast<const uint4*>(x + d + i);
#pragma unroll
      for (int j = 0; j < U; ++j) v[i + j] = Elem<T>::to_f(b.e[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = Elem<T>::to_f(x[d + i]);
  }
}
// The same, rotated by table row rp (rp < 0: as they are), in fp32.
template <typename T>
__device__ __forceinline__ void load_q16(const FaDec8Params& p, const T* x, int d, int rp, bool vec, float* v) {
  load16(x, d, vec, v);
  if (rp < 0 || d >= p.rot_dim) return;
  const int half = p.rot_dim / 2;
  const float* ct = p.cos + (long long)rp * half;
  const float* sn = p.sin + (long long)rp * half;
  if (p.rot_interleaved) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      if (d + i >= p.rot_dim) break;
      const float c = __ldg(ct + (d + i) / 2), s = __ldg(sn + (d + i) / 2), a = v[i], b = v[i + 1];
      v[i] = a * c - b * s;
      v[i + 1] = b * c + a * s;
    }
  } else if (half % 16 == 0) {   // the partners are a piece too
    const bool low = d < half;
    float w[16];
    load16(x, low ? d + half : d - half, vec, w);
    ct += low ? d : d - half;
    sn += low ? d : d - half;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float c = __ldg(ct + i), s = __ldg(sn + i);
      v[i] = low ? v[i] * c - w[i] * s : v[i] * c + w[i] * s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (d + i >= p.rot_dim) break;
      const bool low = d + i < half;
      const int j = low ? d + i : d + i - half;
      const float c = __ldg(ct + j), s = __ldg(sn + j), b = Elem<T>::to_f(x[low ? d + i + half : d + i - half]);
      v[i] = low ? v[i] * c - b * s : v[i] * c + b * s;
    }
  }
}

__device__ __forceinline__ void store_n(void* o, int dtype, long long at, const float* v, int n) {
  if (dtype == FA_DTYPE_BF16) {
    __nv_bfloat16* x = (__nv_bfloat16*)o + at;
#pragma unroll
    for (int i = 0; i < n; i += 8) {
      uint4 u;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[i + 2 * j], v[i + 2 * j + 1]);
      *reinterpret_cast<uint4*>(x + i) = u;
    }
  } else if (dtype == FA_DTYPE_F16) {
    __half* x = (__half*)o + at;
#pragma unroll
    for (int i = 0; i < n; i += 8) {
      uint4 u;
      __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(v[i + 2 * j], v[i + 2 * j + 1]);
      *reinterpret_cast<uint4*>(x + i) = u;
    }
  } else {
    float* x = (float*)o + at;
#pragma unroll
    for (int i = 0; i < n; i += 4) *reinterpret_cast<float4*>(x + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  }
}

__device__ __forceinline__ void store_lse(const FaDec8Params& p, long long row, int head, float m, float l) {
  if (p.lse) p.lse[head * p.total + row] = l == 0.f ? -INFINITY : (m + lg2(l)) * FA_LN2;
}

struct Cut {   // the row tile of a sequence whose strips begin in a warp's range and end in a later one
  long long first;   // the sequence's first row
  int tile, rows;    // row tile; rows of a kv head in the sequence (tokens x query heads)
  int parts, pad[3]; // ranges that it lies in; 0: none
};
static_assert(sizeof(Cut) == 32, "the slots behind the records are stored to 16 bytes at a time");

// ---------------------------------------------------------------- the pass over the cache
template <int W, typename Q, int RT, bool TMA>
__global__ void __launch_bounds__((Cfg<W, RT>::NW * 32), (Cfg<W, RT>::CTAS))
    dec8_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const FaDec8Params p,
                const Pages pg, const int dtype, const int ranges) {
  using C = Cfg<W, RT>;
  constexpr int ST = C::ST, NW = C::NW, STAGES = C::STAGES, KS = C::KS, NT = W / 8, KC = W / 64, VC = W == 256 ? 2 : 1;
  constexpr int JT = C::JT, NP = 2 * JT;   // n tiles of S, positions of a thread
  constexpr unsigned ALL = ST == 32 ? ~0u : 0xffffu;
  constexpr int RPT = RT / 8;        // rows of a thread: g, g + 8
  constexpr bool INT = std::is_same<Q, I8>::value;
  extern __shared__ unsigned char smem_raw[];
  __shared__ unsigned long long s_full[NW][STAGES];   // mbarrier of a stage
  __shared__ unsigned s_have[NW][STAGES];             // its positions that lie in a page (bits)
  __shared__ long long s_pre[NW * 32 + 1], s_warp[NW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int NKV = p.NH / p.gqa;

  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) sm100::mbar_init(sm100::smem_u32(&s_full[warp][i]), 1);
    sm100::fence_barrier_init();
    sm100::prefetch_tmap(&tmK);
    sm100::prefetch_tmap(&tmV);
  }
  pdl_wait();      // what comes before on the stream (an append) is done
  pdl_trigger();   // the merge may be set up; it waits for this grid itself
  // ---- the line of strips: every thread sums a run of sequences
  const int CB = (p.batch + NW * 32 - 1) / (NW * 32);
  {
    long long mine = 0;
    for (int z = tid * CB; z < min(p.batch, (tid + 1) * CB); ++z) {
      const Seq s = seq_of<RT, C::ST>(p, pg, z);
      mine += (long long)s.strips * s.tiles;
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(~0u, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    for (int w = 0; w < warp; ++w) inc += s_warp[w];
    s_pre[tid] = inc - mine;
    if (tid == NW * 32 - 1) s_pre[NW * 32] = inc;
    __syncthreads();
  }
  const long long total = s_pre[NW * 32];
  const int gw = blockIdx.x * NW + warp, range = gw / NKV, kvh = gw % NKV;
  if (range >= ranges) return;
  Cut* const cuts = reinterpret_cast<Cut*>(p.scratch);
  float* const slots = p.scratch + (long long)ranges * NKV * (sizeof(Cut) / 4) + (long long)gw * 2 * C::SLOT;
  Cut cut{};
  const long long per = max(1ll, (total + ranges - 1) / ranges);
  const long long begin = range * per, end = min(total, begin + per);

  const uint32_t base = (sm100::smem_u32(smem_raw) + 1023u) & ~1023u, ring = base + warp * C::RING_B;
  const unsigned char* const mine = smem_raw + (ring - sm100::smem_u32(smem_raw));
  unsigned char* const own = smem_raw + (base - sm100::smem_u32(smem_raw)) + NW * C::RING_B + warp * (C::Q_B + STAGES * C::SCALE_B);
  uint4* const qs = reinterpret_cast<uint4*>(own);
  const float* const scales = reinterpret_cast<const float*>(own + C::Q_B);   // a stage: ST of K, ST of V
  const uint32_t scales_u = sm100::smem_u32(scales) + lane * 4;
  const int bshift = log2_of(p.block), per_page = p.page >> bshift;
  const int run = min(p.page, ST);                  // slots of a box
  const bool two = run < ST;                        // a page is half a strip
  // the thread's pieces within K or V of a stage
  const auto piece = [](int row, int i) { return row * C::ROW + (C::ROW == 128 ? (i ^ (row & 7)) : (i ^ ((row >> 1) & 3))) * 16; };
  const int kat = piece(col_pos(g), t4);
  const int vat0 = W == 64 ? piece(2 * t4, g >> 1) + (g & 1) * 8 : piece(2 * t4, g);
  const int vat1 = W == 64 ? piece(col_pos(2 * t4 + 1), g >> 1) + (g & 1) * 8 : piece(col_pos(2 * t4 + 1), g);
  int stage = 0, parity = 0;                        // of the next strip to consume; a piece fills the ring from there

  // ---- the sequence that holds the range's first strip
  int z = 0;
  long long off = 0;                                // line position of sequence z
  Seq sq{};
  if (begin < end) {
    int a = 0, b = NW * 32 - 1;                     // last run that starts at or before `begin`
    while (a < b) {
      const int mid = (a + b + 1) >> 1;
      if (s_pre[mid] <= begin) a = mid;
      else b = mid - 1;
    }
    z = a * CB;
    off = s_pre[a];
    sq = seq_of<RT, C::ST>(p, pg, z);
    while (off + (long long)sq.strips * sq.tiles <= begin) {
      off += (long long)sq.strips * sq.tiles;
      sq = seq_of<RT, C::ST>(p, pg, ++z);
    }
  }

  for (long long at = begin; at < end;) {
    // ---- a piece: strips [k0, k1) of row tile `tile` of sequence z
    const int tile = (int)((at - off) / sq.strips), k0 = (int)((at - off) % sq.strips);
    const int k1 = (int)min((long long)sq.strips, k0 + (end - at));

    // Strip k of the sequence into a stage: lane 0 the codes, the lanes one scale each (two where a strip has 32).
    // What no row sees is not read: its weights are 0, and its V rows are cleared where they are used.  The pages of
    // the next strip (two where a page is half a strip) are looked up an issue ahead.
    int b0 = pg.of(z, (sq.s0 + k0) * ST), b1 = run < ST ? pg.of(z, (sq.s0 + k0) * ST + run) : b0;
    auto load = [&](int r, int slot, int to) {
      const uint32_t bar = sm100::smem_u32(&s_full[warp][to]), dst = ring + to * C::STAGE_B + r * C::ROW;
#pragma unroll
      for (int c = 0; c < C::PANELS; ++c) {
        sm100::tma_load_3d(dst + c * ST * C::ROW, &tmK, c * C::ROW, kvh, slot, bar);
        sm100::tma_load_3d(dst + C::HALF_B + c * ST * C::ROW, &tmV, c * C::ROW, kvh, slot, bar);
      }
    };
    auto scale_to = [&](int e, int b, int in_page, int to) {   // entry e of a stage's scales
      cp_async4(scales_u + to * C::SCALE_B + (e - lane) * 4,
                (e < ST ? p.Ks : p.Vs) + ((long long)b * NKV + kvh) * per_page + (in_page >> bshift));
    };
    auto issue = [&](int k, int to) {
      const int pos0 = (sq.s0 + k) * ST, in_page = pos0 & (p.page - 1);
      // do rows see something of the slots of either page; are they there
      const bool see0 = pos0 + run > sq.lo && pos0 < sq.L, see1 = two && pos0 + ST > sq.lo && pos0 + run < sq.L;
      const bool go0 = see0 && b0 >= 0, go1 = see1 && b1 >= 0;
      if (UNLIKELY(see0 != go0 || see1 != go1)) record(ERR_PAGE);
      if (lane == 0) {
        const uint32_t half = (uint32_t)run * (2 * W);
        s_have[warp][to] = (go0 ? (two ? 0xffffu : ALL) : 0u) | (go1 ? 0xffff0000u : 0u);
        sm100::mbar_expect_tx(sm100::smem_u32(&s_full[warp][to]), (go0 ? half : 0) + (go1 ? half : 0));
        if (go0) load(0, b0 * p.page + in_page, to);
        if (UNLIKELY(go1)) load(run, b1 * p.page, to);
      }
#pragma unroll
      for (int i = 0; i < ST / 16; ++i) {
        const int e = lane + 32 * i, r = e % ST;
        const bool first = ST == 16 || r < run;
        if (first ? go0 : go1) scale_to(e, first ? b0 : b1, (in_page + r) & (p.page - 1), to);
      }
      if (in_page + ST >= p.page && k + 1 < k1) {
        b0 = pg.of(z, pos0 + ST);
        if (UNLIKELY(two)) b1 = pg.of(z, pos0 + ST + run);
      }
    };
    // Pages of less than 16 slots: the whole warp copies slot by slot, piece by piece, into the same places.
    auto issue_small = [&](int k, int to) {
      const int pos0 = (sq.s0 + k) * ST;
      unsigned have = 0;
#pragma unroll 1
      for (int i = 0; i < ST / 16; ++i) {           // lane's entry: K or V of position pos0 + r
        const int e = lane + 32 * i, r = e % ST, pos = pos0 + r;
        const bool in = pos >= sq.lo && pos < sq.L;
        const int b = in ? pg.of(z, pos) : -1;
        if (in && b < 0) record(ERR_PAGE);
        have = __ballot_sync(~0u, b >= 0) & ALL;
        const unsigned char* src = (const unsigned char*)(e < ST ? p.Kc : p.Vc);
        if (b >= 0) src += (((long long)b * p.page + (pos & (p.page - 1))) * NKV + kvh) * p.dim;
        const uint32_t dst = ring + to * C::STAGE_B + (e < ST ? 0 : C::HALF_B);
        for (int j = 0; j < W / 16; ++j) {
          const bool ok = b >= 0 && 16 * j < p.dim;
          cp_async16(dst + (16 * j / C::ROW) * ST * C::ROW + piece(r, j % (C::ROW / 16)), ok ? src + 16 * j : src, ok);
        }
        if (b >= 0) scale_to(e, b, pos & (p.page - 1), to);
      }
      if (lane == 0) s_have[warp][to] = have;
    };
    __syncwarp();                                   // the last piece's stages and q are free
    for (int i = 0, to = stage; i < STAGES; ++i) {
      if (k0 + i < k1) {
        if constexpr (TMA) issue(k0 + i, to);
        else issue_small(k0 + i, to);
      }
      cp_commit();
      to = to + 1 == STAGES ? 0 : to + 1;
    }
    const bool cap = p.softcap > 0.f;
    const int q_unit = dtype == FA_DTYPE_F32 ? 4 : 8;
    const bool q_vec = (uintptr_t)p.q % 16 == 0 && p.q_row % q_unit == 0 && p.q_head % q_unit == 0;
    // ---- the rows: ranges of keys, factors, q operands
    float qf[RPT], slope[RPT], qpos[RPT];
    int rlo[RPT], rhi[RPT];
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      const int row = tile * RT + g + 8 * r, tok = row / p.gqa, head = kvh * p.gqa + row % p.gqa;
      const bool live = tok < sq.n;
      const int pos = p.ctx_len[z] - sq.n + tok;
      rlo[r] = max(sq.lo, p.win_left >= 0 ? pos - p.win_left : 0);
      rhi[r] = !live ? 0 : p.win_right >= 0 ? (int)min((long long)sq.L, (long long)pos + p.win_right + 1) : sq.L;
      qpos[r] = (float)pos;
      slope[r] = p.alibi && live ? p.alibi[head] * FA_LOG2E : 0.f;
      int rp = -1;
      if (p.cos && rlo[r] < rhi[r]) {
        rp = p.rot_pos ? p.rot_pos[z] + tok : pos;
        if (rp < 0 || rp >= p.rot_seqlen_ro) {
          record(ERR_ROTARY);
          rp = -1;
        }
      }
      const long long qe = (sq.first + tok) * p.q_row + head * p.q_head;
      float x[KS * 4], most = 0.f, bad = 0.f;       // 16 i + 4 w: piece t4 + 4 i, word w; bad: NaN where one is not finite
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const int d = 16 * (t4 + 4 * i);
        float* v = x + 16 * i;
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = 0.f;
        if (live && d < p.dim) {
          if (dtype == FA_DTYPE_BF16) load_q16(p, (const __nv_bfloat16*)p.q + qe, d, rp, q_vec, v);
          else if (dtype == FA_DTYPE_F16) load_q16(p, (const __half*)p.q + qe, d, rp, q_vec, v);
          else load_q16(p, (const float*)p.q + qe, d, rp, q_vec, v);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          most = fmaxf(most, fabsf(v[j]));
          if constexpr (INT) bad = fmaf(v[j], 0.f, bad);
        }
      }
      // rows are brought to [1, 2) by a power of two, so that fp16 holds them whatever their size
      most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
      most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
      const int e = min(exponent(most), 126);
      const float down = pow2(-e);
      qf[r] = p.scale * pow2(e) * (cap ? 1.f / p.softcap : FA_LOG2E);
      if constexpr (INT) {   // q as integers of 24 bits, 2^22 to 1: three bytes, the upper one signed
        bad += __shfl_xor_sync(~0u, bad, 1);
        bad += __shfl_xor_sync(~0u, bad, 2);
        qf[r] = fmaf(qf[r], 0x1p-22f, bad);
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          int n[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) n[i] = min(__float2int_rn(x[4 * c + i] * down * 0x1p22f), (1 << 23) - 1);
          uint32_t* const at = reinterpret_cast<uint32_t*>(qs);
          const int step = (c >> 1) * 32 + lane;
          if constexpr (RT == 8) {   // the upper bytes of a step's two words; of each, the middle ones and the lower ones
            at[2 * step + (c & 1)] = bytes_of(n, 2);
            uint32_t* const low = at + KS * 32 + 4 * step + 2 * (c & 1);
            low[0] = bytes_of(n, 1);
            low[1] = bytes_of(n, 0);
          } else {                   // as the operand has them: word 0 of rows g, g + 8, word 1 of both
#pragma unroll
            for (int i = 0; i < 3; ++i) at[i * (KS * 64) + 4 * step + 2 * (c & 1) + r] = bytes_of(n, 2 - i);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          uint32_t h0, l0, h1, l1;
          split(x[4 * c] * down, x[4 * c + 1] * down, h0, l0);
          split(x[4 * c + 2] * down, x[4 * c + 3] * down, h1, l1);
          if constexpr (RT == 8) {
            qs[c * 32 + lane] = make_uint4(h0, l0, h1, l1);
          } else {   // operand words: 0 row g, 1 row g + 8 (first pair); 2, 3 (second pair); low parts behind
            uint32_t* const hi = reinterpret_cast<uint32_t*>(qs) + (c * 32 + lane) * 4;
            uint32_t* const lo = hi + KS * 128;
            hi[r] = h0; hi[2 + r] = h1;
            lo[r] = l0; lo[2 + r] = l1;
          }
        }
      }
    }
    // keys that every row of the warp sees
    int all_lo = rlo[0], all_hi = rhi[0];
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      const bool live = tile * RT + g + 8 * r < sq.n * p.gqa;   // rows past the last token see nothing and are not written
      all_lo = max(all_lo, live ? rlo[r] : all_lo);
      all_hi = min(all_hi, live ? rhi[r] : all_hi);
      if (!live && r == 0) { all_lo = 0; all_hi = 0x7fffffff; }
    }
    all_lo = __reduce_max_sync(~0u, all_lo);
    all_hi = cap || p.alibi ? 0 : __reduce_min_sync(~0u, all_hi);

    float o[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[RPT], above[RPT], l[RPT], up[RPT];      // above: how far over m a score moves it
#pragma unroll
    for (int r = 0; r < RPT; ++r) { m[r] = l[r] = 0.f; above[r] = -INFINITY; up[r] = pow2(126); }
    const float cap_out = p.softcap * FA_LOG2E;

    int k_lost = -1;
    for (int k = k0; k < k1; ++k) {
      cp_wait<STAGES - 1>();
      __syncwarp();
      if (TMA && UNLIKELY(!__all_sync(~0u, sm100::mbar_wait(sm100::smem_u32(&s_full[warp][stage]), parity)))) {
        record(ERR_WAIT);                           // copies that never land: give up (they are waited for below)
        k_lost = k;
        break;
      }
      const unsigned char* const src = mine + stage * C::STAGE_B;

      // ---- S = Q K^T: column c of n tile j is position pos0 + 8 j + col_pos(c)
      float s[RPT][NP];                             // as the weights are, below
      if constexpr (INT) {
        // Integer mma on the codes as they are.  With q = 65536 h + 256 m + l the three sums stay below 2^31 for 256
        // dims, and so does 256 m + l.  8 rows: h in one, m and l in the two halves of another.  (K as fp16: 175 against
        // 166 us for 16 x 16-32k tokens of 4 heads a kv head, 279 against 256 us with 16 heads.)
        constexpr int ACCS = RT == 8 ? 2 : 3;
        int a[ACCS][JT][4];
#pragma unroll
        for (int i = 0; i < ACCS; ++i)
#pragma unroll
          for (int j = 0; j < JT; ++j) a[i][j][0] = a[i][j][1] = a[i][j][2] = a[i][j][3] = 0;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          uint4 kk[JT];
#pragma unroll
          for (int j = 0; j < JT; ++j)
            kk[j] = *reinterpret_cast<const uint4*>(src + (c >> 1) * (ST * 128) + (kat ^ ((c & 1) * 64)) + j * 8 * C::ROW);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int step = (2 * c + w) * 32 + lane;
            if constexpr (RT == 8) {
              const uint2 h = reinterpret_cast<const uint2*>(qs)[step];
              const uint4 ml = qs[KS * 8 + step];
#pragma unroll
              for (int j = 0; j < JT; ++j) {
                const uint32_t k0 = (&kk[j].x)[2 * w], k1 = (&kk[j].x)[2 * w + 1];
                mma8<true>(a[0][j], h.x, 0, h.y, 0, k0, k1);
                mma8<false>(a[1][j], ml.x, ml.y, ml.z, ml.w, k0, k1);
              }
            } else {
              const uint4 h = qs[step], m = qs[KS * 16 + step], l = qs[KS * 32 + step];
#pragma unroll
              for (int j = 0; j < JT; ++j) {
                const uint32_t k0 = (&kk[j].x)[2 * w], k1 = (&kk[j].x)[2 * w + 1];
                mma8<true>(a[0][j], h.x, h.y, h.z, h.w, k0, k1);
                mma8<false>(a[1][j], m.x, m.y, m.z, m.w, k0, k1);
                mma8<false>(a[2][j], l.x, l.y, l.z, l.w, k0, k1);
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int j = i >> 1, e = i & 1;
#pragma unroll
          for (int h = 0; h < RPT; ++h) {
            const int ml = RT == 8 ? a[1][j][e] * 256 + a[1][j][2 + e] : a[1][j][2 * h + e] * 256 + a[ACCS - 1][j][2 * h + e];
            s[h][i] = fmaf((float)a[0][j][2 * h + e], 65536.f, (float)ml);
          }
        }
      } else {
        float a[JT][4];
#pragma unroll
        for (int j = 0; j < JT; ++j) a[j][0] = a[j][1] = a[j][2] = a[j][3] = 0.f;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          uint4 kk[JT];
#pragma unroll
          for (int j = 0; j < JT; ++j)
            kk[j] = *reinterpret_cast<const uint4*>(src + (c >> 1) * (ST * 128) + (kat ^ ((c & 1) * 64)) + j * 8 * C::ROW);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint4 qu = qs[(4 * c + w) * 32 + lane];
            const uint32_t qv[4] = {qu.x, qu.y, qu.z, qu.w};
            uint32_t ql[4];
            if constexpr (RT == 16) {
              const uint4 lu = qs[(KS + 4 * c + w) * 32 + lane];
              ql[0] = lu.x; ql[1] = lu.y; ql[2] = lu.z; ql[3] = lu.w;
            }
#pragma unroll
            for (int j = 0; j < JT; ++j) {
              uint32_t k0, k1;
              Conv<Q>::along((&kk[j].x)[w], k0, k1);
              mma(a[j], qv, k0, k1);
              if constexpr (RT == 16) mma(a[j], ql, k0, k1);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int h = 0; h < RPT; ++h)
            s[h][i] = RT == 8 ? a[i >> 1][i & 1] + a[i >> 1][2 + (i & 1)] : a[i >> 1][2 * h + (i & 1)];
      }

      // ---- weights of positions pos0 + 8 j + col_pos(2 t4 + e), row g (+ 8 r), at [2 j + e]; x: scores less m, rounded
      // once (a score of 50 by itself is good to 2^-19 only, and so would its weight be).  What a softcap takes is the score
      // itself, not its difference from m, which would be rounded at m's size.
      const int pos0 = (sq.s0 + k) * ST;
      const unsigned have = s_have[warp][stage];
      // strips that every row sees whole, with scores that are nothing but products, run code without masks (16 x 16-32k
      // int8 tokens: one form with branches 182 us, two forms 173; e4m3 165 and 160)
      const auto weigh = [&](auto plain) {
      constexpr bool PLAIN = decltype(plain)::value;
      float x[RPT][NP], vs[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = 8 * (i >> 1) + col_pos(2 * t4 + (i & 1));
        const float ks = scales[stage * (2 * ST) + r];
        vs[i] = scales[stage * (2 * ST) + ST + r];
#pragma unroll
        for (int h = 0; h < RPT; ++h) x[h][i] = fmaf(s[h][i], ks * qf[h], !PLAIN && cap ? 0.f : -m[h]);
      }
      if constexpr (!PLAIN) {
        if (cap) {
#pragma unroll
          for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int h = 0; h < RPT; ++h) x[h][i] = fmaf(cap_out, tanh_rel(x[h][i]), -m[h]);
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int r = 8 * (i >> 1) + col_pos(2 * t4 + (i & 1)), pos = pos0 + r;
#pragma unroll
          for (int h = 0; h < RPT; ++h) {
            if (p.alibi) x[h][i] = fmaf(slope[h], (float)pos - qpos[h], x[h][i]);
            if (!(pos >= rlo[h] && pos < rhi[h] && ((have >> r) & 1))) x[h][i] = -INFINITY;
          }
        }
      }
      bool move = false;
#pragma unroll
      for (int r = 0; r < RPT; ++r) move |= max_of(x[r]) > above[r];
      if (UNLIKELY(__any_sync(~0u, move))) {
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
          // the reference moves by what fp32 has room for, and everything else by the same
          float top = above[r] == LAZY ? 0.f : -INFINITY;   // a row's first keys may lower it
          raise(top, x[r]);
          if (top == -INFINITY) continue;          // nothing seen yet
          const float by = (m[r] + top) - m[r];
          // before a row's first keys l and o hold 0 (or NaN): scaled by 2^-by, infinite where by <= -128, they would be NaN
          if (above[r] == LAZY) {
            // u rises by what whole powers of two the weights so far fall by: o keeps its size, and the weights that count
            // from now on keep their bits however large the V scales of keys that no longer do
            const int lift = min(__float2int_rz(by), 253 - (__float_as_int(up[r]) >> 23));   // to 2^126 at most
            up[r] = __int_as_float(__float_as_int(up[r]) + (lift << 23));
            l[r] *= ex2(-by);
            scale_rows<NT, RT>(o, r, ex2((float)lift - by));
          }
          m[r] += by;
          above[r] = LAZY;
#pragma unroll
          for (int i = 0; i < NP; ++i) x[r][i] -= by;
        }
      }
      float w[RPT][NP];
      move = false;
#pragma unroll
      for (int r = 0; r < RPT; ++r) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const float e = ex2(x[r][i]);
          l[r] += e;
          w[r][i] = e * vs[i];
        }
        if constexpr (!PLAIN)
#pragma unroll
          for (int i = 0; i < NP; ++i)
            if (x[r][i] == -INFINITY) w[r][i] = 0.f;   // whatever the scale is
        move |= max_of(w[r]) * up[r] > MOST;
      }
      if (UNLIKELY(__any_sync(~0u, move))) {
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
          float most = 0.f;
          raise(most, w[r]);
          const float to = fminf(up[r], pow2(LIFT - min(exponent(most), 128)));
          scale_rows<NT, RT>(o, r, to * (1.f / up[r]));
          up[r] = to;
        }
      }

      // ---- O += W V, 16 positions (two n tiles of S) a time
#pragma unroll
      for (int b = 0; b < ST / 16; ++b) {
        uint32_t wa[4], wl[4];
#pragma unroll
        for (int r = 0; r < RPT; ++r)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t hi, lo;
            split(w[r][4 * b + 2 * j] * up[r], w[r][4 * b + 2 * j + 1] * up[r], hi, lo);
            if constexpr (RT == 8) {
              wa[2 * j] = hi;
              wa[2 * j + 1] = lo;
            } else {
              wa[2 * j + r] = hi;
              wl[2 * j + r] = lo;
            }
          }
        // the thread's rows: positions 16 b + 8 (j >> 1) + col_pos(2 t4 + (j & 1)); what no row sees may be
        // anything, and 0 * NaN is not 0
        const unsigned char* const vsrc = src + C::HALF_B + b * 16 * C::ROW;
        unsigned hidden = 0;
        if constexpr (!PLAIN) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 16 * b + 8 * (j >> 1) + col_pos(2 * t4 + (j & 1));
            if (!(pos0 + r >= sq.lo && pos0 + r < sq.L && ((have >> r) & 1))) hidden |= 1u << j;
          }
        }
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          using Piece = std::conditional_t<W == 64, uint2, uint4>;
          Piece v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[j] = *reinterpret_cast<const Piece*>(vsrc + c * (ST * 128) + ((j & 1) ? vat1 : vat0) + (j >> 1) * 8 * C::ROW);
          if (UNLIKELY(hidden)) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if ((hidden >> j) & 1) v[j] = Piece{};
          }
#pragma unroll
          for (int i = 0; i < (int)sizeof(Piece) / 4; ++i) {
            uint32_t v0[4], v1[4];
            Conv<Q>::across((&v[0].x)[i], (&v[1].x)[i], v0);
            Conv<Q>::across((&v[2].x)[i], (&v[3].x)[i], v1);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              mma(o[16 * c + 4 * i + n], wa, v0[n], v1[n]);
              if constexpr (RT == 16) mma(o[16 * c + 4 * i + n], wl, v0[n], v1[n]);
            }
          }
        }
      }

      };
      if (have == ALL && pos0 >= all_lo && pos0 + ST <= all_hi) weigh(std::true_type{});
      else weigh(std::false_type{});

      __syncwarp();                                 // every lane has read the stage
      if (k + STAGES < k1) {
        if constexpr (TMA) issue(k + STAGES, stage);
        else issue_small(k + STAGES, stage);
      }
      cp_commit();
      if (++stage == STAGES) { stage = 0; parity ^= 1; }
    }
    if (k_lost >= 0) {   // let what is in flight land before the CTA's memory goes
      for (int i = 0; i < STAGES && k_lost + i < k1; ++i) {
        sm100::mbar_wait(sm100::smem_u32(&s_full[warp][stage]), parity, 1000000000ull);
        if (++stage == STAGES) { stage = 0; parity ^= 1; }
      }
      break;
    }

    // ---- the piece's result.  Column 2 t4 + h of n tile i belongs to thread g' = 2 t4 + h of the B
    // operand: dims PIECE * (g' + 8 c) + i, i < PIECE
    constexpr int PIECE = W == 64 ? 8 : 16;
    const bool whole_seq = k0 == 0 && k1 == sq.strips;
    float* const slot = slots + (k0 == 0 ? C::SLOT : 0);
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      l[r] += __shfl_xor_sync(~0u, l[r], 1);
      l[r] += __shfl_xor_sync(~0u, l[r], 2);
      const float back = 1.f / up[r];
      const float f = whole_seq ? (l[r] == 0.f ? 0.f : back / l[r]) : back;
      const int row = tile * RT + g + 8 * r, tok = row / p.gqa, head = kvh * p.gqa + row % p.gqa;
      if (tok >= sq.n) continue;
      if (t4 == 0) {
        if (whole_seq) {
          store_lse(p, sq.first + tok, head, m[r], l[r]);
        } else {
          slot[g + 8 * r] = above[r] == LAZY ? m[r] : NONE;
          slot[RT + g + 8 * r] = l[r];
        }
      }
#pragma unroll
      for (int c = 0; c < VC; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d = PIECE * (2 * t4 + h + 8 * c);
          float v[PIECE];
#pragma unroll
          for (int i = 0; i < PIECE; ++i)
            v[i] = (RT == 8 ? o[PIECE * c + i][h] + o[PIECE * c + i][2 + h] : o[PIECE * c + i][2 * r + h]) * f;
          if (whole_seq) {
            if (d < p.dim) store_n(p.o, dtype, ((sq.first + tok) * p.NH + head) * p.dim + d, v, PIECE);
          } else {
            store_n(slot, FA_DTYPE_F32, 2 * RT + (g + 8 * r) * W + d, v, PIECE);
          }
        }
    }
    if (k0 == 0 && k1 < sq.strips) {   // goes on in the ranges that follow
      cut.first = sq.first;
      cut.tile = tile;
      cut.rows = sq.n * p.gqa;
      cut.parts = (int)((at + sq.strips - 1) / per - range) + 1;
    }
    at += k1 - k0;
    if (at < end && at - off >= (long long)sq.strips * sq.tiles) {
      do {
        off += (long long)sq.strips * sq.tiles;
        sq = seq_of<RT, C::ST>(p, pg, ++z);
      } while (sq.tiles == 0);
    }
  }
  if (lane == 0) cuts[gw] = cut;
}

// ---------------------------------------------------------------- the join of cut sequences
// A row of a cut sequence and kv head is one item.  Which ranges a cut begins in stands in their records, the same for every kv
// head: each CTA lists them for itself (a few KB from L2, in the same order everywhere).  Items of few parts, the rule in a batch,
// are taken by a warp each; those of many, a long sequence's, by a CTA each, so that one sequence's items spread over the
// whole GPU.  Either way an item takes two rounds of loads, all of each under way at once: the parts' maxima and
// sums, a thread each, then their outputs.  (Every item by a CTA: 27 us of 128 for 48 sequences of 1-9k tokens.)
constexpr int MW = 8, FEW = 16;
template <int E>
__device__ __forceinline__ void store_row(const FaDec8Params& p, int dtype, long long at, int d, const float* v) {
  if (d >= p.dim) return;
  at = at * p.dim + d;
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    if (dtype == FA_DTYPE_BF16) *reinterpret_cast<__nv_bfloat162*>((__nv_bfloat16*)p.o + at + e) = __floats2bfloat162_rn(v[e], v[e + 1]);
    else if (dtype == FA_DTYPE_F16) *reinterpret_cast<__half2*>((__half*)p.o + at + e) = __floats2half2_rn(v[e], v[e + 1]);
    else *reinterpret_cast<float2*>((float*)p.o + at + e) = make_float2(v[e], v[e + 1]);
  }
}
template <int W, int RT>
__global__ void __launch_bounds__(MW * 32) dec8_merge_kernel(const FaDec8Params p, const int dtype, const int ranges) {
  using C = Cfg<W, RT>;
  extern __shared__ int s_cut[];                    // ranges that a cut begins in, few parts from the front, many from
  float* const s_f = reinterpret_cast<float*>(s_cut + ranges);   // the back; the factors of an item's parts
  __shared__ int s_few[MW], s_many[MW];
  __shared__ float s_m[MW], s_l[MW];
  __shared__ __align__(16) float s_v[MW][W];
  const int NKV = p.NH / p.gqa, tid = threadIdx.x, w = tid / 32, lane = tid % 32;
  pdl_wait();
  pdl_trigger();
  const Cut* const cuts = reinterpret_cast<const Cut*>(p.scratch);
  int few = 0, many = 0;
  for (int base = 0; base < ranges; base += MW * 32) {
    const int parts = base + tid < ranges ? cuts[(long long)(base + tid) * NKV].parts : 0;
    const unsigned vf = __ballot_sync(~0u, parts > 0 && parts <= FEW), vm = __ballot_sync(~0u, parts > FEW);
    if (lane == 0) {
      s_few[w] = __popc(vf);
      s_many[w] = __popc(vm);
    }
    __syncthreads();
    const unsigned below = (1u << lane) - 1;
    int af = few + __popc(vf & below), am = many + __popc(vm & below);
#pragma unroll
    for (int i = 0; i < MW; ++i) {
      if (i < w) {
        af += s_few[i];
        am += s_many[i];
      }
      few += s_few[i];
      many += s_many[i];
    }
    if (parts > FEW) s_cut[ranges - 1 - am] = base + tid;
    else if (parts > 0) s_cut[af] = base + tid;
    __syncthreads();
  }
  const float* const slots = p.scratch + (long long)ranges * NKV * (sizeof(Cut) / 4);
  constexpr int E = W / 32;
  // part 0 of a cut that begins in the range of warp gw: its second slot; part i: first slot of the warp i ranges on
  auto part = [&](int gw, int i) { return slots + ((long long)(gw + i * NKV) * 2 + (i == 0)) * C::SLOT; };

  for (int item = blockIdx.x * MW + w; item < few * NKV * RT; item += gridDim.x * MW) {
    const int r = item % RT, kvh = item / RT % NKV, gw = s_cut[item / RT / NKV] * NKV + kvh;
    const Cut cut = cuts[gw];
    const int row = cut.tile * RT + r;
    if (row >= cut.rows) continue;
    float m = NONE, f = 0.f, l = 0.f, v[E];
    if (lane < cut.parts) {
      m = part(gw, lane)[r];
      l = part(gw, lane)[RT + r];
    }
    float all = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(~0u, all, o));
    if (lane < cut.parts) f = ex2(m - all);
    l *= f;
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int i = 0; i < cut.parts; ++i) {
      const float* const o = part(gw, i) + 2 * RT + r * W + lane * E;
      const float fi = __shfl_sync(~0u, f, i);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 u = *reinterpret_cast<const float2*>(o + e);
        v[e] = fmaf(u.x, fi, v[e]);
        v[e + 1] = fmaf(u.y, fi, v[e + 1]);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = l == 0.f ? 0.f : v[e] / l;
    const int head = kvh * p.gqa + row % p.gqa;
    store_row<E>(p, dtype, (cut.first + row / p.gqa) * p.NH + head, lane * E, v);
    if (lane == 0) store_lse(p, cut.first + row / p.gqa, head, all, l);
  }

  for (int item = blockIdx.x; item < many * NKV * RT; item += gridDim.x) {
    const int r = item % RT, kvh = item / RT % NKV, gw = s_cut[ranges - 1 - item / RT / NKV] * NKV + kvh;
    const Cut cut = cuts[gw];
    const int row = cut.tile * RT + r;
    if (row >= cut.rows) continue;
    float m = NONE;
    for (int i = tid; i < cut.parts; i += MW * 32) {
      s_f[i] = part(gw, i)[r];
      m = fmaxf(m, s_f[i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (lane == 0) s_m[w] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MW; ++i) m = fmaxf(m, s_m[i]);
    float l = 0.f;
    for (int i = tid; i < cut.parts; i += MW * 32) {
      const float f = ex2(s_f[i] - m);
      s_f[i] = f;
      l = fmaf(part(gw, i)[RT + r], f, l);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
    if (lane == 0) s_l[w] = l;
    __syncthreads();
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 8
    for (int i = w; i < cut.parts; i += MW) {
      const float* const o = part(gw, i) + 2 * RT + r * W + lane * E;
      const float f = s_f[i];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 u = *reinterpret_cast<const float2*>(o + e);
        v[e] = fmaf(u.x, f, v[e]);
        v[e + 1] = fmaf(u.y, f, v[e + 1]);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_v[w][lane * E + e] = v[e];
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int i = 0; i < MW; ++i) l += s_l[i];
    const int head = kvh * p.gqa + row % p.gqa;
    for (int d = 2 * tid; d < p.dim; d += MW * 64) {
      float x[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < MW; ++i) {
        x[0] += s_v[i][d];
        x[1] += s_v[i][d + 1];
      }
      x[0] = l == 0.f ? 0.f : x[0] / l;
      x[1] = l == 0.f ? 0.f : x[1] / l;
      store_row<2>(p, dtype, (cut.first + row / p.gqa) * p.NH + head, d, x);
    }
    if (tid == 0) store_lse(p, cut.first + row / p.gqa, head, m, l);
    __syncthreads();
  }

  if (!p.cu_q) return;   // rows of no sequence (a padded batch's): 0 and -infinity, a warp a row and head
  const long long from = min(max((long long)__ldg(p.cu_q), 0ll), p.total), to = min(max((long long)__ldg(p.cu_q + p.batch), from), p.total);
  for (long long item = blockIdx.x * MW + w; item < (from + p.total - to) * p.NH; item += gridDim.x * MW) {
    const long long i = item / p.NH, row = i < from ? i : to + i - from;
    const int head = (int)(item % p.NH);
    const float zero[2] = {0.f, 0.f};
    for (int d = 2 * lane; d < p.dim; d += 64) store_row<2>(p, dtype, row * p.NH + head, d, zero);
    if (lane == 0) store_lse(p, row, head, 0.f, 0.f);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }
  return fn;
}

// The cache as rows of `dim` bytes: (dim, kv heads, slots); a box is `row` bytes of one head in `run` slots, what lies past dim
// comes as zeros.
int map_of(CUtensorMap* m, const void* base, const FaDec8Params& p, int row, int strip) {
  const auto enc = encode_fn();
  const cuuint64_t heads = p.NH / p.gqa;
  const cuuint64_t dims[3] = {(cuuint64_t)p.dim, heads, (cuuint64_t)p.num_blocks * p.page};
  const cuuint64_t strides[2] = {(cuuint64_t)p.dim, heads * p.dim};
  const cuuint32_t box[3] = {(cuuint32_t)row, 1, (cuuint32_t)std::min(p.page, strip)};
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult e = !enc ? CUDA_ERROR_NOT_FOUND
                          : enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, one,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (e == CUDA_SUCCESS) return FA_OK;
  fa::set_error("8-bit decode: cuTensorMapEncodeTiled failed (%d)", (int)e);
  return FA_ERR_CUDA;
}

template <int W, typename Q, int RT, bool TMA>
int launch(const FaDec8Params& p, int dtype, cudaStream_t st) {
  using C = Cfg<W, RT>;
  static unsigned long long done = 0;
  if (int rc = fa::ensure_smem((const void*)dec8_kernel<W, Q, RT, TMA>, C::SMEM, &done)) return rc;
  CUtensorMap mk, mv;
  if (int rc = map_of(&mk, p.Kc, p, C::ROW, C::ST)) return rc;
  if (int rc = map_of(&mv, p.Vc, p, C::ROW, C::ST)) return rc;
  const Pages pg{p.block_table, log2_of(p.page), p.max_blocks, p.num_blocks};
  const int NKV = p.NH / p.gqa, warps = fa::num_sms() * C::CTAS * C::NW;
  // no more ranges than the block table's width allows strips for: a small call then starts and joins few warps
  const long long tiles = ((long long)(p.cu_q ? p.max_tokens : p.tokens) * p.gqa + RT - 1) / RT;
  const long long strips = p.batch * tiles * (((long long)p.max_blocks * p.page + C::ST - 1) / C::ST);
  const int ranges = (int)std::max(1ll, std::min<long long>(warps / NKV, strips));
  const int need = (ranges * NKV + C::NW - 1) / C::NW;
  cudaError_t e = fa::launch_pdl(dec8_kernel<W, Q, RT, TMA>, dim3(need), dim3(C::NW * 32), C::SMEM, st, mk, mv, p, pg, dtype, ranges);
  fa::count_launch();
  if (int rc = fa::cuda_status(e, "8-bit decode launch")) return rc;
  e = fa::launch_pdl(dec8_merge_kernel<W, RT>, dim3(std::min(4 * fa::num_sms(), ranges * NKV * RT)), dim3(MW * 32),
                                       (size_t)ranges * 8, st, p, dtype, ranges);
  fa::count_launch();
  return fa::cuda_status(e, "8-bit decode merge launch");
}

// A box takes slots of one page: pages of 8 and less would make four or more copies of a strip of 32, and go by the warp's own
// 16-byte copies.
template <int W, typename Q, int RT>
int by_page(const FaDec8Params& p, int dtype, cudaStream_t st) {
  return p.page < 16 ? launch<W, Q, RT, false>(p, dtype, st) : launch<W, Q, RT, true>(p, dtype, st);
}
template <int W, typename Q>
int by_rows(const FaDec8Params& p, int dtype, cudaStream_t st) {
  // More than 8 rows a sequence: one pass over the cache with 16 rows, or tiles of 8 that each make a pass.  16 rows win
  // where every sequence has them (16 x 16-32k tokens, 16 heads a kv head, headdim 128: int8 252 against 301 us, e4m3 254
  // against 299; headdim 64, int8: 205 against 193); tiles win where counts are ragged, since most tiles of 16 are then half
  // empty (1 to 4 tokens of 4 heads, 24 x 1-20k int8 tokens, window 4096 and softcap: 104 against 88 us, without either 185
  // against 157), and for rows of 256, whose 16-row form has one warp a scheduler (16 x 1-9k tokens, 16 heads, before int8 took
  // integer mma: 127 against 108 us).
  const bool full = p.gqa > 8 || (!p.cu_q && (long long)p.gqa * p.tokens > 8);
  if constexpr (W <= 128)
    if (full) return by_page<W, Q, 16>(p, dtype, st);
  return by_page<W, Q, 8>(p, dtype, st);
}
template <typename Q>
int by_dim(const FaDec8Params& p, int dtype, cudaStream_t st) {
  if (p.dim <= 64) return by_rows<64, Q>(p, dtype, st);
  if (p.dim <= 128) return by_rows<128, Q>(p, dtype, st);
  return by_rows<256, Q>(p, dtype, st);
}

template <int W, int RT>
long long scratch_of(int NKV) {
  using C = Cfg<W, RT>;
  const long long warps = (long long)fa::num_sms() * C::CTAS * C::NW, used = std::max<long long>(1, warps / NKV) * NKV;
  return used * (sizeof(Cut) / 4 + 2ll * C::SLOT);
}

}  // namespace

namespace fa {
int dec8_device_error(int clear) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_dec8_error, sizeof(int));
  if (clear && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_dec8_error, &zero, sizeof(int));
  }
  return v;
}
}  // namespace fa

extern "C" FA_API long long fa_decode8_scratch_floats(int NH, int gqa, int dim) {
  if (NH <= 0 || gqa <= 0 || NH % gqa || dim <= 0) return 0;
  const int n = NH / gqa;
  if (dim <= 64) return std::max(scratch_of<64, 8>(n), scratch_of<64, 16>(n));
  if (dim <= 128) return std::max(scratch_of<128, 8>(n), scratch_of<128, 16>(n));
  return scratch_of<256, 8>(n);
}

extern "C" FA_API int fa_decode8_launch(const FaDec8Params* pp, int dtype, void* stream) {
  FA_ABI_GUARD(pp, FaDec8Params);
  FaDec8Params p = *pp;
  FA_CHECK_ARG(dtype == FA_DTYPE_F16 || dtype == FA_DTYPE_BF16 || dtype == FA_DTYPE_F32, "8-bit decode: dtype code %d", dtype);
  FA_CHECK_ARG(p.code == FA_CODE_I8 || p.code == FA_CODE_E4M3, "8-bit decode: cache element code %d", p.code);
  FA_CHECK_ARG(p.q && p.Kc && p.Vc && p.Ks && p.Vs && p.block_table && p.ctx_len && p.o,
               "8-bit decode: q, Kc, Vc, Ks, Vs, block_table, ctx_len, o must be non-null");
  FA_CHECK_ARG(p.batch >= 0 && p.NH > 0 && p.gqa > 0 && p.NH % p.gqa == 0, "8-bit decode: batch=%d NH=%d gqa=%d", p.batch,
               p.NH, p.gqa);
  FA_CHECK_ARG(p.page > 0 && (p.page & (p.page - 1)) == 0 && p.max_blocks > 0 && p.num_blocks > 0,
               "8-bit decode: page=%d must be a power of two, max_blocks=%d and num_blocks=%lld positive", p.page,
               p.max_blocks, p.num_blocks);
  FA_CHECK_ARG(p.block > 0 && (p.block & (p.block - 1)) == 0 && p.block <= p.page && p.block <= 256,
               "8-bit decode: block=%d must be a power of two, at most page=%d and 256", p.block, p.page);
  FA_CHECK_ARG(p.total >= 0 && (p.cu_q || p.total == (long long)p.batch * p.tokens),
               "8-bit decode: total=%lld rows, batch=%d tokens=%d", p.total, p.batch, p.tokens);
  if (p.cos)
    FA_CHECK_ARG(p.sin && p.rot_dim > 0 && p.rot_dim % 2 == 0 && p.rot_dim <= p.dim && p.rot_seqlen_ro > 0,
                 "8-bit decode: rotary needs sin, an even rot_dim=%d in (0, dim], rot_seqlen_ro=%d > 0", p.rot_dim,
                 p.rot_seqlen_ro);
  if (!(p.dim > 0 && p.dim % 16 == 0 && p.dim <= 256)) {
    fa::set_error("8-bit decode: dim=%d must be a multiple of 16 up to 256", p.dim);
    return FA_ERR_UNSUPPORTED;
  }
  if (p.total == 0) return FA_OK;
  FA_CHECK_ARG(p.batch > 0, "8-bit decode: %lld rows of no sequence", p.total);
  if (p.total * p.NH >= 1ll << 31) {
    fa::set_error("8-bit decode: %lld rows of %d heads are more than one call takes", p.total, p.NH);
    return FA_ERR_SIZE;
  }
  FA_CHECK_ARG(p.scratch, "8-bit decode: scratch must be non-null");
  FA_CHECK_ARG(((uintptr_t)p.Kc | (uintptr_t)p.Vc | (uintptr_t)p.o | (uintptr_t)p.scratch) % 16 == 0,
               "8-bit decode: Kc, Vc, o and scratch must be 16-byte aligned");
  if (p.num_blocks * (long long)p.page >= 1ll << 31) {
    fa::set_error("8-bit decode: a cache of %lld pages of %d slots is more than one call takes", p.num_blocks, p.page);
    return FA_ERR_SIZE;
  }
  p.win_left = std::min(p.win_left, 1 << 30);   // position - win_left stays within 32 bits
  p.win_right = std::min(p.win_right, 1 << 30);
  cudaStream_t st = (cudaStream_t)stream;
  return p.code == FA_CODE_I8 ? by_dim<I8>(p, dtype, st) : by_dim<E4M3>(p, dtype, st);
}
