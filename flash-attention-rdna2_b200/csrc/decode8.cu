// decode8.cu — attention of new tokens over a paged cache held in 8 bits (fa_decode8_launch of
// fable_attn.h).
//
// One pass over the cache with a running maximum and sum.  For a key j with codes c_j, d_j and block
// scales ks_j, vs_j, and in base 2:  x_j = scale log2(e) ks_j (q . c_j),  o = sum 2^(x_j - m) vs_j d_j / sum 2^(x_j - m).
// The value scale joins the weight, w_j = 2^(x_j - m) vs_j u, where u is a power of two of the row's own that keeps the
// largest weight so far in fp16's range whatever the scales: the tensor cores take codes (exact in
// fp16) and weights (fp16 high and low part, 22 bits) as they are, and dividing by u at the end is exact.
//
// Bound by the bytes of the cache.  What is read goes through registers to mma.sync (m16n8k16, fp16
// operands, fp32 sums): with 8 query rows the tensor pipe has twice the time that the bytes need, and the conversion of codes
// has to pass through registers anyway.  A strip is 16 positions of one kv head.  Its K rows are the B operand of
// S = Q K^T, its V rows that of O += W V.  The order of an mma's k index and of its n columns is free as long as both operands
// agree, so each thread's operands are whole 16-byte pieces of cache rows: K, row g = lane / 4, pieces
// lane % 4 + 4 i; V, positions 2 (lane % 4) + {0, 1, 8, 9}, piece g.  A thread copies those pieces into
// shared memory with cp.async and reads back only its own: no barrier, no bank conflict, no ldmatrix.
// S leaves the tensor cores in the layout in which W enters them.
//
// Rows of a warp are (new token, query head) pairs of one kv head.  8 rows: the upper 8 rows of the
// m16 tile carry the low parts of q and of w, so that both have 22 bits for nothing.  16 rows: a second mma.
//
// Work split: the strips of all sequences (times the row tiles of each) form one line, cut into equal
// ranges, one for each warp of a kv head; the warps of a CTA take the heads of one range, so that the heads' rows,
// adjacent in memory, are read together.  A warp's range is cut at sequence ends; a piece that is a whole sequence
// writes its output, others leave (m, l, o) in one of the warp's two slots, and a merge kernel joins the slots of each
// cut sequence in order (no atomics: same bits on every call).
#include <algorithm>
#include <type_traits>
#include "fa_launch.h"
#include "kv8_common.cuh"

namespace {

using namespace fa_kv;

__device__ int g_dec8_error = 0;
__device__ __forceinline__ void record(int bit) { atomicOr(&g_dec8_error, bit); }

constexpr int ST = 16;             // positions of a strip
constexpr int NW = 4;              // warps of a CTA
constexpr float NONE = -1e30f;     // a running maximum that nothing has moved yet
constexpr float LAZY = 8.f;        // a score may exceed the running maximum by 8 (base 2) before it is moved
constexpr int LIFT = 6;            // weights are brought to [2^6, 2^7) ...
constexpr float MOST = 16384.f;    // ... when one exceeds 2^14: fp16 then reaches 2^-30 of the largest
constexpr int MIN_STRIPS = 2;      // least strips of a range

template <int W, int RT>
struct Cfg {
  // warps of an SM and their stages: what 64 K registers and 227 KB of shared memory hold
  static constexpr int CTAS = W == 256 ? (RT == 16 ? 1 : 2) : RT == 16 ? 2 : W == 64 ? 4 : 3;   // per SM
  static constexpr int STAGES = W == 256 && RT == 8 ? 2 : 4;
  static constexpr bool QREG = RT == 8 && W <= 128;                        // q operands stay in registers
  static constexpr int KS = W / 16;                                        // k steps of S
  static constexpr int STAGE_B = W * 32;                                   // K and V of a strip
  static constexpr int Q_B = QREG ? 0 : KS * 512 * (RT / 8);
  static constexpr int WARP_B = STAGES * (STAGE_B + 128 + 16) + Q_B;
  static constexpr int SMEM = NW * WARP_B;
  static_assert(SMEM * CTAS <= 227 * 1024, "shared memory of an SM");
  static constexpr int SLOT = RT * (W + 2);                                // floats of a slot: m[RT], l[RT], o[RT][W]
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ int exponent(float x) { return max(((__float_as_int(x) >> 23) & 255) - 127, -120); }
// m raised to the largest of it and a row's four values in each of its four threads; returns it
__device__ __forceinline__ float raise(float& m, const float* v) {
  float a = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
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
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool valid) {   // N bytes, zeros where not valid
  const int n = valid ? N : 0;
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
  // 4 bytes of one word -> (0, 1), (2, 3)
  static __device__ __forceinline__ void along(uint32_t w, uint32_t& p0, uint32_t& p1) {
    const uint32_t x = w ^ 0x80808080u;
    p0 = half_pair(x, 0x4140);
    p1 = half_pair(x, 0x4342);
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
  static __device__ __forceinline__ uint32_t two(uint32_t x, int up) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(up ? x >> 16 : x & 0xffffu), __NV_E4M3);
    return (uint32_t)r.x | ((uint32_t)r.y << 16);
  }
  static __device__ __forceinline__ void along(uint32_t w, uint32_t& p0, uint32_t& p1) {
    p0 = two(w, 0);
    p1 = two(w, 1);
  }
  static __device__ __forceinline__ void across(uint32_t a, uint32_t b, uint32_t* p) {
    const uint32_t x = __byte_perm(a, b, 0x5140), y = __byte_perm(a, b, 0x7362);
    p[0] = two(x, 0); p[1] = two(x, 1); p[2] = two(y, 0); p[3] = two(y, 1);
  }
};

// ---------------------------------------------------------------- geometry
struct Seq {
  int n, L, lo;           // new tokens, cached tokens, first key that any of them sees
  int s0, strips, tiles;  // first strip, strips (at least one, so that somebody writes the rows), row tiles
  long long first;        // its first row
};

template <int RT>
__device__ __forceinline__ Seq seq_of(const FaDec8Params& p, const Pages& pg, int z) {
  Seq s;
  const RowMap rm{p.cu_q, p.tokens, p.batch};
  s.first = rm.first(z);
  s.n = (int)max(0ll, min((long long)rm.count(z), p.total - s.first));
  if (s.first < 0) s.n = 0;
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

// element d.. of a q row; rotated by table row rp (rp < 0: as it is), in fp32
template <typename T>
__device__ __noinline__ void load_q4(const FaDec8Params& p, const void* row, int d, int rp, float* v) {
  const T* x = (const T*)row;
  const int half = p.rot_dim / 2;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = Elem<T>::to_f(x[d + e]);
  if (rp < 0 || d >= p.rot_dim) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = d + e;
    if (i >= p.rot_dim) break;
    const bool low = p.rot_interleaved ? !(i & 1) : i < half;
    const int j = p.rot_interleaved ? i / 2 : low ? i : i - half;
    const float b = Elem<T>::to_f(x[p.rot_interleaved ? i ^ 1 : low ? i + half : i - half]);
    const float c = __ldg(p.cos + (long long)rp * half + j), s = __ldg(p.sin + (long long)rp * half + j);
    v[e] = low ? v[e] * c - b * s : v[e] * c + b * s;
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

__device__ __forceinline__ void store_lse(const FaDec8Params& p, int z, long long row, int t, int head, float m, float l) {
  if (!p.lse) return;
  p.lse[p.cu_q ? head * p.total + row : ((long long)z * p.NH + head) * p.tokens + t] =
      l == 0.f ? -INFINITY : (m + lg2(l)) * FA_LN2;
}

struct Cut {   // the sequence whose strips begin in a warp's range and end in a later one
  int z, tile, parts, pad;
};

// ---------------------------------------------------------------- the pass over the cache
template <int W, typename Q, int RT>
__global__ void __launch_bounds__(NW * 32, (Cfg<W, RT>::CTAS))
    dec8_kernel(const FaDec8Params p, const Pages pg, const int dtype, const int ranges) {
  using C = Cfg<W, RT>;
  constexpr int STAGES = C::STAGES, KS = C::KS, NT = W / 8, KC = W / 64, VC = W == 256 ? 2 : 1;
  constexpr int RPT = RT / 8;        // rows of a thread: g, g + 8
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ long long s_pre[NW * 32 + 1], s_warp[NW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int NKV = p.NH / p.gqa;

  // ---- the line of strips: every thread sums a run of sequences
  const int CB = (p.batch + NW * 32 - 1) / (NW * 32);
  {
    long long mine = 0;
    for (int z = tid * CB; z < min(p.batch, (tid + 1) * CB); ++z) {
      const Seq s = seq_of<RT>(p, pg, z);
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
  Cut cut{0, 0, 0, 0};
  const long long per = max((long long)MIN_STRIPS, (total + ranges - 1) / ranges);
  const long long begin = range * per, end = min(total, begin + per);

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * C::WARP_B;
  const uint32_t scales = ring + STAGES * C::STAGE_B, masks = scales + STAGES * 128, qs = masks + STAGES * 16;
  const typename Q::T* const Kc = (const typename Q::T*)p.Kc;
  const typename Q::T* const Vc = (const typename Q::T*)p.Vc;
  const int pmask = p.page - 1, bshift = log2_of(p.block), per_page = p.page >> bshift;
  const bool wide = p.page >= ST;                   // a strip lies in one page

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
    sq = seq_of<RT>(p, pg, z);
    while (off + (long long)sq.strips * sq.tiles <= begin) {
      off += (long long)sq.strips * sq.tiles;
      sq = seq_of<RT>(p, pg, ++z);
    }
  }

  for (long long at = begin; at < end;) {
    // ---- a piece: strips [k0, k1) of row tile `tile` of sequence z
    const int tile = (int)((at - off) / sq.strips), k0 = (int)((at - off) % sq.strips);
    const int k1 = (int)min((long long)sq.strips, k0 + (end - at));

    auto issue = [&](int k, int stage) {            // strip k of the sequence into a stage
      const int pos0 = (sq.s0 + k) * ST;
      const uint32_t dst = ring + stage * C::STAGE_B;
      long long blk = 0;
      if (wide) blk = pg.of(z, pos0);
      auto slot_of = [&](int r) -> long long {      // cache row of position pos0 + r, -1 for none
        const int pos = pos0 + r;
        if (pos < sq.lo || pos >= sq.L) return -1;
        const long long b = wide ? blk : pg.of(z, pos);
        return b < 0 ? -1 : b * p.page + (pos & pmask);
      };
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const long long s = slot_of(g + 8 * j);
        const typename Q::T* src = Kc + (s < 0 ? 0 : (s * NKV + kvh) * p.dim);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const int d = 16 * (t4 + 4 * c);
          const bool ok = s >= 0 && d < p.dim;
          cp_async<16>(dst + (j * KC + c) * 512 + lane * 16, ok ? src + d : Kc, ok);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long s = slot_of(2 * t4 + (j & 1) + 8 * (j >> 1));
        const typename Q::T* src = Vc + (s < 0 ? 0 : (s * NKV + kvh) * p.dim);
        if constexpr (W == 64) {
          const bool ok = s >= 0 && 8 * g < p.dim;
          cp_async<8>(dst + 2 * KC * 512 + j * 256 + lane * 8, ok ? src + 8 * g : Vc, ok);
        } else {
#pragma unroll
          for (int c = 0; c < VC; ++c) {
            const int d = 16 * (g + 8 * c);
            const bool ok = s >= 0 && d < p.dim;
            cp_async<16>(dst + 2 * KC * 512 + (j * VC + c) * 512 + lane * 16, ok ? src + d : Vc, ok);
          }
        }
      }
      {   // lanes 0-15: K scale of position lane; 16-31: V scale
        const int r = lane & 15;
        const long long s = slot_of(r);
        const float* sc = lane < 16 ? p.Ks : p.Vs;
        const long long b = s < 0 ? 0 : (wide ? blk : s / p.page);
        const long long i = s < 0 ? 0 : (b * NKV + kvh) * per_page + (((pos0 + r) & pmask) >> bshift);
        cp_async<4>(scales + stage * 128 + lane * 4, sc + i, s >= 0);
        const bool in = pos0 + r >= sq.lo && pos0 + r < sq.L;
        const uint32_t have = __ballot_sync(~0u, s >= 0) & 0xffffu;
        if (in && s < 0) record(ERR_PAGE);
        if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(masks + stage * 16), "r"(have) : "memory");
      }
    };

    __syncwarp();                                   // the last piece's stages and q are free
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      if (k0 + i < k1) issue(k0 + i, i);
      cp_commit();
    }

    // ---- the rows: ranges of keys, factors, q operands
    uint32_t qa[C::QREG ? KS : 1][4];
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
      float x[KS * 4], most = 0.f;
#pragma unroll
      for (int c = 0; c < KS; ++c) {                // step c = 4 i + w: piece t4 + 4 i, word w
        const int d = 16 * (t4 + 4 * (c / 4)) + 4 * (c % 4);
        float* v = x + 4 * c;
        v[0] = v[1] = v[2] = v[3] = 0.f;
        if (live && d < p.dim) {
          if (dtype == FA_DTYPE_BF16) load_q4<__nv_bfloat16>(p, (const __nv_bfloat16*)p.q + qe, d, rp, v);
          else if (dtype == FA_DTYPE_F16) load_q4<__half>(p, (const __half*)p.q + qe, d, rp, v);
          else load_q4<float>(p, (const float*)p.q + qe, d, rp, v);
        }
        most = fmaxf(most, fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));
      }
      // rows are brought to [1, 2) by a power of two, so that fp16 holds them whatever their size
      most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
      most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
      const int e = min(exponent(most), 126);
      const float down = pow2(-e);
      qf[r] = p.scale * pow2(e);
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        uint32_t h0, l0, h1, l1;
        split(x[4 * c] * down, x[4 * c + 1] * down, h0, l0);
        split(x[4 * c + 2] * down, x[4 * c + 3] * down, h1, l1);
        if constexpr (C::QREG) {
          qa[c][0] = h0; qa[c][1] = l0; qa[c][2] = h1; qa[c][3] = l1;
        } else if constexpr (RT == 8) {
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(qs + c * 512 + lane * 16), "r"(h0), "r"(l0), "r"(h1),
                       "r"(l1) : "memory");
        } else {   // operand words: 0 row g, 1 row g + 8 (first pair); 2, 3 (second pair); low parts behind
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(qs + c * 512 + lane * 16 + 4 * r), "r"(h0) : "memory");
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(qs + c * 512 + lane * 16 + 8 + 4 * r), "r"(h1) : "memory");
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(qs + (KS + c) * 512 + lane * 16 + 4 * r), "r"(l0) : "memory");
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(qs + (KS + c) * 512 + lane * 16 + 8 + 4 * r), "r"(l1) : "memory");
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
    all_hi = __reduce_min_sync(~0u, all_hi);

    float o[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[RPT], l[RPT], up[RPT];
#pragma unroll
    for (int r = 0; r < RPT; ++r) { m[r] = NONE; l[r] = 0.f; up[r] = pow2(126); }
    const bool cap = p.softcap > 0.f;
    const float cap_in = cap ? 1.f / p.softcap : FA_LOG2E, cap_out = p.softcap * FA_LOG2E;

    for (int k = k0; k < k1; ++k) {
      const int stage = (k - k0) % STAGES;
      cp_wait<STAGES - 2>();
      __syncwarp();
      if (k + STAGES - 1 < k1) issue(k + STAGES - 1, (k - k0 + STAGES - 1) % STAGES);
      cp_commit();
      const uint32_t src = ring + stage * C::STAGE_B + lane * 16;

      // ---- S = Q K^T: columns j * 8 + 2 t4 + {0, 1}
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        uint4 kk[2];
        kk[0] = lds128(src + c * 512);
        kk[1] = lds128(src + (KC + c) * 512);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t qv[4], ql[4];
          if constexpr (C::QREG) {
#pragma unroll
            for (int i = 0; i < 4; ++i) qv[i] = qa[4 * c + w][i];
          } else {
            const uint4 u = lds128(qs + (4 * c + w) * 512 + lane * 16);
            qv[0] = u.x; qv[1] = u.y; qv[2] = u.z; qv[3] = u.w;
            if constexpr (RT == 16) {
              const uint4 v = lds128(qs + (KS + 4 * c + w) * 512 + lane * 16);
              ql[0] = v.x; ql[1] = v.y; ql[2] = v.z; ql[3] = v.w;
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t b0, b1;
            Conv<Q>::along((&kk[j].x)[w], b0, b1);
            mma(s[j], qv, b0, b1);
            if constexpr (RT == 16) mma(s[j], ql, b0, b1);
          }
        }
      }

      // ---- weights of positions pos0 + 8 j + 2 t4 + e, row g (+ 8 r)
      const int pos0 = (sq.s0 + k) * ST;
      uint32_t have;
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(have) : "r"(masks + stage * 16) : "memory");
      const bool whole = have == 0xffffu && pos0 >= all_lo && pos0 + ST <= all_hi;
      float x[RPT][4], vs[4];
      bool move = false;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint2 ku = lds64(scales + stage * 128 + (8 * j + 2 * t4) * 4), vu = lds64(scales + stage * 128 + (16 + 8 * j + 2 * t4) * 4);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ks = __uint_as_float(e ? ku.y : ku.x);
          vs[2 * j + e] = __uint_as_float(e ? vu.y : vu.x);
          const int pos = pos0 + 8 * j + 2 * t4 + e;
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            float v = (RT == 8 ? s[j][e] + s[j][2 + e] : s[j][2 * r + e]) * ks * qf[r] * cap_in;
            if (cap) v = cap_out * fa_tanh(v);
            if (p.alibi) v = fmaf(slope[r], (float)pos - qpos[r], v);
            if (!whole && !(pos >= rlo[r] && pos < rhi[r] && ((have >> (pos - pos0)) & 1))) v = -INFINITY;
            x[r][2 * j + e] = v;
            move |= v > m[r] + LAZY;
          }
        }
      }
      if (__any_sync(~0u, move)) {
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
          const float was = m[r], f = ex2(was - raise(m[r], x[r]));
          l[r] *= f;
          scale_rows<NT, RT>(o, r, f);
        }
      }
      float w[RPT][4];
      move = false;
#pragma unroll
      for (int r = 0; r < RPT; ++r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = ex2(x[r][i] - m[r]);
          l[r] += e;
          w[r][i] = x[r][i] == -INFINITY ? 0.f : e * vs[i];
          move |= w[r][i] * up[r] > MOST;
        }
      }
      if (__any_sync(~0u, move)) {
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
          float most = 0.f;
          raise(most, w[r]);
          const float to = fminf(up[r], pow2(LIFT - min(exponent(most), 128)));
          scale_rows<NT, RT>(o, r, to * (1.f / up[r]));
          up[r] = to;
        }
      }
      uint32_t wa[4], wl[4];
#pragma unroll
      for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t hi, lo;
          split(w[r][2 * j] * up[r], w[r][2 * j + 1] * up[r], hi, lo);
          if constexpr (RT == 8) {
            wa[2 * j] = hi;
            wa[2 * j + 1] = lo;
          } else {
            wa[2 * j + r] = hi;
            wl[2 * j + r] = lo;
          }
        }

      // ---- O += W V
      const uint32_t vsrc = ring + stage * C::STAGE_B + 2 * KC * 512;
      if constexpr (W == 64) {
        uint2 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = lds64(vsrc + j * 256 + lane * 8);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t b0[4], b1[4];
          Conv<Q>::across((&v[0].x)[w], (&v[1].x)[w], b0);
          Conv<Q>::across((&v[2].x)[w], (&v[3].x)[w], b1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            mma(o[4 * w + i], wa, b0[i], b1[i]);
            if constexpr (RT == 16) mma(o[4 * w + i], wl, b0[i], b1[i]);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          uint4 v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = lds128(vsrc + (j * VC + c) * 512 + lane * 16);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t b0[4], b1[4];
            Conv<Q>::across((&v[0].x)[w], (&v[1].x)[w], b0);
            Conv<Q>::across((&v[2].x)[w], (&v[3].x)[w], b1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              mma(o[16 * c + 4 * w + i], wa, b0[i], b1[i]);
              if constexpr (RT == 16) mma(o[16 * c + 4 * w + i], wl, b0[i], b1[i]);
            }
          }
        }
      }
    }
    cp_wait<0>();

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
          store_lse(p, z, sq.first + tok, tok, head, m[r], l[r]);
        } else {
          slot[g + 8 * r] = m[r];
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
      cut.z = z;
      cut.tile = tile;
      cut.parts = (int)((at + sq.strips - 1) / per - range) + 1;
    }
    at += k1 - k0;
    if (at < end && at - off >= (long long)sq.strips * sq.tiles) {
      do {
        off += (long long)sq.strips * sq.tiles;
        sq = seq_of<RT>(p, pg, ++z);
      } while (sq.tiles == 0);
    }
  }
  if (lane == 0) cuts[gw] = cut;
  pdl_trigger();
}

// ---------------------------------------------------------------- the join of cut sequences
// One CTA for the warp whose range a cut sequence begins in, one warp per row.
template <int W, int RT>
__global__ void __launch_bounds__(RT * 32)
    dec8_merge_kernel(const FaDec8Params p, const Pages pg, const int dtype, const int ranges) {
  using C = Cfg<W, RT>;
  pdl_wait();
  const int NKV = p.NH / p.gqa, gw = blockIdx.x, kvh = gw % NKV, r = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Cut cut = reinterpret_cast<const Cut*>(p.scratch)[gw];
  if (cut.parts == 0) return;
  const Seq sq = seq_of<RT>(p, pg, cut.z);
  const int row = cut.tile * RT + r, tok = row / p.gqa, head = kvh * p.gqa + row % p.gqa;
  if (tok >= sq.n) return;
  const float* slots = p.scratch + (long long)ranges * NKV * (sizeof(Cut) / 4);
  // part 0: second slot of warp gw; part i: first slot of the warp i ranges on
  auto part = [&](int i) { return slots + ((long long)(gw + i * NKV) * 2 + (i == 0)) * C::SLOT; };
  float m = NONE;
  for (int i = lane; i < cut.parts; i += 32) m = fmaxf(m, part(i)[r]);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  constexpr int E = W / 32;
  float l = 0.f, v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < cut.parts; ++i) {
    const float* s = part(i);
    const float f = ex2(s[r] - m);
    l = fmaf(s[RT + r], f, l);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 u = *reinterpret_cast<const float2*>(s + 2 * RT + r * W + lane * E + e);
      v[e] = fmaf(u.x, f, v[e]);
      v[e + 1] = fmaf(u.y, f, v[e + 1]);
    }
  }
  const float f = l == 0.f ? 0.f : 1.f / l;
  const long long at = ((sq.first + tok) * p.NH + head) * p.dim;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane * E + e;
    if (d >= p.dim) break;
    if (dtype == FA_DTYPE_BF16) ((__nv_bfloat16*)p.o)[at + d] = __float2bfloat16_rn(v[e] * f);
    else if (dtype == FA_DTYPE_F16) ((__half*)p.o)[at + d] = __float2half_rn(v[e] * f);
    else ((float*)p.o)[at + d] = v[e] * f;
  }
  if (lane == 0) store_lse(p, cut.z, sq.first + tok, tok, head, m, l);
}

template <int W, typename Q, int RT>
int launch(const FaDec8Params& p, int dtype, cudaStream_t st) {
  using C = Cfg<W, RT>;
  static unsigned long long done = 0;
  if (int rc = fa::ensure_smem((const void*)dec8_kernel<W, Q, RT>, C::SMEM, &done)) return rc;
  const Pages pg{p.block_table, log2_of(p.page), p.max_blocks, p.num_blocks};
  const int NKV = p.NH / p.gqa, grid = fa::num_sms() * C::CTAS, warps = grid * NW;
  const int ranges = std::max(1, warps / NKV), need = (ranges * NKV + NW - 1) / NW;
  dec8_kernel<W, Q, RT><<<need, NW * 32, C::SMEM, st>>>(p, pg, dtype, ranges);
  fa::count_launch();
  if (int rc = fa::cuda_status(cudaGetLastError(), "8-bit decode launch")) return rc;
  const cudaError_t e = fa::launch_pdl(dec8_merge_kernel<W, RT>, dim3(ranges * NKV), dim3(RT * 32), 0, st, p, pg, dtype, ranges);
  fa::count_launch();
  return fa::cuda_status(e, "8-bit decode merge launch");
}

template <int W, typename Q>
int by_rows(const FaDec8Params& p, int dtype, cudaStream_t st) {
  // more than 8 rows share one pass over the cache; fp32 keeps to 8, whose q and weights have 22 bits
  const long long rows = (long long)p.gqa * (p.cu_q ? p.max_tokens : p.tokens);
  return rows > 8 ? launch<W, Q, 16>(p, dtype, st) : launch<W, Q, 8>(p, dtype, st);
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
  const long long warps = (long long)fa::num_sms() * C::CTAS * NW, used = std::max<long long>(1, warps / NKV) * NKV;
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
  return std::max(scratch_of<256, 8>(n), scratch_of<256, 16>(n));
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
  if (p.total == 0 || p.batch == 0) return FA_OK;
  if (p.total * p.NH >= 1ll << 31) {
    fa::set_error("8-bit decode: %lld rows of %d heads are more than one call takes", p.total, p.NH);
    return FA_ERR_SIZE;
  }
  FA_CHECK_ARG(p.scratch, "8-bit decode: scratch must be non-null");
  FA_CHECK_ARG(((uintptr_t)p.Kc | (uintptr_t)p.Vc | (uintptr_t)p.o | (uintptr_t)p.scratch) % 16 == 0,
               "8-bit decode: Kc, Vc, o and scratch must be 16-byte aligned");
  p.win_left = std::min(p.win_left, 1 << 30);   // position - win_left stays within 32 bits
  p.win_right = std::min(p.win_right, 1 << 30);
  cudaStream_t st = (cudaStream_t)stream;
  return p.code == FA_CODE_I8 ? by_dim<I8>(p, dtype, st) : by_dim<E4M3>(p, dtype, st);
}
