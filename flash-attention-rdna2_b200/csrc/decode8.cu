// decode8.cu — attention of new tokens over a paged cache held in 8 bits (fa_decode8_launch of
// fable_attn.h).
//
// One warp per (new token, query head): it walks the keys that the row sees with an online
// softmax, every quantity in fp32.
#include "fa_launch.h"
#include "kv8_common.cuh"

namespace {

using namespace fa_kv;

__device__ int g_dec8_error = 0;
__device__ __forceinline__ void record(int bit) { atomicOr(&g_dec8_error, bit); }

template <typename T, typename Q>
__global__ void __launch_bounds__(128) dec8_kernel(const FaDec8Params p, const Pages pg) {
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  if (w >= p.total * p.NH) return;
  const int lane = threadIdx.x % 32, h = (int)(w % p.NH), kvh = h / p.gqa, NKV = p.NH / p.gqa;
  const long long row = w / p.NH;
  const RowMap rm{p.cu_q, p.tokens, p.batch};
  const int z = rm.seq_of_row(row), n = rm.count(z), t = (int)(row - rm.first(z)), L = p.ctx_len[z];
  const int pos = L - n + t;
  const bool mine = t >= 0 && t < n;   // else a row of no sequence
  int lo = p.leftpad ? max(p.leftpad[z], 0) : 0, hi = L;
  if (p.win_left >= 0) lo = max(lo, pos - p.win_left);
  if (p.win_right >= 0) hi = (int)min((long long)hi, (long long)pos + p.win_right + 1);
  if (!mine) hi = lo;
  float q[8], acc[8];
  const T* x = (const T*)p.q + row * p.q_row + h * p.q_head;
  int rp = -1;
  if (p.cos && lo < hi) {
    rp = p.rot_pos ? p.rot_pos[z] + t : pos;
    if (rp < 0 || rp >= p.rot_seqlen_ro) {
      record(ERR_ROTARY);
      rp = -1;
    }
  }
  const int half = p.rot_dim / 2;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    acc[i] = 0.f;
    q[i] = d < p.dim ? Elem<T>::to_f(x[d]) : 0.f;
    if (rp >= 0 && d < p.rot_dim) {
      const bool low = p.rot_interleaved ? !(d & 1) : d < half;
      const int j = p.rot_interleaved ? d / 2 : d % half;
      const float b = Elem<T>::to_f(x[p.rot_interleaved ? d ^ 1 : low ? d + half : d - half]);
      const float c = p.cos[(long long)rp * half + j], s = p.sin[(long long)rp * half + j];
      q[i] = low ? q[i] * c - b * s : q[i] * c + b * s;
    }
  }
  float m = -INFINITY, l = 0.f;
  for (int key = lo; key < hi; ++key) {
    const long long blk = pg.of(z, key);
    if (blk < 0) {
      record(ERR_PAGE);
      continue;
    }
    const int in_page = key & (p.page - 1);
    const long long at = ((blk * p.page + in_page) * NKV + kvh) * p.dim;
    const long long sc = (blk * NKV + kvh) * (p.page / p.block) + in_page / p.block;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.dim) s += q[i] * Q::to_f(((const typename Q::T*)p.Kc)[at + lane + 32 * i]);
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    s *= p.Ks[sc] * p.scale;
    if (p.softcap > 0.f) s = p.softcap * fa_tanh(s / p.softcap);
    if (p.alibi) s += p.alibi[h] * (float)(key - pos);
    const float mn = fmaxf(m, s), corr = m == -INFINITY ? 0.f : expf(m - mn), e = expf(s - mn), ev = e * p.Vs[sc];
    m = mn;
    l = l * corr + e;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.dim) acc[i] = acc[i] * corr + ev * Q::to_f(((const typename Q::T*)p.Vc)[at + lane + 32 * i]);
  }
  T* o = (T*)p.o + (row * p.NH + h) * p.dim;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < p.dim) o[lane + 32 * i] = Elem<T>::from_f(l == 0.f ? 0.f : acc[i] / l);
  if (p.lse && lane == 0)
    p.lse[p.cu_q ? h * p.total + row : ((long long)z * p.NH + h) * p.tokens + t] = l == 0.f ? -INFINITY : m + logf(l);
}

template <typename T>
int run(const FaDec8Params& p, cudaStream_t st) {
  const Pages pg{p.block_table, log2_of(p.page), p.max_blocks, p.num_blocks};
  const unsigned grid = (unsigned)((p.total * p.NH + 3) / 4);
  if (p.code == FA_CODE_I8) dec8_kernel<T, I8><<<grid, 128, 0, st>>>(p, pg);
  else dec8_kernel<T, E4M3><<<grid, 128, 0, st>>>(p, pg);
  fa::count_launch();
  return fa::cuda_status(cudaGetLastError(), "8-bit decode launch");
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
  (void)NH; (void)gqa; (void)dim;
  return 0;
}

extern "C" FA_API int fa_decode8_launch(const FaDec8Params* pp, int dtype, void* stream) {
  FA_ABI_GUARD(pp, FaDec8Params);
  const FaDec8Params& p = *pp;
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
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == FA_DTYPE_F16) return run<__half>(p, st);
  if (dtype == FA_DTYPE_BF16) return run<__nv_bfloat16>(p, st);
  return run<float>(p, st);
}
