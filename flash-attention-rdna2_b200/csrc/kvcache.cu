// kvcache.cu — writing to and reading back from paged caches (fa_kv_append_launch,
// fa_kv_gather_launch of fable_attn.h): new K/V rows are rotated and stored behind each
// sequence's cached tokens, as they are or in 8 bits with a scale for each block of slots and
// head; ranges of the caches come back as packed rows.
#include <algorithm>
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

// one thread per (row, head, element): K and V
template <typename T, typename C, bool SCALED>
__global__ void __launch_bounds__(256) gather_kernel(const FaKvGatherParams p, const Pages pg) {
  const long long per = (long long)p.heads * p.dim, e = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (e >= p.total * per) return;
  const long long row = e / per;
  const int h = (int)(e % per / p.dim), d = (int)(e % p.dim);
  const RowMap rm{p.cu_k, 0, p.batch};
  const int z = rm.seq_of_row(row), i = (int)(row - rm.first(z)), pos = i + (p.starts ? p.starts[z] : 0);
  const bool mine = i >= 0 && i < rm.count(z);   // else a row of no sequence
  const long long blk = mine ? pg.of(z, pos) : -1;
  float k = 0.f, v = 0.f;
  if (blk >= 0) {
    const int in_page = pos & (p.page - 1);
    const long long at = ((blk * p.page + in_page) * p.heads + h) * p.dim + d;
    if constexpr (SCALED) {
      const long long sc = (blk * p.heads + h) * (p.page / p.block) + in_page / p.block;
      k = C::to_f(((const typename C::T*)p.Kc)[at]) * p.Ks[sc];
      v = C::to_f(((const typename C::T*)p.Vc)[at]) * p.Vs[sc];
    } else {
      k = Elem<C>::to_f(((const C*)p.Kc)[at]);
      v = Elem<C>::to_f(((const C*)p.Vc)[at]);
    }
  } else if (mine) {
    record(ERR_PAGE);
  }
  ((T*)p.k)[e] = Elem<T>::from_f(k);
  ((T*)p.v)[e] = Elem<T>::from_f(v);
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

template <typename T>
int append(const FaKvAppendParams& p, cudaStream_t st) {
  const Pages pg = pages_of(p);
  if (p.code == FA_CODE_I8 || p.code == FA_CODE_E4M3) {
    const long long slots = p.total / p.block + 2ll * p.batch, warps = slots * p.heads * 2;
    const unsigned grid = (unsigned)((warps + 3) / 4);
    if (p.code == FA_CODE_I8) append8_kernel<T, I8><<<grid, 128, 0, st>>>(p, pg, slots);
    else append8_kernel<T, E4M3><<<grid, 128, 0, st>>>(p, pg, slots);
  } else {
    const unsigned grid = (unsigned)((p.total * p.heads * 2 + 3) / 4);
    append_kernel<T, T><<<grid, 128, 0, st>>>(p, pg);
  }
  fa::count_launch();
  return fa::cuda_status(cudaGetLastError(), "kv append launch");
}

template <typename T>
int gather(const FaKvGatherParams& p, cudaStream_t st) {
  const Pages pg = pages_of(p);
  const unsigned grid = (unsigned)((p.total * p.heads * p.dim + 255) / 256);
  if (p.code == FA_CODE_I8) gather_kernel<T, I8, true><<<grid, 256, 0, st>>>(p, pg);
  else if (p.code == FA_CODE_E4M3) gather_kernel<T, E4M3, true><<<grid, 256, 0, st>>>(p, pg);
  else if (p.code == FA_DTYPE_F16) gather_kernel<T, __half, false><<<grid, 256, 0, st>>>(p, pg);
  else if (p.code == FA_DTYPE_BF16) gather_kernel<T, __nv_bfloat16, false><<<grid, 256, 0, st>>>(p, pg);
  else gather_kernel<T, float, false><<<grid, 256, 0, st>>>(p, pg);
  fa::count_launch();
  return fa::cuda_status(cudaGetLastError(), "kv gather launch");
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
