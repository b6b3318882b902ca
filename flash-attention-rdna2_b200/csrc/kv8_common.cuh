// kv8_common.cuh — shared by the kernels over paged 8-bit caches (kvcache.cu, decode8.cu): the
// codes' conversions, the bounds-checked page lookup, the sequence of a packed row.
#pragma once
#include <cuda_fp8.h>
#include "fa_common.cuh"

namespace fa_kv {

struct I8 {
  using T = signed char;
  static constexpr float QMAX = 127.f;
  static __device__ __forceinline__ float to_f(T c) { return (float)c; }
  // x within the code range up to rounding: the clamp only takes what rounding put past QMAX
  static __device__ __forceinline__ T from_f(float x) {
    const int c = __float2int_rn(x);
    return (T)(c > 127 ? 127 : c < -127 ? -127 : c);
  }
};
struct E4M3 {
  using T = __nv_fp8_storage_t;
  static constexpr float QMAX = 448.f;
  static __device__ __forceinline__ float to_f(T c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }
  static __device__ __forceinline__ T from_f(float x) { return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }
};

constexpr float MIN_SCALE = 7.888609052210118e-31f;   // 2^-100: 1 / scale stays finite for a block of zeros

// error bits of fa_device_error
constexpr int ERR_PAGE = 8192, ERR_ROTARY = 16384;

struct Pages {
  const int* table;
  int shift, max_blocks;   // page = 1 << shift
  long long num_blocks;
  // page of position pos of sequence z, or -1 where there is none
  __device__ __forceinline__ int of(int z, int pos) const {
    const int i = pos >> shift;
    if (pos < 0 || i >= max_blocks) return -1;
    const int b = __ldg(table + (long long)z * max_blocks + i);
    return b >= 0 && b < num_blocks ? b : -1;
  }
};

// Rows of sequence z in a packed layout: [first(z), first(z + 1)) of `cu`, or dense rows of
// `tokens` each.  With a group size g = 1 << gs, slot(z) = first(z) / g + 2 z gives every sequence
// enough slots for the aligned groups that its rows can touch wherever they start
// ((n - 1) / g + 2 at most), so a grid of total / g + 2 batch slots covers them with no host
// knowledge of the lengths.
struct RowMap {
  const int* cu;
  int tokens, batch;
  __device__ __forceinline__ long long first(int z) const { return cu ? (long long)__ldg(cu + z) : (long long)z * tokens; }
  // rows of sequence z, of those that lie in [0, total): the offsets come from the device, unchecked by the host
  __device__ __forceinline__ int count(int z, long long total) const {
    const long long a = first(z), n = cu ? __ldg(cu + z + 1) - a : tokens;
    return a < 0 ? 0 : (int)max(0ll, min(n, total - a));
  }
  __device__ __forceinline__ int seq_of_slot(long long slot, int gs) const {
    int lo = 0, hi = batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((first(mid) >> gs) + 2 * mid <= slot) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
  __device__ __forceinline__ int seq_of_row(long long row) const {
    int lo = 0, hi = batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first(mid) <= row) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
};

__host__ __device__ __forceinline__ int log2_of(int x) {   // of a power of two
#ifdef __CUDA_ARCH__
  return 31 - __clz(x);
#else
  return 31 - __builtin_clz((unsigned)x);
#endif
}

// n / d for 0 <= n < 2^31 / d, d known to the host: one multiplication
struct Div {
  unsigned d, m;
  Div() = default;
  explicit Div(int d_) : d((unsigned)d_), m((unsigned)((0x100000000ull + d_ - 1) / d_)) {}
  __device__ __forceinline__ int of(int n) const { return d == 1 ? n : (int)__umulhi((unsigned)n, m); }
};

}  // namespace fa_kv
