// What the operators of an experts' feed-forward (norm_rows.hip, experts.hip, expert_gemm.hip) share: the requant in 64 bits and
// the checks of operands that may not overlap.
#pragma once

#include "common.h"

namespace anvil {

// clamp((acc * m + 2^(s-1)) >> s, lo, hi) with the product and the sum in 64 bits, left as a clamped int to be shifted right by `rest`.
// HI: s >= 33, where the sum's upper word alone is needed: one multiply-add of 32 x 32 + 64 bits, clamped before the last s - 32 bits go. A
// product's m / 2^s lies well below 1 / 4, so a smaller s is moved up to 33 where m has room (lift_shift). The lower word of 2^(s-1), zero
// there, comes from where the compiler does not see it: knowing it, it multiplies and adds in two instructions.
struct WideRequant {
  int s, rest, clo, chi, lo, hi;
  long long half;
  __device__ __forceinline__ WideRequant(int shift, int lo_, int hi_) : s(shift), rest(0), clo(lo_), chi(hi_), lo(lo_), hi(hi_), half(0) {
    if (s < 33) return;
    rest = s - 32;
    int zero = 0;
    asm("" : "+s"(zero));
    half = (long long)((unsigned long long)(1u << (rest - 1)) << 32 | (unsigned)zero);
    const long long a = (long long)lo << rest, b = (((long long)hi + 1) << rest) - 1;
    clo = a < I32_MIN ? (int)I32_MIN : (int)a;
    chi = b > I32_MAX ? (int)I32_MAX : (int)b;
  }
  __device__ __forceinline__ bool high() const { return s >= 33; }
  template <bool HI>
  __device__ __forceinline__ int unshifted(int acc, int m) const {
    if constexpr (HI) return med3i((int)(((long long)acc * m + half) >> 32), clo, chi);
    const long long r = ((long long)acc * m + (s ? 1ll << (s - 1) : 0)) >> s;
    return (int)(r < lo ? lo : r > hi ? hi : r);
  }
  template <bool HI>
  __device__ __forceinline__ int of(int acc, int m) const { return unshifted<HI>(acc, m) >> rest; }
};

// (m, s) with s moved up to 33 where m keeps within int32: the same products and roundings. From below 2 only m = 0 would keep, and the product
// here leaves 64 bits (-2^31 from 0).
__host__ __device__ inline void lift_shift(int& m, int& s) {
  if (s >= 33 || s < 2) return;
  const long long w = (long long)m * (1ll << (33 - s));
  if (w < I32_MIN || w > I32_MAX) return;
  m = (int)w;
  s = 33;
}

template <int L>
__device__ __forceinline__ int lane_group_max(int v) {       // maximum over aligned groups of L lanes
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));
  if constexpr (L > 16) v = max(v, __builtin_amdgcn_ds_swizzle(v, (16 << 10) | 0x1F));
  if constexpr (L > 32) v = max(v, __shfl_xor(v, 32));
  return v;
}

// sixteen bytes, at any alignment if ANY
template <bool ANY>
__device__ __forceinline__ v4i load16(const void* p) {
  if constexpr (!ANY) return *reinterpret_cast<const v4i*>(p);
  v4i v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// The last `bytes` of the 4 N bytes w that would end at `end` (fewer than all): a store for each bit of their number, the largest the
// last in memory. What is left after each lies in one half of the words before.
template <int N>
struct Words {                                           // a vector: an array chosen from at run time would go to memory
  typedef unsigned type __attribute__((ext_vector_type(N)));
  typedef type any __attribute__((aligned(1)));
};
template <int N>
__device__ __forceinline__ void store_last(char* end, typename Words<N>::type w, int bytes) {
  if constexpr (N > 1) {
    const bool upper = bytes & 2 * N;
    typename Words<N / 2>::type left, high;
#pragma unroll
    for (int q = 0; q < N / 2; ++q) left[q] = upper ? w[q] : w[N / 2 + q], high[q] = w[N / 2 + q];
    if (upper) {
      end -= 2 * N;
      *reinterpret_cast<typename Words<N / 2>::any*>(end) = high;
    }
    store_last<N / 2>(end, left, bytes);
  } else {
    unsigned v = w[0];
    if (bytes & 2) {
      end -= 2;
      const unsigned short u = (unsigned short)(v >> 16);
      __builtin_memcpy(end, &u, 2);
      v <<= 16;
    }
    if (bytes & 1) end[-1] = (char)(v >> 24);
  }
}

// Memory of `rows` rows of `width` bytes, `ld` bytes apart.
struct Span {
  const void* p;
  long long rows, ld, width;
};
// No byte of both: apart as ranges, or rows of equal stride between each other's.
inline bool apart(const Span& a, const Span& b) {
  if (!a.p || !b.p || !a.rows || !b.rows || !a.width || !b.width) return true;
  const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
  const uintptr_t a1 = a0 + (a.rows - 1) * a.ld + a.width, b1 = b0 + (b.rows - 1) * b.ld + b.width;
  if (a1 <= b0 || b1 <= a0) return true;
  if (a.ld != b.ld || a.rows < 2 || b.rows < 2) return false;
  const long long d = (long long)((b0 >= a0 ? b0 - a0 : (uintptr_t)a.ld - (a0 - b0) % (uintptr_t)a.ld) % (uintptr_t)a.ld);
  return d >= a.width && d + b.width <= a.ld;
}

// a row stride of at least `width` that keeps every byte offset within 64 bits
inline bool stride_ok(long long ld, int width) { return ld >= width && ld <= INT32_MAX; }

inline bool narrow(int dtype) { return dtype == ANVIL_I8 || dtype == ANVIL_I16; }

// |a| * |ma| + |b| * |mb| + 2^(s-1) for every a and b of their dtypes is an int32
inline bool sum_fits(int a_dtype, long long ma, int b_dtype, long long mb, int s) {
  const long long a = -(long long)dtype_lo(a_dtype), b = -(long long)dtype_lo(b_dtype);
  return a * (ma < 0 ? -ma : ma) + b * (mb < 0 ? -mb : mb) + (s ? 1ll << (s - 1) : 0) <= I32_MAX;
}

}  // namespace anvil
