// What the operators of an experts' feed-forward (norm_rows.hip, experts.hip, expert_gemm.hip) share: the requant in 64 bits and
// the checks of operands that may not overlap.
#pragma once

#include "common.h"

namespace anvil {

// clamp((acc * m + 2^(s-1)) >> s, lo, hi) with the product and the sum in 64 bits. HI: s >= 32, so that all of the result is in
// the sum's upper word, which is clamped before its shift by s - 32: one 32 x 32 -> 64-bit multiply-add, a clamp and a shift.
// A product's multiplier is m / 2^s below 1 / 2, so the host and the kernels move a smaller s up to 32 where m has room.
struct Requant {
  long long rnd;
  int s, lo, hi;
  __device__ Requant(int shift, int lo_, int hi_) : rnd(shift ? 1ll << (shift - 1) : 0), s(shift), lo(lo_), hi(hi_) {}
  template <bool HI>
  __device__ __forceinline__ int of(int acc, int m) const {
    const long long v = (long long)acc * m + rnd;
    if constexpr (HI) return min(max((int)(v >> 32) >> (s - 32), lo), hi);
    const long long r = v >> s;
    return (int)(r < lo ? lo : r > hi ? hi : r);
  }
};

// (m, s) with s moved up to 32 where m keeps within int32: the same products and roundings
__host__ __device__ inline void lift_shift(int& m, int& s) {
  if (s >= 32) return;
  const long long w = (long long)m * (1ll << (32 - s));
  if (w < I32_MIN || w > I32_MAX) return;
  m = (int)w;
  s = 32;
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
