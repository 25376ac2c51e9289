// The residual's addition and a root-mean-square norm of each row into int8 codes with a scale of the row's own.
//
// With t_c = r_c w_c the norm's result is t_c / rms: one factor for the whole row, so code_c = round(127 t_c / max |t|) does not
// depend on it, and the scale is max |t| / rms. Both need only the row's sum of r^2 and its largest |t|, so a row is read once,
// held, and written once: what bounds the call is memory.
#include <algorithm>

#include "experts.h"

namespace anvil {

struct NormArgs {
  anvil_add_norm n;
  int nbits;                                             // bit length of lut_len
  unsigned* flags;
};

__device__ __forceinline__ long long load_any(const void* p, int dtype, long long i) {
  return dtype == ANVIL_I8 ? (long long)((const int8_t*)p)[i] : (long long)((const int16_t*)p)[i];
}

// r of one element
__device__ __forceinline__ int sum_of(const anvil_add_norm& n, long long row, int c, int lo, int hi) {
  const int x = (int)load_any(n.X, n.x_dtype, row * n.ldx + c);
  if (!n.Y) return x;
  const int y = (int)load_any(n.Y, n.y_dtype, row * n.ldy + c);
  const int v = (x * n.ma + y * n.mb + (int)round_term(n.shift)) >> n.shift;
  return min(max(v, lo), hi);
}

// sign(t) floor((254 |t| + a) / (2 a)) for |t| <= a: the quotient is at most 127, so a reciprocal in 32 bits is off by at most one,
// which the remainder shows
__device__ __forceinline__ int code_of(int t, unsigned a, float inv) {
  const unsigned num = 254u * (unsigned)abs(t) + a;      // below 2^31: |t| <= 2^22
  unsigned q = (unsigned)((float)num * inv);
  const int rem = (int)(num - q * 2 * a);
  q += rem < 0 ? -1 : (rem >= (int)(2 * a) ? 1 : 0);
  return t < 0 ? -(int)q : (int)q;
}

__device__ __forceinline__ int scale_of(const anvil_add_norm& n, unsigned a, unsigned long long ss, int nbits) {
  ss += (unsigned)n.eps;
  const int b = 64 - __builtin_clzll(ss | 1);            // the bit length of a sum that is not 0
  const int k0 = max(0, (b - nbits + 1) >> 1);
  const int k = k0 + ((ss >> (2 * k0)) >= (unsigned)n.lut_len ? 1 : 0);
  const long long v = (long long)a * max(0, n.lut[ss >> (2 * k)]);
  const int s = n.lut_shift + k;
  const long long r = (v + round_term(s)) >> s;
  return (int)min(r, 32767ll);
}

// One workgroup a row, any width, stride and alignment; the row is read twice.
__global__ __launch_bounds__(256) void add_norm_any(NormArgs g) {
  const anvil_add_norm& n = g.n;
  __shared__ unsigned long long sums[4];
  __shared__ unsigned tops[4];
  const int lo = n.r_dtype == ANVIL_I8 ? -128 : -32768, hi = -lo - 1;
  for (long long row = blockIdx.x; row < n.rows; row += gridDim.x) {
    unsigned long long ss = 0;
    unsigned a = 0;
    for (int c = threadIdx.x; c < n.cols; c += 256) {
      const int r = sum_of(n, row, c, lo, hi);
      ss += (unsigned)(r * r);
      a = max(a, (unsigned)abs(r * n.w[c]));
    }
    for (int o = 32; o; o >>= 1) {
      ss += __shfl_xor(ss, o);
      a = max(a, (unsigned)__shfl_xor((int)a, o));
    }
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = ss, tops[threadIdx.x >> 6] = a;
    __syncthreads();
    ss = sums[0] + sums[1] + sums[2] + sums[3];
    a = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    const float inv = a ? 1.0f / (2.0f * (float)a) : 0.0f;
    for (int c = threadIdx.x; c < n.cols; c += 256) {
      const int r = sum_of(n, row, c, lo, hi);
      if (n.Y) {
        if (n.r_dtype == ANVIL_I8) ((int8_t*)n.R)[row * n.ldr + c] = (int8_t)r;
        else ((int16_t*)n.R)[row * n.ldr + c] = (int16_t)r;
      }
      n.H[row * n.ldh + c] = a ? (int8_t)code_of(r * n.w[c], a, inv) : (int8_t)0;
    }
    if (threadIdx.x == 0) n.scale[row] = (int16_t)scale_of(n, a, ss, g.nbits);
    __syncthreads();
  }
}

}  // namespace anvil

using namespace anvil;

extern "C" int anvil_add_norm_i8(anvil_ctx* ctx, const anvil_add_norm* n) {
  const char* who = "anvil_add_norm_i8";
  if (!n) return set_error(ANVIL_E_VALUE, "%s: null arguments", who);
  if (n->rows < 0 || n->cols < 1 || n->cols > 65536)
    return set_error(ANVIL_E_VALUE, "%s: %d rows of %d", who, n->rows, n->cols);
  if (!narrow(n->x_dtype) || !narrow(n->r_dtype) || (n->Y && !narrow(n->y_dtype)))
    return set_error(ANVIL_E_VALUE, "%s: x, y and r must be i8 or i16", who);
  if ((n->Y != nullptr) != (n->R != nullptr) || (!n->Y && n->r_dtype != n->x_dtype))
    return set_error(ANVIL_E_VALUE, "%s: R goes with Y, and without them r is x", who);
  if (!stride_ok(n->ldx, n->cols) || !stride_ok(n->ldh, n->cols) || (n->Y && !(stride_ok(n->ldy, n->cols) && stride_ok(n->ldr, n->cols))))
    return set_error(ANVIL_E_VALUE, "%s: a row stride is not in [%d, 2^31)", who, n->cols);
  if (n->lut_len < 2 || n->lut_len > 65536 || n->eps < 0 || n->lut_shift < 0 || n->lut_shift > 31)
    return set_error(ANVIL_E_VALUE, "%s: table of %d, eps %d, lut_shift %d", who, n->lut_len, n->eps, n->lut_shift);
  if (n->Y) {
    if (n->shift < 0 || n->shift > 31) return set_error(ANVIL_E_VALUE, "%s: shift %d outside [0, 31]", who, n->shift);
    if (!sum_fits(n->x_dtype, n->ma, n->y_dtype, n->mb, n->shift))
      return set_error(ANVIL_E_OVERFLOW, "%s: x * %d + y * %d may leave int32", who, n->ma, n->mb);
  }
  if (!n->rows) return check_ctx(ctx);
  if (!n->X || !n->w || !n->lut || !n->H || !n->scale) return set_error(ANVIL_E_VALUE, "%s: null pointer", who);
  if ((uintptr_t)n->X % n->x_dtype || (n->Y && ((uintptr_t)n->Y % n->y_dtype || (uintptr_t)n->R % n->r_dtype)) ||
      (uintptr_t)n->lut % 4 || (uintptr_t)n->scale % 2)
    return set_error(ANVIL_E_VALUE, "%s: a pointer is not aligned to its type", who);
  const auto span = [&](const void* p, long long ld, int size) { return Span{p, n->rows, ld * size, (long long)n->cols * size}; };
  const Span x = span(n->X, n->ldx, n->x_dtype), y = span(n->Y, n->ldy, n->Y ? n->y_dtype : 1), w{n->w, 1, n->cols, n->cols},
             lut{n->lut, 1, 4ll * n->lut_len, 4ll * n->lut_len};
  const Span r = span(n->R, n->ldr, n->r_dtype), h = span(n->H, n->ldh, 1), scale{n->scale, 1, 2ll * n->rows, 2ll * n->rows};
  const bool on_x = n->R == n->X && n->r_dtype == n->x_dtype && n->ldr == n->ldx;
  const bool on_y = n->R && n->R == n->Y && n->r_dtype == n->y_dtype && n->ldr == n->ldy;
  const Span out[3] = {r, h, scale};
  for (int i = 0; i < 3; ++i) {
    bool ok = apart(out[i], w) && apart(out[i], lut) && (i == 0 && on_x ? true : apart(out[i], x)) &&
              (i == 0 && on_y ? true : apart(out[i], y));
    for (int j = 0; j < i; ++j) ok = ok && apart(out[i], out[j]);
    if (!ok) return set_error(ANVIL_E_VALUE, "%s: the results overlap each other or what is read", who);
  }
  if (int e = check_ctx(ctx)) return e;
  NormArgs g{*n, 32 - __builtin_clz((unsigned)n->lut_len), ctx->flags};
  ANVIL_LAUNCH(add_norm_any, dim3((unsigned)std::min(n->rows, 1 << 20)), dim3(256), 0, ctx->stream, g);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
