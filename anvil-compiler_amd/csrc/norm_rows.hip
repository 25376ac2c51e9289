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

// floor(u / d) of u < 2^31 for one d in [2, 2^23]: (u m) >> (31 + l) with 2^(l-1) < d <= 2^l and m = ceil(2^(31+l) / d), which lies in
// [2^31, 2^32) and is too large by less than d / 2^(31+l) of a unit in 2^-(31+l): below 2^31 that is less than 1 / d, so no quotient
// changes.
// m comes from single precision and remainders. d is exact there, the hardware's reciprocal off by at most 2^-23 of it and every other
// step by 2^-24; taken 2^-21 smaller, the first quotient is too small by at most 11 / 2^24 of itself, 2817 units and a fraction, and the second,
// of what remains, leaves less than 2 d.
struct Divider {
  unsigned m;
  int sh;                                                // of the product's upper word
  __device__ __forceinline__ explicit Divider(unsigned d) {
    const int l = 32 - __builtin_clz(d - 1);
    const float r = __builtin_amdgcn_rcpf((float)d) * (1.0f - 0x1p-21f);
    m = (unsigned)__builtin_ldexpf(r, 31 + l);
    const unsigned long long whole = 1ull << (31 + l);
    m += (unsigned)((float)(whole - (unsigned long long)m * d) * r);
    const unsigned left = (unsigned)(whole - (unsigned long long)m * d);
    m += (left > 0) + (left > d);
    sh = l - 1;
  }
};

typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

// R chunks of eight elements, raw: 16 bytes of i16, or 8 of i8 in a chunk's first half. All loads go out before the first is looked
// at (unpack), whatever the dtype, and chunks past the row (`off` is OOB there) are zeros.
template <int R, typename OFF>
__device__ __forceinline__ void load_chunks(v4i (&v)[R], __amdgpu_buffer_rsrc_t p, int dtype, OFF&& off) {
  if (dtype == ANVIL_I16) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(p, off(i), 0, 0));
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const v2u b = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(p, off(i), 0, 0));
      v[i] = v4i{(int)b[0], (int)b[1], 0, 0};
    }
  }
}

// raw chunks as pairs of int16
template <int R>
__device__ __forceinline__ void unpack(v4i (&v)[R], int dtype) {
  if (dtype == ANVIL_I16) return;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const unsigned b0 = (unsigned)v[i][0], b1 = (unsigned)v[i][1];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const unsigned b = q < 2 ? b0 : b1;
      const int lo = (int)(b << (24 - 16 * (q & 1))) >> 24, hi = (int)(b << (16 - 16 * (q & 1))) >> 24;
      v[i][q] = (int)__builtin_amdgcn_perm((unsigned)hi, (unsigned)lo, 0x05040100u);
    }
  }
}

// The types of X (and of R) and Y that a kernel is made for: Y 0 none, -1 as the call says.
template <int X, int Y>
struct NormTypes {
  static constexpr int x = X, y = Y;
};

// Rows of at most 8 L R columns, 16-byte aligned, in registers: L lanes a row (64 / L rows a wave, or the workgroup's 256), R chunks of
// eight elements a lane, and a lane has the same columns of every row it takes, so its weights stay in registers.
//
// What bounds it is memory: 6 bytes an element (an i16 stream and an i8 addend), some 22 instructions. 32768 x 768: 30.4 us, 4.97
// TB/s, a copy's rate (one workgroup a row, each row read twice: 149). 32 lanes of three chunks for 768 columns: 64 would leave a quarter of
// them idle in the second chunk, 16 hold six chunks each and leave room for few waves.
//
// Codes. floor((254 |t| + a) / 2a) with t's sign is floor((254 t + a - [t < 0]) / 2a); with 256 a added it is 128 larger and its
// numerator lies in [0, 511 a], below 2^31 (a <= 2^22), so one multiplication by the row's reciprocal (Divider) and a shift
// straight into the code's byte give it exactly.
//
// ANY: rows at any alignment and of any width from eight columns on. The last chunk is the row's last eight columns, of which those that the
// chunk before has count as zeros and are not stored. 32768 x 769: 41 us (a workgroup a row that reads it twice 167).
template <int L, int R, typename T, bool ANY>
__global__ __launch_bounds__(256) void add_norm_rows(NormArgs g) {
  const anvil_add_norm& n = g.n;
  constexpr bool WHOLE = L == 256;                       // a workgroup a row
  const int xt = T::x < 0 ? n.x_dtype : T::x, yt = T::y < 0 ? n.y_dtype : T::y, rt = T::x < 0 ? n.r_dtype : T::x;
  const bool added = T::y < 0 ? n.Y != nullptr : T::y > 0;
  constexpr int ROWS = WHOLE ? 1 : 64 / L;               // of a wave at a time
  __shared__ unsigned long long sums[2][4];
  __shared__ int tops[2][4];
  const int lane = threadIdx.x & 63, sub = threadIdx.x & (L - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int mine = WHOLE ? 0 : lane / L;                 // row of those
  const int chunks = (n.cols + 7) >> 3, over = ANY ? 8 * chunks - n.cols : 0;  // columns that the last two chunks share
  const int last = ANY ? (chunks - 1) / L : -1;          // its number with its lane
  const bool shares = ANY && over && sub == (chunks - 1) % L;
  const unsigned back = shares ? over : 0;
  const int lo = rt == ANVIL_I8 ? -128 : -32768, hi = -lo - 1;
  const int rnd = (int)round_term(n.shift), ma = n.ma, mb = n.mb, shift = n.shift;
  v2u w[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    w[i] = v2u{0, 0};
    if (sub + L * i < chunks) __builtin_memcpy(&w[i], __builtin_assume_aligned(n.w + 8 * (sub + L * i) - (i == last ? back : 0), ANY ? 1 : 8), 8);
  }
  v4i keep;                                              // of the last chunk's pairs
#pragma unroll
  for (int q = 0; q < 4; ++q) keep[q] = (back <= 2 * q ? 0xFFFF : 0) | (back <= 2 * q + 1 ? ~0xFFFF : 0);
  // a lane's first chunk from that of its wave's rows (the launch checks ROWS rows against 2^31); chunk i is i steps on
  const auto offset = [&](long long ld, int size) { return (unsigned)(mine * ld + 8 * sub) * (unsigned)size; };
  const unsigned ox = offset(n.ldx, xt), oy = added ? offset(n.ldy, yt) : 0, oz = added ? offset(n.ldr, rt) : 0,
                 oh = offset(n.ldh, 1);
  const long long group = WHOLE ? blockIdx.x : (long long)blockIdx.x * 4 + wave, groups = WHOLE ? gridDim.x : 4ll * gridDim.x;
  int turn = 0;                                          // a wave is at most one barrier ahead, so two sets of sums do
  for (long long first = group * ROWS; first < n.rows; first += groups * ROWS, turn ^= 1) {
    const long long row = first + mine;
    const bool live = row < n.rows;
    const int rows = (int)min((long long)ROWS, n.rows - first);
    const auto span = [&](const void* p, long long ld, int size) {
      return uniform_rsrc((const char*)p + first * ld * size, (int)((rows - 1) * ld + n.cols) * size);
    };
    const auto at = [&](unsigned o, int size) {
      return [=](int i) { return live && sub + L * i < chunks ? o + (8 * L * i - (ANY && i == last ? back : 0)) * size : OOB; };
    };
    const auto but = [&](unsigned o, int size) {         // the same without a chunk that shares columns
      const auto f = at(o, size);
      return [=](int i) { return ANY && i == last && shares ? OOB : f(i); };
    };
    v4i x[R], y[R];
    load_chunks(x, span(n.X, n.ldx, xt), xt, at(ox, xt));
    if (added) {
      load_chunks(y, span(n.Y, n.ldy, yt), yt, at(oy, yt));
      unpack(x, xt);
      unpack(y, yt);
#pragma unroll
      for (int i = 0; i < R; ++i)                        // past the row's end x, y and so r are 0
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int v0 = (__mul24((int)(short)x[i][q], ma) + __mul24((int)(short)y[i][q], mb) + rnd) >> shift;
          const int v1 = (__mul24(x[i][q] >> 16, ma) + __mul24(y[i][q] >> 16, mb) + rnd) >> shift;
          x[i][q] = (int)__builtin_amdgcn_perm((unsigned)med3i(v1, lo, hi), (unsigned)med3i(v0, lo, hi), 0x05040100u);
        }
      const __amdgpu_buffer_rsrc_t pr = span(n.R, n.ldr, rt);
      const auto off = but(oz, rt);
      if (rt == ANVIL_I16) {
#pragma unroll
        for (int i = 0; i < R; ++i) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, x[i]), pr, off(i), 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const v2u b = {__builtin_amdgcn_perm((unsigned)x[i][1], (unsigned)x[i][0], 0x06040200u),
                         __builtin_amdgcn_perm((unsigned)x[i][3], (unsigned)x[i][2], 0x06040200u)};
          __builtin_amdgcn_raw_buffer_store_b64(b, pr, off(i), 0, 0);
        }
      }
      if constexpr (ANY) {
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (i == last && shares && live) {
            char* const end = (char*)n.R + (row * n.ldr + n.cols) * rt;
            const v4u v = __builtin_bit_cast(v4u, x[i]);
            if (rt == ANVIL_I16) store_last<4>(end, v, 2 * (8 - over));
            else store_last<2>(end, v2u{__builtin_amdgcn_perm(v[1], v[0], 0x06040200u), __builtin_amdgcn_perm(v[3], v[2], 0x06040200u)}, 8 - over);
          }
      }
    } else {
      unpack(x, xt);
    }
    if constexpr (ANY) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (i == last) x[i] &= keep;
    }
    unsigned long long ss = 0;
    int top = 0, low = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned p = (unsigned)x[i][q];
        ss += (unsigned)square_half<0>(p) + (unsigned)square_half<1>(p);       // at most 2^31
        const unsigned wq = w[i][q >> 1];
        const int t0 = q & 1 ? mul_half_byte<0, 2>(p, wq) : mul_half_byte<0, 0>(p, wq);
        const int t1 = q & 1 ? mul_half_byte<1, 3>(p, wq) : mul_half_byte<1, 1>(p, wq);
        top = max(top, max(t0, t1));
        low = min(low, min(t0, t1));
      }
    }
    constexpr int W = WHOLE ? 64 : L;
    unsigned a = (unsigned)lane_group_max<W>(max(top, -low));
    const unsigned s0 = (unsigned)lane_group_sum<W>((int)(ss & 0xFFFFFF)), s1 = (unsigned)lane_group_sum<W>((int)(ss >> 24));
    ss = ((unsigned long long)s1 << 24) + s0;
    if constexpr (WHOLE) {
      if (lane == 0) sums[turn][wave] = ss, tops[turn][wave] = (int)a;
      __syncthreads();
      ss = sums[turn][0] + sums[turn][1] + sums[turn][2] + sums[turn][3];
      a = (unsigned)max(max(tops[turn][0], tops[turn][1]), max(tops[turn][2], tops[turn][3]));
    }
    // the products t again, rather than held since the sums: 8 R registers of a wave's budget
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(x[i][q]));
    const Divider div(2 * max(a, 1u));                   // a row of zeros: every code is 257 / 2 - 128
    const __amdgpu_buffer_rsrc_t ph = span(n.H, n.ldh, 1);
    const auto to = but(oh, 1);
    const int bias = 257 * (int)max(a, 1u);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      v2u h;
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        unsigned u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned p = (unsigned)x[i][2 * d + (e >> 1)];
          const int t = e == 0   ? mul_half_byte<0, 0>(p, w[i][d])
                        : e == 1 ? mul_half_byte<1, 1>(p, w[i][d])
                        : e == 2 ? mul_half_byte<0, 2>(p, w[i][d])
                                 : mul_half_byte<1, 3>(p, w[i][d]);
          u[e] = __umulhi((unsigned)(mad_i24v(t, 254, bias) + (t >> 31)), div.m);
        }
        h[d] = sra_pack4v((int)u[0], (int)u[1], (int)u[2], (int)u[3], div.sh) ^ 0x80808080u;
      }
      __builtin_amdgcn_raw_buffer_store_b64(h, ph, to(i), 0, 0);
      if constexpr (ANY) {
        if (i == last && shares && live) store_last<2>((char*)n.H + row * n.ldh + n.cols, h, 8 - over);
      }
    }
    if (live && sub == 0) n.scale[row] = (int16_t)scale_of(n, a, ss, g.nbits);
  }
}

// One workgroup a row, which is read twice: rows of fewer than 8 or more than 16384 columns, multipliers of more than 24 bits, rows far apart.
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
  // eight elements a load: 16 bytes of i16, 8 of i8; multipliers that a 24-bit product takes; four rows within 32-bit offsets
  const auto even = [&](const void* p, long long ld, int size) { return (uintptr_t)p % (8 * size) == 0 && ld % 8 == 0; };
  const auto m24 = [](int m) { return m >= -(1 << 23) && m < 1 << 23; };
  const auto near = [](long long ld) { return ld < 1 << 28; };
  const int chunks = (n->cols + 7) / 8;
  if (n->cols >= 8 && chunks <= 2048 && near(n->ldx) && near(n->ldh) && (!n->Y || (near(n->ldy) && near(n->ldr) && m24(n->ma) && m24(n->mb)))) {
    const bool aligned = n->cols % 8 == 0 && even(n->X, n->ldx, n->x_dtype) && even(n->H, n->ldh, 1) && even(n->w, 8, 1) &&
                         (!n->Y || (even(n->Y, n->ldy, n->y_dtype) && even(n->R, n->ldr, n->r_dtype)));
    const auto launch = [&](auto lanes, auto per, auto types, auto any) {
      constexpr int L = decltype(lanes)::value, R = decltype(per)::value;
      const int rows = 256 / L;                          // of a workgroup at a time
      ANVIL_LAUNCH((add_norm_rows<L, R, decltype(types), decltype(any)::value>), dim3((unsigned)std::min((n->rows + rows - 1) / rows, 64 * ctx->num_cu)), dim3(256), 0,
                   ctx->stream, g);
    };
    // Streams of one type, alone or with an int8 addend, have kernels of their own: 32768 rows of 768 (i16 and i8) 30.4 us, 32.4 with types
    // told apart at run time; 8192 of 4096 37.5 and 41.0 (40.0 with workgroups for eight a CU that walk over the rows).
    const auto go = [&](auto lanes, auto per) {
      const bool same = n->r_dtype == n->x_dtype;
      const std::false_type whole;
      if (!aligned) launch(lanes, per, NormTypes<-1, -1>{}, std::true_type{});
      else if (same && !n->Y && n->x_dtype == ANVIL_I16) launch(lanes, per, NormTypes<ANVIL_I16, 0>{}, whole);
      else if (same && n->Y && n->x_dtype == ANVIL_I16 && n->y_dtype == ANVIL_I8) launch(lanes, per, NormTypes<ANVIL_I16, ANVIL_I8>{}, whole);
      else if (same && n->Y && n->x_dtype == ANVIL_I8 && n->y_dtype == ANVIL_I8) launch(lanes, per, NormTypes<ANVIL_I8, ANVIL_I8>{}, whole);
      else launch(lanes, per, NormTypes<-1, -1>{}, whole);
    };
    using std::integral_constant;
    const integral_constant<int, 1> c1;
    const integral_constant<int, 2> c2;
    const integral_constant<int, 3> c3;
    const integral_constant<int, 4> c4;
    // Lanes a row, us of an i16 stream with an i8 addend. 16 / 32: 32768 rows of 256 10.7 / 11.6, of 512 22.5 / 20.8, of 768 32.7 / 30.5. 32 / 64: 32768
    // of 768 30.5 / 33.5, 8192 9.5 / 9.8, 2048 5.0 / 5.2. 64 / 256: 32768 of 1024 37.6 / 84.6, 8192 of 1536 15.9 / 23.8, 16384 of 2048 38.6 / 50.0, 8192
    // of 2560 28.9 / 28.3.
    if (chunks <= 32) {
      const integral_constant<int, 16> l;
      if (chunks <= 16) go(l, c1);
      else go(l, c2);
    } else if (chunks <= 96) {
      const integral_constant<int, 32> l;
      if (chunks <= 64) go(l, c2);
      else go(l, c3);
    } else if (chunks <= 256) {
      const integral_constant<int, 64> l;
      if (chunks <= 128) go(l, c2);
      else go(l, c4);
    } else {
      const integral_constant<int, 256> l;
      if (chunks <= 512) go(l, c2);
      else if (chunks <= 1024) go(l, c4);
      else go(l, integral_constant<int, 8>{});
    }
    ANVIL_LAUNCHED();
    return ANVIL_OK;
  }
  ANVIL_LAUNCH(add_norm_any, dim3((unsigned)std::min(n->rows, 1 << 20)), dim3(256), 0, ctx->stream, g);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
