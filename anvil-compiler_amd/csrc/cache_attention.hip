// Attention of the newest tokens over the 4-bit paged cache.
//
// Mathematics. softmax_lut's exponentials are table entries at x - max, so a maximum found later cannot rescale a sum that was
// begun; but a score is one of 256 values, and with the histogram of a row's scores its maximum, its sum and the probability of each
// value follow exactly. So a row is evaluated in two passes: its scores (one byte a key, kept) with their histogram, then a
// 256-entry table of probabilities and the sum of p V, looked up by score. K is read once, V once.
//
// Tiles. Up to 16 rows share a pass over a cache head's keys: the query heads of its group, for one token or several. 64 keys (a
// page) are one step of a wave:
//   scores  keys x channels codes (their four bits in a byte's upper half, so that no sign has to be extended: 16 x the product)
//           times channels x columns queries, 16 keys a product; each group of 32 channels times the key's step of that group
//   values  channels x keys codes times keys x columns of p x step, whose 12 to 20 bits go through as 7-bit digits
// A product has 16 columns. With RP = 4 or 8 row slots the 16 / RP columns of a row are put to use: for the scores each takes
// groups of its own (zeros elsewhere), which are summed across them after the steps; for the values each takes a digit. So the
// instructions around the products, which are what bounds the kernel, are shared out over the lanes.
// The operand rows are ordered so that the lanes of (row, q) receive the scores of keys 16 q .. 16 q + 15 in order, which are the keys
// whose p they supply to the second product: a wave reads back what it wrote.
#include <algorithm>

#include "cache.h"

namespace anvil {

struct AttendArgs {
  const int8_t* q;
  int8_t* o;
  long long q_row, q_head, o_row, o_head;
  const int* lut;
  int m_s, s_s, one, m_o, s_o, window, sinks;
  int group, rows;                                       // query heads of a cache head; rows of a tile that can exist
  int seq0, tile0, tiles, splits, bound;                 // this launch's part; pages that a tile can see at most
  uint8_t* scores;                                       // workspace: [unit][tile][page][row][64], a score + 128; or widened
                                                         //            pages, [unit][page]
  unsigned* hist;                                        //            [unit][tile][split][row][256]
  int* sums;                                             //            [unit][tile][split][row][32 NG], 16 x sum p V
};

constexpr int HIST = 257;                                // dwords of a row's histogram in LDS: rows start in different banks

constexpr int ONE_NARROW = ((1 << 14) - 1) / STEP_MAX;   // 910: p x step is two 7-bit digits
constexpr int ONE_FIFTEEN = 7 * (1 + 15 + 225 + 3375);   // 25312: four digits of base 15

typedef unsigned short __attribute__((may_alias)) u16_alias;

// What a workgroup evaluates: the rows of one tile, and the pages that some row of it may see, numbered from 0 (first those of the
// sinks, then from the window's first page on).
struct Tile {
  NewRows r;
  int seq, head, unit, tile, first, rows, lo, hi;        // its first row, rows in use; positions of its first and last token
  int sink_pages, window_page, pages;
};

template <int ROWS = 16>
__device__ __forceinline__ bool find_tile(const CacheView& c, const AttendArgs& a, Tile& t) {
  t.unit = blockIdx.x, t.tile = (int)blockIdx.y;
  t.seq = a.seq0 + t.unit / c.heads, t.head = t.unit % c.heads;
  const int first = t.first = (a.tile0 + t.tile) * ROWS;
  new_rows(c, t.seq, t.r, first == 0 && blockIdx.z == 0 && t.head == 0 && threadIdx.x == 0);
  t.r.first = __builtin_amdgcn_readfirstlane(t.r.first), t.r.n = __builtin_amdgcn_readfirstlane(t.r.n);   // the same in every lane
  t.r.len = __builtin_amdgcn_readfirstlane(t.r.len);
  const long long all = (long long)t.r.n * a.group;
  if (first >= all) return false;
  t.rows = (int)min((long long)ROWS, all - first);
  t.lo = t.r.len - t.r.n + first / a.group;
  t.hi = t.r.len - t.r.n + (first + t.rows - 1) / a.group;
  t.window_page = a.window && t.lo >= a.window ? (t.lo - a.window + 1) >> PAGE_SHIFT : 0;
  t.sink_pages = min((a.sinks + PAGE - 1) >> PAGE_SHIFT, t.window_page);
  t.pages = t.sink_pages + (t.hi >> PAGE_SHIFT) - t.window_page + 1;
  return true;
}

__device__ __forceinline__ int slot_of(const Tile& t, int page) {
  return page < t.sink_pages ? page : t.window_page + page - t.sink_pages;
}

// The table's entry of a page, -1 where it names none. An entry out of range is reported.
__device__ __forceinline__ int entry_of(const CacheView& c, const Tile& t, int page, int end) {
  int entry = -1;
  if (page < end) entry = c.table[(long long)t.seq * c.slots + slot_of(t, page)];
  if (entry >= c.pages || entry < -1) {
    raise_flag(c.flags, FLAG_CACHE);
    entry = -1;
  }
  return entry;
}

// whether every row of the tile sees every key of a page
__device__ __forceinline__ bool whole(const Tile& t, const AttendArgs& a, int slot) {
  const int first = slot * PAGE, last = first + PAGE - 1;
  return last <= t.lo && (!a.window || first > t.hi - a.window || last < a.sinks);
}

// One row of the tile as its lanes know it.
struct Row {
  int pos, after, sinks;                                 // sees keys <= pos that are > after or < sinks
  bool on;
  __device__ __forceinline__ Row(const Tile& t, const AttendArgs& a, int r) {
    on = r < t.rows;
    pos = t.r.len - t.r.n + (t.first + r) / a.group;
    after = a.window ? pos - a.window : -1;
    sinks = a.sinks;
  }
  // bits of the 16 keys from `key` on that the row sees
  __device__ __forceinline__ unsigned mask(int key) const {
    const auto below = [](int n) { return n <= 0 ? 0u : (n >= 16 ? 0xFFFFu : (1u << n) - 1u); };   // keys before key + n
    return below(pos + 1 - key) & (~below(after + 1 - key) | below(sinks - key));
  }
};

template <int N>
struct Words {
  unsigned w[N];
};
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
template <int N>
__device__ __forceinline__ Words<N> load_words(__amdgpu_buffer_rsrc_t blk, int at) {
  Words<N> r;
  if constexpr (N == 1) {
    r.w[0] = __builtin_amdgcn_raw_buffer_load_b32(blk, at, 0, 0);
  } else if constexpr (N == 2) {
    const u2 v = __builtin_bit_cast(u2, __builtin_amdgcn_raw_buffer_load_b64(blk, at, 0, 0));
    r.w[0] = v.x, r.w[1] = v.y;
  } else {
    const u4 v = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(blk, at, 0, 0));
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  }
  return r;
}

// How a product's 16 columns are shared out: VN columns a row, of which GV hold different groups (NA groups each).
template <int NG, int RP>
struct Columns {
  static constexpr int VN = 16 / RP, GV = VN < NG ? VN : NG, NA = NG / GV, NE = 4 / VN;
};

// A lane's part of a page's keys: of 16 keys in each of four products the four bits of 8 channels a group, and the steps (of the
// lane's groups) of the 16 keys whose sums it receives.
template <int NG, int RP>
struct KeyPage {
  using C = Columns<NG, RP>;
  Words<NG> code[4];
  Words<C::NA> step[4];                                  // [i]: keys 16 q + 4 i .. + 3
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t blk, int lane) {
    const int row = lane & 15, q = lane >> 4;
    const int codes = key_of(row, 0) * Block<NG>::ROW + 4 * q * NG, steps = Block<NG>::K_STEPS + 16 * q * NG + 4 * (row % C::GV);
#pragma unroll
    for (int k = 0; k < 4; ++k) code[k] = load_words<NG>(blk, codes + k * key_of(0, 1) * Block<NG>::ROW);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (C::GV == 1) {
        step[e] = load_words<C::NA>(blk, steps + 4 * NG * e);
      } else {
#pragma unroll
        for (int n = 0; n < C::NA; ++n) step[e].w[n] = load_words<1>(blk, steps + 4 * NG * e + 4 * C::GV * n).w[0];
      }
    }
  }
  // the key of operand row `row` in product k. Sum e of product k (operand row 4 q + e) is that of key 16 q + 4 e + k, so that a lane
  // that keeps one e has four keys in a row; with a column a row, which keeps all, 16 q + 4 k + e: whole cache lines a load.
  static __device__ __forceinline__ int key_of(int row, int k) { return C::VN > 1 ? 4 * row + k : 16 * (row >> 2) + 4 * k + (row & 3); }
  __device__ __forceinline__ int step_of(int n, int e, int k) const {
    return (int)(C::VN > 1 ? (step[e].w[n] >> (8 * k)) & 255u : (step[k].w[n] >> (8 * e)) & 255u);
  }
};

// A lane's part of a page's values: 16 keys of two channels a group, and their steps.
template <int NG>
struct ValuePage {
  Words<4> code[NG], step[NG];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t blk, int lane) {
    const int row = lane & 15, q = lane >> 4;
    const int codes = Block<NG>::V + row * PAGE + 16 * q, steps = Block<NG>::V_STEPS + 16 * q;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      code[g] = load_words<4>(blk, codes + 16 * PAGE * g);
      step[g] = load_words<4>(blk, steps + PAGE * g);
    }
  }
};

// clamp((acc * m + rnd) >> s) of scores: |acc| below 2^22 (128 x 126 x 128 channels) and the product with the rounding inside int32
// by the caller's check, so 24-bit multiply-adds and a clamp before the shift are exact.
struct Requant {
  int m, s, rnd, lo, hi;
  __device__ Requant(int mult, int shift) : m(mult), s(shift), rnd(shift ? 1 << (shift - 1) : 0) {
    lo = (int)max(-128ll << shift, (long long)INT32_MIN);
    hi = (int)min((128ll << shift) - 1, (long long)INT32_MAX);
  }
};

// The query operand: the lane's column holds row column / VN; lane quarter q channels 8 q .. 8 q + 7 of each group that is the
// column's, zeros for the others (one group a product with VN = 1, two otherwise).
template <int NG, int RP>
struct Query {
  long w[NG];
  __device__ __forceinline__ void load(const CacheView& c, const AttendArgs& a, const Tile& t, int lane, int first = 0) {
    using C = Columns<NG, RP>;
    const int col = lane & 15, row = first + col / C::VN, r = t.first + row, ch = 8 * (lane >> 4);
    const int8_t* p = a.q + (long long)(t.r.first + r / a.group) * a.q_row + (long long)(t.head * a.group + r % a.group) * a.q_head + ch;
#pragma unroll
    for (int g = 0; g < NG; ++g)
      w[g] = row < t.rows && 32 * g + ch < c.dim && (C::GV == 1 || col % C::GV == g % C::GV) ? *(const long*)(p + 32 * g) : 0;
  }
};

// v of lane ^ 1 or lane ^ 2
template <int X>
__device__ __forceinline__ int lane_xor(int v) {
  return __builtin_amdgcn_update_dpp(0, v, X == 1 ? 0xB1 : 0x4E, 0xF, 0xF, false);
}

// The lane's scores of a page, a byte each, + 128: dword i holds keys 16 q + 4 e + 0..3 with e = NE v + i, v the lane's column of its
// row. The products hold 16 x code: their sum is divided exactly.
template <int NG, int RP>
__device__ __forceinline__ Words<Columns<NG, RP>::NE> score_page(const KeyPage<NG, RP>& k, const Query<NG, RP>& q, const Requant& rq) {
  using C = Columns<NG, RP>;
  const int v = threadIdx.x % C::VN;
  int x[C::NE][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v4i d[C::NA];
    if constexpr (NG == 1 || C::VN == 1) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const unsigned long low = (k.code[i].w[g] << 4) & 0xF0F0F0F0u, high = k.code[i].w[g] & 0xF0F0F0F0u;
        d[g] = __builtin_amdgcn_mfma_i32_16x16x32_i8((long)(high << 32 | low), q.w[g], v4i{0, 0, 0, 0}, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int g = 0; g < NG; g += 2) {
        const unsigned w0 = k.code[i].w[g], w1 = k.code[i].w[g + 1];
        const v4i keys = {(int)((w0 << 4) & 0xF0F0F0F0u), (int)(w0 & 0xF0F0F0F0u), (int)((w1 << 4) & 0xF0F0F0F0u), (int)(w1 & 0xF0F0F0F0u)};
        const v4i rows = {(int)q.w[g], (int)(q.w[g] >> 32), (int)q.w[g + 1], (int)(q.w[g + 1] >> 32)};
        const bool again = C::GV == 4 && g > 0;          // four columns of a group each: one sum for both products
        d[g / C::GV] = __builtin_amdgcn_mfma_i32_16x16x64_i8(keys, rows, again ? d[0] : v4i{0, 0, 0, 0}, 0, 0, 0);
      }
    }
    int acc[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[e] = 0;
#pragma unroll
      for (int n = 0; n < C::NA; ++n) acc[e] += __mul24(d[n][e], k.step_of(n, e, i));
    }
    // the sum over the row's columns; each keeps its NE of the four keys
    if constexpr (C::VN == 4) {
      int a0, a1;
      if constexpr (C::GV == 4) {
        a0 = (v & 2 ? acc[2] : acc[0]) + lane_xor<2>(v & 2 ? acc[0] : acc[2]);
        a1 = (v & 2 ? acc[3] : acc[1]) + lane_xor<2>(v & 2 ? acc[1] : acc[3]);
      } else {
        a0 = v & 2 ? acc[2] : acc[0];
        a1 = v & 2 ? acc[3] : acc[1];
      }
      acc[0] = C::GV == 1 ? (v & 1 ? a1 : a0) : (v & 1 ? a1 : a0) + lane_xor<1>(v & 1 ? a0 : a1);
    } else if constexpr (C::VN == 2) {
      const int a0 = v ? acc[2] : acc[0], a1 = v ? acc[3] : acc[1];
      if constexpr (C::GV == 2) {
        const int b0 = v ? acc[0] : acc[2], b1 = v ? acc[1] : acc[3];
        acc[0] = a0 + lane_xor<1>(b0), acc[1] = a1 + lane_xor<1>(b1);
      } else {
        acc[0] = a0, acc[1] = a1;
      }
    }
#pragma unroll
    for (int n = 0; n < C::NE; ++n) {
      const int v = med3i(__mul24(acc[n] >> 4, rq.m) + rq.rnd, rq.lo, rq.hi);
      if constexpr (C::VN > 1) x[n][i] = v;
      else x[i][n] = v;
    }
  }
  Words<C::NE> out;
#pragma unroll
  for (int n = 0; n < C::NE; ++n) out.w[n] = sra_pack4(x[n][0], x[n][1], x[n][2], x[n][3], rq.s) ^ 0x80808080u;
  return out;
}

__device__ __forceinline__ unsigned word(const uint4& v, int i) { return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)); }

// The scores of a page into the row's histogram: all of them, or with a mask, a bit a key.
template <int N>
__device__ __forceinline__ void count_scores(unsigned* hist, const Words<N>& sc) {
#pragma unroll
  for (int i = 0; i < 4 * N; ++i) atomicAdd(&hist[(sc.w[i >> 2] >> (8 * (i & 3))) & 255u], 1u);
}
template <int N>
__device__ __forceinline__ void count_scores(unsigned* hist, const Words<N>& sc, unsigned mask) {
#pragma unroll
  for (int i = 0; i < 4 * N; ++i)
    if (mask >> i & 1u) atomicAdd(&hist[(sc.w[i >> 2] >> (8 * (i & 3))) & 255u], 1u);
}

// Digits. With four columns a row, p as four digits of base 15 from -7 to 7 (p <= 25312), a column and a table of bytes each: a digit
// times a step (at most 18) is an int8 as it stands. Else a table entry is 2 p, or 2 (p & 127) and 2 (p >> 7) in two tables (WIDE).
// Its product with a step is below 2^15 (p <= 910, 127 or 255), so two keys are one 16-bit packed product, whose low byte halved is
// the low 7-bit digit of p x step (bit 0 is 0) and whose high byte the high one.
//   RP  4        columns: digits of base 15
//   RP  8        columns: low and high digit of p x step
//   RP  8 WIDE   columns: p & 127, p >> 7; a product each for the low and the high digit
//   RP 16        a product each for the low and the high digit of p x step
//   RP 16 WIDE   products for both digits of p & 127 and of p >> 7, the middle two into one sum
enum { TABLE_P = 1, TABLE_SEVEN = 2, TABLE_FIFTEEN = 4, TABLE_BYTES = 5, TABLE_PAIRS = 6 };
template <int RP, bool WIDE>
struct Digits {
  static constexpr int TABLE = RP == 4 ? TABLE_FIFTEEN : (RP == 8 && WIDE ? TABLE_SEVEN : TABLE_P);   // RP 16 takes 2 p apart itself
  static constexpr int SUMS = RP == 16 ? (WIDE ? 3 : 2) : (RP == 8 && WIDE ? 2 : 1);
  // the weight of a column's sum n
  static __device__ __forceinline__ unsigned weight(int v, int n) {
    if constexpr (RP == 4) return v == 0 ? 1u : (v == 1 ? 15u : (v == 2 ? 225u : 3375u));
    else if constexpr (RP == 8 && !WIDE) return 1u << (7 * v);
    else if constexpr (RP == 8) return 1u << (7 * (v + n));
    else return 1u << (7 * n);
  }
};
// byte B of d = a x byte B of st
template <int B>
__device__ __forceinline__ void mul_to_byte(unsigned& d, int a, unsigned st) {
  if constexpr (B == 0)
    asm("v_mul_i32_i24_sdwa %0, %1, %2 dst_sel:BYTE_0 dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0"
        : "=v"(d) : "v"(a), "v"(st));
  else if constexpr (B == 1)
    asm("v_mul_i32_i24_sdwa %0, %1, %2 dst_sel:BYTE_1 dst_unused:UNUSED_PRESERVE src0_sel:DWORD src1_sel:BYTE_1"
        : "+v"(d) : "v"(a), "v"(st));
  else if constexpr (B == 2)
    asm("v_mul_i32_i24_sdwa %0, %1, %2 dst_sel:BYTE_2 dst_unused:UNUSED_PRESERVE src0_sel:DWORD src1_sel:BYTE_2"
        : "+v"(d) : "v"(a), "v"(st));
  else
    asm("v_mul_i32_i24_sdwa %0, %1, %2 dst_sel:BYTE_3 dst_unused:UNUSED_PRESERVE src0_sel:DWORD src1_sel:BYTE_3"
        : "+v"(d) : "v"(a), "v"(st));
}
typedef unsigned short v2u __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned mul_pair(unsigned a, unsigned b) {
  return __builtin_bit_cast(unsigned, (v2u)(__builtin_bit_cast(v2u, a) * __builtin_bit_cast(v2u, b)));
}

// acc += digits of p x step times 16 x code over a page, for the 16 keys of the lane's quarter: sc their scores, a bit of mask a key
// (`all`: every key, for every lane).
template <int NG, int RP, bool WIDE>
__device__ __forceinline__ void add_page(const ValuePage<NG>& v, const uint4& sc, const uint8_t* table, bool all, unsigned mask,
                                         v4i (&acc)[Digits<RP, WIDE>::SUMS][2 * NG]) {
  int one[RP == 4 ? 16 : 1];                             // a key's digit
  unsigned p[8];                                         // or the table entries of two keys each
  if constexpr (RP == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) one[i] = (int8_t)table[(word(sc, i >> 2) >> (8 * (i & 3))) & 255u];
    if (!all) {
#pragma unroll
      for (int i = 0; i < 16; ++i) one[i] = mask >> i & 1u ? one[i] : 0;
    }
  } else {
    const u16_alias* t = (const u16_alias*)table;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned w = word(sc, j >> 1) >> (16 * (j & 1));
      p[j] = t[w & 255u] | (unsigned)t[(w >> 8) & 255u] << 16;
    }
    if (!all) {
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] &= (mask >> (2 * j) & 1u ? 0xFFFFu : 0u) | (mask >> (2 * j + 1) & 1u ? 0xFFFF0000u : 0u);
    }
  }
  constexpr unsigned LOW = 0x06040200u, HIGH = 0x07050301u;
  const bool high = threadIdx.x % (16 / RP);             // RP 8: the digit of the lane's column
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    constexpr int ND = RP == 4 || (RP == 8 && !WIDE) ? 1 : (RP == 16 && WIDE ? 4 : 2);
    v4i digit[ND];
    if constexpr (RP == 4) {
      unsigned d[4];                                     // byte by byte: a byte's write and the next one's are four apart
      static_for<4>([&](auto b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) mul_to_byte<b>(d[i], one[4 * i + b], v.step[g].w[i]);
      });
      // a matrix instruction reads a vector register two wait states after its write at the earliest; the compiler sees to that, but
      // not behind inline assembly
      asm("s_nop 1" : "+v"(d[0]), "+v"(d[1]), "+v"(d[2]), "+v"(d[3]));
      digit[0] = {(int)d[0], (int)d[1], (int)d[2], (int)d[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned st = v.step[g].w[i];
        const unsigned s0 = __builtin_amdgcn_perm(0, st, 0x0c010c00u), s1 = __builtin_amdgcn_perm(0, st, 0x0c030c02u);
        if constexpr (ND == 4) {
          const unsigned y0 = mul_pair(p[2 * i] & 0x00FE00FEu, s0), y1 = mul_pair(p[2 * i + 1] & 0x00FE00FEu, s1);
          const unsigned z0 = mul_pair((p[2 * i] >> 7) & 0x01FE01FEu, s0), z1 = mul_pair((p[2 * i + 1] >> 7) & 0x01FE01FEu, s1);
          digit[0][i] = (int)(__builtin_amdgcn_perm(y1, y0, LOW) >> 1);
          digit[1][i] = (int)__builtin_amdgcn_perm(y1, y0, HIGH);
          digit[2][i] = (int)(__builtin_amdgcn_perm(z1, z0, LOW) >> 1);
          digit[ND - 1][i] = (int)__builtin_amdgcn_perm(z1, z0, HIGH);
        } else {
          const unsigned y0 = mul_pair(p[2 * i], s0), y1 = mul_pair(p[2 * i + 1], s1);
          if constexpr (ND == 1) {
            digit[0][i] = (int)(__builtin_amdgcn_perm(y1, y0, high ? HIGH : LOW) >> (high ? 0 : 1));
          } else {
            digit[0][i] = (int)(__builtin_amdgcn_perm(y1, y0, LOW) >> 1);
            digit[ND - 1][i] = (int)__builtin_amdgcn_perm(y1, y0, HIGH);
          }
        }
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      v4i code;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned w = v.code[g].w[i];
        code[i] = (int)((half ? w : w << 4) & 0xF0F0F0F0u);
      }
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        const int sum = ND == 4 && n > 1 ? n - 1 : n;
        acc[sum][2 * g + half] = __builtin_amdgcn_mfma_i32_16x16x64_i8(code, digit[n], acc[sum][2 * g + half], 0, 0, 0);
      }
    }
  }
}

// A wave's pages of a tile, begin + wave, begin + wave + waves, .. below end, one after the other, AHEAD of them in flight. One is
// enough: with two or three, whose steps are unrolled for as many sets of registers, the longer code costs a short walk more (its
// instructions come from memory too) than the loads in flight bring a long one. 32 x 12 heads over up to 1024 tokens: none
// 11.9 us, one 11.6, three and two 12.9; 64 x 32 heads over up to 8192: 79.0, 69.7, 70.1. Table entries come 64 at a time, one a lane;
// the first of them are known when the walk begins (`entry`).
template <int NG, int AHEAD, typename Page>
struct Walk {
  Page ring[AHEAD + 1];
  const CacheView& c;
  const Tile& t;
  const int first, end, waves, lane;
  int entry, n;

  __device__ __forceinline__ Walk(const CacheView& view, const Tile& tile, int begin, int stop, int entries)
      : c(view), t(tile), first(begin + (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), end(stop), waves(blockDim.x >> 6),
        lane(threadIdx.x & 63), entry(entries) {
    n = min(64, (end - first + waves - 1) / waves);
    static_for<AHEAD>([&](auto d) { fetch(d, ring[d]); });
  }
  // behind the last page, and where the table names none, an empty descriptor: the loads are issued, so that every step waits for
  // the same number of them, and touch no memory
  __device__ __forceinline__ void fetch(int i, Page& p) {
    const int e = i < n ? __builtin_amdgcn_readlane(entry, i & 63) : -1;
    const uint8_t* blk = c.pool + ((long long)max(e, 0) * c.heads + t.head) * Block<NG>::BYTES;
    p.load(uniform_rsrc(blk, e < 0 ? 0 : Block<NG>::BYTES), lane);
  }
  // step(page's lane part, page) for those that the table names
  template <typename Step>
  __device__ __forceinline__ void run(Step&& step) {
    for (int at = first; at < end; at += 64 * waves) {
      if (at != first) {
        entry = entry_of(c, t, at + lane * waves, end);
        n = min(64, (end - at + waves - 1) / waves);
        static_for<AHEAD>([&](auto d) { fetch(d, ring[d]); });
      }
      for (int i = 0; i < n; i += AHEAD + 1)
        static_for<AHEAD + 1>([&](auto d) {
          if (i + d < n) {
            fetch(i + d + AHEAD, ring[(d + AHEAD) % (AHEAD + 1)]);
            if (__builtin_amdgcn_readlane(entry, i + d) >= 0) step(ring[d], at + (i + d) * waves);
          }
        });
    }
  }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {     // 0 where the control names no lane
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xF, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xF, false);
  return v + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_max(int v) {
  return max(v, __builtin_amdgcn_update_dpp(INT32_MIN, v, CTRL, ROWS, 0xF, false));
}
// over 64 or 16 lanes, in each of them
template <int LANES>
__device__ __forceinline__ double lanes_sum(double v) {
  v = dpp_add<0xB1, 0xF>(v);                             // quad_perm [1,0,3,2]
  v = dpp_add<0x4E, 0xF>(v);                             // quad_perm [2,3,0,1]
  v = dpp_add<0x141, 0xF>(v);                            // row_half_mirror
  v = dpp_add<0x140, 0xF>(v);                            // row_mirror: each row of 16 its sum
  if constexpr (LANES == 16) return v;
  v = dpp_add<0x142, 0xA>(v);                            // row_bcast:15 into rows 1 and 3
  v = dpp_add<0x143, 0xC>(v);                            // row_bcast:31 into rows 2 and 3: lane 63 has them all
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_readlane((int)u, 63), hi = __builtin_amdgcn_readlane((int)(u >> 32), 63);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
template <int LANES>
__device__ __forceinline__ int lanes_max(int v) {
  v = dpp_max<0xB1, 0xF>(v);
  v = dpp_max<0x4E, 0xF>(v);
  v = dpp_max<0x141, 0xF>(v);
  v = dpp_max<0x140, 0xF>(v);
  if constexpr (LANES == 16) return v;
  v = dpp_max<0x142, 0xA>(v);
  v = dpp_max<0x143, 0xC>(v);
  return __builtin_amdgcn_readlane(v, 63);
}

// A row's table in place of its histogram, by LANES lanes (64 or 16, which stay together): lane l has counts 4 (l + LANES i) + j.
//
// p = floor(n / S) with n = e one + floor(S / 2), S the sum of e x count; whole numbers below 2^53, so sums in double are exact. For
// S < 2^34 the quotient is e (one / S) + (floor(S / 2) / S + 2^-35), truncated. Two Newton steps leave 1 / S good to 2^-51 whatever
// v_rcp_f64 is off by up to 2^-20, and with the roundings (2^-53 each) of a quotient below 2^15 the sum is off by less than
// 2^15 (2^-51 + 2 2^-53) + 2^-51 < 2^-35: it is not below the quotient, and above it by less than 2^-34 < 1 / S, so no whole number
// lies between the two. For a larger S the quotient is put right by its remainder.
//
// That p is at most `one`, and so fits its part of a packed entry, holds for the scores that the row has: their e is part of S. A table need
// not rise, and the entry of a score that no key has may be larger than S by any factor: it counts as 0.
template <int TABLE, int LANES>
__device__ __forceinline__ void probabilities(unsigned* table, const int* lut, int one, unsigned* flags) {
  constexpr int N = 64 / LANES;
  const int lane = threadIdx.x & (LANES - 1);
  uint4 count[N];
  int top = -1;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    unsigned* h = table + 4 * (lane + LANES * i);        // rows start at any dword
    count[i] = {h[0], h[1], h[2], h[3]};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (word(count[i], j)) top = 4 * LANES * i + j;
  }
  top = lanes_max<LANES>(top < 0 ? -1 : top + 4 * lane);
  unsigned p[N][4];
  double e[N][4], S = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int x = min(4 * (lane + LANES * i) + j, max(top, 0)) - max(top, 0) + 255;        // larger scores do not occur
      e[i][j] = (double)(unsigned)max(0, lut[x]);
      S = __builtin_fma(e[i][j], (double)word(count[i], j), S);
    }
  S = lanes_sum<LANES>(S);
  if (S == 0) {                                          // nothing seen, or nothing but zeros
    if (top >= 0 && lane == 0) raise_flag(flags, FLAG_ZERODIV);
    S = 1;
    one = 0;
  }
  const double half = __builtin_trunc(0.5 * S);
  double inv = __builtin_amdgcn_rcp(S);
  inv = __builtin_fma(inv, __builtin_fma(-S, inv, 1.0), inv);
  inv = __builtin_fma(inv, __builtin_fma(-S, inv, 1.0), inv);
  const double by = (double)one * inv, start = __builtin_fma(half, inv, 0x1p-35);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) p[i][j] = (unsigned)__builtin_fma(e[i][j], by, start);
  if (S >= 0x1p34) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double n = __builtin_fma(e[i][j], (double)one, half);
        double k = __builtin_trunc(n * inv);
        const double rest = __builtin_fma(-k, S, n);
        k += rest < 0 ? -1.0 : (rest >= S ? 1.0 : 0.0);
        p[i][j] = (unsigned)k;
      }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[i][j] = word(count[i], j) ? p[i][j] : 0u;
    const int at = lane + LANES * i;
    if constexpr (TABLE == TABLE_FIFTEEN) {              // a byte each of four tables
      int x[4] = {(int)p[i][0], (int)p[i][1], (int)p[i][2], (int)p[i][3]};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        int d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int up = (int)((unsigned)__umul24(x[j] + 7, 34953) >> 19);        // / 15, exact below 2^19 / 7
          d[j] = x[j] - 15 * up, x[j] = up;
        }
        table[64 * v + at] = pack4(d[0], d[1], d[2], d[3]);
      }
    } else if constexpr (TABLE == TABLE_BYTES) {
      table[at] = pack4((int)p[i][0], (int)p[i][1], (int)p[i][2], (int)p[i][3]);
    } else if constexpr (TABLE == TABLE_PAIRS) {         // a low digit from -128 on and a high one, a byte each
      unsigned d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = (p[i][j] & 255u) | ((p[i][j] + 128u) & 0xFF00u);
      table[2 * at] = d[0] | d[1] << 16, table[2 * at + 1] = d[2] | d[3] << 16;
    } else if constexpr (TABLE == TABLE_SEVEN) {
      table[2 * at] = 2 * (p[i][0] & 127u) | (p[i][1] & 127u) << 17, table[2 * at + 1] = 2 * (p[i][2] & 127u) | (p[i][3] & 127u) << 17;
      table[128 + 2 * at] = 2 * (p[i][0] >> 7) | (p[i][1] >> 7) << 17;
      table[129 + 2 * at] = 2 * (p[i][2] >> 7) | (p[i][3] >> 7) << 17;
    } else {
      table[2 * at] = 2 * p[i][0] | p[i][1] << 17, table[2 * at + 1] = 2 * p[i][2] | p[i][3] << 17;
    }
  }
}

// The tables of a tile's rows. A wave takes a row at a time, or four where there are many: the sums over lanes and what is one number
// a row cost a row less.
template <int TABLE, bool MANY>
__device__ __forceinline__ void make_tables(unsigned* rows, int n_rows, const int* lut, int one, unsigned* flags) {
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if constexpr (MANY) {
    for (int i = 4 * wave + ((threadIdx.x >> 4) & 3); i < n_rows; i += 4 * waves) probabilities<TABLE, 16>(rows + i * HIST, lut, one, flags);
  } else {
    for (int i = wave; i < n_rows; i += waves) probabilities<TABLE, 64>(rows + i * HIST, lut, one, flags);
  }
}

// A wave's accumulators as 16 x sums of p V (modulo 2^32, in which the sum itself lies) into row-major int32.
template <int NG, int RP, bool WIDE>
__device__ __forceinline__ void spill(const v4i (&acc)[Digits<RP, WIDE>::SUMS][2 * NG], int* rows, int stride, int n_rows) {
  using D = Digits<RP, WIDE>;
  constexpr int VN = 16 / RP;
  const int lane = threadIdx.x & 63, r = (lane & 15) / VN, v = lane % VN, q = lane >> 4;
#pragma unroll
  for (int m = 0; m < 2 * NG; ++m) {
    v4i s;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      unsigned x = 0;
#pragma unroll
      for (int n = 0; n < D::SUMS; ++n) x += (unsigned)acc[n][m][e] * D::weight(v, n);
      if constexpr (VN > 1) x += (unsigned)lane_xor<1>((int)x);
      if constexpr (VN > 2) x += (unsigned)lane_xor<2>((int)x);
      s[e] = (int)x;
    }
    if (v == 0 && r < n_rows) *(v4i*)(rows + r * stride + 16 * m + 4 * q) = s;
  }
}

// four results of a row from its sums
__device__ __forceinline__ unsigned finish4(const v4i& sum, const AttendArgs& a) {
  int o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const long long v = ((long long)sum[e] * a.m_o + round_term(a.s_o)) >> a.s_o;
    o[e] = v < -128 ? -128 : (v > 127 ? 127 : (int)v);
  }
  return pack4(o[0], o[1], o[2], o[3]);
}

__device__ __forceinline__ unsigned* out_word(const AttendArgs& a, const Tile& t, int r, int ch) {
  const int at = t.first + r;
  return (unsigned*)(a.o + (long long)(t.r.first + at / a.group) * a.o_row + (long long)(t.head * a.group + at % a.group) * a.o_head + ch);
}

// The sum over the workgroup's waves of what each holds, in LDS (`red`: waves x rows x SUM_STRIDE), then f(row, channel, sum).
template <int NG>
constexpr int SUM_STRIDE = 32 * NG + 4;
template <int NG, int RP, bool WIDE, typename F>
__device__ __forceinline__ void join_waves(const v4i (&acc)[Digits<RP, WIDE>::SUMS][2 * NG], int* red, const Tile& t, F&& f) {
  constexpr int STRIDE = SUM_STRIDE<NG>;
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  spill<NG, RP, WIDE>(acc, red + wave * t.rows * STRIDE, STRIDE, t.rows);
  __syncthreads();
  for (int i = threadIdx.x; i < t.rows * 8 * NG; i += blockDim.x) {
    const int r = i / (8 * NG), ch = 4 * (i % (8 * NG));
    v4i s = {0, 0, 0, 0};
    for (int w = 0; w < waves; ++w) s += *(const v4i*)(red + (w * t.rows + r) * STRIDE + ch);
    f(r, ch, s);
  }
}

constexpr int WAVES_MAX = 8;

// Where a lane stands in the first pass: its row, and which of the row's 64 scores of a page are its NE dwords.
template <int NG, int RP>
struct Place {
  using C = Columns<NG, RP>;
  int r, word, bit;
  __device__ __forceinline__ Place() {
    const int lane = threadIdx.x & 63;
    r = (lane & 15) / C::VN;
    word = 4 * (lane >> 4) + C::NE * (lane % C::VN);
    bit = 4 * C::NE * (lane % C::VN);                    // of the quarter's 16 keys
  }
};

template <int NG, int RP>
using KeyWalk = Walk<NG, 1, KeyPage<NG, RP>>;
template <int NG>
using ValueWalk = Walk<NG, 1, ValuePage<NG>>;

template <int NG, int RP>
__device__ __forceinline__ void score_pages(KeyWalk<NG, RP>& walk, const CacheView& c, const AttendArgs& a, const Tile& t,
                                            unsigned* hist, unsigned* scores, int row_slots) {
  using C = Columns<NG, RP>;
  const int lane = threadIdx.x & 63, q = lane >> 4;
  const Place<NG, RP> at;
  const Row row(t, a, at.r);
  Query<NG, RP> query;
  query.load(c, a, t, lane);
  const Requant rq(a.m_s, a.s_s);
  walk.run([&](const KeyPage<NG, RP>& page, int n) {
    const Words<C::NE> sc = score_page<NG, RP>(page, query, rq);
    const int slot = slot_of(t, n);
    if (!row.on) return;
    unsigned* out = scores + ((long long)n * row_slots + at.r) * (PAGE / 4) + at.word;
    if constexpr (C::NE == 4) *(uint4*)out = {sc.w[0], sc.w[1], sc.w[2], sc.w[3]};
    else if constexpr (C::NE == 2) *(uint2*)out = {sc.w[0], sc.w[1]};
    else *out = sc.w[0];
    if (whole(t, a, slot)) count_scores(hist + at.r * HIST, sc);
    else count_scores(hist + at.r * HIST, sc, row.mask(slot * PAGE + 16 * q) >> at.bit);
  });
}

template <int NG, int RP, bool WIDE>
__device__ __forceinline__ void add_pages(ValueWalk<NG>& walk, const AttendArgs& a, const Tile& t, const unsigned* tables,
                                          const unsigned* scores, int row_slots, v4i (&acc)[Digits<RP, WIDE>::SUMS][2 * NG]) {
  constexpr int VN = 16 / RP;
  const int lane = threadIdx.x & 63, q = lane >> 4, v = lane % VN;
  const Row row(t, a, (lane & 15) / VN);
  const int r = row.on ? (lane & 15) / VN : 0;
  const int which = RP == 4 ? 64 * v : (RP == 8 && WIDE ? 128 * v : 0);          // of the row's tables
  const uint8_t* table = (const uint8_t*)(tables + r * HIST + which);
  walk.run([&](const ValuePage<NG>& page, int n) {
    const int slot = slot_of(t, n);
    const uint4 sc = *(const uint4*)(scores + ((long long)n * row_slots + r) * (PAGE / 4) + 4 * q);
    add_page<NG, RP, WIDE>(page, sc, table, whole(t, a, slot), row.mask(slot * PAGE + 16 * q), acc);
  });
}

// What a workgroup clears and fetches before it knows its tile, whose numbers come from memory themselves: the histograms, the
// exponentials' table, and without a window the wave's first table entries.
struct Early {
  int lut, entry;
  __device__ __forceinline__ Early(const CacheView& c, const AttendArgs& a, unsigned* hist, bool entries) {
    lut = threadIdx.x < 256 ? a.lut[threadIdx.x] : 0;
    entry = -1;
    const int page = (int)(threadIdx.x >> 6) + (int)(threadIdx.x & 63) * (int)(blockDim.x >> 6);
    if (entries && !a.window && page < c.slots) entry = c.table[(long long)(a.seq0 + (int)blockIdx.x / c.heads) * c.slots + page];
    for (int i = threadIdx.x; i < a.rows * HIST; i += blockDim.x) hist[i] = 0;
  }
  __device__ __forceinline__ void keep(int* table) const {
    if (threadIdx.x < 256) table[threadIdx.x] = lut;
  }
  // the wave's first entries of a walk over pages begin .. end - 1; `mine`: read ahead
  __device__ __forceinline__ int entries(const CacheView& c, const AttendArgs& a, const Tile& t, int begin, int end, bool mine) const {
    const int page = begin + (int)(threadIdx.x >> 6) + (int)(threadIdx.x & 63) * (int)(blockDim.x >> 6);
    if (!mine || a.window) return entry_of(c, t, page, end);
    if (page >= end || entry == -1) return -1;
    if (entry < -1 || entry >= c.pages) {
      raise_flag(c.flags, FLAG_CACHE);
      return -1;
    }
    return entry;
  }
};

// Both passes of a tile in one workgroup, its scores in LDS.
template <int NG, int RP, bool WIDE>
__global__ __launch_bounds__(64 * WAVES_MAX) void attend_tile_kernel(CacheView c, AttendArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  int* lut = (int*)lds;
  unsigned* hist = lds + 256;
  unsigned* scores = hist + (a.rows * HIST + 3) / 4 * 4;
  const Early early(c, a, hist, true);
  Tile t;
  if (!find_tile(c, a, t)) return;
  const int entry = early.entries(c, a, t, 0, t.pages, true);
  {
    KeyWalk<NG, RP> keys(c, t, 0, t.pages, entry);
    early.keep(lut);
    __syncthreads();
    score_pages<NG, RP>(keys, c, a, t, hist, scores, t.rows);
  }
  ValueWalk<NG> values(c, t, 0, t.pages, entry);         // on their way while the tables are made
  __syncthreads();
  make_tables<Digits<RP, WIDE>::TABLE, RP == 16>(hist, t.rows, lut, a.one, c.flags);
  __syncthreads();
  v4i acc[Digits<RP, WIDE>::SUMS][2 * NG] = {};
  add_pages<NG, RP, WIDE>(values, a, t, hist, scores, t.rows, acc);
  __syncthreads();                                       // the scores have been read
  join_waves<NG, RP, WIDE>(acc, (int*)scores, t, [&](int i, int ch, const v4i& s) {
    if (ch < c.dim) *out_word(a, t, i, ch) = finish4(s >> 4, a);
  });
}

// ---- one tile over several workgroups: scores and histograms, then sums, then their total

// pages of a part: parts are of equal size, at least a page a wave
__device__ __forceinline__ int part_pages(const Tile& t, const AttendArgs& a, int waves) { return max(waves, (t.pages + a.splits - 1) / a.splits); }

template <int NG, int RP>
__global__ __launch_bounds__(64 * WAVES_MAX) void attend_scores_kernel(CacheView c, AttendArgs a) {
  __shared__ unsigned hist[RP * HIST];
  for (int i = threadIdx.x; i < a.rows * HIST; i += blockDim.x) hist[i] = 0;
  Tile t;
  if (!find_tile(c, a, t)) return;
  const int per = part_pages(t, a, blockDim.x >> 6), begin = (int)blockIdx.z * per, end = min(begin + per, t.pages);
  if (begin >= end) return;
  const int page = begin + (int)(threadIdx.x >> 6) + (int)(threadIdx.x & 63) * (int)(blockDim.x >> 6);
  KeyWalk<NG, RP> keys(c, t, begin, end, entry_of(c, t, page, end));
  __syncthreads();
  const long long unit = (long long)t.unit * a.tiles + t.tile;
  score_pages<NG, RP>(keys, c, a, t, hist, (unsigned*)a.scores + unit * a.bound * a.rows * (PAGE / 4), a.rows);
  __syncthreads();
  unsigned* out = a.hist + (unit * a.splits + blockIdx.z) * a.rows * 256;
  for (int i = threadIdx.x; i < t.rows * 256; i += blockDim.x) out[i] = hist[(i >> 8) * HIST + (i & 255)];
}

template <int NG, int RP, bool WIDE>
__global__ __launch_bounds__(64 * WAVES_MAX) void attend_values_kernel(CacheView c, AttendArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  int* lut = (int*)lds;
  unsigned* tables = lds + 256;
  int* red = (int*)(tables + (a.rows * HIST + 3) / 4 * 4);
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  for (int i = tid; i < 256; i += blockDim.x) lut[i] = a.lut[i];
  for (int i = tid; i < a.rows * HIST; i += blockDim.x) tables[i] = 0;
  Tile t;
  if (!find_tile(c, a, t)) return;
  const int per = part_pages(t, a, waves), parts = (t.pages + per - 1) / per;
  const int begin = (int)blockIdx.z * per, end = min(begin + per, t.pages);
  if (begin >= end) return;
  ValueWalk<NG> values(c, t, begin, end, entry_of(c, t, begin + (tid >> 6) + lane * waves, end));
  __syncthreads();
  const long long unit = (long long)t.unit * a.tiles + t.tile;
  const uint4* slices = (const uint4*)(a.hist + unit * a.splits * a.rows * 256) + lane;
  // all parts' histograms: a wave takes a row of every several parts, eight of them at once
  const int share = max(1, waves / t.rows);
  for (int i = tid >> 6; i < t.rows * share; i += waves) {
    const int row = i % t.rows;
    uint4 sum = {0, 0, 0, 0};
    for (int p = i / t.rows; p < parts; p += 8 * share) {
      uint4 x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] = {0, 0, 0, 0};
        if (p + k * share < parts) x[k] = slices[((long long)(p + k * share) * a.rows + row) * 64];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sum.x += x[k].x, sum.y += x[k].y, sum.z += x[k].z, sum.w += x[k].w;
    }
    unsigned* h = tables + row * HIST + 4 * lane;
    atomicAdd(h, sum.x), atomicAdd(h + 1, sum.y), atomicAdd(h + 2, sum.z), atomicAdd(h + 3, sum.w);
  }
  __syncthreads();
  make_tables<Digits<RP, WIDE>::TABLE, RP == 16>(tables, t.rows, lut, a.one, c.flags);
  __syncthreads();
  v4i acc[Digits<RP, WIDE>::SUMS][2 * NG] = {};
  add_pages<NG, RP, WIDE>(values, a, t, tables, (const unsigned*)a.scores + unit * a.bound * a.rows * (PAGE / 4), a.rows, acc);
  int* sums = a.sums + (unit * a.splits + blockIdx.z) * a.rows * 32 * NG;
  join_waves<NG, RP, WIDE>(acc, red, t, [&](int i, int ch, const v4i& s) { *(v4i*)(sums + i * 32 * NG + ch) = s; });
}

// One wave a row and 16 channels: four lanes to the channels, 16 to the parts.
constexpr int JOIN_THREADS = 64;
template <int NG>
__global__ __launch_bounds__(JOIN_THREADS) void attend_join_kernel(CacheView c, AttendArgs a, int waves) {
  Tile t;
  if (!find_tile(c, a, t)) return;
  const int r = (int)blockIdx.z / (2 * NG), ch = 16 * ((int)blockIdx.z % (2 * NG)) + 4 * (threadIdx.x & 3);
  if (r >= t.rows || ch >= c.dim) return;
  const long long unit = (long long)t.unit * a.tiles + t.tile;
  const int per = part_pages(t, a, waves), parts = (t.pages + per - 1) / per;
  const int* p = a.sums + (unit * a.splits * a.rows + r) * 32 * NG + ch;
  v4i s = {0, 0, 0, 0};
  for (int n = threadIdx.x >> 2; n < parts; n += 16) s += *(const v4i*)(p + (long long)n * a.rows * 32 * NG);
#pragma unroll
  for (int d = 4; d < 64; d *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += __shfl_xor(s[e], d);
  if (threadIdx.x < 4) *out_word(a, t, r, ch) = finish4(s >> 4, a);
}

// ---- many rows: pages made int8 once, in the workspace, then tiles of 32 rows
//
// Where a sequence has many rows its pages are worth multiplying out first: a score is then the product itself, a digit of p an
// operand as it stands, and nothing is left between the products but the requant and the two tables. Scores are not kept but made again
// in the second pass, so that a tile needs LDS for its histograms alone and has any length. 4 sequences of 32 heads over 8 of 128
// channels, 1024 new tokens of 16384 each: 3134 us with tiles of 16 rows, 1154 with these; 2 of up to 512 new of up to 4096: 188 and 92.
// Of the latter's time VALU instructions take 28 % on a SIMD, the LDS 30 % (20 % conflicts on histograms and tables), MFMAs 12 %; a wave
// lives 37 of the 92 us, and of the two workgroups that a CU has room for one is there on average, as the tiles with rows come unevenly.
// The second with 16, 32, 48 and 64 rows a tile: 114, 92, 106, 100 us; with 2, 3, 4 and 8 waves 90, 114, 92, 105, and with 2 a third
// more where tiles are short (4 x 12 heads of 64, 512 new, the last 1024 seen).

constexpr int WIDE_TILES = 2, WIDE_ROWS = 16 * WIDE_TILES, WIDE_WAVES = 4;
constexpr int ONE_PAIR = 127 * 256 + 127;                // 32639: two digits, the low one from -128 on
__device__ __forceinline__ unsigned mad_pair(unsigned a, unsigned b, unsigned c) {
  return __builtin_bit_cast(unsigned, (v2u)(__builtin_bit_cast(v2u, a) * __builtin_bit_cast(v2u, b) + __builtin_bit_cast(v2u, c)));
}

// A lane's part of a page's keys: of keys 4 row + k, k in 0..3, the codes of 8 channels a group, and the steps.
template <int NG>
struct KeyRows {
  Words<NG> code[4], step;
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t blk, int lane) {
    const int row = lane & 15, q = lane >> 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) code[k] = load_words<NG>(blk, (4 * row + k) * Block<NG>::ROW + 4 * q * NG);
    step = load_words<NG>(blk, Block<NG>::K_STEPS + 4 * NG * row);
  }
  // Key k's values, four bytes a dword: two codes + 8 = u as a number u1 256 + u0, times the step, less 8 x 257 steps and with 128 added,
  // so that the low byte does not borrow from the high one.
  template <int k>
  __device__ __forceinline__ void values(unsigned (&x)[2 * NG]) const {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const unsigned s = __builtin_amdgcn_perm(0, step.w[g], 0x0c000c00u | k << 16 | k), c = mad_pair(s, 0xF7F8F7F8u, 0x00800080u);
      const unsigned u = code[k].w[g] ^ 0x88888888u;
      x[2 * g] = mad_pair(u & 0x0F0F0F0Fu, s, c) ^ 0x00800080u;
      x[2 * g + 1] = mad_pair((u >> 4) & 0x0F0F0F0Fu, s, c) ^ 0x00800080u;
    }
  }
};

// Group g's values, 16 keys of two channels: a product's low byte is that of its operands' low bytes, whatever lies above them.
template <int NG>
__device__ __forceinline__ void values_of(const ValuePage<NG>& v, int g, v4i (&x)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned u = v.code[g].w[i] ^ 0x88888888u, s0 = v.step[g].w[i], s1 = s0 >> 8;
    const unsigned c0 = mul_pair(s0, 0xFFF8FFF8u), c1 = mul_pair(s1, 0xFFF8FFF8u);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const unsigned n = (half ? u >> 4 : u) & 0x0F0F0F0Fu;
      x[half][i] = (int)__builtin_amdgcn_perm(mad_pair(n >> 8, s1, c1), mad_pair(n, s0, c0), 0x06020400u);
    }
  }
}

// A page in the workspace: the operands of its products, a lane's next to the next one's.
template <int NG>
struct Wide {
  static constexpr int KN = NG == 1 ? 1 : NG / 2, KB = NG == 1 ? 8 : 16;         // products and bytes a lane of 16 keys
  static constexpr int K = 64 * KB, V = 4 * KN * K, BYTES = V + 2 * NG * 1024;
};

// The pages that some new row of a sequence may see, numbered as a tile's are; a tile's own are among them.
struct Span {
  int sink_pages, window_page, pages;
  __device__ __forceinline__ Span(const NewRows& r, const AttendArgs& a) {
    const int lo = r.len - r.n;
    window_page = a.window && lo >= a.window ? (lo - a.window + 1) >> PAGE_SHIFT : 0;
    sink_pages = min((a.sinks + PAGE - 1) >> PAGE_SHIFT, window_page);
    pages = sink_pages + ((r.len - 1) >> PAGE_SHIFT) - window_page + 1;
  }
  __device__ __forceinline__ int slot(int page) const { return page < sink_pages ? page : window_page + page - sink_pages; }
  __device__ __forceinline__ int page(int slot) const { return slot < sink_pages ? slot : slot - window_page + sink_pages; }
};

// blockIdx: cache head of a sequence, page (a wave each, four a workgroup).
template <int NG>
__global__ __launch_bounds__(256) void attend_widen_kernel(CacheView c, AttendArgs a) {
  const int unit = blockIdx.x, seq = a.seq0 + unit / c.heads, head = unit % c.heads, lane = threadIdx.x & 63;
  const int page = 4 * (int)blockIdx.y + (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  NewRows r;
  if (!new_rows(c, seq, r, blockIdx.y == 0 && head == 0 && threadIdx.x == 0) || !r.n) return;
  const Span span(r, a);
  if (page >= span.pages) return;
  const uint8_t* blk = page_block<NG>(c, seq, span.slot(page), head, head == 0 && lane == 0);
  if (!blk) return;
  KeyRows<NG> k;
  ValuePage<NG> v;
  k.load(uniform_rsrc(blk, Block<NG>::BYTES), lane);
  v.load(uniform_rsrc(blk, Block<NG>::BYTES), lane);
  uint8_t* out = a.scores + ((long long)unit * a.bound + page) * Wide<NG>::BYTES;
  static_for<4>([&](auto i) {
    unsigned x[2 * NG];
    k.template values<i>(x);
    uint8_t* o = out + i * Wide<NG>::KN * Wide<NG>::K;
    if constexpr (NG == 1) {
      *(uint2*)(o + 8 * lane) = {x[0], x[1]};
    } else {
#pragma unroll
      for (int n = 0; n < NG / 2; ++n) *(uint4*)(o + 1024 * n + 16 * lane) = {x[4 * n], x[4 * n + 1], x[4 * n + 2], x[4 * n + 3]};
    }
  });
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    v4i x[2];
    values_of<NG>(v, g, x);
#pragma unroll
    for (int half = 0; half < 2; ++half) *(v4i*)(out + Wide<NG>::V + 1024 * (2 * g + half) + 16 * lane) = x[half];
  }
}

template <int NG>
struct WideKeys {
  static constexpr int N = Wide<NG>::KN, W = Wide<NG>::KB / 4;
  Words<W> k[4][N];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t page, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < N; ++n) k[i][n] = load_words<W>(page, (i * N + n) * Wide<NG>::K + 4 * W * lane);
  }
};
template <int NG>
struct WideValues {
  Words<4> v[2 * NG];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t page, int lane) {
#pragma unroll
    for (int m = 0; m < 2 * NG; ++m) v[m] = load_words<4>(page, Wide<NG>::V + 1024 * m + 16 * lane);
  }
};

// A wave's pages of a tile in the workspace, as Walk's in the pool. step(page, its resource, ahead): ahead() when `page` is done with.
template <int NG, int AHEAD>
struct WideWalk {
  WideKeys<NG> ring[AHEAD + 1];
  const CacheView& c;
  const Tile& t;
  const Span span;
  const uint8_t* base;
  const int first, waves, lane;
  int entry, n;

  __device__ __forceinline__ WideWalk(const CacheView& view, const AttendArgs& a, const Tile& tile, int entries)
      : c(view), t(tile), span(tile.r, a), base(a.scores + (long long)tile.unit * a.bound * Wide<NG>::BYTES),
        first(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), waves(blockDim.x >> 6), lane(threadIdx.x & 63), entry(entries) {
    n = min(64, (t.pages - first + waves - 1) / waves);
    static_for<AHEAD>([&](auto d) { ring[d].load(page_of(first, d), lane); });
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t page_of(int at, int i) const {
    const int e = i < n ? __builtin_amdgcn_readlane(entry, i & 63) : -1;
    const int page = e < 0 ? 0 : span.page(slot_of(t, at + i * waves));
    return uniform_rsrc(base + (long long)page * Wide<NG>::BYTES, e < 0 ? 0 : Wide<NG>::BYTES);
  }
  template <typename Step>
  __device__ __forceinline__ void run(Step&& step) {
    for (int at = first; at < t.pages; at += 64 * waves) {
      if (at != first) {
        entry = entry_of(c, t, at + lane * waves, t.pages);
        n = min(64, (t.pages - at + waves - 1) / waves);
        static_for<AHEAD>([&](auto d) { ring[d].load(page_of(at, d), lane); });
      }
      for (int i = 0; i < n; i += AHEAD + 1)
        static_for<AHEAD + 1>([&](auto d) {
          if (i + d < n) {
            ring[(d + AHEAD) % (AHEAD + 1)].load(page_of(at, i + d + AHEAD), lane);
            if (__builtin_amdgcn_readlane(entry, i + d) >= 0) step(ring[d], at + (i + d) * waves, page_of(at, i + d));
          }
        });
    }
  }
};

// f(tile r, e, k, score) for the lane's 16 keys 16 q + 4 e + k of the R rows that are its columns.
template <int NG, int R, typename F>
__device__ __forceinline__ void scores_of(const WideKeys<NG>& page, const Query<NG, 16> (&query)[R], const Requant& rq, F&& f) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      v4i d = {0, 0, 0, 0};
      if constexpr (NG == 1) {
        d = __builtin_amdgcn_mfma_i32_16x16x32_i8((long)((unsigned long)page.k[k][0].w[1] << 32 | page.k[k][0].w[0]), query[r].w[0], d, 0, 0, 0);
      } else {
#pragma unroll
        for (int n = 0; n < NG / 2; ++n) {
          const Words<4>& w = page.k[k][n];
          const v4i keys = {(int)w.w[0], (int)w.w[1], (int)w.w[2], (int)w.w[3]};
          const v4i rows = {(int)query[r].w[2 * n], (int)(query[r].w[2 * n] >> 32), (int)query[r].w[2 * n + 1], (int)(query[r].w[2 * n + 1] >> 32)};
          d = __builtin_amdgcn_mfma_i32_16x16x64_i8(keys, rows, d, 0, 0, 0);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) f(r, e, k, med3i(__mul24(d[e], rq.m) + rq.rnd, rq.lo, rq.hi) >> rq.s);
    }
}

template <int NG, int ND>
__global__ __launch_bounds__(64 * WIDE_WAVES) void attend_rows_kernel(CacheView c, AttendArgs a) {
  constexpr int R = WIDE_TILES;
  extern __shared__ __align__(16) unsigned lds[];
  int* lut = (int*)lds;
  unsigned* hist = lds + 256;
  const Early early(c, a, hist, true);
  Tile t;
  if (!find_tile<WIDE_ROWS>(c, a, t)) return;
  const int lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4, wave = threadIdx.x >> 6;
  const int entry = early.entries(c, a, t, 0, t.pages, true);
  Query<NG, 16> query[R];
#pragma unroll
  for (int r = 0; r < R; ++r) query[r].load(c, a, t, lane, 16 * r);
  const Requant rq(a.m_s, a.s_s);
  {
    WideWalk<NG, 1> keys(c, a, t, entry);
    early.keep(lut);
    __syncthreads();
    unsigned* mine = hist + col * HIST + 128;            // of a score of 0
    keys.run([&](const WideKeys<NG>& page, int n, __amdgpu_buffer_rsrc_t) {
      const int slot = slot_of(t, n);
      if (whole(t, a, slot)) {
        scores_of<NG, R>(page, query, rq, [&](int r, int, int, int x) { atomicAdd(mine + 16 * HIST * r + x, 1u); });
      } else {
        unsigned mask[R];
#pragma unroll
        for (int r = 0; r < R; ++r) mask[r] = Row(t, a, 16 * r + col).mask(slot * PAGE + 16 * q);
        scores_of<NG, R>(page, query, rq,
                         [&](int r, int e, int k, int x) { atomicAdd(mine + 16 * HIST * r + x, mask[r] >> (4 * e + k) & 1u); });
      }
    });
  }
  WideWalk<NG, (R * NG * ND > 8 ? 0 : 1)> keys(c, a, t, entry);                  // on their way while the tables are made
  __syncthreads();
  make_tables<ND == 1 ? TABLE_BYTES : TABLE_PAIRS, true>(hist, t.rows, lut, a.one, c.flags);
  __syncthreads();
  v4i acc[R][2 * NG][ND] = {};
  keys.run([&](const WideKeys<NG>& page, int n, __amdgpu_buffer_rsrc_t rsrc) {
    WideValues<NG> v;
    v.load(rsrc, lane);
    unsigned p[R][4][ND] = {};                           // digits of 4 keys a dword, or both of two
    if constexpr (ND == 1) {
      const uint8_t* mine = (const uint8_t*)(hist + col * HIST) + 128;
      scores_of<NG, R>(page, query, rq, [&](int r, int i, int k, int x) { p[r][i][0] |= (unsigned)mine[4 * 16 * HIST * r + x] << (8 * k); });
    } else {
      const u16_alias* mine = (const u16_alias*)(hist + col * HIST) + 128;
      scores_of<NG, R>(page, query, rq,
                       [&](int r, int i, int k, int x) { p[r][i][k >> 1] |= (unsigned)mine[2 * 16 * HIST * r + x] << (16 * (k & 1)); });
    }
    v4i digit[R][ND];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (ND == 1) {
          digit[r][0][i] = (int)p[r][i][0];
        } else {
          digit[r][0][i] = (int)__builtin_amdgcn_perm(p[r][i][1], p[r][i][0], 0x06040200u);
          digit[r][1][i] = (int)__builtin_amdgcn_perm(p[r][i][1], p[r][i][0], 0x07050301u);
        }
      }
    const int slot = slot_of(t, n);
    if (!whole(t, a, slot)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const unsigned mask = Row(t, a, 16 * r + col).mask(slot * PAGE + 16 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {                    // a byte of ones a key that is seen
          const unsigned seen = (((mask >> (4 * i) & 15u) * 0x00204081u) & 0x01010101u) * 255u;
#pragma unroll
          for (int d = 0; d < ND; ++d) digit[r][d][i] &= (int)seen;
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 2 * NG; ++m) {
      const v4i x = {(int)v.v[m].w[0], (int)v.v[m].w[1], (int)v.v[m].w[2], (int)v.v[m].w[3]};
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[r][m][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, digit[r][d], acc[r][m][d], 0, 0, 0);
    }
  });
  // the waves' sums, 16 rows at a time, where the tables were
  constexpr int STRIDE = SUM_STRIDE<NG>;
  int* red = (int*)hist;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    __syncthreads();
    if (16 * r >= t.rows) break;
#pragma unroll
    for (int m = 0; m < 2 * NG; ++m) {
      v4i s = acc[r][m][0];
      if constexpr (ND == 2) s += acc[r][m][1] * 256;
      *(v4i*)(red + (16 * wave + col) * STRIDE + 16 * m + 4 * q) = s;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(16, t.rows - 16 * r) * 8 * NG; i += blockDim.x) {
      const int row = i / (8 * NG), ch = 4 * (i % (8 * NG));
      v4i s = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < WIDE_WAVES; ++w) s += *(const v4i*)(red + (16 * w + row) * STRIDE + ch);
      if (ch < c.dim) *out_word(a, t, 16 * r + row, ch) = finish4(s, a);
    }
  }
}

constexpr int LDS_MAX = 160 * 1024;                      // of a CU
constexpr long long WIDE_MAX = 2ll << 30;                // bytes of widened pages in the workspace
constexpr long long SCORES_MAX = 1ll << 30;              // bytes of scores in the workspace, unless one tile has more

template <typename K>
static int launch_lds(K kernel, dim3 grid, int threads, size_t lds, anvil_ctx* ctx, const CacheView& c, const AttendArgs& a) {
  if (lds > 64 * 1024)
    ANVIL_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS_MAX));
  ANVIL_LAUNCH(kernel, grid, dim3((unsigned)threads), lds, ctx->stream, c, a);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}

// The pages that the rows of a run of `tokens` tokens can see at most.
static int pages_seen(const CacheView& c, const AttendArgs& a, int tokens) {
  if (!a.window) return c.slots;
  const long long seen = ((long long)a.window + tokens + PAGE - 2) / PAGE + 1 + (a.sinks + PAGE - 1) / PAGE;
  return (int)std::min<long long>(c.slots, seen);
}

// As many sequences at once as the workspace holds widened pages of.
template <int NG, int ND>
static int attend_rows(anvil_ctx* ctx, const CacheView& c, AttendArgs a, long long all) {
  const long long tiles = (all + WIDE_ROWS - 1) / WIDE_ROWS, seq_bytes = (long long)c.heads * a.bound * Wide<NG>::BYTES;
  const int seqs = (int)std::min<long long>(c.seqs, WIDE_MAX / seq_bytes);
  const size_t lds = sizeof(int) * (256 + std::max<size_t>(WIDE_ROWS * HIST, (size_t)WIDE_WAVES * 16 * SUM_STRIDE<NG>));
  char* ws;
  if (int r = decode_workspace(ctx, (size_t)(seqs * seq_bytes), &ws)) return r;
  a.rows = WIDE_ROWS, a.scores = (uint8_t*)ws;
  for (a.seq0 = 0; a.seq0 < c.seqs; a.seq0 += seqs) {
    const unsigned units = (unsigned)(std::min(seqs, c.seqs - a.seq0) * c.heads);
    ANVIL_LAUNCH(attend_widen_kernel<NG>, dim3(units, (unsigned)(a.bound + 3) / 4), dim3(256), 0, ctx->stream, c, a);
    ANVIL_LAUNCHED();
    for (long long t0 = 0; t0 < tiles; t0 += 65535) {
      a.tile0 = (int)t0, a.tiles = (int)std::min<long long>(tiles - t0, 65535);
      if (int r = launch_lds(attend_rows_kernel<NG, ND>, dim3(units, (unsigned)a.tiles), 64 * WIDE_WAVES, lds, ctx, c, a)) return r;
    }
  }
  return ANVIL_OK;
}

template <int NG, int RP, bool WIDE>
static int attend(anvil_ctx* ctx, const CacheView& c, AttendArgs a) {
  const long long all = (long long)c.max_new * a.group;    // rows of a cache head at most
  a.rows = (int)std::min(16ll, all);
  const long long tiles = (all + 15) / 16;
  const int tokens = (int)std::min<long long>(c.max_new, (a.rows - 1) / a.group + 2);
  a.bound = pages_seen(c, a, tokens);
  const long long units = (long long)c.seqs * c.heads, groups = units * tiles;
  if constexpr (RP == 16) {
    // Widened pages pay where eight or more tiles of 32 rows read each, and where there are enough tiles for the CUs, which a tile of
    // twice the rows keeps busy twice as long: 2 tiles of 16 rows a CU over 2048 keys or more (32 heads over 8 of 128, 256 new of
    // 4096: 50.4 us with 16 rows, 40.2 with 32; of 1024 18.2 and 20.8), 8 over fewer (1024 new of 1024: 47.2 and 37.1). With few rows
    // (16 x 12 heads of 64, 64 new of 4096): 54.4 and 69.6. The numbers are those of max_new, as if every sequence had as many. Where one of
    // many has them, each as long, the two differ by the heads: 1 of 64 sequences with 512 of 8192, the others with one token, 32 heads over
    // 8 of 128 992 and 994 us, 16 over 4 of 64 613 and 365, but 12 of 64 305 and 541.
    AttendArgs wide = a;
    wide.bound = pages_seen(c, a, c.max_new);
    if (all >= 256 && groups >= 2ll * ctx->num_cu && (a.bound >= 32 || groups >= 8ll * ctx->num_cu) && a.one <= ONE_PAIR &&
        (long long)c.heads * wide.bound * Wide<NG>::BYTES <= WIDE_MAX)
      return a.one <= 127 ? attend_rows<NG, 1>(ctx, c, wide, all) : attend_rows<NG, 2>(ctx, c, wide, all);
  }
  const size_t fixed = sizeof(int) * (256 + (size_t)(a.rows * HIST + 3) / 4 * 4), row_sums = sizeof(int) * (size_t)a.rows * SUM_STRIDE<NG>;
  const size_t scores = (size_t)a.bound * a.rows * PAGE;
  // Four waves a workgroup where there are more tiles than CUs and two such workgroups fit a CU's LDS, else eight. Heads of 128 and 16-row
  // tiles take more than 128 registers a lane, so that eight waves leave no room for another workgroup: 32 heads over 8 of 128, 1024
  // tokens, with 256 tiles 12.2 us with four and 11.9 with eight, with 288 15.3 and 20.0, with 704 22.0 and 29.5; 12 heads of 64, 64 new of
  // 2048, 288 tiles: 20.9 and 24.7 (of 4096, where two do not fit the LDS, 48.5 and 37.5). The others have room for two of either: from 257 to
  // 512 tiles heads of 64 and 32 take 12.4 and 12.6, 11.3 and 11.0 over 1024 tokens, 29.4 and 28.9, 28.2 and 26.3 over 4096; with 576 tiles
  // and 1024 tokens 15.5 and 17.7, 14.1 and 14.4.
  const bool fit = fixed + std::max(scores, 4 * row_sums) <= LDS_MAX / 2;
  const bool many = NG == 4 || RP == 16 ? groups > ctx->num_cu : 2 * groups >= 3ll * ctx->num_cu;
  const int waves = many && fit ? 4 : 8;
  const size_t sums = waves * row_sums, lds = fixed + std::max(scores, sums);
  // Parts of a tile only where they bring CUs to work that the tiles leave idle, and where a tile is long: three launches cost what
  // one does over 32 pages.
  const bool whole_tiles = a.bound <= 32 || 3 * groups > ctx->num_cu;
  a.splits = whole_tiles ? 1 : (int)std::min<long long>(ctx->num_cu / groups, (a.bound + 7) / 8);
  if (a.splits == 1 && lds <= LDS_MAX) {
    for (long long t0 = 0; t0 < tiles; t0 += 65535) {    // a grid dimension's limit
      a.tile0 = (int)t0, a.tiles = (int)std::min<long long>(tiles - t0, 65535);
      if (int r = launch_lds(attend_tile_kernel<NG, RP, WIDE>, dim3((unsigned)units, (unsigned)a.tiles), 64 * waves, lds, ctx, c, a)) return r;
    }
    return ANVIL_OK;
  }
  // scores, histograms and sums of so many sequences and tiles at once
  const long long tile_scores = (long long)a.bound * a.rows * PAGE, tile_hist = 1024ll * a.splits * a.rows,
                  tile_sums = 128ll * NG * a.splits * a.rows, tile_bytes = tile_scores + tile_hist + tile_sums;
  const int seqs = (int)std::max<long long>(1, std::min<long long>(c.seqs, SCORES_MAX / (tile_bytes * c.heads * tiles)));
  const int step = (int)std::min<long long>(65535, seqs > 1 ? tiles : std::max<long long>(1, std::min(tiles, SCORES_MAX / (tile_bytes * c.heads))));
  const long long held = (long long)seqs * c.heads * std::min<long long>(step, tiles);
  char* ws;
  if (int r = decode_workspace(ctx, (size_t)(held * tile_bytes), &ws)) return r;
  a.scores = (uint8_t*)ws;
  a.hist = (unsigned*)(ws + held * tile_scores);
  a.sums = (int*)(ws + held * (tile_scores + tile_hist));
  for (a.seq0 = 0; a.seq0 < c.seqs; a.seq0 += seqs)
    for (long long t0 = 0; t0 < tiles; t0 += step) {
      a.tile0 = (int)t0, a.tiles = (int)std::min<long long>(tiles - t0, step);
      const unsigned n = (unsigned)(std::min(seqs, c.seqs - a.seq0) * c.heads);
      const dim3 grid(n, (unsigned)a.tiles, (unsigned)a.splits);
      if (int r = launch_lds(attend_scores_kernel<NG, RP>, grid, 64 * waves, 0, ctx, c, a)) return r;
      if (int r = launch_lds(attend_values_kernel<NG, RP, WIDE>, grid, 64 * waves, fixed + sums, ctx, c, a)) return r;
      ANVIL_LAUNCH(attend_join_kernel<NG>, dim3(n, (unsigned)a.tiles, (unsigned)(2 * NG * a.rows)), dim3(JOIN_THREADS), 0, ctx->stream, c,
                   a, waves);
      ANVIL_LAUNCHED();
    }
  return ANVIL_OK;
}

// Whether a head's row of O may share a byte with one of Q: where their extents meet, with row strides alike, each pair of heads
// settles it (modulo the stride), and strides that differ are taken to meet.
static bool rows_meet(const AttendArgs& a, int rows, int heads, int dim) {
  using wide = __int128;
  const wide apart = (wide)(uintptr_t)a.o - (wide)(uintptr_t)a.q, q_rows = (wide)a.q_row * (rows - 1), q_heads = (wide)a.q_head * (heads - 1),
             o_last = (wide)a.o_row * (rows - 1) + (wide)a.o_head * (heads - 1);
  if (apart >= std::max<wide>(q_rows, 0) + std::max<wide>(q_heads, 0) + dim ||
      apart + o_last + dim <= std::min<wide>(q_rows, 0) + std::min<wide>(q_heads, 0))
    return false;
  if (a.q_row != a.o_row || heads > 4096) return true;
  const wide row = a.o_row;                              // at least dim
  for (int ho = 0; ho < heads; ++ho)
    for (int hq = 0; hq < heads; ++hq) {
      const wide d = apart + (wide)ho * a.o_head - (wide)hq * a.q_head;
      wide k = d / row;
      k -= d < k * row;                                  // rounded down
      const wide rest = d - k * row;
      if ((rest < dim && k < rows && -k < rows) || (row - rest < dim && k + 1 < rows && -k - 1 < rows)) return true;
    }
  return false;
}

}  // namespace anvil

using namespace anvil;

extern "C" int anvil_attention_cache_i4(anvil_ctx* ctx, const anvil_cache* cache, int layer, const int8_t* Q, int8_t* O,
                                        const int32_t* starts, int rows, int max_new, int heads_q, const int64_t* strides,
                                        int32_t m_s, int s_s, const int32_t* lut, int32_t one, int32_t m_o, int s_o,
                                        int window, int sinks) {
  const char* who = "anvil_attention_cache_i4";
  CacheView c;
  if (int r = cache_view(who, ctx, cache, layer, starts, rows, max_new, &c)) return r;
  if (heads_q < 1 || heads_q % c.heads) return set_error(ANVIL_E_VALUE, "%s: %d query heads over %d", who, heads_q, c.heads);
  if (s_s < 0 || s_s > 31 || s_o < 0 || s_o > 31) return set_error(ANVIL_E_VALUE, "%s: shifts %d, %d outside [0, 31]", who, s_s, s_o);
  if (one < 1 || one > 32767) return set_error(ANVIL_E_VALUE, "%s: one = %d outside [1, 32767]", who, one);
  if (window < 0 || sinks < 0) return set_error(ANVIL_E_VALUE, "%s: window %d, sinks %d", who, window, sinks);
  if (!strides || !lut || (uintptr_t)lut % 4) return set_error(ANVIL_E_VALUE, "%s: strides or lut null or not aligned", who);
  const long long top = 128ll * 126 * c.dim * (m_s < 0 ? -(long long)m_s : m_s) + (s_s ? 1ll << (s_s - 1) : 0);
  if (top > INT32_MAX) return set_error(ANVIL_E_OVERFLOW, "%s: a score's requant with multiplier %d may leave int32", who, m_s);
  if ((long long)c.seqs * c.heads > 1 << 22 || (long long)c.max_new * (heads_q / c.heads) > 1 << 30)
    return set_error(ANVIL_E_VALUE, "%s: %d sequences of %d tokens, %d query heads over %d", who, c.seqs, c.max_new, heads_q, c.heads);
  if (!c.seqs || !rows) return check_ctx(ctx);
  if (!Q || !O || (uintptr_t)Q % 16 || (uintptr_t)O % 4) return set_error(ANVIL_E_VALUE, "%s: Q must be 16- and O 4-byte aligned", who);
  if (strides[0] % 16 || strides[1] % 16 || strides[2] % 4 || strides[3] % 4 || strides[2] < c.dim || strides[3] < c.dim)
    return set_error(ANVIL_E_VALUE, "%s: strides %lld, %lld, %lld, %lld", who, (long long)strides[0], (long long)strides[1],
                     (long long)strides[2], (long long)strides[3]);
  if (int r = check_ctx(ctx)) return r;
  AttendArgs a{};
  a.q = Q, a.o = O, a.q_row = strides[0], a.q_head = strides[1], a.o_row = strides[2], a.o_head = strides[3];
  a.lut = lut, a.m_s = m_s, a.s_s = s_s, a.one = one, a.m_o = m_o, a.s_o = s_o;
  if (rows_meet(a, rows, heads_q, c.dim))
    return set_error(ANVIL_E_VALUE, "%s: O overlaps Q, which other workgroups still read", who);
  const int most = c.slots * PAGE;                       // keys; a window that holds them all is none
  a.window = window < most ? window : 0, a.sinks = std::min(sinks, most), a.group = heads_q / c.heads;
  int r = ANVIL_OK;
  by_groups(c.dim, [&](auto ng) {
    constexpr int NG = decltype(ng)::value;
    const long long rows = (long long)c.max_new * a.group;
    if (rows <= 4 && one <= ONE_FIFTEEN) r = attend<NG, 4, false>(ctx, c, a);
    else if (rows <= 8) r = one <= ONE_NARROW ? attend<NG, 8, false>(ctx, c, a) : attend<NG, 8, true>(ctx, c, a);
    else r = one <= ONE_NARROW ? attend<NG, 16, false>(ctx, c, a) : attend<NG, 16, true>(ctx, c, a);
  });
  return r;
}
