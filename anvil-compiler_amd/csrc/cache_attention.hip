// Attention of the newest tokens over the 4-bit paged cache.
//
// Mathematics. softmax_lut's exponentials are table entries at x - max, so a maximum found later cannot rescale a sum that was
// begun; but a score is one of 256 values, and with the histogram of a row's scores its maximum, its sum and the probability of each
// value follow exactly. So a row is evaluated in two passes: its scores (one byte a key, kept) with their histogram, then a
// 256-entry table of probabilities and the sum of p V, looked up by score. K is read once, V once.
//
// Tiles. 16 rows share a pass over a cache head's keys: the query heads of its group, for one token or several. 64 keys (a page)
// are one step of a wave:
//   scores  v_mfma_i32_16x16x32_i8 for each 16 keys and group of 32 channels: keys x channels codes (their four bits in a byte's
//           upper half, so that no sign has to be extended: 16 x the product), channels x rows queries; times the key's step
//   values  v_mfma_i32_16x16x64_i8 for each 16 channels: channels x keys codes, keys x rows of p x step, which takes 12 to 20
//           bits and goes through as two or three 7-bit digits
// The operand row of key 16 q + 4 k + i in the k-th product is 4 q + i, so lane (row, q) receives the scores of keys 16 q .. 16 q + 15
// in order, which are the keys whose p it supplies to the second product: a lane reads back what it wrote, without a barrier.
#include <algorithm>

#include "cache.h"

namespace anvil {

struct AttendArgs {
  const int8_t* q;
  int8_t* o;
  long long q_row, q_head, o_row, o_head;
  const int* lut;
  int heads_q, m_s, s_s, one, m_o, s_o, window, sinks;
  int group, rows;                                       // query heads of a cache head; rows of a tile that can exist (<= 16)
  int seq0, tile0, tiles, splits, bound;                 // this launch's part; pages that a tile can see at most
  uint8_t* scores;                                       // workspace: [unit][tile][page][row][64], a score + 128
  unsigned* hist;                                        //            [unit][tile][split][row][256]
  int* sums;                                             //            [unit][tile][split][row][32 NG], 16 x sum p V
};

constexpr int WAVES = 4, ATTEND_THREADS = 64 * WAVES;
constexpr int HIST = 257;                                // dwords of a row's histogram in LDS: rows start in different banks

constexpr int ONE_TWO_DIGITS = ((1 << 14) - 1) / STEP_MAX;   // 910: p x step below 2^14

typedef unsigned short __attribute__((may_alias)) u16_alias;

// What a workgroup evaluates: the rows of one tile, and the pages that some row of it may see, numbered from 0 (first those of the
// sinks, then from the window's first page on).
struct Tile {
  NewRows r;
  int seq, head, unit, tile, rows, lo, hi;               // rows in use; positions of its first and last token
  int sink_pages, window_page, pages;
};

__device__ __forceinline__ bool find_tile(const CacheView& c, const AttendArgs& a, Tile& t) {
  t.unit = blockIdx.x, t.tile = (int)blockIdx.y;
  t.seq = a.seq0 + t.unit / c.heads, t.head = t.unit % c.heads;
  const int first = (a.tile0 + t.tile) * 16;
  new_rows(c, t.seq, t.r, first == 0 && blockIdx.z == 0 && t.head == 0 && threadIdx.x == 0);
  const long long all = (long long)t.r.n * a.group;
  if (first >= all) return false;
  t.rows = (int)min(16ll, all - first);
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

// whether every row of the tile sees every key of a page
__device__ __forceinline__ bool whole(const Tile& t, const AttendArgs& a, int slot) {
  const int first = slot * PAGE, last = first + PAGE - 1;
  return last <= t.lo && (!a.window || first > t.hi - a.window || last < a.sinks);
}

// One row as its lanes know it: row l % 16 of the tile.
struct Row {
  int pos, after, sinks;                                 // sees keys <= pos that are > after or < sinks
  bool on;
  __device__ __forceinline__ Row(const Tile& t, const AttendArgs& a, int r) {
    on = r < t.rows;
    pos = t.r.len - t.r.n + ((a.tile0 + t.tile) * 16 + r) / a.group;
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
template <int N>
__device__ __forceinline__ Words<N> load_words(const uint8_t* p) {
  Words<N> r;
  if constexpr (N == 1) {
    r.w[0] = *(const unsigned*)p;
  } else if constexpr (N == 2) {
    const uint2 v = *(const uint2*)p;
    r.w[0] = v.x, r.w[1] = v.y;
  } else {
    const uint4 v = *(const uint4*)p;
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  }
  return r;
}

// A lane's part of a page's keys: of 16 keys in each of four products the four bits of 8 channels a group, and the steps of the
// four keys whose scores it receives.
template <int NG>
struct KeyPage {
  Words<NG> code[4], step[4];
  __device__ __forceinline__ void load(const uint8_t* blk, int lane) {
    const int row = lane & 15, q = lane >> 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      code[k] = load_words<NG>(blk + Block<NG>::K + (16 * (row >> 2) + 4 * k + (row & 3)) * Block<NG>::ROW + 4 * q * NG);
      step[k] = load_words<NG>(blk + Block<NG>::K_STEPS + (4 * q + k) * 4 * NG);
    }
  }
};

// A lane's part of a page's values: 16 keys of two channels a group, and their steps.
template <int NG>
struct ValuePage {
  uint4 code[NG], step[NG];
  __device__ __forceinline__ void load(const uint8_t* blk, int lane) {
    const int row = lane & 15, q = lane >> 4;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      code[g] = *(const uint4*)(blk + Block<NG>::V + (16 * g + row) * PAGE + 16 * q);
      step[g] = *(const uint4*)(blk + Block<NG>::V_STEPS + PAGE * g + 16 * q);
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

// The lane's 16 scores of a page, a byte each, + 128. The products hold 16 x code: their sum is divided exactly.
template <int NG>
__device__ __forceinline__ uint4 score_page(const KeyPage<NG>& k, const long (&q)[NG], const Requant& rq) {
  unsigned out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int acc[4];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const unsigned w = k.code[i].w[g], st = k.step[i].w[g];
      const unsigned long low = (w << 4) & 0xF0F0F0F0u, high = w & 0xF0F0F0F0u;
      const v4i d = __builtin_amdgcn_mfma_i32_16x16x32_i8((long)(high << 32 | low), q[g], v4i{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int part = __mul24(d[e], (int)((st >> (8 * e)) & 255u));
        acc[e] = g ? acc[e] + part : part;
      }
    }
    int x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = med3i(__mul24(acc[e] >> 4, rq.m) + rq.rnd, rq.lo, rq.hi);
    out[i] = sra_pack4(x[0], x[1], x[2], x[3], rq.s) ^ 0x80808080u;
  }
  return {out[0], out[1], out[2], out[3]};
}

__device__ __forceinline__ unsigned word(const uint4& v, int i) { return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)); }

// The scores of a page into the row's histogram.
__device__ __forceinline__ void count_scores(unsigned* hist, const uint4& sc, unsigned mask) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (mask >> i & 1u) atomicAdd(&hist[(word(sc, i >> 2) >> (8 * (i & 3))) & 255u], 1u);
}

// acc[digit][16 channels] += digits of p x step times 16 x code over a page. The table holds 2 p, so that bit 0 of 2 p x step is 0
// and the low 7-bit digit is its low byte halved. Two digits (p <= 910): below 2^15, two keys a 16-bit packed product. Three:
// 24-bit products below 2^21.
template <int NG, int ND>
__device__ __forceinline__ void add_page(const ValuePage<NG>& v, const uint4& sc, const u16_alias* table, unsigned mask,
                                         v4i (&acc)[ND][2 * NG]) {
  unsigned p[8];                                         // 2 p of two keys each
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned w = word(sc, j >> 1) >> (16 * (j & 1));
    p[j] = table[w & 255u] | (unsigned)table[(w >> 8) & 255u] << 16;
  }
  if (mask != 0xFFFFu) {
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] &= (mask >> (2 * j) & 1u ? 0xFFFFu : 0u) | (mask >> (2 * j + 1) & 1u ? 0xFFFF0000u : 0u);
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    v4i digit[ND];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned st = word(v.step[g], i);
      if constexpr (ND == 2) {
        typedef unsigned short v2u __attribute__((ext_vector_type(2)));
        const unsigned s0 = __builtin_amdgcn_perm(0, st, 0x0c010c00u), s1 = __builtin_amdgcn_perm(0, st, 0x0c030c02u);
        const unsigned y0 = __builtin_bit_cast(unsigned, (v2u)(__builtin_bit_cast(v2u, p[2 * i]) * __builtin_bit_cast(v2u, s0)));
        const unsigned y1 = __builtin_bit_cast(unsigned, (v2u)(__builtin_bit_cast(v2u, p[2 * i + 1]) * __builtin_bit_cast(v2u, s1)));
        digit[0][i] = (int)(__builtin_amdgcn_perm(y1, y0, 0x06040200u) >> 1);
        digit[1][i] = (int)__builtin_amdgcn_perm(y1, y0, 0x07050301u);
      } else {
        unsigned y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[e] = (unsigned)__umul24((p[2 * i + (e >> 1)] >> (16 * (e & 1))) & 0xFFFFu, (st >> (8 * e)) & 255u);
        const unsigned b0 = pack4((int)y[0], (int)y[1], (int)y[2], (int)y[3]);
        const unsigned b1 = pack4((int)(y[0] >> 8), (int)(y[1] >> 8), (int)(y[2] >> 8), (int)(y[3] >> 8));
        const unsigned b2 = pack4((int)(y[0] >> 16), (int)(y[1] >> 16), (int)(y[2] >> 16), (int)(y[3] >> 16));
        digit[0][i] = (int)(b0 >> 1);
        digit[1][i] = (int)(b1 & 0x7F7F7F7Fu);
        digit[ND - 1][i] = (int)(b2 << 1 | (b1 >> 7 & 0x01010101u));
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      v4i code;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned w = word(v.code[g], i);
        code[i] = (int)((half ? w : w << 4) & 0xF0F0F0F0u);
      }
#pragma unroll
      for (int n = 0; n < ND; ++n)
        acc[n][2 * g + half] = __builtin_amdgcn_mfma_i32_16x16x64_i8(code, digit[n], acc[n][2 * g + half], 0, 0, 0);
    }
  }
}

// The query operand: lane (row, q) holds channels 8 q .. 8 q + 7 of each group.
template <int NG>
__device__ __forceinline__ void load_query(const CacheView& c, const AttendArgs& a, const Tile& t, int lane, long (&q)[NG]) {
  const int r = (a.tile0 + t.tile) * 16 + (lane & 15), ch = 8 * (lane >> 4);
  const int8_t* p = a.q + (long long)(t.r.first + r / a.group) * a.q_row + (long long)(t.head * a.group + r % a.group) * a.q_head + ch;
#pragma unroll
  for (int g = 0; g < NG; ++g) q[g] = (lane & 15) < t.rows && 32 * g + ch < c.dim ? *(const long*)(p + 32 * g) : 0;
}

// Pages begin + wave, begin + wave + WAVES, .. below end of a tile, one after the other: step(page, slot, block) for those that the
// table names, with `ahead` holding what load(block) of the next one returns, issued before step runs on this one. Table
// entries come 64 at a time, one a lane.
template <int NG, typename Page, typename Step>
__device__ __forceinline__ void walk(const CacheView& c, const Tile& t, int begin, int end, bool report, Step&& step) {
  const int lane = threadIdx.x & 63;
  const int first = begin + (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long stride = (long long)c.heads * Block<NG>::BYTES;
  const uint8_t* base = c.pool + (long long)t.head * Block<NG>::BYTES;
  for (int at = first; at < end; at += 64 * WAVES) {
    const int mine = at + lane * WAVES;
    int entry = -1;
    if (mine < end) entry = c.table[(long long)t.seq * c.slots + slot_of(t, mine)];
    if (entry >= c.pages || entry < -1) {
      if (report) raise_flag(c.flags, FLAG_CACHE);
      entry = -1;
    }
    const int n = min(64, (end - at + WAVES - 1) / WAVES);
    // a page that the table does not name reads page 0's bytes, which step never sees
    const auto fetch = [&](int i, Page& p) {
      const int e = __builtin_amdgcn_readlane(entry, i);
      p.load(base + max(e, 0) * stride, lane);
    };
    Page a, b;
    fetch(0, a);
    for (int i = 0; i < n; i += 2) {
      if (i + 1 < n) fetch(i + 1, b);
      if (__builtin_amdgcn_readlane(entry, i) >= 0) step(a, at + i * WAVES);
      if (i + 1 >= n) break;
      if (i + 2 < n) fetch(i + 2, a);
      if (__builtin_amdgcn_readlane(entry, i + 1) >= 0) step(b, at + (i + 1) * WAVES);
    }
  }
}

// From a row's histogram (counts of scores 4 lane .. 4 lane + 3, less 128) the lane's four probabilities, as pairs of 2 p: every
// operand is a whole number below 2^53, so double arithmetic is exact but for the quotient, which is put right by its remainder.
__device__ __forceinline__ uint2 probabilities(const uint4& count, const int* lut, int one, unsigned* flags) {
  const int lane = threadIdx.x & 63;
  const int mine = count.w ? 3 : (count.z ? 2 : (count.y ? 1 : (count.x ? 0 : -1)));
  const unsigned long long any = __ballot(mine >= 0);
  if (!any) return {0, 0};                               // the row sees nothing
  const int at = 63 - __builtin_clzll(any), top = 4 * at + __builtin_amdgcn_readlane(mine, at);
  int e[4];
  unsigned long long sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = 4 * lane + i;
    e[i] = x <= top ? max(0, lut[x - top + 255]) : 0;
    sum += (unsigned long long)e[i] * word(count, i);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if (!sum) {
    if (lane == 0) raise_flag(flags, FLAG_ZERODIV);
    return {0, 0};
  }
  const double S = (double)sum, half = (double)(sum >> 1), inv = 1.0 / S;
  unsigned p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double n = (double)e[i] * one + half;
    double k = __builtin_trunc(n * inv);
    const double rest = __builtin_fma(-k, S, n);
    k += rest < 0 ? -1.0 : (rest >= S ? 1.0 : 0.0);
    p[i] = 2u * (unsigned)k;
  }
  return {p[0] | p[1] << 16, p[2] | p[3] << 16};
}

// A wave's accumulators as 16 x sums of p V (modulo 2^32, in which the sum itself lies) into row-major int32.
template <int NG, int ND>
__device__ __forceinline__ void spill(const v4i (&acc)[ND][2 * NG], int* rows, int stride, int n_rows) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  if (r >= n_rows) return;
#pragma unroll
  for (int m = 0; m < 2 * NG; ++m) {
    v4i s;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      unsigned x = (unsigned)acc[0][m][e] + ((unsigned)acc[1][m][e] << 7);
      if constexpr (ND == 3) x += (unsigned)acc[ND - 1][m][e] << 14;
      s[e] = (int)x;
    }
    *(v4i*)(rows + r * stride + 16 * m + 4 * q) = s;
  }
}

// four results of a row from 16 x its sums
__device__ __forceinline__ unsigned finish4(const v4i& sum, const AttendArgs& a) {
  int o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const long long v = ((long long)(sum[e] >> 4) * a.m_o + round_term(a.s_o)) >> a.s_o;
    o[e] = v < -128 ? -128 : (v > 127 ? 127 : (int)v);
  }
  return pack4(o[0], o[1], o[2], o[3]);
}

__device__ __forceinline__ unsigned* out_word(const AttendArgs& a, const Tile& t, int r, int ch) {
  const int at = (a.tile0 + t.tile) * 16 + r;
  return (unsigned*)(a.o + (long long)(t.r.first + at / a.group) * a.o_row + (long long)(t.head * a.group + at % a.group) * a.o_head + ch);
}

// The sum over the workgroup's waves of what each holds, in LDS (`red`: WAVES x rows x stride), then f(row, channel, sum).
template <int NG, int ND, typename F>
__device__ __forceinline__ void join_waves(const v4i (&acc)[ND][2 * NG], int* red, const Tile& t, F&& f) {
  constexpr int STRIDE = 32 * NG + 4;
  const int wave = threadIdx.x >> 6;
  spill<NG, ND>(acc, red + wave * t.rows * STRIDE, STRIDE, t.rows);
  __syncthreads();
  for (int i = threadIdx.x; i < t.rows * 8 * NG; i += ATTEND_THREADS) {
    const int r = i / (8 * NG), ch = 4 * (i % (8 * NG));
    v4i s = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += *(const v4i*)(red + (w * t.rows + r) * STRIDE + ch);
    f(r, ch, s);
  }
}

// Both passes of a tile in one workgroup, its scores in LDS.
template <int NG, int ND>
__global__ __launch_bounds__(ATTEND_THREADS) void attend_tile_kernel(CacheView c, AttendArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  __shared__ int lut[256];
  Tile t;
  if (!find_tile(c, a, t)) return;
  unsigned* hist = lds;
  uint4* scores = (uint4*)(lds + (a.rows * HIST + 3) / 4 * 4);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
  const Row row(t, a, r);
  long query[NG];
  load_query<NG>(c, a, t, lane, query);
  lut[tid] = a.lut[tid];
  for (int i = tid; i < t.rows * HIST; i += ATTEND_THREADS) hist[i] = 0;
  __syncthreads();
  const Requant rq(a.m_s, a.s_s);
  walk<NG, KeyPage<NG>>(c, t, 0, t.pages, true, [&](const KeyPage<NG>& page, int at) {
    const uint4 sc = score_page<NG>(page, query, rq);
    const int slot = slot_of(t, at);
    if (!row.on) return;
    scores[(at * t.rows + r) * 4 + q] = sc;
    if (whole(t, a, slot)) count_scores(hist + r * HIST, sc, 0xFFFFu);
    else count_scores(hist + r * HIST, sc, row.mask(slot * PAGE + 16 * q));
  });
  __syncthreads();
  for (int i = wave; i < t.rows; i += WAVES) {           // the row's table takes its histogram's place
    unsigned* h = hist + i * HIST;
    const uint4 count = {h[4 * lane], h[4 * lane + 1], h[4 * lane + 2], h[4 * lane + 3]};
    const uint2 p = probabilities(count, lut, a.one, c.flags);
    h[2 * lane] = p.x;
    h[2 * lane + 1] = p.y;
  }
  __syncthreads();
  v4i acc[ND][2 * NG] = {};
  const u16_alias* table = (const u16_alias*)(hist + (row.on ? r : 0) * HIST);
  walk<NG, ValuePage<NG>>(c, t, 0, t.pages, false, [&](const ValuePage<NG>& page, int at) {
    const int slot = slot_of(t, at);
    const uint4 sc = scores[(at * t.rows + (row.on ? r : 0)) * 4 + q];
    add_page<NG, ND>(page, sc, table, whole(t, a, slot) ? 0xFFFFu : row.mask(slot * PAGE + 16 * q), acc);
  });
  __syncthreads();                                       // the scores have been read
  join_waves<NG, ND>(acc, (int*)scores, t, [&](int i, int ch, const v4i& s) {
    if (ch < c.dim) *out_word(a, t, i, ch) = finish4(s, a);
  });
}

// ---- one tile over several workgroups: scores and histograms, then sums, then their total

__device__ __forceinline__ void split_range(const Tile& t, const AttendArgs& a, int& begin, int& end) {
  const int per = max(2 * WAVES, (t.pages + a.splits - 1) / a.splits);
  begin = min((int)blockIdx.z * per, t.pages);
  end = min(begin + per, t.pages);
}

template <int NG>
__global__ __launch_bounds__(ATTEND_THREADS) void attend_scores_kernel(CacheView c, AttendArgs a) {
  __shared__ unsigned hist[16 * HIST];
  Tile t;
  if (!find_tile(c, a, t)) return;
  int begin, end;
  split_range(t, a, begin, end);
  if (begin >= end) return;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const Row row(t, a, r);
  long query[NG];
  load_query<NG>(c, a, t, lane, query);
  for (int i = tid; i < t.rows * HIST; i += ATTEND_THREADS) hist[i] = 0;
  __syncthreads();
  const Requant rq(a.m_s, a.s_s);
  const long long unit = (long long)t.unit * a.tiles + t.tile;
  uint4* scores = (uint4*)a.scores + unit * a.bound * a.rows * 4;
  walk<NG, KeyPage<NG>>(c, t, begin, end, true, [&](const KeyPage<NG>& page, int at) {
    const uint4 sc = score_page<NG>(page, query, rq);
    const int slot = slot_of(t, at);
    if (!row.on) return;
    scores[((long long)at * a.rows + r) * 4 + q] = sc;
    if (whole(t, a, slot)) count_scores(hist + r * HIST, sc, 0xFFFFu);
    else count_scores(hist + r * HIST, sc, row.mask(slot * PAGE + 16 * q));
  });
  __syncthreads();
  unsigned* out = a.hist + (unit * a.splits + blockIdx.z) * a.rows * 256;
  for (int i = tid; i < t.rows * 256; i += ATTEND_THREADS) out[i] = hist[(i >> 8) * HIST + (i & 255)];
}

template <int NG, int ND>
__global__ __launch_bounds__(ATTEND_THREADS) void attend_values_kernel(CacheView c, AttendArgs a) {
  __shared__ int lut[256];
  __shared__ __align__(16) unsigned tables[16 * HIST];
  __shared__ __align__(16) int red[WAVES * 16 * (32 * NG + 4)];
  Tile t;
  if (!find_tile(c, a, t)) return;
  int begin, end;
  split_range(t, a, begin, end);
  if (begin >= end) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
  const Row row(t, a, r);
  lut[tid] = a.lut[tid];
  __syncthreads();
  const long long unit = (long long)t.unit * a.tiles + t.tile;
  const int per = max(2 * WAVES, (t.pages + a.splits - 1) / a.splits), parts = (t.pages + per - 1) / per;
  for (int i = wave; i < t.rows; i += WAVES) {
    const uint4* h = (const uint4*)(a.hist + (unit * a.splits * a.rows + i) * 256) + lane;
    uint4 count = {0, 0, 0, 0};
    for (int p = 0; p < parts; ++p) {
      const uint4 x = h[(long long)p * a.rows * 64];
      count.x += x.x, count.y += x.y, count.z += x.z, count.w += x.w;
    }
    const uint2 p = probabilities(count, lut, a.one, c.flags);
    tables[i * HIST + 2 * lane] = p.x;
    tables[i * HIST + 2 * lane + 1] = p.y;
  }
  __syncthreads();
  v4i acc[ND][2 * NG] = {};
  const u16_alias* table = (const u16_alias*)(tables + (row.on ? r : 0) * HIST);
  const uint4* scores = (const uint4*)a.scores + unit * a.bound * a.rows * 4;
  walk<NG, ValuePage<NG>>(c, t, begin, end, false, [&](const ValuePage<NG>& page, int at) {
    const int slot = slot_of(t, at);
    const uint4 sc = scores[((long long)at * a.rows + (row.on ? r : 0)) * 4 + q];
    add_page<NG, ND>(page, sc, table, whole(t, a, slot) ? 0xFFFFu : row.mask(slot * PAGE + 16 * q), acc);
  });
  int* sums = a.sums + (unit * a.splits + blockIdx.z) * a.rows * 32 * NG;
  join_waves<NG, ND>(acc, red, t, [&](int i, int ch, const v4i& s) { *(v4i*)(sums + i * 32 * NG + ch) = s; });
}

template <int NG>
__global__ __launch_bounds__(ATTEND_THREADS) void attend_join_kernel(CacheView c, AttendArgs a) {
  Tile t;
  if (!find_tile(c, a, t)) return;
  const long long unit = (long long)t.unit * a.tiles + t.tile;
  const int per = max(2 * WAVES, (t.pages + a.splits - 1) / a.splits), parts = (t.pages + per - 1) / per;
  for (int i = threadIdx.x; i < t.rows * 8 * NG; i += ATTEND_THREADS) {
    const int r = i / (8 * NG), ch = 4 * (i % (8 * NG));
    if (ch >= c.dim) continue;
    const int* p = a.sums + (unit * a.splits * a.rows + r) * 32 * NG + ch;
    v4i s = {0, 0, 0, 0};
    for (int n = 0; n < parts; ++n) s += *(const v4i*)(p + (long long)n * a.rows * 32 * NG);
    *out_word(a, t, r, ch) = finish4(s, a);
  }
}

constexpr int TILE_LDS_MAX = 63 * 1024;                  // a tile's scores and histograms: two workgroups a CU
constexpr long long SCORES_MAX = 1ll << 30;              // bytes of scores in the workspace, unless one tile has more
constexpr int FILL = 512;                                // workgroups that fill the card

template <int NG, int ND>
static int attend(anvil_ctx* ctx, const CacheView& c, AttendArgs a, int max_new) {
  const long long all = (long long)max_new * a.group;    // rows of a cache head at most
  a.rows = (int)std::min(16ll, all);
  const long long tiles = (all + 15) / 16;
  const int tokens = (int)std::min<long long>(max_new, (a.rows - 1) / a.group + 2);
  a.bound = c.slots;
  if (a.window) {
    const long long seen = ((long long)a.window + tokens + PAGE - 2) / PAGE + 1 + (a.sinks + PAGE - 1) / PAGE;
    a.bound = (int)std::min<long long>(c.slots, seen);
  }
  const long long units = (long long)c.seqs * c.heads;
  const size_t lds = sizeof(int) * ((size_t)(a.rows * HIST + 3) / 4 * 4) +
                     std::max<size_t>((size_t)a.bound * a.rows * PAGE, sizeof(int) * WAVES * a.rows * (32 * NG + 4));
  const long long wanted = std::min<long long>((FILL + units * tiles - 1) / (units * tiles), (a.bound + 2 * WAVES - 1) / (2 * WAVES));
  a.splits = (int)std::max(1ll, wanted);
  if (a.splits == 1 && lds <= TILE_LDS_MAX) {
    for (long long t0 = 0; t0 < tiles; t0 += 65535) {    // a grid dimension's limit
      a.tile0 = (int)t0, a.tiles = (int)std::min<long long>(tiles - t0, 65535);
      ANVIL_LAUNCH((attend_tile_kernel<NG, ND>), dim3((unsigned)units, (unsigned)a.tiles), dim3(ATTEND_THREADS), lds, ctx->stream, c, a);
      ANVIL_LAUNCHED();
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
      ANVIL_LAUNCH(attend_scores_kernel<NG>, grid, dim3(ATTEND_THREADS), 0, ctx->stream, c, a);
      ANVIL_LAUNCHED();
      ANVIL_LAUNCH((attend_values_kernel<NG, ND>), grid, dim3(ATTEND_THREADS), 0, ctx->stream, c, a);
      ANVIL_LAUNCHED();
      ANVIL_LAUNCH(attend_join_kernel<NG>, dim3(n, (unsigned)a.tiles), dim3(ATTEND_THREADS), 0, ctx->stream, c, a);
      ANVIL_LAUNCHED();
    }
  return ANVIL_OK;
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
  if (!c.seqs || !rows) return check_ctx(ctx);
  if (!Q || !O || (uintptr_t)Q % 16 || (uintptr_t)O % 4) return set_error(ANVIL_E_VALUE, "%s: Q must be 16- and O 4-byte aligned", who);
  if (strides[0] % 16 || strides[1] % 16 || strides[2] % 4 || strides[3] % 4 || strides[2] < c.dim || strides[3] < c.dim)
    return set_error(ANVIL_E_VALUE, "%s: strides %lld, %lld, %lld, %lld", who, (long long)strides[0], (long long)strides[1],
                     (long long)strides[2], (long long)strides[3]);
  if (int r = check_ctx(ctx)) return r;
  AttendArgs a{};
  a.q = Q, a.o = O, a.q_row = strides[0], a.q_head = strides[1], a.o_row = strides[2], a.o_head = strides[3];
  a.lut = lut, a.heads_q = heads_q, a.m_s = m_s, a.s_s = s_s, a.one = one, a.m_o = m_o, a.s_o = s_o;
  const int most = c.slots * PAGE;                       // keys; a window that holds them all is none
  a.window = window < most ? window : 0, a.sinks = std::min(sinks, most), a.group = heads_q / c.heads;
  int r = ANVIL_OK;
  by_groups(c.dim, [&](auto ng) {
    constexpr int NG = decltype(ng)::value;
    r = one <= ONE_TWO_DIGITS ? attend<NG, 2>(ctx, c, a, max_new) : attend<NG, 3>(ctx, c, a, max_new);
  });
  return r;
}
