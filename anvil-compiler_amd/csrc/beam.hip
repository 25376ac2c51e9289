// Beam search's selection over beams and vocabulary from int8 logits.
//
// A logit is one of 256 values, so the histogram of a row gives its softmax's sum exactly, and the k-th best value of a stretch of
// it: above that value fewer than k tokens lie, and of those at it the first few in token order are taken. Each stretch of
// 16384 logits is read once into registers by one workgroup, which leaves its histogram and its k best; one workgroup a group then
// joins them. Rows of at most 4096 logits take a wave each of that last workgroup instead, in one launch.
//
// 64 x 8 rows of 100003 logits: 27 us of the stretches (12 of reading, 11 of counting, an LDS atomic a logit at 8.4 clocks a wave's, 5
// of collecting) and 8 of joining; 8 x 4 rows of 512: 8 us, most of it the launch and one chain.
#include "common.h"

namespace anvil {

constexpr long long NO_SCORE = INT64_MIN;
constexpr int WAVE_TOKENS = 4096;                        // 64 lanes x 4 blocks x 16 logits
constexpr int BLOCKS = WAVE_TOKENS / 1024;
constexpr int PART_WAVES = 4, PART_TOKENS = PART_WAVES * WAVE_TOKENS, PART_THREADS = 64 * PART_WAVES;
constexpr int PICK_WAVES = 8, PICK_THREADS = 64 * PICK_WAVES;
constexpr int VOCAB_MAX = 1 << 28;                       // 2^14 stretches
constexpr int KEEP_MAX = 64;                             // of beams too: one a lane

typedef unsigned long long u64;

// A candidate of a row: the logit + 128, then tokens ascending, as one number to be as large as possible; 0: none.
__device__ __forceinline__ u64 key_of(unsigned u, int token) { return (u64)u << 32 | ~(unsigned)token; }
__device__ __forceinline__ int token_of(u64 key) { return (int)~(unsigned)key; }

__device__ __forceinline__ uint4 load16(const void* p) {                         // at any alignment
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ unsigned word(const uint4& v, int i) { return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)); }
__device__ __forceinline__ unsigned byte(const uint4& v, int i) { return (word(v, i >> 2) >> (8 * (i & 3))) & 255u; }

// a byte by an index that the compiler does not know
__device__ __forceinline__ unsigned byte_at(const uint4& v, int i) {
  const unsigned x = v.x, y = v.y, z = v.z, w = v.w;     // values: of lvalues ?: selects an address, which keeps v in memory
  const unsigned a = i & 4 ? y : x, b = i & 4 ? w : z;
  return (i & 8 ? b : a) >> (8 * (i & 3)) & 255u;
}

template <int W>
__device__ __forceinline__ void together() {             // what the W waves of a stretch wrote to LDS is there
  if constexpr (W > 1) __syncthreads();
  else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// The want-th best of the values that a histogram counts, and how many lie above it; -1 and all of them where there are no more.
struct Edge {
  int value, higher;
  __device__ __forceinline__ Edge(const unsigned* hist, int want) {
    const int lane = threadIdx.x & 63;
    const uint4 c = ((const uint4*)hist)[lane];
    const int mine = (int)(c.x + c.y + c.z + c.w);
    const int upto = wave_scan(mine), all = __builtin_amdgcn_readlane(upto, 63);
    const int above = all - upto + mine;                 // of the lane's four values and higher ones
    value = -1, higher = all;
    if (higher <= want) return;
    int e = 3, h = above - mine;
#pragma unroll
    for (int i = 3; i > 0; --i) {
      const int n = (int)word(c, i);
      if (e == i && h + n < want) h += n, e = i - 1;
    }
    const int at = 63 - __builtin_clzll(__ballot(above >= want));
    value = 4 * at + __builtin_amdgcn_readlane(e, at), higher = __builtin_amdgcn_readlane(h, at);
  }
};

// What the W waves of a stretch share: counts of all values, of those of allowed tokens (near the best), and each wave's finds.
template <int W>
struct alignas(16) Shared {
  unsigned hist[256], fit[256];
  int high[W], equal[W];
};

// One wave's 4096 logits of a row, in registers, and its share of the stretch's `keep` best.
template <int W>
struct Stretch {
  uint4 u[BLOCKS];                                       // logits + 128; block b, lane l: tokens 1024 b + 16 l ..
  int have[BLOCKS];                                      // of them the row has
  unsigned valid[BLOCKS];                                // the same as `from` says it

  __device__ __forceinline__ Stretch(const int8_t* x, int n) {
    const int lane = threadIdx.x & 63;
    static_for<BLOCKS>([&](auto b) {
      const int at = 1024 * b + 16 * lane;
      have[b] = min(16, max(0, n - at));
      valid[b] = 0x0F0F0F0Fu;
      uint4 v = {0, 0, 0, 0};
      if (have[b] == 16) {
        v = load16(x + at);
      } else {
        unsigned w[4] = {0, 0, 0, 0};
        valid[b] = 0;
        for (int i = 0; i < have[b]; ++i) {
          const unsigned xi = (uint8_t)x[at + i];
          valid[b] |= 1u << (8 * (i & 3) + (i >> 2));
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] |= (i >> 2) == j ? xi << (8 * (i & 3)) : 0u;
        }
        v = {w[0], w[1], w[2], w[3]};
      }
      u[b] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
    });
  }

  __device__ __forceinline__ void count(unsigned* hist) const {
    static_for<BLOCKS>([&](auto b) {
      if (have[b] == 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) atomicAdd(&hist[byte(u[b], i)], 1u);
      } else {
        for (int i = 0; i < have[b]; ++i) {
          atomicAdd(&hist[byte_at(u[b], i)], 1u);
        }
      }
    });
  }

  // A bit for each of a block's tokens whose value is at least `least`: bit 8 i + j is token 4 j + i, so that four bytes at a time the
  // carry out of 7 bits and the eighth decide it. Tokens that the row has not are 0 bits.
  template <int b>
  __device__ __forceinline__ unsigned from(int least) const {
    const unsigned add = (0x80u - ((unsigned)least & 0x7Fu)) * 0x01010101u, upper = least >= 128 ? 0u : ~0u;
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned w = word(u[b], j), t = (w & 0x7F7F7F7Fu) + add;
      const unsigned ge = (w & t) | ((w | t) & upper);   // least >= 128: both bits, else one of them
      m |= (ge & 0x80808080u) >> (7 - j);
    }
    return least > 255 ? 0 : m & valid[b];
  }
  // the tokens of such a mask in order, a bit each
  static __device__ __forceinline__ unsigned in_order(unsigned m) {
    unsigned r = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) r |= (((m >> j & 0x01010101u) * 0x01020408u) >> 24 & 15u) << (4 * j);
    return r;
  }

  // The stretch's `keep` best allowed tokens into list (zeros where there are fewer), the waves' together. s.hist holds the counts.
  __device__ __forceinline__ void collect(Shared<W>& s, int wave, const uint8_t* allowed, int keep, int token0, u64* list) const {
    const int lane = threadIdx.x & 63;
    unsigned mask[BLOCKS];
    // with forbidden tokens the best 2 keep + 32 of all hold the best `keep` allowed ones, but for the rare row that is looked
    // through whole
    Edge edge(s.hist, allowed ? 2 * keep + 32 : keep);
    for (int least = max(edge.value, 0);; least = 0) {
      static_for<BLOCKS>([&](auto b) {
        mask[b] = from<b>(least);
        if (!allowed) return;
        for (unsigned todo = mask[b]; todo; todo &= todo - 1) {
          const int bit = __builtin_ctz(todo), i = 4 * (bit & 3) + (bit >> 3);
          if (allowed[1024 * b + 16 * lane + i]) atomicAdd(&s.fit[byte_at(u[b], i)], 1u);
          else mask[b] &= ~(1u << bit);
        }
      });
      if (!allowed) break;
      together<W>();
      const Edge fit(s.fit, keep);
      edge = fit;
      if (least == 0 || fit.higher >= keep || fit.value >= 0) break;
      together<W>();                                     // every wave has read the counts
      for (int i = threadIdx.x & (64 * W - 1); i < 256; i += 64 * W) s.fit[i] = 0;
      together<W>();
    }
    const int at_edge = edge.value < 0 ? 0 : keep - edge.higher;
    unsigned equal[BLOCKS];
    int highs = 0, equals = 0;
    static_for<BLOCKS>([&](auto b) {
      equal[b] = 0;
      if (edge.value >= 0 && __ballot(mask[b])) {
        const unsigned above = mask[b] & from<b>(edge.value + 1);
        equal[b] = mask[b] & ~above & from<b>(edge.value);
        mask[b] = above;
      }
      highs += __builtin_popcount(mask[b]), equals += __builtin_popcount(equal[b]);
    });
    int high_at = 0, equal_at = 0;                       // of the waves before this one
    if constexpr (W > 1) {
      const int high_sum = __builtin_amdgcn_readlane(wave_scan(highs), 63), equal_sum = __builtin_amdgcn_readlane(wave_scan(equals), 63);
      if (lane == 0) s.high[wave] = high_sum, s.equal[wave] = equal_sum;
      together<W>();
      for (int w = 0; w < wave; ++w) high_at += s.high[w], equal_at += s.equal[w];
    }
    if (wave == 0)
      for (int i = edge.higher + at_edge + lane; i < keep; i += 64) list[i] = 0;
    int h = high_at + wave_scan(highs) - highs;          // where the lane's higher ones go, in any order
    static_for<BLOCKS>([&](auto b) {
      for (unsigned todo = mask[b]; todo; todo &= todo - 1) {
        const int bit = __builtin_ctz(todo), i = 4 * (bit & 3) + (bit >> 3);
        list[h++] = key_of(byte_at(u[b], i), token0 + 1024 * b + 16 * lane + i);
      }
      const unsigned same = equal_at < at_edge ? equal[b] : 0;                   // those at the edge in token order
      if (!__ballot(same)) return;
      const int mine = __builtin_popcount(same), upto = wave_scan(mine);
      int e = equal_at + upto - mine;
      equal_at += __builtin_amdgcn_readlane(upto, 63);
      for (unsigned todo = in_order(same); todo && e < at_edge; todo &= todo - 1)
        list[edge.higher + e++] = key_of((unsigned)edge.value, token0 + 1024 * b + 16 * lane + __builtin_ctz(todo));
    });
  }
};

// 64 keys, one a lane, from the largest down
__device__ __forceinline__ u64 sort_down(u64 key) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int size = 2; size <= 64; size *= 2)
#pragma unroll
    for (int d = size / 2; d; d /= 2) {
      const u64 other = __shfl_xor(key, d);
      const bool larger = ((lane & d) == 0) == ((lane & size) == 0);
      key = larger ? max(key, other) : min(key, other);
    }
  return key;
}

// the largest 64 of two lists, each from the largest down
__device__ __forceinline__ u64 merge_down(u64 a, u64 b) {
  const int lane = threadIdx.x & 63;
  u64 key = max(a, (u64)__shfl(b, 63 - lane));
#pragma unroll
  for (int d = 32; d; d /= 2) {
    const u64 other = __shfl_xor(key, d);
    key = (lane & d) == 0 ? max(key, other) : min(key, other);
  }
  return key;
}

template <int CTRL>
__device__ __forceinline__ long long dpp_max(long long v) {
  const int lo = __builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false);
  const int hi = __builtin_amdgcn_update_dpp((int)(v >> 32), (int)(v >> 32), CTRL, 0xF, 0xF, false);
  return max(v, (long long)((u64)(unsigned)hi << 32 | (unsigned)lo));
}
__device__ __forceinline__ long long wave_max(long long v) {
  v = dpp_max<0xB1>(v);                                  // quad_perm [1,0,3,2]
  v = dpp_max<0x4E>(v);                                  // quad_perm [2,3,0,1]
  v = dpp_max<0x141>(v);                                 // row_half_mirror
  v = dpp_max<0x140>(v);                                 // row_mirror
  v = dpp_max<0x142>(v);                                 // row_bcast:15
  v = dpp_max<0x143>(v);                                 // row_bcast:31: lane 63 has seen all
  const unsigned lo = __builtin_amdgcn_readlane((int)v, 63), hi = __builtin_amdgcn_readlane((int)(v >> 32), 63);
  return (long long)((u64)hi << 32 | lo);
}

__device__ __forceinline__ long long log_fixed(const anvil_beams& b, u64 v) {
  int k = v < (u64)b.nlogs ? 0 : max(0, 64 - __builtin_clzll(v) - (32 - __builtin_clz((unsigned)b.nlogs)));
  while (v >> k >= (u64)b.nlogs) ++k;                    // bit lengths leave one step open
  return b.logs[v >> k] + (long long)k * b.step;
}

// What a wave knows of a row before its candidates: live (it has some of its own), ended, and from the row's counts (lane l:
// logits + 128 of 4 l .. 4 l + 3) what a candidate's score adds to logit * mult.
struct BeamRow {
  long long score, base;
  bool ended, live;
  __device__ __forceinline__ BeamRow(const anvil_beams& b, long long row) {
    score = b.scores[row];
    ended = score != NO_SCORE && b.ended && b.ended[row];
    live = score != NO_SCORE && !ended;
    base = score;
  }
  __device__ __forceinline__ void weigh(const anvil_beams& b, const unsigned (&count)[4], unsigned* flags) {
    const int lane = threadIdx.x & 63;
    const int mine = count[3] ? 3 : (count[2] ? 2 : (count[1] ? 1 : (count[0] ? 0 : -1)));
    const int at = 63 - __builtin_clzll(__ballot(mine >= 0) | 1ull), top = 4 * at + __builtin_amdgcn_readlane(mine, at);
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * lane + i <= top) sum += (u64)max(0, b.lut[4 * lane + i - top + 255]) * count[i];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    const int one = b.lut[255];
    if (live && (sum < 1 || one < 1)) {
      if (lane == 0) raise_flag(flags, FLAG_ZERODIV);
      live = false;
    }
    if (live) base = score - (long long)(top - 128) * b.mult - (log_fixed(b, sum) - log_fixed(b, (u64)one));
  }
};

// The group's best of its rows' sorted lists, by one wave: lane l walks row l's.
__device__ __forceinline__ void pick(const anvil_beams& b, int group, const u64* lists, const long long* bases) {
  const int lane = threadIdx.x & 63;
  int at = 0;
  u64 key = lane < b.beams ? lists[lane * b.keep] : 0;
  const long long base = lane < b.beams ? bases[lane] : 0, row = (long long)group * b.beams + lane;
  const bool ended = lane < b.beams && b.ended && b.ended[row];
  for (int n = 0; n < b.keep; ++n) {
    const long long score = key ? base + (long long)((int)(key >> 32) - 128) * b.mult : NO_SCORE;
    const long long best = wave_max(score), out = (long long)group * b.keep + n;
    if (best == NO_SCORE) {                              // nothing left
      if (lane == 0) b.scores_out[out] = NO_SCORE, b.parent[out] = -1, b.token[out] = -1, b.ended_out[out] = 0;
      continue;
    }
    if (lane == __builtin_ctzll(__ballot(score == best))) {
      const int token = token_of(key);
      b.scores_out[out] = best, b.parent[out] = (int)row, b.token[out] = token, b.ended_out[out] = ended || token == b.eos;
      key = ++at < b.keep ? lists[lane * b.keep + at] : 0;
    }
  }
}

// One stretch of a row a workgroup (blockIdx: row, stretch).
__global__ __launch_bounds__(PART_THREADS) void beam_part_kernel(anvil_beams b, u64* lists, unsigned* hists, int parts) {
  __shared__ Shared<PART_WAVES> s;
  const long long row = blockIdx.x;
  const int part = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
  const int token0 = part * PART_TOKENS + wave * WAVE_TOKENS;
  const Stretch<PART_WAVES> x(b.logits + row * b.ld + token0, b.vocab - token0);
  const BeamRow r(b, row);
  if (!r.live) return;                                   // the joining workgroup does not read its lists
  s.hist[tid] = 0, s.fit[tid] = 0;
  __syncthreads();
  x.count(s.hist);
  __syncthreads();
  hists[(row * parts + part) * 256 + tid] = s.hist[tid];
  x.collect(s, wave, b.allowed ? b.allowed + token0 : nullptr, b.keep, token0, lists + (row * parts + part) * b.keep);
}

// One group a workgroup, a wave a row: its stretches' histograms and lists joined, then the rows'.
__global__ __launch_bounds__(PICK_THREADS) void beam_join_kernel(anvil_beams b, const u64* lists, const unsigned* hists, int parts,
                                                                 unsigned* flags) {
  __shared__ u64 sorted[KEEP_MAX * KEEP_MAX];
  __shared__ long long bases[KEEP_MAX];
  const int group = blockIdx.x, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  for (int i = threadIdx.x >> 6; i < b.beams; i += waves) {
    const long long row = (long long)group * b.beams + i;
    BeamRow r(b, row);
    u64 key = 0;
    if (r.live) {
      const long long n = (long long)parts * b.keep;
      const u64* all = lists + row * n;
      u64 next = lane < n ? all[lane] : 0;               // on its way beside the histograms
      unsigned count[4] = {0, 0, 0, 0};
      for (int p = 0; p < parts; p += 8) {
        uint4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          x[k] = {0, 0, 0, 0};
          if (p + k < parts) x[k] = ((const uint4*)(hists + (row * parts + p + k) * 256))[lane];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) count[0] += x[k].x, count[1] += x[k].y, count[2] += x[k].z, count[3] += x[k].w;
      }
      r.weigh(b, count, flags);
      if (r.live) {
        for (long long at = 64;; at += 64) {
          const u64 now = sort_down(next);
          key = at > 64 ? merge_down(key, now) : now;
          if (at >= n) break;
          next = at + lane < n ? all[at + lane] : 0;
        }
      }
    } else if (r.ended && lane == 0) {
      key = key_of(128, b.eos);                          // a logit of 0: its own score
    }
    if (lane < b.keep) sorted[i * b.keep + lane] = key;
    if (lane == 0) bases[i] = r.base;
  }
  __syncthreads();
  if (threadIdx.x < 64) pick(b, group, sorted, bases);
}

// Rows of at most WAVE_TOKENS logits: one group a workgroup, a wave a row, in one launch.
__global__ __launch_bounds__(PICK_THREADS) void beam_small_kernel(anvil_beams b, unsigned* flags) {
  __shared__ u64 sorted[KEEP_MAX * KEEP_MAX];
  __shared__ long long bases[KEEP_MAX];
  __shared__ Shared<1> shared[PICK_WAVES];
  const int group = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  Shared<1>& s = shared[wave];
  for (int i = wave; i < b.beams; i += waves) {
    const long long row = (long long)group * b.beams + i;
    BeamRow r(b, row);
    u64* list = sorted + i * b.keep;
    u64 key = 0;
    if (r.live) {
      const Stretch<1> x(b.logits + row * b.ld, b.vocab);
      for (int j = lane; j < 256; j += 64) s.hist[j] = 0, s.fit[j] = 0;
      together<1>();
      x.count(s.hist);
      together<1>();
      const uint4 c = ((const uint4*)s.hist)[lane];
      const unsigned count[4] = {c.x, c.y, c.z, c.w};
      x.collect(s, 0, b.allowed, b.keep, 0, list);
      together<1>();
      r.weigh(b, count, flags);
      if (r.live) key = sort_down(lane < b.keep ? list[lane] : 0);
      together<1>();
    }
    if (r.ended && lane == 0) key = key_of(128, b.eos);
    if (lane < b.keep) list[lane] = key;
    if (lane == 0) bases[i] = r.base;
  }
  __syncthreads();
  if (threadIdx.x < 64) pick(b, group, sorted, bases);
}

}  // namespace anvil

using namespace anvil;

extern "C" int anvil_beam_select_i8(anvil_ctx* ctx, const anvil_beams* b) {
  const char* who = "anvil_beam_select_i8";
  if (!b) return set_error(ANVIL_E_VALUE, "%s: null arguments", who);
  if (b->groups < 0 || b->beams < 1 || b->beams > KEEP_MAX || (long long)b->groups * b->beams > 1 << 22 || b->keep < 1 ||
      b->keep > KEEP_MAX || b->vocab < 1 || b->vocab > VOCAB_MAX || b->ld < b->vocab)
    return set_error(ANVIL_E_VALUE, "%s: %d groups of %d beams, %d kept, vocabulary %d, row stride %lld", who, b->groups,
                     b->beams, b->keep, b->vocab, (long long)b->ld);
  if (b->nlogs < 2 || b->mult < 1 || b->step < 0)
    return set_error(ANVIL_E_VALUE, "%s: %d logs, step %d, mult %d", who, b->nlogs, b->step, b->mult);
  if (b->eos < -1 || b->eos >= b->vocab || (b->ended && b->eos < 0))
    return set_error(ANVIL_E_VALUE, "%s: eos %d of %d (ended rows need one)", who, b->eos, b->vocab);
  if (!b->groups) return check_ctx(ctx);
  if (!b->logits || !b->scores || !b->lut || !b->logs || !b->scores_out || !b->parent || !b->token || !b->ended_out)
    return set_error(ANVIL_E_VALUE, "%s: null pointer", who);
  if ((uintptr_t)b->scores % 8 || (uintptr_t)b->scores_out % 8 || (uintptr_t)b->lut % 4 || (uintptr_t)b->logs % 4 ||
      (uintptr_t)b->parent % 4 || (uintptr_t)b->token % 4)
    return set_error(ANVIL_E_VALUE, "%s: a pointer is not aligned to its type", who);
  const auto apart = [](const void* a, size_t na, const void* b, size_t nb) {
    return (uintptr_t)a + na <= (uintptr_t)b || (uintptr_t)b + nb <= (uintptr_t)a;
  };
  const size_t in = (size_t)b->groups * b->beams, out = (size_t)b->groups * b->keep;
  const void* const read[2] = {b->scores, b->ended};
  void* const written[4] = {b->scores_out, b->parent, b->token, b->ended_out};
  const size_t size[4] = {8, 4, 4, 1};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 2; ++j)                          // a group's rows are read while another's results are written
      if (read[j] && !apart(read[j], in * (j ? 1 : 8), written[i], out * size[i]))
        return set_error(ANVIL_E_VALUE, "%s: the results overlap the scores or ended rows that are read", who);
  if (int r = check_ctx(ctx)) return r;
  const unsigned pick_threads = 64u * (unsigned)(b->beams < PICK_WAVES ? b->beams : PICK_WAVES);
  if (b->vocab <= WAVE_TOKENS) {
    ANVIL_LAUNCH(beam_small_kernel, dim3((unsigned)b->groups), dim3(pick_threads), 0, ctx->stream, *b, ctx->flags);
    ANVIL_LAUNCHED();
    return ANVIL_OK;
  }
  const long long rows = (long long)b->groups * b->beams;
  const int parts = (b->vocab + PART_TOKENS - 1) / PART_TOKENS;
  const long long bytes = rows * parts * 1024;           // histograms; as many lists of at most half the size follow
  char* ws;
  if (int r = decode_workspace(ctx, (size_t)(bytes + rows * parts * b->keep * 8), &ws)) return r;
  ANVIL_LAUNCH(beam_part_kernel, dim3((unsigned)rows, (unsigned)parts), dim3(PART_THREADS), 0, ctx->stream, *b, (u64*)(ws + bytes),
               (unsigned*)ws, parts);
  ANVIL_LAUNCHED();
  ANVIL_LAUNCH(beam_join_kernel, dim3((unsigned)b->groups), dim3(pick_threads), 0, ctx->stream, *b, (const u64*)(ws + bytes),
               (const unsigned*)ws, parts, ctx->flags);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
