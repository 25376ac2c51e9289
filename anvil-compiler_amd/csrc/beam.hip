// Beam search's selection over beams and vocabulary from int8 logits.
//
// A logit is one of 256 values, so the histogram of a row gives its softmax's sum exactly, and the k-th best value of a stretch of
// it: above that value fewer than k tokens lie, and of those at it the first few in token order are taken. Each stretch of
// 16384 logits is read once into registers by one workgroup, which leaves its histogram and its k best; one workgroup a group then
// joins them. Rows of at most 4096 logits take a wave each of that last workgroup instead, in one launch.
#include "common.h"

namespace anvil {

constexpr long long NO_SCORE = INT64_MIN;
constexpr int WAVE_TOKENS = 4096;                        // 64 lanes x 4 blocks x 16 logits
constexpr int BLOCKS = WAVE_TOKENS / 1024;
constexpr int PART_WAVES = 4, PART_TOKENS = PART_WAVES * WAVE_TOKENS, PART_THREADS = 64 * PART_WAVES;
constexpr int PICK_WAVES = 16, PICK_THREADS = 64 * PICK_WAVES;
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

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// One wave's 4096 logits of a row: registers, histogram, and its share of the stretch's k best. W waves share a stretch, each with a
// histogram of its own (counts of a value below, of its allowed tokens above bit 16).
template <int W>
struct Stretch {
  uint4 u[BLOCKS];                                       // logits + 128; block b, lane l: tokens 1024 b + 16 l ..
  unsigned mask[BLOCKS];                                 // allowed ones

  __device__ __forceinline__ void count(const int8_t* x, const uint8_t* allowed, int n, unsigned* hist) {
    const int lane = threadIdx.x & 63;
    for (int i = lane; i < 256; i += 64) hist[i] = 0;
    int have[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const int at = 1024 * b + 16 * lane;
      have[b] = min(16, max(0, n - at));
      uint4 v = {0, 0, 0, 0};
      unsigned m = (1u << have[b]) - 1u;
      if (have[b] == 16) {
        v = load16(x + at);
        if (allowed) {
          const uint4 ok = load16(allowed + at);
          m = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) m |= (byte(ok, i) ? 1u : 0u) << i;
        }
      } else {
        unsigned w[4] = {0, 0, 0, 0};
        for (int i = 0; i < have[b]; ++i) {
          const unsigned xi = (uint8_t)x[at + i];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] |= (i >> 2) == j ? xi << (8 * (i & 3)) : 0u;
          if (allowed && !allowed[at + i]) m &= ~(1u << i);
        }
        v = {w[0], w[1], w[2], w[3]};
      }
      u[b] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
      mask[b] = m;
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < have[b]) atomicAdd(&hist[byte(u[b], i)], 1u + ((mask[b] >> i & 1u) << 16));
  }

  // The wave's share of the `keep` best of all W waves' tokens into list (keep entries, cleared where there are fewer).
  __device__ __forceinline__ void collect(const unsigned* hists, int wave, int keep, int token0, u64* list) const {
    const int lane = threadIdx.x & 63;
    int c[4], lane_sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) c[i] += hists[256 * w + 4 * lane + i] >> 16;
      lane_sum += c[i];
    }
    int above = lane_sum;                                // allowed tokens of this lane's values and higher ones
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int y = __shfl_down(above, d);
      if (lane + d < 64) above += y;
    }
    const int all = __builtin_amdgcn_readfirstlane(above);
    int edge = -1, higher = all;                         // the k-th best value, and how many lie above it
    if (all > keep) {
      int e = 0, h = above - lane_sum;
      bool found = false;
#pragma unroll
      for (int i = 3; i >= 0; --i)
        if (!found) {
          if (h + c[i] >= keep) found = true, e = 4 * lane + i;
          else h += c[i];
        }
      const int at = 63 - __builtin_clzll(__ballot(above >= keep));
      edge = __builtin_amdgcn_readlane(e, at), higher = __builtin_amdgcn_readlane(h, at);
    }
    int high_at = 0, edge_at = 0;                        // of the waves before this one
    if constexpr (W > 1) {
      int before = 0;
      for (int w = 0; w < wave; ++w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) before += 4 * lane + i > edge ? (int)(hists[256 * w + 4 * lane + i] >> 16) : 0;
        if (edge >= 0) edge_at += hists[256 * w + edge] >> 16;
      }
      high_at = wave_sum(before);
    }
    const int at_edge = edge < 0 ? 0 : keep - higher;
    if (wave == 0)
      for (int i = higher + at_edge + lane; i < keep; i += 64) list[i] = 0;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      unsigned high = 0, equal = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int v = (int)byte(u[b], i);
        high |= (v > edge ? 1u : 0u) << i;
        equal |= (v == edge ? 1u : 0u) << i;
      }
      high &= mask[b], equal &= edge_at < at_edge ? mask[b] : 0;
      if (!__ballot(high | equal)) continue;
      const int mine = __builtin_popcount(high) | __builtin_popcount(equal) << 16;
      int sum = mine;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(sum, d);
        if (lane >= d) sum += y;
      }
      int h = high_at + ((sum - mine) & 0xFFFF), e = edge_at + ((sum - mine) >> 16);
      const int total = __builtin_amdgcn_readlane(sum, 63);
      high_at += total & 0xFFFF, edge_at += total >> 16;
      for (unsigned todo = high | equal; todo; todo &= todo - 1) {
        const int i = __builtin_ctz(todo);
        const unsigned v = i < 8 ? (i < 4 ? u[b].x : u[b].y) : (i < 12 ? u[b].z : u[b].w);
        const u64 key = key_of(v >> (8 * (i & 3)) & 255u, token0 + 1024 * b + 16 * lane + i);
        if (high >> i & 1u) list[h++] = key;
        else if (e < at_edge) list[higher + e++] = key;
      }
    }
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
  __shared__ unsigned hist[PART_WAVES * 256];
  const long long row = blockIdx.x;
  const int part = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
  const BeamRow r(b, row);
  if (!r.live) return;                                   // the joining workgroup does not read its lists
  const int token0 = part * PART_TOKENS + wave * WAVE_TOKENS;
  Stretch<PART_WAVES> s;
  s.count(b.logits + row * b.ld + token0, b.allowed ? b.allowed + token0 : nullptr, b.vocab - token0, hist + 256 * wave);
  __syncthreads();
  s.collect(hist, wave, b.keep, token0, lists + (row * parts + part) * b.keep);
  unsigned sum = 0;
#pragma unroll
  for (int w = 0; w < PART_WAVES; ++w) sum += hist[256 * w + tid] & 0xFFFFu;
  hists[(row * parts + part) * 256 + tid] = sum;
}

// One group a workgroup, a wave a row: its stretches' histograms and lists joined, then the rows'.
__global__ __launch_bounds__(PICK_THREADS) void beam_join_kernel(anvil_beams b, const u64* lists, const unsigned* hists, int parts,
                                                                 unsigned* flags) {
  __shared__ u64 sorted[KEEP_MAX * KEEP_MAX];
  __shared__ long long bases[KEEP_MAX];
  const int group = blockIdx.x, lane = threadIdx.x & 63;
  for (int i = threadIdx.x >> 6; i < b.beams; i += PICK_WAVES) {
    const long long row = (long long)group * b.beams + i;
    BeamRow r(b, row);
    u64 key = 0;
    if (r.live) {
      unsigned count[4] = {0, 0, 0, 0};
      for (int p = 0; p < parts; ++p) {
        const uint4 x = ((const uint4*)(hists + (row * parts + p) * 256))[lane];
        count[0] += x.x, count[1] += x.y, count[2] += x.z, count[3] += x.w;
      }
      r.weigh(b, count, flags);
    }
    if (r.live) {
      const long long n = (long long)parts * b.keep;
      for (long long at = 0; at < n; at += 64) {
        const u64 next = sort_down(at + lane < n ? lists[row * n + at + lane] : 0);
        key = at ? merge_down(key, next) : next;
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
  __shared__ unsigned hists[PICK_WAVES * 256];
  const int group = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned* hist = hists + 256 * wave;
  for (int i = wave; i < b.beams; i += PICK_WAVES) {
    const long long row = (long long)group * b.beams + i;
    BeamRow r(b, row);
    u64* list = sorted + i * b.keep;
    u64 key = 0;
    if (r.live) {
      Stretch<1> s;
      s.count(b.logits + row * b.ld, b.allowed, b.vocab, hist);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      s.collect(hist, 0, b.keep, 0, list);
      unsigned count[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) count[j] = hist[4 * lane + j] & 0xFFFFu;
      r.weigh(b, count, flags);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      if (r.live) key = sort_down(lane < b.keep ? list[lane] : 0);
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
  if (b->groups < 0 || b->groups > (1 << 24) || b->beams < 1 || b->beams > 64 || b->keep < 1 || b->keep > 64 || b->vocab < 1 || b->vocab > VOCAB_MAX ||
      b->ld < b->vocab)
    return set_error(ANVIL_E_VALUE, "%s: %d groups of %d beams, %d kept, vocabulary %d, row stride %lld", who, b->groups,
                     b->beams, b->keep, b->vocab, (long long)b->ld);
  if (b->nlogs < 2 || b->mult < 1 || b->step < 0) return set_error(ANVIL_E_VALUE, "%s: %d logs, step %d, mult %d", who, b->nlogs, b->step, b->mult);
  if (b->eos < -1 || b->eos >= b->vocab || (b->ended && b->eos < 0))
    return set_error(ANVIL_E_VALUE, "%s: eos %d of %d (ended rows need one)", who, b->eos, b->vocab);
  if (!b->groups) return check_ctx(ctx);
  if (!b->logits || !b->scores || !b->lut || !b->logs || !b->scores_out || !b->parent || !b->token || !b->ended_out)
    return set_error(ANVIL_E_VALUE, "%s: null pointer", who);
  if ((uintptr_t)b->scores % 8 || (uintptr_t)b->scores_out % 8 || (uintptr_t)b->lut % 4 || (uintptr_t)b->logs % 4 ||
      (uintptr_t)b->parent % 4 || (uintptr_t)b->token % 4)
    return set_error(ANVIL_E_VALUE, "%s: a pointer is not aligned to its type", who);
  if (int r = check_ctx(ctx)) return r;
  if (b->vocab <= WAVE_TOKENS) {
    ANVIL_LAUNCH(beam_small_kernel, dim3((unsigned)b->groups), dim3(PICK_THREADS), 0, ctx->stream, *b, ctx->flags);
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
  ANVIL_LAUNCH(beam_join_kernel, dim3((unsigned)b->groups), dim3(PICK_THREADS), 0, ctx->stream, *b, (const u64*)(ws + bytes),
               (const unsigned*)ws, parts, ctx->flags);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
