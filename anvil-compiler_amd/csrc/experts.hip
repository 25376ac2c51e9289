// The router of an experts' feed-forward and the way back: each row's best experts and their weights, the rows sorted by expert,
// and the weighted sums of their results.
//
// Route. Sixteen lanes take a row (64 of many experts or choices), so that its maxima are four data-parallel moves: the j-th choice is the
// largest key below the one before.
// Sorting. Workgroups count their rows' pairs by expert; the rows of counts meet in a second launch, where every workgroup adds up all of
// them and those before its own, and places its pairs. Within a workgroup the waves own runs of consecutive pairs, and a pair's
// rank among the 64 of a step is the number of lower lanes with its expert (ballots over the bits of its number). Atomics add counts, none
// decides an order: positions are the same each time. 32749 rows, six of 64 experts each: 7.2 + 8.0 us for 5 MB, chains of reductions and of
// waits for counts, not bandwidth.
#include <algorithm>

#include "experts.h"

namespace anvil {

// Rows of a workgroup, at least, and workgroups, at most: each reads the counts of all. 4096 rows over 8 (two each), 64
// (six) and 256 experts (eight) take 9.6, 9.6 and 12.8 us with 32 rows, 11.0, 13.0 and 20.4 with 128. 32768 rows
// over 64: 14.4 us by 256 workgroups, 20.4 by 128, 24.8 by 512.
constexpr int ROUTE_ROWS = 32, ROUTE_BLOCKS = 256;
// Rows that one workgroup routes and sorts by itself: 64 rows over 8, 64 and 256 experts take it 5.8, 6.7 and 9.7 us, 128 rows 6.8, 8.6 and
// 14.2; two launches take 128 rows in 8.9, 8.9 and 9.9.
constexpr int ROUTE_ONE = 64;

// Rows of a workgroup that take sixteen waves, not eight: 32768 rows over 8, 64, 256 and 1024 experts (four each) take 12.3, 14.8, 25.0 and
// 73 us with them, 12.0, 15.9, 27.6 and 99 with eight.
constexpr int ROUTE_WIDE = 64;

struct RouteArgs {
  anvil_route r;
  int* counts;                                           // blocks x experts
  int blocks, block_rows;
  unsigned* flags;
};

// (e one + S / 2) / S of e <= 2^31 - 1, one <= 2^15 - 1, at most 32767: single precision is off by less than 1 / 50 of one, the remainder
// shows by which way
__device__ __forceinline__ int share(long long e, int one, long long S) {
  const long long num = e * one + S / 2;
  int q = (int)((float)num * __builtin_amdgcn_rcpf((float)S));
  const long long left = num - q * S;
  q += left < 0 ? -1 : left >= S ? 1 : 0;
  return q;
}

// sums over aligned groups of L lanes
template <int L>
__device__ __forceinline__ long long group_sum(long long v) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// A row's choices by L lanes, PER experts a lane (lane `sub` of them has experts sub, sub + L, ...): lane j's expert and weight of choice j.
// A key is the score with the expert's number below it, turned round, so keys differ and the order of ties is theirs.
template <int L, int PER>
__device__ __forceinline__ void choose(const RouteArgs& g, long long row, int sub, bool live, int& expert, int& weight) {
  const anvil_route& r = g.r;
  int key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = sub + L * i;
    key[i] = e < r.experts ? (int)r.scores[row * r.ld + e] * 1024 + (1023 - e) : INT32_MIN;
  }
  int best = INT32_MAX, mine = 0, top = 0;
  for (int j = 0; j < r.top; ++j) {                      // the largest key below the one before
    int m = INT32_MIN;
#pragma unroll
    for (int i = 0; i < PER; ++i) m = max(m, key[i] < best ? key[i] : INT32_MIN);
    best = lane_group_max<L>(m);
    if (j == 0) top = best >> 10;
    if (sub == j) mine = best;
  }
  const long long e = sub < r.top ? max(0, r.lut[(mine >> 10) - top + 255]) : 0;
  long long S = e;
  if (r.flags & ANVIL_ROUTE_EVERY) {
    S = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (sub + L * i < r.experts) S += max(0, r.lut[(key[i] >> 10) - top + 255]);
  }
  S = group_sum<L>(S);
  if (!live) return;
  expert = 1023 - (mine & 1023);
  weight = S ? share(e, r.one, S) : 0;
  if (!S && sub == 0) raise_flag(g.flags, FLAG_ZERODIV);
}

// Experts and weights of rows first .. first + n - 1, by the whole workgroup: also into pairs (n x top) unless null, counted by expert.
template <int L, int PER>
__device__ __forceinline__ void choose_rows(const RouteArgs& g, long long first, int n, int* pairs, int* count) {
  const anvil_route& r = g.r;
  const int sub = threadIdx.x & (L - 1), at = threadIdx.x / L, step = blockDim.x / L;
  for (int i0 = 0; i0 < n; i0 += step) {                 // whole waves: the reductions need every lane
    const int i = i0 + at;
    const long long row = first + min(i, n - 1);
    int expert = -1, weight = 0;
    const bool live = i < n && (!r.live || r.live[row]);
    choose<L, PER>(g, row, sub, live, expert, weight);
    if (i < n && sub < r.top) {
      r.expert[row * r.top + sub] = expert;
      r.weight[row * r.top + sub] = (int16_t)weight;
      if (pairs) pairs[i * r.top + sub] = expert;
      if (live) atomicAdd(&count[expert], 1);
    }
  }
}

// The pairs 0 .. n - 1 of `expert` that the calling wave owns, 64 a step: f(pair or -1, expert or -1, rank among this step's lower lanes
// of the same expert, whether it is the expert's last lane, how many it has)
template <typename F>
__device__ __forceinline__ void for_pairs(const int* expert, int n, int lane, F&& f) {
  for (int i = 0; i < n; i += 64) {
    const bool in = i + lane < n;
    const int e = in ? expert[i + lane] : -1;
    unsigned long long same = __ballot(e >= 0);
    for (int b = 0; b < 10; ++b) {
      const unsigned long long set = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1)), all = __popcll(same);
    f(in ? i + lane : -1, e, rank, rank == all - 1, all);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// Positions of a workgroup's pairs first .. first + n - 1, whose experts are expert[0 .. n - 1]. base[e]: the position of its
// first pair of expert e; at: a row of experts ints a wave, zeros.
__device__ __forceinline__ void place_pairs(const anvil_route& r, const int* expert, long long first, int n, const int* base, int* at) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int run = (n + waves - 1) / waves;
  const int lo = min(n, wave * run), hi = min(n, lo + run);
  int* mine = at + wave * r.experts;
  for_pairs(expert + lo, hi - lo, lane, [&](int, int e, int, bool last, int all) {
    if (e >= 0 && last) mine[e] += all;
  });
  __syncthreads();
  for (int e = threadIdx.x; e < r.experts; e += blockDim.x) {
    int p = base[e];
    for (int w = 0; w < waves; ++w) {
      const int c = at[w * r.experts + e];
      at[w * r.experts + e] = p;
      p += c;
    }
  }
  __syncthreads();
  for_pairs(expert + lo, hi - lo, lane, [&](int pair, int e, int rank, bool last, int) {
    const int p = e >= 0 ? mine[e] + rank : -1;
    const long long to = first + lo + pair;
    if (pair >= 0) r.slot[to] = p;
    if (e >= 0) r.row[p] = (int)((unsigned)to / (unsigned)r.top);
    __builtin_amdgcn_wave_barrier();
    if (e >= 0 && last) mine[e] = p + 1;
  });
}

// starts (written where `write`) and base[e] = starts[e] + before[e], of the experts' totals: total and before are experts ints in LDS
__device__ __forceinline__ void start_experts(const anvil_route& r, const int* total, const int* before, int* base, bool write, int* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int carry = 0;
  for (int e0 = 0; e0 < r.experts; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    const int c = e < r.experts ? total[e] : 0, incl = wave_scan(c);
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int start = carry + incl - c;
    for (int w = 0; w < waves; ++w) {
      if (w < wave) start += sums[w];
      carry += sums[w];
    }
    if (e < r.experts) {
      base[e] = start + (before ? before[e] : 0);
      if (write) r.starts[e] = start;
    }
    __syncthreads();
  }
  if (write && threadIdx.x == 0) r.starts[r.experts] = carry;
}

// Few rows: all of it by one workgroup. LDS: the pairs' experts, experts counts and bases, a row of experts a wave.
template <int L, int PER>
__global__ __launch_bounds__(1024) void route_one(RouteArgs g) {
  extern __shared__ int lds[];
  __shared__ int sums[16];
  const anvil_route& r = g.r;
  const int waves = blockDim.x >> 6, n = r.rows * r.top;
  int *count = lds, *base = lds + r.experts, *at = base + r.experts, *pairs = at + waves * r.experts;
  for (int e = threadIdx.x; e < (2 + waves) * r.experts; e += blockDim.x) lds[e] = 0;
  __syncthreads();
  choose_rows<L, PER>(g, 0, r.rows, pairs, count);
  __syncthreads();
  start_experts(r, count, nullptr, base, true, sums);
  place_pairs(r, pairs, 0, n, base, at);
}

// Many rows, first launch: each workgroup's experts and weights, and its counts.
template <int L, int PER>
__global__ __launch_bounds__(1024) void route_choose(RouteArgs g) {
  __shared__ int count[L * PER];
  for (int e = threadIdx.x; e < L * PER; e += blockDim.x) count[e] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * g.block_rows;
  choose_rows<L, PER>(g, first, (int)min((long long)g.block_rows, g.r.rows - first), nullptr, count);
  __syncthreads();
  for (int e = threadIdx.x; e < g.r.experts; e += blockDim.x) g.counts[(long long)blockIdx.x * g.r.experts + e] = count[e];
}

// Second launch: every workgroup adds up the counts of all, and of those before it, and places its pairs. LDS: totals, those before,
// bases, a row of experts a wave.
__global__ __launch_bounds__(1024) void route_place(RouteArgs g) {
  extern __shared__ int lds[];
  __shared__ int sums[16];
  const anvil_route& r = g.r;
  const int E = r.experts;
  int *total = lds, *before = lds + E, *base = before + E, *at = base + E;
  for (int e = threadIdx.x; e < (3 + (int)(blockDim.x >> 6)) * E; e += blockDim.x) lds[e] = 0;
  __syncthreads();
  // thread t: expert t % pitch, workgroups t / pitch, + blockDim.x / pitch, ...
  const int pitch = min((int)blockDim.x, (E + 63) / 64 * 64);
  const int parts = (int)blockDim.x / pitch, part = threadIdx.x / pitch;
  if (part < parts)
    for (int e = threadIdx.x % pitch; e < E; e += pitch) {
      int all = 0, prior = 0;
#pragma unroll 16
      for (int b = part; b < g.blocks; b += parts) {
        const int c = g.counts[(long long)b * E + e];
        all += c;
        prior += b < (int)blockIdx.x ? c : 0;
      }
      atomicAdd(&total[e], all);
      atomicAdd(&before[e], prior);
    }
  __syncthreads();
  start_experts(r, total, before, base, blockIdx.x == 0, sums);
  const long long first = (long long)blockIdx.x * g.block_rows * r.top, left = (long long)r.rows * r.top - first;
  place_pairs(r, r.expert + first, first, (int)min((long long)g.block_rows * r.top, left), base, at);
}

// ------------------------------------------------------------------------------------------------- combine

struct CombineArgs {
  anvil_expert_combine c;
  int mult, lifted;                                      // of WideRequant's upper word, where c.mult / 2^c.shift allows it (c.shift then 33 or more)
  unsigned* flags;
};

// Sixteen columns a thread, operands 16-byte aligned: a row's slots and weights first, then up to four of its results at a time. A slot
// that adds nothing reads row 0 with weight 0, so no load waits for a branch. RSZ, DSZ: bytes of R's (0: none) and D's elements.
// What bounds it is memory: top + 4 bytes an element (an i16 residual and result), two instructions a result's element and nine more.
// 32768 rows of 768, two results each: 30.7 us, 4.9 TB/s (with types told apart at run time and a branch a result 37.1, eight columns a thread
// so 40, an element a thread 147); int8 residual and result 21.0 (31.0), none 15.7 (19.6).
// ANY: rows at any alignment and of any width from 16 columns on. A row's last thread then takes its last 16 columns and stores those that no
// other thread has, so it reads no byte past the row, and in place what it has read of another's columns is dropped. 32768 rows of 769: 33.3 us
// (an element a thread 166).
template <int RSZ, int DSZ, bool ANY>
__global__ __launch_bounds__(256) void combine_rows(CombineArgs g) {
  const anvil_expert_combine& c = g.c;
  const WideRequant rq(c.shift, -128, 127);
  constexpr int lo = DSZ == 1 ? -128 : -32768, hi = -lo - 1;
  const int rnd2 = (int)round_term(c.shift2), wide = DSZ == 1 ? 24 : 16;       // a shift from which lo and hi leave int32
  const int clo = c.shift2 < wide ? lo * (1 << c.shift2) : (int)I32_MIN, chi = c.shift2 < wide ? -lo * (1 << c.shift2) - 1 : (int)I32_MAX;
  const int chunks = (c.cols + 15) >> 4;
  const long long n = (long long)c.rows * chunks;
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
    const long long i = n <= UINT32_MAX ? (unsigned)at / (unsigned)chunks : at / chunks;
    const int first = (int)(at - i * chunks) * 16, col = ANY ? min(first, c.cols - 16) : first;
    const int* const slot = c.slot + i * c.top;
    const int16_t* const weight = c.weight + i * c.top;
    v4i r[RSZ == 2 ? 2 : 1];
    if constexpr (RSZ > 0) {
      const char* p = (const char*)c.R + (i * c.ldr + col) * RSZ;
#pragma unroll
      for (int q = 0; q < RSZ; ++q) r[q] = load16<ANY>(p + 16 * q);
    }
    int acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0;
    const auto add = [&](int j0, auto count) {
      constexpr int N = decltype(count)::value;
      int p[N], w[N];
      v4i y[N];
#pragma unroll
      for (int k = 0; k < N; ++k) p[k] = slot[j0 + k], w[k] = weight[j0 + k];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const bool in = p[k] >= 0 && p[k] < c.positions;
        if (!in && p[k] != -1) raise_flag(g.flags, FLAG_EXPERTS);
        w[k] = in ? w[k] : 0;
        y[k] = load16<ANY>(c.Y + (in ? p[k] : 0) * c.ldy + col);
      }
#pragma unroll
      for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] += __mul24((int)(int8_t)((unsigned)y[k][e >> 2] >> (8 * (e & 3))), w[k]);
    };
    if (c.positions) {
      int j = 0;
      for (; j + 4 <= c.top; j += 4) add(j, std::integral_constant<int, 4>{});
      if (c.top & 2) add(j, std::integral_constant<int, 2>{}), j += 2;
      if (c.top & 1) add(j, std::integral_constant<int, 1>{});
    }
    const auto finish = [&](auto hi_c) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        acc[e] = rq.of<decltype(hi_c)::value>(acc[e], g.mult);
        if constexpr (RSZ > 0) {
          const unsigned h = (unsigned)r[RSZ == 2 ? e >> 3 : 0][RSZ == 2 ? e >> 1 & 3 : e >> 2];
          const int x = RSZ == 1 ? (int)(int8_t)(h >> (8 * (e & 3))) : e & 1 ? (int)h >> 16 : (int)(int16_t)h;
          acc[e] = med3i(mad_i24v(x, c.ma, mad_i24v(acc[e], c.mb, rnd2)), clo, chi);
        }
      }
    };
    if (g.lifted) finish(std::true_type{});
    else finish(std::false_type{});
    const int shift2 = RSZ ? c.shift2 : 0;
    typename Words<4 * DSZ>::type w;
    if constexpr (DSZ == 1) {
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = sra_pack4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3], shift2);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) w[q] = __builtin_amdgcn_perm((unsigned)(acc[2 * q + 1] >> shift2), (unsigned)(acc[2 * q] >> shift2), 0x05040100u);
    }
    char* const d = (char*)c.D + (i * c.ldd + col) * DSZ;
    if (ANY && col != first) {
      store_last<4 * DSZ>(d + 16 * DSZ, w, (c.cols & 15) * DSZ);
    } else {
#pragma unroll
      for (int q = 0; q < DSZ; ++q) {
        const v4i v = {(int)w[4 * q], (int)w[4 * q + 1], (int)w[4 * q + 2], (int)w[4 * q + 3]};
        if constexpr (ANY) __builtin_memcpy(d + 16 * q, &v, 16);
        else *reinterpret_cast<v4i*>(d + 16 * q) = v;
      }
    }
  }
}

// Slots of a Y without rows, which combine_rows does not look at: every one but -1 is out of range. (Looked at there, they cost it four registers and
// with them a wave a SIMD.)
__global__ __launch_bounds__(256) void report_slots(CombineArgs g) {
  const long long n = (long long)g.c.rows * g.c.top;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256)
    if (g.c.slot[i] != -1) raise_flag(g.flags, FLAG_EXPERTS);
}

// One element a thread: rows of fewer than 16 columns, multipliers of more than 24 bits.
__global__ __launch_bounds__(256) void combine_any(CombineArgs g) {
  const anvil_expert_combine& c = g.c;
  const WideRequant rq(c.shift, -128, 127);
  const int lo = c.d_dtype == ANVIL_I8 ? -128 : -32768, hi = -lo - 1;
  const long long n = (long long)c.rows * c.cols;
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
    const long long i = n <= UINT32_MAX ? (unsigned)at / (unsigned)c.cols : at / c.cols;
    const int col = (int)(at - i * c.cols);
    int acc = 0;                                         // 32 x 2^15 x 2^7 at most
    for (int j = 0; j < c.top; ++j) {
      const int p = c.slot[i * c.top + j];
      if (p >= 0 && p < c.positions) acc += (int)c.weight[i * c.top + j] * (int)c.Y[p * c.ldy + col];
      else if (p != -1) raise_flag(g.flags, FLAG_EXPERTS);
    }
    int d = g.lifted ? rq.of<true>(acc, g.mult) : rq.of<false>(acc, g.mult);
    if (c.R) {
      const int r = c.r_dtype == ANVIL_I8 ? (int)((const int8_t*)c.R)[i * c.ldr + col] : (int)((const int16_t*)c.R)[i * c.ldr + col];
      d = min(max((r * c.ma + d * c.mb + (int)round_term(c.shift2)) >> c.shift2, lo), hi);
    }
    if (c.d_dtype == ANVIL_I8) ((int8_t*)c.D)[i * c.ldd + col] = (int8_t)d;
    else ((int16_t*)c.D)[i * c.ldd + col] = (int16_t)d;
  }
}

}  // namespace anvil

using namespace anvil;

extern "C" int anvil_expert_route_i8(anvil_ctx* ctx, const anvil_route* r) {
  const char* who = "anvil_expert_route_i8";
  if (!r) return set_error(ANVIL_E_VALUE, "%s: null arguments", who);
  if (r->rows < 0 || r->experts < 1 || r->experts > ANVIL_EXPERTS_MAX || r->top < 1 || r->top > ANVIL_ROUTE_TOP_MAX ||
      r->top > r->experts || (long long)r->rows * r->top >= 1 << 30 || !stride_ok(r->ld, r->experts))
    return set_error(ANVIL_E_VALUE, "%s: %d rows, %d of %d experts, row stride %lld", who, r->rows, r->top, r->experts, (long long)r->ld);
  if (r->flags & ~ANVIL_ROUTE_EVERY) return set_error(ANVIL_E_VALUE, "%s: unknown flags %d", who, r->flags);
  if (r->one < 1 || r->one > 32767) return set_error(ANVIL_E_VALUE, "%s: one %d outside [1, 32767]", who, r->one);
  if (!r->starts || (r->rows && (!r->scores || !r->lut || !r->expert || !r->weight || !r->slot || !r->row)))
    return set_error(ANVIL_E_VALUE, "%s: null pointer", who);
  if ((uintptr_t)r->lut % 4 || (uintptr_t)r->expert % 4 || (uintptr_t)r->weight % 2 || (uintptr_t)r->slot % 4 || (uintptr_t)r->row % 4 ||
      (uintptr_t)r->starts % 4)
    return set_error(ANVIL_E_VALUE, "%s: a pointer is not aligned to its type", who);
  const long long pairs = (long long)r->rows * r->top;
  const auto flat = [](const void* p, long long bytes) { return Span{p, 1, bytes, bytes}; };
  const Span in[3] = {{r->scores, r->rows, r->ld, r->experts}, flat(r->live, r->rows), flat(r->lut, 1024)};
  const Span out[5] = {flat(r->expert, 4 * pairs), flat(r->weight, 2 * pairs), flat(r->slot, 4 * pairs), flat(r->row, 4 * pairs),
                       flat(r->starts, 4ll * r->experts + 4)};
  for (int i = 0; i < 5; ++i) {
    bool ok = true;
    for (int j = 0; j < 3; ++j) ok = ok && apart(out[i], in[j]);
    for (int j = 0; j < i; ++j) ok = ok && apart(out[i], out[j]);
    if (!ok) return set_error(ANVIL_E_VALUE, "%s: the results overlap each other or what is read", who);
  }
  if (int e = check_ctx(ctx)) return e;
  if (!r->rows) return zero_fill(ctx->stream, r->starts, 4ull * r->experts + 4);
  const int block_rows = std::max(ROUTE_ROWS, (r->rows + ROUTE_BLOCKS - 1) / ROUTE_BLOCKS);
  RouteArgs g{*r, nullptr, (r->rows + block_rows - 1) / block_rows, block_rows, ctx->flags};
  const size_t E = (size_t)r->experts * sizeof(int);
  const int lanes = r->top <= 16 && r->experts <= 256 ? 16 : 64;
  // one workgroup: as many waves as its rows fill at a time, where its LDS has room for them
  const int waves = std::max(1, std::min(16, (r->rows * lanes + 63) / 64));
  const size_t lds_one = (2 + waves) * E + (size_t)r->rows * r->top * sizeof(int);
  const bool one = r->rows <= ROUTE_ONE && lds_one <= 60 << 10;
  const int wide = block_rows >= ROUTE_WIDE ? 16 : 8, placing = (3 + wide) * E <= 60 << 10 ? wide : 8;
  if (!one) {
    char* ws;
    if (int e = decode_workspace(ctx, g.blocks * E, &ws)) return e;
    g.counts = (int*)ws;
  }
  const auto run = [&](auto l, auto per) {
    constexpr int L = decltype(l)::value, PER = decltype(per)::value;
    if (one) {
      ANVIL_LAUNCH((route_one<L, PER>), dim3(1), dim3(64 * waves), lds_one, ctx->stream, g);
      return;
    }
    ANVIL_LAUNCH((route_choose<L, PER>), dim3((unsigned)g.blocks), dim3(64 * wide), 0, ctx->stream, g);
    ANVIL_LAUNCH(route_place, dim3((unsigned)g.blocks), dim3(64 * placing), (3 + placing) * E, ctx->stream, g);
  };
  using std::integral_constant;
  if (lanes == 16) {
    const integral_constant<int, 16> l;
    if (r->experts <= 16) run(l, integral_constant<int, 1>{});
    else if (r->experts <= 32) run(l, integral_constant<int, 2>{});
    else if (r->experts <= 64) run(l, integral_constant<int, 4>{});
    else if (r->experts <= 128) run(l, integral_constant<int, 8>{});
    else run(l, integral_constant<int, 16>{});
  } else {
    const integral_constant<int, 64> l;
    if (r->experts <= 64) run(l, integral_constant<int, 1>{});
    else if (r->experts <= 256) run(l, integral_constant<int, 4>{});
    else run(l, integral_constant<int, 16>{});
  }
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}

extern "C" int anvil_expert_combine_i8(anvil_ctx* ctx, const anvil_expert_combine* c) {
  const char* who = "anvil_expert_combine_i8";
  if (!c) return set_error(ANVIL_E_VALUE, "%s: null arguments", who);
  if (c->rows < 0 || c->cols < 1 || c->cols > 1 << 20 || c->top < 1 || c->top > ANVIL_ROUTE_TOP_MAX || c->positions < 0 ||
      (long long)c->rows * c->top >= 1 << 30)
    return set_error(ANVIL_E_VALUE, "%s: %d rows of %d, %d of %d positions each", who, c->rows, c->cols, c->top, c->positions);
  if (!narrow(c->d_dtype) || (c->R ? !narrow(c->r_dtype) : c->d_dtype != ANVIL_I8))
    return set_error(ANVIL_E_VALUE, "%s: R and D must be i8 or i16, D without R i8", who);
  if (!stride_ok(c->ldy, c->cols) || !stride_ok(c->ldd, c->cols) || (c->R && !stride_ok(c->ldr, c->cols)))
    return set_error(ANVIL_E_VALUE, "%s: a row stride is not in [%d, 2^31)", who, c->cols);
  if (c->shift < 0 || c->shift > 62) return set_error(ANVIL_E_VALUE, "%s: shift %d outside [0, 62]", who, c->shift);
  if (c->R) {
    if (c->shift2 < 0 || c->shift2 > 31) return set_error(ANVIL_E_VALUE, "%s: shift2 %d outside [0, 31]", who, c->shift2);
    if (!sum_fits(c->r_dtype, c->ma, ANVIL_I8, c->mb, c->shift2))
      return set_error(ANVIL_E_OVERFLOW, "%s: R * %d + y * %d may leave int32", who, c->ma, c->mb);
  }
  if (!c->rows) return check_ctx(ctx);
  if (!c->slot || !c->weight || !c->D || (c->positions && !c->Y)) return set_error(ANVIL_E_VALUE, "%s: null pointer", who);
  if ((uintptr_t)c->slot % 4 || (uintptr_t)c->weight % 2 || (uintptr_t)c->D % c->d_dtype || (c->R && (uintptr_t)c->R % c->r_dtype))
    return set_error(ANVIL_E_VALUE, "%s: a pointer is not aligned to its type", who);
  const long long pairs = (long long)c->rows * c->top;
  const Span d{c->D, c->rows, c->ldd * c->d_dtype, (long long)c->cols * c->d_dtype};
  const Span y{c->Y, c->positions, c->ldy, c->cols}, slot{c->slot, 1, 4 * pairs, 4 * pairs}, weight{c->weight, 1, 2 * pairs, 2 * pairs};
  const bool on_r = c->D == c->R && c->d_dtype == c->r_dtype && c->ldd == c->ldr;
  if (!apart(d, y) || !apart(d, slot) || !apart(d, weight) ||
      (c->R && !on_r && !apart(d, Span{c->R, c->rows, c->ldr * c->r_dtype, (long long)c->cols * c->r_dtype})))
    return set_error(ANVIL_E_VALUE, "%s: the result overlaps what is read", who);
  if (int e = check_ctx(ctx)) return e;
  CombineArgs g{*c, c->mult, 0, ctx->flags};
  lift_shift(g.mult, g.c.shift);
  g.lifted = g.c.shift >= 33;
  const long long n = (long long)c->rows * c->cols;
  const auto even = [](const void* p, long long ld, int size) { return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0; };
  const auto m24 = [](int m) { return m >= -(1 << 23) && m < 1 << 23; };         // multipliers that a 24-bit product takes
  if (c->cols >= 16 && (!c->R || (m24(c->ma) && m24(c->mb)))) {
    const bool aligned = c->cols % 16 == 0 && even(c->Y, c->ldy, 1) && even(c->D, c->ldd, c->d_dtype) && (!c->R || even(c->R, c->ldr, c->r_dtype));
    const long long threads = (long long)c->rows * ((c->cols + 15) / 16);
    const dim3 grid((unsigned)std::min<long long>((threads + 255) / 256, 1 << 20));
    if (!c->positions) {
      ANVIL_LAUNCH(report_slots, dim3((unsigned)std::min<long long>((pairs + 255) / 256, 1 << 16)), dim3(256), 0, ctx->stream, g);
      ANVIL_LAUNCHED();
    }
    const auto run = [&](auto rsz, auto dsz) {
      constexpr int RSZ = decltype(rsz)::value, DSZ = decltype(dsz)::value;
      if (aligned) ANVIL_LAUNCH((combine_rows<RSZ, DSZ, false>), grid, dim3(256), 0, ctx->stream, g);
      else ANVIL_LAUNCH((combine_rows<RSZ, DSZ, true>), grid, dim3(256), 0, ctx->stream, g);
    };
    const std::integral_constant<int, 0> none;
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    if (!c->R) run(none, one);
    else if (c->r_dtype == ANVIL_I8 && c->d_dtype == ANVIL_I8) run(one, one);
    else if (c->r_dtype == ANVIL_I8) run(one, two);
    else if (c->d_dtype == ANVIL_I8) run(two, one);
    else run(two, two);
    ANVIL_LAUNCHED();
    return ANVIL_OK;
  }
  ANVIL_LAUNCH(combine_any, dim3((unsigned)std::min<long long>((n + 255) / 256, 1 << 20)), dim3(256), 0, ctx->stream, g);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
