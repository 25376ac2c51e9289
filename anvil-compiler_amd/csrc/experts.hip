// The router of an experts' feed-forward and the way back: each row's best experts and their weights, the rows sorted by expert,
// and the weighted sums of their results.
//
// Route. A wave takes a row: lane l holds the scores of experts l, l + 64, ..., each with its expert's number below it in one int
// (larger score first, then lower expert), so the j-th choice is a maximum over the wave of what is below the one before.
// Sorting. Workgroups of ROWS rows count their pairs by expert; the rows of counts meet in a second launch, where every workgroup adds up
// those before its own and places its pairs. Within a workgroup the waves own runs of consecutive pairs, and a pair's
// rank among the 64 of a step is the number of lower lanes with its expert (ballots over the bits of its number). No atomic decides
// an order: positions are the same each time.
#include <algorithm>

#include "experts.h"

namespace anvil {

constexpr int ROUTE_WAVES = 4, ROUTE_THREADS = 64 * ROUTE_WAVES;
constexpr int ROUTE_ROWS = 128;                          // rows of a workgroup, at least
constexpr int ROUTE_BLOCKS = 1024;                       // workgroups, at most

struct RouteArgs {
  anvil_route r;
  int* counts;                                           // blocks x experts
  int blocks, block_rows;
  unsigned* flags;
};

__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ long long wave_total(long long v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// (e one + S / 2) / S of e <= 2^31 - 1, one <= 2^15 - 1: the quotient of doubles is off by at most one
__device__ __forceinline__ int share(long long e, int one, long long S) {
  const long long num = e * one + S / 2;
  long long q = (long long)((double)num / (double)S);
  if (q * S > num) --q;
  else if ((q + 1) * S <= num) ++q;
  return (int)q;
}

// A row's choices: lane j's expert and weight of choice j
template <int PER>
__device__ __forceinline__ void choose(const RouteArgs& g, long long row, int lane, int& expert, int& weight) {
  const anvil_route& r = g.r;
  int key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 64 * i;
    key[i] = e < r.experts ? (int)r.scores[row * r.ld + e] * 1024 + (1023 - e) : INT32_MIN;
  }
  int best = 0, mine = 0, top = 0;
  for (int j = 0; j < r.top; ++j) {
    int m = INT32_MIN;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (j == 0 || key[i] < best) m = max(m, key[i]);
    best = wave_max(m);
    if (j == 0) top = best >> 10;
    if (lane == j) mine = best;
  }
  const bool has = lane < r.top;
  const long long e = has ? max(0, r.lut[(mine >> 10) - top + 255]) : 0;
  long long S = e;
  if (r.flags & ANVIL_ROUTE_EVERY) {
    S = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 64 * i < r.experts) S += max(0, r.lut[(key[i] >> 10) - top + 255]);
  }
  S = wave_total(S);
  expert = 1023 - (mine & 1023);
  weight = S ? share(e, r.one, S) : 0;
  if (!S && lane == 0) raise_flag(g.flags, FLAG_ZERODIV);
}

// The pairs first .. first + n - 1 (in the order of rows and choices) that the calling wave owns, 64 a step:
// f(pair or -1, expert or -1, rank among this step's lower lanes of the same expert, whether it is the expert's last lane, its count)
template <typename F>
__device__ __forceinline__ void for_pairs(const int* expert, long long first, int n, int lane, F&& f) {
  for (int i = 0; i < n; i += 64) {
    const bool in = i + lane < n;
    const int e = in ? expert[first + i + lane] : -1;
    unsigned long long same = __ballot(e >= 0);
    for (int b = 0; b < 10; ++b) {
      const unsigned long long set = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1)), all = __popcll(same);
    f(in ? first + i + lane : -1ll, e, rank, rank == all - 1, all);
  }
}

// The rows' experts and weights, and the counts of each workgroup's pairs by expert.
template <int PER>
__global__ __launch_bounds__(ROUTE_THREADS) void route_choose(RouteArgs g) {
  const anvil_route& r = g.r;
  __shared__ int count[64 * PER];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int e = threadIdx.x; e < 64 * PER; e += ROUTE_THREADS) count[e] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * g.block_rows;
  const int n = (int)min((long long)g.block_rows, r.rows - first);
  for (int i = wave; i < n; i += ROUTE_WAVES) {
    const long long row = first + i;
    int expert = -1, weight = 0;
    const bool live = !r.live || r.live[row];
    if (live) choose<PER>(g, row, lane, expert, weight);
    if (lane < r.top) {
      r.expert[row * r.top + lane] = expert;
      r.weight[row * r.top + lane] = (int16_t)weight;
      if (live) atomicAdd(&count[expert], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < r.experts; e += ROUTE_THREADS) g.counts[(long long)blockIdx.x * r.experts + e] = count[e];
}

// Positions of each workgroup's pairs.
template <int PER>
__global__ __launch_bounds__(ROUTE_THREADS) void route_place(RouteArgs g) {
  const anvil_route& r = g.r;
  __shared__ int base[64 * PER], at[ROUTE_WAVES][64 * PER];
  __shared__ int sums[ROUTE_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // thread t: experts PER' t .. : totals of all workgroups, those before this one, and the exclusive sums over experts
  constexpr int MINE = (64 * PER + ROUTE_THREADS - 1) / ROUTE_THREADS;
  int total[MINE], before[MINE], sum = 0;
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int e = threadIdx.x * MINE + i;
    total[i] = before[i] = 0;
    if (e < r.experts)
      for (int b = 0; b < g.blocks; ++b) {
        const int c = g.counts[(long long)b * r.experts + e];
        total[i] += c;
        if (b < (int)blockIdx.x) before[i] += c;
      }
    sum += total[i];
  }
  const int incl = wave_scan(sum);
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int start = incl - sum;
  for (int w = 0; w < wave; ++w) start += sums[w];
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int e = threadIdx.x * MINE + i;
    if (e < r.experts) {
      base[e] = start + before[i];
      if (blockIdx.x == 0) r.starts[e] = start;
    }
    start += total[i];
  }
  if (blockIdx.x == 0 && threadIdx.x == ROUTE_THREADS - 1) r.starts[r.experts] = start;
  for (int e = threadIdx.x; e < ROUTE_WAVES * 64 * PER; e += ROUTE_THREADS) (&at[0][0])[e] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * g.block_rows * r.top;
  const int n = (int)min((long long)g.block_rows * r.top, (long long)r.rows * r.top - first);
  const int run = (n + ROUTE_WAVES - 1) / ROUTE_WAVES;
  const int lo = min(n, wave * run), hi = min(n, lo + run);
  for_pairs(r.expert, first + lo, hi - lo, lane, [&](long long, int e, int, bool last, int all) {
    if (e >= 0 && last) at[wave][e] += all;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  });
  __syncthreads();
  for (int e = threadIdx.x; e < r.experts; e += ROUTE_THREADS) {
    int p = base[e];
#pragma unroll
    for (int w = 0; w < ROUTE_WAVES; ++w) {
      const int c = at[w][e];
      at[w][e] = p;
      p += c;
    }
  }
  __syncthreads();
  for_pairs(r.expert, first + lo, hi - lo, lane, [&](long long pair, int e, int rank, bool last, int all) {
    const int p = e >= 0 ? at[wave][e] + rank : -1;
    if (pair >= 0) r.slot[pair] = p;
    if (e >= 0) r.row[p] = (int)(pair / r.top);
    __builtin_amdgcn_wave_barrier();
    if (e >= 0 && last) at[wave][e] = p + 1;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  });
}

// ------------------------------------------------------------------------------------------------- combine

struct CombineArgs {
  anvil_expert_combine c;
  unsigned* flags;
};

// One element a thread, any alignment.
__global__ __launch_bounds__(256) void combine_any(CombineArgs g) {
  const anvil_expert_combine& c = g.c;
  const Requant rq(c.shift, -128, 127);
  const int lo = c.d_dtype == ANVIL_I8 ? -128 : -32768, hi = -lo - 1;
  const long long n = (long long)c.rows * c.cols;
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
    const long long i = at / c.cols;
    const int col = (int)(at - i * c.cols);
    int acc = 0;                                         // 32 x 2^15 x 2^7 at most
    for (int j = 0; j < c.top; ++j) {
      const int p = c.slot[i * c.top + j];
      if (p >= 0 && p < c.positions) acc += (int)c.weight[i * c.top + j] * (int)c.Y[p * c.ldy + col];
      else if (p != -1) raise_flag(g.flags, FLAG_EXPERTS);
    }
    int d = rq.of<false>(acc, c.mult);
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
  char* ws;
  if (int e = decode_workspace(ctx, (size_t)g.blocks * r->experts * sizeof(int), &ws)) return e;
  g.counts = (int*)ws;
  const auto run = [&](auto per) {
    constexpr int PER = decltype(per)::value;
    ANVIL_LAUNCH(route_choose<PER>, dim3((unsigned)g.blocks), dim3(ROUTE_THREADS), 0, ctx->stream, g);
    ANVIL_LAUNCH(route_place<PER>, dim3((unsigned)g.blocks), dim3(ROUTE_THREADS), 0, ctx->stream, g);
  };
  if (r->experts <= 64) run(std::integral_constant<int, 1>{});
  else if (r->experts <= 256) run(std::integral_constant<int, 4>{});
  else run(std::integral_constant<int, 16>{});
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
  CombineArgs g{*c, ctx->flags};
  const long long n = (long long)c->rows * c->cols;
  ANVIL_LAUNCH(combine_any, dim3((unsigned)std::min<long long>((n + 255) / 256, 1 << 20)), dim3(256), 0, ctx->stream, g);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
