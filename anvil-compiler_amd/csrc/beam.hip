// Beam search's selection over beams and vocabulary from int8 logits.
#include "common.h"

namespace anvil {

constexpr long long NO_SCORE = INT64_MIN;
constexpr int BEAM_THREADS = 256;

__device__ __forceinline__ long long log_fixed(const anvil_beams& b, long long v) {
  int k = 0;
  while ((v >> k) >= b.nlogs) ++k;
  return b.logs[v >> k] + (long long)k * b.step;
}

// base[row]: what a candidate's score adds to logit * mult; NO_SCORE where the row has no candidates of its own.
__global__ __launch_bounds__(BEAM_THREADS) void beam_rows_kernel(anvil_beams b, long long* base, unsigned* flags) {
  const long long row = blockIdx.x;
  const int tid = threadIdx.x;
  __shared__ int hist[256];
  __shared__ unsigned long long sum;
  __shared__ int top;
  hist[tid] = 0;
  if (tid == 0) sum = 0, top = 0;
  __syncthreads();
  for (int v = tid; v < b.vocab; v += BEAM_THREADS) atomicAdd(&hist[b.logits[row * b.ld + v] + 128], 1);
  __syncthreads();
  if (hist[tid]) atomicMax(&top, tid);
  __syncthreads();
  if (hist[tid]) atomicAdd(&sum, (unsigned long long)max(0, b.lut[tid - top + 255]) * hist[tid]);
  __syncthreads();
  if (tid == 0) {
    const bool live = b.scores[row] != NO_SCORE && !(b.ended && b.ended[row]);
    const long long S = (long long)sum, one = b.lut[255];
    if (live && (S < 1 || one < 1)) raise_flag(flags, FLAG_ZERODIV);
    base[row] = live && S >= 1 && one >= 1
                    ? b.scores[row] - (long long)(top - 128) * b.mult - (log_fixed(b, S) - log_fixed(b, one))
                    : NO_SCORE;
  }
}

// One group a workgroup: the best candidate behind the last one taken, `keep` times.
__global__ __launch_bounds__(BEAM_THREADS) void beam_pick_kernel(anvil_beams b, const long long* base) {
  const int group = blockIdx.x, tid = threadIdx.x;
  __shared__ long long score[BEAM_THREADS];
  __shared__ long long where[BEAM_THREADS];
  long long last_score = INT64_MAX, last = -1;
  const long long size = (long long)b.beams * b.vocab;
  for (int n = 0; n < b.keep; ++n) {
    long long best = NO_SCORE, at = -1;
    for (long long i = tid; i < size; i += BEAM_THREADS) {
      const long long row = (long long)group * b.beams + i / b.vocab;
      const int v = (int)(i % b.vocab);
      long long c = NO_SCORE;
      if (b.ended && b.ended[row]) {
        if (v == b.eos) c = b.scores[row];
      } else if (base[row] != NO_SCORE && !(b.allowed && !b.allowed[v])) {
        c = base[row] + (long long)b.logits[row * b.ld + v] * b.mult;
      }
      if (c == NO_SCORE || c > last_score || (c == last_score && i <= last)) continue;
      if (c > best) best = c, at = i;                    // i ascends: the lowest of equals stays
    }
    score[tid] = best, where[tid] = at;
    __syncthreads();
    for (int d = BEAM_THREADS / 2; d; d /= 2) {
      if (tid < d) {
        const long long s2 = score[tid + d], w2 = where[tid + d];
        if (w2 >= 0 && (where[tid] < 0 || s2 > score[tid] || (s2 == score[tid] && w2 < where[tid]))) score[tid] = s2, where[tid] = w2;
      }
      __syncthreads();
    }
    best = score[0], at = where[0];
    __syncthreads();
    if (tid == 0) {
      const long long out = (long long)group * b.keep + n, row = (long long)group * b.beams + at / b.vocab;
      const int v = (int)(at % b.vocab);
      b.scores_out[out] = at < 0 ? NO_SCORE : best;
      b.parent[out] = at < 0 ? -1 : (int)row;
      b.token[out] = at < 0 ? -1 : v;
      b.ended_out[out] = at >= 0 && (v == b.eos || (b.ended && b.ended[row]));
    }
    if (at < 0) last_score = NO_SCORE, last = size;      // nothing left: the rest is empty too
    else last_score = best, last = at;
  }
}

}  // namespace anvil

using namespace anvil;

extern "C" int anvil_beam_select_i8(anvil_ctx* ctx, const anvil_beams* b) {
  const char* who = "anvil_beam_select_i8";
  if (!b) return set_error(ANVIL_E_VALUE, "%s: null arguments", who);
  if (b->groups < 0 || b->groups > (1 << 24) || b->beams < 1 || b->beams > 64 || b->keep < 1 || b->keep > 64 || b->vocab < 1 || b->ld < b->vocab)
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
  char* ws;
  const long long rows = (long long)b->groups * b->beams;
  if (int r = decode_workspace(ctx, (size_t)rows * 8, &ws)) return r;
  ANVIL_LAUNCH(beam_rows_kernel, dim3((unsigned)rows), dim3(BEAM_THREADS), 0, ctx->stream, *b, (long long*)ws, ctx->flags);
  ANVIL_LAUNCHED();
  ANVIL_LAUNCH(beam_pick_kernel, dim3((unsigned)b->groups), dim3(BEAM_THREADS), 0, ctx->stream, *b, (const long long*)ws);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
