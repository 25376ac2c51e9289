// Attention of the newest tokens over the 4-bit paged cache.
#include "cache.h"

namespace anvil {

struct AttendArgs {
  const int8_t* q;
  int8_t* o;
  long long q_row, q_head, o_row, o_head;
  const int* lut;
  int heads_q, m_s, s_s, one, m_o, s_o, window, sinks;
};

__device__ __forceinline__ bool sees(int j, int i, int window, int sinks) {
  return j <= i && (!window || j > i - window || j < sinks);
}

__device__ __forceinline__ int clamp_i8(long long v) { return v < -128 ? -128 : (v > 127 ? 127 : (int)v); }

constexpr int ATTEND_THREADS = 256;

// One query row and head a workgroup, one key a thread: the scores twice (their histogram, then their probabilities).
template <int NG>
__global__ __launch_bounds__(ATTEND_THREADS) void attend_kernel(CacheView c, AttendArgs a) {
  using B = Block<NG>;
  const int s = blockIdx.y, t = (int)blockIdx.x / a.heads_q, hq = (int)blockIdx.x % a.heads_q, tid = threadIdx.x;
  const int h = hq / (a.heads_q / c.heads);
  NewRows r;
  new_rows(c, s, r, blockIdx.x == 0 && tid == 0);
  if (t >= r.n) return;
  const int pos = r.len - r.n + t;
  __shared__ int hist[256], probs[256], part[ATTEND_THREADS];
  __shared__ unsigned long long sum;
  __shared__ int top;
  __shared__ int8_t qs[32 * NG];
  for (int i = tid; i < 256; i += ATTEND_THREADS) hist[i] = 0;
  for (int i = tid; i < 32 * NG; i += ATTEND_THREADS)
    qs[i] = i < c.dim ? a.q[(r.first + t) * a.q_row + hq * a.q_head + i] : 0;
  if (tid == 0) sum = 0, top = 0;
  __syncthreads();
  auto score = [&](const uint8_t* blk, int key) {
    long long acc = 0;
    for (int g = 0; g < NG; ++g) {
      int dot = 0;
      for (int q = 0; q < 4; ++q) {
        const unsigned w = *(const unsigned*)(blk + B::K + key * B::ROW + 4 * (q * NG + g));
        for (int e = 0; e < 8; ++e) dot += ((int)(w << (28 - 4 * (2 * (e & 3) + (e >> 2)))) >> 28) * qs[32 * g + 8 * q + e];
      }
      acc += dot * (int)blk[B::K_STEPS + ((key >> 2) * NG + g) * 4 + (key & 3)];
    }
    return clamp_i8((acc * a.m_s + round_term(a.s_s)) >> a.s_s);
  };
  for (int j = tid; j <= pos; j += ATTEND_THREADS) {
    if (!sees(j, pos, a.window, a.sinks)) continue;
    const uint8_t* blk = page_block<NG>(c, s, j / PAGE, h, true);
    if (blk) atomicAdd(&hist[score(blk, j % PAGE) + 128], 1);
  }
  __syncthreads();
  if (hist[tid]) atomicMax(&top, tid);
  __syncthreads();
  const long long e = tid <= top ? max(0, a.lut[tid - top + 255]) : 0;
  if (hist[tid]) atomicAdd(&sum, (unsigned long long)(e * hist[tid]));
  __syncthreads();
  const long long S = (long long)sum;
  probs[tid] = S ? (int)((e * a.one + S / 2) / S) : 0;
  if (tid == 0 && S == 0 && hist[top]) raise_flag(c.flags, FLAG_ZERODIV);
  long long acc = 0;
  const int d = tid & 127, half = tid >> 7;
  const int ch = d < 32 * NG ? d : 0, g = ch / 32, i = ch % 16, high = (ch / 16) & 1;
  for (int base = 0; base <= pos; base += ATTEND_THREADS) {
    __syncthreads();
    const int j = base + tid;
    int p = 0;
    if (j <= pos && sees(j, pos, a.window, a.sinks)) {
      const uint8_t* blk = page_block<NG>(c, s, j / PAGE, h, false);
      if (blk) p = probs[score(blk, j % PAGE) + 128];
    }
    part[tid] = p;
    __syncthreads();
    for (int k = half; k < ATTEND_THREADS; k += 2) {
      if (part[k] == 0) continue;
      const int key = base + k;
      const uint8_t* blk = page_block<NG>(c, s, key / PAGE, h, false);
      const unsigned b = blk[B::V + (16 * g + i) * PAGE + key % PAGE];
      acc += (long long)part[k] * (((int)(b << (28 - 4 * high)) >> 28) * (int)blk[B::V_STEPS + PAGE * g + key % PAGE]);
    }
  }
  __syncthreads();
  part[tid] = (int)acc;
  __syncthreads();
  if (tid < c.dim)
    a.o[(r.first + t) * a.o_row + hq * a.o_head + tid] =
        (int8_t)clamp_i8(((long long)(part[tid] + part[tid + 128]) * a.m_o + round_term(a.s_o)) >> a.s_o);
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
  const AttendArgs a{Q, O, strides[0], strides[1], strides[2], strides[3], lut, heads_q, m_s, s_s, one, m_o, s_o, window, sinks};
  by_groups(c.dim, [&](auto ng) {
    ANVIL_LAUNCH(attend_kernel<decltype(ng)::value>, dim3((unsigned)((long long)max_new * heads_q), (unsigned)c.seqs),
                 dim3(ATTEND_THREADS), 0, ctx->stream, c, a);
  });
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
