// The 4-bit paged cache: new rows rounded into their pages, read back, and the page tables of the next step.
#include <algorithm>
#include <cmath>

#include "cache.h"

namespace anvil {

int check_cache(const char* who, const anvil_cache* c, bool refs) {
  if (!c) return set_error(ANVIL_E_VALUE, "%s: null cache", who);
  if (c->dim != 16 && c->dim != 32 && c->dim != 64 && c->dim != 128)
    return set_error(ANVIL_E_VALUE, "%s: head dim %d is not 16, 32, 64 or 128", who, c->dim);
  if (c->seqs < 0 || c->seqs > 65535 || c->slots < 1 || c->slots > ANVIL_CACHE_SLOTS_MAX || c->pages < 1 ||
      c->pages > (1 << 24) || c->heads < 1 || c->heads > 4096 || c->layers < 1 || c->layers > 65535)
    return set_error(ANVIL_E_VALUE, "%s: %d sequences of %d slots, %d pages of %d heads, %d layers", who, c->seqs,
                     c->slots, c->pages, c->heads, c->layers);
  if (!c->pool || (uintptr_t)c->pool % 16) return set_error(ANVIL_E_VALUE, "%s: the pool is null or not 16-byte aligned", who);
  if (c->seqs && (!c->table || !c->lens || (uintptr_t)c->table % 4 || (uintptr_t)c->lens % 4))
    return set_error(ANVIL_E_VALUE, "%s: table and lens must be aligned and not null", who);
  if (refs && (!c->refs || (uintptr_t)c->refs % 4)) return set_error(ANVIL_E_VALUE, "%s: refs must be aligned and not null", who);
  return ANVIL_OK;
}

int cache_view(const char* who, anvil_ctx* ctx, const anvil_cache* c, int layer, const int32_t* starts, int rows,
               int max_new, CacheView* v) {
  if (int r = check_cache(who, c, false)) return r;
  if (layer < 0 || layer >= c->layers) return set_error(ANVIL_E_VALUE, "%s: layer %d of %d", who, layer, c->layers);
  if (rows < 0 || max_new < 1 || max_new > ANVIL_CACHE_SLOTS_MAX * PAGE)
    return set_error(ANVIL_E_VALUE, "%s: %d rows, at most %d of a sequence", who, rows, max_new);
  if (!starts && (rows != c->seqs || max_new != 1))
    return set_error(ANVIL_E_VALUE, "%s: without starts every sequence has one row (rows %d, sequences %d, max_new %d)", who,
                     rows, c->seqs, max_new);
  if ((uintptr_t)starts % 4) return set_error(ANVIL_E_VALUE, "%s: starts is not aligned", who);
  v->pool = (uint8_t*)c->pool + (long long)layer * c->pages * c->heads * 2176 * groups_of(c->dim);
  v->table = c->table, v->lens = c->lens, v->starts = starts;
  v->seqs = c->seqs, v->slots = c->slots, v->pages = c->pages, v->heads = c->heads, v->dim = c->dim;
  v->rows = rows, v->max_new = std::min(max_new, std::max(rows, 1)), v->flags = ctx ? ctx->flags : nullptr;
  return ANVIL_OK;
}

// ------------------------------------------------------------------------------------------- append and read

struct RowPtrs {
  int8_t *k, *v;
  long long k_row, k_head, v_row, v_head;
};

// Eight consecutive channels as 4-bit codes and their group's step: lanes 4 i .. 4 i + 3 hold a group's 32 channels.
// code + 8 = floor((2 x + 17 step) / (2 step)), from 1 to 15 whatever x (|x| <= 7 step, and at step 18 the ends of int8 still round to
// 7 steps). With d = 2 step <= 36 and n <= 562 the quotient is (n m) >> 16 for every m from 2^16 / d to 2^16 / d + 2, as
// n (m d - 2^16) < 2^16: a reciprocal that may be one off either way will do. (a + 6) / 7 is a multiply by 2^16 / 7, rounded up. The
// dword's nibble e is channel e's code.
__device__ __forceinline__ unsigned round4(uint2 x, int& step) {
  int v[8], top = 0, least = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (int8_t)((e < 4 ? x.x : x.y) >> (8 * (e & 3)));
#pragma unroll
  for (int e = 0; e < 8; e += 2) top = max(max(top, v[e]), v[e + 1]), least = min(min(least, v[e]), v[e + 1]);
  int a = max(top, -least);
  a = max(a, (int)__builtin_amdgcn_update_dpp(0, a, 0xB1, 0xF, 0xF, false));     // quad_perm [1,0,3,2]
  a = max(a, (int)__builtin_amdgcn_update_dpp(0, a, 0x4E, 0xF, 0xF, false));     // quad_perm [2,3,0,1]
  step = min(STEP_MAX, max(1, __umul24(a + 6, 9363) >> 16));
  const int m = (int)(65536.0f * __builtin_amdgcn_rcpf((float)(2 * step))) + 2, start = 17 * step;
  unsigned w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= ((unsigned)__umul24(2 * v[e] + start, m) >> 16 & 15u) << (4 * e);
  return w ^ 0x88888888u;
}

// nibbles 0..3 of w into the low halves of four bytes, nibbles 4..7 into the high ones: the K code order
__device__ __forceinline__ unsigned interleave_k(unsigned w) {
  unsigned d = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) d |= (((w >> (4 * i)) & 15u) | ((w >> (12 + 4 * i)) & 0xF0u)) << (8 * i);
  return d;
}

constexpr int ROW_THREADS = 256;
constexpr int TILE = PAGE + 4;                           // bytes of a row of V codes in LDS: rows start in different banks

// A workgroup's part of a call: the tokens t0 .. t1 - 1 of one page of one sequence, and the row of the page's token 0.
struct PageRows {
  int t0, t1;
  long long row0;
  uint8_t* blk;
};
template <int NG>
__device__ __forceinline__ bool page_rows(const CacheView& c, PageRows& p) {
  const int s = blockIdx.y, h = blockIdx.z;
  NewRows r;
  new_rows(c, s, r, blockIdx.x == 0 && h == 0 && threadIdx.x == 0);
  const int begin = r.len - r.n, slot = (begin >> PAGE_SHIFT) + (int)blockIdx.x;
  p.t0 = max(begin - slot * PAGE, 0), p.t1 = min(r.len - slot * PAGE, PAGE);
  if (r.n == 0 || p.t1 <= 0) return false;
  p.row0 = (long long)r.first + slot * PAGE - begin;
  p.blk = page_block<NG>(c, s, slot, h, threadIdx.x == 0);
  return true;
}

// One page of one sequence and head a workgroup (blockIdx: page among those with new rows, sequence, head). Four
// lanes a group of 32 channels; all of a thread's rows are on their way before the first is rounded. K codes go straight to their
// rows; V codes, which the page holds channel by channel, meet in LDS and leave as whole 64-byte rows where the page is new from end
// to end. 8 prompts of up to 2048 tokens, 8 heads of 128: 11.4 us, 1.6 TB/s of rows read and pages written. 36 % of wave cycles wait for
// memory or the LDS, 40 % for a turn to issue; VALU instructions take 38 % of a SIMD's time.
template <int NG>
__global__ __launch_bounds__(ROW_THREADS) void append_kernel(CacheView c, RowPtrs p) {
  using B = Block<NG>;
  const int h = blockIdx.z, tid = threadIdx.x;
  PageRows r;
  if (!page_rows<NG>(c, r)) return;
  if (!r.blk) {
    if (tid == 0) raise_flag(c.flags, FLAG_CACHE);
    return;
  }
  __shared__ __align__(16) uint8_t vt[16 * NG][TILE];
  __shared__ __align__(16) uint8_t steps[2][PAGE * NG];
  const int items = (r.t1 - r.t0) * NG * 4;
  uint2 xk[NG], xv[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int i = tid + n * ROW_THREADS, t = r.t0 + i / (NG * 4), ch = 8 * (i % (NG * 4));
    xk[n] = {0, 0}, xv[n] = {0, 0};
    if (i < items && ch < c.dim) {
      xk[n] = *(const uint2*)(p.k + (r.row0 + t) * p.k_row + h * p.k_head + ch);
      xv[n] = *(const uint2*)(p.v + (r.row0 + t) * p.v_row + h * p.v_head + ch);
    }
  }
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int i = tid + n * ROW_THREADS;
    if (n * ROW_THREADS + (tid & ~63) >= items) break;   // whole waves: lanes exchange values
    const int t = r.t0 + i / (NG * 4), g = (i / 4) % NG, q = i & 3;
    int sk, sv;
    const unsigned wk = round4(xk[n], sk), wv = round4(xv[n], sv);
    const unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)wv, 0x4E, 0xF, 0xF, false);   // lane q ^ 2
    if (i >= items) continue;
    *(unsigned*)(r.blk + B::K + t * B::ROW + 4 * (q * NG + g)) = interleave_k(wk);
    // lane q holds channels 8 q .. of the group: with q ^ 2 it has both halves of V bytes i = 8 (q & 1) .., four each
    const unsigned low = q < 2 ? wv : other >> 16, high = q < 2 ? other : wv >> 16;
    const int i0 = 8 * (q & 1) + (q < 2 ? 0 : 4);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      vt[16 * g + i0 + e][t] = (uint8_t)(((low >> (4 * e)) & 15u) | (((high >> (4 * e)) & 15u) << 4));
    if (q == 0) {
      steps[0][((t >> 2) * NG + g) * 4 + (t & 3)] = (uint8_t)sk;
      steps[1][PAGE * g + t] = (uint8_t)sv;
    }
  }
  __syncthreads();
  if (r.t1 - r.t0 == PAGE) {
    for (int i = tid; i < 16 * NG * 4; i += ROW_THREADS) {
      const unsigned* row = (const unsigned*)(&vt[i >> 2][16 * (i & 3)]);
      *(uint4*)(r.blk + B::V + 16 * i) = {row[0], row[1], row[2], row[3]};
    }
    const int v = tid / (4 * NG), at = 16 * (tid % (4 * NG));
    if (v < 2) *(uint4*)(r.blk + (v ? B::V_STEPS : B::K_STEPS) + at) = *(const uint4*)(&steps[v][at]);
  } else {
    for (int i = tid; i < 2 * NG * (r.t1 - r.t0); i += ROW_THREADS) {
      const int g = i % NG, v = i / NG & 1, t = r.t0 + i / (2 * NG), at = v ? PAGE * g + t : ((t >> 2) * NG + g) * 4 + (t & 3);
      r.blk[(v ? B::V_STEPS : B::K_STEPS) + at] = steps[v][at];
    }
    for (int i = tid; i < 16 * NG * (r.t1 - r.t0); i += ROW_THREADS) {
      const int j = i / (r.t1 - r.t0), t = r.t0 + i % (r.t1 - r.t0);
      r.blk[B::V + j * PAGE + t] = vt[j][t];
    }
  }
}

__device__ __forceinline__ int code_of(unsigned w, int e) { return (int)(w << (28 - 4 * e)) >> 28; }

// The values of the same rows, one page of one sequence and head a workgroup. V's codes come through LDS: a token's are 64 bytes
// apart.
template <int NG>
__global__ __launch_bounds__(ROW_THREADS) void read_kernel(CacheView c, RowPtrs p) {
  using B = Block<NG>;
  const int h = blockIdx.z, tid = threadIdx.x;
  PageRows r;
  if (!page_rows<NG>(c, r)) return;
  __shared__ __align__(16) uint8_t vt[16 * NG][TILE];
  const int items = (r.t1 - r.t0) * NG * 4, blocks = (r.t1 + 15) / 16 - r.t0 / 16;
  if (r.blk)
    for (int i = tid; i < 16 * NG * blocks; i += ROW_THREADS) {
      const int j = i / blocks, at = 16 * (r.t0 / 16 + i % blocks);
      const uint4 x = *(const uint4*)(r.blk + B::V + j * PAGE + at);
      unsigned* row = (unsigned*)(&vt[j][at]);
      row[0] = x.x, row[1] = x.y, row[2] = x.z, row[3] = x.w;
    }
  unsigned wk[NG];
  int sk[NG], sv[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int i = tid + n * ROW_THREADS, t = r.t0 + i / (NG * 4), g = (i / 4) % NG, q = i & 3;
    wk[n] = 0, sk[n] = 0, sv[n] = 0;                     // a page given back reads as zeros
    if (r.blk && i < items) {
      wk[n] = *(const unsigned*)(r.blk + B::K + t * B::ROW + 4 * (q * NG + g));
      sk[n] = r.blk[B::K_STEPS + ((t >> 2) * NG + g) * 4 + (t & 3)], sv[n] = r.blk[B::V_STEPS + PAGE * g + t];
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int i = tid + n * ROW_THREADS, t = r.t0 + i / (NG * 4), g = (i / 4) % NG, q = i & 3;
    if (i >= items || 32 * g + 8 * q >= c.dim) continue;
    int k[8], v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      k[e] = code_of(wk[n], 2 * (e & 3) + (e >> 2)) * sk[n];
      v[e] = r.blk ? code_of(vt[16 * g + 8 * (q & 1) + e][t], q >> 1) * sv[n] : 0;
    }
    const uint2 xk = {pack4(k[0], k[1], k[2], k[3]), pack4(k[4], k[5], k[6], k[7])};
    const uint2 xv = {pack4(v[0], v[1], v[2], v[3]), pack4(v[4], v[5], v[6], v[7])};
    *(uint2*)(p.k + (r.row0 + t) * p.k_row + h * p.k_head + 32 * g + 8 * q) = xk;
    *(uint2*)(p.v + (r.row0 + t) * p.v_row + h * p.v_head + 32 * g + 8 * q) = xv;
  }
}

static int rows_call(const char* who, anvil_ctx* ctx, const anvil_cache* cache, int layer, const int8_t* K, const int8_t* V,
                     const int32_t* starts, int rows, int max_new, const int64_t* strides, bool write) {
  CacheView c;
  if (int r = cache_view(who, ctx, cache, layer, starts, rows, max_new, &c)) return r;
  if (!strides) return set_error(ANVIL_E_VALUE, "%s: null strides", who);
  if (!c.seqs || !rows) return check_ctx(ctx);
  if (!K || !V || (uintptr_t)K % 16 || (uintptr_t)V % 16) return set_error(ANVIL_E_VALUE, "%s: K and V must be 16-byte aligned", who);
  for (int i = 0; i < 4; ++i)
    if (strides[i] % 16 || (!write && (strides[i] < c.dim)))
      return set_error(ANVIL_E_VALUE, "%s: stride %lld (strides are multiples of 16, a result's at least the head dim)", who,
                       (long long)strides[i]);
  if (int r = check_ctx(ctx)) return r;
  const RowPtrs p{(int8_t*)K, (int8_t*)V, strides[0], strides[1], strides[2], strides[3]};
  const dim3 grid((unsigned)((c.max_new + PAGE - 2) / PAGE + 1), (unsigned)c.seqs, (unsigned)c.heads);
  by_groups(c.dim, [&](auto ng) {
    constexpr int NG = decltype(ng)::value;
    ANVIL_LAUNCH(write ? append_kernel<NG> : read_kernel<NG>, grid, dim3(ROW_THREADS), 0, ctx->stream, c, p);
  });
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}

// ------------------------------------------------------------------------------------------------- embedding

struct EmbedArgs {
  const int* ids;
  const float *wte, *wpe;
  int C, vocab, positions, lo, hi;
  double scale;
};

// One token a workgroup (blockIdx: token of its sequence, striding, and sequence).
template <typename TO>
__global__ __launch_bounds__(256) void embed_new_kernel(CacheView c, EmbedArgs e, TO* out) {
  NewRows r;
  new_rows(c, blockIdx.y, r, blockIdx.x == 0 && threadIdx.x == 0);
  for (int t = blockIdx.x; t < r.n; t += gridDim.x) {
    const int id = e.ids[r.first + t], i = r.len - r.n + t;
    const bool ok = id >= 0 && id < e.vocab && i < e.positions;
    if (!ok && threadIdx.x == 0) raise_flag(c.flags, FLAG_RANGE);
    for (int col = threadIdx.x; col < e.C; col += 256) {
      double v = 0;
      if (ok) v = rint(((double)e.wte[(long long)id * e.C + col] + (double)e.wpe[(long long)i * e.C + col]) / e.scale);
      out[(long long)(r.first + t) * e.C + col] = (TO)(v < e.lo ? e.lo : (v > e.hi ? e.hi : v));
    }
  }
}

// ---------------------------------------------------------------------------------------- fork and compact

constexpr int META = 1024;                               // threads of the workgroup that writes the tables

// exclusive prefix sum of v over the workgroup's META threads, and the total
__device__ __forceinline__ int prefix(int v, int& total) {
  __shared__ int sums[META / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = wave_scan(v);
  __syncthreads();                                       // the last call's sums have been read
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < META / 64; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  return before + x - v;
}

struct ForkArgs {
  const int *table, *lens, *refs, *parent, *add;
  int *table_out, *lens_out, *refs_out;
  int* list;                                             // scratch: free pages in order
  int2* copies;                                          // scratch: (from, to) pages, `*n` of them
  int* n;
  int seqs, seqs_out, slots, pages, window, sinks;
  unsigned* flags;
};

// A page's references while they are counted: in LDS, or with larger tables in refs_out, past the caches.
template <bool LDS>
struct Count {
  int* n;
  __device__ __forceinline__ int get(int p) const {
    if constexpr (LDS) return n[p];
    else return __hip_atomic_load(n + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ __forceinline__ void set(int p, int v) const {
    if constexpr (LDS) n[p] = v;
    else atomicExch(n + p, v);
  }
  __device__ __forceinline__ void add(int p, int v) const { atomicAdd(n + p, v); }
};

// Entry j of row `row`, which was `was` and continues row par's len tokens (par -1: an empty row): table_out's, and the references of
// what the entry was and is, where the two differ.
template <bool LDS>
__device__ __forceinline__ void carry_entry(const ForkArgs& a, const Count<LDS>& count, int row, int j, int was, int par, int len) {
  int is = -1;
  const bool gone = a.window && j * PAGE >= a.sinks && j * PAGE + PAGE - 1 <= len - a.window;
  if (par >= 0 && j < (len + PAGE - 1) / PAGE && !gone) is = a.table[(long long)par * a.slots + j];
  if (is < 0 || is >= a.pages) is = -1;
  if (was < -1 || was >= a.pages) {
    raise_flag(a.flags, FLAG_CACHE);
    was = -1;
  }
  if (row < a.seqs_out) a.table_out[(long long)row * a.slots + j] = is;
  if (was == is) return;
  if (was >= 0) count.add(was, -1);
  if (is >= 0) count.add(is, 1);
}

// Larger tables: counts that start as refs, and the entries, by as many workgroups as there are rows or more.
__global__ __launch_bounds__(256) void fork_refs_kernel(ForkArgs a) {
  for (int p = (int)blockIdx.x * 256 + (int)threadIdx.x; p < a.pages; p += (int)gridDim.x * 256) a.refs_out[p] = a.refs[p];
}
__global__ __launch_bounds__(256) void fork_entries_kernel(ForkArgs a) {
  const int row = blockIdx.y;
  int par = -1, len = 0;
  if (row < a.seqs_out) par = a.parent ? a.parent[row] : row;
  if (par >= a.seqs) par = -1;
  if (par >= 0) len = a.lens[par];
  if (len < 0 || len > a.slots * PAGE) len = 0;          // reported with the rows
  for (int j = (int)blockIdx.x * 256 + (int)threadIdx.x; j < a.slots; j += (int)gridDim.x * 256)
    carry_entry(a, Count<false>{a.refs_out}, row, j, row < a.seqs ? a.table[(long long)row * a.slots + j] : -1, par, len);
}

// Tables of at most so many entries are one workgroup's, with counts in LDS. A step of 64 rows with one workgroup and with many: 8.7 us
// and 12.9 with 16 entries a row, 16.5 and 13.9 with 256, 60 and 14.2 with 2048.
constexpr int FORK_LDS_ENTRIES = 8192;
constexpr int FORK_LDS_PAGES = 12288;                    // 96 KiB of counts and free pages beside 48 KiB of rows
constexpr int ROWS_EACH = ANVIL_CACHE_ROWS_MAX / META;

// A step's tables by one workgroup, or (LDS false) what is left when fork_entries_kernel has carried the entries: copies and new pages
// row by row, lowest free page first. A thread's rows stay in its registers. What it takes are the waits for memory one behind the
// other: parents, lengths, entries, and what is written in the end.
template <bool LDS>
__global__ __launch_bounds__(META) void fork_kernel(ForkArgs a) {
  extern __shared__ int pages_lds[];
  __shared__ int last[ANVIL_CACHE_ROWS_MAX];             // the shared-candidate page that a row extends into, -1 none
  __shared__ int2 rows[ANVIL_CACHE_ROWS_MAX];            // parent (-1: none), length
  __shared__ int bad, copied;                            // FLAG_* bits of what rules the step out; pages copied so far
  constexpr int EACH = LDS ? FORK_LDS_ENTRIES / META : 1;
  int was[EACH];                                         // on their way beside the rows
  if constexpr (LDS) {
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int i = (int)threadIdx.x + k * META;
      was[k] = i < a.seqs * a.slots ? a.table[i] : -1;
    }
  }
  const Count<LDS> count{LDS ? pages_lds : a.refs_out};
  int* list = LDS ? pages_lds + a.pages : a.list;        // free pages in order
  const int tid = threadIdx.x;
  if (tid == 0) bad = 0, copied = 0;
  int par[ROWS_EACH], len[ROWS_EACH], add[ROWS_EACH];
#pragma unroll
  for (int k = 0; k < ROWS_EACH; ++k) {
    const int row = tid + k * META;
    par[k] = -1, len[k] = 0, add[k] = 0;
    if (row < a.seqs_out) {
      par[k] = a.parent ? a.parent[row] : row;
      add[k] = a.add ? a.add[row] : 0;
    }
  }
  if constexpr (LDS)
    for (int p = tid; p < a.pages; p += META) count.set(p, a.refs[p]);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ROWS_EACH; ++k) {
    const int row = tid + k * META;
    if (row >= a.seqs_out) break;
    unsigned wrong = 0;
    if (par[k] < -1 || par[k] >= a.seqs) par[k] = -1, raise_flag(a.flags, FLAG_CACHE);
    if (par[k] < 0) {
      add[k] = 0;
    } else {
      len[k] = a.lens[par[k]];
      if (len[k] < 0 || len[k] > a.slots * PAGE || add[k] < 0) wrong = FLAG_CACHE;
      else if ((long long)len[k] + add[k] > a.slots * PAGE) wrong = FLAG_PAGES;
    }
    if (wrong) {
      atomicOr(&bad, (int)wrong);
      raise_flag(a.flags, wrong);
      len[k] = 0, add[k] = 0;
    }
    rows[row] = {par[k], len[k]};
    last[row] = -1;
    if (add[k] > 0 && len[k] % PAGE) last[row] = a.table[(long long)par[k] * a.slots + len[k] / PAGE];
  }
  const int out_entries = a.seqs_out * a.slots;
  __syncthreads();
  if constexpr (LDS) {
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int i = tid + k * META, row = i / a.slots;
      if (i >= max(a.seqs, a.seqs_out) * a.slots) break;
      const int2 r = row < a.seqs_out ? rows[row] : int2{-1, 0};
      carry_entry(a, count, row, i - row * a.slots, was[k], r.x, r.y);
    }
    __syncthreads();
  }
  // pages wanted by each row, in order; the copies first
  int wanted = 0, from[ROWS_EACH];
  bool copy[ROWS_EACH];
#pragma unroll
  for (int k = 0; k < ROWS_EACH; ++k) {
    if (k * META >= a.seqs_out) break;
    const int row = tid + k * META, page = row < a.seqs_out ? last[row] : -1;
    copy[k] = false;
    if (page >= 0 && page < a.pages) {
      int others = count.get(page) - 1;                  // sharers that have not copied by then
      if (others > 0) {
        for (int i = 0; i < row; ++i) others -= last[i] == page;
        copy[k] = others > 0;
      }
    }
    int total;
    from[k] = wanted + prefix((len[k] + add[k] + PAGE - 1) / PAGE - (len[k] + PAGE - 1) / PAGE + copy[k], total);
    wanted += total;
  }
  // the first `wanted` free pages, a run of RUN a thread at a time
  constexpr int RUN = LDS ? 2 : 8;
  int found = 0;
  if (!bad)
    for (int p0 = 0; found < wanted && p0 < a.pages; p0 += META * RUN) {
      int free = 0;
      const int p = p0 + RUN * tid;
#pragma unroll
      for (int k = 0; k < RUN; ++k) free |= (p + k < a.pages && count.get(p + k) == 0) << k;
      int all;
      int at = found + prefix(__builtin_popcount(free), all);
      found += all;
      for (; free && at < wanted; free &= free - 1) list[at++] = p + __builtin_ctz(free);
    }
  const bool fail = bad || found < wanted;
  __syncthreads();
  if (fail) {
    if (tid == 0 && !bad) raise_flag(a.flags, FLAG_PAGES);
    for (int i = tid; i < out_entries; i += META) a.table_out[i] = -1;
    for (int row = tid; row < a.seqs_out; row += META) a.lens_out[row] = 0;
    if (tid == 0) *a.n = 0;
    for (int p = tid; p < a.pages; p += META) a.refs_out[p] = a.refs[p];
    return;
  }
#pragma unroll
  for (int k = 0; k < ROWS_EACH; ++k) {
    const int row = tid + k * META;
    if (row >= a.seqs_out) break;
    const int* take = list + from[k];
    int* entries = a.table_out + (long long)row * a.slots;
    if (copy[k]) {
      const int2 pair = {last[row], *take++};
      entries[len[k] / PAGE] = pair.y;
      count.add(pair.x, -1);
      count.set(pair.y, 1);
      a.copies[atomicAdd(&copied, 1)] = pair;            // in any order: no page is in two of them but as a source
    }
    for (int j = (len[k] + PAGE - 1) / PAGE; j < (len[k] + add[k] + PAGE - 1) / PAGE; ++j) {
      entries[j] = *take;
      count.set(*take++, 1);
    }
    a.lens_out[row] = len[k] + add[k];
  }
  __syncthreads();
  if (tid == 0) *a.n = copied;
  if constexpr (LDS)
    for (int p = tid; p < a.pages; p += META) a.refs_out[p] = count.get(p);
}

struct CompactArgs {
  const int *table, *lens, *refs;
  int *table_out, *lens_out, *refs_out, *map;
  int2* moves;                                           // scratch: (from, to), `*n` of them
  int* n;
  int seqs, slots, pages;
  unsigned* flags;
};

// map and refs_out by one workgroup, a run of pages a thread at a time: first how many are used, then each place. A call on 105000 pages
// takes 135 us, 301 with one long run a thread.
__global__ __launch_bounds__(META) void compact_map_kernel(CompactArgs a) {
  constexpr int RUN = 4;
  const int tid = threadIdx.x;
  int used = 0, n;
  for (int p0 = RUN * tid; p0 < a.pages; p0 += RUN * META)
#pragma unroll
    for (int k = 0; k < RUN; ++k) used += p0 + k < a.pages && a.refs[p0 + k] > 0;
  prefix(used, n);
  int holes = 0, movers = 0;                             // holes below n, used pages from n on
  for (int p0 = 0; p0 < a.pages; p0 += RUN * META) {
    int refs[RUN], count = 0, total;                     // of movers in the upper half
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      const int p = p0 + RUN * tid + k;
      refs[k] = p < a.pages ? a.refs[p] : 0;
      if (p < a.pages) count += p < n ? refs[k] <= 0 : (refs[k] > 0) << 16;
    }
    const int before = prefix(count, total);
    int hole = holes + (before & 0xFFFF), mover = movers + (before >> 16);
    holes += total & 0xFFFF, movers += total >> 16;
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      const int p = p0 + RUN * tid + k;
      if (p >= a.pages) break;
      if (refs[k] > 0 && p >= n) a.moves[mover++].x = p;
      else if (refs[k] <= 0 && p < n) a.moves[hole++].y = p;
      if (refs[k] > 0 && p < n) a.map[p] = p, a.refs_out[p] = refs[k];
      if (refs[k] <= 0) a.map[p] = -1;
      if (p >= n) a.refs_out[p] = 0;
    }
  }
  __syncthreads();
  for (int i = tid; i < movers; i += META) {
    const int2 m = a.moves[i];
    a.map[m.x] = m.y;
    a.refs_out[m.y] = a.refs[m.x];
  }
  if (tid == 0) *a.n = movers;
}

// Pages pairs[i].x -> pairs[i].y of every layer (blockIdx: part of a page, pair, striding, layer).
// 16 bytes a thread: with four of them, loads before stores, a compaction of 156 MB ran in 76.5 us instead of 63.2.
constexpr int COPY_THREADS = 256;
struct CopyArgs {
  uint8_t* pool;
  const int2* pairs;
  const int* n;
  int pages, page_bytes, step;                           // step: workgroups of a part and layer
};
__device__ __forceinline__ void copy_pages(const CopyArgs& a) {
  const long long layer = (long long)blockIdx.z * a.pages;
  const int at = (int)blockIdx.x * COPY_THREADS + (int)threadIdx.x, n = *a.n;
  int2 pair = a.pairs[blockIdx.y];                       // beside n: there is room for a pair each
  if (at >= a.page_bytes / 16) return;
  for (int i = blockIdx.y; i < n; i += a.step) {
    if (i != (int)blockIdx.y) pair = a.pairs[i];
    ((uint4*)(a.pool + (layer + pair.y) * a.page_bytes))[at] = ((const uint4*)(a.pool + (layer + pair.x) * a.page_bytes))[at];
  }
}

__global__ __launch_bounds__(COPY_THREADS) void fork_copy_kernel(CopyArgs a) { copy_pages(a); }

// The moved pages, and by the workgroups behind them (blockIdx.y = step) the tables, which the map now tells.
__global__ __launch_bounds__(COPY_THREADS) void compact_move_kernel(CopyArgs a, CompactArgs t) {
  if ((int)blockIdx.y < a.step) {
    copy_pages(a);
    return;
  }
  // parts x layers x COPY_THREADS passes 2^31 in a pool of few large pages
  const long long step = (long long)gridDim.x * gridDim.z * COPY_THREADS;
  const int entries = t.seqs * t.slots;
  for (long long at = ((long long)blockIdx.z * gridDim.x + blockIdx.x) * COPY_THREADS + threadIdx.x; at < entries; at += step) {
    const int i = (int)at;
    const int p = t.table[i];
    int to = -1;
    if (p >= 0 && p < t.pages) to = t.map[p];
    if (p != -1 && to < 0) raise_flag(t.flags, FLAG_CACHE);                      // out of range, or a page nothing counts
    t.table_out[i] = to;
    if (i % t.slots == 0) t.lens_out[i / t.slots] = t.lens[i / t.slots];
  }
}

static int check_pair(const char* who, const anvil_cache* in, const anvil_cache* out) {
  if (int r = check_cache(who, in, true)) return r;
  if (int r = check_cache(who, out, true)) return r;
  if (in->pool != out->pool || in->slots != out->slots || in->pages != out->pages || in->heads != out->heads ||
      in->dim != out->dim || in->layers != out->layers)
    return set_error(ANVIL_E_VALUE, "%s: both caches must share one pool, its shape and their slots", who);
  if (in->seqs > ANVIL_CACHE_ROWS_MAX || out->seqs > ANVIL_CACHE_ROWS_MAX)
    return set_error(ANVIL_E_VALUE, "%s: %d and %d rows, at most %d", who, in->seqs, out->seqs, ANVIL_CACHE_ROWS_MAX);
  const auto apart = [](const int* a, long long na, const int* b, long long nb) {
    return !na || !nb || (uintptr_t)(a + na) <= (uintptr_t)b || (uintptr_t)(b + nb) <= (uintptr_t)a;
  };
  const int* ins[3] = {in->table, in->lens, in->refs};
  const int* outs[3] = {out->table, out->lens, out->refs};
  const long long ni[3] = {(long long)in->seqs * in->slots, in->seqs, in->pages};
  const long long no[3] = {(long long)out->seqs * out->slots, out->seqs, out->pages};
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 3; ++j)
      if (!apart(ins[i], ni[i], outs[j], no[j]))
        return set_error(ANVIL_E_VALUE, "%s: the tables written overlap those read", who);
  return ANVIL_OK;
}

// The copies of at most so many pairs, and their grid. A step copies little, and 278000 workgroups that find nothing to do take 60 us
// (512 rows of 32 layers, 8 heads of 128: 73 us a step, 14 with at most 16384); a compaction of 400 pages of 12 layers takes 63.9 us
// with 16384 workgroups, 66.3 with half or twice as many, 74 with one a pair.
constexpr int COPY_GROUPS = 16384;
static dim3 copy_grid(const anvil_cache* c, const int2* pairs, const int* n, int most, CopyArgs* a) {
  *a = {(uint8_t*)c->pool, pairs, n, c->pages, c->heads * 2176 * groups_of(c->dim), 0};
  const int parts = (a->page_bytes + 16 * COPY_THREADS - 1) / (16 * COPY_THREADS);
  a->step = (int)std::max<long long>(1, std::min<long long>(most, COPY_GROUPS / ((long long)parts * c->layers)));
  return dim3((unsigned)parts, (unsigned)a->step, (unsigned)c->layers);
}

}  // namespace anvil

using namespace anvil;

extern "C" {

int anvil_cache_bytes(int layers, int pages, int heads, int dim, long long* bytes) {
  if (!bytes) return set_error(ANVIL_E_VALUE, "anvil_cache_bytes: null output pointer");
  *bytes = 0;
  if (dim != 16 && dim != 32 && dim != 64 && dim != 128)
    return set_error(ANVIL_E_VALUE, "anvil_cache_bytes: head dim %d is not 16, 32, 64 or 128", dim);
  if (layers < 1 || layers > 65535 || pages < 1 || pages > (1 << 24) || heads < 1 || heads > 4096)
    return set_error(ANVIL_E_VALUE, "anvil_cache_bytes: %d layers of %d pages of %d heads", layers, pages, heads);
  *bytes = (long long)layers * pages * heads * 2176 * groups_of(dim);
  return ANVIL_OK;
}

int anvil_cache_append_i4(anvil_ctx* ctx, const anvil_cache* cache, int layer, const int8_t* K, const int8_t* V,
                          const int32_t* starts, int rows, int max_new, const int64_t* strides) {
  return rows_call("anvil_cache_append_i4", ctx, cache, layer, K, V, starts, rows, max_new, strides, true);
}

int anvil_cache_read_i4(anvil_ctx* ctx, const anvil_cache* cache, int layer, int8_t* K, int8_t* V, const int32_t* starts,
                        int rows, int max_new, const int64_t* strides) {
  return rows_call("anvil_cache_read_i4", ctx, cache, layer, K, V, starts, rows, max_new, strides, false);
}

int anvil_embed_quantize_new(anvil_ctx* ctx, const anvil_cache* cache, const int32_t* ids, const int32_t* starts, int rows,
                             int max_new, int C, const float* wte, int vocab, const float* wpe, int positions, double scale,
                             void* out, int out_dtype) {
  const char* who = "anvil_embed_quantize_new";
  CacheView c;
  if (int r = cache_view(who, ctx, cache, 0, starts, rows, max_new, &c)) return r;
  if (C < 1 || vocab < 1 || positions < 1)
    return set_error(ANVIL_E_VALUE, "%s: C %d, vocab %d, positions %d", who, C, vocab, positions);
  if (!(scale > 0) || std::isinf(scale)) return set_error(ANVIL_E_VALUE, "%s: scale must be > 0", who);
  if (out_dtype != ANVIL_I8 && out_dtype != ANVIL_I16) return set_error(ANVIL_E_VALUE, "%s: result dtype must be i8 or i16", who);
  if (!c.seqs || !rows) return check_ctx(ctx);
  if (!ids || !wte || !wpe || !out) return set_error(ANVIL_E_VALUE, "%s: null pointer", who);
  if ((uintptr_t)ids % 4 || (uintptr_t)wte % 4 || (uintptr_t)wpe % 4 || (uintptr_t)out % out_dtype)
    return set_error(ANVIL_E_VALUE, "%s: a pointer is not aligned to its type", who);
  if (int r = check_ctx(ctx)) return r;
  const EmbedArgs e{ids, wte, wpe, C, vocab, positions, dtype_lo(out_dtype), dtype_hi(out_dtype), scale};
  const dim3 grid((unsigned)std::min(c.max_new, 4096), (unsigned)c.seqs);
  if (out_dtype == ANVIL_I8) ANVIL_LAUNCH(embed_new_kernel<int8_t>, grid, dim3(256), 0, ctx->stream, c, e, (int8_t*)out);
  else ANVIL_LAUNCH(embed_new_kernel<int16_t>, grid, dim3(256), 0, ctx->stream, c, e, (int16_t*)out);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}

int anvil_cache_fork(anvil_ctx* ctx, const anvil_cache* in, const anvil_cache* out, const int32_t* parent,
                     const int32_t* add, int window, int sinks) {
  if (int r = check_pair("anvil_cache_fork", in, out)) return r;
  if (window < 0 || sinks < 0) return set_error(ANVIL_E_VALUE, "anvil_cache_fork: window %d, sinks %d", window, sinks);
  if (!parent && in->seqs != out->seqs)
    return set_error(ANVIL_E_VALUE, "anvil_cache_fork: without parents both caches have the same rows (%d, %d)", in->seqs,
                     out->seqs);
  if ((uintptr_t)parent % 4 || (uintptr_t)add % 4) return set_error(ANVIL_E_VALUE, "anvil_cache_fork: parent or add is not aligned");
  if (int r = check_ctx(ctx)) return r;
  char* ws;
  const size_t pairs = (sizeof(int2) * (size_t)out->seqs + 255) / 256 * 256;
  if (int r = decode_workspace(ctx, 256 + pairs + sizeof(int) * (size_t)in->pages, &ws)) return r;
  int* copied = (int*)ws;
  ws += 256;
  ForkArgs a{in->table, in->lens, in->refs, parent, add, out->table, out->lens, out->refs,
             (int*)(ws + pairs), (int2*)ws, copied,
             in->seqs, out->seqs, in->slots, in->pages, window, sinks, ctx->flags};
  const int rows = std::max(in->seqs, out->seqs);
  if (in->pages <= FORK_LDS_PAGES && (long long)rows * in->slots <= FORK_LDS_ENTRIES) {
    ANVIL_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(fork_kernel<true>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                  2 * sizeof(int) * FORK_LDS_PAGES));
    ANVIL_LAUNCH(fork_kernel<true>, dim3(1), dim3(META), 2 * sizeof(int) * in->pages, ctx->stream, a);
  } else {
    ANVIL_LAUNCH(fork_refs_kernel, dim3((unsigned)std::min(1024, (in->pages + 255) / 256)), dim3(256), 0, ctx->stream, a);
    ANVIL_LAUNCHED();
    if (rows) {
      ANVIL_LAUNCH(fork_entries_kernel, dim3((unsigned)(in->slots + 255) / 256, (unsigned)rows), dim3(256), 0, ctx->stream, a);
      ANVIL_LAUNCHED();
    }
    ANVIL_LAUNCH(fork_kernel<false>, dim3(1), dim3(META), 0, ctx->stream, a);
  }
  ANVIL_LAUNCHED();
  if (!add || !out->seqs) return ANVIL_OK;
  CopyArgs copy;
  const dim3 grid = copy_grid(out, a.copies, copied, out->seqs, &copy);
  ANVIL_LAUNCH(fork_copy_kernel, grid, dim3(COPY_THREADS), 0, ctx->stream, copy);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}

int anvil_cache_compact(anvil_ctx* ctx, const anvil_cache* in, const anvil_cache* out, int32_t* map) {
  if (int r = check_pair("anvil_cache_compact", in, out)) return r;
  if (in->seqs != out->seqs) return set_error(ANVIL_E_VALUE, "anvil_cache_compact: %d rows into %d", in->seqs, out->seqs);
  if (!map || (uintptr_t)map % 4) return set_error(ANVIL_E_VALUE, "anvil_cache_compact: map must be aligned and not null");
  if (int r = check_ctx(ctx)) return r;
  char* ws;
  const size_t moves = (sizeof(int2) * (size_t)in->pages + 255) / 256 * 256;
  if (int r = decode_workspace(ctx, moves + 256, &ws)) return r;
  CompactArgs a{in->table, in->lens, in->refs, out->table, out->lens, out->refs, map, (int2*)ws, (int*)(ws + moves),
                in->seqs, in->slots, in->pages, ctx->flags};
  ANVIL_LAUNCH(compact_map_kernel, dim3(1), dim3(META), 0, ctx->stream, a);
  ANVIL_LAUNCHED();
  CopyArgs copy;
  dim3 grid = copy_grid(in, a.moves, a.n, in->pages / 2, &copy);                 // at most half of the pages have a hole before them
  ++grid.y;                                              // the tables
  ANVIL_LAUNCH(compact_move_kernel, grid, dim3(COPY_THREADS), 0, ctx->stream, copy, a);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}

}  // extern "C"
