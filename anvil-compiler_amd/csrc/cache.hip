// The 4-bit paged cache: new rows rounded into their pages, read back, and the page tables of the next step.
#include <algorithm>

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
  v->rows = rows, v->max_new = max_new, v->flags = ctx ? ctx->flags : nullptr;
  return ANVIL_OK;
}

// ------------------------------------------------------------------------------------------- append and read

struct RowPtrs {
  int8_t *k, *v;
  long long k_row, k_head, v_row, v_head;
};

// Eight consecutive channels as 4-bit codes and their group's step: lanes 4 i .. 4 i + 3 hold a group's 32 channels.
// code + 8 = floor((2 x + 17 step) / (2 step)) with a positive numerator n <= 562; its quotient by d = 2 step <= 36 is
// (n ceil(2^16 / d)) >> 16, exact as n d < 2^16. The dword's nibble e is channel e's code.
__device__ __forceinline__ unsigned round4(uint2 x, int& step) {
  int v[8], a = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = (int8_t)((e < 4 ? x.x : x.y) >> (8 * (e & 3)));
    a = max(a, abs(v[e]));
  }
  a = max(a, (int)__builtin_amdgcn_update_dpp(0, a, 0xB1, 0xF, 0xF, false));     // quad_perm [1,0,3,2]
  a = max(a, (int)__builtin_amdgcn_update_dpp(0, a, 0x4E, 0xF, 0xF, false));     // quad_perm [2,3,0,1]
  step = min(STEP_MAX, max(1, (a + 6) / 7));
  const unsigned m = (65535u + 2u * step) / (2u * step);
  unsigned w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int code = (int)(((unsigned)(2 * v[e] + 17 * step) * m) >> 16) - 8;
    w |= ((unsigned)min(7, max(-7, code)) & 15u) << (4 * e);
  }
  return w;
}

// nibbles 0..3 of w into the low halves of four bytes, nibbles 4..7 into the high ones: the K code order
__device__ __forceinline__ unsigned interleave_k(unsigned w) {
  unsigned d = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) d |= (((w >> (4 * i)) & 15u) | ((w >> (12 + 4 * i)) & 0xF0u)) << (8 * i);
  return d;
}

constexpr int ROW_THREADS = 256;

// One page of one sequence and head a workgroup (blockIdx: page among those with new rows, sequence, head). Four
// lanes a group of 32 channels. K codes go straight to their rows; V codes, which the page holds channel by channel, meet
// in LDS and leave as whole 64-byte rows where the page is new from end to end.
template <int NG>
__global__ __launch_bounds__(ROW_THREADS) void append_kernel(CacheView c, RowPtrs p) {
  using B = Block<NG>;
  const int s = blockIdx.y, h = blockIdx.z, tid = threadIdx.x;
  NewRows r;
  new_rows(c, s, r, blockIdx.x == 0 && h == 0 && tid == 0);
  const int begin = r.len - r.n, slot = (begin >> PAGE_SHIFT) + (int)blockIdx.x;
  const int t0 = max(begin - slot * PAGE, 0), t1 = min(r.len - slot * PAGE, PAGE);
  if (r.n == 0 || t1 <= 0) return;
  uint8_t* blk = page_block<NG>(c, s, slot, h, tid == 0);
  if (!blk) {
    if (tid == 0) raise_flag(c.flags, FLAG_CACHE);
    return;
  }
  __shared__ __align__(16) uint8_t vt[16 * NG][PAGE];
  const long long row0 = (long long)r.first + slot * PAGE - begin;               // the row of the page's token 0
  const int items = (t1 - t0) * NG * 4;
  for (int i = tid; i < (items + 63) / 64 * 64; i += ROW_THREADS) {              // whole waves: lanes exchange values
    const bool on = i < items;
    const int t = t0 + (on ? i / (NG * 4) : 0), g = (i / 4) % NG, q = i & 3;
    const bool real = on && 32 * g + 8 * q < c.dim;
    uint2 xk = {0, 0}, xv = {0, 0};
    if (real) {
      xk = *(const uint2*)(p.k + (row0 + t) * p.k_row + h * p.k_head + 32 * g + 8 * q);
      xv = *(const uint2*)(p.v + (row0 + t) * p.v_row + h * p.v_head + 32 * g + 8 * q);
    }
    int sk, sv;
    const unsigned wk = round4(xk, sk), wv = round4(xv, sv);
    const unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)wv, 0x4E, 0xF, 0xF, false);   // lane q ^ 2
    if (!on) continue;
    *(unsigned*)(blk + B::K + t * B::ROW + 4 * (q * NG + g)) = interleave_k(wk);
    // lane q holds channels 8 q .. of the group: with q ^ 2 it has both halves of V bytes i = 8 (q & 1) .., four each
    const unsigned low = q < 2 ? wv : other >> 16, high = q < 2 ? other : wv >> 16;
    const int i0 = 8 * (q & 1) + (q < 2 ? 0 : 4);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      vt[16 * g + i0 + e][t] = (uint8_t)(((low >> (4 * e)) & 15u) | (((high >> (4 * e)) & 15u) << 4));
    if (q == 0) {
      blk[B::K_STEPS + ((t >> 2) * NG + g) * 4 + (t & 3)] = (uint8_t)sk;
      blk[B::V_STEPS + PAGE * g + t] = (uint8_t)sv;
    }
  }
  __syncthreads();
  if (t1 - t0 == PAGE) {
    for (int i = tid; i < 16 * NG * 4; i += ROW_THREADS)
      *(uint4*)(blk + B::V + 16 * i) = *(const uint4*)(&vt[i >> 2][16 * (i & 3)]);
  } else {
    for (int i = tid; i < 16 * NG * (t1 - t0); i += ROW_THREADS) {
      const int j = i / (t1 - t0), t = t0 + i % (t1 - t0);
      blk[B::V + j * PAGE + t] = vt[j][t];
    }
  }
}

__device__ __forceinline__ int code_of(unsigned w, int e) { return (int)(w << (28 - 4 * e)) >> 28; }

// The values of the same rows, one page of one sequence and head a workgroup.
template <int NG>
__global__ __launch_bounds__(ROW_THREADS) void read_kernel(CacheView c, RowPtrs p) {
  using B = Block<NG>;
  const int s = blockIdx.y, h = blockIdx.z, tid = threadIdx.x;
  NewRows r;
  new_rows(c, s, r, blockIdx.x == 0 && h == 0 && tid == 0);
  const int begin = r.len - r.n, slot = (begin >> PAGE_SHIFT) + (int)blockIdx.x;
  const int t0 = max(begin - slot * PAGE, 0), t1 = min(r.len - slot * PAGE, PAGE);
  if (r.n == 0 || t1 <= 0) return;
  const uint8_t* blk = page_block<NG>(c, s, slot, h, tid == 0);
  const long long row0 = (long long)r.first + slot * PAGE - begin;
  for (int i = tid; i < (t1 - t0) * NG * 4; i += ROW_THREADS) {
    const int t = t0 + i / (NG * 4), g = (i / 4) % NG, q = i & 3;
    if (32 * g + 8 * q >= c.dim) continue;
    uint2 xk = {0, 0}, xv = {0, 0};                                              // a page given back reads as zeros
    if (blk) {
      const unsigned wk = *(const unsigned*)(blk + B::K + t * B::ROW + 4 * (q * NG + g));
      const int sk = blk[B::K_STEPS + ((t >> 2) * NG + g) * 4 + (t & 3)], sv = blk[B::V_STEPS + PAGE * g + t];
      unsigned k[8], v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        k[e] = (unsigned)(code_of(wk, 2 * (e & 3) + (e >> 2)) * sk) & 255u;
        const unsigned b = blk[B::V + (16 * g + 8 * (q & 1) + e) * PAGE + t];
        v[e] = (unsigned)(code_of(b, q >> 1) * sv) & 255u;
      }
      xk = {k[0] | k[1] << 8 | k[2] << 16 | k[3] << 24, k[4] | k[5] << 8 | k[6] << 16 | k[7] << 24};
      xv = {v[0] | v[1] << 8 | v[2] << 16 | v[3] << 24, v[4] | v[5] << 8 | v[6] << 16 | v[7] << 24};
    }
    *(uint2*)(p.k + (row0 + t) * p.k_row + h * p.k_head + 32 * g + 8 * q) = xk;
    *(uint2*)(p.v + (row0 + t) * p.v_row + h * p.v_head + 32 * g + 8 * q) = xv;
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
  const dim3 grid((unsigned)((max_new + PAGE - 2) / PAGE + 1), (unsigned)c.seqs, (unsigned)c.heads);
  by_groups(c.dim, [&](auto ng) {
    constexpr int NG = decltype(ng)::value;
    ANVIL_LAUNCH(write ? append_kernel<NG> : read_kernel<NG>, grid, dim3(ROW_THREADS), 0, ctx->stream, c, p);
  });
  ANVIL_LAUNCHED();
  return ANVIL_OK;
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
  int *count, *list;                                     // scratch: references of each page (pages), free pages in order
  int2* copies;                                          // scratch: (from, to) page of each row, from = -1: none
  int seqs, seqs_out, slots, pages, window, sinks;
  unsigned* flags;
};

__device__ __forceinline__ int counted(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The whole step's tables by one workgroup: a few thousand entries, whose order (references, then copies and new pages row
// by row, lowest free page first) would need a launch for each step otherwise.
__global__ __launch_bounds__(META) void fork_kernel(ForkArgs a) {
  __shared__ int last[ANVIL_CACHE_ROWS_MAX];             // the shared-candidate page that a row extends into, -1 none
  __shared__ int bad;                                    // FLAG_* bits of what rules the step out
  const int tid = threadIdx.x;
  if (tid == 0) bad = 0;
  for (int p = tid; p < a.pages; p += META) atomicExch(&a.count[p], a.refs[p]);
  __syncthreads();
  const int in_entries = a.seqs * a.slots, out_entries = a.seqs_out * a.slots;
  for (int i = tid; i < in_entries; i += META) {
    const int p = a.table[i];
    if (p >= 0 && p < a.pages) atomicAdd(&a.count[p], -1);
    else if (p != -1) raise_flag(a.flags, FLAG_CACHE);
  }
  for (int i = tid; i < out_entries; i += META) {
    const int row = i / a.slots, j = i % a.slots;
    const int par = a.parent ? a.parent[row] : row;
    int p = -1;
    if (par >= 0 && par < a.seqs) {
      const int len = a.lens[par];
      const bool used = len >= 0 && j < (len + PAGE - 1) / PAGE;
      const bool gone = a.window && j * PAGE >= a.sinks && j * PAGE + PAGE - 1 <= len - a.window;
      if (used && !gone) p = a.table[(long long)par * a.slots + j];
      if (p < 0 || p >= a.pages) p = -1;
      if (p >= 0) atomicAdd(&a.count[p], 1);
    }
    a.table_out[i] = p;
  }
  __syncthreads();
  // each row's last page, and whether its numbers are in range
  for (int row = tid; row < a.seqs_out; row += META) {
    const int par = a.parent ? a.parent[row] : row;
    int page = -1;
    if (par < -1 || par >= a.seqs) raise_flag(a.flags, FLAG_CACHE);
    if (par >= 0 && par < a.seqs) {
      const int len = a.lens[par], add = a.add ? a.add[row] : 0;
      if (len < 0 || len > a.slots * PAGE || add < 0) {
        atomicOr(&bad, (int)FLAG_CACHE);
      } else if ((long long)len + add > a.slots * PAGE) {
        atomicOr(&bad, (int)FLAG_PAGES);
      } else if (add > 0 && len % PAGE) {
        page = a.table_out[(long long)row * a.slots + len / PAGE];
      }
    }
    last[row] = page;
  }
  __syncthreads();
  // pages wanted by each row, in order; the copies first
  int wanted = 0;
  for (int base = 0; base < a.seqs_out; base += META) {
    const int row = base + tid;
    int need = 0;
    bool copy = false;
    if (row < a.seqs_out && !bad) {
      const int par = a.parent ? a.parent[row] : row;
      if (par >= 0 && par < a.seqs) {
        const int len = a.lens[par], add = a.add ? a.add[row] : 0;
        need = (len + add + PAGE - 1) / PAGE - (len + PAGE - 1) / PAGE;
        const int page = last[row];
        if (page >= 0) {
          int others = counted(&a.count[page]) - 1;                              // sharers that have not copied by then
          if (others > 0) {
            for (int k = 0; k < row; ++k) others -= last[k] == page;
            copy = others > 0;
          }
        }
        need += copy;
      }
      a.copies[row] = {copy ? last[row] : -1, 0};
    }
    int total;
    const int at = prefix(need, total);
    if (row < a.seqs_out) a.lens_out[row] = wanted + at;                         // for now: where the row's pages begin
    wanted += total;
  }
  // the first `wanted` free pages: each thread its run of pages
  const int run = (a.pages + META - 1) / META, lo = min(tid * run, a.pages), hi = min(lo + run, a.pages);
  int free = 0;
  for (int p = lo; p < hi; ++p) free += counted(&a.count[p]) == 0;
  int all;
  int at = prefix(free, all);
  const bool fail = bad || all < wanted;
  if (!fail)
    for (int p = lo; p < hi && at < wanted; ++p)
      if (counted(&a.count[p]) == 0) a.list[at++] = p;
  __syncthreads();
  if (fail) {
    if (tid == 0) raise_flag(a.flags, bad ? (unsigned)bad : (unsigned)FLAG_PAGES);
    for (int i = tid; i < out_entries; i += META) a.table_out[i] = -1;
    for (int row = tid; row < a.seqs_out; row += META) {
      a.lens_out[row] = 0;
      a.copies[row] = {-1, 0};
    }
    for (int p = tid; p < a.pages; p += META) a.refs_out[p] = a.refs[p];
    return;
  }
  for (int row = tid; row < a.seqs_out; row += META) {
    const int par = a.parent ? a.parent[row] : row;
    int from = a.lens_out[row], len = 0;
    if (par >= 0 && par < a.seqs) {
      const int* take = a.list + from;
      len = a.lens[par];
      const int add = a.add ? a.add[row] : 0;
      int* entries = a.table_out + (long long)row * a.slots;
      int2 copy = a.copies[row];
      if (copy.x >= 0) {
        copy.y = *take++;
        a.copies[row] = copy;
        entries[len / PAGE] = copy.y;
        atomicAdd(&a.count[copy.x], -1);
        atomicExch(&a.count[copy.y], 1);
      }
      for (int j = (len + PAGE - 1) / PAGE; j < (len + add + PAGE - 1) / PAGE; ++j) {
        entries[j] = *take;
        atomicExch(&a.count[*take++], 1);
      }
      len += add;
    }
    a.lens_out[row] = len;
  }
  __syncthreads();
  for (int p = tid; p < a.pages; p += META) a.refs_out[p] = counted(&a.count[p]);
}

// Pages copies[i].x -> copies[i].y of every layer (blockIdx: part of a page, pair, layer).
constexpr int COPY_THREADS = 256, COPY_VECS = 4;         // 16 KiB a workgroup
__global__ __launch_bounds__(COPY_THREADS) void copy_pages_kernel(uint8_t* pool, const int2* copies, const int* n, int first,
                                                                  int pages, int page_bytes) {
  const int pair = first + (int)blockIdx.y;
  if (n && pair >= *n) return;
  const int2 c = copies[pair];
  if (c.x < 0) return;
  const long long layer = (long long)blockIdx.z * pages;
  const uint4* src = (const uint4*)(pool + (layer + c.x) * page_bytes);
  uint4* dst = (uint4*)(pool + (layer + c.y) * page_bytes);
  const int vecs = page_bytes / 16, v0 = (int)blockIdx.x * COPY_THREADS * COPY_VECS + (int)threadIdx.x;
  uint4 x[COPY_VECS];
#pragma unroll
  for (int i = 0; i < COPY_VECS; ++i)
    if (v0 + i * COPY_THREADS < vecs) x[i] = src[v0 + i * COPY_THREADS];
#pragma unroll
  for (int i = 0; i < COPY_VECS; ++i)
    if (v0 + i * COPY_THREADS < vecs) dst[v0 + i * COPY_THREADS] = x[i];
}

struct CompactArgs {
  const int *table, *lens, *refs;
  int *table_out, *lens_out, *refs_out, *map;
  int2* moves;                                           // scratch: (from, to), `*n` of them
  int* n;
  int seqs, slots, pages;
  unsigned* flags;
};

// map and refs_out by one workgroup: thread t's run of pages is counted, then placed behind the runs before it.
__global__ __launch_bounds__(META) void compact_map_kernel(CompactArgs a) {
  const int tid = threadIdx.x;
  const int run = (a.pages + META - 1) / META, lo = min(tid * run, a.pages), hi = min(lo + run, a.pages);
  int used = 0;
  for (int p = lo; p < hi; ++p) used += a.refs[p] > 0;
  int n, movers, total;
  prefix(used, n);
  int holes = 0, late = 0;
  for (int p = lo; p < hi; ++p) {
    const bool u = a.refs[p] > 0;
    holes += !u && p < n;
    late += u && p >= n;
  }
  int hole = prefix(holes, total), mover = prefix(late, movers);
  for (int p = lo; p < hi; ++p) {
    const int refs = a.refs[p];
    if (refs > 0 && p >= n) a.moves[mover++].x = p;
    else if (refs <= 0 && p < n) a.moves[hole++].y = p;
    if (refs > 0 && p < n) a.map[p] = p, a.refs_out[p] = refs;
    if (refs <= 0) a.map[p] = -1;
    if (p >= n) a.refs_out[p] = 0;
  }
  __syncthreads();
  for (int i = tid; i < movers; i += META) {
    const int2 m = a.moves[i];
    a.map[m.x] = m.y;
    a.refs_out[m.y] = a.refs[m.x];
  }
  if (tid == 0) *a.n = movers;
}

__global__ __launch_bounds__(256) void compact_table_kernel(CompactArgs a) {
  const int i = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (i < a.seqs * a.slots) {
    const int p = a.table[i];
    int to = -1;
    if (p >= 0 && p < a.pages) to = a.map[p];
    if (p != -1 && to < 0) raise_flag(a.flags, FLAG_CACHE);                      // out of range, or a page nothing counts
    a.table_out[i] = to;
  }
  if (i < a.seqs) a.lens_out[i] = a.lens[i];
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

static int copy_pages(anvil_ctx* ctx, const anvil_cache* c, const int2* copies, const int* n, int pairs) {
  const int page_bytes = c->heads * 2176 * groups_of(c->dim);
  const int per = 16 * COPY_THREADS * COPY_VECS;
  for (int lo = 0; lo < pairs; lo += 65535) {            // a grid dimension's limit
    ANVIL_LAUNCH(copy_pages_kernel, dim3((unsigned)((page_bytes + per - 1) / per), (unsigned)std::min(pairs - lo, 65535),
                 (unsigned)c->layers), dim3(COPY_THREADS), 0, ctx->stream, (uint8_t*)c->pool, copies, n, lo, c->pages, page_bytes);
    ANVIL_LAUNCHED();
  }
  return ANVIL_OK;
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
  if (int r = decode_workspace(ctx, pairs + 2 * sizeof(int) * (size_t)in->pages, &ws)) return r;
  ForkArgs a{in->table, in->lens, in->refs, parent, add, out->table, out->lens, out->refs,
             (int*)(ws + pairs), (int*)(ws + pairs) + in->pages, (int2*)ws,
             in->seqs, out->seqs, in->slots, in->pages, window, sinks, ctx->flags};
  ANVIL_LAUNCH(fork_kernel, dim3(1), dim3(META), 0, ctx->stream, a);
  ANVIL_LAUNCHED();
  return add ? copy_pages(ctx, out, a.copies, nullptr, out->seqs) : ANVIL_OK;
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
  if (in->seqs) {
    const long long n = std::max<long long>((long long)in->seqs * in->slots, in->seqs);
    ANVIL_LAUNCH(compact_table_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, ctx->stream, a);
    ANVIL_LAUNCHED();
  }
  return copy_pages(ctx, in, a.moves, a.n, in->pages / 2);          // at most half of the pages have a hole before them
}

}  // extern "C"
