// The 4-bit paged cache as its kernels see it: layout of a page, rows of new tokens, argument checks.
#pragma once

#include "common.h"

namespace anvil {

constexpr int PAGE = ANVIL_CACHE_PAGE;
constexpr int PAGE_SHIFT = 6;
static_assert(PAGE == 1 << PAGE_SHIFT, "a page is a power of two");
constexpr int STEP_MAX = 18;                             // 7 x 18 = 126 is the largest multiple of 7 in an int8

// One head's block of a page for NG groups of 32 channels: byte offsets (anvil_mi355x.h has the order within each part).
template <int NG>
struct Block {
  static constexpr int ROW = 16 * NG;                    // bytes of one token's K codes
  static constexpr int K = 0, K_STEPS = PAGE * ROW, V = K_STEPS + PAGE * NG, V_STEPS = V + PAGE * ROW,
                       BYTES = V_STEPS + PAGE * NG;
  static_assert(BYTES == 68 * 32 * NG, "68 bytes a channel");
};
inline int groups_of(int dim) { return dim <= 32 ? 1 : dim / 32; }

// One layer of a cache, and the rows of new tokens (anvil_cache_append_i4 and its kind), by value.
struct CacheView {
  uint8_t* pool;
  const int* table;
  const int* lens;
  const int* starts;                                     // null: one row a sequence that is not empty
  int seqs, slots, pages, heads, dim, rows, max_new;
  unsigned* flags;
};

struct NewRows {
  int first, n, len;                                     // packed rows first .. first + n - 1, positions len - n .. len - 1
};

// The new rows of sequence s; false (and n = 0) where the caller's numbers leave their range, which `report` reports.
__device__ __forceinline__ bool new_rows(const CacheView& c, int s, NewRows& r, bool report) {
  const int lo = c.starts ? c.starts[s] : s, hi = c.starts ? c.starts[s + 1] : s + 1;
  r.len = c.lens[s];
  r.first = lo;
  r.n = 0;
  if (!c.starts && r.len == 0) return true;              // an empty sequence has no row
  const bool ok = lo >= 0 && hi >= lo && hi <= c.rows && hi - lo <= c.max_new && r.len >= 0 &&
                  r.len <= c.slots * PAGE && hi - lo <= r.len;
  if (ok) r.n = hi - lo;
  else if (report) raise_flag(c.flags, FLAG_CACHE);
  return ok;
}

// The block of head h in the page of slot j of sequence s; null where the table names none.
template <int NG>
__device__ __forceinline__ uint8_t* page_block(const CacheView& c, int s, int j, int h, bool report) {
  const int p = c.table[(long long)s * c.slots + j];
  if (p < 0 || p >= c.pages) {
    if (report && p != -1) raise_flag(c.flags, FLAG_CACHE);
    return nullptr;
  }
  return c.pool + ((long long)p * c.heads + h) * Block<NG>::BYTES;
}

// argument checks shared by the entry points
int check_cache(const char* who, const anvil_cache* c, bool refs);
int cache_view(const char* who, anvil_ctx* ctx, const anvil_cache* c, int layer, const int32_t* starts, int rows,
               int max_new, CacheView* v);

// f(std::integral_constant<int, NG>) for the head dims of a cache
template <typename F>
void by_groups(int dim, F&& f) {
  switch (groups_of(dim)) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    default: return f(std::integral_constant<int, 4>{});
  }
}

}  // namespace anvil
