// Products of sorted rows with their experts' weights, on int8 matrix instructions.
//
// How many rows an expert has is known on the device alone. The grid covers the most tiles there can be (rows / BM + experts, times
// the column tiles), and every workgroup finds its own by a scan over the experts' row counts; those past the last tile end at once. Tiles
// are numbered so that an XCD's are consecutive, in bands of row tiles that share their experts' weights in its L2.
#include <algorithm>

#include "experts.h"
#include "gemm.h"

namespace anvil {

constexpr long long GRID_MAX = (1ll << 24) - 8;          // workgroups of 256: a grid has fewer than 2^32 threads

struct ExpertArgs {
  anvil_expert_gemm g;
  int tiles_n;
  int tiles_m;                                           // as many as `rows` rows of ascending starts can have
  int a_bytes;                                           // of A, as a buffer descriptor takes them: below 2^32
  unsigned* flags;
};

// an offset past an operand's last byte, by more than a row: A and a tile's weights span less
constexpr unsigned PAST = 0xFFF00000u;

struct ExpertTile {
  int e, p0, rows, n0;                                   // expert, first position, rows of the tile, first column
};

// The number of rows of expert e; 0 where its starts leave their range, which `report` reports.
__device__ __forceinline__ int expert_rows(const ExpertArgs& a, int e, bool report, int& lo) {
  lo = a.g.starts[e];
  const int hi = a.g.starts[e + 1];
  if (lo >= 0 && hi >= lo && hi <= a.g.rows) return hi - lo;
  if (report) raise_flag(a.flags, FLAG_EXPERTS);
  return 0;
}

// Tile number `w` of a grid of row tiles of BM x column tiles of BN; false past the last. Starts that decrease (expert_rows reports them) may count
// positions again; where that gives more tiles than the grid was made for there is none at all, rather than those that it reaches.
template <int BM, int BN>
__device__ __forceinline__ bool find_tile(const ExpertArgs& a, int w, int lane, ExpertTile& t) {
  const int E = a.g.experts;
  int lo = 0, n = 0, mt = 0;                             // of the last 64 experts or fewer
  for (int e0 = 0; e0 < E; e0 += 64) {
    n = e0 + lane < E ? expert_rows(a, e0 + lane, w == 0, lo) : 0;
    mt += (n + BM - 1) / BM;
  }
  if (__ballot(mt > (int)GRID_MAX)) return false;        // past what the sums hold
  int incl = wave_scan(mt);
  const int tiles_m = __builtin_amdgcn_readlane(incl, 63);
  if (tiles_m > a.tiles_m) return false;
  const unsigned tiles = (unsigned)tiles_m * (unsigned)a.tiles_n;
  const unsigned per = (tiles + 7) / 8, pid = (w & 7) * per + (w >> 3);
  if ((unsigned)(w >> 3) >= per || pid >= tiles) return false;
  const unsigned in_group = GROUP_M * a.tiles_n;
  const int first_m = (int)(pid / in_group) * GROUP_M, in = (int)(pid % in_group);
  const int gsize = min(tiles_m - first_m, GROUP_M);
  const int gm = first_m + in % gsize;
  t.n0 = in / gsize * BN;
  int before = 0;
  for (int e0 = 0;; e0 += 64) {
    if (E > 64) {
      n = e0 + lane < E ? expert_rows(a, e0 + lane, false, lo) : 0;
      mt = (n + BM - 1) / BM;
      incl = wave_scan(mt);
    }
    const unsigned long long past = __ballot(gm < before + incl);
    if (past || e0 + 64 >= E) {
      const int l = past ? __builtin_ctzll(past) : 63;   // the first expert whose tiles reach past gm
      const int skip = (gm - before - __builtin_amdgcn_readlane(incl - mt, l)) * BM;
      t.e = e0 + l;
      t.p0 = __builtin_amdgcn_readlane(lo, l) + skip;
      t.rows = min(BM, __builtin_amdgcn_readlane(n, l) - skip);
      return past != 0;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
}

// Row i of A for position p; -1 where the caller's number leaves its range.
__device__ __forceinline__ int row_of(const ExpertArgs& a, int p, bool report) {
  const int i = a.g.row ? a.g.row[p] : p;
  if (i >= 0 && i < a.g.rows_a) return i;
  if (report) raise_flag(a.flags, FLAG_EXPERTS);
  return -1;
}

// An expert's multiplier; false where it does not leave room for a row's scale.
__device__ __forceinline__ bool expert_mult(const ExpertArgs& a, const int* mults, int mult, int e, bool report, int& m) {
  m = mults ? mults[e] : mult;
  if (!a.g.scale || (m >= -32767 && m <= 32767)) return true;
  if (report) raise_flag(a.flags, FLAG_EXPERTS);
  return false;
}

// What follows a product's requants: the table, the gated product and the bounds of its value before its shift.
struct Epilogue {
  WideRequant q, q2;
  bool high, lut;
  int mult3, rnd3, shift3, clo3, chi3;
  __device__ __forceinline__ Epilogue(const anvil_expert_gemm& g, int shift, int shift2, int lo)
      : q(shift, lo, -lo - 1), q2(shift2, -128, 127), lut(g.lut != nullptr), mult3(g.mult3), rnd3((int)round_term(g.shift3)), shift3(g.shift3) {
    high = q.high() && q.rest <= 24 && (!g.B2 || q2.high());                   // 24: the table's index is eight bits of an int
    if (!high) q.rest = q2.rest = 0;                     // the 64-bit form shifts by all of it
    clo3 = shift3 < 24 ? -128 * (1 << shift3) : (int)I32_MIN;
    chi3 = shift3 < 24 ? 128 * (1 << shift3) - 1 : (int)I32_MAX;
  }
};

// A lane's results: n accumulators of one row (and n of the gate's partner) as n values of the result's dtype in words.
template <int n, int OSZ, bool GATED, bool HI, typename V>
__device__ __forceinline__ void finish_n(const V& acc, const V& acc2, int m, int m2, const Epilogue& p, const int8_t* lut_s, unsigned* w) {
  int v[n];
#pragma unroll
  for (int e = 0; e < n; ++e) {
    v[e] = p.q.unshifted<HI>(acc[e], m);
    if (OSZ == 1 && (GATED || p.lut)) v[e] = lut_s[__builtin_amdgcn_ubfe((unsigned)v[e], (unsigned)p.q.rest, 8u)];      // rotated: v at index v & 255
    if constexpr (GATED) {
      const int u = p.q2.unshifted<HI>(acc2[e], m2) >> p.q2.rest;
      v[e] = med3i(mad_i24v(__mul24(v[e], u), p.mult3, p.rnd3), p.clo3, p.chi3);
    }
  }
#pragma unroll
  for (int q = 0; q < n / 4; ++q) {
    int* x = v + 4 * q;
    if constexpr (OSZ == 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[2 * q + h] = __builtin_amdgcn_perm((unsigned)(x[2 * h + 1] >> p.q.rest), (unsigned)(x[2 * h] >> p.q.rest), 0x05040100u);
    } else if (GATED) {
      w[q] = sra_pack4(x[0], x[1], x[2], x[3], p.shift3);
    } else if (p.lut) {
      w[q] = pack4(x[0], x[1], x[2], x[3]);
    } else {
      w[q] = sra_pack4(x[0], x[1], x[2], x[3], p.q.rest);
    }
  }
}

// Columns c .. c + n - 1 of the result's row p, those there are, at any alignment: n values in words.
template <int n, int OSZ>
__device__ __forceinline__ void store_n(const anvil_expert_gemm& g, long long p, int c, const unsigned* w) {
  char* out = (char*)g.C + (p * g.ldc + c) * OSZ;
  if (c + n <= g.N) {
    __builtin_memcpy(out, w, n * OSZ);
    return;
  }
#pragma unroll
  for (int e = 0; e < n; ++e)
    if (c + e < g.N) {
      if (OSZ == 1) out[e] = (char)(w[e >> 2] >> (8 * (e & 3)));
      else ((int16_t*)out)[e] = (int16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
}

// sixteen bytes with the first n, if any, zeros
__device__ __forceinline__ v4i without_first(v4i v, int n) {
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] &= n >= 4 * q + 4 ? 0 : n <= 4 * q ? -1 : -1 << (8 * (n - 4 * q));
  return v;
}

// the same address in scalar registers (uniform_rsrc)
__device__ __forceinline__ void* uniform_ptr(const void* p) {
  const unsigned long long a = (unsigned long long)p;
  return (void*)((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(a >> 32)) << 32 |
                 (unsigned)__builtin_amdgcn_readfirstlane((unsigned)a));
}

// One workgroup of 2 x 2 waves a BM x BN tile, operands 16-byte aligned, K in stages of BK bytes, NS of them in LDS and NS - 1 on their way.
//
// 128 x 256 tiles (waves of 64 x 128, three stages of 64 bytes, two workgroups a CU): 65536 gated positions of 768 to 2048 columns, 412 GOP,
// 270 to 275 us in a row of calls, 1.5 POPS (ten from rest 296, as clocks go); 65536 of 2048 to 768, 206 GOP, 132 to 134. On a card where these
// were 267 and 126 it took 181 and 80 without its loads, 205 and 102 without its matrix instructions, 220 and 111 without its epilogue (239 and
// 118 without the epilogue's stores): loads from L2 cost most, 2.4 GB in lines of which a stage takes half. The epilogue is eleven
// instructions a gated result (with fifteen the call took 2 % longer). 256 x 256 tiles of eight waves, one workgroup a CU, load a third less
// and take 300 and 133 us, as no other workgroup's products run beside their epilogue (283 and 136 where a workgroup walks its tiles and the
// next one's first stages load under the results; 128 x 256 tiles walked that way 298 and 130); 128 x 128 tiles 316 and 138. A load's offset
// is one register and the stage's scalar (KFULL): selecting an offset past K for each load instead took 2 % longer.
// KFULL: K is a whole number of stages, so a load's offset is its lane's own and the stage's, which lies within the descriptor's bytes (the range
// check subtracts it from them); stages past K have empty descriptors and no offset.
template <int BM, int BN, int BK, int NS, int OSZ, bool GATED, bool KFULL>
__global__ __launch_bounds__(256, 2) void expert_tile(ExpertArgs a) {
  constexpr int T = 256, NW = 4, WGN = 2, CPR = BK / 16, KS = BK / 32;
  constexpr int WM = BM / (NW / WGN), WN = BN / WGN, TM = WM / 32, TN = WN / 32;
  constexpr int COLS = GATED ? BN / 2 : BN;              // columns of the result
  static_assert(TM >= 1 && TN >= (GATED ? 2 : 1) && (!GATED || TN % 2 == 0) && NS >= 2 && NS <= 3, "wave tile and stages");
  constexpr int JA = BM * CPR / T, JB = BN * CPR / T, G = JA + JB;       // a wave's loads per stage
  static_assert(JA * T == BM * CPR && JB * T == BN * CPR && (NS - 2) * G < 64, "whole loads");
  constexpr int STAGE = (BM + BN) * BK;
  __shared__ __attribute__((aligned(1024))) int8_t L0[STAGE], L1[STAGE], L2[NS > 2 ? STAGE : 16];
  __shared__ __attribute__((aligned(2048))) int8_t lut_s[256];            // before the stages, where a read's own offset reaches it
  auto arr = [&](auto u) -> int8_t* {                    // the array of stage u, known at compile time
    constexpr int U = decltype(u)::value % NS;
    if constexpr (U == 0) return L0;
    else if constexpr (U == 1) return L1;
    else return L2;
  };
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), wm = wave / WGN, wn = wave % WGN;
  const int half = lane >> 5, l32 = lane & 31;
  const anvil_expert_gemm& g = a.g;
  ExpertTile tile;
  if (!find_tile<BM, COLS>(a, blockIdx.x, lane, tile)) return;
  const int K = g.K;

  // operand rows in LDS: A's as they are; B's in bperm order within each 32, a wave's gate columns before its partner columns
  const int cols = min(g.N - tile.n0, COLS);
  const long long b_at = tile.e * g.sb + (long long)tile.n0 * g.ldb;
  const int b_bytes = __builtin_amdgcn_readfirstlane((int)((cols - 1) * g.ldb + K));
  void *const pa = uniform_ptr(g.A), *const pb = uniform_ptr(g.B + b_at), *const pb2 = uniform_ptr(GATED ? g.B2 + b_at : g.B);
  int mult, mult2 = 0, shift = g.shift, shift2 = g.shift2;
  if (!expert_mult(a, g.mults, g.mult, tile.e, t == 0, mult)) return;
  if (GATED && !expert_mult(a, g.mults2, g.mult2, tile.e, t == 0, mult2)) return;
  if (!g.scale) lift_shift(mult, shift), lift_shift(mult2, shift2);
  // The first loads in the order of what waits for what: the table and the rows' numbers, the first stages of B, and once the numbers
  // are there the rows' scales and the first stages of A.
  const int8_t entry = g.lut ? g.lut[t] : (int8_t)0;
  int rows[JA], mine[TM];
#pragma unroll
  for (int j = 0; j < JA; ++j) {
    const int r = ((wave + NW * j) * 64 + lane) / CPR;
    rows[j] = r < tile.rows ? row_of(a, tile.p0 + r, tile.n0 == 0) : -1;
  }
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int r = wm * WM + 32 * j + l32;
    mine[j] = g.scale && r < tile.rows ? row_of(a, tile.p0 + r, false) : -1;
  }
  unsigned offa[JA], offb[JB];                           // OOB stays out of range for every k below it: K is at most 2^16
  int ka[JA], kb[JB];
#pragma unroll
  for (int j = 0; j < JB; ++j) {
    const int P = (wave + NW * j) * 64 + lane, r = P / CPR, c = swz<BK>(r, P % CPR);
    const int col = GATED ? r / WN * (WN / 2) + (r % (WN / 2) & ~31) + bperm(r & 31) : (r & ~31) + bperm(r & 31);
    offb[j] = col < cols ? (unsigned)(col * g.ldb + c * 16) : PAST;
    kb[j] = c * 16;
  }
  // chunks past K load zeros; a stage past K is issued all the same, which keeps the wait counts fixed
  auto load = [&](__amdgpu_buffer_rsrc_t r, int8_t* s, unsigned off, int k, int k0) {
    if constexpr (KFULL)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)s, 16, off, k0 < K ? k0 : 0, 0, 0);
    else
      dma16(r, s, k0 + k < K ? off + k0 : OOB);
  };
  auto within = [&](void* p, int bytes, int k0) {
    return __builtin_amdgcn_make_buffer_rsrc(p, (short)0, KFULL && k0 >= K ? 0 : bytes, RSRC_DW3);
  };
  auto issue_b = [&](int8_t* s, int k0) {
    const __amdgpu_buffer_rsrc_t r1 = within(pb, b_bytes, k0), r2 = within(pb2, b_bytes, k0);
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      const bool second = GATED && ((wave + NW * j) * (64 / CPR) % WN) >= WN / 2;
      load(second ? r2 : r1, s + BM * BK + (wave + NW * j) * 1024, offb[j], kb[j], k0);
    }
  };
  auto issue_a = [&](int8_t* s, int k0) {
    const __amdgpu_buffer_rsrc_t r = within(pa, a.a_bytes, k0);
#pragma unroll
    for (int j = 0; j < JA; ++j) load(r, s + (wave + NW * j) * 1024, offa[j], ka[j], k0);
  };
  static_for<NS - 1>([&](auto u) { issue_b(arr(u), decltype(u)::value * BK); });
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < JA; ++j) {
    const int P = (wave + NW * j) * 64 + lane, r = P / CPR, c = swz<BK>(r, P % CPR);
    offa[j] = rows[j] >= 0 ? (unsigned)(rows[j] * g.lda + c * 16) : PAST;
    ka[j] = c * 16;
  }
  int scale[TM];
#pragma unroll
  for (int j = 0; j < TM; ++j) scale[j] = !g.scale ? 1 : mine[j] < 0 ? 0 : (int)g.scale[mine[j]];
  static_for<NS - 1>([&](auto u) { issue_a(arr(u), decltype(u)::value * BK); });
  lut_s[t ^ 128] = entry;

  v16i acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = v16i{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  v4i af[2][TM], bf[2][TN];
  auto load_frags = [&](int set, const int8_t* s, int ks) {
    const int ch = ks * 2 + half;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int r = wm * WM + j * 32 + l32;
      af[set][j] = *reinterpret_cast<const v4i*>(s + r * BK + (swz<BK>(r, ch) << 4));
    }
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      const int r = wn * WN + i * 32 + l32;
      bf[set][i] = *reinterpret_cast<const v4i*>(s + BM * BK + r * BK + (swz<BK>(r, ch) << 4));
    }
  };
  auto mm = [&](int set) {
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf[set][i], af[set][j], acc[i][j], 0, 0, 0);
  };
  const int nk = (K + BK - 1) / BK;
  // stage kt + NS - 1 loads into the array of stage kt - 1; before its last k-step a wave waits for its share of stage kt + 1
  // and meets the others
  auto step = [&](int kt, const int8_t* cur, int8_t* nxt, const int8_t* next) {
    issue_b(nxt, (kt + NS - 1) * BK);
    issue_a(nxt, (kt + NS - 1) * BK);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < KS - 1; ++ks) {
      load_frags((ks + 1) & 1, cur, ks + 1);
      __builtin_amdgcn_sched_barrier(0);
      mm(ks & 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_vm_lgkm0<(NS - 2) * G>();
    stage_barrier();
    load_frags(0, next, 0);
    __builtin_amdgcn_sched_barrier(0);
    mm((KS - 1) & 1);
  };
  wait_vm_lgkm0<(NS - 2) * JA>();                        // all of B's first stages and A's first
  stage_barrier();
  load_frags(0, L0, 0);
#define ANVIL_EXPERT_STEP(u)                                                                               \
  if constexpr (NS > u) {                                                                                  \
    step(kt, arr(std::integral_constant<int, u>{}), arr(std::integral_constant<int, u + NS - 1>{}),          \
         arr(std::integral_constant<int, u + 1>{}));                                                       \
    if (++kt == nk) break;                                                                                 \
  }
  for (int kt = 0;;) {
    ANVIL_EXPERT_STEP(0) ANVIL_EXPERT_STEP(1) ANVIL_EXPERT_STEP(2)
  }
#undef ANVIL_EXPERT_STEP

  const Epilogue ep(g, shift, shift2, OSZ == 1 ? -128 : -32768);
  constexpr int TC = GATED ? TN / 2 : TN;                // column groups of 32 a wave has of the result
  auto finish = [&](auto hi_c) {
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int r = wm * WM + 32 * j + l32;
      if (r >= tile.rows) continue;
      const int m = mult * scale[j], m2 = mult2 * scale[j];
#pragma unroll
      for (int i = 0; i < TC; ++i) {
        const int n = tile.n0 + (wn * TC + i) * 32 + 16 * half;
        if (n >= g.N) continue;
        unsigned w[4 * OSZ];
        finish_n<16, OSZ, GATED, decltype(hi_c)::value>(acc[i][j], acc[GATED ? TC + i : i][j], m, m2, ep, lut_s, w);
        store_n<16, OSZ>(g, tile.p0 + r, n, w);
      }
    }
  };
  if (ep.high) finish(std::true_type{});
  else finish(std::false_type{});
  wait_vmcnt(0);                                         // the trailing zero loads land before the LDS is released
}

// Few rows an expert: 16 MT rows x 16 CT columns a workgroup, operands straight from memory into registers.
//
// What bounds it is the weights' way from memory, so nothing stands in it: each of the four waves takes every fourth 64 bytes of K, asks
// for STEPS of them at a time, and its matrix instructions (16 x 16 x 64) take the loads' registers as they are; no LDS, no barrier before
// the end, where the waves' sums meet in LDS. A lane's results are four consecutive columns of its row.
//
// ANY: rows at any alignment and K from 16 on. K's last chunk is the rows' last 16 bytes, of which those that the chunk before has are zeros in A.
template <int MT, int CT, int OSZ, bool GATED, bool ANY>
__global__ __launch_bounds__(256) void expert_few(ExpertArgs a) {
  constexpr int NB = GATED ? 2 : 1, STEPS = 4, COLS = 16 * CT;
  __shared__ __attribute__((aligned(16))) v4i sums[4][MT * CT * NB][64];
  __shared__ int8_t lut_s[256];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r16 = lane & 15, quad = lane >> 4;
  const anvil_expert_gemm& g = a.g;
  ExpertTile tile;
  if (!find_tile<16 * MT, COLS>(a, blockIdx.x, lane, tile)) return;
  int mult, mult2 = 0, shift = g.shift, shift2 = g.shift2;
  if (!expert_mult(a, g.mults, g.mult, tile.e, t == 0, mult)) return;
  if (GATED && !expert_mult(a, g.mults2, g.mult2, tile.e, t == 0, mult2)) return;
  if (!g.scale) lift_shift(mult, shift), lift_shift(mult2, shift2);
  const int K = g.K;
  int row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = 16 * m + r16;
    row[m] = r < tile.rows ? row_of(a, tile.p0 + r, tile.n0 == 0 && wave == 0 && quad == 0) : -1;
  }
  const int8_t entry = g.lut ? g.lut[t] : (int8_t)0;
  const int cols = min(g.N - tile.n0, COLS);
  const long long b_at = tile.e * g.sb + (long long)tile.n0 * g.ldb;
  const int b_bytes = (int)((cols - 1) * g.ldb + K);
  const __amdgpu_buffer_rsrc_t ra = uniform_rsrc(g.A, a.a_bytes), rb = uniform_rsrc(g.B + b_at, b_bytes),
                               rb2 = uniform_rsrc(GATED ? g.B2 + b_at : g.B, GATED ? b_bytes : 0);
  unsigned offb[CT], offa[MT];
#pragma unroll
  for (int c = 0; c < CT; ++c) offb[c] = 16 * c + r16 < cols ? (unsigned)((16 * c + r16) * g.ldb) : PAST;
  const auto load = [](__amdgpu_buffer_rsrc_t r, unsigned off) {
    return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
  };
  v4i acc[NB][CT][MT];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[b][c][m] = v4i{0, 0, 0, 0};
  v4i fb[STEPS][NB][CT], fa[STEPS][MT];
  const auto within = [&](unsigned off, int k) {         // of the lane's chunk of the 64 bytes from k on; chunks past K are zeros
    const int at = k + 16 * quad;
    return at < K ? off + (ANY ? min(at, K - 16) : at) : OOB;
  };
  const auto ask_b = [&](int k0) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int k = k0 + 256 * s;
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const unsigned off = within(offb[c], k);
        fb[s][0][c] = load(rb, off);
        if constexpr (GATED) fb[s][NB - 1][c] = load(rb2, off);
      }
    }
  };
  const auto ask_a = [&](int k0) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int k = k0 + 256 * s;
#pragma unroll
      for (int m = 0; m < MT; ++m) fa[s][m] = load(ra, within(offa[m], k));
    }
  };
  ask_b(64 * wave);                                      // before the rows' numbers are there
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int m = 0; m < MT; ++m) offa[m] = row[m] >= 0 ? (unsigned)(row[m] * g.lda) : PAST;
  int scale[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) scale[m] = !g.scale ? 1 : row[m] < 0 ? 0 : (int)g.scale[row[m]];
  for (int k0 = 64 * wave;;) {
    ask_a(k0);
    if constexpr (ANY) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int k = k0 + 256 * s;
        if (k < K && k + 64 > K) {
#pragma unroll
          for (int m = 0; m < MT; ++m) fa[s][m] = without_first(fa[s][m], k + 16 * quad - (K - 16));
        }
      }
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int m = 0; m < MT; ++m)
            acc[b][c][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[s][b][c], fa[s][m], acc[b][c][m], 0, 0, 0);
    k0 += 256 * STEPS;
    if (k0 >= K) break;
    ask_b(k0);
  }
  lut_s[t ^ 128] = entry;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int m = 0; m < MT; ++m) sums[wave][(m * CT + c) * NB + b][lane] = acc[b][c][m];
  __syncthreads();
  const Epilogue ep(g, shift, shift2, OSZ == 1 ? -128 : -32768);
#pragma unroll
  for (int i = 0; i < MT * CT; ++i) {                    // block i of 16 x 16: wave i % 4
    if (i % 4 != wave) continue;
    const int r = 16 * (i / CT) + r16, n = tile.n0 + 16 * (i % CT) + 4 * quad;
    if (r >= tile.rows || n >= g.N) continue;
    v4i x[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) x[b] = sums[0][i * NB + b][lane] + sums[1][i * NB + b][lane] + sums[2][i * NB + b][lane] + sums[3][i * NB + b][lane];
    const int sc = scale[i / CT];
    unsigned w[OSZ];
    const auto finish = [&](auto hi_c) {
      finish_n<4, OSZ, GATED, decltype(hi_c)::value>(x[0], x[NB - 1], mult * sc, mult2 * sc, ep, lut_s, w);
    };
    if (ep.high) finish(std::true_type{});
    else finish(std::false_type{});
    store_n<4, OSZ>(g, tile.p0 + r, n, w);
  }
}

// Operands at any alignment and stride, and past 2^32 bytes: 64 TM x 64 tiles, chunks through registers into LDS, the next stage's on their
// way while one is multiplied. 3001 rows of 500, three of 11 experts each, to 333 columns: 11.3 us (12.4 with 64 bytes of a row a load, for
// which unaligned rows' lines are asked twice as often, 17 with results stored a byte at a time as well). One array of LDS and two barriers
// a stage, for more workgroups a CU: 20000 x 2 rows of 700 to 1001, gated, by 64 x 64 tiles 133 us (150 with two arrays), by 128 x 64 122. More
// stages on their way: no faster.
template <int TM, int OSZ, bool GATED>
__global__ __launch_bounds__(256) void expert_any(ExpertArgs a) {
  constexpr int BM = 64 * TM, BN = 64, BK = 128, NB = GATED ? 2 : 1, PER = 2, PA = PER * TM;
  __shared__ __attribute__((aligned(16))) int8_t As[BM * BK], Bs[NB][BN * BK];
  __shared__ int8_t lut_s[256];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave >> 1, wn = wave & 1, half = lane >> 5, l32 = lane & 31;
  const anvil_expert_gemm& g = a.g;
  ExpertTile tile;
  if (!find_tile<BM, BN>(a, blockIdx.x, lane, tile)) return;
  int mult, mult2 = 0;
  if (!expert_mult(a, g.mults, g.mult, tile.e, t == 0, mult)) return;
  if (GATED && !expert_mult(a, g.mults2, g.mult2, tile.e, t == 0, mult2)) return;
  if (g.lut) lut_s[t] = g.lut[t];

  // thread t stages chunk t % 8 of rows t / 8 and t / 8 + 32 of each operand: 128 bytes of a row an eighth of a wave
  const int sr = t >> 3, sc = t & 7;
  const int8_t *arow[PA], *brow[NB][PER];                // past the last column some other row: what it gives is not stored
#pragma unroll
  for (int i = 0; i < PA; ++i) {
    const int r = sr + 32 * i, src = r < tile.rows ? row_of(a, tile.p0 + r, tile.n0 == 0 && sc == 0) : -1;
    arow[i] = src < 0 ? nullptr : g.A + (long long)src * g.lda;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b) brow[b][i] = (b ? g.B2 : g.B) + tile.e * g.sb + (long long)min(tile.n0 + sr + 32 * i, g.N - 1) * g.ldb;
  const int K = g.K;
  v4i av[PA], bv[NB][PER];
  // K's last chunk is the rows' last 16 bytes, of which those that the chunk before has are zeros in A, as are chunks past K
  const auto ask = [&](int k0) {
    const int k = k0 + 16 * sc, at = min(k, K - 16);
#pragma unroll
    for (int i = 0; i < PA; ++i) {
      av[i] = v4i{0, 0, 0, 0};
      if (arow[i]) {
        if (K >= 16) __builtin_memcpy(&av[i], arow[i] + at, 16);
        else av[i] = row_chunk(arow[i], k, K);
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (K >= 16) __builtin_memcpy(&bv[b][i], brow[b][i] + at, 16);
        else bv[b][i] = row_chunk(brow[b][i], k, K);
      }
    if (k0 + BK > K && K >= 16) {
#pragma unroll
      for (int i = 0; i < PA; ++i) av[i] = without_first(av[i], k - (K - 16));
    }
  };
  v16i acc[TM][NB];
#pragma unroll
  for (int j = 0; j < TM; ++j)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[j][b] = v16i{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  ask(0);
  for (int k = 0; k < K; k += BK) {
    if (k) __syncthreads();
#pragma unroll
    for (int i = 0; i < PA; ++i) *reinterpret_cast<v4i*>(As + (sr + 32 * i) * BK + 16 * swz<BK>(sr + 32 * i, sc)) = av[i];
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b) *reinterpret_cast<v4i*>(Bs[b] + (sr + 32 * i) * BK + 16 * swz<BK>(sr + 32 * i, sc)) = bv[b][i];
    __syncthreads();
    if (k + BK < K) ask(k + BK);
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      const int rb = wn * 32 + bperm(l32), ch = 2 * ks + half;
      v4i af[TM];
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int ra = wm * 32 * TM + 32 * j + l32;
        af[j] = *reinterpret_cast<const v4i*>(As + ra * BK + 16 * swz<BK>(ra, ch));
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const v4i bf = *reinterpret_cast<const v4i*>(Bs[b] + rb * BK + 16 * swz<BK>(rb, ch));
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[j][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf, af[j], acc[j][b], 0, 0, 0);
      }
    }
  }
  const int n0 = tile.n0 + wn * 32 + 16 * half;          // this lane's 16 columns
  const int lo = OSZ == 1 ? -128 : -32768;
  const WideRequant q1(g.shift, lo, -lo - 1), q2(g.shift2, -128, 127);
  const auto of = [](const WideRequant& q, int acc, int mul) { return q.high() ? q.of<true>(acc, mul) : q.of<false>(acc, mul); };
  const int rnd3 = (int)round_term(g.shift3);
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int m = wm * 32 * TM + 32 * j + l32;
    if (m >= tile.rows) continue;
    const int i = row_of(a, tile.p0 + m, false);
    const int scale = g.scale ? (i < 0 ? 0 : (int)g.scale[i]) : 1;
    int v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      v[e] = of(q1, acc[j][0][e], mult * scale);
      if (g.lut) v[e] = lut_s[(v[e] + 128) & 255];
      if constexpr (GATED) v[e] = min(max((v[e] * of(q2, acc[j][NB - 1][e], mult2 * scale) * g.mult3 + rnd3) >> g.shift3, -128), 127);
    }
    unsigned w[4 * OSZ];
#pragma unroll
    for (int q = 0; q < 4 * OSZ; ++q)
      w[q] = OSZ == 1 ? pack4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3])
                      : __builtin_amdgcn_perm((unsigned)v[2 * q + 1], (unsigned)v[2 * q], 0x05040100u);
    store_n<16, OSZ>(g, tile.p0 + m, n0, w);
  }
}

}  // namespace anvil

using namespace anvil;

extern "C" int anvil_expert_gemm_i8(anvil_ctx* ctx, const anvil_expert_gemm* g) {
  const char* who = "anvil_expert_gemm_i8";
  if (!g) return set_error(ANVIL_E_VALUE, "%s: null arguments", who);
  if (g->rows < 0 || g->rows >= 1 << 30 || g->rows_a < 0 || g->experts < 1 || g->experts > ANVIL_EXPERTS_MAX || g->N < 1 || g->N > 1 << 20 ||
      g->K < 1 || g->K > 1 << 16)
    return set_error(ANVIL_E_VALUE, "%s: %d rows of %d, %d experts, N %d, K %d", who, g->rows, g->rows_a, g->experts, g->N, g->K);
  if (!narrow(g->out_dtype) || ((g->lut || g->B2) && g->out_dtype != ANVIL_I8))
    return set_error(ANVIL_E_VALUE, "%s: results are i8, or i16 without a table", who);
  if (g->B2 && !g->lut) return set_error(ANVIL_E_VALUE, "%s: a gated product needs its gate's table", who);
  if (g->shift < 0 || g->shift > 62 || (g->B2 && (g->shift2 < 0 || g->shift2 > 62 || g->shift3 < 0 || g->shift3 > 31)))
    return set_error(ANVIL_E_VALUE, "%s: shifts %d, %d, %d outside [0, 62], [0, 62], [0, 31]", who, g->shift, g->shift2, g->shift3);
  if (!stride_ok(g->lda, g->K) || !stride_ok(g->ldb, g->K) || !stride_ok(g->ldc, g->N) ||
      (g->experts > 1 && (g->sb < g->ldb * (g->N - 1) + g->K || g->sb > 1ll << 51)))
    return set_error(ANVIL_E_VALUE, "%s: a stride is below its operand's width or past 2^31", who);
  const auto wide = [](int m) { return m < -32767 || m > 32767; };
  if (g->scale && ((!g->mults && wide(g->mult)) || (g->B2 && !g->mults2 && wide(g->mult2))))
    return set_error(ANVIL_E_OVERFLOW, "%s: multipliers %d, %d times a row's scale may leave int32", who, g->mult, g->mult2);
  if (g->B2 && (1ll << 14) * std::abs((long long)g->mult3) + (g->shift3 ? 1ll << (g->shift3 - 1) : 0) > I32_MAX)
    return set_error(ANVIL_E_OVERFLOW, "%s: the gated product's multiplier %d may leave int32", who, g->mult3);
  if (!g->rows) return check_ctx(ctx);
  if (!g->B || !g->starts || !g->C || (g->rows_a && !g->A)) return set_error(ANVIL_E_VALUE, "%s: null pointer", who);
  if ((uintptr_t)g->row % 4 || (uintptr_t)g->scale % 2 || (uintptr_t)g->starts % 4 || (uintptr_t)g->mults % 4 || (uintptr_t)g->mults2 % 4 ||
      (uintptr_t)g->C % g->out_dtype)
    return set_error(ANVIL_E_VALUE, "%s: a pointer is not aligned to its type", who);
  const auto flat = [](const void* p, long long bytes) { return Span{p, 1, bytes, bytes}; };
  const Span c{g->C, g->rows, g->ldc * g->out_dtype, (long long)g->N * g->out_dtype};
  const long long weights = (g->experts - 1) * g->sb + (g->N - 1) * g->ldb + g->K;
  const Span in[9] = {{g->A, g->rows_a, g->lda, g->K}, flat(g->row, 4ll * g->rows), flat(g->scale, 2ll * g->rows_a), flat(g->B, weights),
                      flat(g->B2, weights), flat(g->starts, 4ll * g->experts + 4), flat(g->mults, 4ll * g->experts),
                      flat(g->mults2, 4ll * g->experts), flat(g->lut, 256)};
  for (const Span& s : in)
    if (!apart(c, s)) return set_error(ANVIL_E_VALUE, "%s: the result overlaps what is read", who);
  if (int e = check_ctx(ctx)) return e;
  ExpertArgs a{*g, 0, 0, 0, ctx->flags};
  const auto grid = [&](int bm, int cols) -> unsigned {   // 0: more tiles than a grid has
    a.tiles_n = (g->N + cols - 1) / cols;
    a.tiles_m = g->rows / bm + std::min(g->experts, g->rows);
    const long long tiles = (long long)a.tiles_m * a.tiles_n;
    return tiles > GRID_MAX ? 0 : (unsigned)((tiles + 7) / 8 * 8);
  };
  const auto by_type = [&](auto&& f) {
    if (g->B2) f(std::integral_constant<int, 1>{}, std::true_type{});
    else if (g->out_dtype == ANVIL_I8) f(std::integral_constant<int, 1>{}, std::false_type{});
    else f(std::integral_constant<int, 2>{}, std::false_type{});
  };
  // 16-byte loads, 32-bit offsets into A and into a tile's weights
  const long long a_bytes = (g->rows_a - 1) * g->lda + g->K;
  unsigned wgs = 0;
  const auto tiles = [&](auto bm, auto bn, auto bk, auto ns) {
    by_type([&](auto osz, auto gated) {
      constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, BK = decltype(bk)::value, NS = decltype(ns)::value;
      constexpr int OSZ = decltype(osz)::value;
      constexpr bool GATED = decltype(gated)::value;
      wgs = grid(BM, GATED ? BN / 2 : BN);
      if (!wgs) return;
      if (g->K % BK == 0) ANVIL_LAUNCH((expert_tile<BM, BN, BK, NS, OSZ, GATED, true>), dim3(wgs), dim3(256), 0, ctx->stream, a);
      else ANVIL_LAUNCH((expert_tile<BM, BN, BK, NS, OSZ, GATED, false>), dim3(wgs), dim3(256), 0, ctx->stream, a);
    });
  };
  using std::integral_constant;
  const bool once = g->rows <= 8ll * g->experts;         // most experts have one tile of 16 rows and read their weights once
  const auto few = [&](auto any) {
    const auto go = [&](auto mt) {
      by_type([&](auto osz, auto gated) {
        constexpr int MT = decltype(mt)::value;
        constexpr bool GATED = decltype(gated)::value;
        constexpr int CT = GATED ? 1 : 2;
        wgs = grid(16 * MT, 16 * CT);
        if (wgs) ANVIL_LAUNCH((expert_few<MT, CT, decltype(osz)::value, GATED, decltype(any)::value>), dim3(wgs), dim3(256), 0, ctx->stream, a);
      });
    };
    if (once) go(integral_constant<int, 1>{});
    else go(integral_constant<int, 2>{});
  };
  const bool near = g->rows_a && g->K >= 16 && a_bytes <= (long long)PAST && g->ldb < 1 << 23;
  const bool aligned = aligned16(g->A) && aligned16(g->B) && aligned16(g->B2) && g->K % 16 == 0 && g->lda % 16 == 0 && g->ldb % 16 == 0 &&
                       (g->experts == 1 || g->sb % 16 == 0);
  a.a_bytes = near ? (int)(unsigned)a_bytes : 0;
  if (near && aligned) {
    const integral_constant<int, 128> i128;
    const integral_constant<int, 64> i64;
    // Kernels by size, us on one box (rows x the experts of each). Few rows / 64 x 128, by the few rows' workgroups (more than five a CU wait for each
    // other; past half of that only where they read the weights once):
    //   16 x 2 of 8, 2048 -> 768 (240), 6.9 / 14; 64 x 2 of 4, 4096 -> 1024 (256), 13.0 / 22.5; 200 x 2 of 8, 2048 -> 768 (480), 11.6 / 14; 2048 of one,
    //     4096 -> 256 (520), 18.8 / 22.7; once: 16 x 2 of 8, 4096 -> 4096 (1280), 33 / 36; 2 x 2 of 8, gated 4096 -> 8192 (1024), 48 / 57
    //   but 30000 of one, 768 -> 16 (938), 9.4 / 9.2; 4096 of one, 1024 -> 256 (1032), 11.4 / 7.9; 64 x 2 of 8, gated 768 -> 2048 (1536), 11.2 / 9.6; 16 x 4 of
    //     32, gated 768 -> 1024 (2304), 12.3 / 11.6; 1000 x 2 of 8, 64 -> 1024 (2240), 12.1 / 6.4; 40 x 4 of 100, 1024 -> 1408 (4840), 24 / 20.5
    // 128 x 256 / 64 x 128:
    //   32768 x 2 of 8, gated 768 -> 2048, 271 / 382; 32768 x 2 of 8, 2048 -> 768, 133 / 161; 4096 x 2 of 8, gated 768 -> 2048, 46 / 55; 8192 x 2 of 16,
    //     2048 -> 768, 41 / 47; 2048 x 2 of 8, gated 768 -> 2048 (640 tiles), 29 / 31;
    //   but 4096 x 2 of 8, 768 -> 2048 (576), 34 / 30: with few tiles the last round of them is half empty, and a short K has little to make up
    //     for it
    const long long shares = ((long long)g->rows / (once ? 16 : 32) + std::min(g->experts, g->rows)) * (g->B2 ? (g->N + 15) / 16 : (g->N + 31) / 32);
    const long long width = (long long)g->N * (g->B2 ? 2 : 1);                         // of the operand B, and B2 beside it
    const long long large = ((long long)g->rows / 128 + std::min(g->experts, g->rows)) * ((width + 255) / 256);
    if (2 * shares <= (once ? 10 : 5) * ctx->num_cu) {
      few(std::false_type{});
    } else if (large >= (g->K >= 2048 ? 3 : 5) * ctx->num_cu / 2) {
      tiles(i128, integral_constant<int, 256>{}, i64, integral_constant<int, 3>{});
    } else {
      tiles(i64, i128, i128, integral_constant<int, 2>{});
    }
  } else if (near && g->rows <= 64ll * g->experts && ((long long)g->rows / 64 + std::min(g->experts, g->rows)) * ((g->N + 63) / 64) < 3 * ctx->num_cu) {
    // Rows at any alignment, us. Few rows / 64 x 64: 200 x 2 of 8, gated 700 -> 1001, 9.5 / 11.8; 64 x 4 of 16, 1001 -> 333, 7.3 / 9.0; 30 x 4 of 40, gated
    // 1500 -> 1001, 26 / 28; but 40 x 4 of 100, 2001 -> 700 (1120 tiles of 64 x 64), 35 / 24.5; 600 x 2 of 8, gated 700 -> 1001 (150 rows an expert),
    // 18.7 / 13.2: more rows read their weights again, and many tiles hide their stages' waits behind each other's.
    few(std::true_type{});
  } else {
    const auto go = [&](auto tm) {
      wgs = grid(64 * decltype(tm)::value, 64);
      if (wgs)
        by_type([&](auto osz, auto gated) {
          ANVIL_LAUNCH((expert_any<decltype(tm)::value, decltype(osz)::value, decltype(gated)::value>), dim3(wgs), dim3(256), 0, ctx->stream, a);
        });
    };
    // 128 rows / 64, us: 20000 x 2 of 8, gated 700 -> 1001, 122 / 133; 6000 x 2 of 16, 1501 -> 1501, 84 / 96; but 300 x 4 of 100, 2001 -> 700, 51 / 44; 3001 x
    // 3 of 11, 500 -> 333, 12.1 / 11.3. Between them little is lost either way: 2000 x 2 of 8, gated 700 -> 1001 (624 tiles of 128), 23.1 / 24.5
    const long long tall = ((long long)g->rows / 128 + std::min(g->experts, g->rows)) * ((g->N + 63) / 64);
    if (tall >= 8 * ctx->num_cu && g->rows >= 128ll * g->experts) go(integral_constant<int, 2>{});
    else go(integral_constant<int, 1>{});
  }
  if (!wgs) return set_error(ANVIL_E_VALUE, "%s: %d rows of %d columns are more tiles than a grid has", who, g->rows, g->N);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
