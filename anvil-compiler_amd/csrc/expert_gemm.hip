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
  unsigned* flags;
};

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

// Tile number `w` of a grid of row tiles of BM x column tiles of BN; false past the last.
template <int BM, int BN>
__device__ __forceinline__ bool find_tile(const ExpertArgs& a, int w, int lane, ExpertTile& t) {
  const int E = a.g.experts;
  int lo, mt = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int n = e0 + lane < E ? expert_rows(a, e0 + lane, w == 0, lo) : 0;
    mt += (n + BM - 1) / BM;
  }
  const int tiles_m = __builtin_amdgcn_readlane(wave_scan(mt), 63);
  const long long tiles = (long long)tiles_m * a.tiles_n;
  const long long per = (tiles + 7) / 8;
  if ((w >> 3) >= per) return false;
  const long long pid = (w & 7) * per + (w >> 3);
  if (pid >= tiles) return false;
  const int in_group = GROUP_M * a.tiles_n;
  const int first_m = (int)(pid / in_group) * GROUP_M, in = (int)(pid % in_group);
  const int gsize = min(tiles_m - first_m, GROUP_M);
  const int gm = first_m + in % gsize;
  t.n0 = in / gsize * BN;
  int before = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int n = e0 + lane < E ? expert_rows(a, e0 + lane, false, lo) : 0;
    const int mine = (n + BM - 1) / BM, incl = wave_scan(mine);
    const int all = __builtin_amdgcn_readlane(incl, 63);
    if (gm < before + all) {
      const int l = __builtin_ctzll(__ballot(gm < before + incl));       // the first expert whose tiles reach past gm
      const int skip = (gm - before - __builtin_amdgcn_readlane(incl - mine, l)) * BM;
      t.e = e0 + l;
      t.p0 = __builtin_amdgcn_readlane(lo, l) + skip;
      t.rows = min(BM, __builtin_amdgcn_readlane(n, l) - skip);
      return true;
    }
    before += all;
  }
  return false;
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

// Operands at any alignment and stride: 64 x 64 tiles, chunks through registers into LDS.
template <int OSZ, bool GATED>
__global__ __launch_bounds__(256) void expert_any(ExpertArgs a) {
  constexpr int BM = 64, BN = 64, BK = 64, NB = GATED ? 2 : 1;
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

  // thread t stages chunk t % 4 of row t / 4 of each operand
  const int sr = t >> 2, sc = t & 3;
  const int src = sr < tile.rows ? row_of(a, tile.p0 + sr, tile.n0 == 0 && sc == 0) : -1;
  const int8_t* arow = src < 0 ? nullptr : g.A + (long long)src * g.lda;
  const int n = tile.n0 + sr;
  const int8_t* brow[2] = {nullptr, nullptr};
  if (n < g.N) {
    brow[0] = g.B + tile.e * g.sb + (long long)n * g.ldb;
    if (GATED) brow[1] = g.B2 + tile.e * g.sb + (long long)n * g.ldb;
  }
  const v4i zero = {0, 0, 0, 0};
  v16i acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = v16i{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  for (int k = 0; k < g.K; k += BK) {
    const v4i av = arow ? row_chunk(arow, k + 16 * sc, g.K) : zero;
    v4i bv[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) bv[b] = brow[b] ? row_chunk(brow[b], k + 16 * sc, g.K) : zero;
    __syncthreads();
    *reinterpret_cast<v4i*>(As + sr * BK + 16 * swz<BK>(sr, sc)) = av;
#pragma unroll
    for (int b = 0; b < NB; ++b) *reinterpret_cast<v4i*>(Bs[b] + sr * BK + 16 * swz<BK>(sr, sc)) = bv[b];
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      const int ra = wm * 32 + l32, rb = wn * 32 + bperm(l32), ch = 2 * ks + half;
      const v4i af = *reinterpret_cast<const v4i*>(As + ra * BK + 16 * swz<BK>(ra, ch));
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const v4i bf = *reinterpret_cast<const v4i*>(Bs[b] + rb * BK + 16 * swz<BK>(rb, ch));
        acc[b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf, af, acc[b], 0, 0, 0);
      }
    }
  }
  const int m = wm * 32 + l32, n0 = tile.n0 + wn * 32 + 16 * half;       // this lane's row and its 16 columns
  if (m >= tile.rows) return;
  const int i = row_of(a, tile.p0 + m, false);
  const int scale = g.scale ? (i < 0 ? 0 : (int)g.scale[i]) : 1;
  const int lo = OSZ == 1 ? -128 : -32768, hi = -lo - 1;
  const Requant q1(g.shift, lo, hi), q2(g.shift2, -128, 127);
  const int rnd3 = (int)round_term(g.shift3);
  char* out = (char*)g.C + ((tile.p0 + m) * g.ldc + n0) * OSZ;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    int v = q1.of<false>(acc[0][e], mult * scale);
    if (g.lut) v = lut_s[(v + 128) & 255];
    if constexpr (GATED) v = min(max((v * q2.of<false>(acc[NB - 1][e], mult2 * scale) * g.mult3 + rnd3) >> g.shift3, -128), 127);
    if (n0 + e >= g.N) break;
    if (OSZ == 1) out[e] = (char)v;
    else ((int16_t*)out)[e] = (int16_t)v;
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
  ExpertArgs a{*g, (g->N + 63) / 64, ctx->flags};
  const long long tiles = ((long long)g->rows / 64 + std::min(g->experts, g->rows)) * a.tiles_n;
  if (tiles > GRID_MAX) return set_error(ANVIL_E_VALUE, "%s: %d rows of %d columns are more tiles than a grid has", who, g->rows, g->N);
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8));
  if (g->B2) ANVIL_LAUNCH((expert_any<1, true>), grid, dim3(256), 0, ctx->stream, a);
  else if (g->out_dtype == ANVIL_I8) ANVIL_LAUNCH((expert_any<1, false>), grid, dim3(256), 0, ctx->stream, a);
  else ANVIL_LAUNCH((expert_any<2, false>), grid, dim3(256), 0, ctx->stream, a);
  ANVIL_LAUNCHED();
  return ANVIL_OK;
}
