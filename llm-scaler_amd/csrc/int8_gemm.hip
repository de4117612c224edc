// The linears of a W8A8 layer: rows of activations to codes (int8_quant.hip), then the product (int8_gemm.hpp).
#include "int8_gemm.hpp"
#include "int8_rows.hpp"
#include "../../include/mi355x_qlinear.h"

namespace qlin {

template <class Act, int BM, int BN, int WM, int WN, int KG, int SA, int SB>
static int launch_tiles(Int8GemmArgs p, hipStream_t st) {
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  const long long tiles = (long long)p.tiles_m * p.tiles_n, grid = (tiles + 7) / 8 * 8;          // linear_sizes: below 2^23
  auto* kernel = int8_gemm_kernel<Act, BM, BN, WM, WN, KG, SA, SB, kEpiOut, false>;
  constexpr size_t lds = int8_gemm_lds(BM, BN, KG, SA, SB);
  if constexpr (lds > 64 * 1024) {
    static std::atomic<unsigned long long> raised{0};
    const int rc = int8_raise_lds(kernel, raised, lds);
    if (rc != MI_OK) return rc;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WM * WN * KG), lds, st, p);
  return launch_status();
}

// The tiles, and what a round of the CUs costs with each: us = fixed + step x (steps of 128 KG of K), fitted to 675 problems (M 17 .. 2048,
// N 512 .. 14336, K 1024 .. 14336); the last three have room for two workgroups on a CU, whose pair costs less than two rounds.  The
// tile with the least sum of rounds is 0.3 % behind the best one in the mean.  Some of them, us with the best / the second best of another shape,
// all tiles one after the other (the clocks of the large ones are lower then than in a call alone): 2048 x 4096 x 14336 256 x 256 135 / 256 x 192 147;
// 2048 x 14336 x 4096 256 x 128 116 / 128 x 128 135; 1000 x 4096 x 6144 128 x 192 29.6 / 256 x 128 32.5; 201 x 2048 x 5120 128 x 64 9.3 / 64 x 64 9.7;
// 64 x 5120 x 5120 64 x 32 10.3 / 64 x 64 12.3; 32 x 14336 x 4096 32 x 16 13.4 / 64 x 16 14.8.  A smaller
// tile reads more through the loads to LDS (68 GB/s per CU for whole lines, 54 for half lines of 64 bytes), a larger one leaves CUs without
// work.  Eight wavefronts in every tile: 128 x 64 with four is 3 % slower in the median, 11 % at most.
struct Int8Tile {
  int bm, bn, kg;
  float fixed, step, pair_fixed, pair_step;            // the pair: 0 where a workgroup fills the CU
};
constexpr Int8Tile kTiles[] = {{256, 256, 1, 9.77f, 1.34f, 0, 0},        {256, 192, 1, 7.54f, 1.11f, 0, 0}, {256, 128, 1, 6.45f, 0.82f, 0, 0},
                               {128, 192, 1, 6.76f, 0.64f, 0, 0},        {128, 128, 1, 4.21f, 0.52f, 0, 0}, {64, 96, 2, 4.89f, 0.52f, 0, 0},
                               {64, 64, 2, 3.92f, 0.37f, 0, 0},          {64, 32, 4, 4.22f, 0.52f, 0, 0},   {64, 16, 4, 4.06f, 0.38f, 0, 0},
                               {32, 16, 8, 3.92f, 0.49f, 0, 0},          {64, 64, 1, 3.49f, 0.24f, 3.39f, 0.40f},
                               {64, 32, 2, 3.70f, 0.28f, 4.10f, 0.53f},  {128, 64, 1, 3.52f, 0.34f, 3.92f, 0.62f}};

static int pick_tile(long long M, long long N, long long K) {
  const long long cus = int8_cu_count();
  int best = 0;
  double least = 0;
  for (int i = 0; i < (int)(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
    const Int8Tile& t = kTiles[i];
    const long long tiles = ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn), rounds = (tiles + cus - 1) / cus;
    const double steps = (double)((K + 128 * t.kg - 1) / (128 * t.kg)), one = t.fixed + t.step * steps;
    const double cost = t.pair_step > 0 ? (rounds % 2) * one + (rounds / 2) * (t.pair_fixed + t.pair_step * steps) : rounds * one;
    if (!i || cost < least) {
      least = cost;
      best = i;
    }
  }
  return best;
}
// Sizes that every launch of a call holds: a grid has less than 2^32 threads.
static bool linear_sizes(int M, int N, int K) {
  if (!int8_sizes(M, N, K)) return false;
  if ((long long)M * N < (1LL << 31)) return true;     // M N / 512 + M / 32 + N / 16 + 1 tiles of 512 threads at most
  const Int8Tile& t = kTiles[pick_tile(M, N, K)];
  return (((long long)M + t.bm - 1) / t.bm) * (((long long)N + t.bn - 1) / t.bn) < (1LL << 23) - 8;
}

template <class Act>
static int launch_product(const Int8GemmArgs& p, hipStream_t st) {
  switch (pick_tile(p.M, p.N, p.K)) {                  // rows, columns, wavefronts along both, KG, buffers of A and B
    case 0: return launch_tiles<Act, 256, 256, 4, 2, 1, 3, 2>(p, st);
    case 1: return launch_tiles<Act, 256, 192, 4, 2, 1, 3, 2>(p, st);
    case 2: return launch_tiles<Act, 256, 128, 4, 2, 1, 3, 3>(p, st);
    case 3: return launch_tiles<Act, 128, 192, 2, 4, 1, 3, 3>(p, st);
    case 4: return launch_tiles<Act, 128, 128, 2, 4, 1, 3, 3>(p, st);
    case 5: return launch_tiles<Act, 64, 96, 2, 2, 2, 3, 3>(p, st);
    case 6: return launch_tiles<Act, 64, 64, 2, 2, 2, 4, 3>(p, st);
    case 7: return launch_tiles<Act, 64, 32, 2, 1, 4, 3, 3>(p, st);
    case 8: return launch_tiles<Act, 64, 16, 2, 1, 4, 3, 3>(p, st);
    case 9: return launch_tiles<Act, 32, 16, 1, 1, 8, 3, 3>(p, st);
    case 10: return launch_tiles<Act, 64, 64, 4, 2, 1, 4, 4>(p, st);
    case 11: return launch_tiles<Act, 64, 32, 2, 2, 2, 3, 3>(p, st);
    default: return launch_tiles<Act, 128, 64, 4, 2, 1, 3, 3>(p, st);
  }
}

struct Linear {
  int from;                   // kFrom*
  QuantArgs q;                // q, scale: filled in here
  const float* x_scale;       // kFromCodes: x is codes
};

static long long round256(long long v) { return (v + 255) / 256 * 256; }
static long long codes_workspace(int M, int K) { return round256((long long)M * K) + round256(4LL * M); }

// Whether the rows are quantised by the launch that multiplies them.  The new residual must not be what other workgroups still read.
static bool one_launch(int from, bool in_place, int M, int N, int K) {
  return from != kFromCodes && N && int8_rows_quantise(from, M, K) && !in_place;
}

static int run_linear(Linear l, const void* w, const float* w_scale, const void* bias, void* out, void* workspace,
                      long long workspace_bytes, int M, int N, int K, int act_dtype, void* stream) {
  if (act_dtype != DT_F16 && act_dtype != DT_BF16) return MI_ERR_ARG;
  if (!linear_sizes(M, N, K)) return MI_ERR_SHAPE;
  if (!M) return MI_OK;
  if (!l.q.x || (N && (!w || !w_scale || !out))) return MI_ERR_ARG;
  if (!aligned16(l.q.x) || !aligned16(w)) return MI_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  Int8RowsArgs r{l.q.x, l.x_scale, l.q.residual, l.q.residual_out, l.q.norm_weight, (const int8_t*)w, w_scale, bias, out, M, N, K, 0, l.q.eps};
  if (one_launch(l.from, l.from == kFromNorm && l.q.residual_out == l.q.residual, M, N, K)) return launch_int8_rows(l.from, r, act_dtype, st);
  Int8GemmArgs p{};
  p.a = (const int8_t*)l.q.x;
  p.a_scale = l.x_scale;
  if (l.from != kFromCodes) {
    if (!workspace || !aligned16(workspace) || workspace_bytes < codes_workspace(M, K)) return MI_ERR_ARG;
    l.q.q = (int8_t*)workspace;
    l.q.scale = (float*)((char*)workspace + round256((long long)M * K));
    l.q.rows = M;
    l.q.K = K;
    const int rc = launch_int8_quant(l.from, l.q, act_dtype, st);
    if (rc != MI_OK) return rc;
    p.a = l.q.q;
    p.a_scale = l.q.scale;
  }
  if (!N) return MI_OK;
  if (int8_rows_codes(M, K)) {
    r.x = p.a;
    r.x_scale = p.a_scale;
    return launch_int8_rows(kFromCodes, r, act_dtype, st);
  }
  p.w = (const int8_t*)w;
  p.w_scale = w_scale;
  p.bias = bias;
  p.out = out;
  p.M = M;
  p.N = N;
  p.K = K;
  return act_dtype == DT_F16 ? launch_product<ActF16>(p, st) : launch_product<ActBF16>(p, st);
}

}  // namespace qlin

using namespace qlin;

extern "C" {

int mi_gemm_int8_workspace(int rows_from, int M, int N, int K, long long* bytes) {
  if (!bytes || rows_from < MI_INT8_CODES || rows_from > MI_INT8_SILU_MUL) return MI_ERR_ARG;
  if (!linear_sizes(M, N, K)) return MI_ERR_SHAPE;
  const int from = rows_from == MI_INT8_CODES ? kFromCodes : rows_from == MI_INT8_ACT ? kFromAct : rows_from == MI_INT8_SILU_MUL ? kFromSilu : kFromNorm;
  *bytes = from == kFromCodes || one_launch(from, rows_from == MI_INT8_RESADD_NORM_IN_PLACE, M, N, K) ? 0 : codes_workspace(M, K);
  return MI_OK;
}

int mi_gemm_int8_ws(const void* x, const float* x_scale, const void* w, const float* w_scale, const void* bias, void* out,
                    void* workspace, long long workspace_bytes, int M, int N, int K, int act_dtype, void* stream) {
  Linear l{x_scale ? kFromCodes : kFromAct, {}, x_scale};
  l.q.x = x;
  return run_linear(l, w, w_scale, bias, out, workspace, workspace_bytes, M, N, K, act_dtype, stream);
}

int mi_resadd_norm_gemm_int8_ws(const void* x, const void* residual, void* residual_out, const void* norm_weight, float eps,
                                const void* w, const float* w_scale, const void* bias, void* out, void* workspace,
                                long long workspace_bytes, int M, int N, int K, int act_dtype, void* stream) {
  if (M > 0 && (!residual || !residual_out || !norm_weight)) return MI_ERR_ARG;
  if (!aligned16(residual) || !aligned16(residual_out) || !aligned16(norm_weight)) return MI_ERR_ARG;
  Linear l{kFromNorm, {}, nullptr};
  l.q.x = x;
  l.q.residual = residual;
  l.q.residual_out = residual_out;
  l.q.norm_weight = norm_weight;
  l.q.eps = eps;
  return run_linear(l, w, w_scale, bias, out, workspace, workspace_bytes, M, N, K, act_dtype, stream);
}

int mi_silu_mul_gemm_int8_ws(const void* gate_up, const void* w, const float* w_scale, const void* bias, void* out, void* workspace,
                             long long workspace_bytes, int M, int N, int K, int act_dtype, void* stream) {
  Linear l{kFromSilu, {}, nullptr};
  l.q.x = gate_up;
  return run_linear(l, w, w_scale, bias, out, workspace, workspace_bytes, M, N, K, act_dtype, stream);
}

}  // extern "C"
