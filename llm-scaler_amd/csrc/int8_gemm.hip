// The linears of a W8A8 layer: rows of activations to codes (int8_quant.hip), then the product (int8_gemm.hpp).
#include "int8_gemm.hpp"
#include "int8_rows.hpp"
#include "../../include/mi355x_qlinear.h"

namespace qlin {

template <class Act, int BM, int BN, int WM, int WN, int STAGES>
static int launch_tiles(Int8GemmArgs p, hipStream_t st) {
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  const long long tiles = (long long)p.tiles_m * p.tiles_n, grid = (tiles + 7) / 8 * 8;
  if (grid > 0x7FFFFFFFLL) return MI_ERR_SHAPE;
  auto* kernel = int8_gemm_kernel<Act, BM, BN, WM, WN, STAGES, kEpiOut, false>;
  constexpr size_t lds = (size_t)STAGES * (BM + BN) * kInt8Step;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WM * WN), lds, st, p);
  return launch_status();
}

template <class Act>
static int launch_product(const Int8GemmArgs& p, hipStream_t st) {
  return launch_tiles<Act, 128, 128, 2, 2, 2>(p, st);
}

struct Linear {
  int from;                   // kFrom*
  QuantArgs q;                // q, scale: filled in here
  const float* x_scale;       // kFromCodes: x is codes
};

static long long round256(long long v) { return (v + 255) / 256 * 256; }

static int run_linear(Linear l, const void* w, const float* w_scale, const void* bias, void* out, void* workspace,
                      long long workspace_bytes, int M, int N, int K, int act_dtype, void* stream) {
  if (act_dtype != DT_F16 && act_dtype != DT_BF16) return MI_ERR_ARG;
  if (!int8_sizes(M, N, K)) return MI_ERR_SHAPE;
  if (!M) return MI_OK;
  if (!l.q.x || (N && (!w || !w_scale || !out))) return MI_ERR_ARG;
  if (!aligned16(l.q.x) || !aligned16(w)) return MI_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  Int8RowsArgs r{l.q.x, l.x_scale, l.q.residual, l.q.residual_out, l.q.norm_weight, (const int8_t*)w, w_scale, bias, out, M, N, K, 0, l.q.eps};
  // one launch; the new residual must not be what other workgroups still read
  if (l.from != kFromCodes && N && int8_rows_quantise(l.from, M, K) && (l.from != kFromNorm || l.q.residual_out != l.q.residual))
    return launch_int8_rows(l.from, r, act_dtype, st);
  Int8GemmArgs p{};
  if (l.from == kFromCodes) {
    p.a = (const int8_t*)l.q.x;
    p.a_scale = l.x_scale;
  } else {
    long long need = 0;
    const int rc = mi_gemm_int8_workspace(M, N, K, &need);
    if (rc != MI_OK) return rc;
    if (!workspace || !aligned16(workspace) || workspace_bytes < need) return MI_ERR_ARG;
    l.q.q = (int8_t*)workspace;
    l.q.scale = (float*)((char*)workspace + round256((long long)M * K));
    l.q.rows = M;
    l.q.K = K;
    const int qc = launch_int8_quant(l.from, l.q, act_dtype, st);
    if (qc != MI_OK) return qc;
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
  p.wide_out = N % 4 == 0 && ((uintptr_t)out & 7) == 0;
  p.M = M;
  p.N = N;
  p.K = K;
  return act_dtype == DT_F16 ? launch_product<ActF16>(p, st) : launch_product<ActBF16>(p, st);
}

}  // namespace qlin

using namespace qlin;

extern "C" {

int mi_gemm_int8_workspace(int M, int N, int K, long long* bytes) {
  if (!bytes) return MI_ERR_ARG;
  if (!int8_sizes(M, N, K)) return MI_ERR_SHAPE;
  *bytes = round256((long long)M * K) + round256(4LL * M);
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
