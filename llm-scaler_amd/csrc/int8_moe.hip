// A mixture-of-experts layer on 8-bit integer experts (W8A8), from the router's logits to the layer's output:
//
//   out[t] = sum_j top_w[t][j] expert(ids[t][j], x[t]) + sigmoid(x[t] . gate_weight) shared(x[t]),
//   expert(e, x) = W2[e] q(h),   h = SiLU(g) u,   (g, u) = W13[e] q(x)
//
// with q() the rows' quantisation of int8_common.hpp; g, u, h and the experts' results stay in fp32, the output is rounded once.
//
// Selection, codes of x, pairs sorted by expert, a tile table, the grouped product with SiLU(gate) x up, codes of h, the grouped down product
// and the weighted sum.  The shared expert is one more expert, with a row for every token.
#include "int8_gemm.hpp"
#include "int8_moe.hpp"
#include "../../include/mi355x_qlinear.h"

namespace qlin {

constexpr int kTileThreads = 1024;

// Tiles of `bm` rows that cover each expert's rows (expert E: the T rows behind the P sorted pairs), and the row of x of every position.
__global__ __launch_bounds__(kTileThreads) void int8_tiles_kernel(const int32_t* __restrict__ start, int32_t* __restrict__ tile,
                                                                  int32_t* __restrict__ row, int E, int P, int T, int bm, int most) {
  __shared__ int32_t total[kTileThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int first = tid < E ? start[tid] : 0, n = tid < E ? start[tid + 1] - first : 0;   // E <= kTileThreads
  const int mine = (n + bm - 1) / bm;
  int sum = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(sum, off, 64);
    if (lane >= off) sum += o;
  }
  if (lane == 63) total[wave] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kTileThreads / 64; ++w) {
    if (w < wave) before += total[w];
    all += total[w];
  }
  const int at = before + sum - mine;
  for (int i = 0; i < mine; ++i) {
    int32_t* t = tile + 4 * (at + i);
    t[0] = tid;
    t[1] = first + i * bm;
    t[2] = n - i * bm < bm ? n - i * bm : bm;
  }
  const int shared = (T + bm - 1) / bm;               // T = 0: no shared expert
  for (int i = tid; i < shared; i += kTileThreads) {
    int32_t* t = tile + 4 * (all + i);
    t[0] = E;
    t[1] = P + i * bm;
    t[2] = T - i * bm < bm ? T - i * bm : bm;
  }
  for (int i = tid; i < T; i += kTileThreads) row[P + i] = i;
  if (tid == 0) tile[4 * most] = all + shared;
}

// out[t] = sum_j w[t][j] y[inv[t k + j]] + gate[t] y[P + t], fp32, one rounding.  Eight columns per thread.
template <class Act>
__global__ __launch_bounds__(256) void int8_combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ inv,
                                                           const typename Act::elem* __restrict__ top_w, const float* __restrict__ gate,
                                                           typename Act::elem* __restrict__ out, int T, int k, int H) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int per = H / 8;
  const long long t = i / per;
  if (t >= T) return;
  const int c = (int)(i - t * per) * 8;
  float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](size_t row, float w) __attribute__((always_inline)) {
    const f32v4* src = reinterpret_cast<const f32v4*>(y + row * H + c);
    const f32v4 a = src[0], b = src[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) { s[j] += w * a[j]; s[4 + j] += w * b[j]; }
  };
  for (int j = 0; j < k; ++j) add((size_t)inv[t * k + j], Act::to_f32(top_w[t * k + j]));
  if (gate) add((size_t)T * k + t, gate[t]);
  typename Act::v8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = Act::from_f32(s[j]);
  *reinterpret_cast<typename Act::v8*>(out + t * H + c) = o;
}

constexpr int kGroupRows = 128;

struct MoeLayout {                                    // byte offsets into the workspace
  long long top_w, ids, gate, pairs, start, inv, row, tile, xq, xs, h, hq, hs, y, bytes;
  long long P, rows, tiles;
};
static MoeLayout moe_layout(int T, int k, int E, int H, int I, int shared) {
  MoeLayout l{};
  l.P = (long long)T * k;
  const long long S = shared ? T : 0;
  l.rows = l.P + S;
  l.tiles = l.P / kGroupRows + (l.P < E ? l.P : E) + (S + kGroupRows - 1) / kGroupRows;
  auto take = [&](long long n) { const long long at = l.bytes; l.bytes += (n + 255) / 256 * 256; return at; };
  l.top_w = take(2 * l.P);
  l.ids = take(4 * l.P);
  l.gate = take(4LL * T);
  l.pairs = take(4 * l.P);
  l.start = take(4LL * (E + 1));
  l.inv = take(4 * l.P);
  l.row = take(4 * l.rows);
  l.tile = take(16 * (l.tiles + 1));
  l.xq = take((long long)T * H);
  l.xs = take(4LL * T);
  l.h = take(4 * l.rows * I);
  l.hq = take(l.rows * I);
  l.hs = take(4 * l.rows);
  l.y = take(4 * l.rows * H);
  return l;
}

template <class Act, int EPI, int BM, int BN, int WM, int WN, int KG, int SA, int SB>
static int launch_tiles(Int8GemmArgs p, long long tiles, hipStream_t st) {
  constexpr int BNO = EPI == kEpiAct ? BN / 2 : BN;
  const int NO = EPI == kEpiAct ? p.N / 2 : p.N;
  p.tiles_m = (int)tiles;
  p.tiles_n = (NO + BNO - 1) / BNO;
  const long long grid = (tiles * p.tiles_n + 7) / 8 * 8;
  if (grid > 0x7FFFFFFFLL) return MI_ERR_SHAPE;
  auto* kernel = int8_gemm_kernel<Act, BM, BN, WM, WN, KG, SA, SB, EPI, true>;
  constexpr size_t lds = int8_gemm_lds(BM, BN, WM * WN, KG, SA, SB);
  if constexpr (lds > 64 * 1024) {
    static std::atomic<unsigned long long> raised{0};
    const int rc = int8_raise_lds(kernel, raised, lds);
    if (rc != MI_OK) return rc;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WM * WN * KG), lds, st, p);
  return launch_status();
}

template <class Act, int EPI>
static int launch_grouped(const Int8GemmArgs& p, long long tiles, hipStream_t st) {
  return launch_tiles<Act, EPI, kGroupRows, 128, 2, 2, 1, 2, 2>(p, tiles, st);
}

static bool moe_sizes(int T, int k, int E, int H, int I) {
  if (T < 0 || E < 1 || E > 1024 || k < 1 || k > 64 || k > E) return false;
  if (!int8_sizes(T, 2, H) || !int8_sizes(T, 2, I)) return false;
  const long long pairs = (long long)T * (k + 1);
  return 2LL * I * H < (1LL << 31) && (long long)T * H < (1LL << 31) && pairs * I < (1LL << 31) && pairs < (1LL << 31) - 1024;
}

template <class Act>
static int run_moe(const Int8MoeArgs& m, char* ws, hipStream_t st) {
  const int T = m.T, k = m.k, E = m.E, H = m.H, I = m.I;
  const void *x = m.x, *logits = m.logits;
  const bool shared = m.shared_w13 != nullptr;
  const MoeLayout l = moe_layout(T, k, E, H, I, shared);
  int32_t *ids = (int32_t*)(ws + l.ids), *start = (int32_t*)(ws + l.start), *inv = (int32_t*)(ws + l.inv), *row = (int32_t*)(ws + l.row);
  int32_t* tile = (int32_t*)(ws + l.tile);
  float* gate = shared ? (float*)(ws + l.gate) : nullptr;
  int rc = mi_moe_topk(logits, ws + l.top_w, ids, T, E, k, 1, nullptr, shared ? x : nullptr, m.gate_weight, gate, H, Act::dt, st);
  if (rc != MI_OK) return rc;
  QuantArgs q{};
  q.x = x;
  q.q = (int8_t*)(ws + l.xq);
  q.scale = (float*)(ws + l.xs);
  q.rows = T;
  q.K = H;
  rc = launch_int8_quant(kFromAct, q, Act::dt, st);
  if (rc != MI_OK) return rc;
  rc = mi_moe_sort(ids, (int32_t*)(ws + l.pairs), start, inv, row, nullptr, T, k, E, st);
  if (rc != MI_OK) return rc;
  hipLaunchKernelGGL(int8_tiles_kernel, dim3(1), dim3(kTileThreads), 0, st, start, tile, row, E, (int)l.P, shared ? T : 0, kGroupRows,
                     (int)l.tiles);
  Int8GemmArgs p{};
  p.a = q.q;
  p.a_scale = q.scale;
  p.w = m.w13;
  p.w_scale = m.s13;
  p.out = ws + l.h;
  p.M = T;
  p.N = 2 * I;
  p.K = H;
  p.g_tile = tile;
  p.g_row = row;
  p.shared_w = m.shared_w13;
  p.shared_scale = m.shared_s13;
  p.E = E;
  rc = launch_grouped<Act, kEpiAct>(p, l.tiles, st);
  if (rc != MI_OK) return rc;
  q.x = ws + l.h;
  q.q = (int8_t*)(ws + l.hq);
  q.scale = (float*)(ws + l.hs);
  q.rows = l.rows;
  q.K = I;
  rc = launch_int8_quant(kFromF32, q, Act::dt, st);
  if (rc != MI_OK) return rc;
  p.a = q.q;
  p.a_scale = q.scale;
  p.w = m.w2;
  p.w_scale = m.s2;
  p.out = ws + l.y;
  p.M = (int)l.rows;
  p.N = H;
  p.K = I;
  p.g_row = nullptr;
  p.shared_w = m.shared_w2;
  p.shared_scale = m.shared_s2;
  rc = launch_grouped<Act, kEpiF32>(p, l.tiles, st);
  if (rc != MI_OK) return rc;
  hipLaunchKernelGGL(int8_combine_kernel<Act>, dim3((unsigned)(((long long)T * (H / 8) + 255) / 256)), dim3(256), 0, st,
                     (const float*)(ws + l.y), inv, (const typename Act::elem*)(ws + l.top_w), gate, (typename Act::elem*)m.out, T, k, H);
  return launch_status();
}

}  // namespace qlin

using namespace qlin;

extern "C" {

int mi_moe_forward_full_int8_workspace(int T, int topk, int num_experts, int H, int I, int shared, long long* bytes) {
  if (!bytes) return MI_ERR_ARG;
  if (!moe_sizes(T, topk, num_experts, H, I)) return MI_ERR_SHAPE;
  *bytes = moe_layout(T, topk, num_experts, H, I, shared).bytes;
  return MI_OK;
}

int mi_moe_forward_full_int8_ws(const void* x, const void* logits, void* out, const void* w13, const float* w13_scale,
                                const void* shared_w13, const float* shared_w13_scale, const void* w2, const float* w2_scale,
                                const void* shared_w2, const float* shared_w2_scale, const void* gate_weight, void* workspace,
                                long long workspace_bytes, int T, int topk, int num_experts, int H, int I, int act_dtype, void* stream) {
  if (act_dtype != DT_F16 && act_dtype != DT_BF16) return MI_ERR_ARG;
  if (!moe_sizes(T, topk, num_experts, H, I)) return MI_ERR_SHAPE;
  if (!T) return MI_OK;
  if (!x || !logits || !out || !w13 || !w13_scale || !w2 || !w2_scale) return MI_ERR_ARG;
  const bool shared = shared_w13 != nullptr;           // all five or none
  if (shared != (shared_w13_scale != nullptr) || shared != (shared_w2 != nullptr) || shared != (shared_w2_scale != nullptr) ||
      shared != (gate_weight != nullptr))
    return MI_ERR_ARG;
  for (const void* q : {x, (const void*)out, w13, w2, shared_w13, shared_w2, gate_weight, (const void*)workspace})
    if (!aligned16(q)) return MI_ERR_ARG;
  if (!workspace || workspace_bytes < moe_layout(T, topk, num_experts, H, I, shared).bytes) return MI_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  const MoeLayout l = moe_layout(T, topk, num_experts, H, I, shared);
  char* ws = (char*)workspace;
  const Int8MoeArgs m{x, logits, out, (const int8_t*)w13, (const int8_t*)w2, w13_scale, w2_scale, (const int8_t*)shared_w13,
                      (const int8_t*)shared_w2, shared_w13_scale, shared_w2_scale, gate_weight, ws + l.top_w, (int32_t*)(ws + l.ids),
                      (float*)(ws + l.gate), (float*)(ws + l.h), T, topk, num_experts, H, I};
  if (int8_moe_decode_pays(T, topk, H, I, shared)) return launch_int8_moe_decode(m, act_dtype, st);
  return act_dtype == DT_F16 ? run_moe<ActF16>(m, ws, st) : run_moe<ActBF16>(m, ws, st);
}

}  // extern "C"
