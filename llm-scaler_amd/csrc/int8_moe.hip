// A mixture-of-experts layer on 8-bit integer experts (W8A8), from the router's logits to the layer's output:
//
//   out[t] = sum_j top_w[t][j] expert(ids[t][j], x[t]) + sigmoid(x[t] . gate_weight) shared(x[t]),
//   expert(e, x) = W2[e] q(h),   h = SiLU(g) u,   (g, u) = W13[e] q(x)
//
// with q() the rows' quantisation of int8_common.hpp; g, u, h and the sums stay in fp32, the output is rounded once.
//
// Few tokens: int8_moe_decode.hip.  Otherwise six launches: selection beside the codes of x, pairs sorted by expert with a tile table, the grouped
// product with SiLU(gate) x up, codes of h, the grouped down product, the weighted sum.  The shared expert is one more expert, with a
// row for every token.
#include "int8_gemm.hpp"
#include "int8_moe.hpp"
#include "int8_quant.hpp"
#include "moe_topk.hpp"
#include "../../include/mi355x_qlinear.h"

namespace qlin {

constexpr int kSortThreads = 1024;                    // E <= kSortThreads
// The shared expert's row tiles come last and have fewer rows, so that the last round of workgroups is a short one.  The whole layer, us (with results
// of 16 bits), with / without: 128 experts, top 8, 2048 / 768, 4096 tokens 349 / 358; 8 experts, top 2, 4096 / 1536, 4096 tokens 327 / 341; of 128 rows 346 and 359.
__host__ __device__ static inline int shared_rows(int bm) { return bm < 192 ? bm : 192; }
constexpr int kSortPairs = 8;                         // pairs per thread of int8_sort_kernel

// Tiles of at most `bm` rows that cover the `n` rows of every expert (thread = expert) from its first position on, and those of the
// shared expert (E): the T rows behind the P sorted pairs.  Returns the expert's first position.  A workgroup of kSortThreads.
__device__ __forceinline__ int write_tiles(int n, int32_t* __restrict__ tile, int32_t* __restrict__ row, int E, int P, int T, int bm, int most) {
  __shared__ int32_t totals[2][kSortThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int mine = (n + bm - 1) / bm;
  int tiles = mine, pairs = n;                        // inclusive sums
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int a = __shfl_up(tiles, off, 64), b = __shfl_up(pairs, off, 64);
    if (lane >= off) { tiles += a; pairs += b; }
  }
  if (lane == 63) { totals[0][wave] = tiles; totals[1][wave] = pairs; }
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kSortThreads / 64; ++w) {
    if (w < wave) { tiles += totals[0][w]; pairs += totals[1][w]; }
    all += totals[0][w];
  }
  const int first = pairs - n;
  for (int i = 0; i < mine; ++i) {
    int32_t* t = tile + 4 * (tiles - mine + i);
    t[0] = tid;
    t[1] = first + i * bm;
    t[2] = n - i * bm < bm ? n - i * bm : bm;
  }
  const int sm = shared_rows(bm), shared = (T + sm - 1) / sm;               // T = 0: no shared expert
  for (int i = tid; i < shared; i += kSortThreads) {
    int32_t* t = tile + 4 * (all + i);
    t[0] = E;
    t[1] = P + i * sm;
    t[2] = T - i * sm < sm ? T - i * sm : sm;
  }
  for (int i = tid; i < T; i += kSortThreads) row[P + i] = i;
  if (tid == 0) tile[4 * most] = all + shared;
  return first;
}

// After mi_moe_sort: the tiles alone.
__global__ __launch_bounds__(kSortThreads) void int8_tiles_kernel(const int32_t* __restrict__ start, int32_t* __restrict__ tile,
                                                                  int32_t* __restrict__ row, int E, int P, int T, int bm, int most) {
  const int e = threadIdx.x;
  write_tiles(e < E ? start[e + 1] - start[e] : 0, tile, row, E, P, T, bm, most);
}

// Up to kSortPairs x kSortThreads pairs: sorted by expert and tiled by one workgroup.  inv: a pair's position, row: a position's token.  The order
// inside an expert is that of the LDS atomics; every row's result is its own, so the outputs do not depend on it.
__global__ __launch_bounds__(kSortThreads) void int8_sort_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ inv,
                                                                 int32_t* __restrict__ row, int32_t* __restrict__ tile, int E, int k, int P, int T,
                                                                 int bm, int most) {
  __shared__ int32_t count[kSortThreads];
  const int tid = threadIdx.x;
  count[tid] = 0;
  __syncthreads();
  int id[kSortPairs], rank[kSortPairs];
#pragma unroll
  for (int i = 0; i < kSortPairs; ++i) {
    if (i * kSortThreads >= P) break;
    id[i] = ids[min(i * kSortThreads + tid, P - 1)];
  }
#pragma unroll
  for (int i = 0; i < kSortPairs; ++i) {
    if (i * kSortThreads >= P) break;
    if (i * kSortThreads + tid < P) rank[i] = atomicAdd(&count[id[i]], 1);
  }
  __syncthreads();
  const int n = count[tid];
  const int first = write_tiles(n, tile, row, E, P, T, bm, most);              // a barrier inside: every count is read
  count[tid] = first;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortPairs; ++i) {
    const int p = i * kSortThreads + tid;
    if (i * kSortThreads >= P) break;
    if (p < P) {
      const int at = count[id[i]] + rank[i];
      inv[p] = at;
      row[at] = p / k;
    }
  }
}

// Selection of a token's experts (with the shared expert's gate) and codes of its row do not depend on each other: one launch, a
// wavefront per token for the first, workgroups behind them for the second.
template <class Act, int SLOTS, int NV>
__global__ __launch_bounds__(256) void int8_route_kernel(const Int8MoeArgs p, int8_t* __restrict__ q, float* __restrict__ scale, int routing) {
  using Elem = typename Act::elem;
  using V8 = typename Act::v8;
  if ((int)blockIdx.x < routing) {
    moe_topk_body<Act, SLOTS>((const Elem*)p.logits, (Elem*)p.top_w, p.ids, p.T, p.E, p.k, 1, nullptr, (const V8*)p.x, (const V8*)p.gate_weight,
                              p.shared_w13 ? p.gate : nullptr, p.H >> 3, blockIdx.x * 4 + (threadIdx.x >> 6));
    return;
  }
  QuantArgs a{};
  a.x = p.x;
  a.q = q;
  a.scale = scale;
  a.rows = p.T;
  a.K = p.H;
  int8_quant_rows<Act, kFromAct, 256, NV>(a, (int)blockIdx.x - routing);
}

// out[t] = sum_j w[t][j] y[inv[t k + j]] + gate[t] y[P + t], fp32, one rounding; y as kEpiFloat24 leaves it.  Eight columns per thread.
// Bound: HBM (4096 tokens of 9 rows of 2048: 40 us, 6.1 TB/s).
template <class Act>
__global__ __launch_bounds__(256) void int8_combine_kernel(const uint16_t* __restrict__ y, const unsigned char* __restrict__ y_low,
                                                           const int32_t* __restrict__ inv, const typename Act::elem* __restrict__ top_w,
                                                           const float* __restrict__ gate, typename Act::elem* __restrict__ out, int T, int k, int H) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int per = H / 8;
  const long long t = i / per;
  if (t >= T) return;
  const int c = (int)(i - t * per) * 8;
  float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](size_t row, float w) __attribute__((always_inline)) {
    const u32x4 high = *reinterpret_cast<const u32x4*>(y + row * H + c);
    const u32x2 low = *reinterpret_cast<const u32x2*>(y_low + row * H + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bytes = (j & 1 ? 0x07060000u : 0x05040000u) | (uint32_t)(j & 3) << 8 | 0x0Cu;
      s[j] += w * __builtin_bit_cast(float, __builtin_amdgcn_perm(high[j >> 1], low[j >> 2], bytes));
    }
  };
  for (int j0 = 0; j0 < k; j0 += 8) {                  // eight rows' positions, then eight rows
    int at[8];
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long p = t * k + (j0 + j < k ? j0 + j : k - 1);
      at[j] = inv[p];
      w[j] = Act::to_f32(top_w[p]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j0 + j < k) add((size_t)at[j], w[j]);
  }
  if (gate) add((size_t)T * k + t, gate[t]);
  typename Act::v8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = Act::from_f32(s[j]);
  *reinterpret_cast<typename Act::v8*>(out + t * H + c) = o;
}

// Rows of a tile, by the rows that an expert has on average: most experts in one row tile, up to 318, then in two.  Up to 192 rows there is
// room for two workgroups on a CU, of eight wavefronts each: one begins and ends its tile while the other multiplies (four wavefronts per workgroup:
// 3 % slower).  The whole layer, us, tile / next: 128 experts, top 8, 2048 / 768: 200 tokens 32 x 128 144 / 64 x 128 146; 600 tokens 64 x 128 168 /
// 128 x 128 189; 1500 tokens 128 x 128 232 / 192 x 128 245; 2300 tokens 192 x 128 280 / 256 x 256 290; 3500 tokens 256 x 256 344 / 320 x 192 355; 4096 tokens
// 320 x 192 386 / 256 x 256 405; 5600 tokens 192 x 128 529 / 256 x 256 566, 7000 tokens 256 x 256 638 / 192 x 128 676; 64 experts, top 6, 2048 / 1408:
// 900 tokens 128 x 128 197 / 192 x 128 212, 1700 tokens 192 x 128 250 / 256 x 256 255; 8 experts, top 2, 4096 / 1536: 1200 tokens 320 x 192 140 /
// 192 x 128 151, 4096 tokens 256 x 256 347 / 192 x 128 373.
enum : int { kRows32, kRows64, kRows128, kRows192, kRows256, kRows320 };
constexpr int kGroupRows[] = {32, 64, 128, 192, 256, 320};
static int group_tile(long long pairs, int E) {
  if (pairs <= 24LL * E) return kRows32;
  if (pairs <= 66LL * E) return kRows64;
  if (pairs <= 125LL * E) return kRows128;
  if (pairs <= 182LL * E) return kRows192;
  if (pairs <= 245LL * E) return kRows256;
  if (pairs <= 318LL * E) return kRows320;
  return pairs <= 385LL * E ? kRows192 : kRows256;     // two of 192, two and more of 256
}

struct MoeLayout {                                    // byte offsets into the workspace
  long long top_w, ids, gate, pairs, start, inv, row, tile, xq, xs, h, hq, hs, y, yl, bytes;
  long long P, rows, tiles;
  int tile_kind, bm;
};
static MoeLayout moe_layout(int T, int k, int E, int H, int I, int shared) {
  MoeLayout l{};
  l.P = (long long)T * k;
  const long long S = shared ? T : 0;
  l.rows = l.P + S;
  l.tile_kind = group_tile(l.P, E);
  l.bm = kGroupRows[l.tile_kind];
  l.tiles = l.P / l.bm + (l.P < E ? l.P : E) + (S + shared_rows(l.bm) - 1) / shared_rows(l.bm);
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
  l.y = take(2 * l.rows * H);
  l.yl = take(l.rows * H);
  return l;
}

template <class Act, int EPI, int BM, int BN, int WM, int WN, int KG, int SA, int SB>
static int launch_tiles(Int8GemmArgs p, long long tiles, hipStream_t st) {
  constexpr int BNO = EPI == kEpiAct ? BN / 2 : BN;
  const int NO = EPI == kEpiAct ? p.N / 2 : p.N;
  p.tiles_m = (int)tiles;
  p.tiles_n = (NO + BNO - 1) / BNO;
  const long long grid = (tiles + 7) / 8 * 8 * p.tiles_n;
  if (grid > 0x7FFFFFFFLL) return MI_ERR_SHAPE;
  auto* kernel = int8_gemm_kernel<Act, BM, BN, WM, WN, KG, SA, SB, EPI, true>;
  constexpr size_t lds = int8_gemm_lds(BM, BN, KG, SA, SB);
  if constexpr (lds > 64 * 1024) {
    static std::atomic<unsigned long long> raised{0};
    const int rc = int8_raise_lds(kernel, raised, lds);
    if (rc != MI_OK) return rc;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WM * WN * KG), lds, st, p);
  return launch_status();
}

template <class Act, int EPI>
static int launch_grouped(const Int8GemmArgs& p, const MoeLayout& l, hipStream_t st) {
  switch (l.tile_kind) {
    case kRows32: return launch_tiles<Act, EPI, 32, 128, 2, 4, 1, 3, 3>(p, l.tiles, st);
    case kRows64: return launch_tiles<Act, EPI, 64, 128, 2, 4, 1, 3, 3>(p, l.tiles, st);
    case kRows128: return launch_tiles<Act, EPI, 128, 128, 2, 4, 1, 2, 3>(p, l.tiles, st);
    case kRows192: return launch_tiles<Act, EPI, 192, 128, 4, 2, 1, 2, 2>(p, l.tiles, st);
    case kRows256: return launch_tiles<Act, EPI, 256, 256, 4, 2, 1, 2, 3>(p, l.tiles, st);
    default: return launch_tiles<Act, EPI, 320, 192, 4, 2, 1, 2, 3>(p, l.tiles, st);
  }
}

template <class Act, int SLOTS>
static void launch_route2(const Int8MoeArgs& m, int8_t* q, float* scale, hipStream_t st) {
  const int routing = (m.T + 3) / 4, pieces = m.H / 8;
  const dim3 grid((unsigned)(routing + m.T)), block(256);
  if (pieces <= 256) hipLaunchKernelGGL((int8_route_kernel<Act, SLOTS, 1>), grid, block, 0, st, m, q, scale, routing);
  else if (pieces <= 512) hipLaunchKernelGGL((int8_route_kernel<Act, SLOTS, 2>), grid, block, 0, st, m, q, scale, routing);
  else if (pieces <= 1024) hipLaunchKernelGGL((int8_route_kernel<Act, SLOTS, 4>), grid, block, 0, st, m, q, scale, routing);
  else hipLaunchKernelGGL((int8_route_kernel<Act, SLOTS, 0>), grid, block, 0, st, m, q, scale, routing);
}
template <class Act>
static int launch_route(const Int8MoeArgs& m, int8_t* q, float* scale, hipStream_t st) {
  if (m.E <= 128) launch_route2<Act, 2>(m, q, scale, st);
  else if (m.E <= 256) launch_route2<Act, 4>(m, q, scale, st);
  else launch_route2<Act, 16>(m, q, scale, st);
  return launch_status();
}

static bool moe_sizes(int T, int k, int E, int H, int I) {
  if (T < 0 || E < 1 || E > 1024 || k < 1 || k > 64 || k > E) return false;
  if (!int8_sizes(T, 2, H) || !int8_sizes(T, 2, I)) return false;
  const long long pairs = (long long)T * (k + 1);
  return 2LL * I * H < (1LL << 31) && (long long)T * H < (1LL << 31) && pairs * I < (1LL << 31) && pairs <= kInt8MaxRows;
}

template <class Act>
static int run_moe(const Int8MoeArgs& m, char* ws, hipStream_t st) {
  const int T = m.T, k = m.k, E = m.E, H = m.H, I = m.I;
  const bool shared = m.shared_w13 != nullptr;
  const MoeLayout l = moe_layout(T, k, E, H, I, shared);
  int32_t *start = (int32_t*)(ws + l.start), *inv = (int32_t*)(ws + l.inv), *row = (int32_t*)(ws + l.row);
  int32_t* tile = (int32_t*)(ws + l.tile);
  QuantArgs q{};
  q.q = (int8_t*)(ws + l.xq);
  q.scale = (float*)(ws + l.xs);
  int rc = launch_route<Act>(m, q.q, q.scale, st);
  if (rc != MI_OK) return rc;
  if (l.P <= (long long)kSortPairs * kSortThreads) {
    hipLaunchKernelGGL(int8_sort_kernel, dim3(1), dim3(kSortThreads), 0, st, m.ids, inv, row, tile, E, k, (int)l.P, shared ? T : 0, l.bm,
                       (int)l.tiles);
  } else {
    rc = mi_moe_sort(m.ids, (int32_t*)(ws + l.pairs), start, inv, row, nullptr, T, k, E, st);
    if (rc != MI_OK) return rc;
    hipLaunchKernelGGL(int8_tiles_kernel, dim3(1), dim3(kSortThreads), 0, st, start, tile, row, E, (int)l.P, shared ? T : 0, l.bm, (int)l.tiles);
  }
  rc = launch_status();
  if (rc != MI_OK) return rc;
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
  rc = launch_grouped<Act, kEpiAct>(p, l, st);
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
  p.low = (unsigned char*)(ws + l.yl);
  p.M = (int)l.rows;
  p.N = H;
  p.K = I;
  p.g_row = nullptr;
  p.shared_w = m.shared_w2;
  p.shared_scale = m.shared_s2;
  rc = launch_grouped<Act, kEpiFloat24>(p, l, st);
  if (rc != MI_OK) return rc;
  hipLaunchKernelGGL(int8_combine_kernel<Act>, dim3((unsigned)(((long long)T * (H / 8) + 255) / 256)), dim3(256), 0, st,
                     (const uint16_t*)(ws + l.y), p.low, inv, (const typename Act::elem*)m.top_w, shared ? m.gate : nullptr,
                     (typename Act::elem*)m.out, T, k, H);
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
  if (int8_moe_decode_pays(T, topk, num_experts, H, I, shared)) return launch_int8_moe_decode(m, act_dtype, st);
  return act_dtype == DT_F16 ? run_moe<ActF16>(m, ws, st) : run_moe<ActBF16>(m, ws, st);
}

}  // extern "C"
