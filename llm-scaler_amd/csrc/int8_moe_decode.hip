// The expert layer of int8_moe.hip for a few tokens, in two launches.  Bound: the weights of the selected experts, once per token, behind
// two round trips each: one token of 128 experts, top 8, 2048 / 768 with a shared expert (43 MB) takes 13.3 us (7.3 + 6.0), a copy of its bytes 8.3.
// With a selection and a quantised row in every wavefront 14.6.
//
// int8_gate_up_kernel: the first wavefront of a workgroup picks the experts of its columns (as many rounds of the selection as they are down
// the list); gate and up rows of a wavefront's columns are requested, all of them, and the workgroup quantises the token's row in the
// meantime, eight values a thread; SiLU(gate) x up goes out in fp32.  One more workgroup per token writes the selection for the second launch.
//
// int8_down_kernel: a workgroup quantises the h of a token's routes and of the shared expert into LDS; the k + 1 weight rows that make
// up an output are one sequence of 16-byte pieces over a wavefront's lanes, every lane scales its partial sums itself (route's weight, h's
// and the channel's scale), and one reduction ends the row.
#include "int8_moe.hpp"
#include "moe_topk.hpp"

namespace qlin {

constexpr int kGateWaves = 8, kDownWaves = 8, kGateMaxH = 4096;
constexpr int kDownPieces = 8;                        // weight pieces in flight per lane and row
constexpr int kDownHeld = 6;                          // pieces of 8 values of h per thread

template <int CTRL>
__device__ __forceinline__ int dpp_addi(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ int wave_isum(int v) {
  v = dpp_addi<0xB1>(v);
  v = dpp_addi<0x4E>(v);
  v = dpp_addi<0x141>(v);
  v = dpp_addi<0x140>(v);
  return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) + (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
}
__device__ __forceinline__ int dot16(i32x4 a, i32x4 b, int c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_sdot4(a[i], b[i], c, false);
  return c;
}

// SLOTS: experts per lane; NI: 1024-byte pieces of a weight row; RP: consecutive columns of the sequence (route, column) per wavefront
template <class Act, int SLOTS, int NI, int RP>
__global__ __launch_bounds__(64 * kGateWaves) void int8_gate_up_kernel(const Int8MoeArgs p) {
  using Elem = typename Act::elem;
  using V8 = typename Act::v8;
  static_assert(64 * kGateWaves * 8 >= kGateMaxH && NI * 1024 <= kGateMaxH && kGateWaves * RP <= 16, "a piece of x per thread; two routes");
  __shared__ __attribute__((aligned(16))) unsigned char codes[kGateMaxH];
  __shared__ uint32_t tops[kGateWaves];
  __shared__ int chosen[2];                           // the expert of the first and of the last column
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.y, k = p.k, E = p.E, H = p.H, I = p.I;
  const bool shared = p.shared_w13 != nullptr;
  if (blockIdx.x == gridDim.x - 1) {                  // this one hands the selection and the shared expert's gate on
    if (wave == 0)
      moe_topk_body<Act, SLOTS>((const Elem*)p.logits, (Elem*)p.top_w, p.ids, p.T, E, k, 1, nullptr, (const V8*)p.x, (const V8*)p.gate_weight,
                                shared ? p.gate : nullptr, H >> 3, t);
    return;
  }
  // the workgroup's columns are of one route or two (kGateWaves RP <= 16 <= I); a wavefront past the last has none
  const int columns = (k + (shared ? 1 : 0)) * I, c0 = blockIdx.x * kGateWaves * RP, q0 = c0 + wave * RP;
  const int ra = c0 / I, rb = (min(c0 + kGateWaves * RP, columns) - 1) / I;
  const int pieces = H >> 4;                          // 16-byte pieces of a weight row
  const int mine_at = threadIdx.x * 8;                // this thread's eight values of x
  const V8 xv = *reinterpret_cast<const V8*>((const Elem*)p.x + (size_t)t * H + (mine_at < H ? mine_at : 0));
  if (wave == 0 && ra < k) {
    Elem raws[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) raws[s] = ((const Elem*)p.logits)[(size_t)t * E + min(s * 64 + lane, E - 1)];
    uint32_t key[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int e = s * 64 + lane;
      key[s] = e < E ? (f16_order((uint32_t)__builtin_bit_cast(uint16_t, raws[s])) << 16) | (0xFFFFu - (uint32_t)e) : 0u;
    }
    int first = 0, last = 0;
    for (int r = 0; r <= min(rb, k - 1); ++r) {
      uint32_t best = 0;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) best = key[s] > best ? key[s] : best;
      best = wave_max_u32(best);
      last = (int)(0xFFFFu - (best & 0xFFFFu));
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
        if (s * 64 + lane == last) key[s] = 0u;
      if (r == ra) first = last;
    }
    if (lane == 0) {
      chosen[0] = first;
      chosen[1] = last;
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = umax32(top, abs_bits(Act::to_f32(xv[j])));         // past the row's end: its first piece again
  top = wave_max_u32(top);
  if (lane == 0) tops[wave] = top;
  lds_barrier();
  const int e0 = __builtin_amdgcn_readfirstlane(chosen[0]), e1 = __builtin_amdgcn_readfirstlane(chosen[1]);
  const int q1 = min(q0 + RP, columns) - 1;
  i32x4 wv[RP][2][NI];
  float ws[RP][2];
  if (q0 < columns) {
#pragma unroll
    for (int j = 0; j < RP; ++j) {
      const int q = min(q0 + j, q1), r = q >= rb * I ? rb : ra, n = q - r * I;
      const size_t e = (size_t)(r == ra ? e0 : e1);
      const int8_t* w = r >= k ? p.shared_w13 : p.w13 + e * 2 * (size_t)I * H;
      const float* sc = r >= k ? p.shared_s13 : p.s13 + e * 2 * (size_t)I;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const size_t row = (size_t)(n + u * I);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int c = i * 64 + lane < pieces ? i * 64 + lane : pieces - 1;
          wv[j][u][i] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(w + row * H) + c);
        }
        ws[j][u] = sc[row];
      }
    }
  }
  top = 0;
#pragma unroll
  for (int w = 0; w < kGateWaves; ++w) top = umax32(top, tops[w]);
  const RowScale s = row_scale(top);
  if (mine_at < H) {
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = code_of<true>(Act::to_f32(xv[j]), s.inv);
    *reinterpret_cast<u32x2*>(codes + mine_at) = u32x2{pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7])};
  }
  lds_barrier();
  if (q0 >= columns) return;
  i32x4 xq[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const bool in = i * 64 + lane < pieces;
    xq[i] = *reinterpret_cast<const i32x4*>(codes + (in ? i * 64 + lane : 0) * 16);
    if (!in) xq[i] = i32x4{0, 0, 0, 0};
  }
  float mine = 0.0f;                                  // lane j: column q0 + j
#pragma unroll
  for (int j = 0; j < RP; ++j) {
    int sum[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int d = 0;
#pragma unroll
      for (int i = 0; i < NI; ++i) d = dot16(wv[j][u][i], xq[i], d);
      sum[u] = wave_isum(d);
    }
    const float h = silu_mul((float)sum[0] * (s.scale * ws[j][0]), (float)sum[1] * (s.scale * ws[j][1]));
    mine = lane == j ? h : mine;
  }
  const int q = q0 + lane;
  if (lane < RP && q <= q1) p.h[q < k * I ? (size_t)t * k * I + q : ((size_t)p.T * k + t) * I + (q - k * I)] = mine;
}

template <class Act, int RPW>                         // output rows per wavefront
__global__ __launch_bounds__(64 * kDownWaves) void int8_down_kernel(const Int8MoeArgs p) {
  using Elem = typename Act::elem;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];        // [routes][I] codes
  __shared__ uint32_t tops[kDownHeld * kDownWaves];
  __shared__ float row_s[72];                         // of a route: its weight x the scale of its h; at most 65 routes
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t = blockIdx.y, k = p.k, H = p.H, I = p.I, routes = k + (p.shared_w13 ? 1 : 0);
  const int n0 = (blockIdx.x * kDownWaves + wave) * RPW;
  const unsigned per = (unsigned)I >> 4, total = per * (unsigned)routes;       // 16-byte pieces of a route's row, of an output row
  // h of all routes: pieces of 8 values, whole wavefronts per route; requested first
  const int waves_per_row = (I / 8 + 63) / 64, held = waves_per_row * routes;
  auto route_of = [&](int i) __attribute__((always_inline)) { return (i * kDownWaves + wave) / waves_per_row; };
  auto at_of = [&](int i, int r) __attribute__((always_inline)) { return ((i * kDownWaves + wave - r * waves_per_row) * 64 + lane) * 8; };
  f32v4 hv[kDownHeld][2];
#pragma unroll
  for (int i = 0; i < kDownHeld; ++i) {
    if (i * kDownWaves >= held) break;
    const int r = min(route_of(i), routes - 1), c = at_of(i, r), in = c < I ? c : 0;
    const f32v4* src = reinterpret_cast<const f32v4*>(p.h + (r < k ? (size_t)t * k + r : (size_t)p.T * k + t) * I + in);
    hv[i][0] = src[0];
    hv[i][1] = src[1];
  }
  i32x4 wv[RPW][kDownPieces];
  float f[RPW][kDownPieces];
  int route[kDownPieces];
  auto request = [&](unsigned s0) __attribute__((always_inline)) {
    unsigned s[kDownPieces];
    int e[kDownPieces];
#pragma unroll
    for (int i = 0; i < kDownPieces; ++i) {
      s[i] = s0 + i * 64 + lane;
      if (s[i] >= total) s[i] = total - 1;
      route[i] = (int)(s[i] / per);
      e[i] = p.ids[(size_t)t * k + min(route[i], k - 1)];
    }
#pragma unroll
    for (int i = 0; i < kDownPieces; ++i) {
      const bool shared = route[i] >= k;
      const unsigned c = s[i] - (unsigned)route[i] * per;
      const int8_t* w = shared ? p.shared_w2 : p.w2 + (size_t)e[i] * H * I;
      const float* sc = shared ? p.shared_s2 : p.s2 + (size_t)e[i] * H;
#pragma unroll
      for (int q = 0; q < RPW; ++q) {
        const int n = n0 + q < H ? n0 + q : H - 1;
        wv[q][i] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(w + (size_t)n * I) + c);
        f[q][i] = sc[n];
      }
    }
  };
  // a route's weight, or the shared expert's gate: for the thread that keeps the route's scale
  const int mine_r = min(tid, routes - 1);
  const float weight = mine_r < k ? Act::to_f32(((const Elem*)p.top_w)[(size_t)t * k + mine_r]) : p.gate[t];
  request(0);
#pragma unroll
  for (int i = 0; i < kDownHeld; ++i) {
    if (i * kDownWaves >= held) break;
    const int r = route_of(i);
    uint32_t top = 0;
    if (r < routes && at_of(i, r) < I) {
#pragma unroll
      for (int j = 0; j < 8; ++j) top = umax32(top, abs_bits(hv[i][j >> 2][j & 3]));
    }
    top = wave_max_u32(top);
    if (lane == 0) tops[i * kDownWaves + wave] = top;
  }
  lds_barrier();
#pragma unroll
  for (int i = 0; i < kDownHeld; ++i) {
    const int r = route_of(i), c = at_of(i, r);
    if (i * kDownWaves >= held || r >= routes) break;
    uint32_t top = 0;
    for (int q = 0; q < waves_per_row; ++q) top = umax32(top, tops[r * waves_per_row + q]);
    const RowScale s = row_scale(top);
    if (c < I) {
      uint32_t b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = code_of<false>(hv[i][j >> 2][j & 3], s.inv);
      *reinterpret_cast<u32x2*>(smem + (size_t)r * I + c) = u32x2{pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7])};
    }
  }
  if (tid < routes) {
    uint32_t top = 0;
    for (int q = 0; q < waves_per_row; ++q) top = umax32(top, tops[tid * waves_per_row + q]);
    row_s[tid] = weight * row_scale(top).scale;
  }
  lds_barrier();
  float acc[RPW];
#pragma unroll
  for (int q = 0; q < RPW; ++q) acc[q] = 0.0f;
  for (unsigned s0 = 0; s0 < total; s0 += 64 * kDownPieces) {
    if (s0) request(s0);
#pragma unroll
    for (int i = 0; i < kDownPieces; ++i) {
      unsigned s = s0 + i * 64 + lane;
      const bool in = s < total;                      // selected: what is repeated may be NaN
      if (!in) s = total - 1;
      const i32x4 a = *reinterpret_cast<const i32x4*>(smem + (size_t)s * 16);
      const float m = row_s[route[i]];
#pragma unroll
      for (int q = 0; q < RPW; ++q) {
        const float d = (float)dot16(wv[q][i], a, 0) * (f[q][i] * m);
        acc[q] = in ? acc[q] + d : acc[q];
      }
    }
  }
#pragma unroll
  for (int q = 0; q < RPW; ++q) {
    const float v = wave_sum(acc[q]);
    if (lane == 0 && n0 + q < H) ((Elem*)p.out)[(size_t)t * H + n0 + q] = Act::from_f32(v);
  }
}

template <class Act, int SLOTS, int NI>
static void launch_gate_up2(const Int8MoeArgs& p, hipStream_t st) {
  const int columns = (p.k + (p.shared_w13 ? 1 : 0)) * p.I;
  auto go = [&](auto rp) {
    constexpr int RP = decltype(rp)::value;
    const int per = kGateWaves * RP;
    hipLaunchKernelGGL((int8_gate_up_kernel<Act, SLOTS, NI, RP>), dim3((unsigned)((columns + per - 1) / per + 1), (unsigned)p.T),
                       dim3(64 * kGateWaves), 0, st, p);
  };
  // columns per wavefront, one / two, us: 1 token of 4096 / 1536 17.7 / 18.4, 4 tokens of 2048 / 768 35.6 / 34.2
  if (p.T == 1) go(std::integral_constant<int, 1>{});
  else go(std::integral_constant<int, 2>{});
}
template <class Act, int NI>
static void launch_gate_up1(const Int8MoeArgs& p, hipStream_t st) {
  if (p.E <= 128) launch_gate_up2<Act, 2, NI>(p, st);
  else if (p.E <= 256) launch_gate_up2<Act, 4, NI>(p, st);
  else launch_gate_up2<Act, 16, NI>(p, st);
}
template <class Act>
static int launch_decode(const Int8MoeArgs& p, hipStream_t st) {
  if (p.H <= 1024) launch_gate_up1<Act, 1>(p, st);
  else if (p.H <= 2048) launch_gate_up1<Act, 2>(p, st);
  else launch_gate_up1<Act, 4>(p, st);
  const size_t lds = (size_t)(p.k + (p.shared_w13 ? 1 : 0)) * p.I;
  auto go = [&](auto rpw) {
    constexpr int RPW = decltype(rpw)::value;
    hipLaunchKernelGGL((int8_down_kernel<Act, RPW>), dim3((unsigned)((p.H + kDownWaves * RPW - 1) / (kDownWaves * RPW)), (unsigned)p.T),
                       dim3(64 * kDownWaves), lds, st, p);
  };
  // one round of workgroups: every one of them quantises all of h (twice as many: 4 tokens of 2048 / 768 34.8 -> 38.0 us)
  const int cus = int8_cu_count(), groups = (p.H + kDownWaves - 1) / kDownWaves * p.T;
  if (groups <= cus) go(std::integral_constant<int, 1>{});
  else if (groups <= 2 * cus) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, 4>{});
  return launch_status();
}

// Every token reads the experts of its routes and the shared expert for itself; sorted by expert they are read once, by four launches more.
// The two launches are ahead while what is expected to be read again stays below 100 MB (two launches / six, us, with a shared expert; E, top, H, I):
// 128, 8, 2048, 768: 1 token 14.8 / 29.6, 8 tokens (91 MB) 60 / 74, 10 tokens (133) 76 / 78, 14 tokens 102 / 92; 8, 2, 4096, 1536: 2 tokens 26 / 37,
// 3 tokens (64) 39 / 41, 4 tokens (104) 44 / 41, 6 tokens 63 / 47; 64, 6, 2048, 1408: 4 tokens (53) 47 / 62, 6 tokens (108) 71 / 72, 8 tokens 82 / 80; 16, 2,
// 2048, 1024: 6 tokens (51) 30 / 31, 8 tokens (79) 34 / 33, 12 tokens (140) 47 / 34; 32, 4, 1024, 512: 8 tokens (28) 19 / 27, 16 tokens (80) 30 / 28.
bool int8_moe_decode_pays(int T, int k, int E, int H, int I, bool shared) {
  const int routes = k + (shared ? 1 : 0);
  if (H > kGateMaxH || (I / 8 + 63) / 64 * routes > kDownHeld * kDownWaves || routes * I > 60 * 1024) return false;
  if ((long long)T * k > 96) return false;
  double missed = 1.0;                                // the share of the experts that no token takes
  for (int t = 0; t < T; ++t) missed *= 1.0 - (double)k / E;
  const double again = (double)T * routes - E * (1.0 - missed) - (shared ? 1 : 0);
  return again * 3.0 * H * I <= 100e6;
}
int launch_int8_moe_decode(const Int8MoeArgs& p, int act_dtype, hipStream_t st) {
  return act_dtype == DT_F16 ? launch_decode<ActF16>(p, st) : launch_decode<ActBF16>(p, st);
}

}  // namespace qlin
