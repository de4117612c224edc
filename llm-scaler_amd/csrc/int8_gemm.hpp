// Product of 8-bit codes on the matrix cores: out[m][n] = (sum_k a[m][k] w[n][k]) a_scale[m] w_scale[n].
//
// A workgroup owns a BM x BN tile.  Both operands go to LDS straight from memory (128-byte pieces of a row per step, no registers
// and no vector instructions in between) into rings of SA and SB buffers; a wavefront multiplies (16 TM) x (16 TN) of the tile with
// v_mfma_i32_16x16x64_i8; where a tile's K is long beside its rows and columns, KG groups of wavefronts take a 128-byte piece of every
// step each, which keeps more loads under way, and their sums meet at the end.  16-byte chunk c of tile row r lies at
// place c ^ f(r) of its 128 bytes, so that the eight lanes that read at a time find eight different places.  The weights are the first
// operand: a lane ends with consecutive output columns of one row, 4 per MFMA tile, and the weight rows of GJ tiles are interleaved so that
// these are 4 GJ in a row.
//
// Bound: the matrix cores and the loads that feed them for many rows (2048 x 4096 x 14336 116 us, 2.1 POP/s; 8192^3 454 us, 2.4), the weights' way
// from HBM through LDS for few (64 x 5120 x 5120 10.0 us, 2.9 TB/s).
#pragma once
#include "int8_common.hpp"

#include <type_traits>

namespace qlin {

struct Int8GemmArgs {
  const int8_t* a;            // [rows, K]
  const float* a_scale;       // [rows]
  const int8_t* w;            // [N, K]; grouped [E, N, K]
  const float* w_scale;       // [N]; grouped [E, N]
  const void* bias;           // [N] in the output's type, or null
  void* out;
  unsigned char* low;         // kEpiFloat24
  int M, N, K;                // M: rows of a
  int tiles_m, tiles_n;
  // Grouped: tile i covers the rows [g_tile[4 i + 1], + g_tile[4 i + 2]) of the expert-sorted order and multiplies them with expert
  // g_tile[4 i]; row r of that order is row g_row[r] of a (null: r).  Expert E is the shared one.  g_tile[4 tiles_m]: tiles in use.
  const int32_t* g_tile;
  const int32_t* g_row;
  const int8_t* shared_w;
  const float* shared_scale;
  int E;
};

// What becomes of the sums: 16-bit outputs with a bias; floats of 24 bits, which another launch adds up; SiLU(gate) x up as fp32 rows,
// gate = weight rows [0, N / 2).
//
// kEpiFloat24: an fp32 number's upper 16 bits in out [rows, N], the next 8 in low [rows, N].  Every value is off by 2^-16 of itself, a 32nd of
// an fp16 output's rounding, whatever the channels beside it are scaled by, for three quarters of the bytes that both launches wait for.
// (The whole layer of 4096 tokens, 128 experts, top 8, 2048 / 768, us: 383; fp32 numbers 400; 16-bit integers with one scale for a row's 32 to 128
// columns 346, but beside a channel of 1000 times their scale the others had six bits left.)
enum : int { kEpiOut = 0, kEpiFloat24 = 1, kEpiAct = 2 };

constexpr int kInt8Step = 128;                        // bytes of a row per step

// LDS of a tile: the rings
constexpr size_t int8_gemm_lds(int BM, int BN, int KG, int SA, int SB) { return (size_t)KG * (SA * BM + SB * BN) * kInt8Step; }

template <class Act, int BM, int BN, int WM, int WN, int KG, int SA, int SB, int EPI, bool GROUPED>
__global__ __launch_bounds__(64 * WM * WN * KG) void int8_gemm_kernel(const Int8GemmArgs p) {
  using Elem = typename Act::elem;
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  // 1 KiB loads of a wavefront per step.  Grouped: half of the wavefronts load A, half B.  Loads are waited for in the order of their requests,
  // so a wavefront that loads both can have hardly more of one under way than of the other; an expert's weights come from HBM for few
  // rows and take the deeper ring (128 experts, 4096 tokens, top 8, 2048 / 768: 193 + 166 us with both, 160 + 141 with these roles; dense
  // products, whose operands are in L2 half of the time: 0 to 3 % slower).
  constexpr bool ROLES = GROUPED && NW % 2 == 0;
  constexpr int NL = ROLES ? NW / 2 : NW, LA = BM / (8 * NL), LB = BN / (8 * NL);
  constexpr int HN = EPI == kEpiAct ? TN / 2 : TN;    // MFMA tiles of gate (or all) columns
  // columns in a row per lane: a store instruction writes 64 bytes of 16 rows then (with 4 tiles in a row, half sectors: 85 us for 302 MB)
  constexpr int GJ = EPI != kEpiAct && HN % 2 == 0 ? 2 : 1;
  constexpr int A_PART = BM * kInt8Step, B_PART = BN * kInt8Step, B_RING = SA * KG * A_PART;   // the ring of A, that of B
  static_assert(SA >= 2 && SB >= 2 && (ROLES || SA == SB || SA == SB + 1), "rings");
  static_assert((!GROUPED || TM <= 5) && TM * 16 * WM == BM && TN * 16 * WN == BN && LA * 8 * NL == BM && LB * 8 * NL == BN, "tile");
  static_assert(HN * (EPI == kEpiAct ? 2 : 1) == TN && HN % GJ == 0, "columns");
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave / NW, wg = wave % NW, wm = wg % WM, wn = wg / WM;        // part of the step, place in the tile
  const int K = p.K, N = p.N;
  constexpr int BNO = EPI == kEpiAct ? BN / 2 : BN;   // output columns of a tile
  const int NO = EPI == kEpiAct ? N / 2 : N;

  int tm, tn, m0, rows;
  const int8_t* w = p.w;
  const float* ws = p.w_scale;
  // workgroups go to the 8 XCDs in turn
  const int xcd = blockIdx.x & 7, nth = blockIdx.x >> 3;
  if constexpr (GROUPED) {
    tm = nth / p.tiles_n * 8 + xcd;                    // every 8th row tile to an XCD: its column tiles share its rows
    tn = nth % p.tiles_n;
    if (tm >= p.tiles_m || tm >= p.g_tile[4 * p.tiles_m]) return;
    const int e = p.g_tile[4 * tm];
    m0 = p.g_tile[4 * tm + 1];
    rows = p.g_tile[4 * tm + 2];
    w = e == p.E ? p.shared_w : p.w + (size_t)e * N * K;
    ws = e == p.E ? p.shared_scale : p.w_scale + (size_t)e * N;
  } else {
    // a run of tiles each, in bands of 8 row tiles that share the weights' tile
    const int total = p.tiles_m * p.tiles_n, per = (total + 7) / 8, id = xcd * per + nth;
    if (nth >= per || id >= total) return;
    const int band = id / (8 * p.tiles_n), in = id - band * 8 * p.tiles_n;
    const int high = p.tiles_m - band * 8 < 8 ? p.tiles_m - band * 8 : 8;
    tn = in / high;
    tm = band * 8 + in - tn * high;
    m0 = tm * BM;
    rows = p.M - m0 < BM ? p.M - m0 : BM;
  }
  const int n0 = tn * BNO;

  // where this lane's 16 bytes of each load come from
  const int wl = wg % NL;
  const bool loads_a = !ROLES || wg < NL, loads_b = !ROLES || wg >= NL;
  constexpr int FIRST_B = ROLES ? 0 : LA, LOADS = ROLES ? (LA > LB ? LA : LB) : LA + LB;
  uint32_t from[LOADS];
  int chunk[LOADS];
  if (loads_a) {
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const int r = (wl * LA + i) * 8 + (lane >> 3);
      chunk[i] = wk * kInt8Step + ((lane & 7) ^ (r & 7)) * 16;
      uint32_t row = (uint32_t)r;
      if constexpr (GROUPED) {
        const int at = m0 + (r < rows ? r : 0);
        row = (uint32_t)(p.g_row ? p.g_row[at] : at);
      }
      from[i] = r < rows ? row * (uint32_t)K + chunk[i] : kOOB;
    }
  }
  if (loads_b) {
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const int r = (wl * LB + i) * 8 + (lane >> 3);
      chunk[FIRST_B + i] = wk * kInt8Step + ((lane & 7) ^ ((r & 3) | ((r / (4 * GJ)) & 1) << 2)) * 16;
      int row = r;
      bool in = n0 + r < N;
      if constexpr (EPI == kEpiAct) {
        const int q = r % (TN * 16), col = r / (TN * 16) * (TN * 8) + q % (TN * 8);
        in = n0 + col < NO;
        row = q < TN * 8 ? col : NO + col;
      }
      from[FIRST_B + i] = in ? (uint32_t)row * (uint32_t)K + chunk[FIRST_B + i] : kOOB;
    }
  }
  const int8_t* a0 = GROUPED ? p.a : p.a + (size_t)m0 * K;
  const unsigned long long a_bytes = (unsigned long long)(GROUPED ? p.M : rows) * K, w_bytes = (unsigned long long)(N - n0) * K;
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(a0, (uint32_t)(a_bytes < 0x7FFFFFFFull ? a_bytes : 0x7FFFFFFFull));
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(w + (size_t)n0 * K, (uint32_t)(w_bytes < 0x7FFFFFFFull ? w_bytes : 0x7FFFFFFFull));

  constexpr int STEP = KG * kInt8Step;
  const int steps = (K + STEP - 1) / STEP;
  auto request = [&](auto is_a, int s, int slot) __attribute__((always_inline)) {
    constexpr bool A = decltype(is_a)::value;
    constexpr int COUNT = A ? LA : LB, FIRST = A ? 0 : FIRST_B;
    if (!(A ? loads_a : loads_b)) return;
    const int to = A ? (slot * KG + wk) * A_PART + wl * LA * 1024 : B_RING + (slot * KG + wk) * B_PART + wl * LB * 1024;
    const int k0 = s * STEP;
    const bool whole = k0 + STEP <= K;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const uint32_t f = whole || k0 + chunk[FIRST + i] < K ? from[FIRST + i] : kOOB;   // past the row's end: zeros
      __builtin_amdgcn_raw_ptr_buffer_load_lds(A ? ra : rb, (lds_ptr)(smem + to + i * 1024), 16, f, k0, 0, 0);
    }
  };
  constexpr std::true_type a_tag{};
  constexpr std::false_type b_tag{};

  i32x4 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int t = 0; t < TM; ++t) acc[j][t] = i32x4{0, 0, 0, 0};

  const int r16 = lane & 15, g = lane >> 4;
  int place[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) place[h] = ((h * 4 + g) ^ (r16 & 7)) * 16;
  const int a_at = (wm * 16 + r16) * kInt8Step;       // row tile t of the wavefront: row tile t WM + wm of the workgroup
  const int b_at = (wn * TN * 16 + (r16 >> 2) * 4 * GJ + (r16 & 3)) * kInt8Step;

  i32x4 fa[2][TM], fb[2][TN];
  auto read = [&](auto live, int h, int slot_a, int slot_b) __attribute__((always_inline)) {
    const unsigned char* a = smem + (slot_a * KG + wk) * A_PART + a_at + place[h];
    const unsigned char* b = smem + B_RING + (slot_b * KG + wk) * B_PART + b_at + place[h];
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[h][j] = *reinterpret_cast<const i32x4*>(b + (j / GJ * GJ * 16 + j % GJ * 4) * kInt8Step);
#pragma unroll
    for (int t = 0; t < decltype(live)::value; ++t) fa[h][t] = *reinterpret_cast<const i32x4*>(a + t * WM * 16 * kInt8Step);
  };
  auto multiply = [&](auto live, int h) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int t = 0; t < decltype(live)::value; ++t) acc[j][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[h][j], fa[h][t], acc[j][t], 0, 0, 0);
  };

  // One barrier per step, in its middle: the operands of a half step are read while the half before it is multiplied.  Behind the barrier
  // every wavefront has read all of step s, whose places take B of step s + SB and A of step s + SA, and step s + 1 has landed.  Past
  // the end nothing but zeros is fetched, so that the loads can be counted.
  auto wait_step = [&](auto older) __attribute__((always_inline)) {            // steps behind the one that is needed: requested, not waited for
    constexpr int O = decltype(older)::value;
    if constexpr (!ROLES) wait_loads<(SB - 2 + O) * (LA + LB) + (SA > SB ? LA : 0)>();           // B's goes out before A's
    else if (loads_a) wait_loads<(SA - 2 + O) * LA>();
    else wait_loads<(SB - 2 + O) * LB>();
  };
  asm volatile("" ::: "memory");
#pragma unroll
  for (int s = SB > SA ? SA - SB : 0; s < SA; ++s) {
    if (s >= SA - SB) request(b_tag, s - (SA - SB), s - (SA - SB));
    if (s >= 0) request(a_tag, s, s);
  }
  wait_step(std::integral_constant<int, 1>{});
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  auto run = [&](auto live) __attribute__((always_inline)) {
    read(live, 0, 0, 0);
    int slot_a = 0, slot_b = 0;
    for (int s = 0; s < steps; ++s) {
      read(live, 1, slot_a, slot_b);
      multiply(live, 0);
      wait_step(std::integral_constant<int, 0>{});
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const int next_a = slot_a + 1 < SA ? slot_a + 1 : 0, next_b = slot_b + 1 < SB ? slot_b + 1 : 0;
      read(live, 0, next_a, next_b);
      request(b_tag, s + SB, slot_b);
      request(a_tag, s + SA, slot_a);
      multiply(live, 1);
      slot_a = next_a;
      slot_b = next_b;
    }
  };
  if constexpr (GROUPED && TM > 1) {                   // an expert's last tile is hardly ever full: only row tiles with rows are multiplied
    const int live = ((rows + 15) / 16 - wm + WM - 1) / WM;
    if (live >= TM) run(std::integral_constant<int, TM>{});
    else if (TM > 4 && live == 4) run(std::integral_constant<int, (TM > 4 ? 4 : 1)>{});
    else if (TM > 3 && live == 3) run(std::integral_constant<int, (TM > 3 ? 3 : 1)>{});
    else if (TM > 2 && live == 2) run(std::integral_constant<int, (TM > 2 ? 2 : 1)>{});
    else run(std::integral_constant<int, 1>{});
  } else {
    run(std::integral_constant<int, TM>{});
  }
  wait_loads<0>();                                     // nothing is on its way to LDS when the workgroup ends

  if constexpr (KG > 1) {                              // the parts' sums meet in LDS
    lds_barrier();
    i32x4* sums = reinterpret_cast<i32x4*>(smem) + wg * (TN * TM) * 64 + lane;
    constexpr int SUMS = NW * TN * TM * 64;
    static_assert((KG - 1) * SUMS * 16 <= KG * (SA * A_PART + SB * B_PART), "the ring holds the sums");
    if (wk > 0) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int t = 0; t < TM; ++t) sums[(wk - 1) * SUMS + (j * TM + t) * 64] = acc[j][t];
    }
    lds_barrier();
    if (wk > 0) return;
#pragma unroll
    for (int q = 0; q < KG - 1; ++q)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[j][t] += sums[q * SUMS + (j * TM + t) * 64];
  }

  // lane: row m of the tile, columns [c, c + 4 GJ) per group of GJ tiles.  The factors of all of its columns are requested together, four at
  // a time (in the tile at N's end one by one, indices held inside the row).
  typedef __attribute__((ext_vector_type(4), aligned(4))) float Floats;
  typedef __attribute__((ext_vector_type(4), aligned(2))) Elem Elems;
  f32v4 cs[EPI == kEpiAct ? 2 : 1][HN];
  float add[EPI == kEpiOut ? HN : 1][4];
  auto column = [&](int q) __attribute__((always_inline)) { return n0 + wn * HN * 16 + q / GJ * GJ * 16 + g * 4 * GJ + q % GJ * 4; };
  if (n0 + BNO <= NO) {
#pragma unroll
    for (int q = 0; q < HN; ++q) {
      cs[0][q] = *reinterpret_cast<const Floats*>(ws + column(q));
      if constexpr (EPI == kEpiAct) cs[1][q] = *reinterpret_cast<const Floats*>(ws + NO + column(q));
    }
  } else {
#pragma unroll
    for (int q = 0; q < HN; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = column(q) + i < NO ? column(q) + i : NO - 1;
        cs[0][q][i] = ws[at];
        if constexpr (EPI == kEpiAct) cs[1][q][i] = ws[NO + at];
      }
  }
  if constexpr (EPI == kEpiFloat24) {                  // a NaN of all ones would be rounded to a number
#pragma unroll
    for (int q = 0; q < HN; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) cs[0][q][i] = cs[0][q][i] == cs[0][q][i] ? cs[0][q][i] : __builtin_nanf("");
  }
  if constexpr (EPI == kEpiOut) {
#pragma unroll
    for (int q = 0; q < HN; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) add[q][i] = 0.0f;
    if (p.bias) {
      const Elem* bias = (const Elem*)p.bias;
      Elems raw[HN];
      if (n0 + BNO <= NO) {
#pragma unroll
        for (int q = 0; q < HN; ++q) raw[q] = *reinterpret_cast<const Elems*>(bias + column(q));
      } else {
#pragma unroll
        for (int q = 0; q < HN; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) raw[q][i] = bias[column(q) + i < NO ? column(q) + i : NO - 1];
      }
#pragma unroll
      for (int q = 0; q < HN; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) add[q][i] = Act::to_f32(raw[q][i]);
    }
  }
  float as[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const int r = (t * WM + wm) * 16 + r16, at = m0 + (r < rows ? r : 0);
    as[t] = p.a_scale[GROUPED && p.g_row ? p.g_row[at] : at];
  }
  constexpr int W = GJ;                                // MFMA tiles per store
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const int r = (t * WM + wm) * 16 + r16;
    const size_t row = (size_t)(m0 + r) * NO;
    if (r < rows) {
#pragma unroll
      for (int q = 0; q < HN; q += W) {
        const int n = column(q);
        if (n >= NO) continue;
        float v[W * 4];
#pragma unroll
        for (int i = 0; i < W * 4; ++i) {              // the sum times a large row scale may pass fp32: the factors first
          const int u = q + i / 4;
          v[i] = (float)acc[u][t][i & 3] * (as[t] * cs[0][u][i & 3]);
          if constexpr (EPI == kEpiAct) v[i] = silu_mul(v[i], (float)acc[HN + u][t][i & 3] * (as[t] * cs[1][u][i & 3]));
          if constexpr (EPI == kEpiOut) v[i] += add[u][i & 3];
        }
        if constexpr (EPI == kEpiOut) {
          // one store wherever a row starts: global memory takes any address (201 x 2048 x 12290 through LDS to words 14.5 us, like this 12.1)
          typedef __attribute__((ext_vector_type(W * 4), aligned(sizeof(Elem)))) Elem VW;
          Elem* o = (Elem*)p.out + row + n;
          VW x;
#pragma unroll
          for (int i = 0; i < W * 4; ++i) x[i] = Act::from_f32(v[i]);
          if (n + W * 4 <= N) {
            *reinterpret_cast<VW*>(o) = x;
          } else {
#pragma unroll
            for (int i = 0; i < W * 4; ++i)
              if (n + i < N) o[i] = x[i];
          }
        } else if constexpr (EPI == kEpiFloat24) {     // N a multiple of 16
          typedef __attribute__((ext_vector_type(W * 2))) uint32_t High;
          typedef __attribute__((ext_vector_type(W))) uint32_t Low;
          uint32_t b[W * 4];
#pragma unroll
          for (int i = 0; i < W * 4; ++i) b[i] = __builtin_bit_cast(uint32_t, v[i]) + 0x80u;
          High x;
          Low y;
#pragma unroll
          for (int i = 0; i < W * 2; ++i) x[i] = __builtin_amdgcn_perm(b[i * 2 + 1], b[i * 2], 0x07060302u);
#pragma unroll
          for (int i = 0; i < W; ++i)                  // the second bytes of four
            y[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[i * 4 + 3], b[i * 4 + 2], 0x0C0C0501u), __builtin_amdgcn_perm(b[i * 4 + 1], b[i * 4], 0x0C0C0501u), 0x05040100u);
          *reinterpret_cast<High*>((uint16_t*)p.out + row + n) = x;
          *reinterpret_cast<Low*>(p.low + row + n) = y;
        } else {
          *reinterpret_cast<f32v4*>((float*)p.out + row + n) = f32v4{v[0], v[1], v[2], v[3]};
        }
      }
    }
  }
}

}  // namespace qlin
