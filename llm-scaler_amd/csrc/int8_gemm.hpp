// Product of 8-bit codes on the matrix cores: out[m][n] = (sum_k a[m][k] w[n][k]) a_scale[m] w_scale[n].
//
// A workgroup owns a BM x BN tile.  Both operands go to LDS straight from memory (128-byte pieces of a row per step, no registers
// and no vector instructions in between) into a ring of STAGES buffers; a wavefront multiplies (16 TM) x (16 TN) of the tile with
// v_mfma_i32_16x16x64_i8.  16-byte chunk c of tile row r lies at place c ^ f(r) of its 128 bytes, so that the eight lanes that
// read at a time find eight different places.  The weights are the first operand: a lane ends with consecutive output columns of
// one row, 4 per MFMA tile, and the weight rows of GJ tiles are interleaved so that these are 4 GJ in a row.
#pragma once
#include "int8_common.hpp"

namespace qlin {

struct Int8GemmArgs {
  const int8_t* a;            // [rows, K]
  const float* a_scale;       // [rows]
  const int8_t* w;            // [N, K]; grouped [E, N, K]
  const float* w_scale;       // [N]; grouped [E, N]
  const void* bias;           // [N] in the output's type, or null
  void* out;
  int M, N, K;                // M: rows of a
  int wide_out;               // four outputs per store: N and out allow it
  int tiles_m, tiles_n;
  // Grouped: tile i covers the rows [g_tile[4 i + 1], + g_tile[4 i + 2]) of the expert-sorted order and multiplies them with expert
  // g_tile[4 i]; row r of that order is row g_row[r] of a (null: r).  Expert E is the shared one.  g_tile[4 tiles_m]: tiles in use.
  const int32_t* g_tile;
  const int32_t* g_row;
  const int8_t* shared_w;
  const float* shared_scale;
  int E;
};

// What becomes of the sums: 16-bit outputs with a bias; fp32 rows; SiLU(gate) x up as fp32 rows, gate = weight rows [0, N / 2).
enum : int { kEpiOut = 0, kEpiF32 = 1, kEpiAct = 2 };

constexpr int kInt8Step = 128;                        // bytes of a row per step

template <class Act, int BM, int BN, int WM, int WN, int STAGES, int EPI, bool GROUPED>
__global__ __launch_bounds__(64 * WM * WN) void int8_gemm_kernel(const Int8GemmArgs p) {
  using Elem = typename Act::elem;
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW;   // 1 KiB loads of a wavefront per step
  constexpr int HN = EPI == kEpiAct ? TN / 2 : TN;    // MFMA tiles of gate (or all) columns
  constexpr int GJ = HN < 4 ? HN : 4;
  constexpr int STAGE = (BM + BN) * kInt8Step;
  static_assert(LA * 8 * NW == BM && LB * 8 * NW == BN && TM * 16 * WM == BM && TN * 16 * WN == BN, "tile");
  static_assert(HN * (EPI == kEpiAct ? 2 : 1) == TN && HN % GJ == 0, "columns");
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int K = p.K, N = p.N;
  constexpr int BNO = EPI == kEpiAct ? BN / 2 : BN;   // output columns of a tile
  const int NO = EPI == kEpiAct ? N / 2 : N;

  int tm, tn, m0, rows;
  const int8_t* w = p.w;
  const float* ws = p.w_scale;
  if constexpr (GROUPED) {
    tm = blockIdx.x / p.tiles_n;
    tn = blockIdx.x - tm * p.tiles_n;
    if (tm >= p.g_tile[4 * p.tiles_m]) return;
    const int e = p.g_tile[4 * tm];
    m0 = p.g_tile[4 * tm + 1];
    rows = p.g_tile[4 * tm + 2];
    w = e == p.E ? p.shared_w : p.w + (size_t)e * N * K;
    ws = e == p.E ? p.shared_scale : p.w_scale + (size_t)e * N;
  } else {
    // workgroups go to the 8 XCDs in turn: each takes a run of tiles, in bands of 8 row tiles that share the weights' tile
    const int total = p.tiles_m * p.tiles_n, per = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= total || (int)(blockIdx.x >> 3) >= per) return;
    const int band = id / (8 * p.tiles_n), in = id - band * 8 * p.tiles_n;
    const int high = p.tiles_m - band * 8 < 8 ? p.tiles_m - band * 8 : 8;
    tn = in / high;
    tm = band * 8 + in - tn * high;
    m0 = tm * BM;
    rows = p.M - m0 < BM ? p.M - m0 : BM;
  }
  const int n0 = tn * BNO;

  // where this lane's 16 bytes of each load come from
  uint32_t from[LA + LB];
  int chunk[LA + LB];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int r = (wave * LA + i) * 8 + (lane >> 3);
    chunk[i] = ((lane & 7) ^ (r & 7)) * 16;
    uint32_t row = (uint32_t)r;
    if constexpr (GROUPED) {
      const int at = m0 + (r < rows ? r : 0);
      row = (uint32_t)(p.g_row ? p.g_row[at] : at);
    }
    from[i] = r < rows ? row * (uint32_t)K + chunk[i] : kOOB;
  }
#pragma unroll
  for (int i = 0; i < LB; ++i) {
    const int r = (wave * LB + i) * 8 + (lane >> 3);
    chunk[LA + i] = ((lane & 7) ^ ((r & 3) | ((r / (4 * GJ)) & 1) << 2)) * 16;
    int row = r;
    bool in = n0 + r < N;
    if constexpr (EPI == kEpiAct) {
      const int q = r % (TN * 16), col = r / (TN * 16) * (TN * 8) + q % (TN * 8);
      in = n0 + col < NO;
      row = q < TN * 8 ? col : NO + col;
    }
    from[LA + i] = in ? (uint32_t)row * (uint32_t)K + chunk[LA + i] : kOOB;
  }
  const int8_t* a0 = GROUPED ? p.a : p.a + (size_t)m0 * K;
  const unsigned long long a_bytes = (unsigned long long)(GROUPED ? p.M : rows) * K, w_bytes = (unsigned long long)(N - n0) * K;
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(a0, (uint32_t)(a_bytes < 0x7FFFFFFFull ? a_bytes : 0x7FFFFFFFull));
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(w + (size_t)n0 * K, (uint32_t)(w_bytes < 0x7FFFFFFFull ? w_bytes : 0x7FFFFFFFull));

  const int steps = (K + kInt8Step - 1) / kInt8Step;
  auto request = [&](int s) __attribute__((always_inline)) {
    unsigned char* to = smem + (s % STAGES) * STAGE;
    const int k0 = s * kInt8Step;
    const bool whole = k0 + kInt8Step <= K;
#pragma unroll
    for (int i = 0; i < LA + LB; ++i) {
      const int at = i < LA ? wave * LA + i : BM / 8 + wave * LB + (i - LA);
      const uint32_t f = whole || k0 + chunk[i] < K ? from[i] : kOOB;   // past the row's end: zeros
      __builtin_amdgcn_raw_ptr_buffer_load_lds(i < LA ? ra : rb, (lds_ptr)(to + at * 1024), 16, f, k0, 0, 0);
    }
  };

  i32x4 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int t = 0; t < TM; ++t) acc[j][t] = i32x4{0, 0, 0, 0};

  const int r16 = lane & 15, g = lane >> 4;
  int place[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) place[h] = ((h * 4 + g) ^ (r16 & 7)) * 16;
  const int a_at = (wm * TM * 16 + r16) * kInt8Step;
  const int b_at = (BM + wn * TN * 16 + (r16 >> 2) * 4 * GJ + (r16 & 3)) * kInt8Step;

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) request(s);
  for (int s = 0; s < steps; ++s) {
    wait_loads<(STAGES - 2) * (LA + LB)>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    request(s + STAGES - 1);                           // into the buffer that every wavefront has left; past the end it fetches zeros
    const unsigned char* from_lds = smem + (s % STAGES) * STAGE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x4 fa[TM], fb[TN];
#pragma unroll
      for (int t = 0; t < TM; ++t) fa[t] = *reinterpret_cast<const i32x4*>(from_lds + a_at + t * 16 * kInt8Step + place[h]);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = j / GJ * GJ * 16 + j % GJ * 4;
        fb[j] = *reinterpret_cast<const i32x4*>(from_lds + b_at + row * kInt8Step + place[h]);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[j][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j], fa[t], acc[j][t], 0, 0, 0);
    }
  }
  wait_loads<0>();                                     // nothing is on its way to LDS when the workgroup ends

  // lane: row m of the tile, columns [c, c + 4 GJ) per group of GJ tiles
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const int r = wm * TM * 16 + t * 16 + r16;
    if (r >= rows) continue;
    size_t row = (size_t)(m0 + r);
    const float as = p.a_scale[GROUPED && p.g_row ? (size_t)p.g_row[m0 + r] : row];
#pragma unroll
    for (int jb = 0; jb < HN / GJ; ++jb) {
      const int c = n0 + wn * HN * 16 + jb * GJ * 16 + g * 4 * GJ;
#pragma unroll
      for (int j = 0; j < GJ; ++j) {
        const int n = c + j * 4;
        if (n >= NO) continue;
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = n + i < NO ? n + i : NO - 1;
          v[i] = (float)acc[jb * GJ + j][t][i] * (as * ws[at]);   // the sum times a large row scale may pass fp32
          if constexpr (EPI == kEpiAct) v[i] = silu_mul(v[i], (float)acc[HN + jb * GJ + j][t][i] * (as * ws[NO + at]));
          if constexpr (EPI == kEpiOut)
            if (p.bias) v[i] += Act::to_f32(((const Elem*)p.bias)[at]);
        }
        if constexpr (EPI == kEpiOut) {
          Elem* o = (Elem*)p.out + row * NO + n;
          if (p.wide_out) {
            typedef __attribute__((ext_vector_type(4))) Elem v4;
            *reinterpret_cast<v4*>(o) = v4{Act::from_f32(v[0]), Act::from_f32(v[1]), Act::from_f32(v[2]), Act::from_f32(v[3])};
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n + i < NO) o[i] = Act::from_f32(v[i]);
          }
        } else {
          *reinterpret_cast<f32v4*>((float*)p.out + row * NO + n) = f32v4{v[0], v[1], v[2], v[3]};   // NO % 4 == 0
        }
      }
    }
  }
}

}  // namespace qlin
