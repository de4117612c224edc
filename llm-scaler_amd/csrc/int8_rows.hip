// The product of few rows (M <= 16) with 8-bit weights: out[m][n] = (sum_k q[m][k] w[n][k]) s[m] w_scale[n].  Bound: HBM, the weights once.
//
// A workgroup of 16 wavefronts owns 16 columns per slot; the KS = 16 / slots wavefronts of a slot each take a part of K, so that all of a
// CU's loads are in flight at once however few columns there are.  Weights go to LDS straight from memory, 128 bytes of 16 rows
// (2 KiB) at a time into a ring of kUnits that is the wavefront's own: whole lines for the loads, and the operands of
// v_mfma_i32_16x16x64_i8 read back without a barrier.  16-byte chunk c of row r lies at place c ^ (r & 7) of its 128 bytes.  The
// codes lie in LDS in operand order.  The parts of K meet in LDS as integers.
//
// Rows that are not codes yet (16-bit activations, residual + norm, SiLU x up) are quantised by every workgroup for itself while its
// first weights are on their way: the rows are few KiB and come from L2, a launch in front would be a round trip.
//
// The same product with the operands loaded into registers (consecutive lanes read consecutive rows, a tag look-up each) took
// 15.8 us for 1 x 4096 x 14336; like this 10.9 (5.4 TB/s), 8 rows 11.7, 16 rows of K = 2048 7.8, 1 x 4096 x 4096 5.1.  Rings of 3 and 4
// units: within 3 %.
#include "int8_rows.hpp"

namespace qlin {

constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr int kPieces = 2;                            // pieces of 8 values per thread that a workgroup quantises
constexpr int kChunks = 4;                            // chunks of 16 codes per thread that it takes as they are
constexpr int kUnit = 2048, kUnits = 2;               // bytes of a ring's unit: 16 rows x 128; units of a ring

template <class Act, int FROM>
__global__ __launch_bounds__(kThreads) void int8_rows_kernel(const Int8RowsArgs p) {
  using Elem = typename Act::elem;
  using V8 = typename Act::v8;
  constexpr bool kCodes = FROM == kFromCodes;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];       // rings, codes
  __shared__ float row_s[16];
  __shared__ float part_sum[kWaves * kPieces];
  __shared__ uint32_t part_top[kWaves * kPieces];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int M = p.M, N = p.N, K = p.K, KS = 1 << p.ks_log2, slots = kWaves >> p.ks_log2;
  const int slot = wave >> p.ks_log2, part = wave & (KS - 1);
  const int blocks = (K + 127) / 128, per = (blocks + KS - 1) >> p.ks_log2;
  const int b0 = part * per, b1 = b0 + per < blocks ? b0 + per : blocks;
  const int n0 = (blockIdx.x * slots + slot) * 16, cols = n0 < N ? (N - n0 < 16 ? N - n0 : 16) : 0;
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(cols ? p.w + (size_t)n0 * K : p.w, (uint32_t)cols * (uint32_t)K);
  unsigned char* const ring = smem + wave * (kUnits * kUnit);
  unsigned char* const codes = smem + kWaves * kUnits * kUnit;                  // [block of 64][row][64]

  // rows to be quantised: pieces of 8 values, whole wavefronts per row
  static_assert(kNormPart == 64 * 8, "a part of the norm's sum is a piece");
  const int waves_per_row = (K / 8 + 63) / 64, pieces = waves_per_row * 64 * M;
  auto row_of = [&](int i) __attribute__((always_inline)) { return (i * kWaves + wave) / waves_per_row; };
  auto k_of = [&](int i, int row) __attribute__((always_inline)) { return ((i * kWaves + wave - row * waves_per_row) * 64 + lane) * 8; };
  // all of them requested before the weights, whose loads they must not wait for: addresses held inside the rows
  constexpr int kRaw = FROM == kFromNorm ? 3 : FROM == kFromSilu ? 2 : 1;
  V8 raw[kCodes ? 1 : kPieces][kRaw];
  if constexpr (!kCodes) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i * kThreads >= pieces) break;
      const int row = row_of(i), at = row < M ? row : M - 1, k = k_of(i, row), in = k < K ? k : 0;
      const Elem* src = (const Elem*)p.x + (size_t)at * (FROM == kFromSilu ? 2 * K : K) + in;
      raw[i][0] = *reinterpret_cast<const V8*>(src);
      if constexpr (FROM == kFromSilu) raw[i][1] = *reinterpret_cast<const V8*>(src + K);
      if constexpr (FROM == kFromNorm) {
        raw[i][1] = *reinterpret_cast<const V8*>((const Elem*)p.residual + (size_t)at * K + in);
        raw[i][2] = *reinterpret_cast<const V8*>((const Elem*)p.norm_weight + in);
      }
    }
  }
  const int chunks = blocks * 8;                       // of 16 codes, a row's behind each other, to the end of the last unit
  u32x4 given[kCodes ? kChunks : 1];
  if constexpr (kCodes) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      if (i * kThreads >= chunks * M) break;
      const int at = i * kThreads + tid, row = at / chunks, c = at - row * chunks;
      given[i] = *reinterpret_cast<const u32x4*>((const int8_t*)p.x + (size_t)(row < M ? row : M - 1) * K + (c * 16 < K ? c * 16 : 0));
    }
  }

  // every thread stores outputs of one column
  const int width = slots * 16, n = blockIdx.x * width + (tid & (width - 1)), n_in = n < N ? n : N - 1;
  const float w_scale = p.w_scale[n_in];
  const Elem bias = p.bias ? ((const Elem*)p.bias)[n_in] : *(const Elem*)p.w_scale;      // some address, so that nothing branches here

  // Unit b of the part into its place of the ring; past the part nothing is fetched (out of range: zeros).  What stands behind a row's
  // end in the last unit meets codes that are zero.
  const uint32_t from0 = (uint32_t)(lane >> 3) * (uint32_t)K + ((lane & 7) ^ (lane >> 3)) * 16, from1 = from0 + 8u * (uint32_t)K;
  auto request = [&](int u, int b) __attribute__((always_inline)) {
    const uint32_t off = b < b1 ? (uint32_t)b * 128u : kOOB;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr)(ring + u * kUnit), 16, from0 + off, 0, 0, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr)(ring + u * kUnit + 1024), 16, from1 + off, 0, 0, 2);
  };
  asm volatile("" ::: "memory");
#pragma unroll
  for (int u = 0; u < kUnits; ++u) request(u, b0 + u);

  if constexpr (!kCodes) {
    float v[kPieces][8];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i * kThreads >= pieces) break;
      const int row = row_of(i);
      const bool in = row < M && k_of(i, row) < K;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = Act::to_f32(raw[i][0][j]);
        if constexpr (FROM == kFromSilu) v[i][j] = silu_mul(a, Act::to_f32(raw[i][1][j]));
        else if constexpr (FROM == kFromNorm) v[i][j] = a + Act::to_f32(raw[i][1][j]);
        else v[i][j] = a;
        v[i][j] = in ? v[i][j] : 0.0f;
      }
    }
    if constexpr (FROM == kFromNorm) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        if (i * kThreads >= pieces) break;
        const float ss = norm_part(v[i]);
        if (lane == 0) part_sum[i * kWaves + wave] = ss;
      }
      lds_barrier();
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int row = row_of(i), k = k_of(i, row);
        if (i * kThreads >= pieces || row >= M) break;
        float ss = 0.0f;
        for (int q = 0; q < waves_per_row; ++q) ss += part_sum[row * waves_per_row + q];
        const float r = rsqrtf(ss / (float)K + p.eps);
        if (k < K) {
#pragma unroll
          for (int j = 0; j < 8; ++j) raw[i][0][j] = Act::from_f32(v[i][j]);     // the new residual, stored at the end
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * r * Act::to_f32(raw[i][2][j]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i * kThreads >= pieces) break;
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = umax32(top, abs_bits(v[i][j]));
      top = wave_max_u32(top);
      if (lane == 0) part_top[i * kWaves + wave] = top;
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int row = row_of(i), k = k_of(i, row);
      if (i * kThreads >= pieces || row >= M) break;
      uint32_t top = 0;
      for (int q = 0; q < waves_per_row; ++q) top = umax32(top, part_top[row * waves_per_row + q]);
      const RowScale s = row_scale(top);
      if (k == 0) row_s[row] = s.scale;
      if (k < blocks * 128) {                          // past K: zeros, to the end of the last unit
        uint32_t c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = code_of<FROM == kFromAct>(v[i][j], s.inv);
        *reinterpret_cast<u32x2*>(codes + ((k >> 6) * M + row) * 64 + (k & 63)) =
            u32x2{pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7])};
      }
    }
  }
  if constexpr (kCodes) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int at = i * kThreads + tid, row = at / chunks, c = at - row * chunks;
      if (at < chunks * M)                             // past K zeros
        *reinterpret_cast<u32x4*>(codes + ((c >> 2) * M + row) * 64 + (c & 3) * 16) = c * 16 < K ? given[i] : u32x4{0, 0, 0, 0};
    }
  }
  lds_barrier();                                       // the codes are there

  i32x4 acc[2] = {i32x4{0, 0, 0, 0}, i32x4{0, 0, 0, 0}};
  const unsigned char* x_at = codes + (r16 < M ? r16 : M - 1) * 64 + g * 16;   // a column of the product past M is not stored
  int w_at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) w_at[h] = r16 * 128 + (((h * 4 + g) ^ (r16 & 7)) * 16);
  for (int b = b0; b < b1; b += kUnits) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int at = b + u < blocks ? b + u : blocks - 1;        // the weights beyond are zeros
      wait_loads<2 * (kUnits - 1)>();
      i32x4 w[2], x[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        w[h] = *reinterpret_cast<const i32x4*>(ring + u * kUnit + w_at[h]);
        x[h] = *reinterpret_cast<const i32x4*>(x_at + (at * 2 + h) * M * 64);
      }
      wait_loads<63>();                                // read before the unit is asked for again
      request(u, b + kUnits + u);
#pragma unroll
      for (int h = 0; h < 2; ++h) acc[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[h], x[h], acc[h], 0, 0, 0);
    }
  }

  // the parts' sums, then one thread per output
  wait_loads<0>();
  __syncthreads();
  int32_t* sums = reinterpret_cast<int32_t*>(smem);
  *reinterpret_cast<i32x4*>(sums + wave * 256 + lane * 4) = acc[0] + acc[1];
  __syncthreads();
  const int c = tid & (width - 1), step = kThreads / width;
  if constexpr (FROM == kFromNorm) {
    if (blockIdx.x == 0) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int row = row_of(i), k = k_of(i, row);
        if (i * kThreads < pieces && row < M && k < K) *reinterpret_cast<V8*>((Elem*)p.residual_out + (size_t)row * K + k) = raw[i][0];
      }
    }
  }
  if (n >= N) return;
  for (int m = tid / width; m < M; m += step) {
    const int32_t* from = sums + ((c >> 4) << p.ks_log2) * 256 + (((c & 15) >> 2) * 16 + m) * 4 + (c & 3);
    int sum = 0;
    for (int q = 0; q < KS; ++q) sum += from[q * 256];
    const float o = (float)sum * ((kCodes ? p.x_scale[m] : row_s[m]) * w_scale) + (p.bias ? Act::to_f32(bias) : 0.0f);
    ((Elem*)p.out)[(size_t)m * N + n] = Act::from_f32(o);
  }
}

static long long codes_bytes(int M, int K) { return (long long)M * ((K + 127) / 128) * 128; }

// Every workgroup repeats the work on the rows, a launch in front does it once.  This / a launch of its own, us, bf16: 1 x 4096 x 4096 5.7 / 7.2,
// 4 x 4096 x 4096 7.0 / 7.9, 8 x 4096 x 4096 9.1 / 8.1, 16 x 2048 x 14336 11.4 / 9.7; SiLU 1 x 14336 x 4096 13.6 / 13.8, 4 x 8192 x 4096 12.3 / 10.9;
// norm 1 x 4096 x 14336 13.3 / 14.0, 4 x 4096 x 14336 15.0 / 14.0.
bool int8_rows_quantise(int from, int M, int K) {
  return M <= 16 && (long long)M * ((K / 8 + 63) / 64) <= (from == kFromNorm ? 1 : kPieces) * kWaves;
}
bool int8_rows_codes(int M, int K) { return M <= 16 && codes_bytes(M, K) <= kChunks * kThreads * 16; }

template <class Act, int FROM>
static int go(const Int8RowsArgs& p, hipStream_t st) {
  const int width = (kWaves >> p.ks_log2) * 16;
  auto* kernel = int8_rows_kernel<Act, FROM>;
  static std::atomic<unsigned long long> raised{0};
  const int rc = int8_raise_lds(kernel, raised, kWaves * kUnits * kUnit + (FROM == kFromCodes ? 64 : 16) * 1024);
  if (rc != MI_OK) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((p.N + width - 1) / width)), dim3(kThreads),
                     kWaves * kUnits * kUnit + (size_t)codes_bytes(p.M, p.K), st, p);
  return launch_status();
}

template <class Act>
static int launch(int from, Int8RowsArgs p, hipStream_t st) {
  const long tiles = (p.N + 15) / 16, cus = int8_cu_count();
  p.ks_log2 = 4;                                       // as many parts of K as leave the columns in one round of the CUs
  while (p.ks_log2 > 0 && tiles > cus * (kWaves >> p.ks_log2)) --p.ks_log2;
  switch (from) {
    case kFromAct: return go<Act, kFromAct>(p, st);
    case kFromNorm: return go<Act, kFromNorm>(p, st);
    case kFromSilu: return go<Act, kFromSilu>(p, st);
  }
  return go<Act, kFromCodes>(p, st);
}

int launch_int8_rows(int from, const Int8RowsArgs& p, int act_dtype, hipStream_t st) {
  return act_dtype == DT_F16 ? launch<ActF16>(from, p, st) : launch<ActBF16>(from, p, st);
}

}  // namespace qlin
