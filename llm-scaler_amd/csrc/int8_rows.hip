// The product of few rows (M <= 64) with 8-bit weights: out[m][n] = (sum_k q[m][k] w[n][k]) s[m] w_scale[n].  Bound: HBM, the weights once.
//
// A workgroup of 16 wavefronts owns 16 NT columns per slot; the KS = 16 / slots wavefronts of a slot each take a part of K, so that all
// of a CU's loads are in flight at once however few columns there are.  A wavefront keeps a ring of U pieces (64 bytes of 16 weight rows: the
// operand of v_mfma_i32_16x16x64_i8 as it comes from memory) under way; the parts of K meet in LDS as integers.
//
// Rows that are not codes yet (16-bit activations, residual + norm, SiLU x up) are quantised by every workgroup for itself while its
// first weights are on their way: the rows are few KiB and come from L2, a launch in front would be a round trip.
#include "int8_rows.hpp"

namespace qlin {

constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr int kPieces = 4;                            // pieces of 8 values per thread that a workgroup quantises

// MT tiles of 16 rows, NT of 16 columns per wavefront, U pieces under way
template <class Act, int FROM, int MT, int NT, int U>
__global__ __launch_bounds__(kThreads) void int8_rows_kernel(const Int8RowsArgs p) {
  using Elem = typename Act::elem;
  using V8 = typename Act::v8;
  constexpr bool kCodes = FROM == kFromCodes;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ float row_s[16];
  __shared__ float part_sum[kWaves * kPieces];
  __shared__ uint32_t part_top[kWaves * kPieces];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int M = p.M, N = p.N, K = p.K, KS = 1 << p.ks_log2, slots = kWaves >> p.ks_log2;
  const int slot = wave >> p.ks_log2, part = wave & (KS - 1);
  const int blocks = (K + 63) / 64, per = (blocks + KS - 1) >> p.ks_log2;
  const int b0 = part * per, b1 = b0 + per < blocks ? b0 + per : blocks;
  const int n0 = (blockIdx.x * slots + slot) * NT * 16, cols = n0 < N ? (N - n0 < NT * 16 ? N - n0 : NT * 16) : 0;
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(cols ? p.w + (size_t)n0 * K : p.w, (uint32_t)cols * (uint32_t)K);
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x, kCodes ? (uint32_t)M * (uint32_t)K : 0u);

  // rows to be quantised: pieces of 8 values, whole wavefronts per row
  const int waves_per_row = (K / 8 + 63) / 64, pieces = waves_per_row * 64 * M;
  float v[kCodes ? 1 : kPieces][8];
  auto row_of = [&](int i) __attribute__((always_inline)) { return (i * kWaves + wave) / waves_per_row; };
  auto k_of = [&](int i, int row) __attribute__((always_inline)) { return ((i * kWaves + wave - row * waves_per_row) * 64 + lane) * 8; };
  if constexpr (!kCodes) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
      const int row = row_of(i), k = k_of(i, row);
      if (i * kThreads < pieces && row < M && k < K) {
        const Elem* src = (const Elem*)p.x + (size_t)row * (FROM == kFromSilu ? 2 * K : K) + k;
        const V8 a = *reinterpret_cast<const V8*>(src);
        if constexpr (FROM == kFromSilu) {
          const V8 b = *reinterpret_cast<const V8*>(src + K);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = silu_mul(Act::to_f32(a[j]), Act::to_f32(b[j]));
        } else if constexpr (FROM == kFromNorm) {
          const V8 b = *reinterpret_cast<const V8*>((const Elem*)p.residual + (size_t)row * K + k);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = Act::to_f32(a[j]) + Act::to_f32(b[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = Act::to_f32(a[j]);
        }
      }
    }
  }

  i32x4 wr[U][NT], xr[U][kCodes ? MT : 1];
  uint32_t w_at[NT], x_at[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) w_at[j] = (uint32_t)(j * 16 + r16) * (uint32_t)K + g * 16;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = t * 16 + r16 < M ? t * 16 + r16 : M - 1;      // a column of the product past M is not stored
    x_at[t] = (uint32_t)m * (uint32_t)K + g * 16;
  }
  // piece b of the part: past its end, zeros; of codes, zeros past the row's end too (what the weights bring there does not count)
  auto request = [&](int u, int b) __attribute__((always_inline)) {
    const uint32_t off = b < b1 ? (uint32_t)b * 64u : kOOB;
#pragma unroll
    for (int j = 0; j < NT; ++j) wr[u][j] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, w_at[j] + off, 0, 2));
    if constexpr (kCodes) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
        xr[u][t] = __builtin_bit_cast(i32x4, buf_load16(rx, b * 64 + g * 16 < K ? x_at[t] + off : kOOB));
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) request(u, b0 + u);

  if constexpr (!kCodes) {
    if constexpr (FROM == kFromNorm) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        if (i * kThreads >= pieces) break;
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
        ss = wave_sum(ss);
        if (lane == 0) part_sum[i * kWaves + wave] = ss;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int row = row_of(i), k = k_of(i, row);
        if (i * kThreads >= pieces || row >= M) break;
        float ss = 0.0f;
        for (int q = 0; q < waves_per_row; ++q) ss += part_sum[row * waves_per_row + q];
        const float r = rsqrtf(ss / (float)K + p.eps);
        if (k < K) {
          if (blockIdx.x == 0) {
            V8 o;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = Act::from_f32(v[i][j]);
            *reinterpret_cast<V8*>((Elem*)p.residual_out + (size_t)row * K + k) = o;
          }
          const V8 nw = *reinterpret_cast<const V8*>((const Elem*)p.norm_weight + k);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * r * Act::to_f32(nw[j]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i * kThreads >= pieces) break;
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = umax32(top, abs_bits(v[i][j]));
      top = wave_umax(top);
      if (lane == 0) part_top[i * kWaves + wave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int row = row_of(i), k = k_of(i, row);
      if (i * kThreads >= pieces || row >= M) break;
      uint32_t top = 0;
      for (int q = 0; q < waves_per_row; ++q) top = umax32(top, part_top[row * waves_per_row + q]);
      const RowScale s = row_scale(top);
      if (k == 0) row_s[row] = s.scale;
      if (k < blocks * 64) {                           // past K: zeros, to the end of the last piece of 64
        int c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = code_of<FROM == kFromAct>(v[i][j], s.inv);
        *reinterpret_cast<u32x2*>(smem + ((k >> 6) * M + row) * 64 + (k & 63)) =
            u32x2{pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7])};
      }
    }
    __syncthreads();
  }

  i32x4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[j][t] = i32x4{0, 0, 0, 0};
  const unsigned char* mine = smem + (r16 < M ? r16 : M - 1) * 64 + g * 16;
  for (int b = b0; b < b1; b += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      i32x4 x[MT];
      if constexpr (kCodes) {
#pragma unroll
        for (int t = 0; t < MT; ++t) x[t] = xr[u][t];
      } else {
        const int at = b + u < blocks ? b + u : blocks - 1;      // the weights beyond are zeros
        x[0] = *reinterpret_cast<const i32x4*>(mine + at * M * 64);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[j][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wr[u][j], x[t], acc[j][t], 0, 0, 0);
      request(u, b + U + u);
    }
  }

  // the parts' sums, then one thread per output
  if constexpr (!kCodes) __syncthreads();              // the codes are read
  int32_t* sums = reinterpret_cast<int32_t*>(smem);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) *reinterpret_cast<i32x4*>(sums + ((wave * NT + j) * MT + t) * 256 + lane * 4) = acc[j][t];
  __syncthreads();
  const int width = slots * NT * 16, first = blockIdx.x * width;
  for (int i = tid; i < M * width; i += kThreads) {
    const int m = i / width, c = i - m * width, n = first + c;
    if (n >= N) continue;
    const int tile = c >> 4, s = tile / NT, j = tile - s * NT, t = m >> 4;
    const int32_t* from = sums + (((s << p.ks_log2) * NT + j) * MT + t) * 256 + (((c & 15) >> 2) * 16 + (m & 15)) * 4 + (c & 3);
    int sum = 0;
    for (int q = 0; q < KS; ++q) sum += from[q * NT * MT * 256];
    float o = (float)sum * ((kCodes ? p.x_scale[m] : row_s[m]) * p.w_scale[n]);
    if (p.bias) o += Act::to_f32(((const Elem*)p.bias)[n]);
    ((Elem*)p.out)[(size_t)m * N + n] = Act::from_f32(o);
  }
}

// Rows that a workgroup quantises for itself.
bool int8_rows_quantise(int M, int K) {
  return M <= 16 && (long long)M * ((K / 8 + 63) / 64) <= kPieces * kWaves;
}

template <class Act, int FROM, int MT, int NT, int U>
static int go(const Int8RowsArgs& p, hipStream_t st) {
  const int slots = kWaves >> p.ks_log2, width = slots * NT * 16;
  constexpr size_t sums = (size_t)kWaves * NT * MT * 1024;
  const size_t codes = FROM == kFromCodes ? 0 : (size_t)p.M * ((p.K + 63) / 64) * 64;
  auto* kernel = int8_rows_kernel<Act, FROM, MT, NT, U>;
  if constexpr (sums > 32 * 1024) {
    static std::atomic<unsigned long long> raised{0};
    const int rc = int8_raise_lds(kernel, raised, sums);
    if (rc != MI_OK) return rc;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)((p.N + width - 1) / width)), dim3(kThreads), sums > codes ? sums : codes, st, p);
  return launch_status();
}

template <class Act>
static int launch(int from, Int8RowsArgs p, hipStream_t st) {
  const int NT = from == kFromCodes && p.M > 16 ? 2 : 1;
  const long tiles = (p.N + 16 * NT - 1) / (16 * NT), cus = int8_cu_count();
  p.ks_log2 = 4;                                       // as many parts of K as leave the columns in one round of the CUs
  while (p.ks_log2 > 0 && tiles > cus * (kWaves >> p.ks_log2)) --p.ks_log2;
  switch (from) {
    case kFromAct: return go<Act, kFromAct, 1, 1, 8>(p, st);
    case kFromNorm: return go<Act, kFromNorm, 1, 1, 8>(p, st);
    case kFromSilu: return go<Act, kFromSilu, 1, 1, 8>(p, st);
  }
  if (p.M <= 16) return go<Act, kFromCodes, 1, 1, 8>(p, st);
  if (p.M <= 32) return go<Act, kFromCodes, 2, 2, 4>(p, st);
  if (p.M <= 48) return go<Act, kFromCodes, 3, 2, 3>(p, st);
  return go<Act, kFromCodes, 4, 2, 3>(p, st);
}

int launch_int8_rows(int from, const Int8RowsArgs& p, int act_dtype, hipStream_t st) {
  return act_dtype == DT_F16 ? launch<ActF16>(from, p, st) : launch<ActBF16>(from, p, st);
}

}  // namespace qlin
