// 8-bit integer activations and weights (W8A8): what the launches share.
//
// A row v of activations becomes codes and a scale,
//
//   m = max(max|v|, 2^-40),   s = m / 127,   q = rint(127 v / m)  (ties to even),
//
// and the product with weights that were quantised per output channel is out[i][n] = (sum_k q[i][k] w[n][k]) s[i] w_scale[n].
// The sums are 32-bit integers: exact, and the same in any order, for K < 2^17.  A row that holds an infinity or a NaN has the scale NaN.
#pragma once
#include "qlinear_common.hpp"

#include <atomic>

namespace qlin {

typedef __attribute__((ext_vector_type(4))) float f32v4;

constexpr int kInt8MaxK = (1 << 17) - 16;             // |sum| <= 2^14 K < 2^31
constexpr float kInt8Floor = 0x1p-40f;

__device__ __forceinline__ uint32_t umax32(uint32_t a, uint32_t b) { return a > b ? a : b; }
// |v| as an ordered integer: NaN above infinity above every number
__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

// LDS that is written straight from memory (no registers in between): the compiler does not see when such a load lands, so every kernel
// here waits for itself.  N: loads that may still be under way, the newest ones; LDS reads and writes of the wavefront are done too.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
  asm volatile("" ::: "memory");
}
// A barrier that leaves loads under way, unlike __syncthreads.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  wait_loads<63>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
using lds_ptr = __attribute__((address_space(3))) void*;

// What a row's largest |v| gives: the factor that makes codes (0 where the row has none) and the scale.
struct RowScale {
  float inv, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t largest) {
  if (largest >= 0x7F800000u) return {0.0f, __builtin_nanf("")};
  const float m = fmaxf(__builtin_bit_cast(float, largest), kInt8Floor);
  return {127.0f / m, m / 127.0f};
}

// The code of v.  EXACT, for a v and an m of 11 significant bits: v inv is off by less than 2^-22 of itself, a quotient that is no tie is at
// least 2^-19 of itself away from one (2 * 127 v - (2 n + 1) m is a multiple of v's last place), so the quotient rounded to 21 bits
// is on the right side of every tie or on it.
// The code is the low byte of the result: the number added is a multiple of 256, and the sum's last place is 1.  In the row of an infinity
// or a NaN the codes mean nothing.
template <bool EXACT>
__device__ __forceinline__ uint32_t code_of(float v, float inv) {
#pragma clang fp contract(off)
  float t = v * inv;
  if constexpr (EXACT) {
    const float c = t * 9.0f;
    const float d = c - t;
    t = c - d;
  }
  return __builtin_bit_cast(uint32_t, t + 0x1.8p23f);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}

// SiLU(g) u, off by a few units in the last place: the exponential and the reciprocal are the hardware's (1 unit each), the rounding of
// -g log2(e) adds |g| / 2 units where g is negative.  With expf and a division the vector ALU bounds the rows that every workgroup of a
// decode step makes for itself: the call took 1.6 times as long.
__device__ __forceinline__ float silu_mul(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -0x1.715476p0f)) * u;
}

// The sum of squares of a wavefront's consecutive values, eight per lane.  A row's sum is that of these parts in their order, in every kernel, and
// the multiplications and additions are told apart here: a row has the same bits wherever it is quantised.
constexpr int kNormPart = 512;
__device__ __forceinline__ float norm_part(const float* v) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s = __builtin_fmaf(v[j], v[j], s);
  return wave_sum(s);
}

// Where a row comes from.
enum : int { kFromAct = 0, kFromNorm = 1, kFromSilu = 2, kFromF32 = 3, kFromCodes = 4 };

// K a multiple of 16 that the integer sums hold; M and N such that a workgroup of 256 per row is a grid of less than 2^32 threads (a larger one
// is not refused by the runtime: it starts fewer workgroups).
constexpr int kInt8MaxRows = (1 << 24) - 1;
static inline bool int8_sizes(int M, int N, int K) {
  return M >= 0 && N >= 0 && M <= kInt8MaxRows && N <= kInt8MaxRows && K > 0 && K % 16 == 0 && K <= kInt8MaxK;
}
static inline int int8_cu_count() {
  static const int count = [] {
    int dev = 0;
    hipDeviceProp_t prop;
    const bool known = hipGetDevice(&dev) == hipSuccess && hipGetDeviceProperties(&prop, dev) == hipSuccess && prop.multiProcessorCount > 0;
    return known ? prop.multiProcessorCount : 256;
  }();
  return count;
}
// A kernel that asks for more LDS than a launch gets unasked: once per device.
template <class Kernel>
static inline int int8_raise_lds(Kernel* kernel, std::atomic<unsigned long long>& raised, size_t bytes) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return MI_ERR_LAUNCH;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (raised.load(std::memory_order_relaxed) & bit)) return MI_OK;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess) {
    (void)hipGetLastError();
    return MI_ERR_LAUNCH;
  }
  if (dev < 64) raised.fetch_or(bit, std::memory_order_relaxed);
  return MI_OK;
}
static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Codes and scales of `rows` rows: from 16-bit activations (kFromAct), residual add and RMS norm (kFromNorm), SiLU(gate) x up of 16-bit
// rows of 2 K (kFromSilu) or fp32 rows (kFromF32).
struct QuantArgs {
  const void* x;
  const void* residual;
  void* residual_out;
  const void* norm_weight;
  int8_t* q;
  float* scale;
  long long rows;
  int K;
  float eps;
};
int launch_int8_quant(int from, const QuantArgs& p, int act_dtype, hipStream_t st);

}  // namespace qlin
