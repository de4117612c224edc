// Rows of activations as 8-bit codes and a scale (int8_quant.hip; the expert layer's first launch too).  Bound: HBM (2 bytes in and 1 out per
// value; 6 and 1 with the residual): SiLU rows of 2048 x 14336 26 us, 5.6 TB/s; 36864 rows of 768 in fp32 22 us, 6.4 TB/s.
//
// A row belongs to a wavefront (short rows) or a workgroup, and its values stay in registers from the one read to the codes: the norm's sum and
// the row's maximum are reductions in between.  Rows longer than the registers hold are read again for each of these steps.
#pragma once
#include "int8_common.hpp"

namespace qlin {

template <class Act, int FROM>
struct RowSource {
  using Elem = typename Act::elem;
  using V8 = typename Act::v8;
  const QuantArgs& p;
  size_t row;
  __device__ __forceinline__ RowSource(const QuantArgs& a, size_t r) : p(a), row(r) {}
  // eight values from k on, before the norm
  __device__ __forceinline__ void load(int k, float* v) const {
    if constexpr (FROM == kFromF32) {
      const f32v4* src = reinterpret_cast<const f32v4*>((const float*)p.x + row * p.K + k);
      const f32v4 a = src[0], b = src[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else if constexpr (FROM == kFromSilu) {
      const V8 g = *reinterpret_cast<const V8*>((const Elem*)p.x + row * 2 * p.K + k);
      const V8 u = *reinterpret_cast<const V8*>((const Elem*)p.x + row * 2 * p.K + p.K + k);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = silu_mul(Act::to_f32(g[i]), Act::to_f32(u[i]));
    } else {
      const V8 a = *reinterpret_cast<const V8*>((const Elem*)p.x + row * p.K + k);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = Act::to_f32(a[i]);
      if constexpr (FROM == kFromNorm) {
        const V8 b = *reinterpret_cast<const V8*>((const Elem*)p.residual + row * p.K + k);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += Act::to_f32(b[i]);
      }
    }
  }
  // the new residual, from the values that load() gave; the norm is taken of the 32-bit sums
  __device__ __forceinline__ void keep(int k, const float* v) const {
    V8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = Act::from_f32(v[i]);
    *reinterpret_cast<V8*>((Elem*)p.residual_out + row * p.K + k) = o;
  }
  __device__ __forceinline__ void norm(int k, float* v, float r) const {
    const V8 w = *reinterpret_cast<const V8*>((const Elem*)p.norm_weight + k);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * r * Act::to_f32(w[i]);
  }
  __device__ __forceinline__ void write(int k, const float* v, float inv) const {
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = code_of<FROM == kFromAct>(v[i], inv);
    *reinterpret_cast<u32x2*>(p.q + row * p.K + k) = u32x2{pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7])};
  }
};

// TPR threads per row, NV pieces of 8 values per thread in registers; NV = 0: the row is read again for every step.  TPR = 64: four rows in a
// workgroup of 256; otherwise a workgroup per row.
template <class Act, int FROM, int TPR, int NV>
__device__ __forceinline__ void int8_quant_rows(const QuantArgs& p, int block) {
  constexpr int WAVES = TPR == 64 ? 4 : TPR / 64;
  __shared__ float sums[FROM != kFromNorm || TPR == 64 ? 1 : NV ? WAVES * NV : (kInt8MaxK + kNormPart - 1) / kNormPart];
  __shared__ uint32_t tops[WAVES];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, at = TPR == 64 ? lane : threadIdx.x;
  const long long row = TPR == 64 ? (long long)block * 4 + wave : (long long)block;
  if (TPR == 64 && row >= p.rows) return;
  const RowSource<Act, FROM> src(p, (size_t)row);
  const int K = p.K;
  float v[NV ? NV : 1][8];
  float r = 0.0f;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = (i * TPR + at) * 8;
      if (k < K) src.load(k, v[i]);
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
      }
    }
  }
  if constexpr (FROM == kFromNorm) {
    float ss = 0.0f;
    if constexpr (TPR == 64) {
#pragma unroll
      for (int i = 0; i < NV; ++i) ss += norm_part(v[i]);
    } else {
      if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const float part = norm_part(v[i]);
          if (lane == 0) sums[i * WAVES + wave] = part;
        }
      } else {
        for (int k0 = wave * kNormPart; k0 < K; k0 += TPR * 8) {
          const int k = k0 + lane * 8;
          if (k < K) src.load(k, v[0]);
          else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[0][j] = 0.0f;
          }
          const float part = norm_part(v[0]);
          if (lane == 0) sums[k0 / kNormPart] = part;
        }
      }
      __syncthreads();
      for (int q = 0; q < (K + kNormPart - 1) / kNormPart; ++q) ss += sums[q];
    }
    r = rsqrtf(ss / (float)K + p.eps);
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = (i * TPR + at) * 8;
        if (k < K) {
          src.keep(k, v[i]);
          src.norm(k, v[i], r);
        }
      }
    }
  }
  uint32_t top = 0;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = umax32(top, abs_bits(v[i][j]));
  } else {
    for (int k = at * 8; k < K; k += TPR * 8) {
      src.load(k, v[0]);
      if constexpr (FROM == kFromNorm) src.norm(k, v[0], r);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = umax32(top, abs_bits(v[0][j]));
    }
  }
  top = wave_max_u32(top);
  if constexpr (TPR > 64) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = umax32(top, tops[w]);
  }
  const RowScale s = row_scale(top);
  if (at == 0) p.scale[row] = s.scale;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = (i * TPR + at) * 8;
      if (k < K) src.write(k, v[i], s.inv);
    }
  } else {
    for (int k = at * 8; k < K; k += TPR * 8) {
      src.load(k, v[0]);                               // a thread reads what it alone overwrites: residual_out may be residual
      if constexpr (FROM == kFromNorm) {
        src.keep(k, v[0]);
        src.norm(k, v[0], r);
      }
      src.write(k, v[0], s.inv);
    }
  }
}

}  // namespace qlin
