// What lies between the fused q, k, v projection of a layer and its attention, in one pass over the projection's rows: an RMS norm of every query
// and key head (optional weights), the rotation by the token's place on the first `rot` elements of a head, queries to q_out, keys to k_out
// (optional) and keys and values to their slots of the cache (optional).
//
//   y = x rsqrt(mean(x^2) + eps) w,   (a, b) -> (a cos - b sin, b cos + a sin),   pairs (i, i + rot / 2), or (2 i, 2 i + 1) interleaved
//
// in fp32, rounded once.  A head belongs to D / 16 lanes that hold two pieces of 8 elements each, chosen so that the two elements of a pair are in
// one lane: no exchange but the sum of squares.
//
// Bound: HBM, in and out once (8192 tokens of 64 + 2 x 8 heads of 128: 338 MB in 68 us, 5.0 TB/s, what a copy reaches); a token alone: the launch
// (2.8 us, the host's call 7).
#include "int8_common.hpp"

#include "../../include/mi355x_qlinear.h"

namespace qlin {

struct RopeArgs {
  const void *x, *qw, *kw, *table;
  const int64_t *positions, *slots;
  void *q, *k, *kc, *vc;
  long long x_token, q_token, q_head, k_token, k_head;           // strides in elements
  long long page, token, head;
  int page_size, T, Hq, Hkv, rot, places;
  long long places_of_cache;
  float eps;
};

template <class Elem>
__device__ __forceinline__ void load8(const Elem* p, float* f) {
  typedef __attribute__((ext_vector_type(8))) Elem e8;
  const e8 x = *(const e8*)p;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)x[i];
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float* f) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
}

template <class Act, class Table, int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const RopeArgs p) {
  using Elem = typename Act::elem;
  typedef __attribute__((ext_vector_type(8))) Elem e8;
  constexpr int L = D / 16;                            // lanes of a head
  const int heads = p.Hq + 2 * p.Hkv, u = threadIdx.x % L;
  const long long item = ((long long)blockIdx.x * 256 + threadIdx.x) / L;
  const int t = (int)(item / heads), head = (int)(item - (long long)t * heads);
  if (t >= p.T) return;
  const bool is_q = head < p.Hq, is_v = head >= p.Hq + p.Hkv;
  long long slot = -1;
  if (!is_q && p.slots) slot = p.slots[t];
  const bool cached = slot >= 0 && slot < p.places_of_cache;
  const Elem* x = (const Elem*)p.x + t * p.x_token + (long long)head * D;
  const int kv = head - p.Hq - (is_v ? p.Hkv : 0);
  long long at = 0;
  if (cached) {
    const long long page = slot / p.page_size;
    at = page * p.page + (slot - page * p.page_size) * p.token + kv * p.head;
  }
  // the two pieces of this lane
  const int turns = p.rot / 16;
  int first = 8 * u, second = 8 * u + p.rot / 2;
  if (INTERLEAVED || u >= turns) first = 16 * u, second = 16 * u + 8;
  if (is_v) {
    if (!cached) return;
    *(e8*)((Elem*)p.vc + at + first) = *(const e8*)(x + first);
    *(e8*)((Elem*)p.vc + at + second) = *(const e8*)(x + second);
    return;
  }
  float a[8], b[8];
  load8(x + first, a);
  load8(x + second, b);
  const Elem* w = (const Elem*)(is_q ? p.qw : p.kw);
  if (w) {
    auto squares = [&]() {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += a[i] * a[i] + b[i] * b[i];
#pragma unroll
      for (int d = 1; d < L; d <<= 1) sum += __shfl_xor(sum, d, 64);
      return sum;
    };
    float sum = squares(), eps = p.eps;
    if (sum == __builtin_inff()) {                     // bf16 from 1e18 on: the same for all lanes of a head
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] *= 0x1p-68f, b[i] *= 0x1p-68f;    // x 2^-68: the norm takes it out again; eps, 2^-136 of itself, no longer counts
      sum = squares();
      eps = 0.f;
    }
    const float f = 1.f / sqrtf(sum * (1.f / D) + eps);
    float wa[8], wb[8];
    load8(w + first, wa);
    load8(w + second, wb);
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] *= f * wa[i], b[i] *= f * wb[i];
  }
  if (u < turns) {
    const long long place = p.positions[t];
    const Table* row = (const Table*)p.table + (place >= 0 && place < p.places ? place : 0) * p.rot + 8 * u;
    float c[8], s[8];
    load8(row, c);
    load8(row + p.rot / 2, s);
    if (place < 0 || place >= p.places)                // no such row: nothing that could pass for a result
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = __builtin_nanf("");
    if constexpr (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
        a[2 * i] = a0 * c[i] - a1 * s[i];
        a[2 * i + 1] = a1 * c[i] + a0 * s[i];
        b[2 * i] = b0 * c[4 + i] - b1 * s[4 + i];
        b[2 * i + 1] = b1 * c[4 + i] + b0 * s[4 + i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a0 = a[i], b0 = b[i];
        a[i] = a0 * c[i] - b0 * s[i];
        b[i] = b0 * c[i] + a0 * s[i];
      }
    }
  }
  e8 ya, yb;
#pragma unroll
  for (int i = 0; i < 8; ++i) ya[i] = Act::from_f32(a[i]), yb[i] = Act::from_f32(b[i]);
  auto store = [&](Elem* to) {
    *(e8*)(to + first) = ya;
    *(e8*)(to + second) = yb;
  };
  if (is_q) return store((Elem*)p.q + t * p.q_token + head * p.q_head);
  if (p.k) store((Elem*)p.k + t * p.k_token + kv * p.k_head);
  if (cached) store((Elem*)p.kc + at);
}

template <class Act, class Table, int D>
static int launch(const RopeArgs& p, int interleaved, hipStream_t st) {
  const long long threads = (long long)p.T * (p.Hq + 2 * p.Hkv) * (D / 16);
  const unsigned grid = (unsigned)((threads + 255) / 256);
  if (interleaved) qk_norm_rope_kernel<Act, Table, D, true><<<grid, 256, 0, st>>>(p);
  else qk_norm_rope_kernel<Act, Table, D, false><<<grid, 256, 0, st>>>(p);
  return launch_status();
}
template <class Act, class Table>
static int pick(const RopeArgs& p, int D, int interleaved, hipStream_t st) {
  return D == 64 ? launch<Act, Table, 64>(p, interleaved, st) : D == 128 ? launch<Act, Table, 128>(p, interleaved, st)
                                                                         : launch<Act, Table, 256>(p, interleaved, st);
}

}  // namespace qlin

using namespace qlin;

extern "C" int mi_qk_norm_rope(const void* qkv, long long qkv_stride, const void* q_weight, const void* k_weight, const void* cos_sin,
                               int table_f32, const int64_t* positions, void* q_out, long long q_token_stride, long long q_head_stride,
                               void* k_out, long long k_token_stride, long long k_head_stride, const MiPagedCache* cache,
                               const int64_t* slots, int T, int num_heads, int num_kv_heads, int head_dim, int rot, int places, float eps,
                               int interleaved, int act_dtype, void* stream) {
  if (act_dtype != DT_F16 && act_dtype != DT_BF16) return MI_ERR_ARG;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return MI_ERR_SHAPE;
  if (T < 0 || num_heads <= 0 || num_kv_heads <= 0 || rot < 0 || rot % 16 || rot > head_dim || places < 0) return MI_ERR_SHAPE;
  if (num_heads > 1 << 16 || num_kv_heads > 1 << 16 || (long long)T * (num_heads + 2LL * num_kv_heads) * (head_dim / 16) >= 1LL << 31)
    return MI_ERR_SHAPE;
  if (!T) return MI_OK;
  if (!qkv || !q_out || (rot && (!cos_sin || !positions || !places)) || (!k_out && !cache) || !cache != !slots) return MI_ERR_ARG;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(q_weight) || !aligned16(k_weight) || !aligned16(cos_sin))
    return MI_ERR_ARG;
  if (qkv_stride % 8 || q_token_stride % 8 || q_head_stride % 8 || k_token_stride % 8 || k_head_stride % 8) return MI_ERR_SHAPE;
  RopeArgs p{};
  p.x = qkv;
  p.qw = q_weight;
  p.kw = k_weight;
  p.table = cos_sin;
  p.positions = positions;
  p.q = q_out;
  p.k = k_out;
  p.x_token = qkv_stride;
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.k_token = k_token_stride;
  p.k_head = k_head_stride;
  p.page_size = 1;
  if (cache) {
    if (!cache->key || !cache->value || !aligned16(cache->key) || !aligned16(cache->value)) return MI_ERR_ARG;
    if (cache->pages <= 0 || cache->page_size <= 0 || cache->page_stride % 8 || cache->token_stride % 8 || cache->head_stride % 8)
      return MI_ERR_SHAPE;
    p.slots = slots;
    p.kc = cache->key;
    p.vc = cache->value;
    p.page = cache->page_stride;
    p.token = cache->token_stride;
    p.head = cache->head_stride;
    p.page_size = cache->page_size;
    p.places_of_cache = (long long)cache->pages * cache->page_size;
  }
  p.T = T;
  p.Hq = num_heads;
  p.Hkv = num_kv_heads;
  p.rot = rot;
  p.places = places;
  p.eps = eps;
  hipStream_t st = (hipStream_t)stream;
  if (act_dtype == DT_F16)
    return table_f32 ? pick<ActF16, float>(p, head_dim, interleaved, st) : pick<ActF16, _Float16>(p, head_dim, interleaved, st);
  return table_f32 ? pick<ActBF16, float>(p, head_dim, interleaved, st) : pick<ActBF16, __bf16>(p, head_dim, interleaved, st);
}
