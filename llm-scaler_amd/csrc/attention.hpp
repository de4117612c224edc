// Attention over a paged cache: what its two kernels share.
//
//   o_i = sum_j p_ij v_j,   p_ij = 2^(c (s_ij - m_i)) / l_i,   s_ij = q_i . k_j,   c = scale log2(e)
//
// in one pass over the keys: m follows the largest s of a row, l is the running sum, and both o and l are multiplied by
// 2^(c (m_old - m_new)) where m moves.  s, m, l and o are fp32; p is rounded to the type of the values in front of its product with
// them (off by half a step of a 16-bit number, below the output's rounding, as v_j is already such a number), and l sums the rounded p.
//
// The rows of a kv head are (token, head of the group) pairs of a sequence, token first: row r is head r % G of token r / G.  A wavefront holds 32
// rows as columns of v_mfma_f32_32x32x16: S^T = K Q^T has a row's scores in the registers of two lanes (16 of 32 keys each), so that maximum and sum
// take one exchange, and those 16 values, rounded, are what the second product O^T = V^T P^T takes as its operand: the keys of V^T come in the order
// that they have in the registers (ds_read_b64_tr_b16 gathers four keys of a column).
//
// Keys and values come to LDS straight from memory, 16 bytes a lane.  What no row of a tile sees (behind the end, outside the window, on a page
// outside the cache) reaches nothing, NaN included, in one of two ways.  A lane looks up the page of one key, and such a key reads zeros instead: the
// rows kernel, and the tiles kernel where pages hold no groups of 8 places.  Or a wavefront looks up the page of 8 places at once and reads them as
// they are, or some place of the cache for a group that nothing sees: AttnRows::hide takes their scores out and AttnRows::clean puts zeros where their
// values are no numbers, in every block that holds such a key.
#pragma once
#include "int8_common.hpp"

namespace qlin {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(4))) unsigned short u16x4;

struct AttnArgs {
  const void *q, *k, *v;
  void* out;                   // [T, Hq, D]
  const int32_t *table, *seq_lens, *cu;
  const int64_t* tree;         // [T, tree_words]: tree_attention; null: causal
  float* part;                 // partial results
  long long q_token, q_head;   // strides of q in elements
  uint32_t page16, row16, head16;        // strides of the cache in 16 bytes
  uint32_t page_mul, page_shift;         // key / page
  int T, B, Hq, Hkv, G, page, width, pages;
  int window, sinks, tree_words;         // window 0: none
  float c, far;                // far: 2^10 / c
  int groups, tile_rows;       // rows kernel: workgroups; rows of a tile, as the caller says
  bool wide, many_parts;       // its work may count 2^30 blocks or more; a tile is in many parts
  int slots, shares;           // tiles kernel: a workgroup per tile (slots of them), or in that many equal shares
  int rows_from;               // sequences with that many rows (tokens x G) or more belong to the tiles kernel
};

constexpr uint32_t kNoRow = 0xFFFFFFFFu;
constexpr int kBlock = 64;                            // keys of a block of work

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
// v of lanes l % 32 and 32 + l % 32
struct Halves { float low, high; };
__device__ __forceinline__ Halves both_halves(float v) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const uint32_t low = r[0], high = r[1];              // a bit cast of r[1] itself would be one of r[0]
  return {__builtin_bit_cast(float, low), __builtin_bit_cast(float, high)};
}

// ---- a sequence of the call -------------------------------------------------------------------
struct AttnSeq {
  int q0, n;                   // its tokens
  int first;                   // place of its first token: length - n
  int cap;                     // keys that can be there: min(length, places of the table)
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& p, int b) {
  AttnSeq s;
  s.q0 = min(max(p.cu[b], 0), p.T);
  s.n = min(max(p.cu[b + 1], s.q0), p.T) - s.q0;
  const int len = max(p.seq_lens[b], 0);
  s.first = len - s.n;
  s.cap = min(len, p.width * p.page);
  return s;
}

// The blocks of BLOCK keys that tokens t0 .. t1 of a sequence see some of: first the `head` blocks with visible first tokens, then all from `from` on.
struct AttnRange { int lo, hi, head, from, blocks; };
template <int BLOCK>
__device__ __forceinline__ AttnRange attn_range(const AttnArgs& p, const AttnSeq& s, int t0, int t1) {
  AttnRange r;
  r.lo = 0;
  r.hi = s.cap;
  if (!p.tree) {
    r.hi = min(s.cap, max(s.first + t1 + 1, 0));
    if (p.window) r.lo = min(max(s.first + t0 - p.window + 1, 0), r.hi);
  }
  r.from = r.lo / BLOCK * BLOCK;
  r.head = min(r.from, (min(p.sinks, r.hi) + BLOCK - 1) / BLOCK * BLOCK) / BLOCK;
  r.blocks = r.head + (r.hi - r.from + BLOCK - 1) / BLOCK;
  return r;
}
template <int BLOCK>
__device__ __forceinline__ int attn_key(const AttnRange& r, int block) {
  return block < r.head ? block * BLOCK : r.from + (block - r.head) * BLOCK;
}

// The column of the table with the page of key `key`
__device__ __forceinline__ int attn_page_of(const AttnArgs& p, int key) {
  return (int)((__umulhi((uint32_t)key, p.page_mul) + (uint32_t)key) >> p.page_shift);
}
__device__ __forceinline__ bool attn_in(const AttnArgs& p, const AttnRange& r, int key) { return key < r.hi && (key >= r.lo || key < p.sinks); }
// Where key `key` lies, on page `page`, in 16 bytes from the cache's start; kNoRow: not in the cache
__device__ __forceinline__ uint32_t attn_place(const AttnArgs& p, int page, int key, int head) {
  if ((uint32_t)page >= (uint32_t)p.pages) return kNoRow;
  return (uint32_t)page * p.page16 + (uint32_t)(key - attn_page_of(p, key) * p.page) * p.row16 + (uint32_t)head * p.head16;
}

// Bit i: a token sees key kb + i.  The token stands at place first + t (negative: before the cache's start), its tree bits in `tree`.
__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
__device__ __forceinline__ uint32_t low_bits32(int n) { return n >= 32 ? ~0u : (1u << max(n, 0)) - 1; }
__device__ __forceinline__ uint32_t attn_sees(const AttnArgs& p, int first, int t, const int64_t* tree, int kb) {
  if (p.tree) {
    const int at = kb - first;                         // the drafted token of key kb
    if (at <= -32) return ~0u;
    auto word = [&](int w) { return w < 2 * p.tree_words ? ((const uint32_t*)tree)[w] : 0u; };
    if (at < 0) return low_bits32(-at) | word(0) << -at;
    const int w = at >> 5, by = at & 31;
    return word(w) >> by | (by ? word(w + 1) << (32 - by) : 0u);
  }
  const int place = first + t;
  uint32_t m = low_bits32(place - kb + 1);
  if (p.window) m &= ~low_bits32(place - p.window + 1 - kb) | low_bits32(p.sinks - kb);
  return m;
}
// Whether every token from t0 to t1 sees all of the N keys from kb on
template <int N>
__device__ __forceinline__ bool attn_all_seen(const AttnArgs& p, int first, int t0, int t1, int kb) {
  if (p.tree) return kb + N <= first;
  return kb + N - 1 <= first + t0 && (!p.window || kb > first + t1 - p.window || kb + N <= p.sinks);
}

// ---- loads ------------------------------------------------------------------------------------
__device__ const u32x4 kZeroRow[64] = {};             // what a key that nothing sees is read from

// 16-byte chunk c of key row r lies at place c ^ swizzle of its row: eight lanes that read a column of K rows at a time, and the four rows of 64
// bytes that a transposing read of V takes, find different banks.
template <int D> __device__ __forceinline__ int k_swizzle(int r) { return D == 64 ? r >> 1 & 7 : r & 15; }
template <int D> __device__ __forceinline__ int v_swizzle(int r) { return D == 64 ? (r >> 1 & 1) << 2 : (r & 3) << 2; }

__device__ const int32_t kNoPage[1] = {-1};

// 16 (4) bytes per lane from memory to LDS, side by side.  As a builtin the compiler waits for all of them in front of every transposing read of
// LDS, loads for the next block included; here the kernels wait for themselves (wait_loads) and the compiler counts none of them.
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }
template <class T> __device__ __forceinline__ __attribute__((address_space(3))) T* in_lds(uint32_t at) {
  return (__attribute__((address_space(3))) T*)(uintptr_t)at;
}
// An address that is the same for all lanes of a wavefront: read by a scalar load, which counts with those of LDS
template <class T> __device__ __forceinline__ T scalar_load(const T* p) { return *(const __attribute__((address_space(4))) T*)(uintptr_t)p; }
__device__ __forceinline__ void to_lds16(const void* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
// from a scalar address and a distance per lane
__device__ __forceinline__ void to_lds16_from(const void* base, uint32_t by, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(by), "s"(base), "s"(to) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(const void* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}

// Rows [first, first + ROWS) of a block of keys to LDS by one wavefront: lane i holds the place of row i of the block, from which every lane takes
// those of the rows that it loads a part of.
template <int D, int ROWS>
struct RowPlaces {
  static constexpr int CH = D / 8, RPI = 64 / CH, N = ROWS / RPI;          // chunks of a row, rows per load
  static_assert(RPI * N == ROWS && (64 % CH) == 0, "rows per load");
  uint32_t of[N];
  __device__ __forceinline__ void take(uint32_t place, int first) {
#pragma unroll
    for (int j = 0; j < N; ++j) of[j] = __shfl(place, first + j * RPI + (int)(threadIdx.x & 63) / CH, 64);
  }
  template <bool IS_K>
  __device__ __forceinline__ void load(const void* from, int first, uint32_t to) const {     // to: in LDS
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int r = first + j * RPI + lane / CH, chunk = (lane % CH) ^ (IS_K ? k_swizzle<D>(r) : v_swizzle<D>(r));
      const unsigned char* a = of[j] != kNoRow ? (const unsigned char*)from + (uint64_t)of[j] * 16 : (const unsigned char*)kZeroRow;
      to_lds16(a + chunk * 16, to + j * 1024);
    }
  }
};

// ---- the rows of a wavefront ------------------------------------------------------------------
// Exponents of the weights: fma(c, s, raise - c m), one instruction, while c |m| < 2^10; raise - c m is then rounded by 2^-14 at most, the same for all
// weights that go by this m.  Of a larger one the last place is worth whole units in the end: there the scores give way to s - m, exact where it matters,
// and the exponent is fma(c, s - m, raise).  Those rows keep their m apart, so that others pay nothing for them (with a comparison more in every step
// 695 against 680 us for chunks of heads of 256, 410 against 405 for a prompt in a window with heads of 64).
// The raise: m may lag, so the largest weight of a row is 2^raise to 2^(raise + 8).  fp16: up to 2^15, so that the weights of a long tail keep
// their bits (half of the smallest number is 2^-32 of the largest weight).  bf16, whose values reach as far as the sums: up to 1, so that no sum is
// larger than the formula's.
template <class Act> constexpr float attn_raise = Act::dt == DT_F16 ? 7.f : -8.f;
// What sums that go by m are multiplied by where they go by `to` >= m; 0 from m = -inf
__device__ __forceinline__ float attn_moved(const AttnArgs& p, float m, float to) { return __builtin_amdgcn_exp2f((m - to) * p.c); }

// 32 rows over steps of 32 keys: scores (K Q^T), their maximum, weights (exp), and the product with V.
template <class Act, int D>
struct AttnRows {
  using v8 = typename Act::v8;
  typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
  typedef __attribute__((ext_vector_type(8))) short i16x8;
  typedef __attribute__((ext_vector_type(4))) typename Act::elem e4;
  static constexpr int DT = D / 32;
  static constexpr float kRaise = attn_raise<Act>;
  static constexpr unsigned short EXPONENT = Act::dt == DT_F16 ? 0x7C00 : 0x7F80;
  struct Weights { v8 p[2]; };                         // p[t][e]: key 16 t + 8 (e / 4) + 4 (lane / 32) + e % 4 of row lane % 32
  // Operands whose reads of LDS go out long before their products: they stay on their side of a `pin`, everything else may move.
  struct Keys { v8 k[D / 16]; };
  struct Values { v8 v[DT]; };
  static __device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0x40E); }

  v8 q[D / 16];
  f32x16 o[DT];                // o[t][i]: column 32 t + 8 (i / 4) + 4 (lane / 32) + i % 4 of row lane % 32
  float m, l;                  // m: the score that a row's exponents are taken from, at most 8 / c below the largest; l: of this lane's keys
  float apart;                 // m where c |m| is 2^10 or more; m is -inf there, as where a row has seen nothing yet
  int ka, va;                  // where this lane reads K and V of a step

  __device__ __forceinline__ void start() {
    const int lane = threadIdx.x & 63, h = lane >> 5, i = lane & 15;
    m = -__builtin_inff();
    l = 0.f;
    apart = m;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x16{};
    ka = (lane & 31) * 2 * D + ((h ^ k_swizzle<D>(lane & 31)) * 16);
    // keys 4 h + i / 4, columns 16 (lane / 16 % 2) + 4 (i % 4)
    va = (4 * h + (i >> 2)) * 2 * D + (((2 * (lane >> 4 & 1) + (i >> 1 & 1)) ^ v_swizzle<D>(i >> 2)) * 16) + (i & 1) * 8;
  }
  __device__ __forceinline__ void load_q(const void* row) {      // null: zeros
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      u32x4 x = {};
      if (row) x = *(const u32x4*)((const unsigned char*)row + s * 32 + h * 16);
      q[s] = as_v8<v8>(x);
    }
  }
  // K of the 32 keys at LDS address k, columns 16 ks ..
  __device__ __forceinline__ v8 k_operand(uint32_t k, int ks) const {
    return as_v8<v8>(in_lds<const u32x4>(k + (ka ^ (ks % 8 * 32)))[ks / 8 * 16]);
  }
  // V^T of 16 keys (from 16 t of those at LDS address v) and columns 32 d ..: element e is key 4 (lane / 32) + e % 4 + 8 (e / 4)
  __device__ __forceinline__ v8 v_operand(uint32_t v, int t, int d) const {
    auto* at = in_lds<i16x4>(v + (va ^ ((d & 3) * 64))) + (d >> 2) * 32 + t * 4 * D;       // one address and distances known to the instruction
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at + 2 * D);
    return __builtin_bit_cast(v8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  __device__ __forceinline__ void read_keys(uint32_t k, Keys& f) const {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) f.k[ks] = k_operand(k, ks);
  }
  __device__ __forceinline__ void read_values(uint32_t v, int t, Values& f) const {
#pragma unroll
    for (int d = 0; d < DT; ++d) f.v[d] = v_operand(v, t, d);
  }

  // Scores: element i is key 8 (i / 4) + 4 (lane / 32) + i % 4 of row lane % 32
  __device__ __forceinline__ f32x16 scores(const Keys& f) const {
    f32x16 x = {};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) x = mfma32(f.k[ks], q[ks], x);
    return x;
  }
  // -inf where the row does not see the key.  mask: bit i of this lane's row, null where a key is not there
  __device__ __forceinline__ void hide(f32x16& x, uint32_t mask) const {
    const uint32_t bits = mask >> (4 * ((threadIdx.x & 63) >> 5));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t sees = (uint32_t)((int32_t)(bits << (31 - 8 * (i / 4) - i % 4)) >> 31);
      const float s = x[i];                            // its own variable: a bit cast of an element is one of element 0
      x[i] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, s) & sees) | (0xFF800000u & ~sees));
    }
  }
  // The largest of a row's scores
  static __device__ __forceinline__ float largest(const f32x16& x) {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
    const Halves y = both_halves(mx);
    return fmaxf(y.low, y.high);
  }
  __device__ __forceinline__ float reference() const { return m == -__builtin_inff() ? apart : m; }
  // Makes m fit the scores x, most their largest.  Sums move to a new m only where an exponent would pass it by 8.
  __device__ __forceinline__ void follow(const AttnArgs& p, f32x16& x, float most) {
    if (!__builtin_amdgcn_ballot_w64((most - m) * p.c > 8.f)) return;         // m = -inf: all that is seen
    const float from = reference();
    const bool moves = (most - from) * p.c > 8.f;      // row by row: a row's bits depend on no other row
    if (__builtin_amdgcn_ballot_w64(moves)) {
      const float to = moves ? most : from, a = moves ? attn_moved(p, from, to) : 1.f;
      l *= a;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        if constexpr (D == 256) asm volatile("" : "+a"(o[d]));   // accumulation registers up to here: not all copied in every step
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= a;
        if constexpr (D == 256) asm volatile("" : "+a"(o[d]));
      }
      const bool far = fabsf(to) >= p.far && to != -__builtin_inff();
      m = far ? -__builtin_inff() : to;
      apart = far ? to : -__builtin_inff();
    }
    if (!__builtin_amdgcn_ballot_w64(apart != -__builtin_inff())) return;
    const float by = apart == -__builtin_inff() ? 0.f : apart;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] -= by;
  }
  __device__ __forceinline__ void weigh(const AttnArgs& p, const f32x16& x, Weights& w) {
    const float add = fabsf(m) >= p.far ? kRaise : __builtin_fmaf(-m, p.c, kRaise);
    typedef __attribute__((ext_vector_type(2))) typename Act::elem e2;
    const e2 one = {(typename Act::elem)1.f, (typename Act::elem)1.f};
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w.p[t][e] = Act::from_f32(__builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * t + e], p.c, add)));
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const e2 two = {w.p[t][e], w.p[t][e + 1]};
        if constexpr (Act::dt == DT_F16) sum = __builtin_amdgcn_fdot2(two, one, sum, false);
        else sum = __builtin_amdgcn_fdot2_f32_bf16(two, one, sum, false);
      }
    }
    l += sum;
  }
  // A step of the tiles kernel: weights of the scores x, the product with their values, and the next step's scores with their largest.  f: the next
  // step's keys, then those at k2; the values are read while the scores are made.
  __device__ __forceinline__ f32x16 step(const AttnArgs& p, const f32x16& x, uint32_t v, Keys& f, uint32_t k2, float& most) {
    Values va, vb;
    Weights w;
    read_values(v, 0, va);
    pin();
    const f32x16 y = scores(f);
    read_values(v, 1, vb);
    pin();
    weigh(p, x, w);
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = mfma32(va.v[d], w.p[0], o[d]);
    read_keys(k2, f);
    most = largest(y);
    pin();
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = mfma32(vb.v[d], w.p[1], o[d]);
    return y;
  }
  __device__ __forceinline__ void add(uint32_t v, const Weights& w) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] = mfma32(v_operand(v, t, d), w.p[t], o[d]);
  }

  // Infinities and NaN among values that a row does not see: 0 times them would not be 0.  They give way to zeros, and go to the rows that see them by
  // themselves.
  //
  // The rows kernel: while the values are read
  __device__ __forceinline__ void add_hidden(uint32_t v, const Weights& w, uint32_t mask) {
    u16x8 all = 0xFFFF;                                // 0 where a value was not finite
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u16x8 x = __builtin_bit_cast(u16x8, v_operand(v, t, d)), finite = are_finite(x);
        all &= finite;
        o[d] = mfma32(__builtin_bit_cast(v8, x & finite), w.p[t], o[d]);
      }
    }
    if (!__builtin_amdgcn_ballot_w64(any_not(all))) return;
#pragma unroll 1
    for (int j = 0; j < 32; ++j)
      add_not_finite(mask >> j & 1, [&](int column) {
        return *in_lds<const u16x4>(v + j * 2 * D + ((column >> 3) ^ v_swizzle<D>(j)) * 16 + (column & 7) * 2);
      });
  }
  // The tiles kernel: zeros in 8 rows of values in LDS, and whether there were any in the rows whose bits `there` has; the values themselves from the
  // cache at the end
  template <int PIECES>
  static __device__ __forceinline__ bool clean(uint32_t v, uint32_t there) {
    bool spoilt = false;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      auto* at = in_lds<u16x8>(v + j * 1024 + (threadIdx.x & 63) * 16);
      const u16x8 x = *at, finite = are_finite(x);
      const bool found = any_not(finite);
      if (!__builtin_amdgcn_ballot_w64(found)) continue;
      *at = x & finite;
      spoilt |= found && there >> (j * (512 / D) + (threadIdx.x & 63) / (D / 8)) & 1;
    }
    return __builtin_amdgcn_ballot_w64(spoilt) != 0;
  }
  // The infinities and NaN of a row of values, four columns from `column` on at a time, where this lane's row sees it
  template <class Read>
  __device__ __forceinline__ void add_not_finite(bool sees, Read read) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u16x4 x = read(32 * d + 8 * i + 4 * h);
        const e4 y = __builtin_bit_cast(e4, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][4 * i + e] += sees && (x[e] & EXPONENT) == EXPONENT ? Act::to_f32(y[e]) : 0.f;
      }
    }
  }
  // All ones where a number is finite: the difference of its exponent and the largest one is below zero
  static __device__ __forceinline__ u16x8 are_finite(u16x8 x) {
    return __builtin_bit_cast(u16x8, __builtin_bit_cast(i16x8, (x & EXPONENT) - EXPONENT) >> 15);
  }
  static __device__ __forceinline__ bool any_not(u16x8 ones) {
    const u32x4 x = __builtin_bit_cast(u32x4, ones);
    return (x[0] & x[1] & x[2] & x[3]) != 0xFFFFFFFFu;
  }
};

// ---- equal shares of the work -------------------------------------------------------------------
// All blocks of KEYS keys of all (sequence, tile of ROWS rows, kv head) in a row, each of these with ITEM blocks more for what beginning it costs, are cut
// into equal shares, one per workgroup, whatever the sequences' lengths are.  A tile whose blocks all lie in one share is finished there; of the
// others a workgroup has at most one that it continues and one that it begins: two parts, unscaled fp32 sums with their m and l, which a second launch
// joins.  FEW: of the sequences with fewer than rows_from rows; otherwise of the others.  Num: int where all work counts less than 2^30 blocks.
template <int ROWS, int KEYS, int ITEM, bool FEW, class Num>
struct Shares {
  // How many tiles a sequence has here, and how many blocks each of them
  struct Seq { AttnSeq s; AttnRange r; int tiles; };
  static __device__ __forceinline__ Seq seq_of(const AttnArgs& p, const AttnSeq& s) {
    Seq x;
    x.s = s;
    x.r = attn_range<KEYS>(p, x.s, 0, x.s.n - 1);
    x.r.blocks = max(x.r.blocks, 1);                   // a row that sees nothing is written too
    const int rows = x.s.n * p.G;
    x.tiles = FEW == (rows >= p.rows_from) ? 0 : (rows + ROWS - 1) / ROWS;
    return x;
  }
  // b the same for all lanes
  __device__ __forceinline__ Seq seq(const AttnArgs& p, int b) const {
    if (per > 1) return seq_of(p, attn_seq(p, b));
    return seq_of(p, {__builtin_amdgcn_readlane(lanes.q0, b), __builtin_amdgcn_readlane(lanes.n, b), __builtin_amdgcn_readlane(lanes.first, b),
                      __builtin_amdgcn_readlane(lanes.cap, b)});
  }
  static __device__ __forceinline__ Num work(const AttnArgs& p, const Seq& x) { return (Num)x.tiles * p.Hkv * (x.r.blocks + ITEM); }

  static __device__ __forceinline__ int from_lane(int v, int lane) { return __shfl(v, lane, 64); }
  static __device__ __forceinline__ long long from_lane(long long v, int lane) {
    return (long long)(uint32_t)__shfl((int)v, lane, 64) | (long long)__shfl((int)(v >> 32), lane, 64) << 32;
  }

  // The same for all lanes: the tiles kernel's addresses have to be scalars, the rows kernel has none to spare.
  static __device__ __forceinline__ int uniform(int v) { return FEW ? v : __builtin_amdgcn_readfirstlane(v); }
  static __device__ __forceinline__ long long uniform(long long v) {
    if (FEW) return v;
    return (long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) | (long long)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
  }

  // Every wavefront finds its share by itself.
  Num incl, before, total, share;                      // work up to, and in front of, this lane's sequences
  int per;
  AttnSeq lanes;                                       // per = 1: this lane's sequence
  __device__ __forceinline__ void plan(const AttnArgs& p, int groups) {
    const int lane = threadIdx.x & 63;
    per = (p.B + 63) / 64;
    Num mine = 0;
    bool wrong = false;                                // sequences that overlap: their work has no bound
    lanes = AttnSeq{};
    for (int i = 0; i < per; ++i) {
      const int b = lane * per + i;
      if (b >= p.B) continue;
      wrong |= p.cu[b] > p.cu[b + 1];
      lanes = attn_seq(p, b);
      mine += work(p, seq_of(p, lanes));
    }
    incl = mine;
    for (int d = 1; d < 64 && d < p.B; d <<= 1) {
      const Num up = from_lane(incl, lane >= d ? lane - d : lane);
      if (lane >= d) incl += up;
    }
    before = incl - mine;
    total = uniform(from_lane(incl, (p.B - 1) / per)); // the last lane with sequences; those behind it have not added all up
    if (__builtin_amdgcn_ballot_w64(wrong)) total = 0;
    // However small: told a length far above the real one, a token of 100, 700 and 2000 keys with heads of 128 takes 10.9, 12.2 and 14.3 us; with shares of
    // at least 2 units 11.8, 13.4 and 13.8, of 5 14.2, 15.7 and 16.9.  Of tiles 40 tokens of 300 and 1000 17.9 and 23.7 us, with at least 9 units 23.2 and 30.3.
    share = uniform((total + groups - 1) / groups);
  }
  // Blocks begin .. end - 1 of the work are workgroup w's; none: begin = end
  __device__ __forceinline__ void of(int w, Num& begin, Num& end) const {
    begin = uniform(share == 0 || (Num)w > total / share ? total : share * (Num)w);
    end = uniform(total - begin < share ? total : begin + share);
  }
  // The sequence with block `at` of the work, and the place of the block in it.  at < total.
  __device__ __forceinline__ void find(const AttnArgs& p, Num at, int& b, Num& in) const {
    const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(at < incl));
    Num rest = at - from_lane(before, owner);
    b = owner * per;
    for (; per > 1 && b + 1 < p.B; ++b) {
      const Num n = work(p, seq(p, b));
      if (rest < n) break;
      rest -= n;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    in = uniform(rest);
  }
  struct Item { int tile, head, rows, unit; };         // unit: of the tile; its first ITEM are none of its blocks
  static __device__ __forceinline__ Item item(const AttnArgs& p, const Seq& x, Num in) {
    const int each = x.r.blocks + ITEM;
    const int n = __builtin_amdgcn_readfirstlane((int)(in / each));
    Item y;
    y.unit = __builtin_amdgcn_readfirstlane((int)(in - (Num)n * each));
    y.tile = n / p.Hkv;
    y.head = n - y.tile * p.Hkv;
    y.rows = min(ROWS, x.s.n * p.G - y.tile * ROWS);
    return y;
  }
  // How many parts are to be joined at the cut in front of share w, at `at`: those of the tile whose blocks it goes through, if it is the first that does
  __device__ __forceinline__ int parts_at(int w, Num at, const Seq& x, const Item& y) const {
    const Num begin = at - y.unit + ITEM;              // of the tile's blocks
    if (at <= begin || ((Num)w - 1) * share > begin) return 0;
    return 1 + (int)((begin + x.r.blocks - 1) / share - (w - 1));
  }
  // Behind what a workgroup did of a sequence (`in`): on to the next one with work
  __device__ __forceinline__ void advance(const AttnArgs& p, const Seq& x, bool more, int& b, Num& in) const {
    if (in < work(p, x)) return;
    in = 0;
    do ++b;
    while (b + 1 < p.B && more && work(p, seq(p, b)) == 0);
  }
};

// Parts: two per workgroup, the one that it continues and the one that it begins; ROWS x D sums, then m and l.  Behind all of them, for the cut in front of
// each share, how many parts are to be joined there (0: none), and the tile.
template <int D, int ROWS> constexpr int kPart = ROWS * (D + 2);
template <int D, int ROWS> __device__ __forceinline__ float* attn_part(const AttnArgs& p, int w, bool begins) {
  return p.part + ((size_t)w * 2 + begins) * kPart<D, ROWS>;
}
template <int D, int ROWS> __device__ __forceinline__ i32x4* attn_cuts(const AttnArgs& p, int groups) {
  return (i32x4*)(p.part + (size_t)groups * 2 * kPart<D, ROWS>);
}
constexpr long long attn_parts_bytes(int groups, int D, int rows) { return (long long)groups * (2LL * rows * (D + 2) * 4 + 16); }
// Row `row` of a sequence's kv head in out
__device__ __forceinline__ long long attn_row(const AttnArgs& p, int q0, int head, int row) {
  const int t = row / p.G;
  return (long long)(q0 + t) * p.Hq + head * p.G + row - t * p.G;
}

// ---- joining parts ------------------------------------------------------------------------------
// A workgroup of THREADS threads makes `rows` rows of out from `parts` parts of each: sums(i, row) points to the D sums of part i, ml(i, row)
// to its m and l (m = -inf: the part has no sums), to(row) to the row of out.  A thread has four columns of a row; where threads are left over they
// share a row's parts, and what they have meets in LDS.  All loads of four parts are under way together.
constexpr int kJoinRows = 8;                          // of a workgroup
template <class Act, int D, int THREADS, class Sums, class Ml, class To>
__device__ __forceinline__ void attn_join(const AttnArgs& p, int rows, int parts, Sums sums, Ml ml, To to) {
  constexpr int Q = D / 4, PLACES = THREADS / Q;         // threads of a row; rows, or shares of rows, at a time
  __shared__ f32x4 part_o[THREADS];
  __shared__ f32x2 part_ml[PLACES];
  const int col = threadIdx.x % Q * 4, place = threadIdx.x / Q;
  int share = 1;
  while (2 * share * rows <= PLACES && 2 * share <= parts) share *= 2;
  for (int row0 = 0; row0 < rows; row0 += PLACES / share) {
    const int row = row0 + place / share, who = place % share;
    float m = -__builtin_inff(), sum = 0.f;
    f32x4 o = {};
    if (row < rows)
      for (int i = who; i < parts; i += 4 * share) {
        f32x2 a[4];
        f32x4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = i + j * share < parts ? i + j * share : i;
          a[j] = *(const f32x2*)ml(at, row);
          x[j] = *(const f32x4*)(sums(at, row) + col);
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (i + j * share >= parts) a[j] = f32x2{-__builtin_inff(), 0.f};
          top = fmaxf(top, a[j][0]);
        }
        if (top == -__builtin_inff()) {                // nothing but rows that see nothing, or see NaN alone
#pragma unroll
          for (int j = 0; j < 4; ++j) sum += a[j][1];
          continue;
        }
        const float f = attn_moved(p, m, top);
        sum *= f;
        o *= f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float g = attn_moved(p, a[j][0], top);
          sum += g * a[j][1];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] += a[j][0] == -__builtin_inff() ? 0.f : g * x[j][e];
        }
        m = top;
      }
    if (share > 1) {
      __syncthreads();
      part_o[threadIdx.x] = o;
      if (col == 0) part_ml[place] = f32x2{m, sum};
      __syncthreads();
      if (who == 0 && row < rows) {
        float top = m;
        for (int j = 1; j < share; ++j) top = fmaxf(top, part_ml[place + j][0]);
        float f = top == -__builtin_inff() ? 1.f : attn_moved(p, m, top);
        sum *= f;
        o *= f;
        for (int j = 1; j < share; ++j) {
          const f32x2 b = part_ml[place + j];
          f = top == -__builtin_inff() ? 1.f : attn_moved(p, b[0], top);
          sum += f * b[1];
          o += f * part_o[threadIdx.x + j * Q];
        }
      }
    }
    if (who == 0 && row < rows) {
      const float f = sum == 0.f ? 0.f : 1.f / sum;
      typedef __attribute__((ext_vector_type(4))) typename Act::elem e4;
      e4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = Act::from_f32(sum != sum ? sum : o[e] * f);
      *(e4*)((typename Act::elem*)to(row) + col) = y;
    }
  }
}

// Workgroup w, y joins rows 8 y .., and every 8 gridDim.y further, of the tile that the cut in front of share w + 1 goes through.
template <class Act, int D, int ROWS, int THREADS>
__global__ __launch_bounds__(THREADS) void attn_join_kernel(const AttnArgs p, int groups) {
  const int w = blockIdx.x + 1;
  const i32x4 cut = attn_cuts<D, ROWS>(p, groups)[w];  // parts, first token, tile, kv head and rows
  const int rows = cut[3] & 511;
  if (!cut[0]) return;
  // the first part is the one that share w - 1 began, the others those that a share continued
  auto part = [&](int i) { return attn_part<D, ROWS>(p, w - 1 + i, i == 0); };
  for (int row0 = blockIdx.y * kJoinRows; row0 < rows; row0 += gridDim.y * kJoinRows)
    attn_join<Act, D, THREADS>(
        p, min(kJoinRows, rows - row0), cut[0], [&](int i, int row) { return part(i) + (row0 + row) * D; },
        [&](int i, int row) { return part(i) + ROWS * D + 2 * (row0 + row); },
        [&](int row) { return (typename Act::elem*)p.out + attn_row(p, cut[1], cut[3] >> 9, cut[2] * ROWS + row0 + row) * D; });
}
template <class Act, int D, int ROWS, int THREADS>
static inline int launch_join(const AttnArgs& p, int groups, int rows, hipStream_t st) {
  if (groups == 1) return MI_OK;
  const dim3 grid(groups - 1, (rows + kJoinRows - 1) / kJoinRows);
  attn_join_kernel<Act, D, ROWS, THREADS><<<grid, THREADS, 0, st>>>(p, groups);
  return launch_status();
}

constexpr int kFewRows = 32;                          // a tile of the rows kernel
int launch_attn_rows(const AttnArgs& p, int D, int act_dtype, hipStream_t st);       // and what joins the parts
int launch_attn_tiles(const AttnArgs& p, int D, int act_dtype, hipStream_t st);
constexpr int attn_tile_rows(int D) { return D == 256 ? 128 : 256; }

}  // namespace qlin
