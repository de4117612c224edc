// Attention of many rows per sequence (prompts, chunks, large trees): a workgroup has 256 rows of a kv head (128 with heads of 256), 32 a wavefront, and
// all of its wavefronts use the same keys and values, which come to LDS a block ahead.
//
// Where there are few tiles, their keys are cut into `splits` parts; a second launch joins them.  Tiles of the last tokens, which see
// the most keys, go first; the kv heads go round the XCDs, so that the tiles of a head share its keys in L2.
//
// Bound: the matrix cores; for a few hundred rows HBM.
#include "attention.hpp"

namespace qlin {

template <int D> struct TilesCfg {
  static constexpr int ROWS = attn_tile_rows(D), NW = ROWS / 32;
  static constexpr int KEYS = D == 256 ? 32 : 64;      // of a step
  static constexpr int HALF = KEYS * D * 2;            // K or V of a step
  static constexpr int LDS = 2 * 2 * HALF;
};

// Slot i of the grid is tile i - start(b) of the sequence b with start(b) <= i < start(b + 1), start(b) = floor(cu[b] G / rows) + b: at least as many
// slots as a sequence has tiles.  64 sequences are looked at at a time.
struct TileOf { int b, tile; };
template <int ROWS>
__device__ __forceinline__ TileOf tile_of(const AttnArgs& p, int slot) {
  const int lane = threadIdx.x & 63;
  auto start = [&](int b) { return (int)((long long)min(max(p.cu[b], 0), p.T) * p.G / ROWS) + b; };
  int lo = 0, n = p.B;                                 // the sequence is one of lo .. lo + n - 1
  while (n > 1) {
    const int step = (n + 63) / 64, b = lo + lane * step;
    const uint64_t in = __builtin_amdgcn_ballot_w64(lane * step < n && start(min(b, p.B - 1)) <= slot);
    const int k = in ? 63 - __builtin_clzll(in) : 0;
    lo += k * step;
    n = min(step, n - k * step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  return {lo, slot - start(lo)};
}

struct Tile {
  AttnSeq s;
  AttnRange r;
  int b, row0, rows;           // row0: of the sequence
};
// false: no such tile, or its sequence belongs to the rows kernel
template <int ROWS, int KEYS>
__device__ __forceinline__ bool tile_at(const AttnArgs& p, int slot, Tile& x) {
  const TileOf at = tile_of<ROWS>(p, slot);
  x.b = at.b;
  x.s = attn_seq(p, at.b);
  const int all = x.s.n * p.G;
  x.row0 = at.tile * ROWS;
  x.rows = min(ROWS, all - x.row0);
  if (at.tile < 0 || x.rows <= 0 || all < p.rows_from) return false;
  x.r = attn_range<KEYS>(p, x.s, x.row0 / p.G, (x.row0 + x.rows - 1) / p.G);
  return true;
}

// Parts: sums [splits][T Hq][D], then m and l [splits][T Hq][2]
__device__ __forceinline__ float* part_sums(const AttnArgs& p, int D, int split, long long row) {
  return p.part + ((long long)split * p.T * p.Hq + row) * D;
}
__device__ __forceinline__ float* part_ml(const AttnArgs& p, int D, int split, long long row) {
  return p.part + (long long)p.splits * p.T * p.Hq * D + ((long long)split * p.T * p.Hq + row) * 2;
}

template <class Act, int D>
__global__ __launch_bounds__(64 * TilesCfg<D>::NW, D == 256 ? 1 : 2) void attn_tiles_kernel(const AttnArgs p) {
  using C = TilesCfg<D>;
  constexpr int KEYS = C::KEYS, NW = C::NW, OWN = KEYS / NW;   // rows of a block that a wavefront loads
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv, split = rest % p.splits, slot = p.slots - 1 - rest / p.splits;
  Tile x;
  if (!tile_at<C::ROWS, KEYS>(p, slot, x)) return;
  const int32_t* table = p.table + (size_t)x.b * p.width;
  const int first = (int)((long long)x.r.blocks * split / p.splits), last = (int)((long long)x.r.blocks * (split + 1) / p.splits);

  const int r = x.row0 + wave * 32 + (lane & 31), t = r / p.G;
  const bool has = wave * 32 + (lane & 31) < x.rows;
  const int wr0 = x.row0 + wave * 32, wr1 = min(wr0 + 31, x.row0 + x.rows - 1);
  const bool live = wr0 <= wr1;
  const int t0 = wr0 / p.G, t1 = max(wr1, wr0) / p.G;
  const int64_t* tree = p.tree ? p.tree + (size_t)(x.s.q0 + (has ? t : 0)) * p.tree_words : nullptr;
  AttnRows<Act, D> a;
  a.start();
  a.load_q(has ? (const typename Act::elem*)p.q + (x.s.q0 + t) * p.q_token + (head * p.G + r - t * p.G) * p.q_head : nullptr);

  const int key = lane % KEYS;
  auto lookup = [&](int i) { return i < last ? attn_lookup(p, table, x.r, attn_key<KEYS>(x.r, i) + key) : -1; };
  auto place = [&](int page, int i) { return i < last ? attn_place(p, page, attn_key<KEYS>(x.r, i) + key, head) : kNoRow; };
  constexpr uint64_t ALL = KEYS == 64 ? ~0ull : (1ull << KEYS) - 1;
  auto request = [&](uint32_t at16, int slot_of) {
    unsigned char* to = smem + slot_of * 2 * C::HALF + wave * OWN * D * 2;
    attn_load<D, OWN>(p.k, p.v, at16, wave * OWN, to, to + C::HALF);
  };

  int page = lookup(first);
  uint32_t at16 = place(page, first);
  page = lookup(first + 1);
  uint64_t there = __builtin_amdgcn_ballot_w64(at16 != kNoRow) & ALL;
  request(at16, 0);
  for (int i = first; i < last; ++i) {
    const int u = (i - first) & 1;
    wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const uint64_t now = there;
    at16 = place(page, i + 1);
    page = lookup(i + 2);
    there = __builtin_amdgcn_ballot_w64(at16 != kNoRow) & ALL;
    if (i + 1 < last) request(at16, u ^ 1);
    const int kb = attn_key<KEYS>(x.r, i);
    // nothing to do where no row of the wavefront sees the block: behind its last token, or in front of its window
    bool some = live;
    if (!p.tree) some = live && kb <= x.s.first + t1 && (!p.window || kb + KEYS - 1 > x.s.first + t0 - p.window || kb < p.sinks);
    if (!some) continue;
    const bool full = now == ALL && attn_all_seen<KEYS>(p, x.s.first, t0, t1, kb);
    uint64_t mask = now;
    if (!full) mask &= attn_sees(p, x.s.first, t, tree, kb);
    const unsigned char* kv = smem + u * 2 * C::HALF;
    a.template block<KEYS>(kv, kv + C::HALF, full, mask, p.c);
  }

  if (!has) return;
  const Halves ls = both_halves(a.l);
  const float l = ls.low + ls.high;
  const long long row = (long long)(x.s.q0 + t) * p.Hq + head * p.G + r - t * p.G;
  if (p.splits == 1) {
    const float f = l == 0.f ? 0.f : 1.f / l;
    typedef __attribute__((ext_vector_type(4))) typename Act::elem e4;
    typename Act::elem* to = (typename Act::elem*)p.out + row * D + (lane >> 5) * 4;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        e4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = Act::from_f32(a.o[d][i + e] * f);
        *(e4*)(to + d * 32 + i * 2) = y;
      }
    return;
  }
  if (lane < 32) *(f32x2*)part_ml(p, D, split, row) = f32x2{a.m, l};
  if (first == last) return;                           // the sums of an empty part are not read
  float* to = part_sums(p, D, split, row) + (lane >> 5) * 4;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) *(f32x4*)(to + d * 32 + i * 2) = f32x4{a.o[d][i], a.o[d][i + 1], a.o[d][i + 2], a.o[d][i + 3]};
}

// A workgroup per slot and kv head.
template <class Act, int D>
__global__ __launch_bounds__(256) void attn_tiles_join_kernel(const AttnArgs p) {
  const int head = blockIdx.x % p.Hkv, slot = blockIdx.x / p.Hkv;
  Tile x;
  if (!tile_at<TilesCfg<D>::ROWS, TilesCfg<D>::KEYS>(p, slot, x)) return;
  for (int idx = threadIdx.x; idx < x.rows * (D / 4); idx += 256) {
    const int r = x.row0 + idx / (D / 4), col = idx % (D / 4) * 4, t = r / p.G;
    const long long row = (long long)(x.s.q0 + t) * p.Hq + head * p.G + r - t * p.G;
    float m = -__builtin_inff(), sum = 0.f;
    for (int i = 0; i < p.splits; ++i) m = fmaxf(m, part_ml(p, D, i, row)[0]);
    const float top = m == -__builtin_inff() ? 0.f : m;
    f32x4 o = {};
    for (int i = 0; i < p.splits; ++i) {
      if ((long long)x.r.blocks * i / p.splits == (long long)x.r.blocks * (i + 1) / p.splits) continue;
      const f32x2 ml = *(const f32x2*)part_ml(p, D, i, row);
      const float f = __builtin_amdgcn_exp2f(ml[0] - top);
      sum += f * ml[1];
      o += f * *(const f32x4*)(part_sums(p, D, i, row) + col);
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    typedef __attribute__((ext_vector_type(4))) typename Act::elem e4;
    e4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = Act::from_f32(o[e] * f);
    *(e4*)((typename Act::elem*)p.out + row * D + col) = y;
  }
}

template <class Act, int D>
static int launch(const AttnArgs& p, hipStream_t st) {
  static std::atomic<unsigned long long> raised{0};
  const int rc = int8_raise_lds(attn_tiles_kernel<Act, D>, raised, TilesCfg<D>::LDS);
  if (rc != MI_OK) return rc;
  attn_tiles_kernel<Act, D><<<(unsigned)(p.slots * p.splits * p.Hkv), 64 * TilesCfg<D>::NW, TilesCfg<D>::LDS, st>>>(p);
  if (p.splits > 1) attn_tiles_join_kernel<Act, D><<<(unsigned)(p.slots * p.Hkv), 256, 0, st>>>(p);
  return launch_status();
}

int launch_attn_tiles(const AttnArgs& p, int D, int act_dtype, hipStream_t st) {
  if (act_dtype == DT_F16) return D == 64 ? launch<ActF16, 64>(p, st) : D == 128 ? launch<ActF16, 128>(p, st) : launch<ActF16, 256>(p, st);
  return D == 64 ? launch<ActBF16, 64>(p, st) : D == 128 ? launch<ActBF16, 128>(p, st) : launch<ActBF16, 256>(p, st);
}

}  // namespace qlin
