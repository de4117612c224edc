// Attention of many rows per sequence (prompts, chunks, large trees): a workgroup of eight wavefronts has 256 rows of a kv head (four and 128 with heads
// of 256), 32 a wavefront, which all use the same keys and values.
//
// A block of 64 keys is two steps.  While the scores of the next step's keys are on the matrix cores, the vector units make weights of this
// step's; then the product with the values goes along with the maximum of the next step's scores.  Keys come to LDS two blocks ahead, values one.
//
// Where there are few tiles, their keys are cut into `splits` parts; a second launch joins them.  Tiles of the last tokens, which see
// the most keys, go first; the kv heads go round the XCDs, so that the tiles of a head share its keys in L2.
//
// Bound: the matrix cores; for a few hundred rows HBM.
#include "attention.hpp"

namespace qlin {

template <int D> struct TilesCfg {
  static constexpr int ROWS = attn_tile_rows(D), NW = ROWS / 32;
  static constexpr int KEYS = D == 256 ? 32 : 64;      // of a block: a step or two
  static constexpr int HALF = KEYS * D * 2;            // K or V of a block
  static constexpr int AHEAD = KEYS == 64 ? 2 : 3;     // how many blocks ahead keys are asked for: two steps are there when a block begins
  static constexpr int PAGES = (AHEAD + 1 + 2) * HALF; // behind the rings of keys and values
  static constexpr int LDS = PAGES + NW * 2 * 4 * KEYS;          // two blocks' pages per wavefront
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
__global__ __launch_bounds__(64 * TilesCfg<D>::NW) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2, D == 256 ? 1 : 2))) void attn_tiles_kernel(const AttnArgs p) {
  using C = TilesCfg<D>;
  constexpr int KEYS = C::KEYS, NW = C::NW, OWN = KEYS / NW, AHEAD = C::AHEAD;     // OWN: rows of a block that a wavefront loads
  using Rows = AttnRows<Act, D, 32, 1>;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv, split = rest % p.splits, slot = p.slots - 1 - rest / p.splits;
  Tile x;
  if (!tile_at<C::ROWS, KEYS>(p, slot, x)) return;
  const int32_t* table = p.table + (size_t)x.b * p.width;
  const int first = (int)((long long)x.r.blocks * split / p.splits), last = (int)((long long)x.r.blocks * (split + 1) / p.splits);

  // the wavefront's rows wr0 .. wr1 of the sequence, tokens t0 .. t1
  const int wr0 = x.row0 + wave * 32, wr1 = min(wr0 + 32, x.row0 + x.rows) - 1;
  const int t0 = wr0 / p.G, t1 = max(wr1, wr0) / p.G;
  const int r = wr0 + (lane & 31), t = r / p.G;
  const bool has = r <= wr1;
  Rows a;
  a.start();
  a.load_q(0, has ? (const typename Act::elem*)p.q + (x.s.q0 + t) * p.q_token + (head * p.G + r - t * p.G) * p.q_head : nullptr);

  // pages of the keys of block i: by direct loads to LDS like the keys, a block ahead of what is asked for with them
  const unsigned char* pages = smem + C::PAGES + wave * (2 * 4 * KEYS);
  auto key_of = [&](int i) { return attn_key<KEYS>(x.r, i); };
  auto lookup = [&](int i, int u) {
    const int key = key_of(i) + lane % KEYS;
    if (KEYS == 64 || lane < KEYS) to_lds4(i < last && attn_in(p, x.r, key) ? table + attn_page_of(p, key) : kNoPage, lds_address(pages + u * 4 * KEYS));
  };
  using Places = RowPlaces<D, OWN>;
  auto place = [&](int i, int u, Places& to) {         // and which keys of the block are there
    const int page = *(const int*)(pages + u * 4 * KEYS + lane % KEYS * 4);
    const uint32_t at = i < last ? attn_place(p, page, key_of(i) + lane % KEYS, head) : kNoRow;
    to.take(at, wave * OWN);
    return __builtin_amdgcn_ballot_w64(at != kNoRow);
  };
  constexpr int OFFSET = OWN * D * 2;

  // Whether the wavefront has something to do with block i, and whether all of its rows see all of it
  auto some_of = [&](int i) {
    if (i >= last || wr0 > wr1) return false;
    const int kb = key_of(i);
    return p.tree || (kb <= x.s.first + t1 && (!p.window || kb + KEYS - 1 > x.s.first + t0 - p.window || kb < p.sinks));
  };
  auto full_of = [&](int i, uint64_t there) { return there == ~0ull && attn_all_seen<KEYS>(p, x.s.first, t0, t1, key_of(i)); };
  auto mask_of = [&](int i, uint64_t there, int half) {
    const int64_t* tree = p.tree ? p.tree + (size_t)(x.s.q0 + (has ? t : 0)) * p.tree_words : nullptr;
    typename Rows::Mask mask;
    mask.of[0] = (there & attn_sees(p, x.s.first, t, tree, key_of(i))) >> (32 * half) & 0xFFFFFFFFull;
    return mask;
  };

  if (first < last) {
    unsigned char* k[AHEAD + 1];                       // keys of blocks i, i + 1 ..
    unsigned char *v0 = smem + (AHEAD + 1) * C::HALF, *v1 = v0 + C::HALF;        // values of blocks i, i + 1
    Places at[AHEAD];                                  // of blocks i + 1 ..
    uint64_t there[AHEAD + 1];                         // keys of blocks i ..
    lookup(first, 0);
    lookup(first + 1, 1);
    wait_loads<0>();
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      k[j] = smem + j * C::HALF;
      Places& to = at[j ? j - 1 : 0];
      there[j] = place(first + j, j & 1, to);
      to.template load<true>(p.k, wave * OWN, k[j] + wave * OFFSET);
      if (j == 0) to.template load<false>(p.v, wave * OWN, v0 + wave * OFFSET);
      lookup(first + j + 2, j & 1);
      if (j >= 1 && j + 1 < AHEAD) wait_loads<0>();
    }
    k[AHEAD] = smem + AHEAD * C::HALF;
    bool some = some_of(first), full = some && full_of(first, there[0]), some1, full1;
    typename Rows::Scores s0, s1;                      // of the two steps of a block (one: s0)
    typename Rows::Weights w;
    float top[1];
    wait_loads<0>();
    there[AHEAD] = place(first + AHEAD, AHEAD & 1, at[AHEAD - 1]);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (some) {
      a.scores(k[0], s0);
      if (!full) a.hide(s0, mask_of(first, there[0], 0));
      a.largest(s0, p.c, top);
      a.follow(top);
    }
    int i = first, u = AHEAD & 1;
    // what a block begins with: its values and the next two steps' keys are there, more of both are asked for
    auto begin = [&]() __attribute__((always_inline)) {
      wait_loads<0>();
      __builtin_amdgcn_s_barrier();                    // everyone's; and block i - 1's are done with
      asm volatile("" ::: "memory");
      if (i + 1 < last) at[0].template load<false>(p.v, wave * OWN, v1 + wave * OFFSET);
      if (i + AHEAD < last) at[AHEAD - 1].template load<true>(p.k, wave * OWN, k[AHEAD] + wave * OFFSET);
      lookup(i + AHEAD + 2, u);
      some1 = some_of(i + 1);
      full1 = some1 && full_of(i + 1, there[1]);
    };
    auto next = [&]() __attribute__((always_inline)) { // the places of one block more, while products go on
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) there[j] = there[j + 1];
#pragma unroll
      for (int j = 0; j + 1 < AHEAD; ++j) at[j] = at[j + 1];
      u ^= 1;
      there[AHEAD] = place(i + AHEAD + 1, u, at[AHEAD - 1]);
    };
    auto end = [&]() __attribute__((always_inline)) {
      unsigned char* to = k[0];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) k[j] = k[j + 1];
      k[AHEAD] = to;
      to = v0;
      v0 = v1;
      v1 = to;
      some = some1;
      full = full1;
      ++i;
    };
    for (;;) {
      begin();
      if (full && full1) {                             // all rows see all of this block and of the next
        typename Rows::Keys f;
        a.read_keys(KEYS == 64 ? k[0] + 64 * D : k[1], f);
        do {
          if constexpr (KEYS == 64) {
            a.step(s0, v0, f, k[1], p.c, s1, top);
            next();
            a.step(s1, v0 + 64 * D, f, k[1] + 64 * D, p.c, s0, top);
          } else {
            a.step(s0, v0, f, k[2], p.c, s1, top);
            next();
            s0 = s1;
          }
          end();
          begin();                                     // there is a next block
        } while (full && full1);
      }
      const uint64_t now = there[0];
      next();
      if (some) {
        typename Rows::Mask mask = mask_of(i, now, 0);
        a.weigh(s0, p.c, w);
        a.add_hidden(v0, w, mask);
        if constexpr (KEYS == 64) {
          mask = mask_of(i, now, 1);
          a.scores(k[0] + 64 * D, s1);
          a.hide(s1, mask);
          a.largest(s1, p.c, top);
          a.follow(top);
          a.weigh(s1, p.c, w);
          a.add_hidden(v0 + 64 * D, w, mask);
        }
      }
      if (some1) {
        a.scores(k[1], s0);
        if (!full1) a.hide(s0, mask_of(i + 1, there[0], 0));
        a.largest(s0, p.c, top);
        a.follow(top);
      }
      end();
      if (i >= last) break;
    }
  }

  const Halves ls = both_halves(a.l[0]);
  const float l = ls.low + ls.high;
  if (!has) return;
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
        for (int e = 0; e < 4; ++e) y[e] = Act::from_f32(a.o[0][d][i + e] * f);
        *(e4*)(to + d * 32 + i * 2) = y;
      }
    return;
  }
  if (lane < 32) *(f32x2*)part_ml(p, D, split, row) = f32x2{a.m[0], l};
  if (first == last) return;                           // m = -inf: the sums are not read
  float* to = part_sums(p, D, split, row) + (lane >> 5) * 4;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *(f32x4*)(to + d * 32 + i * 2) = f32x4{a.o[0][d][i], a.o[0][d][i + 1], a.o[0][d][i + 2], a.o[0][d][i + 3]};
}

// A workgroup per 32 rows of a slot and kv head.
template <class Act, int D>
__global__ __launch_bounds__(kJoin) void attn_tiles_join_kernel(const AttnArgs p) {
  using C = TilesCfg<D>;
  const int piece = blockIdx.x % C::NW, rest = blockIdx.x / C::NW, head = rest % p.Hkv, slot = rest / p.Hkv;
  Tile x;
  if (!tile_at<C::ROWS, C::KEYS>(p, slot, x) || piece * 32 >= x.rows) return;
  auto row_of = [&](int row) {
    const int r = x.row0 + piece * 32 + row, t = r / p.G;
    return (long long)(x.s.q0 + t) * p.Hq + head * p.G + r - t * p.G;
  };
  attn_join<Act, D>(min(32, x.rows - piece * 32), p.splits, [&](int i, int row) { return part_sums(p, D, i, row_of(row)); },
                    [&](int i, int row) { return part_ml(p, D, i, row_of(row)); },
                    [&](int row) { return (typename Act::elem*)p.out + row_of(row) * D; });
}

template <class Act, int D>
static int launch(const AttnArgs& p, hipStream_t st) {
  static std::atomic<unsigned long long> raised{0};
  const int rc = int8_raise_lds(attn_tiles_kernel<Act, D>, raised, TilesCfg<D>::LDS);
  if (rc != MI_OK) return rc;
  attn_tiles_kernel<Act, D><<<(unsigned)(p.slots * p.splits * p.Hkv), 64 * TilesCfg<D>::NW, TilesCfg<D>::LDS, st>>>(p);
  if (p.splits > 1) attn_tiles_join_kernel<Act, D><<<(unsigned)(p.slots * p.Hkv * TilesCfg<D>::NW), kJoin, 0, st>>>(p);
  return launch_status();
}

int launch_attn_tiles(const AttnArgs& p, int D, int act_dtype, hipStream_t st) {
  if (act_dtype == DT_F16) return D == 64 ? launch<ActF16, 64>(p, st) : D == 128 ? launch<ActF16, 128>(p, st) : launch<ActF16, 256>(p, st);
  return D == 64 ? launch<ActBF16, 64>(p, st) : D == 128 ? launch<ActBF16, 128>(p, st) : launch<ActBF16, 256>(p, st);
}

}  // namespace qlin
