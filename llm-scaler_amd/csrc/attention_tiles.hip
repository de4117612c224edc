// Attention of many rows per sequence (prompts, chunks, large trees): a workgroup of eight wavefronts has 256 rows of a kv head (four and 128 with heads
// of 256), 32 a wavefront, which all use the same keys and values.
//
// A step is 32 keys: while the scores of the next step's keys are on the matrix cores, the vector units make weights of this step's; then the product with
// the values goes along with the maximum of the next step's scores.  A block, what comes to LDS together, is two steps (one with heads of
// 256); keys come two blocks ahead (three), values one.  Where pages hold whole groups of 8 places (GROUPS), the keys that a wavefront loads
// lie on one page: their address is a scalar.
//
// Long prompts have a workgroup per tile: tiles of the last tokens, which see the most keys, go first, and the kv heads go round the XCDs, so that
// the tiles of a head share its keys in L2.  Few tokens over long contexts are done in equal shares instead.
//
// Bound: what a wavefront can issue beside the matrix instructions.  8192 tokens, 32 heads of 128 over 8: 560 us, 0.98 PFLOP/s, matrix pipe 47 % busy
// at 2.1 GHz (power); chunks, 16 heads of 256 over 2: 684 us, 0.87 PFLOP/s, 43 %; a window of 1024, 64 heads of 64 over 8: 413 us, 0.65 PFLOP/s, 35 %,
// vector instructions 73 % (the exponentials alone take as long as both products; 12 registers are put aside around the loop).  Each compared on one card, keys and
// values a block further ahead change nothing (699 against 694 us for the chunks, 560 against 556 for the prompt), nor does an order of instructions
// laid down by hand (696 against 694), nor four wavefronts with 64 rows each (copies between register files).
#include "attention.hpp"

#include <type_traits>

namespace qlin {

template <int D> struct TilesCfg {
  static constexpr int ROWS = attn_tile_rows(D), NW = ROWS / 32;
  static constexpr int KEYS = D == 256 ? 32 : 64;      // of a block: a step or two
  static constexpr int HALF = KEYS * D * 2;            // K or V of a block
  static constexpr int WAVES = D == 64 ? 4 : D == 128 ? 2 : 1;   // per SIMD
  static constexpr int AHEAD = KEYS == 64 ? 2 : 3;     // how many blocks ahead keys are asked for: two steps are there when a block begins
  static constexpr int FLAGS = (AHEAD + 1 + 2) * HALF; // behind the rings of keys and values: 8 x 8 and 8 words
  static constexpr int PAGES = FLAGS + 512;            // two blocks' pages per wavefront
  static constexpr int LDS = PAGES + NW * 2 * 4 * KEYS;
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

// Blocks first .. last - 1 of a tile, by a whole workgroup.  part: where sums, m and l go; null: the rows of out are finished.
template <class Act, int D, bool GROUPS>
__device__ __forceinline__ void tile_piece(const AttnArgs& p, const Tile& x, int head, int first, int last, float* part) {
  using C = TilesCfg<D>;
  constexpr int KEYS = C::KEYS, NW = C::NW, OWN = KEYS / NW, AHEAD = C::AHEAD;   // OWN: rows of a block that a wavefront loads
  static_assert(OWN == 8 && NW <= 8, "a group of 8 places per wavefront");
  using Rows = AttnRows<Act, D>;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t* table = p.table + (size_t)x.b * p.width;

  // the wavefront's rows wr0 .. wr1 of the sequence, tokens t0 .. t1
  const int wr0 = x.row0 + wave * 32, wr1 = min(wr0 + 32, x.row0 + x.rows) - 1;
  const int t0 = wr0 / p.G, t1 = max(wr1, wr0) / p.G;
  const bool live = wr0 <= wr1;
  const int r = wr0 + (lane & 31), t = r / p.G;
  const bool has = r <= wr1;
  Rows a;
  a.start();
  a.load_q(has ? (const typename Act::elem*)p.q + (x.s.q0 + t) * p.q_token + (head * p.G + r - t * p.G) * p.q_head : nullptr);

  auto key_of = [&](int i) { return attn_key<KEYS>(x.r, i); };
  constexpr uint64_t ALL = KEYS == 64 ? ~0ull : (1ull << (KEYS % 64)) - 1;
  constexpr int OFFSET = OWN * D * 2;

  // Where the wavefront's rows of a block lie: GROUPS: one place for all of them; otherwise a place per row, of pages that come by direct loads to LDS
  // like the keys, a block ahead of what is asked for with them
  using Places = std::conditional_t<GROUPS, uint32_t, RowPlaces<D, OWN>>;
  using Row = RowPlaces<D, OWN>;
  const uint32_t rings = lds_address(smem), pages = rings + C::PAGES + wave * (2 * 4 * KEYS);
  uint32_t* bad = (uint32_t*)(smem + C::FLAGS);        // [block % 8][wave]: its page is outside the cache
  uint32_t* dirty = bad + 64;                          // [wave]: it put zeros in place of values that some row sees
  uint32_t from_k[Row::N], from_v[Row::N];             // bytes from a group's first place
  if constexpr (GROUPS)
#pragma unroll
    for (int j = 0; j < Row::N; ++j) {
      const int g = j * Row::RPI + lane / Row::CH, row = wave * OWN + g;
      from_k[j] = g * p.row16 * 16 + ((lane % Row::CH) ^ k_swizzle<D>(row)) * 16;
      from_v[j] = g * p.row16 * 16 + ((lane % Row::CH) ^ v_swizzle<D>(row)) * 16;
    }
  // Blocks `inner` .. inner + inners - 1 hold keys that all rows of the tile see; where no page of the call is outside the cache nothing is looked up for
  // them but the page.
  const int tile0 = x.row0 / p.G, tile1 = (x.row0 + x.rows - 1) / p.G;
  int inner = 0, inners = 0, inners_then = 0;          // then: when all pages are known to be inside
  if constexpr (GROUPS) {
    const int from = max(x.r.lo, p.window ? x.s.first + tile1 - p.window + 1 : 0), to = p.tree ? min(x.r.hi, x.s.first) : min(x.r.hi, x.s.first + tile0 + 1);
    inner = max(x.r.head + (max(from - x.r.from, 0) + KEYS - 1) / KEYS, first);
    if (to > x.r.from) inners_then = max(min(x.r.head + (to - x.r.from) / KEYS, last) - inner, 0);
  }
  auto pages_wrong = [&]() {
    bool wrong = false;
    auto scan = [&](int a, int b) {                    // the pages of keys a .. b - 1
      if (a < b)
        for (int i = attn_page_of(p, a) + (int)threadIdx.x; i <= attn_page_of(p, b - 1); i += 64 * NW) wrong |= (uint32_t)table[i] >= (uint32_t)p.pages;
    };
    scan(first * KEYS, min(min(last, x.r.head) * KEYS, min(p.sinks, x.r.hi)));
    scan(max(x.r.lo, attn_key<KEYS>(x.r, max(first, x.r.head))), min(x.r.hi, attn_key<KEYS>(x.r, last - 1) + KEYS));
    return __builtin_amdgcn_ballot_w64(wrong) != 0;
  };
  const int inner_key = x.r.from + (inner - x.r.head) * KEYS;
  auto is_inner = [&](int i) { return GROUPS && (uint32_t)(i - inner) < (uint32_t)inners; };
  int page = 0;                                        // GROUPS: of the block whose place comes next
  auto lookup = [&](int i, int u, bool known = false) {
    if constexpr (GROUPS) {
      if (known || is_inner(i)) {
        page = scalar_load(table + attn_page_of(p, inner_key + (i - inner) * KEYS + wave * OWN));
        return;
      }
      const int key = key_of(i) + wave * OWN;
      const bool seen = i < last && key < x.r.hi && (key + OWN > x.r.lo || key < p.sinks);
      page = 0;
      if (seen) page = scalar_load(table + attn_page_of(p, key));          // a group that nothing sees: some place of the cache
    } else {
      const int key = key_of(i) + lane % KEYS;
      if (KEYS == 64 || lane < KEYS)
        to_lds4(i < last && attn_in(p, x.r, key) ? table + attn_page_of(p, key) : kNoPage, pages + u * 4 * KEYS);
    }
  };
  // the place of block i, and which of its keys are there
  auto place = [&](int i, int u, Places& to, bool known = false) {
    if constexpr (GROUPS) {
      if (known || is_inner(i)) {
        const int key = inner_key + (i - inner) * KEYS + wave * OWN;
        to = (uint32_t)page * p.page16 + (uint32_t)(key - attn_page_of(p, key) * p.page) * p.row16 + (uint32_t)head * p.head16;
        return ALL;
      }
      const int key = key_of(i) + wave * OWN;
      const bool wrong = (uint32_t)page >= (uint32_t)p.pages;
      const bool seen = i < last && key < x.r.hi && (key + OWN > x.r.lo || key < p.sinks);
      const uint32_t in = wrong || !seen ? 0 : (uint32_t)page * p.page16 + (uint32_t)(key - attn_page_of(p, key) * p.page) * p.row16;
      to = in + (uint32_t)head * p.head16;
      if (lane == 0) bad[(i & 7) * 8 + wave] = wrong;
      return ALL;                                      // less what keys_there says when all wavefronts have written theirs
    } else {
      const int it = *in_lds<const int>(pages + u * 4 * KEYS + lane % KEYS * 4);
      const uint32_t at = i < last ? attn_place(p, it, key_of(i) + lane % KEYS, head) : kNoRow;
      to.take(at, wave * OWN);
      return (uint64_t)__builtin_amdgcn_ballot_w64(at != kNoRow) & ALL;
    }
  };
  auto keys_there = [&](int i) {                       // GROUPS
    if (is_inner(i)) return ALL;
    if (i >= last) return (uint64_t)0;
    const int kb = key_of(i);
    uint64_t m = low_bits(x.r.hi - kb) & (~low_bits(x.r.lo - kb) | low_bits(p.sinks - kb));
    uint64_t wrong = __builtin_amdgcn_ballot_w64(lane < NW && bad[(i & 7) * 8 + (lane & 7)]);
    for (; wrong; wrong &= wrong - 1) m &= ~(0xFFull << (8 * __builtin_ctzll(wrong)));
    return m & ALL;
  };
  auto request = [&](auto is_k, const Places& from, uint32_t to) {
    constexpr bool K = decltype(is_k)::value;
    to += wave * OFFSET;
    if constexpr (GROUPS) {
      const unsigned char* base = (const unsigned char*)(K ? p.k : p.v) + (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)from) * 16;
#pragma unroll
      for (int j = 0; j < Row::N; ++j) to_lds16_from(base, K ? from_k[j] : from_v[j], to + j * 1024);
    } else {
      from.template load<K>(K ? p.k : p.v, wave * OWN, to);
    }
  };
  const std::true_type K_;
  const std::false_type V_;

  auto full_of = [&](int i, uint64_t there) { return is_inner(i) || (there == ALL && attn_all_seen<KEYS>(p, x.s.first, t0, t1, key_of(i))); };
  auto edge_of = [&](int i, uint64_t there) { return !is_inner(i) && (there != ALL || !attn_all_seen<KEYS>(p, x.s.first, tile0, tile1, key_of(i))); };
  bool spoilt = false;
  auto mask_of = [&](int i, uint64_t there, int half) {
    int mine = has ? t : 0;
    asm volatile("" : "+v"(mine));                     // made here, not kept in registers all along
    const int64_t* tree = p.tree ? p.tree + (size_t)(x.s.q0 + mine) * p.tree_words : nullptr;
    return (uint32_t)(there >> (32 * half)) & attn_sees(p, x.s.first, mine, tree, key_of(i) + 32 * half);
  };

  if (first < last) {
    uint32_t k[AHEAD + 1];                             // where in LDS: keys of blocks i, i + 1 ..
    uint32_t v0 = rings + (AHEAD + 1) * C::HALF, v1 = v0 + C::HALF;              // values of blocks i, i + 1
    Places at[AHEAD];                                  // of blocks i + 1 ..
    uint64_t there[AHEAD + 1];                         // keys of blocks i .. (GROUPS: of i and i + 1)
    lookup(first, 0);
    if constexpr (!GROUPS) {
      lookup(first + 1, 1);
      wait_loads<0>();
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      k[j] = rings + j * C::HALF;
      Places& to = at[j ? j - 1 : 0];
      there[j] = place(first + j, j & 1, to);
      request(K_, to, k[j]);
      if (j == 0) request(V_, to, v0);
      if constexpr (GROUPS) {
        lookup(first + j + 1, 0);
      } else {
        lookup(first + j + 2, j & 1);
        if (j >= 1 && j + 1 < AHEAD) wait_loads<0>();
      }
    }
    k[AHEAD] = rings + AHEAD * C::HALF;
    f32x16 s0, s1;                                     // scores of the two steps of a block (one: s0)
    typename Rows::Keys f;
    if constexpr (GROUPS) {
      const bool wrong = pages_wrong();
      if (lane == 0) dirty[wave] = wrong;
    }
    wait_loads<0>();
    there[AHEAD] = place(first + AHEAD, AHEAD & 1, at[AHEAD - 1]);
    if constexpr (GROUPS) lookup(first + AHEAD + 1, 0);
    lds_barrier();
    if constexpr (GROUPS) {
      if (!__builtin_amdgcn_ballot_w64(lane < NW && dirty[lane & 7])) inners = inners_then;
      there[0] = keys_there(first);
    }
    bool full = full_of(first, there[0]);
    float most;                                        // the largest of the scores that were made last
    auto follow = [&](f32x16& s, bool all, int i, uint64_t keys, int half) __attribute__((always_inline)) {
      if (!all) {
        a.hide(s, mask_of(i, keys, half));
        most = a.largest(s);
      }
      a.follow(p, s, most);
    };
    if (live) {
      a.read_keys(k[0], f);
      s0 = a.scores(f);
      most = a.largest(s0);
      follow(s0, full, first, there[0], 0);
      a.read_keys(KEYS == 64 ? k[0] + 64 * D : k[1], f);
    }
    auto turn = [&]() __attribute__((always_inline)) { // the rings
      uint32_t to = k[0];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) k[j] = k[j + 1];
      k[AHEAD] = to;
      to = v0;
      v0 = v1;
      v1 = to;
    };
    int u = AHEAD & 1;
    for (int i = first; i < last; ++i) {
      if constexpr (GROUPS)
        // All blocks that are loaded or looked up meanwhile are inner ones: the same without a question.
        for (; live && i >= inner && i + AHEAD + 2 < inner + inners; ++i) {
          wait_loads<0>();
          lds_barrier();
          request(V_, at[0], v1);
          request(K_, at[AHEAD - 1], k[AHEAD]);
#pragma unroll
          for (int j = 0; j + 1 < AHEAD; ++j) at[j] = at[j + 1];
          place(i + AHEAD + 1, 0, at[AHEAD - 1], true);
          lookup(i + AHEAD + 2, 0, true);
          if constexpr (KEYS == 64) {
            s1 = a.step(p, s0, v0, f, k[1], most);
            a.follow(p, s1, most);
            s0 = a.step(p, s1, v0 + 64 * D, f, k[1] + 64 * D, most);
          } else {
            s0 = a.step(p, s0, v0, f, k[2], most);
          }
          a.follow(p, s0, most);
          turn();
        }
      // The block's values and the next two steps' keys are there; more of both are asked for.
      wait_loads<0>();
      // 0 times an infinity or a NaN would not be 0: in blocks that some row does not see all of, the wavefronts look for such among the values that they
      // loaded and put zeros there.
      if (edge_of(i, there[0])) spoilt |= Rows::template clean<Row::N>(v0 + wave * OFFSET, (uint32_t)(there[0] >> (wave * OWN)) & 0xFF);
      lds_barrier();                                   // everyone's; and block i - 1's are done with
      if (i + 1 < last) request(V_, at[0], v1);
      if (i + AHEAD < last) request(K_, at[AHEAD - 1], k[AHEAD]);
      if constexpr (!GROUPS) lookup(i + AHEAD + 2, u);
      const uint64_t now = there[0];
      auto next = [&]() __attribute__((always_inline)) {         // the places of one block more, while products go on
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) there[j] = there[j + 1];
#pragma unroll
        for (int j = 0; j + 1 < AHEAD; ++j) at[j] = at[j + 1];
        u ^= 1;
        there[AHEAD] = place(i + AHEAD + 1, u, at[AHEAD - 1]);
        if constexpr (GROUPS) {
          lookup(i + AHEAD + 2, 0);
          there[0] = keys_there(i + 1);
        }
      };
      bool full1;
      if (!live) {
        next();
        full1 = full_of(i + 1, there[0]);
      } else if constexpr (KEYS == 64) {
        s1 = a.step(p, s0, v0, f, k[1], most);
        follow(s1, full, i, now, 1);
        next();
        full1 = full_of(i + 1, there[0]);
        s0 = a.step(p, s1, v0 + 64 * D, f, k[1] + 64 * D, most);
        follow(s0, full1, i + 1, there[0], 0);
      } else {
        s0 = a.step(p, s0, v0, f, k[2], most);
        next();
        full1 = full_of(i + 1, there[0]);
        follow(s0, full1, i + 1, there[0], 0);
      }
      full = full1;
      turn();
    }
  }

  wait_loads<0>();                                     // nothing is on its way to LDS any more
  // Values that are no numbers, where zeros stood in for them and some row sees them: each goes to the rows that do, from the cache itself.
  if (first < last) {
    if (lane == 0) dirty[wave] = spoilt;
    lds_barrier();
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(lane < NW && dirty[lane & 7]) != 0, 0))
#pragma unroll 1
      for (int i = first; i < last; ++i) {
        const int kb = key_of(i), key = kb + lane % KEYS;
        const uint32_t place = attn_in(p, x.r, key) ? attn_place(p, table[attn_page_of(p, key)], key, head) : kNoRow;
        uint64_t there = __builtin_amdgcn_ballot_w64(place != kNoRow) & ALL;
        if (!edge_of(i, there)) continue;
        const int64_t* tree = p.tree ? p.tree + (size_t)(x.s.q0 + (has ? t : 0)) * p.tree_words : nullptr;
        const uint64_t sees = attn_sees(p, x.s.first, t, tree, kb) | (uint64_t)attn_sees(p, x.s.first, t, tree, kb + 32) << 32;
#pragma unroll 1
        for (; there; there &= there - 1) {
          const int j = __builtin_ctzll(there);
          const unsigned char* v = (const unsigned char*)p.v + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)place, j) * 16;
          a.add_not_finite(sees >> j & 1, [&](int column) { return *(const u16x4*)(v + column * 2); });
        }
      }
  }

  const Halves ls = both_halves(a.l);
  const float l = ls.low + ls.high;
  if (!has) return;
  if (!part) {
    const float f = l == 0.f ? 0.f : 1.f / l;
    typedef __attribute__((ext_vector_type(4))) typename Act::elem e4;
    typename Act::elem* to = (typename Act::elem*)p.out + attn_row(p, x.s.q0, head, r) * D + (lane >> 5) * 4;
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
  const int row = r - x.row0;
  if (lane < 32) *(f32x2*)(part + C::ROWS * D + 2 * row) = f32x2{a.reference(), l};
  float* to = part + row * D + (lane >> 5) * 4;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *(f32x4*)(to + d * 32 + i * 2) = f32x4{a.o[d][i], a.o[d][i + 1], a.o[d][i + 2], a.o[d][i + 3]};
}

template <class Act, int D, bool GROUPS>
__global__ __launch_bounds__(64 * TilesCfg<D>::NW) __attribute__((amdgpu_waves_per_eu(TilesCfg<D>::WAVES, TilesCfg<D>::WAVES)))
void attn_tiles_kernel(const AttnArgs p) {
  using C = TilesCfg<D>;
  Tile x;
  if (!tile_at<C::ROWS, C::KEYS>(p, p.slots - 1 - (int)(blockIdx.x / p.Hkv), x)) return;
  tile_piece<Act, D, GROUPS>(p, x, blockIdx.x % p.Hkv, 0, x.r.blocks, nullptr);
}

// In equal shares.  All tiles of a sequence have the blocks that any of its tokens sees.  66 to 71 scalar registers lie in lanes of vector registers: the
// shares' counts, read again between tiles, none in the loop over inner blocks.
template <class Act, int D, bool GROUPS>
__global__ __launch_bounds__(64 * TilesCfg<D>::NW) __attribute__((amdgpu_waves_per_eu(TilesCfg<D>::WAVES, TilesCfg<D>::WAVES)))
void attn_tiles_shared_kernel(const AttnArgs p) {
  using C = TilesCfg<D>;
  constexpr int kItem = 8;
  using Work = Shares<C::ROWS, C::KEYS, kItem, false, long long>;
  Work shares;
  shares.plan(p, p.shares);
  long long at, end, in;
  shares.of(blockIdx.x, at, end);
  i32x4* cut = attn_cuts<D, C::ROWS>(p, p.shares) + blockIdx.x;
  if (at >= end) {
    if (threadIdx.x == 0) *cut = i32x4{};
    return;
  }
  int b;
  shares.find(p, at, b, in);
  for (bool starts = true; at < end; starts = false) {
    const typename Work::Seq s = shares.seq(p, b);
    const typename Work::Item y = Work::item(p, s, in);
    if (starts && threadIdx.x == 0) *cut = i32x4{shares.parts_at(blockIdx.x, at, s, y), s.s.q0, y.tile, y.head << 9 | y.rows};
    const int take = __builtin_amdgcn_readfirstlane((int)min((long long)(s.r.blocks + kItem - y.unit), end - at));
    const int first = max(y.unit - kItem, 0), last = y.unit + take - kItem;
    at += take;
    in += take;
    if (last > first) {
      const Tile x{s.s, s.r, b, y.tile * C::ROWS, y.rows};
      const bool whole = first == 0 && last == s.r.blocks;
      tile_piece<Act, D, GROUPS>(p, x, y.head, first, last, whole ? nullptr : attn_part<D, C::ROWS>(p, blockIdx.x, first == 0));
      lds_barrier();                                   // before LDS is used for the next tile
    }
    shares.advance(p, s, at < end, b, in);
  }
}

template <class Act, int D, bool GROUPS>
static int launch_tiles(const AttnArgs& p, hipStream_t st) {
  static std::atomic<unsigned long long> raised{0}, raised_shared{0};
  constexpr int THREADS = 64 * TilesCfg<D>::NW, LDS = TilesCfg<D>::LDS;
  if (p.shares) {
    const int rc = int8_raise_lds(attn_tiles_shared_kernel<Act, D, GROUPS>, raised_shared, LDS);
    if (rc != MI_OK) return rc;
    attn_tiles_shared_kernel<Act, D, GROUPS><<<p.shares, THREADS, LDS, st>>>(p);
  } else {
    const int rc = int8_raise_lds(attn_tiles_kernel<Act, D, GROUPS>, raised, LDS);
    if (rc != MI_OK) return rc;
    attn_tiles_kernel<Act, D, GROUPS><<<(unsigned)(p.slots * p.Hkv), THREADS, LDS, st>>>(p);
  }
  return launch_status();
}
template <class Act, int D>
static int launch(const AttnArgs& p, hipStream_t st) {
  const bool groups = p.page % 8 == 0 && p.row16 < 1u << 24;     // a group's rows: 32-bit distances in bytes
  const int rc = groups ? launch_tiles<Act, D, true>(p, st) : launch_tiles<Act, D, false>(p, st);
  return rc != MI_OK || !p.shares ? rc : launch_join<Act, D, TilesCfg<D>::ROWS, 256>(p, p.shares, TilesCfg<D>::ROWS, st);
}

int launch_attn_tiles(const AttnArgs& p, int D, int act_dtype, hipStream_t st) {
  if (act_dtype == DT_F16) return D == 64 ? launch<ActF16, 64>(p, st) : D == 128 ? launch<ActF16, 128>(p, st) : launch<ActF16, 256>(p, st);
  return D == 64 ? launch<ActBF16, 64>(p, st) : D == 128 ? launch<ActBF16, 128>(p, st) : launch<ActBF16, 256>(p, st);
}

}  // namespace qlin
