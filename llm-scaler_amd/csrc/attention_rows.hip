// Attention of few rows per sequence (single tokens, small trees): up to 32 rows are in a tile, a wavefront by itself takes a part of the keys of one
// tile after another, 32 at a time, with its loads two steps ahead.
//
// The work is cut evenly whatever the sequences' lengths are: the blocks of 32 keys of all (sequence, tile, kv head) in a row, each of these with
// kItem blocks more for what beginning it costs, and workgroup w takes [w, w + 1) total / groups of them.  A tile whose blocks all lie in one
// workgroup is finished there; of the others each workgroup has at most one that it continues and one that it begins, kept as unscaled fp32 sums
// with their m and l, and a second launch joins them.
//
// Bound: HBM.
#include "attention.hpp"

namespace qlin {

template <int D> struct RowsCfg {
  static constexpr int KEYS = 32, STAGES = 2;
  static constexpr int HALF = KEYS * D * 2;            // K or V of a step
  static constexpr int LDS = STAGES * 2 * HALF + 512;  // behind the ring: pages of 64 keys, twice
  static constexpr int PART = 32 * (D + 2);            // floats of a part: sums, m, l
};
constexpr int kItem = 3;

// How many tiles a sequence has here, and how many blocks each of them
struct RowsSeq { AttnSeq s; AttnRange r; int tiles; };
__device__ __forceinline__ RowsSeq rows_seq(const AttnArgs& p, int b) {
  RowsSeq x;
  x.s = attn_seq(p, b);
  x.r = attn_range<32>(p, x.s, 0, x.s.n - 1);
  x.r.blocks = max(x.r.blocks, 1);                     // a row that sees nothing is written too
  const int rows = x.s.n * p.G;
  x.tiles = rows >= p.rows_from ? 0 : (rows + 31) / 32;
  return x;
}
// Num: int where all work of the call counts less than 2^31 blocks
template <class Num>
__device__ __forceinline__ Num rows_work(const AttnArgs& p, const RowsSeq& x) { return (Num)x.tiles * p.Hkv * (x.r.blocks + kItem); }

__device__ __forceinline__ int from_lane(int v, int lane) { return __shfl(v, lane, 64); }
__device__ __forceinline__ long long from_lane(long long v, int lane) {
  return (long long)(uint32_t)__shfl((int)v, lane, 64) | (long long)__shfl((int)(v >> 32), lane, 64) << 32;
}

// All work of the call, and the share of a workgroup: every wavefront finds it by itself.
template <class Num> struct RowsPlan { Num incl, before, total, share; int per; };
template <class Num>
__device__ __forceinline__ RowsPlan<Num> rows_plan(const AttnArgs& p) {
  const int lane = threadIdx.x & 63;
  RowsPlan<Num> a;
  a.per = (p.B + 63) / 64;
  Num mine = 0;
  for (int i = 0; i < a.per; ++i) {
    const int b = lane * a.per + i;
    if (b < p.B) mine += rows_work<Num>(p, rows_seq(p, b));
  }
  Num incl = mine;
  for (int d = 1; d < 64 && d < p.B; d <<= 1) {
    const Num up = from_lane(incl, lane >= d ? lane - d : lane);
    if (lane >= d) incl += up;
  }
  a.incl = incl;
  a.before = incl - mine;
  a.total = from_lane(incl, (p.B - 1) / a.per);        // the last lane with sequences; those behind it have not added all up
  a.share = (a.total + p.groups - 1) / p.groups;
  return a;
}
// The sequence with block `at` of the work, and the place of the block in it.  at < total.
template <class Num>
__device__ __forceinline__ void rows_find(const AttnArgs& p, const RowsPlan<Num>& a, Num at, int& b, Num& in) {
  const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(at < a.incl));
  Num rest = at - from_lane(a.before, owner);
  b = owner * a.per;
  for (; a.per > 1 && b + 1 < p.B; ++b) {
    const Num n = rows_work<Num>(p, rows_seq(p, b));
    if (rest < n) break;
    rest -= n;
  }
  in = rest;
}

// A tile's place in the work: its sequence's `in`-th unit
struct RowsItem { int tile, head, rows, unit; };      // unit: of the tile; its first kItem are none of its blocks
template <class Num>
__device__ __forceinline__ RowsItem rows_item(const AttnArgs& p, const RowsSeq& x, Num in) {
  const int per = x.r.blocks + kItem;
  const int item = __builtin_amdgcn_readfirstlane((int)(in / per));
  RowsItem y;
  y.unit = __builtin_amdgcn_readfirstlane((int)(in - (Num)item * per));
  y.tile = item / p.Hkv;
  y.head = item - y.tile * p.Hkv;
  y.rows = min(32, x.s.n * p.G - y.tile * 32);
  return y;
}
// Row `row` of a tile in out
__device__ __forceinline__ long long rows_row(const AttnArgs& p, int q0, int tile, int head, int row) {
  const int r = tile * 32 + row, t = r / p.G;
  return (long long)(q0 + t) * p.Hq + head * p.G + r - t * p.G;
}
// Behind the parts: for the cut in front of each share how many parts are to be joined there (0: none), and the tile
template <int D>
__device__ __forceinline__ i32x4* rows_cuts(const AttnArgs& p) { return (i32x4*)(p.part + (size_t)p.groups * 2 * RowsCfg<D>::PART); }

template <class Act, int D, class Num>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2, D == 256 ? 1 : 2))) void attn_rows_kernel(const AttnArgs p) {
  using C = RowsCfg<D>;
  using Rows = AttnRows<Act, D, 32, 1>;
  constexpr int LOADS = 2 * C::HALF / 1024;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x;

  const RowsPlan<Num> plan = rows_plan<Num>(p);
  // shares: all of them may count up to 2^31 and a share more
  const bool none = plan.share == 0 || (Num)blockIdx.x > plan.total / plan.share;
  Num at = none ? plan.total : plan.share * (Num)blockIdx.x;
  const Num end = plan.total - at < plan.share ? plan.total : at + plan.share;
  if (at >= end) {
    if (lane == 0) rows_cuts<D>(p)[blockIdx.x] = i32x4{};
    return;
  }
  int b;
  Num in;
  rows_find<Num>(p, plan, at, b, in);
  b = __builtin_amdgcn_readfirstlane(b);

  for (bool starts = true; at < end; starts = false) {
    const RowsSeq x = rows_seq(p, b);
    const RowsItem y = rows_item(p, x, in);
    if (starts) {                                      // the cut in front of this share is one to join at if it goes through blocks, as the tile's first
      const Num begin = at - y.unit + kItem, w = blockIdx.x;
      const int parts = at <= begin || (w - 1) * plan.share > begin ? 0 : 1 + (int)((begin + x.r.blocks - 1) / plan.share - (w - 1));
      if (lane == 0) rows_cuts<D>(p)[w] = i32x4{parts, x.s.q0, y.tile, y.head * 64 + y.rows};
    }
    const int take = __builtin_amdgcn_readfirstlane((int)min((Num)(x.r.blocks + kItem - y.unit), end - at));
    const int first = max(y.unit - kItem, 0), last = y.unit + take - kItem;      // blocks
    at += take;
    in += take;
    if (last > first) {
      const int32_t* table = p.table + (size_t)b * p.width;
      const int r = y.tile * 32 + (lane & 31), t = r / p.G;                      // this lane's row
      const bool has = (lane & 31) < y.rows;
      const int64_t* tree = p.tree ? p.tree + (size_t)(x.s.q0 + (has ? t : 0)) * p.tree_words : nullptr;
      const int t0 = y.tile * 32 / p.G, t1 = (y.tile * 32 + y.rows - 1) / p.G;
      Rows a;
      a.start();
      a.load_q(0, has ? (const typename Act::elem*)p.q + (x.s.q0 + t) * p.q_token + (y.head * p.G + r - t * p.G) * p.q_head : nullptr);

      // block i's keys and values lie in half (i - first) % 2 of the ring, the pages of its keys likewise behind it
      const uint32_t ring = lds_address(smem), pages = ring + C::STAGES * 2 * C::HALF;
      auto lookup = [&](int i, int u) {
        const int key = attn_key<32>(x.r, i) + (lane & 31);
        to_lds4(i < last && attn_in(p, x.r, key) ? table + attn_page_of(p, key) : kNoPage, pages + u * 256);
      };
      auto place = [&](int i, int u) {
        const int page = *in_lds<const int>(pages + u * 256 + lane * 4);
        return i < last ? attn_place(p, page, attn_key<32>(x.r, i) + (lane & 31), y.head) : kNoRow;
      };
      auto request = [&](uint32_t at16, int u) {
        RowPlaces<D, 32> rows;
        rows.take(at16, 0);
        rows.template load<true>(p.k, 0, ring + u * 2 * C::HALF);
        rows.template load<false>(p.v, 0, ring + u * 2 * C::HALF + C::HALF);
        return (uint32_t)__builtin_amdgcn_ballot_w64(at16 != kNoRow);
      };
      uint32_t there[2];
      lookup(first, 0);
      lookup(first + 1, 1);
      wait_loads<0>();
      const uint32_t at0 = place(first, 0), at1 = place(first + 1, 1);
      there[0] = request(at0, 0);
      lookup(first + 2, 0);
      there[1] = request(at1, 1);
      for (int i = first; i < last;) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (i >= last) break;
          wait_loads<LOADS>();                         // block i is there, and the pages of block i + 2
          __builtin_amdgcn_sched_barrier(0);
          const uint32_t k = ring + u * 2 * C::HALF, v = k + C::HALF;
          const int kb = attn_key<32>(x.r, i);
          const bool full = there[u] == 0xFFFFFFFFu && attn_all_seen<32>(p, x.s.first, t0, t1, kb);
          typename Rows::Scores s;
          typename Rows::Weights w;
          typename Rows::Mask mask;
          float top[1];
          a.scores(k, s);
          if (!full) {
            mask.of[0] = there[u] & attn_sees(p, x.s.first, t, tree, kb);
            a.hide(s, mask);
          }
          a.largest(s, p.c, top);
          a.follow(top);
          a.weigh(s, p.c, w);
          if (full) a.add(v, w);
          else a.add_hidden(v, w, mask);
          __builtin_amdgcn_sched_barrier(0);
          const uint32_t at16 = place(i + 2, u);
          lookup(i + 3, u ^ 1);
          there[u] = request(at16, u);
          ++i;
        }
      }
      wait_loads<0>();                                 // the ring is filled anew for the next tile

      const Halves ls = both_halves(a.l[0]);
      const float l = ls.low + ls.high;
      if (has) {
        const int h = lane >> 5;
        if (first == 0 && last == x.r.blocks) {
          const float f = l == 0.f ? 0.f : 1.f / l;
          typedef __attribute__((ext_vector_type(4))) typename Act::elem e4;
          typename Act::elem* to = (typename Act::elem*)p.out + rows_row(p, x.s.q0, y.tile, y.head, lane & 31) * D + h * 4;
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              e4 z;
#pragma unroll
              for (int e = 0; e < 4; ++e) z[e] = Act::from_f32(a.o[0][d][j + e] * f);
              *(e4*)(to + d * 32 + j * 2) = z;
            }
        } else {
          float* part = p.part + ((size_t)blockIdx.x * 2 + (first == 0)) * C::PART;
          if (h == 0) *(f32x2*)(part + 32 * D + 2 * lane) = f32x2{a.m[0], l};
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *(f32x4*)(part + (lane & 31) * D + h * 4 + d * 32 + j * 2) =
                  f32x4{a.o[0][d][j], a.o[0][d][j + 1], a.o[0][d][j + 2], a.o[0][d][j + 3]};
        }
      }
    }
    if (in >= rows_work<Num>(p, x)) {
      in = 0;
      do ++b;
      while (b + 1 < p.B && at < end && rows_work<Num>(p, rows_seq(p, b)) == 0);
    }
  }
}

// Workgroup w, y joins rows 8 y .., and every 8 gridDim.y further, of the tile that the cut in front of share w + 1 goes through.
template <class Act, int D, int THREADS>
__global__ __launch_bounds__(THREADS) void attn_rows_join_kernel(const AttnArgs p) {
  constexpr int PART = RowsCfg<D>::PART;
  const int w = blockIdx.x + 1;
  const i32x4 cut = rows_cuts<D>(p)[w];
  const int rows = cut[3] % 64;
  if (!cut[0]) return;
  // the first part is the one that share w - 1 began, the others those that a share continued
  auto part = [&](int i) { return p.part + ((size_t)(w - 1 + i) * 2 + (i == 0)) * PART; };
  for (int row0 = blockIdx.y * kJoinRows; row0 < rows; row0 += gridDim.y * kJoinRows)
    attn_join<Act, D, THREADS>(
        min(kJoinRows, rows - row0), cut[0], [&](int i, int row) { return part(i) + (row0 + row) * D; },
        [&](int i, int row) { return part(i) + 32 * D + 2 * (row0 + row); },
        [&](int row) { return (typename Act::elem*)p.out + rows_row(p, cut[1], cut[2], cut[3] / 64, row0 + row) * D; });
}

long long attn_rows_bytes(int groups, int D) { return (long long)groups * (2 * 32 * (D + 2) * 4 + 16); }

template <class Act, int D, class Num>
static int launch_rows(const AttnArgs& p, hipStream_t st) {
  static std::atomic<unsigned long long> raised{0};
  const int rc = int8_raise_lds(attn_rows_kernel<Act, D, Num>, raised, RowsCfg<D>::LDS);
  if (rc != MI_OK) return rc;
  attn_rows_kernel<Act, D, Num><<<p.groups, 64, RowsCfg<D>::LDS, st>>>(p);
  return launch_status();
}
template <class Act, int D>
static int launch(const AttnArgs& p, hipStream_t st) {
  const int rc = p.wide ? launch_rows<Act, D, long long>(p, st) : launch_rows<Act, D, int>(p, st);
  if (rc != MI_OK || p.groups == 1) return rc;
  const dim3 grid(p.groups - 1, (p.tile_rows + kJoinRows - 1) / kJoinRows);
  if (p.many_parts) attn_rows_join_kernel<Act, D, 1024><<<grid, 1024, 0, st>>>(p);
  else attn_rows_join_kernel<Act, D, 256><<<grid, 256, 0, st>>>(p);
  return launch_status();
}

int launch_attn_rows(const AttnArgs& p, int D, int act_dtype, hipStream_t st) {
  if (act_dtype == DT_F16) return D == 64 ? launch<ActF16, 64>(p, st) : D == 128 ? launch<ActF16, 128>(p, st) : launch<ActF16, 256>(p, st);
  return D == 64 ? launch<ActBF16, 64>(p, st) : D == 128 ? launch<ActBF16, 128>(p, st) : launch<ActBF16, 256>(p, st);
}

}  // namespace qlin
