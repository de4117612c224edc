// Attention of few rows per sequence (single tokens, small trees): up to 32 rows are in a tile, a wavefront by itself takes an equal share of the work,
// 32 keys at a time, with its loads two steps ahead.
//
// A wavefront needs no barrier, and eight (four, two with heads of 64, 128, 256) fill a CU's LDS with loads under way.  Equal shares: whatever the
// lengths, all wavefronts end together (a workgroup per tile and a fixed number of parts took 1.2 to 1.5 times as long for trees over long contexts).
//
// Bound: HBM.  Two sequences of 131072 keys, 8 kv heads of 128: 1.07 GB in 204 us (5.3 TB/s) and 10 to join the parts; 64 sequences of up to 8192:
// 260 MB in 56 us (4.6 TB/s) and 7.  Heads of 256, two wavefronts per CU: 1.07 GB in 185 us and 9, 130 MB of 64 sequences in 34 (3.8 TB/s) and 15.
// Short calls: two launches, of which the second waits for the first (8 and 4 us for a sequence of 700).
// 28, 43 and 91 scalar registers (heads of 64, 128, 256) lie in lanes of vector registers: of the shares, read again between tiles, and of the edges, read in the
// loop (0, 7 and up to 20 reads per two steps).
#include "attention.hpp"

namespace qlin {

template <int D> struct RowsCfg {
  static constexpr int KEYS = 32, STAGES = 2;
  static constexpr int HALF = KEYS * D * 2;            // K or V of a step
  static constexpr int LDS = STAGES * 2 * HALF + 512;  // behind the ring: pages of 64 keys, twice
};

template <class Act, int D, class Num>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2, D == 256 ? 1 : 2))) void attn_rows_kernel(const AttnArgs p) {
  using C = RowsCfg<D>;
  using Rows = AttnRows<Act, D>;
  constexpr int LOADS = 2 * C::HALF / 1024, kItem = 3;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x;

  using Work = Shares<kFewRows, 32, kItem, true, Num>;
  Work shares;
  shares.plan(p, p.groups);
  Num at, end;
  shares.of(blockIdx.x, at, end);
  if (at >= end) {
    if (lane == 0) attn_cuts<D, kFewRows>(p, p.groups)[blockIdx.x] = i32x4{};
    return;
  }
  int b;
  Num in;
  shares.find(p, at, b, in);

  for (bool starts = true; at < end; starts = false) {
    const typename Work::Seq x = shares.seq(p, b);
    const typename Work::Item y = Work::item(p, x, in);
    if (starts) {
      const int parts = shares.parts_at(blockIdx.x, at, x, y);
      if (lane == 0) attn_cuts<D, kFewRows>(p, p.groups)[blockIdx.x] = i32x4{parts, x.s.q0, y.tile, y.head << 9 | y.rows};
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
      a.load_q(has ? (const typename Act::elem*)p.q + (x.s.q0 + t) * p.q_token + (y.head * p.G + r - t * p.G) * p.q_head : nullptr);

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
          typename Rows::Keys f;
          typename Rows::Weights w;
          uint32_t mask = there[u];
          a.read_keys(k, f);
          f32x16 s = a.scores(f);
          if (!full) {
            mask &= attn_sees(p, x.s.first, t, tree, kb);
            a.hide(s, mask);
          }
          a.follow(p, s, a.largest(s));
          a.weigh(p, s, w);
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

      const Halves ls = both_halves(a.l);
      const float l = ls.low + ls.high;
      if (has) {
        const int h = lane >> 5;
        if (first == 0 && last == x.r.blocks) {
          const float f = l == 0.f ? 0.f : 1.f / l;
          typedef __attribute__((ext_vector_type(4))) typename Act::elem e4;
          typename Act::elem* to = (typename Act::elem*)p.out + attn_row(p, x.s.q0, y.head, r) * D + h * 4;
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              e4 z;
#pragma unroll
              for (int e = 0; e < 4; ++e) z[e] = Act::from_f32(a.o[d][j + e] * f);
              *(e4*)(to + d * 32 + j * 2) = z;
            }
        } else {
          float* part = attn_part<D, kFewRows>(p, blockIdx.x, first == 0);
          if (h == 0) *(f32x2*)(part + 32 * D + 2 * lane) = f32x2{a.reference(), l};
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *(f32x4*)(part + (lane & 31) * D + h * 4 + d * 32 + j * 2) =
                  f32x4{a.o[d][j], a.o[d][j + 1], a.o[d][j + 2], a.o[d][j + 3]};
        }
      }
    }
    shares.advance(p, x, at < end, b, in);
  }
}

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
  if (rc != MI_OK) return rc;
  return p.many_parts ? launch_join<Act, D, kFewRows, 1024>(p, p.groups, p.tile_rows, st) : launch_join<Act, D, kFewRows, 256>(p, p.groups, p.tile_rows, st);
}

int launch_attn_rows(const AttnArgs& p, int D, int act_dtype, hipStream_t st) {
  if (act_dtype == DT_F16) return D == 64 ? launch<ActF16, 64>(p, st) : D == 128 ? launch<ActF16, 128>(p, st) : launch<ActF16, 256>(p, st);
  return D == 64 ? launch<ActBF16, 64>(p, st) : D == 128 ? launch<ActBF16, 128>(p, st) : launch<ActBF16, 256>(p, st);
}

}  // namespace qlin
