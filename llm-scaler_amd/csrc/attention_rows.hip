// Attention of few rows per sequence (single tokens, small trees): 32 rows at most are in a tile, and the wavefronts of a workgroup take 32 keys
// each, with their loads two steps ahead and no barrier between them; their results meet in LDS.
//
// The work is cut evenly whatever the sequences' lengths are: all blocks of 64 keys of all (sequence, tile, kv head) in a row, and
// workgroup w takes [w, w + 1) total / groups of them.  A tile whose blocks all lie in one workgroup is finished there; of the others each
// workgroup has at most one that it continues and one that it begins, kept as unscaled fp32 sums with their m and l, and a second
// launch joins them.
//
// Bound: HBM.
#include "attention.hpp"

namespace qlin {

template <int D> struct RowsCfg {
  static constexpr int NW = D == 256 ? 2 : 4;          // wavefronts
  static constexpr int STAGES = 2;
  static constexpr int HALF = 32 * D * 2;              // K or V of a step
  static constexpr int LDS = NW * STAGES * 2 * HALF;
  static constexpr int PITCH = D + 4;                  // of the floats in LDS
  static constexpr int PART = 32 * (D + 2);            // floats of a part: sums, m, l
};

// How many tiles a sequence has here, and how many blocks each of them
struct RowsSeq { AttnSeq s; AttnRange r; int tiles; };
__device__ __forceinline__ RowsSeq rows_seq(const AttnArgs& p, int b) {
  RowsSeq x;
  x.s = attn_seq(p, b);
  x.r = attn_range<kBlock>(p, x.s, 0, x.s.n - 1);
  x.r.blocks = max(x.r.blocks, 1);                     // a row that sees nothing is written too
  const int rows = x.s.n * p.G;
  x.tiles = rows >= p.rows_from ? 0 : (rows + 31) / 32;
  return x;
}
__device__ __forceinline__ long long rows_work(const AttnArgs& p, const RowsSeq& x) { return (long long)x.tiles * p.Hkv * x.r.blocks; }

__device__ __forceinline__ long long shfl64(long long v, int lane) {
  return (long long)(uint32_t)__shfl((int)v, lane, 64) | (long long)__shfl((int)(v >> 32), lane, 64) << 32;
}

// All work of the call, and the share of a workgroup: every wavefront finds it by itself.
struct RowsPlan { long long incl, before, total, share; int per; };
__device__ __forceinline__ RowsPlan rows_plan(const AttnArgs& p) {
  const int lane = threadIdx.x & 63;
  RowsPlan a;
  a.per = (p.B + 63) / 64;
  long long mine = 0;
  for (int i = 0; i < a.per; ++i) {
    const int b = lane * a.per + i;
    if (b < p.B) mine += rows_work(p, rows_seq(p, b));
  }
  long long incl = mine;
  for (int d = 1; d < 64; d <<= 1) {
    const long long up = shfl64(incl, lane >= d ? lane - d : lane);
    if (lane >= d) incl += up;
  }
  a.incl = incl;
  a.before = incl - mine;
  a.total = shfl64(incl, 63);
  a.share = (a.total + p.groups - 1) / p.groups;
  return a;
}
// The sequence with block `at` of the work, and the place of the block in it.  at < total.
__device__ __forceinline__ void rows_find(const AttnArgs& p, const RowsPlan& a, long long at, int& b, long long& in) {
  const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(at < a.incl));
  long long rest = at - shfl64(a.before, owner);
  b = owner * a.per;
  for (;; ++b) {
    const long long n = rows_work(p, rows_seq(p, b));
    if (rest < n || b + 1 >= p.B) break;
    rest -= n;
  }
  in = rest;
}

template <class Act, int D>
__global__ __launch_bounds__(64 * RowsCfg<D>::NW) void attn_rows_kernel(const AttnArgs p) {
  using C = RowsCfg<D>;
  constexpr int NW = C::NW, LOADS = 2 * C::HALF / 1024;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  __shared__ float ml[2][NW][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned char* ring = smem + wave * (C::STAGES * 2 * C::HALF);

  const RowsPlan plan = rows_plan(p);
  long long at = plan.share * blockIdx.x;
  const long long end = min(at + plan.share, plan.total);
  if (at >= end) return;
  int b;
  long long in;
  rows_find(p, plan, at, b, in);
  b = __builtin_amdgcn_readfirstlane(b);

  while (at < end) {
    const RowsSeq x = rows_seq(p, b);
    const int item = __builtin_amdgcn_readfirstlane((int)(in / x.r.blocks));
    const int block0 = __builtin_amdgcn_readfirstlane((int)(in - (long long)item * x.r.blocks));
    const int block1 = __builtin_amdgcn_readfirstlane((int)min((long long)x.r.blocks, block0 + (end - at)));
    const int tile = item / p.Hkv, head = item - tile * p.Hkv, rows = min(32, x.s.n * p.G - tile * 32);
    const int32_t* table = p.table + (size_t)b * p.width;

    // this lane's row
    const int r = tile * 32 + (lane & 31), t = r / p.G;
    const bool has = (lane & 31) < rows;
    const int64_t* tree = p.tree ? p.tree + (size_t)(x.s.q0 + (has ? t : 0)) * p.tree_words : nullptr;
    const int t0 = tile * 32 / p.G, t1 = (tile * 32 + rows - 1) / p.G;
    AttnRows<Act, D> a;
    a.start();
    a.load_q(has ? (const typename Act::elem*)p.q + (x.s.q0 + t) * p.q_token + (head * p.G + r - t * p.G) * p.q_head : nullptr);

    // steps of 32 keys: first + NW i is this wavefront's i-th
    const int first = 2 * block0 + wave, last = 2 * block1;
    auto key_of = [&](int step) { return attn_key<kBlock>(x.r, step >> 1) + (step & 1) * 32; };
    auto lookup = [&](int step) { return step < last ? attn_lookup(p, table, x.r, key_of(step) + (lane & 31)) : -1; };
    auto place = [&](int page, int step) { return step < last ? attn_place(p, page, key_of(step) + (lane & 31), head) : kNoRow; };
    uint64_t there[2];
    int step = first;
    int page = lookup(step);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t at16 = place(page, step + u * NW);
      page = lookup(step + (u + 1) * NW);
      there[u] = __builtin_amdgcn_ballot_w64(at16 != kNoRow) & 0xFFFFFFFFull;
      attn_load<D, 32>(p.k, p.v, at16, 0, ring + u * 2 * C::HALF, ring + u * 2 * C::HALF + C::HALF);
    }
    while (step < last) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (step >= last) break;
        wait_loads<LOADS>();
        __builtin_amdgcn_sched_barrier(0);
        const int kb = key_of(step);
        const bool full = there[u] == 0xFFFFFFFFull && attn_all_seen<32>(p, x.s.first, t0, t1, kb);
        uint64_t mask = there[u];
        if (!full) mask &= attn_sees(p, x.s.first, t, tree, kb);
        a.template block<32>(ring + u * 2 * C::HALF, ring + u * 2 * C::HALF + C::HALF, full, mask, p.c);
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t at16 = place(page, step + 2 * NW);
        page = lookup(step + 3 * NW);
        there[u] = __builtin_amdgcn_ballot_w64(at16 != kNoRow) & 0xFFFFFFFFull;
        attn_load<D, 32>(p.k, p.v, at16, 0, ring + u * 2 * C::HALF, ring + u * 2 * C::HALF + C::HALF);
        step += NW;
      }
    }
    wait_loads<0>();
    __syncthreads();                                   // all rings are free

    float* sums = (float*)smem;
    const Halves ls = both_halves(a.l);
    const float l = ls.low + ls.high;
    if (lane < 32) {
      ml[0][wave][lane] = a.m;
      ml[1][wave][lane] = l;
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *(f32x4*)(sums + (wave * 32 + (lane & 31)) * C::PITCH + d * 32 + i * 2 + (lane >> 5) * 4) =
            f32x4{a.o[d][i], a.o[d][i + 1], a.o[d][i + 2], a.o[d][i + 3]};
    __syncthreads();
    const bool whole = block0 == 0 && block1 == x.r.blocks;
    float* part = p.part + ((size_t)blockIdx.x * 2 + (block0 == 0)) * C::PART;
    for (int idx = threadIdx.x; idx < rows * (D / 4); idx += 64 * NW) {
      const int row = idx / (D / 4), col = idx % (D / 4) * 4;
      float m = ml[0][0][row], sum = 0.f;
#pragma unroll
      for (int w = 1; w < NW; ++w) m = fmaxf(m, ml[0][w][row]);
      const float top = m == -__builtin_inff() ? 0.f : m;
      f32x4 o = {};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(ml[0][w][row] - top);
        sum += f * ml[1][w][row];
        o += f * *(const f32x4*)(sums + (w * 32 + row) * C::PITCH + col);
      }
      if (whole) {
        const float f = sum == 0.f ? 0.f : 1.f / sum;
        const int rr = tile * 32 + row, tt = rr / p.G;
        typename Act::elem* to = (typename Act::elem*)p.out + ((size_t)(x.s.q0 + tt) * p.Hq + head * p.G + rr - tt * p.G) * D + col;
        typedef __attribute__((ext_vector_type(4))) typename Act::elem e4;
        e4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = Act::from_f32(o[i] * f);
        *(e4*)to = y;
      } else {
        *(f32x4*)(part + row * D + col) = o;
        if (col == 0) {
          part[32 * D + row] = m;
          part[32 * D + 32 + row] = sum;
        }
      }
    }
    __syncthreads();                                   // before the rings are filled again
    at += block1 - block0;
    in += block1 - block0;
    if (in >= rows_work(p, x)) {
      in = 0;
      do ++b;
      while (b + 1 < p.B && at < end && rows_work(p, rows_seq(p, b)) == 0);
    }
  }
}

// Workgroup w joins the tile that the boundary in front of share w cuts, if no earlier boundary cuts it too.
template <class Act, int D>
__global__ __launch_bounds__(256) void attn_rows_join_kernel(const AttnArgs p) {
  using C = RowsCfg<D>;
  const RowsPlan plan = rows_plan(p);
  const long long w = blockIdx.x + 1, at = w * plan.share;
  if (at >= plan.total) return;
  int b;
  long long in;
  rows_find(p, plan, at, b, in);
  const RowsSeq x = rows_seq(p, b);
  const int item = (int)(in / x.r.blocks), block0 = (int)(in - (long long)item * x.r.blocks);
  const long long begin = at - block0;
  if (block0 == 0 || (w - 1) * plan.share > begin) return;
  const int parts = 1 + (int)((begin + x.r.blocks - 1) / plan.share - (w - 1));
  const int tile = item / p.Hkv, head = item - tile * p.Hkv, rows = min(32, x.s.n * p.G - tile * 32);
  for (int idx = threadIdx.x; idx < rows * (D / 4); idx += 256) {
    const int row = idx / (D / 4), col = idx % (D / 4) * 4;
    float m = -__builtin_inff(), sum = 0.f;
    auto part = [&](int i) { return p.part + ((size_t)(w - 1 + i) * 2 + (i == 0)) * C::PART; };
    for (int i = 0; i < parts; ++i) m = fmaxf(m, part(i)[32 * D + row]);
    const float top = m == -__builtin_inff() ? 0.f : m;
    f32x4 o = {};
    for (int i = 0; i < parts; ++i) {
      const float* from = part(i);
      const float f = __builtin_amdgcn_exp2f(from[32 * D + row] - top);
      sum += f * from[32 * D + 32 + row];
      o += f * *(const f32x4*)(from + row * D + col);
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    const int rr = tile * 32 + row, tt = rr / p.G;
    typename Act::elem* to = (typename Act::elem*)p.out + ((size_t)(x.s.q0 + tt) * p.Hq + head * p.G + rr - tt * p.G) * D + col;
    typedef __attribute__((ext_vector_type(4))) typename Act::elem e4;
    e4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = Act::from_f32(o[i] * f);
    *(e4*)to = y;
  }
}

long long attn_rows_bytes(int groups, int D) { return (long long)groups * 2 * 32 * (D + 2) * 4; }

template <class Act, int D>
static int launch(const AttnArgs& p, hipStream_t st) {
  static std::atomic<unsigned long long> raised{0};
  const int rc = int8_raise_lds(attn_rows_kernel<Act, D>, raised, RowsCfg<D>::LDS);
  if (rc != MI_OK) return rc;
  attn_rows_kernel<Act, D><<<p.groups, 64 * RowsCfg<D>::NW, RowsCfg<D>::LDS, st>>>(p);
  if (p.groups > 1) attn_rows_join_kernel<Act, D><<<p.groups - 1, 256, 0, st>>>(p);
  return launch_status();
}

int launch_attn_rows(const AttnArgs& p, int D, int act_dtype, hipStream_t st) {
  if (act_dtype == DT_F16) return D == 64 ? launch<ActF16, 64>(p, st) : D == 128 ? launch<ActF16, 128>(p, st) : launch<ActF16, 256>(p, st);
  return D == 64 ? launch<ActBF16, 64>(p, st) : D == 128 ? launch<ActBF16, 128>(p, st) : launch<ActBF16, 256>(p, st);
}

}  // namespace qlin
