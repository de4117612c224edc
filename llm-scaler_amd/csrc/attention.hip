// C entries of the attention over a paged cache: checks, the choice of kernel, the workspace.
#include "attention.hpp"

#include "../../include/mi355x_qlinear.h"

namespace qlin {

// Which kernels a call runs.  Up to 32 rows (tokens x heads of a group) per sequence go to the rows kernel, more to the tiles kernel; where
// sequences of both kinds can be in a call both are launched, and each takes its own.  Measured at 16, 32 and 48 rows, 8 kv heads, us by the rows kernel
// and by tiles:
//   heads of 64    1 sequence of 1000 keys 12.1 / 19.3, 12.3 / 19.4, 13.8 / 20.5; 4 of 1000 14.3 / 19.6, 17.2 / 19.8, 18.9 / 21.0; 4 of 30000 59 / 61, 65 / 61, 104 / 60
//   heads of 128   1 of 1000 14.3 / 15.4, 14.8 / 16.7, 15.8 / 17.0; 4 of 1000 17.4 / 17.2, 21.5 / 17.3, 22.0 / 18.5; 4 of 30000 114 / 110, 121 / 113, 211 / 114
//   heads of 256   1 of 1000 20.7 / 21.7, 21.8 / 23.1, 24.5 / 24.6; 4 of 1000 27.6 / 24.2, 29.3 / 24.9, 31.5 / 26.5; 4 of 30000 201 / 191, 201 / 192, 359 / 192
// One bound for all: at 32 rows it is the better side by up to a third for short calls and heads of 64, and the worse by up to a fifth between.
struct AttnPlan {
  bool rows, tiles;
  int rows_from, groups, slots, shares;
  long long rows_bytes, tiles_bytes;
};

static int cus() {
  static const int n = [] {
    int dev = 0, v = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0) {
      (void)hipGetLastError();
      return 256;                                      // without a device only sizes are asked for
    }
    return v;
  }();
  return n;
}

static long long round256(long long v) { return (v + 255) / 256 * 256; }

// window 0: none
static int attn_plan(int T, int B, int Hq, int Hkv, int D, int max_query_len, int max_seq_len, long long window, long long sinks, AttnPlan& a) {
  if (D != 64 && D != 128 && D != 256) return MI_ERR_SHAPE;
  if (T < 0 || B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || max_query_len < 0 || max_seq_len < 0) return MI_ERR_SHAPE;
  if ((long long)T * Hq >= 1 << 28 || B >= 1 << 24 || Hq > 1 << 16) return MI_ERR_SHAPE;
  const int G = Hq / Hkv, most = max_query_len < T ? max_query_len : T;
  a = AttnPlan{};
  if (!T || !B) return MI_OK;
  // keys that `tokens` tokens side by side see
  const long long keys = max_seq_len < 1 ? 1 : max_seq_len;
  auto reach = [&](long long tokens) { return window && window + sinks + tokens < keys ? window + sinks + tokens : keys; };
  a.rows = a.tiles = true;
  a.rows_from = 33;
  if ((long long)most * G <= 32) {
    a.tiles = false;
    a.rows_from = INT32_MAX;
  } else if (B == 1 || (long long)B * most == T) {     // all sequences are as long as the longest
    a.rows = false;
    a.rows_from = 0;
  }
  if (a.rows) {
    const long long full = (long long)cus() * (D == 64 ? 8 : D == 128 ? 4 : 2);  // workgroups that the device holds
    // shares of two blocks at least: more of one block each make the joining longer (17.8 -> 15.4 us for 8 tiles of 908 keys)
    const long long tiles = ((long long)T * G / kFewRows < B ? B : (long long)T * G / kFewRows) * Hkv;
    const long long some = tiles * (reach(kFewRows) / 32 + 4) / 2 + 1;
    a.groups = (int)(some < full ? some : full);
    a.rows_bytes = round256(attn_parts_bytes(a.groups, D, kFewRows));
  }
  if (a.tiles) {
    const int R = attn_tile_rows(D), hold = cus() * (D == 64 ? 2 : 1);           // workgroups that the device holds
    const long long slots = (long long)T * G / R + B;
    if (slots * Hkv >= (1LL << 32) / (2 * R)) return MI_ERR_SHAPE;               // a grid holds less than 2^32 threads
    a.slots = (int)slots;
    // What the longer of both ways takes, in blocks of keys per workgroup: a workgroup per tile takes as long as the longest tile, and half as long again
    // on top of the even share where workgroups follow each other; equal shares have every tile see what its sequence's last token sees, and
    // parts to write and read.  One and four sequences of 1000 keys, 48 rows, heads of 128: 25.1 and 25.4 us by tiles, 16.4 and 17.7 in shares; four of
    // 500 with 256 rows 25.5 and 26.9, 16 of 700 with 48 20.8 and 26.2; heads of 64, four of 1000: 20.5 and 21.1.  In a window a tile
    // sees little of that: 2048 tokens at the end of 65536 in one of 1024, 64 heads of 128: 111 and 289 us; a prompt of 6000 in one of 512, 8 heads: 31
    // and 245.
    long long tiles = (long long)T * G / R;
    if (tiles < B) tiles = B;
    tiles *= Hkv;
    const long long tile = reach(R / G + 1), half = keys - (most < keys ? most : keys) / 2, seen = half < tile ? half : tile;    // of a tile: the most, the mean
    const long long even = tiles * seen / hold, alone = tiles <= hold ? tile : even + tile / 2, shared = tiles * reach(most) / hold + (D == 64 ? 1024 : 560);
    if (alone > shared) {
      a.shares = hold;
      a.tiles_bytes = round256(attn_parts_bytes(a.shares, D, R));
    }
  }
  return MI_OK;
}

// A window takes no more workspace than the call would without one.
static int attn_plan_within(int T, int B, int Hq, int Hkv, int D, int max_query_len, int max_seq_len, int window, int sinks, AttnPlan& a) {
  AttnPlan whole;
  const int rc = attn_plan(T, B, Hq, Hkv, D, max_query_len, max_seq_len, 0, 0, whole);
  if (rc != MI_OK || !window) {
    a = whole;
    return rc;
  }
  const int r = attn_plan(T, B, Hq, Hkv, D, max_query_len, max_seq_len, window, sinks, a);
  if (!whole.shares) a.shares = 0, a.tiles_bytes = 0;
  return r;
}
// window of a call: 1 and more, or -1: none.  0: none, as no place is 2^30 from another
static int window_of(int window) { return window < 0 || window >= 1 << 30 ? 0 : window; }

// key / d for keys below 2^30: (umulhi(key, mul) + key) >> shift
static void divide_by(uint32_t d, uint32_t& mul, uint32_t& shift) {
  shift = 0;
  while ((1ull << shift) < d) ++shift;
  mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
}

static int run(const AttnArgs& base, const MiPagedCache* cache, int D, float scale, int max_query_len, int max_seq_len, void* workspace,
               long long workspace_bytes, int act_dtype, hipStream_t st) {
  AttnArgs p = base;
  if (act_dtype != DT_F16 && act_dtype != DT_BF16) return MI_ERR_ARG;
  AttnPlan a;
  const int rc = attn_plan_within(p.T, p.B, p.Hq, p.Hkv, D, max_query_len, max_seq_len, p.window, p.sinks, a);
  if (rc != MI_OK) return rc;
  if (!a.rows && !a.tiles) return MI_OK;
  if (!cache || !p.q || !p.out || !p.seq_lens || !p.cu || !cache->key || !cache->value || !(scale > 0.f) || scale > 3e38f) return MI_ERR_ARG;
  if (!aligned16(p.q) || !aligned16(p.out) || !aligned16(cache->key) || !aligned16(cache->value) || !aligned16(workspace)) return MI_ERR_ARG;
  if (p.q_token % 8 || p.q_head % 8 || cache->page_stride % 8 || cache->token_stride % 8 || cache->head_stride % 8) return MI_ERR_SHAPE;
  if (cache->pages <= 0 || cache->page_size <= 0 || p.width < 0 || (p.width && !p.table)) return MI_ERR_ARG;
  if ((long long)p.width * cache->page_size >= 1 << 30) return MI_ERR_SHAPE;
  if (cache->page_stride < 0 || cache->token_stride < 0 || cache->head_stride < 0) return MI_ERR_SHAPE;
  const long long end = (cache->pages - 1LL) * (cache->page_stride / 8) + (cache->page_size - 1LL) * (cache->token_stride / 8) +
                        (p.Hkv - 1LL) * (cache->head_stride / 8) + D / 8;
  if (end >= (long long)kNoRow) return MI_ERR_SHAPE;
  if (a.rows_bytes + a.tiles_bytes > 0 && (!workspace || workspace_bytes < a.rows_bytes + a.tiles_bytes)) return MI_ERR_ARG;
  p.k = cache->key;
  p.v = cache->value;
  p.page16 = (uint32_t)(cache->page_stride / 8);
  p.row16 = (uint32_t)(cache->token_stride / 8);
  p.head16 = (uint32_t)(cache->head_stride / 8);
  p.page = cache->page_size;
  p.pages = cache->pages;
  divide_by((uint32_t)p.page, p.page_mul, p.page_shift);
  p.G = p.Hq / p.Hkv;
  p.c = scale * 1.4426950408889634f;
  p.far = 1024.f / p.c;
  p.rows_from = a.rows_from;
  p.groups = a.groups;
  const long long most = max_query_len < p.T ? max_query_len : p.T;
  p.tile_rows = a.tiles || most * p.G > 32 ? 32 : most < 1 ? p.G : (int)(most * p.G);
  p.many_parts = a.tiles || (long long)a.groups > 16LL * p.B * p.Hkv;          // with tiles beside them hardly any sequence is here
  p.wide = ((long long)p.T * p.G / 32 + p.B) * p.Hkv * ((long long)p.width * cache->page_size / 32 + 8) >= 1LL << 30;
  p.slots = a.slots;
  p.shares = a.shares;
  if (a.tiles) {
    p.part = (float*)((char*)workspace + a.rows_bytes);
    const int r = launch_attn_tiles(p, D, act_dtype, st);
    if (r != MI_OK) return r;
  }
  if (a.rows) {
    p.part = (float*)workspace;
    return launch_attn_rows(p, D, act_dtype, st);
  }
  return MI_OK;
}

}  // namespace qlin

using namespace qlin;

extern "C" {

int mi_paged_attention_workspace(int T, int B, int num_heads, int num_kv_heads, int head_dim, int max_query_len, int max_seq_len,
                                 long long* bytes) {
  if (!bytes) return MI_ERR_ARG;
  AttnPlan a;
  const int rc = attn_plan(T, B, num_heads, num_kv_heads, head_dim, max_query_len, max_seq_len, 0, 0, a);
  if (rc == MI_OK) *bytes = a.rows_bytes + a.tiles_bytes;
  return rc;
}

int mi_paged_attention_window_workspace(int T, int B, int num_heads, int num_kv_heads, int head_dim, int window, int sinks, int max_query_len,
                                        int max_seq_len, long long* bytes) {
  if (!bytes) return MI_ERR_ARG;
  if ((window < 1 && window != -1) || sinks < 0) return MI_ERR_SHAPE;
  AttnPlan a;
  const int rc = attn_plan_within(T, B, num_heads, num_kv_heads, head_dim, max_query_len, max_seq_len, window_of(window), sinks, a);
  if (rc == MI_OK) *bytes = a.rows_bytes + a.tiles_bytes;
  return rc;
}

int mi_paged_attention_ws(const void* query, long long token_stride, long long head_stride, const MiPagedCache* cache,
                          const int32_t* block_table, int table_width, const int32_t* seq_lens, const int32_t* cu_seqlens_q, void* out,
                          void* workspace, long long workspace_bytes, int T, int B, int num_heads, int num_kv_heads, int head_dim,
                          float scale, int window, int sinks, int max_query_len, int max_seq_len, int act_dtype, void* stream) {
  if ((window < 1 && window != -1) || sinks < 0) return MI_ERR_SHAPE;
  AttnArgs p{};
  p.q = query;
  p.q_token = token_stride;
  p.q_head = head_stride;
  p.table = block_table;
  p.width = table_width;
  p.seq_lens = seq_lens;
  p.cu = cu_seqlens_q;
  p.out = out;
  p.T = T;
  p.B = B;
  p.Hq = num_heads;
  p.Hkv = num_kv_heads;
  p.window = window_of(window);
  p.sinks = sinks;
  return run(p, cache, head_dim, scale, max_query_len, max_seq_len, workspace, workspace_bytes, act_dtype, (hipStream_t)stream);
}

int mi_tree_attention_ws(const void* query, long long token_stride, long long head_stride, const MiPagedCache* cache,
                         const int32_t* block_table, int table_width, const int32_t* seq_lens, const int32_t* cu_seqlens_q,
                         const int64_t* tree_mask, int mask_words, void* out, void* workspace, long long workspace_bytes, int T, int B,
                         int num_heads, int num_kv_heads, int head_dim, float scale, int max_query_len, int max_seq_len, int act_dtype,
                         void* stream) {
  if (T > 0 && B > 0 && !tree_mask) return MI_ERR_ARG;
  if (mask_words < 1 || mask_words > 1 << 20) return MI_ERR_SHAPE;
  AttnArgs p{};
  p.q = query;
  p.q_token = token_stride;
  p.q_head = head_stride;
  p.table = block_table;
  p.width = table_width;
  p.seq_lens = seq_lens;
  p.cu = cu_seqlens_q;
  p.tree = tree_mask;
  p.tree_words = mask_words;
  p.out = out;
  p.T = T;
  p.B = B;
  p.Hq = num_heads;
  p.Hkv = num_kv_heads;
  return run(p, cache, head_dim, scale, max_query_len, max_seq_len, workspace, workspace_bytes, act_dtype, (hipStream_t)stream);
}

}  // extern "C"
