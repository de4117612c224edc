// The expert layer on 8-bit integers: its operands, and the two launches for a few tokens (int8_moe_decode.hip).
#pragma once
#include "int8_common.hpp"

#include <type_traits>

namespace qlin {

struct Int8MoeArgs {
  const void *x, *logits;     // [T, H], [T, E]
  void* out;                  // [T, H]
  const int8_t *w13, *w2;     // [E, 2 I, H], [E, H, I]
  const float *s13, *s2;      // [E, 2 I], [E, H]
  const int8_t *shared_w13, *shared_w2;                // null: no shared expert
  const float *shared_s13, *shared_s2;
  const void* gate_weight;    // [H]
  void* top_w;                // [T, k], activation type
  int32_t* ids;               // [T, k]
  float* gate;                // [T]
  float* h;                   // [T k + T, I]: routes in pair order, then the shared expert's rows
  int T, k, E, H, I;
};

bool int8_moe_decode_pays(int T, int k, int E, int H, int I, bool shared);
int launch_int8_moe_decode(const Int8MoeArgs& p, int act_dtype, hipStream_t st);

}  // namespace qlin
