// Few rows against 8-bit weights (int8_rows.hip).
#pragma once
#include "int8_common.hpp"

namespace qlin {

struct Int8RowsArgs {
  const void* x;              // codes [M, K], or 16-bit rows as QuantArgs has them
  const float* x_scale;       // of codes
  const void* residual;
  void* residual_out;         // overlaps no input: one workgroup writes it while others read
  const void* norm_weight;
  const int8_t* w;
  const float* w_scale;
  const void* bias;
  void* out;
  int M, N, K;
  int ks_log2;                // parts of K per slot: filled in by the launch
  float eps;
};

bool int8_rows_codes(int M, int K);                   // whether the kernel takes M rows of codes
bool int8_rows_quantise(int from, int M, int K);      // and of activations
int launch_int8_rows(int from, const Int8RowsArgs& p, int act_dtype, hipStream_t st);

}  // namespace qlin
