// Launches of int8_quant.hpp.
#include "int8_quant.hpp"
#include "../../include/mi355x_qlinear.h"

namespace qlin {

template <class Act, int FROM, int TPR, int NV>
__global__ __launch_bounds__(256) void int8_quant_kernel(const QuantArgs p) {
  int8_quant_rows<Act, FROM, TPR, NV>(p, blockIdx.x);
}

template <class Act, int FROM>
static void launch_quant(const QuantArgs& p, hipStream_t st) {
  const int pieces = p.K / 8;
  const unsigned by4 = (unsigned)((p.rows + 3) / 4), by1 = (unsigned)p.rows;
  if (pieces <= 64) hipLaunchKernelGGL((int8_quant_kernel<Act, FROM, 64, 1>), dim3(by4), dim3(256), 0, st, p);
  else if (pieces <= 128) hipLaunchKernelGGL((int8_quant_kernel<Act, FROM, 64, 2>), dim3(by4), dim3(256), 0, st, p);
  else if (pieces <= 256) hipLaunchKernelGGL((int8_quant_kernel<Act, FROM, 256, 1>), dim3(by1), dim3(256), 0, st, p);
  else if (pieces <= 512) hipLaunchKernelGGL((int8_quant_kernel<Act, FROM, 256, 2>), dim3(by1), dim3(256), 0, st, p);
  else if (pieces <= 1024) hipLaunchKernelGGL((int8_quant_kernel<Act, FROM, 256, 4>), dim3(by1), dim3(256), 0, st, p);
  else if (pieces <= 2048) hipLaunchKernelGGL((int8_quant_kernel<Act, FROM, 256, 8>), dim3(by1), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((int8_quant_kernel<Act, FROM, 256, 0>), dim3(by1), dim3(256), 0, st, p);
}

int launch_int8_quant(int from, const QuantArgs& p, int act_dtype, hipStream_t st) {
  if (!p.rows) return MI_OK;
  if (p.rows > 0x7FFFFFFFLL) return MI_ERR_SHAPE;
  const bool f16 = act_dtype == DT_F16;
  switch (from) {
    case kFromAct: f16 ? launch_quant<ActF16, kFromAct>(p, st) : launch_quant<ActBF16, kFromAct>(p, st); break;
    case kFromNorm: f16 ? launch_quant<ActF16, kFromNorm>(p, st) : launch_quant<ActBF16, kFromNorm>(p, st); break;
    case kFromSilu: f16 ? launch_quant<ActF16, kFromSilu>(p, st) : launch_quant<ActBF16, kFromSilu>(p, st); break;
    case kFromF32: launch_quant<ActF16, kFromF32>(p, st); break;
    default: return MI_ERR_ARG;
  }
  return launch_status();
}

}  // namespace qlin
