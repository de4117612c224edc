// Launches of int8_quant.hpp.
#include "int8_quant.hpp"
#include "../../include/mi355x_qlinear.h"

#include <type_traits>

namespace qlin {

template <int V>
using Int = std::integral_constant<int, V>;

template <class Act, int FROM, int TPR, int NV>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void int8_quant_kernel(const QuantArgs p) {
  int8_quant_rows<Act, FROM, TPR, NV>(p, blockIdx.x);
}

// A thread's chain is as long as its pieces, and a row's barriers as dear as its wavefronts.  With a product of 64 columns behind them, us, as below /
// with the other count of threads: SiLU 2 x 14336 8.4 / 9.4 (256 threads), 2048 x 14336 41.5 / 44.2 (256), 43.3 (512), 2048 x 4096 14.2 / 15.1 (256);
// rows of 8192 17.7 / 19.1 (256), 8192 rows of 4096 27.4 / 28.8 (512), 1000 rows of 4096 with the norm 13.0 / 13.4 (512), 16.6 (64); 2048 rows of 512 6.8 /
// 7.4 (256).
template <class Act, int FROM>
static void launch_quant(const QuantArgs& p, hipStream_t st) {
  const int pieces = p.K / 8;
  auto go = [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
    hipLaunchKernelGGL((int8_quant_kernel<Act, FROM, TPR, NV>), dim3((unsigned)(TPR == 64 ? (p.rows + 3) / 4 : p.rows)), dim3(TPR == 64 ? 256 : TPR), 0, st, p);
  };
  // a grid has less than 2^32 threads: past it rows take 256 threads, and are read again where those do not hold them (rows < 2^24: int8_sizes)
  const auto grid_holds = [&](long long threads) { return p.rows * threads < 1LL << 32; };
  if (pieces <= 64) go(Int<64>{}, Int<1>{});
  else if (pieces <= 128) go(Int<64>{}, Int<2>{});
  else if (pieces <= 256) go(Int<256>{}, Int<1>{});
  else if (pieces <= 512 && FROM != kFromSilu) go(Int<256>{}, Int<2>{});
  else if (!grid_holds(pieces <= 1024 ? 512 : 1024)) go(Int<256>{}, Int<0>{});
  else if (pieces <= 512) go(Int<512>{}, Int<1>{});
  else if (pieces <= 1024) go(Int<512>{}, Int<2>{});
  else if (pieces <= 2048) go(Int<1024>{}, Int<2>{});
  else go(Int<1024>{}, Int<0>{});
}

int launch_int8_quant(int from, const QuantArgs& p, int act_dtype, hipStream_t st) {
  if (!p.rows) return MI_OK;
  if (p.rows > kInt8MaxRows) return MI_ERR_SHAPE;
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
