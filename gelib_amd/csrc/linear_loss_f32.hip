// The logits of a linear layer's classes with their loss's epilogues, of this type.
#include "linear_gemm.h"

namespace gelib_hip {

template <>
int launch_loss_gemm<float>(int epilogue, int tile, const GemmArgs &a, hipStream_t s) {
  if (epilogue == kLossSums) launch_tile<float, true, false, kLossSums>(tile, a, s);
  else launch_tile<float, true, false, kLossGrad>(tile, a, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "linear loss launch");
}

}  // namespace gelib_hip
