// The matrix products of linear layers of this type.
#include "linear_gemm.h"

namespace gelib_hip {
template int launch_gemm<half_t>(GemmForm, int, const GemmArgs &, hipStream_t);
}
