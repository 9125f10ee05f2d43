// The forward pass of attention, bfloat16 (attention_impl.h).
#include "attention_impl.h"

namespace gelib_hip {
template int launch_attention_kernels<kAttnForward, bhalf_t>(const AttnPlan &, const AttnArgs &, hipStream_t);
}
