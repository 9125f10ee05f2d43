// The forward pass of attention, float32 (attention_impl.h).
#include "attention_impl.h"

namespace gelib_hip {
template int launch_attention_kernels<kAttnForward, float>(const AttnPlan &, const AttnArgs &, hipStream_t);
}
