// The gradients of attention by keys, float16 (attention_impl.h).
#include "attention_impl.h"

namespace gelib_hip {
template int launch_attention_kernels<kAttnKeys, half_t>(const AttnPlan &, const AttnArgs &, hipStream_t);
}
