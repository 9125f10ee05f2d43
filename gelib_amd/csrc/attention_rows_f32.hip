// The gradients of attention by query rows, float32 (attention_impl.h).
#include "attention_impl.h"

namespace gelib_hip {
template int launch_attention_kernels<kAttnRows, float>(const AttnPlan &, const AttnArgs &, hipStream_t);
}
