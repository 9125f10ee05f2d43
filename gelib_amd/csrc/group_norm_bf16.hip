// Group norm of this type.
#include "group_norm_impl.h"

namespace gelib_hip {
template int launch_norm_typed<bhalf_t>(bool, const NormDev &, hipStream_t);
}
