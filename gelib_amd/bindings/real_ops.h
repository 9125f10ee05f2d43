// What gelib_base.cpp needs of real_ops.cpp and point_ops.cpp.
#pragma once

#include <torch/extension.h>

#include "gelib_hip.h"

void bind_real_ops(pybind11::module_ &m);
void bind_point_ops(pybind11::module_ &m);
