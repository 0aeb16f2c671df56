// Registration of the fused tensor-parallel, model and serving ops (b200ar._C).
#pragma once

#include <pybind11/pybind11.h>

void register_ops(pybind11::module& m);
void register_serving_ops(pybind11::module& m);
