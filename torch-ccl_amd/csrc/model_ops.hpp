// Tensor front end of the operators around the collectives, registered with the Python module.
#pragma once

#include <pybind11/pybind11.h>

void register_model_ops(pybind11::module_& m);
