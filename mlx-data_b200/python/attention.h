#pragma once

#include <pybind11/pybind11.h>

// Adds the submodule `attention` to the module.
void bind_attention(pybind11::module_& m);
