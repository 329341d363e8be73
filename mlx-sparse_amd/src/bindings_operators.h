// bindings_operators.h - the module's entry points of window attention and
// distillation.
#pragma once

#include <pybind11/pybind11.h>

void bind_operators(pybind11::module_ &m);
