// bindings_operators.h - the module's entry points of window attention and
// distillation, and of rotary positions and paged caches.
#pragma once

#include <pybind11/pybind11.h>

void bind_operators(pybind11::module_ &m);
void bind_paged(pybind11::module_ &m);
