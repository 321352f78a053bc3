// The parts of the extension module that live in files of their own.
#pragma once

#include <torch/extension.h>

void register_linear_ops(pybind11::module& m);
void register_logit_ops(pybind11::module& m);
