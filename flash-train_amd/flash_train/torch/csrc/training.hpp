// The operators around a training step's products, added to the binding's module.
#pragma once

#include <torch/extension.h>

void bindTraining(py::module_& m);
