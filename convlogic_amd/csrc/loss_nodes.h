// The losses' part of the module that nodes.cpp defines.
#pragma once

#include <torch/csrc/utils/pybind.h>

void add_loss_nodes(pybind11::module_ &m);
