// Torch face (arguments, allocation, gradients) of the operators around a block's matrix products.
#pragma once
#include <pybind11/pybind11.h>

namespace pccl {
void bind_block_ops(pybind11::module_& m);
}
