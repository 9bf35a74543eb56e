// Bindings of norm, token order and block-scaled product (implemented in op_bindings.cpp).
#pragma once
#include <torch/extension.h>
namespace nep {
void bind_ops(pybind11::module_& m);
}
