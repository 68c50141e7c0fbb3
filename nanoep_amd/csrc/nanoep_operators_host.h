// What nanoep_torch.cpp, which makes the module, needs of nanoep_operators.cpp.
#ifndef NANOEP_OPERATORS_HOST_H_
#define NANOEP_OPERATORS_HOST_H_

#include <torch/extension.h>

namespace py = pybind11;

namespace nanoep {

// Adds the expert layer's operators to the module.
void bind_operators(py::module_& module);

}  // namespace nanoep

#endif  // NANOEP_OPERATORS_HOST_H_
