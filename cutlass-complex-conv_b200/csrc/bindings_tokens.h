// Registers the token operators (bindings_tokens.cpp) in the extension.
#pragma once

#include <torch/extension.h>

void register_token_operators(pybind11::module_& m);
