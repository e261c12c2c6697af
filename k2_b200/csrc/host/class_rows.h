// Scores of given classes and distillation on torch tensors: class_rows.cc.
#pragma once
#include <torch/extension.h>

// Adds `token_log_probs` and `distillation_loss` to the module.
void BindClassRows(pybind11::module_ &m);
