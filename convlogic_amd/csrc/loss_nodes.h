// The losses' part of the module that nodes.cpp defines, and what its parts share.
#pragma once

#include <ATen/ATen.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

// gradients that cannot be differentiated again
inline torch::autograd::variable_list once_only(torch::autograd::variable_list grads, const char *message)
{
    if (!at::GradMode::is_enabled()) return grads;
    for (at::Tensor &g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(message, (int64_t)grads.size());
    return (*error)(std::move(grads));
}

void add_loss_nodes(pybind11::module_ &m);
