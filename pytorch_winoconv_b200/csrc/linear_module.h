// Native forward and backward of the fully connected layers (linear.py) and the packing of activations (checkpoint.py): layout
// copies, allocation, launches and the autograd node without a trip through Python per call.
#pragma once

#include <cstdint>
#include <initializer_list>
#include <optional>
#include <tuple>

#include <torch/extension.h>

// Raises where the call would be recorded (torch.jit.trace, make_fx, torch.export) or carries a forward-mode gradient: what is
// launched here is seen neither by a tracer, to which the result would be an empty tensor, nor by forward-mode differentiation, to
// which it would be a constant.
void check_eager(const char *what, std::initializer_list<const at::Tensor *> tensors);

// y = act(x weight^T + bias) + residual in x's type (f16 or bf16); act: winoconv_act_t.  weight and bias are of that type or f32
// (the weight is then rounded once, the bias added as it is).  pack: what the backward pass needs of x and of the
// pre-activation is kept in eight bits.
at::Tensor linear_call(const at::Tensor &x, const at::Tensor &weight, const std::optional<at::Tensor> &bias, const std::optional<at::Tensor> &residual,
                       int64_t act, bool pack);

// (e4m3 values of x's shape, scales [..., ceil(C / 32)] as e8m0) of a tensor's rows, and the values they stand for.
std::tuple<at::Tensor, at::Tensor> e4m3_pack(const at::Tensor &x);
at::Tensor e4m3_unpack(const at::Tensor &q, const at::Tensor &scale, at::ScalarType type);
