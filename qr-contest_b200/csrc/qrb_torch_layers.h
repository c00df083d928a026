// qrb200 -- the layer operators as C++ functions on tensors (libqrb200_torch_ops.so), with their
// gradients, for callers that have made sure that nothing listens for operators (no dispatch mode, no
// tensor subclass, no transform).  All others call torch.ops.qrb200.*.
#pragma once
#include <ATen/ATen.h>

#include <tuple>

namespace qrb200 {

using OptTensor = std::optional<at::Tensor>;

std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm(const at::Tensor& x, const OptTensor& weight,
                                                        const OptTensor& residual, double eps,
                                                        std::optional<at::ScalarType> out_dtype);
std::tuple<at::Tensor, at::Tensor> linear(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                                          const OptTensor& residual, int64_t activation, const OptTensor& x_scale,
                                          const OptTensor& weight_scale, std::optional<at::ScalarType> out_dtype,
                                          bool want_slope);

}  // namespace qrb200
