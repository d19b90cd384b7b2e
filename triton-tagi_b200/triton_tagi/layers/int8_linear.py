"""A trained ``Linear`` for serving: weights in 8 bits, both moments from 8-bit products
(kernels/int8.py).

    μ_z = μ_a μ_w + μ_b,   S_z = μ_a² S_w + S_a (μ_w² + S_w) + S_b

with one scale for each token and each output channel of every operand. The weights take
3 bytes instead of 8 and are laid out once, from the ``Linear``'s parameters as they are
at that moment. Inference only.
"""

from __future__ import annotations

import torch
from torch import Tensor

from ..base import Layer
from ..kernels.int8 import Int8Moments, int8_moments_matmul, quantize_moments, quantize_weights


class Int8Linear(Layer):
    """Made by ``Linear.quantize()``; ``Sequential.quantize()`` does so for a network."""

    MAX_IN = 33025  # 255 * 255 * MAX_IN < 2^31: the integer sums hold every reduction

    def __init__(self, linear) -> None:
        if linear.in_features > self.MAX_IN:
            raise ValueError(f"Int8Linear: in_features={linear.in_features} exceeds {self.MAX_IN}, "
                             "the longest reduction that 32-bit sums hold")
        self.in_features, self.out_features = linear.in_features, linear.out_features
        self.has_bias = linear.has_bias
        self.device = linear.mw.device
        self.weight = quantize_weights(linear.mw, linear.Sw)
        self.bias_m = linear.mb.detach().clone().view(-1) if linear.has_bias else None
        self.bias_S = linear.Sb.detach().clone().view(-1) if linear.has_bias else None

    def codes(self, ma: Tensor, Sa: Tensor) -> Int8Moments:
        """The layer's input in 8 bits, leading dimensions flattened to rows."""
        return quantize_moments(ma, Sa)

    def forward_int8(self, x: Int8Moments, leading: torch.Size) -> tuple[Tensor, Tensor]:
        """The layer on tokens that are in 8 bits already; ``leading``: their dimensions."""
        mz, Sz = int8_moments_matmul(x, self.weight, self.bias_m, self.bias_S)
        shape = (*leading, self.out_features)
        return mz.view(shape), Sz.view(shape)

    def forward(self, ma: Tensor, Sa: Tensor) -> tuple[Tensor, Tensor]:
        return self.forward_int8(self.codes(ma, Sa), ma.shape[:-1])

    def backward(self, delta_ma: Tensor, delta_Sa: Tensor) -> tuple[Tensor, Tensor]:
        raise RuntimeError("Int8Linear serves a trained layer: it has no backward pass")

    def update(self, cap_factor: float) -> None:
        raise RuntimeError("Int8Linear serves a trained layer: it has no update")

    @property
    def num_parameters(self) -> int:
        """As the ``Linear``'s: means and variances of weights and biases."""
        return 2 * (self.in_features + (1 if self.has_bias else 0)) * self.out_features

    def __repr__(self) -> str:
        return f"Int8Linear(in={self.in_features}, out={self.out_features}, bias={self.has_bias})"
