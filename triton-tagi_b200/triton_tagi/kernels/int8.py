"""Gaussian rows in 8 bits, and the linear layer's moments from them.

A row of means μ and variances S is held as three rows of codes with one scale each
(``Int8Moments``); value = code × scale:

    q_m   signed    of μ
    q_2   unsigned  of μ² (tokens) or μ² + S (weights)
    q_S   unsigned  of S

which are the operands of the moment product

    μ_z = μ_a μ_w + μ_b,   S_z = μ_a² S_w + S_a (μ_w² + S_w) + S_b

so that both moments come from products of 8-bit integers with exact 32-bit sums and
a scale for each token and each output channel.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from .._lib import call_on, check_f32, check_on, ptr


class Int8Moments(NamedTuple):
    """Codes ``(rows, width)`` and scales ``(3, rows)`` (means, q_2, variances). A row
    that held a value that is not finite has codes 0 and scales NaN."""

    q_m: Tensor
    q_2: Tensor
    q_S: Tensor
    scales: Tensor

    def values(self) -> tuple[Tensor, Tensor, Tensor]:
        """What the codes stand for: three float32 ``(rows, width)`` tensors."""
        dev = check_f32(self.scales)
        q = _checked(self, dev)
        rows, width = q.q_m.shape
        out = [q.scales.new_empty((rows, width)) for _ in range(3)]
        call_on(dev, "tagi_int8_values", *_pointers(q), *(t.data_ptr() for t in out), rows,
                width)
        return tuple(out)


def empty_codes(rows: int, width: int, like: Tensor) -> Int8Moments:
    """Uninitialised codes whose rows start on 16-byte boundaries, as the tensor-core
    product's copies need them."""
    ld = (width + 15) // 16 * 16
    new = like.new_empty_strided
    size, stride = (rows, width), (ld, 1)
    return Int8Moments(new(size, stride, dtype=torch.int8), new(size, stride, dtype=torch.uint8),
                       new(size, stride, dtype=torch.uint8),
                       like.new_empty((3, rows), dtype=torch.float32))


def _ld(t: Tensor) -> int:
    """Bytes between rows of codes (of one row: any multiple of 16 that holds it)."""
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16


def _checked(q: Int8Moments, dev: int) -> Int8Moments:
    """``q`` with the layout the kernels read: unit column stride, one row stride, rows
    on 16-byte boundaries (copied where it differs)."""
    q_m, q_2, q_S, scales = q
    check_on(dev, q_m, q_2, q_S)
    if q_m.dtype != torch.int8 or q_2.dtype != torch.uint8 or q_S.dtype != torch.uint8:
        raise ValueError(f"codes must be int8, uint8, uint8, got {q_m.dtype}, {q_2.dtype}, "
                         f"{q_S.dtype}")
    if q_m.dim() != 2 or q_2.shape != q_m.shape or q_S.shape != q_m.shape \
            or tuple(scales.shape) != (3, q_m.shape[0]):
        raise ValueError(f"codes {tuple(q_m.shape)}, {tuple(q_2.shape)}, {tuple(q_S.shape)} and "
                         f"scales {tuple(scales.shape)} do not belong together")
    ld = _ld(q_m)
    if any(t.stride(1) != 1 or _ld(t) != ld or ld < t.shape[1] or (ld | t.data_ptr()) & 15
           for t in (q_m, q_2, q_S)):
        new = empty_codes(*q_m.shape, scales)
        for a, b in zip(new[:3], (q_m, q_2, q_S)):
            a.copy_(b)
        q = Int8Moments(*new[:3], scales)
    return q if scales.is_contiguous() else q._replace(scales=scales.contiguous())


def _pointers(q: Int8Moments) -> tuple:
    return (q.q_m.data_ptr(), q.q_2.data_ptr(), q.q_S.data_ptr(), q.scales.data_ptr(), _ld(q.q_m))


def _quantize(m: Tensor, S: Tensor, weights: bool) -> Int8Moments:
    dev = check_f32(m, S)
    if m.dim() < 1 or m.shape != S.shape or m.shape[-1] < 1:
        raise ValueError(f"means {tuple(m.shape)} and variances {tuple(S.shape)} must have one "
                         "shape and a last dimension")
    width = m.shape[-1]
    m, S = m.reshape(-1, width).contiguous(), S.reshape(-1, width).contiguous()
    q = empty_codes(m.shape[0], width, m)
    call_on(dev, "tagi_quantize_moments", m.data_ptr(), S.data_ptr(), 1 if weights else 0,
            *_pointers(q), m.shape[0], width)
    return q


def quantize_moments(ma: Tensor, Sa: Tensor) -> Int8Moments:
    """Tokens' moments in 8 bits: the last dimension is a row; leading ones are
    flattened. Negative variances count as 0."""
    return _quantize(ma, Sa, False)


def quantize_weights(mw: Tensor, Sw: Tensor) -> Int8Moments:
    """A ``(K, N)`` weight in 8 bits, one row of K codes for each output channel."""
    if mw.dim() != 2:
        raise ValueError(f"expected a (K, N) weight, got {tuple(mw.shape)}")
    return _quantize(mw.t(), Sw.t(), True)


def int8_moments_matmul(x: Int8Moments, w: Int8Moments, mb: Tensor | None = None,
                        Sb: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """(mz, Sz), each ``(M, N)``: the moments of tokens ``x`` (M, K) through weights
    ``w`` (N, K) plus the biases (N values each, or None)."""
    dev = check_f32(x.scales, w.scales, mb, Sb)
    x, w = _checked(x, dev), _checked(w, dev)
    M, K = x.q_m.shape
    N = w.q_m.shape[0]
    if w.q_m.shape[1] != K:
        raise ValueError(f"Reduction dims disagree: x has {K}, w has {w.q_m.shape[1]}")
    if mb is not None and mb.numel() != N or Sb is not None and Sb.numel() != N:
        raise ValueError(f"biases must hold {N} values")
    mb = None if mb is None else mb.contiguous()
    Sb = None if Sb is None else Sb.contiguous()
    mz = x.scales.new_empty((M, N))
    Sz = torch.empty_like(mz)
    call_on(dev, "tagi_int8_moment_matmul", *_pointers(x), *_pointers(w), ptr(mb), ptr(Sb),
            mz.data_ptr(), Sz.data_ptr(), M, N, K)
    return mz, Sz
