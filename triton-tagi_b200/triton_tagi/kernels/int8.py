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

from .._lib import allocator, call_on, check_f32, check_on, ptr


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
        pointers, rows, width, _hold = _checked(self, dev)
        new, size, stride, f32 = allocator(dev), (rows, width), (width, 1), torch.float32
        v_m, v_2, v_S = new(size, stride, f32), new(size, stride, f32), new(size, stride, f32)
        call_on(dev, "tagi_int8_values", *pointers, v_m.data_ptr(), v_2.data_ptr(), v_S.data_ptr(),
                rows, width)
        return v_m, v_2, v_S


def empty_codes(rows: int, width: int, dev: int) -> Int8Moments:
    """Uninitialised codes whose rows start on 16-byte boundaries, as the tensor-core
    product's copies need them."""
    new, size, stride = allocator(dev), (rows, width), ((width + 15) // 16 * 16, 1)
    return Int8Moments(new(size, stride, torch.int8), new(size, stride, torch.uint8),
                       new(size, stride, torch.uint8), new((3, rows), (rows, 1), torch.float32))


def _checked(q: Int8Moments, dev: int) -> tuple:
    """(pointers and row stride, rows, width, codes) of ``q`` in the layout that the
    kernels read: unit column stride, one row stride, rows on 16-byte boundaries; the
    codes are copied where theirs differs."""
    q_m, q_2, q_S, scales = q
    check_on(dev, q_m, q_2, q_S)
    if q_m.dtype is not torch.int8 or q_2.dtype is not torch.uint8 or q_S.dtype is not torch.uint8:
        raise ValueError(f"codes must be int8, uint8, uint8, got {q_m.dtype}, {q_2.dtype}, "
                         f"{q_S.dtype}")
    shape = q_m.shape
    if len(shape) != 2 or q_2.shape != shape or q_S.shape != shape \
            or scales.shape != (3, shape[0]):
        raise ValueError(f"codes {tuple(shape)}, {tuple(q_2.shape)}, {tuple(q_S.shape)} and "
                         f"scales {tuple(scales.shape)} do not belong together")
    rows, width = shape
    stride = q_m.stride()
    ld = stride[0]
    if rows <= 1:  # the stride of a single row says nothing
        ld = (width + 15) // 16 * 16
        same = q_m.stride(1) == q_2.stride(1) == q_S.stride(1) == 1
    else:
        same = stride[1] == 1 and q_2.stride() == stride and q_S.stride() == stride
    if not same or ld < width \
            or (ld | q_m.data_ptr() | q_2.data_ptr() | q_S.data_ptr()) & 15:
        new = empty_codes(rows, width, dev)
        new.q_m.copy_(q_m)
        new.q_2.copy_(q_2)
        new.q_S.copy_(q_S)
        q_m, q_2, q_S = new[:3]
        ld = (width + 15) // 16 * 16
    scales = scales.contiguous()
    return ((q_m.data_ptr(), q_2.data_ptr(), q_S.data_ptr(), scales.data_ptr(), ld), rows, width,
            (q_m, q_2, q_S, scales))


def _pointers(q: Int8Moments, width: int) -> tuple:
    """Pointers and row stride of codes from ``empty_codes``."""
    return (q.q_m.data_ptr(), q.q_2.data_ptr(), q.q_S.data_ptr(), q.scales.data_ptr(),
            (width + 15) // 16 * 16)


def _quantize(m: Tensor, S: Tensor, weights: bool) -> Int8Moments:
    dev = check_f32(m, S)
    if m.dim() < 1 or m.shape != S.shape or m.shape[-1] < 1:
        raise ValueError(f"means {tuple(m.shape)} and variances {tuple(S.shape)} must have one "
                         "shape and a last dimension")
    width = m.shape[-1]
    rows = m.numel() // width
    m, S = m.contiguous(), S.contiguous()
    q = empty_codes(rows, width, dev)
    call_on(dev, "tagi_quantize_moments", m.data_ptr(), S.data_ptr(), 1 if weights else 0,
            *_pointers(q, width), rows, width)
    return q


def quantize_moments(ma: Tensor, Sa: Tensor) -> Int8Moments:
    """Tokens' moments in 8 bits: the last dimension is a row; leading ones are
    flattened. Finite variances below 0 count as 0."""
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
    px, M, K, _hold_x = _checked(x, dev)
    pw, N, Kw, _hold_w = _checked(w, dev)
    if Kw != K:
        raise ValueError(f"Reduction dims disagree: x has {K}, w has {Kw}")
    if mb is not None and mb.numel() != N or Sb is not None and Sb.numel() != N:
        raise ValueError(f"biases must hold {N} values")
    mb = None if mb is None else mb.contiguous()
    Sb = None if Sb is None else Sb.contiguous()
    new = allocator(dev)
    mz, Sz = new((M, N), (N, 1), torch.float32), new((M, N), (N, 1), torch.float32)
    call_on(dev, "tagi_int8_moment_matmul", *px, *pw, ptr(mb), ptr(Sb),
            mz.data_ptr(), Sz.data_ptr(), M, N, K)
    return mz, Sz
