"""Residual addition and RMSNorm of Gaussian rows in one pass, and its backward.

    h = (μ_a + μ_r, S_a + S_r)                        the residual stream
    inv = 1/√(mean(μ_h² + S_h) + ε)
    μ_z = inv μ_h μ_γ,  S_z = inv² (S_h (μ_γ² + S_γ) + S_γ μ_h²)

(triton_tagi/layers/rms_norm.py:93-137 after resblock.py:138-154.)
"""

from __future__ import annotations

import torch
from torch import Tensor

from .._lib import (WGRAD_DELTAS, WGRAD_SUMS, WGRAD_UPDATE, allocator, call_on, check_f32,
                    check_on, lib, ptr)
from .int8 import Int8Moments, _pointers, empty_codes


def _rows(name: str, mw: Tensor, Sw: Tensor | None, *ts: Tensor | None) -> tuple[int, int, int]:
    """(device, rows, width) of the tensors given (None: absent), after checking them."""
    dev = check_f32(*ts, mw, Sw)
    first = ts[0]
    width = mw.numel()
    if width < 1 or Sw is not None and Sw.numel() != width:
        raise ValueError(f"{name}: scale parameters of {mw.numel()} and "
                         f"{'no' if Sw is None else Sw.numel()} values")
    shape = first.shape
    if not shape or shape[-1] != width:
        raise ValueError(f"{name}: rows of {width} do not fit shape {tuple(shape)}")
    for t in ts:
        if t is not None and t.shape != shape:
            raise ValueError(f"{name}: shape {tuple(t.shape)} does not fit {tuple(first.shape)} "
                             f"with rows of {width}")
    return dev, first.numel() // width, width


def _pair(name: str, a: Tensor | None, b: Tensor | None) -> None:
    if (a is None) != (b is None):
        raise ValueError(f"{name}: mean and variance must be given together")


def _cont(*ts: Tensor | None) -> list:
    return [None if t is None else t.contiguous() for t in ts]


def add_rmsnorm(ma: Tensor, Sa: Tensor, mr: Tensor | None, Sr: Tensor | None, mw: Tensor,
                Sw: Tensor, eps: float = 1e-6) -> tuple:
    """(μ_h, S_h, μ_z, S_z, inv): the stream, its norm and the rows' 1/rms. Without a
    residual (mr, Sr None) the stream is the input itself."""
    _pair("add_rmsnorm", mr, Sr)
    dev, rows, width = _rows("add_rmsnorm", mw, Sw, ma, Sa, mr, Sr)
    ma, Sa, mr, Sr, mw, Sw = _cont(ma, Sa, mr, Sr, mw, Sw)
    new, size, stride, f32 = allocator(dev), tuple(ma.shape), ma.stride(), torch.float32
    hm, hS = (ma, Sa) if mr is None else (new(size, stride, f32), new(size, stride, f32))
    mz, Sz = new(size, stride, f32), new(size, stride, f32)
    inv = new((rows,), (1,), f32)
    if len(size) != 2:
        inv = inv.view(size[:-1])
    call_on(dev, "tagi_add_rmsnorm_forward", ma.data_ptr(), Sa.data_ptr(), ptr(mr), ptr(Sr),
            mw.data_ptr(), Sw.data_ptr(), hm.data_ptr(), hS.data_ptr(), mz.data_ptr(),
            Sz.data_ptr(), inv.data_ptr(), rows, width, eps)
    return hm, hS, mz, Sz, inv


def add_rmsnorm_int8(ma: Tensor, Sa: Tensor, mr: Tensor | None, Sr: Tensor | None, mw: Tensor,
                     Sw: Tensor, eps: float = 1e-6) -> tuple[Tensor, Tensor, Int8Moments]:
    """(μ_h, S_h, codes): as ``add_rmsnorm`` with the norm's output in 8 bits, leading
    dimensions flattened to rows. The codes do not depend on how a row was summed."""
    _pair("add_rmsnorm_int8", mr, Sr)
    dev, rows, width = _rows("add_rmsnorm_int8", mw, Sw, ma, Sa, mr, Sr)
    ma, Sa, mr, Sr, mw, Sw = _cont(ma, Sa, mr, Sr, mw, Sw)
    hm, hS = ma, Sa
    if mr is not None:
        new, size, stride, f32 = allocator(dev), tuple(ma.shape), ma.stride(), torch.float32
        hm, hS = new(size, stride, f32), new(size, stride, f32)
    q = empty_codes(rows, width, dev)
    call_on(dev, "tagi_add_rmsnorm_int8", ma.data_ptr(), Sa.data_ptr(), ptr(mr), ptr(Sr),
            mw.data_ptr(), Sw.data_ptr(), hm.data_ptr(), hS.data_ptr(), *_pointers(q, width), rows,
            width, eps)
    return hm, hS, q


def _backward(mode, dmz, dSz, hm, inv, mw, Sw, rm, rS, sums=None, d_mw=None, d_Sw=None, cap=1.0):
    name = "add_rmsnorm_backward"
    _pair(name, rm, rS)
    dev, rows, width = _rows(name, mw, Sw, dmz, dSz, rm, rS)
    check_f32(dmz, hm, inv)
    if hm.numel() != rows * width or hm.shape[-1:] != (width,) or inv.numel() != rows:
        raise ValueError(f"{name}: the stream {tuple(hm.shape)} and 1/rms {tuple(inv.shape)} do "
                         f"not match {rows} rows of {width}")
    dmz, dSz, hm, inv, rm, rS = _cont(dmz, dSz, hm, inv, rm, rS)
    new, size, stride, f32 = allocator(dev), tuple(dmz.shape), dmz.stride(), torch.float32
    d_m, d_S = new(size, stride, f32), new(size, stride, f32)
    wn = lib().size("tagi_add_rmsnorm_backward_workspace_size", rows, width)
    hold = new((wn,), (1,), torch.uint8)
    call_on(dev, "tagi_add_rmsnorm_backward", dmz.data_ptr(), dSz.data_ptr(), hm.data_ptr(),
            inv.data_ptr(), ptr(rm), ptr(rS), d_m.data_ptr(), d_S.data_ptr(), mode, ptr(sums),
            mw.data_ptr(), ptr(Sw), ptr(d_mw), ptr(d_Sw), cap, rows, width,
            hold.data_ptr(), wn)
    return d_m, d_S


def add_rmsnorm_backward(dmz: Tensor, dSz: Tensor, hm: Tensor, inv: Tensor, mw: Tensor, Sw: Tensor,
                         rm: Tensor | None = None, rS: Tensor | None = None) -> tuple:
    """(δμ, δS, Δμ_γ, ΔS_γ): the deltas of both branches of the addition,
    inv μ_γ δμ_z + δμ_h and (inv μ_γ)² δS_z + δS_h with the deltas (rm, rS) that reach
    the stream behind the norm (None: none), and the deltas of the scale parameters,
    S_γ Σ inv μ_h δμ_z and S_γ² Σ (inv μ_h)² δS_z."""
    _pair("add_rmsnorm_backward", rm, rS)
    mw, Sw = _cont(mw, Sw)
    new, size, stride = allocator(check_f32(mw, Sw)), tuple(mw.shape), mw.stride()
    d_mw, d_Sw = new(size, stride, torch.float32), new(size, stride, torch.float32)
    d_m, d_S = _backward(WGRAD_DELTAS, dmz, dSz, hm, inv, mw, Sw, rm, rS, d_mw=d_mw, d_Sw=d_Sw)
    return d_m, d_S, d_mw, d_Sw


def add_rmsnorm_backward_sums(dmz, dSz, hm, inv, mw, sums, rm=None, rS=None) -> tuple:
    """(δμ, δS), with the raw sums Σ inv μ_h δμ_z and Σ (inv μ_h)² δS_z written to
    ``sums`` (2 × width float64, contiguous), for a data-parallel reduction."""
    if sums.dtype != torch.float64 or sums.numel() != 2 * mw.numel() or not sums.is_contiguous():
        raise ValueError("sums must hold 2 x width contiguous float64 values")
    check_on(dmz.get_device(), sums)
    return _backward(WGRAD_SUMS, dmz, dSz, hm, inv, mw.contiguous(), None, rm, rS, sums=sums)


def add_rmsnorm_backward_update(dmz, dSz, hm, inv, mw, Sw, cap_factor, rm=None, rS=None) -> tuple:
    """(δμ, δS), with the capped update applied to (mw, Sw) in place."""
    if not (mw.is_contiguous() and Sw.is_contiguous()):
        raise ValueError("in-place targets must be contiguous")
    return _backward(WGRAD_UPDATE, dmz, dSz, hm, inv, mw, Sw, rm, rS, cap=float(cap_factor))
