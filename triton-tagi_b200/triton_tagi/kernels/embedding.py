"""Scaled Gaussian embedding lookup and its gradient over tokens sorted by id.

    lookup   mz = s μ_w[id],  Sz = s² S_w[id]
    grad     g_μ[v] = s Σ δμ,  g_S[v] = s² Σ δS   over the tokens of row v

``layers/embedding.py`` scans all ids once per vocabulary row (the reference's
additions in token order, triton_tagi/layers/embedding.py:112-151); these sort the
tokens first, so their cost does not grow with vocabulary × tokens, and
``embedding_update`` touches only the rows that a token names.

``ids`` may be int64, int32 or float32 (truncated toward zero, as in the layer) of
any shape. Ids outside the table and ``padding_idx`` give zero rows and take no
part in the sums.
"""

from __future__ import annotations

import torch
from torch import Tensor

from .._lib import (WGRAD_DELTAS, WGRAD_SUMS, WGRAD_UPDATE, allocator, call_on, check_f32,
                    check_on, lib, ptr)

_ID_TYPES = {torch.float32: 0, torch.int32: 1, torch.int64: 2}


def _id_type(ids: Tensor) -> int:
    code = _ID_TYPES.get(ids.dtype)
    if code is None:
        raise ValueError(f"token ids must be int64, int32 or float32, got {ids.dtype}")
    return code


def _check_table(mw: Tensor, Sw: Tensor) -> tuple[int, int]:
    shape = mw.shape
    if len(shape) != 2 or shape != Sw.shape:
        raise ValueError(f"expected two (V, D) tables, got {tuple(shape)} and {tuple(Sw.shape)}")
    return shape


def embedding_lookup(ids: Tensor, mw: Tensor, Sw: Tensor, scale: float = 1.0,
                     padding_idx: int = -1) -> tuple[Tensor, Tensor]:
    """(mz, Sz), each ``(*ids.shape, D)``: rows s·mw[id] and s²·Sw[id]."""
    code = _id_type(ids)
    dev = check_f32(mw, Sw)
    check_on(dev, ids)
    V, D = _check_table(mw, Sw)
    ids, mw, Sw = ids.contiguous(), mw.contiguous(), Sw.contiguous()
    n, shape = ids.numel(), ids.shape
    new = allocator(dev)
    mz, Sz = new((n, D), (D, 1), torch.float32), new((n, D), (D, 1), torch.float32)
    call_on(dev, "tagi_embedding_lookup", ids.data_ptr(), code, mw.data_ptr(), Sw.data_ptr(),
            mz.data_ptr(), Sz.data_ptr(), n, V, D, padding_idx, scale)
    if len(shape) != 1:
        mz, Sz = mz.view(*shape, D), Sz.view(*shape, D)
    return mz, Sz


def _grad(mode, ids, dmz, dSz, V, D, scale, padding_idx, mw, Sw, out_m, out_S, cap) -> None:
    code = _id_type(ids)
    dev = check_f32(dmz, dSz, mw, Sw, out_m, out_S)
    check_on(dev, ids)
    n = ids.numel()
    if dmz.shape != dSz.shape or dmz.numel() != n * D or (dmz.dim() and dmz.shape[-1] != D):
        raise ValueError(f"deltas {tuple(dmz.shape)} and {tuple(dSz.shape)} do not match "
                         f"{n} tokens of {D} columns")
    ids, dmz, dSz = ids.contiguous(), dmz.contiguous(), dSz.contiguous()
    wn = lib().size("tagi_embedding_grad_workspace_size", n, D)
    hold = allocator(dev)((wn,), (1,), torch.uint8)
    call_on(dev, "tagi_embedding_grad", ids.data_ptr(), code, dmz.data_ptr(), dSz.data_ptr(), n,
            V, D, padding_idx, scale, mode, ptr(mw), ptr(Sw), ptr(out_m), ptr(out_S), cap,
            hold.data_ptr(), wn)


def embedding_grad(ids: Tensor, dmz: Tensor, dSz: Tensor, num_embeddings: int, scale: float = 1.0,
                   padding_idx: int = -1, Sw: Tensor | None = None,
                   out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
    """(g_μ, g_S), each ``(num_embeddings, D)``: the sums of the deltas over the tokens
    of each row. With ``Sw`` the parameter deltas Sw·g_μ and Sw²·g_S instead.
    ``out``: two contiguous tensors to write."""
    D = dmz.shape[-1] if dmz.dim() else 0
    if num_embeddings < 1 or D < 1:
        raise ValueError("embedding_grad: an empty table")
    if Sw is not None:
        if tuple(Sw.shape) != (num_embeddings, D):
            raise ValueError(f"Sw {tuple(Sw.shape)} is not ({num_embeddings}, {D})")
        Sw = Sw.contiguous()
    if out is None:
        new, size = allocator(check_f32(dmz)), (int(num_embeddings), D)
        g_m, g_S = new(size, (D, 1), torch.float32), new(size, (D, 1), torch.float32)
    else:
        g_m, g_S = out
        for t in out:
            if tuple(t.shape) != (num_embeddings, D) or not t.is_contiguous():
                raise ValueError(f"out must be contiguous ({num_embeddings}, {D}) tensors")
    _grad(WGRAD_SUMS if Sw is None else WGRAD_DELTAS, ids, dmz, dSz, num_embeddings, D,
          float(scale), padding_idx, None, Sw, g_m, g_S, 1.0)
    return g_m, g_S


def embedding_update(ids: Tensor, dmz: Tensor, dSz: Tensor, mw: Tensor, Sw: Tensor,
                     cap_factor: float, scale: float = 1.0, padding_idx: int = -1) -> None:
    """The capped update of (mw, Sw) from the deltas, in place, as ``update_parameters``
    with ``embedding_grad(..., Sw=Sw)`` would apply it to the rows that a token names;
    the other rows are neither read nor written."""
    V, D = _check_table(mw, Sw)
    if not (mw.is_contiguous() and Sw.is_contiguous()):
        raise ValueError("in-place targets must be contiguous")
    _grad(WGRAD_UPDATE, ids, dmz, dSz, V, D, float(scale), padding_idx, mw, Sw, None, None,
          float(cap_factor))
