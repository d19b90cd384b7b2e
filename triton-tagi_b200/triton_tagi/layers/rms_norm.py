"""Bayesian RMSNorm (drop-in for triton_tagi/layers/rms_norm.py).

Per row over the feature dim (rms_norm.py:93-110):
    inv = 1/√(mean(μ_a² + S_a) + ε)
    μ_z = inv μ_a μ_γ,   S_z = inv² (S_a (μ_γ² + S_γ) + S_γ μ_a²)
Backward (rms_norm.py:115-128): δμ_a = inv μ_γ δμ_z, δS_a = (inv μ_γ)² δS_z;
γ sums Σ inv μ_a δμ_z and Σ inv² μ_a² δS_z over rows (float64).

``forward(ma, Sa, residual=(mr, Sr))`` adds a residual stream first and keeps the sum in
``stream``, in one pass (kernels/norm.py); ``backward(dmz, dSz, stream_delta=(dm, dS))``
then adds the deltas that reached the stream behind the norm and returns the deltas of
both addends. The backward reads the stream, so what follows adds to a tensor of its own
(``Add``, the next norm's ``residual``); after a change in place ``backward`` raises. ``forward_int8`` gives the output in 8 bits for ``Int8Linear`` (no backward).
"""

from __future__ import annotations

import torch
from torch import Tensor

from .._lib import WGRAD_DELTAS, WGRAD_UPDATE, check_cuda_f32, lib, stream
from ..base import LearnableLayer
from ..kernels.int8 import Int8Moments
from ..kernels.norm import (add_rmsnorm, add_rmsnorm_backward, add_rmsnorm_backward_sums,
                            add_rmsnorm_backward_update, add_rmsnorm_int8)
from ..param_init import init_weight_bias_norm
from ._params import contiguous_params


def _version(t: Tensor) -> int:
    """How often ``t`` (or what it is a view of) was changed in place."""
    return 0 if t.is_inference() else t._version


class RMSNorm(LearnableLayer):
    _kept = ("ma_in", "inv_rms", "stream")

    def __init__(self, normalized_shape, eps: float = 1e-6, gain_w: float = 1.0,
                 device="cuda") -> None:
        if isinstance(normalized_shape, int):
            normalized_shape = [normalized_shape]
        if len(normalized_shape) != 1:
            raise ValueError(
                f"RMSNorm only supports a single normalized dimension, got {normalized_shape}")
        self.normalized_shape = list(normalized_shape)
        self.ni = normalized_shape[0]
        self.eps = eps
        self.gain_w = gain_w
        self.device = torch.device(device)
        self.has_bias = False
        self.mw, self.Sw, _, _ = init_weight_bias_norm(self.ni, gain_w=gain_w, gain_b=1.0,
                                                       device=self.device)
        self.mb = self.Sb = None
        self.ma_in = None
        self.inv_rms = None
        self.stream = None  # (means, variances) of input plus residual, when one was given
        self._input_shape = None
        self.delta_mw = self.delta_Sw = self.delta_mb = self.delta_Sb = None

    def _rows_of(self, *ts: Tensor | None) -> tuple:
        """The tensors, of one shape, with rows of ``ni``: as they are, or split where the
        last dimension is a multiple of it (what does not fit, the kernels refuse)."""
        shape = ts[0].shape
        if not shape or shape[-1] == self.ni or shape[-1] % self.ni:
            return ts
        if any(t is not None and t.shape != shape for t in ts):
            raise ValueError(f"RMSNorm: a shape differs from {tuple(shape)}")
        return tuple(None if t is None else t.reshape(-1, self.ni) for t in ts)

    @staticmethod
    def _shaped(shape: torch.Size, *ts: Tensor) -> tuple:
        return ts if ts[0].shape == shape else tuple(t.view(shape) for t in ts)

    def forward(self, ma: Tensor, Sa: Tensor,
                residual: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
        check_cuda_f32(ma, Sa)
        contiguous_params(self, ("mw", "Sw"))
        self._input_shape = ma.shape
        self.stream = None
        if residual is not None:
            hm, hS, mz, Sz, inv = add_rmsnorm(*self._rows_of(ma, Sa, *residual), self.mw, self.Sw,
                                              float(self.eps))
            self.ma_in, self.inv_rms = hm.view(-1, self.ni), inv.view(-1, 1)
            self._stream_version = _version(self.ma_in)
            hm, hS, mz, Sz = self._shaped(ma.shape, hm, hS, mz, Sz)
            self.stream = (hm, hS)
            return mz, Sz
        a = ma.reshape(-1, self.ni).contiguous()
        s = Sa.reshape(-1, self.ni).contiguous()
        rows = a.shape[0]
        mz = torch.empty_like(a)
        Sz = torch.empty_like(a)
        inv = torch.empty(rows, 1, device=a.device)
        lib()("tagi_rmsnorm_forward", a.data_ptr(), s.data_ptr(), self.mw.data_ptr(),
              self.Sw.data_ptr(), mz.data_ptr(), Sz.data_ptr(), inv.data_ptr(), rows, self.ni,
              float(self.eps), stream(a))
        self.ma_in, self.inv_rms = a, inv
        return mz.reshape(self._input_shape), Sz.reshape(self._input_shape)

    def forward_int8(self, ma: Tensor, Sa: Tensor,
                     residual: tuple[Tensor, Tensor] | None = None) -> Int8Moments:
        """The output in 8 bits, flattened to rows of ``normalized_shape`` (inference only:
        nothing is kept for a backward but ``stream``)."""
        contiguous_params(self, ("mw", "Sw"))
        mr, Sr = (None, None) if residual is None else residual
        hm, hS, q = add_rmsnorm_int8(*self._rows_of(ma, Sa, mr, Sr), self.mw, self.Sw,
                                     float(self.eps))
        self.stream = None if residual is None else self._shaped(ma.shape, hm, hS)
        self.ma_in = self.inv_rms = None
        return q

    def _fused_backward(self, dmz, dSz, delta) -> tuple[Tensor, Tensor]:
        if _version(self.ma_in) != self._stream_version:
            raise RuntimeError("RMSNorm.backward: the residual stream was changed in place after "
                               "the forward pass; add to a tensor of its own")
        mode, shape = self._param_mode, dmz.shape
        dmz, dSz, rm, rS = self._rows_of(dmz, dSz, *((None, None) if delta is None else delta))
        head = (dmz, dSz, self.ma_in, self.inv_rms)
        if mode == "deltas":
            d_m, d_S, self.delta_mw, self.delta_Sw = add_rmsnorm_backward(
                *head, self.mw, self.Sw, rm, rS)
        elif mode == "update":
            d_m, d_S = add_rmsnorm_backward_update(*head, self.mw, self.Sw, self._cap, rm, rS)
            self._updated_in_backward = True
        elif mode == "sums":
            sums = self._reducer.buffer(self, 2 * self.ni, torch.float64)
            d_m, d_S = add_rmsnorm_backward_sums(*head, self.mw, sums, rm, rS)
            self._reducer.ready(self)
        else:
            raise ValueError(f"unknown parameter mode {mode!r}")
        return self._shaped(shape, d_m, d_S)

    def backward(self, delta_mz: Tensor, delta_Sz: Tensor,
                 stream_delta: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
        check_cuda_f32(delta_mz, delta_Sz)
        if self.ma_in is None:
            raise RuntimeError("RMSNorm.backward needs a forward pass in 32 bits before it")
        if self.stream is not None:
            return self._fused_backward(delta_mz, delta_Sz, stream_delta)
        if stream_delta is not None:
            raise ValueError("RMSNorm.backward: stream_delta without a residual in the forward")
        shape = delta_mz.shape
        dm = delta_mz.reshape(-1, self.ni).contiguous()
        dS = delta_Sz.reshape(-1, self.ni).contiguous()
        rows = dm.shape[0]
        dma = torch.empty_like(dm)
        dSa = torch.empty_like(dS)
        mode = self._param_mode
        sums = (self._reducer.buffer(self, 2 * self.ni, torch.float64) if mode == "sums"
                else torch.empty(2 * self.ni, device=dm.device, dtype=torch.float64))
        st = stream(dm)
        L = lib()
        L("tagi_rmsnorm_backward", dm.data_ptr(), dS.data_ptr(), self.ma_in.data_ptr(),
          self.inv_rms.data_ptr(), self.mw.data_ptr(), dma.data_ptr(), dSa.data_ptr(),
          sums.data_ptr(), rows, self.ni, st)
        if mode == "deltas":
            self.delta_mw = torch.empty(self.ni, device=dm.device)
            self.delta_Sw = torch.empty(self.ni, device=dm.device)
            L("tagi_apply_vector_sums", sums.data_ptr(), sums[self.ni:].data_ptr(), self.ni,
              WGRAD_DELTAS, None, self.Sw.data_ptr(), self.delta_mw.data_ptr(),
              self.delta_Sw.data_ptr(), 1.0, st)
        elif mode == "update":
            self._apply_sums(sums, self._cap)
            self._updated_in_backward = True
        elif mode == "sums":
            self._reducer.ready(self)
        else:
            raise ValueError(f"unknown parameter mode {mode!r}")
        return dma.reshape(shape), dSa.reshape(shape)

    def _sums_numel(self) -> int:
        return 2 * self.ni

    def _apply_sums(self, sums: Tensor, cap: float) -> None:
        lib()("tagi_apply_vector_sums", sums.data_ptr(), sums[self.ni:].data_ptr(), self.ni,
              WGRAD_UPDATE, self.mw.data_ptr(), self.Sw.data_ptr(), None, None, float(cap),
              stream(sums))

    def update(self, cap_factor: float) -> None:
        from ..update.parameters import update_parameters

        if self._updated_in_backward:
            self._updated_in_backward = False
            return
        if self._param_mode == "sums":
            return
        update_parameters(self.mw, self.Sw, self.delta_mw, self.delta_Sw, cap_factor)

    @property
    def num_parameters(self) -> int:
        return 2 * self.mw.numel()

    def __repr__(self) -> str:
        return f"RMSNorm(normalized_shape={self.normalized_shape}, eps={self.eps}, gain_w={self.gain_w})"
