"""Refusals and host-side behaviour of the token-path operators that need no GPU."""

from __future__ import annotations

import pytest
import torch

import triton_tagi as tt
from triton_tagi import kernels as K
from triton_tagi._lib import lib

P = 256  # stands for a device pointer; every call here is refused before any launch


def test_cpu_tensors_are_refused():
    x, v = torch.zeros(2, 4), torch.zeros(4)
    ids = torch.zeros(2, dtype=torch.int64)
    t = torch.zeros(3, 4)
    for call in (lambda: K.embedding_lookup(ids, t, t),
                 lambda: K.embedding_grad(ids, x, x, 3),
                 lambda: K.embedding_update(ids, x, x, t, t, 2.0),
                 lambda: K.add_rmsnorm(x, x, x, x, v, v),
                 lambda: K.add_rmsnorm_int8(x, x, None, None, v, v),
                 lambda: K.add_rmsnorm_backward(x, x, x, torch.zeros(2), v, v),
                 lambda: K.quantize_moments(x, x),
                 lambda: K.quantize_weights(x, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    q = K.Int8Moments(x.to(torch.int8), x.to(torch.uint8), x.to(torch.uint8), torch.zeros(3, 2))
    with pytest.raises(ValueError, match="CUDA"):
        K.int8_moments_matmul(q, q)
    with pytest.raises(ValueError, match="CUDA"):
        q.values()


def test_dtypes_are_refused():
    with pytest.raises(ValueError, match="int64, int32 or float32"):
        K.embedding_lookup(torch.zeros(2, dtype=torch.int16), torch.zeros(3, 4), torch.zeros(3, 4))
    with pytest.raises(ValueError, match="float32"):
        K.add_rmsnorm(*(torch.zeros(2, 4, dtype=torch.float64),) * 4, torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="float32"):
        K.quantize_moments(torch.zeros(2, 4, dtype=torch.bfloat16), torch.zeros(2, 4))


def test_residual_halves_go_together():
    x, v = torch.zeros(2, 4), torch.zeros(4)
    with pytest.raises(ValueError, match="together"):
        K.add_rmsnorm(x, x, x, None, v, v)
    with pytest.raises(ValueError, match="together"):
        K.add_rmsnorm_int8(x, x, None, x, v, v)
    with pytest.raises(ValueError, match="together"):
        K.add_rmsnorm_backward(x, x, x, torch.zeros(2), v, v, x, None)


@pytest.mark.parametrize("args,match", [
    ((P, 3, P, P, P, P, 4, 8, 4, -1, 1.0), "id type"),
    ((P, 1, P, P, P, P, -1, 8, 4, -1, 1.0), "bad sizes"),
    ((P, 1, P, P, P, P, 4, 0, 4, -1, 1.0), "bad sizes"),
    ((P, 1, P, P, P, P, 4, 8, 0, -1, 1.0), "bad sizes"),
    ((P, 0, P, P, P, P, 4, 2**24 + 1, 4, -1, 1.0), "float ids"),
    ((None, 1, P, P, P, P, 4, 8, 4, -1, 1.0), "null pointer"),
])
def test_lookup_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        lib()("tagi_embedding_lookup", *args, None)


def test_gradient_refuses():
    L = lib()
    n, V, D = 100, 50, 8
    ws = L.size("tagi_embedding_grad_workspace_size", n, D)
    assert ws > 0 and L.size("tagi_embedding_grad_workspace_size", 0, D) == 0

    def call(ids=P, id_type=2, n=n, V=V, D=D, mode=0, mw=None, Sw=None, out=P, cap=2.0, w=P, wn=ws):
        L("tagi_embedding_grad", ids, id_type, P, P, n, V, D, -1, 1.0, mode, mw, Sw, out, out, cap,
          w, wn, None)

    for kw, match in ((dict(id_type=-1), "id type"), (dict(n=2**30 + 1), "bad sizes"),
                      (dict(D=2**20 + 1), "bad sizes"), (dict(mode=7), "bad mode"),
                      (dict(ids=None), "null pointer"), (dict(out=None), "null pointer"),
                      (dict(mode=1), "null pointer"), (dict(mode=2, out=None), "update args"),
                      (dict(mode=2, mw=P, Sw=P, cap=0.0), "update args"),
                      (dict(w=P + 4), "aligned")):
        with pytest.raises(ValueError, match=match):
            call(**kw)
    for kw in (dict(wn=ws - 1), dict(w=None)):
        with pytest.raises(RuntimeError, match="workspace"):
            call(**kw)


def test_norm_refuses():
    L = lib()
    fwd = lambda mr=P, Sr=P, hm=P, rows=4, ni=8: L(  # noqa: E731
        "tagi_add_rmsnorm_forward", P, P, mr, Sr, P, P, hm, P, P, P, P, rows, ni, 1e-6, None)
    for kw, match in ((dict(rows=-1), "bad sizes"), (dict(ni=0), "bad sizes"),
                      (dict(ni=2**24 + 1), "bad sizes"), (dict(mr=None), "residual"),
                      (dict(hm=None), "residual")):
        with pytest.raises(ValueError, match=match):
            fwd(**kw)
    fwd(rows=0)  # nothing to do
    q = lambda ldq=16, qm=P: L("tagi_add_rmsnorm_int8", P, P, P, P, P, P, P, P, qm, P, P, P, ldq,  # noqa: E731
                               4, 8, 1e-6, None)
    with pytest.raises(ValueError, match="overlap"):
        q(ldq=7)
    with pytest.raises(ValueError, match="null pointer"):
        q(qm=None)
    with pytest.raises(ValueError, match="overlap"):
        L("tagi_quantize_moments", P, P, 0, P, P, P, P, 7, 4, 8, None)
    with pytest.raises(ValueError, match="overlap"):
        L("tagi_int8_values", P, P, P, P, 7, P, P, P, 4, 8, None)
    ws = L.size("tagi_add_rmsnorm_backward_workspace_size", 100, 64)

    def back(rm=None, rS=None, mode=0, sums=P, Sw=None, d=None, cap=1.0, wn=ws):
        L("tagi_add_rmsnorm_backward", P, P, P, P, rm, rS, P, P, mode, sums, P, Sw, d, d, cap, 100,
          64, P, wn, None)

    for kw, match in ((dict(rm=P), "mean and variance"), (dict(sums=None), "bad mode"),
                      (dict(mode=1), "bad mode"), (dict(mode=2, Sw=P, cap=0.0), "bad mode")):
        with pytest.raises(ValueError, match=match):
            back(**kw)
    with pytest.raises(RuntimeError, match="workspace"):
        back(wn=ws - 1)


def test_8bit_product_refuses():
    L = lib()

    def call(x=P, ldx=64, w=P, ldw=64, M=4, N=8, K=64, out=P):
        L("tagi_int8_moment_matmul", x, P, P, P, ldx, w, P, P, P, ldw, None, None, out, P, M, N, K,
          None)

    for kw, match in ((dict(K=0), "bad sizes"), (dict(K=33026, ldx=33040, ldw=33040), "33025"),
                      (dict(M=-1), "bad sizes"), (dict(ldx=48), "overlap"),
                      (dict(x=None), "null pointer"), (dict(out=None), "null pointer"),
                      (dict(x=P + 1), "16-byte"), (dict(ldw=72), "16-byte")):
        with pytest.raises(ValueError, match=match):
            call(**kw)
    call(M=0)
    call(N=0)


def test_layers_describe_themselves_and_refuse():
    emb = tt.Embedding(10, 4, device="cpu", out_scale=2.0)
    assert emb.sorted_grad and "out_scale=2.0" in repr(emb) and "sorted_grad" in repr(emb)
    assert not tt.Embedding(10, 4, device="cpu").sorted_grad
    norm = tt.RMSNorm(4, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        norm.forward(torch.zeros(2, 4), torch.zeros(2, 4),
                     residual=(torch.zeros(2, 4), torch.zeros(2, 4)))
    with pytest.raises(ValueError, match="CUDA"):
        tt.Linear(4, 3, device="cpu").quantize()
    with pytest.raises(ValueError, match="33025"):
        tt.Linear(33026, 1, device="cpu").quantize()
