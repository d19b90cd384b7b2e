"""Token-path operators, further cases: 8-bit products on the CTA-pair route, operators
beside other work on the device, rows of every width class, scales whose squares are not
exact, and what a served network leaves alone.

Tolerances count roundings of u = 2^-24 (half a float32 step, relative), as in
test_gpu_token_path.py, whose plain float64 forms these tests share.
"""

from __future__ import annotations

import pytest
import torch

import test_gpu_token_path as forms
from test_gpu_token_path import DEV, U, gen, operand, plain_linear, rand, randn, within

pytestmark = pytest.mark.gpu


# -- the CTA-pair route of the 8-bit product ----------------------------------------------
# 96 or more tiles of 128 x 128; a pair computes 256 x 256 and there are 74 of them.

PAIRS = [
    # M, N, K
    (3333, 3001, 129),   # 14 x 12 tiles of 256: two and three per pair, all edges ragged
    (5000, 2570, 640),   # 20 x 11: the last channels are 10 of a pair's first CTA alone
    (257, 12300, 40),    # 2 x 49: one token in the last tile; the reduction ends in its block
    (12289, 127, 1),     # 49 x 1: no channel for the second CTA; a reduction of one
    (1536, 1024, 512),   # 6 x 4: no edge at all, fewer tiles than pairs
    (2050, 2305, 1030),  # 9 x 10: more than one round of stages per product
]


@pytest.mark.parametrize("M,N,K", PAIRS)
@pytest.mark.parametrize("bias", [True, False])
def test_int8_moments_matmul_by_pairs(M, N, K, bias):
    """Against the float64 form, over all rows. The sums are exact; each is converted (1
    rounding) and scaled by its token (1); the channel's scale and the bias take 1 on the
    result, and the variance's first product with the bias 1 on a part of it."""
    from triton_tagi._lib import device_status
    from triton_tagi.kernels import int8_moments_matmul

    assert ((M + 127) // 128) * ((N + 127) // 128) >= 96
    g = gen(M + N + K)
    x, w = operand(g, M, K), operand(g, N, K)
    mb, Sb = (randn(g, N), rand(g, N)) if bias else (None, None)
    mz, Sz = int8_moments_matmul(x, w, mb, Sb)
    rm, rS, tm, tS = plain_linear(x, w, mb, Sb)
    within(mz, rm, U * (4 * tm + rm.abs()), "mz")
    within(Sz, rS, U * (4 * tS + 2 * rS.abs()), "Sz")
    again = int8_moments_matmul(x, w, mb, Sb)
    assert torch.equal(mz, again[0]) and torch.equal(Sz, again[1])
    assert device_status() == 0


def test_rows_by_pairs_that_are_not_finite_stay_alone():
    """Scales that are NaN make their own token NaN and no other, in every tile of a pair."""
    from triton_tagi.kernels import int8_moments_matmul

    g = gen(41)
    x, w = operand(g, 3333, 129), operand(g, 3001, 129)
    bad = torch.zeros(3333, dtype=torch.bool, device=DEV)
    bad[[0, 255, 256, 1999, 3332]] = True
    x.scales[:, bad] = float("nan")
    mz, Sz = int8_moments_matmul(x, w)
    assert torch.equal(mz.isnan().all(1), bad) and torch.equal(mz.isnan().any(1), bad)
    assert torch.equal(Sz.isnan().all(1), bad) and torch.equal(Sz.isnan().any(1), bad)


def test_the_abort_path_of_pairs_releases_its_memory_and_reports():
    """As test_the_abort_path_releases_its_memory_and_reports, with several tiles per pair:
    the host's limit makes both CTAs of every pair give up before their first stage."""
    from triton_tagi._lib import device_status, set_wait_limit_ns
    from triton_tagi.kernels import int8_moments_matmul

    g = gen(42)
    x, w = operand(g, 3333, 640), operand(g, 3001, 640)
    ref = int8_moments_matmul(x, w)
    assert device_status(reset=True) == 0
    set_wait_limit_ns(500)
    try:
        int8_moments_matmul(x, w)
        torch.cuda.synchronize()
    finally:
        set_wait_limit_ns(0)
    assert device_status(reset=True) != 0
    assert device_status() == 0
    for _ in range(2):
        got = int8_moments_matmul(x, w)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    assert device_status() == 0
# -- beside other work on the device -----------------------------------------------------


def test_products_in_a_row_beside_training_on_another_stream():
    """8-bit products that are launched while the one before them ends, in both kernels,
    while a Linear trains on another stream (its contractions hold tensor memory too):
    every result is the one of the product alone."""
    import triton_tagi as tt
    from triton_tagi._lib import device_status
    from triton_tagi.kernels import int8_moments_matmul

    g = gen(40)
    sizes = ((16, 512, 512), (40, 1000, 700), (2100, 1300, 300))
    ops = [(operand(g, M, K), operand(g, N, K)) for M, N, K in sizes]
    ref = [int8_moments_matmul(*o) for o in ops]
    net = tt.Sequential([tt.Linear(256, 64, device=DEV), tt.ReLU(), tt.Linear(64, 32, device=DEV)],
                        device=DEV)
    x, y = randn(g, 2048, 256), randn(g, 2048, 32)
    net.step(x, y, 0.1)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            got.append([int8_moments_matmul(*o) for o in ops])
        with torch.cuda.stream(s2):
            net.step(x, y, 0.1)
    torch.cuda.synchronize()
    assert device_status() == 0
    for out in got:
        for a, b in zip(out, ref):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# -- rows of every width class, and values that are not finite -----------------------------


# 129 to 256 vectors of 4 per row: two warps per row; one vector on either side
WIDTHS = [(5, 516), (37, 768), (3, 1020), (6, 1024), (4, 1028)]


@pytest.mark.parametrize("R,D", WIDTHS)
@pytest.mark.parametrize("residual", [True, False])
def test_norm_of_rows_of_two_warps(R, D, residual):
    forms.test_add_rmsnorm(R, D, residual)
    forms.test_add_rmsnorm_int8(R, D, residual)


@pytest.mark.parametrize("R,D", WIDTHS)
@pytest.mark.parametrize("weights", [False, True])
def test_quantize_rows_of_two_warps(R, D, weights):
    forms.test_quantize(R, D, weights)


@pytest.mark.parametrize("D", [5, 512, 768, 4096, 9001])
def test_a_variance_of_minus_infinity_makes_its_row_nan(D):
    """Not finite is not finite, on either side: codes 0 and scales NaN, where a finite
    variance below 0 counts as 0."""
    from triton_tagi.kernels import add_rmsnorm_int8, quantize_moments, quantize_weights

    g = gen(43 + D)
    m, S = randn(g, 5, D), rand(g, 5, D)
    S[1, 0] = -float("inf")
    S[2, D - 1] = -float("inf")
    S[3, D // 2] = -1.0
    bad = torch.tensor([False, True, True, False, False], device=DEV)
    w, Sw = torch.ones(D, device=DEV), torch.full((D,), 0.1, device=DEV)
    for q in (quantize_moments(m, S), quantize_weights(m.t(), S.t()),
              add_rmsnorm_int8(m, S, None, None, w, Sw)[2]):
        assert torch.equal(q.scales.isnan().all(0), bad) and torch.equal(q.scales.isnan().any(0), bad)
        assert not q.q_m[bad].any() and not q.q_2[bad].any() and not q.q_S[bad].any()


# -- scales whose squares are not exact ---------------------------------------------------


@pytest.mark.parametrize("root", [512, 770, 3])
def test_the_square_of_a_scale_is_rounded_once(root):
    """scale = sqrt(512): variances scale by 512, not by the square of sqrt(512) rounded to
    32 bits. Sums of whole numbers are exact, so results are compared for equality."""
    from triton_tagi.kernels import embedding_grad, embedding_lookup

    scale = root ** 0.5
    g = gen(root)
    V, D, n = 40, 24, 3000
    ids = torch.randint(0, V, (n,), device=DEV, generator=g)
    mw, Sw = randn(g, V, D), rand(g, V, D)
    mz, Sz = embedding_lookup(ids, mw, Sw, scale=scale)
    assert torch.equal(mz, mw[ids] * scale)
    assert torch.equal(Sz, Sw[ids] * (scale * scale))
    dm = torch.randint(-3, 4, (n, D), device=DEV, generator=g).float()
    dS = -torch.randint(0, 4, (n, D), device=DEV, generator=g).float()
    for k in (n, 20):  # segments that cross chunks, and ones that do not
        t_m, t_S = (torch.zeros(V, D, device=DEV).index_add_(0, ids[:k], t[:k]) for t in (dm, dS))
        g_m, g_S = embedding_grad(ids[:k], dm[:k], dS[:k], V, scale=scale)
        assert torch.equal(g_m, t_m * scale)
        assert torch.equal(g_S, t_S * (scale * scale))


# -- refusals -------------------------------------------------------------------------------


def test_a_stream_of_other_rows_is_refused():
    """As many values in another shape are not the stream of these deltas."""
    from triton_tagi.kernels import add_rmsnorm_backward

    g = gen(50)
    dm, dS, h, inv, w = randn(g, 6, 4), -rand(g, 6, 4), randn(g, 6, 4), rand(g, 6), rand(g, 4)
    ref = add_rmsnorm_backward(dm, dS, h, inv, w, w)
    got = add_rmsnorm_backward(dm.view(2, 3, 4), dS.view(2, 3, 4), h, inv.view(2, 3), w, w)
    assert all(torch.equal(a.view(b.shape), b) for a, b in zip(got, ref))
    for other in (h.t().contiguous(), h.view(-1), h.view(3, 8)):
        with pytest.raises(ValueError, match="do not match"):
            add_rmsnorm_backward(dm, dS, other, inv, w, w)
