"""Token-path operators against plain float64 forms: scaled embedding lookup and its
gradient over sorted tokens, residual RMSNorm in 32 and 8 bits, 8-bit linear moments.

Tolerances count roundings of u = 2^-24 (half a float32 step, relative):

* sums over tokens: at most 31 fp32 additions in a chunk of 32 tokens, chunks in
  double, one rounding each for the result, the scale and its square: 34 u Σ|x|;
* 1/rms: a thread adds at most 24 terms here (rows up to 9001 over 512 threads: 18),
  then 5 shuffle levels and 16 warps: 45 u on the mean of positive terms, half of it
  on the root, and 3 roundings: 26 u; the mean output adds 2 (28 u), the variance
  output doubles 1/rms and adds 6 (58 u); 32 u and 64 u are used;
* the backward deltas: 4 roundings of the product and 1 of the addition; the
  parameter sums: 4 per term in fp32, double additions, 4 after them;
* 8-bit products: exact sums; one rounding each for the conversion, the scales'
  product, the product with it, the second term and the bias.

8-bit codes and the residual stream are compared for equality.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def rand(g, *shape):
    return torch.rand(*shape, device=DEV, generator=g)


def within(got, ref, tol, what):
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3e} over its tolerance"


def shifted(t):
    """The same values at an address that is 4 bytes off every wider boundary."""
    buf = torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)
    out = buf[1:].view(t.shape)
    out.copy_(t)
    return out


# -- embedding --------------------------------------------------------------------

TOKENS = [
    # n, V, D, pad, id type, how the ids fall
    (1, 1, 1, -1, torch.int64, "even"),
    (31, 7, 3, -1, torch.int32, "even"),
    (32, 64, 4, 0, torch.float32, "even"),
    (33, 300, 6, -1, torch.int64, "even"),
    (1000, 65536, 130, 5, torch.int32, "even"),
    (2500, 70000, 64, 0, torch.int64, "skew"),
    (4097, 64, 512, -1, torch.float32, "even"),
    (5000, 3, 20, 1, torch.int64, "even"),
    (5000, 1000, 36, -1, torch.int64, "one"),
    (5000, 1000, 36, 7, torch.int64, "pad"),
    (20000, 50021, 257, 0, torch.int32, "skew"),
    (70001, 40000, 8, -1, torch.int64, "skew"),
]


def make_ids(g, n, V, pad, dtype, how):
    if how == "one":
        ids = torch.full((n,), V // 2, device=DEV)
    elif how == "pad":
        ids = torch.full((n,), pad, device=DEV)
    elif how == "skew":
        ids = (torch.exp(rand(g, n).double() * torch.log(torch.tensor(V + 1.0))) - 1).long()
        ids = ids.clamp_(0, V - 1)
    else:
        ids = torch.randint(0, V, (n,), device=DEV, generator=g)
    if how == "even" and n > 8:  # some ids outside the table
        ids[3], ids[7] = -1, V
    return ids.to(dtype)


@pytest.mark.parametrize("n,V,D,pad,dtype,how", TOKENS)
def test_lookup(n, V, D, pad, dtype, how):
    from triton_tagi.kernels import embedding_lookup

    g = gen(n + V + D)
    ids = make_ids(g, n, V, pad, dtype, how)
    mw, Sw = randn(g, V, D), rand(g, V, D)
    for scale in (1.0, 22.5):
        for table in ((mw, Sw), (shifted(mw), shifted(Sw))):
            mz, Sz = embedding_lookup(ids, *table, scale=scale, padding_idx=pad)
            i = ids.long()
            keep = ((i >= 0) & (i < V) & (i != pad)).unsqueeze(-1)
            i = i.clamp(0, V - 1)
            assert torch.equal(mz, torch.where(keep, mw[i] * scale, 0.0))
            assert torch.equal(Sz, torch.where(keep, Sw[i] * (scale * scale), 0.0))


def plain_sums(ids, dm, dS, V, pad, s):
    i = ids.long()
    keep = (i >= 0) & (i < V) & (i != pad)
    i, dm, dS = i[keep], dm.double()[keep], dS.double()[keep]
    z = lambda: torch.zeros(V, dm.shape[-1], device=DEV, dtype=torch.float64)  # noqa: E731
    return [z().index_add_(0, i, x) * f for x, f in
            ((dm, s), (dS, s * s), (dm.abs(), s), (dS.abs(), s * s))]


@pytest.mark.parametrize("n,V,D,pad,dtype,how", TOKENS)
def test_grad_sums_and_deltas(n, V, D, pad, dtype, how):
    from triton_tagi.kernels import embedding_grad

    g = gen(n * 3 + V + D)
    ids = make_ids(g, n, V, pad, dtype, how)
    dm, dS = randn(g, n, D), -rand(g, n, D)
    for s, (a, b) in ((1.0, (dm, dS)), (0.75, (shifted(dm), shifted(dS)))):
        r_m, r_S, t_m, t_S = plain_sums(ids, dm, dS, V, pad, s)
        g_m, g_S = embedding_grad(ids, a, b, V, scale=s, padding_idx=pad)
        within(g_m, r_m, 34 * U * t_m, "g_m")
        within(g_S, r_S, 34 * U * t_S, "g_S")
        again = embedding_grad(ids, a, b, V, scale=s, padding_idx=pad)
        assert torch.equal(g_m, again[0]) and torch.equal(g_S, again[1])
    Sw = rand(g, V, D) + 0.1
    d_m, d_S = embedding_grad(ids, dm, dS, V, scale=0.75, padding_idx=pad, Sw=Sw)
    W = Sw.double()
    within(d_m, r_m * W, 35 * U * t_m * W, "deltas of the means")
    within(d_S, r_S * W * W, 36 * U * t_S * W * W, "deltas of the variances")


@pytest.mark.parametrize("n,V,D,pad,dtype,how", TOKENS)
def test_update_touches_the_named_rows_only(n, V, D, pad, dtype, how):
    from triton_tagi.kernels import embedding_update

    g = gen(n * 7 + V + D)
    ids = make_ids(g, n, V, pad, dtype, how)
    dm, dS = randn(g, n, D) * 0.1, -rand(g, n, D) * 1e-3
    mw, Sw = randn(g, V, D), rand(g, V, D) * 0.5 + 0.5
    m0, S0 = mw.double(), Sw.double()
    s, cap = 0.75, 2.0
    r_m, r_S, t_m, t_S = plain_sums(ids, dm, dS, V, pad, s)
    got_m, got_S = mw.clone(), Sw.clone()
    embedding_update(ids, dm, dS, got_m, got_S, cap, scale=s, padding_idx=pad)
    bound = S0.clamp_min(1e-10).sqrt() / cap
    d_m, d_S = S0 * r_m, S0 * S0 * r_S
    e_m = m0 + d_m.sign() * torch.minimum(d_m.abs(), bound)
    e_S = S0 + d_S.sign() * torch.minimum(d_S.abs(), bound)
    e_S = torch.where(e_S <= 0, 1e-5, e_S)
    # the step carries the sums' error and 4 roundings, the result one more; no
    # variance ends near 0 (0.5 - sqrt(0.5) / 2 > 0.14), so none meets the floor
    assert e_S.min() > 0.1
    within(got_m, e_m, S0 * 34 * U * t_m + 5 * U * (m0.abs() + bound), "mw")
    within(got_S, e_S, S0 * S0 * 34 * U * t_S + 5 * U * (S0 + bound), "Sw")
    named = torch.zeros(V, dtype=torch.bool, device=DEV)
    i = ids.long()
    named[i[(i >= 0) & (i < V) & (i != pad)]] = True
    assert torch.equal(got_m[~named], mw[~named]) and torch.equal(got_S[~named], Sw[~named])


def test_empty_batch_of_tokens():
    from triton_tagi.kernels import embedding_grad, embedding_lookup, embedding_update

    ids = torch.empty(0, device=DEV, dtype=torch.int64)
    mw, Sw = torch.ones(5, 3, device=DEV), torch.ones(5, 3, device=DEV)
    assert embedding_lookup(ids, mw, Sw)[0].shape == (0, 3)
    e = torch.empty(0, 3, device=DEV)
    g_m, g_S = embedding_grad(ids, e, e, 5)
    assert not g_m.any() and not g_S.any()
    embedding_update(ids, e, e, mw, Sw, 2.0)
    assert (mw == 1).all() and (Sw == 1).all()


def test_gradient_against_differences():
    """The lookup is linear in the table, so a difference of its outputs along one entry,
    weighted with the deltas, is that entry's sum; variances enter with the scale squared."""
    from triton_tagi.kernels import embedding_grad, embedding_lookup

    g = gen(31)
    V, D, n, s = 12, 5, 90, 1.5
    ids = torch.randint(0, V, (n,), device=DEV, generator=g)
    mw, Sw = randn(g, V, D), rand(g, V, D)
    dm, dS = randn(g, n, D), -rand(g, n, D)
    g_m, g_S = embedding_grad(ids, dm, dS, V, scale=s, padding_idx=3)
    for v, j in ((0, 0), (3, 1), (7, 4), (11, 2)):
        up = [t.clone() for t in (mw, Sw)]
        for t in up:
            t[v, j] = 0.0
        lo = embedding_lookup(ids, *up, scale=s, padding_idx=3)
        for t in up:
            t[v, j] = 1.0
        hi = embedding_lookup(ids, *up, scale=s, padding_idx=3)
        for a, b, d, got in ((hi[0], lo[0], dm, g_m), (hi[1], lo[1], dS, g_S)):
            diff = (a.double() - b.double()) * d.double()
            assert abs(got[v, j].item() - diff.sum().item()) <= 34 * U * diff.abs().sum().item()


def test_strided_operands():
    """Views with other strides give what their contiguous copies give."""
    from triton_tagi import kernels as K

    g = gen(32)
    wide = [randn(g, 48, 60) for _ in range(4)]
    a = [t[::2, ::3].t() for t in wide]  # 20 x 24
    a[1], a[3] = a[1].abs(), a[3].abs()
    c = [t.contiguous() for t in a]
    w, Sw = rand(g, 48)[::2] + 0.5, rand(g, 24)
    for f in (K.add_rmsnorm, K.add_rmsnorm_int8):
        x, y = f(*a, w, Sw), f(*c, w.contiguous(), Sw)
        for p, q in zip(x, y):
            for u, v in zip(p, q) if isinstance(p, tuple) else ((p, q),):
                assert torch.equal(u, v)
    inv = rand(g, 40)[::2] + 0.5
    x = K.add_rmsnorm_backward(a[0], a[1], a[2], inv, w, Sw, a[3], a[0])
    y = K.add_rmsnorm_backward(c[0], c[1], c[2], inv.contiguous(), w.contiguous(), Sw, c[3], c[0])
    assert all(torch.equal(u, v) for u, v in zip(x, y))
    for f in (K.quantize_moments, K.quantize_weights):
        assert all(torch.equal(u, v) for u, v in zip(f(a[0], a[1]), f(c[0], c[1])))
    ids = torch.randint(0, 20, (30, 2), device=DEV, generator=g)[:, 0]
    x, y = K.embedding_lookup(ids, a[0], a[1]), K.embedding_lookup(ids.contiguous(), c[0], c[1])
    assert all(torch.equal(u, v) for u, v in zip(x, y))
    d = randn(g, 24, 30).t()
    x, y = K.embedding_grad(ids, d, -d, 20), K.embedding_grad(ids.contiguous(), d.contiguous(), -d, 20)
    assert all(torch.equal(u, v) for u, v in zip(x, y))
    with pytest.raises(ValueError, match="contiguous"):
        K.embedding_update(ids, d, d, a[0], a[1], 2.0)


def test_update_of_deltas_that_are_not_numbers():
    """As update_parameters: a NaN delta leaves its parameter, an infinite one moves it by
    the cap."""
    from triton_tagi.kernels import embedding_update
    from triton_tagi.update.parameters import update_parameters

    ids = torch.arange(4, device=DEV)
    dm, dS = torch.zeros(4, 4, device=DEV), torch.zeros(4, 4, device=DEV)
    dm[0, 0], dS[0, 1] = float("nan"), float("nan")
    dm[1, 0], dS[1, 1] = float("inf"), -float("inf")
    dm[2, 2] = -float("inf")
    mw, Sw = torch.ones(6, 4, device=DEV), torch.full((6, 4), 0.25, device=DEV)
    m2, S2 = mw[:4].clone(), Sw[:4].clone()
    update_parameters(m2, S2, S2 * dm, S2 * S2 * dS, 2.0)
    embedding_update(ids, dm, dS, mw, Sw, 2.0)
    assert torch.isfinite(mw).all() and torch.isfinite(Sw).all()
    assert torch.equal(mw[:4], m2) and torch.equal(Sw[:4], S2)
    assert (mw[4:] == 1).all() and (Sw[4:] == 0.25).all()


# -- residual RMSNorm ---------------------------------------------------------------

ROWS = [(1, 1), (3, 5), (130, 64), (7, 127), (5, 128), (33, 512), (9, 1001), (4, 2048),
        (3, 4096), (2, 8192), (3, 8196), (2, 9001)]


def norm_inputs(R, D, seed):
    g = gen(seed)
    return (randn(g, R, D), rand(g, R, D) * 1e-2, randn(g, R, D), rand(g, R, D) * 1e-2,
            1 + 0.1 * randn(g, D), rand(g, D) / D)


def plain_norm(hm, hS, w, Sw, eps):
    hm, hS, w, Sw = (t.double() for t in (hm, hS, w, Sw))
    inv = ((hm * hm + hS).mean(-1, keepdim=True) + eps).rsqrt()
    return inv * hm * w, inv * inv * (hS * (w * w + Sw) + Sw * hm * hm), inv


@pytest.mark.parametrize("R,D", ROWS)
@pytest.mark.parametrize("residual", [True, False])
def test_add_rmsnorm(R, D, residual):
    from triton_tagi.kernels import add_rmsnorm

    ma, Sa, mr, Sr, w, Sw = norm_inputs(R, D, R + D)
    for shift in (False, True):
        a = [shifted(t) if shift else t for t in (ma, Sa, mr, Sr, w, Sw)]
        if not residual:
            a[2] = a[3] = None
        hm, hS, mz, Sz, inv = add_rmsnorm(*a, eps=1e-6)
        if residual:
            assert torch.equal(hm, ma + mr) and torch.equal(hS, Sa + Sr)
        else:
            assert torch.equal(hm, ma) and torch.equal(hS, Sa)
        rm, rS, ri = plain_norm(hm, hS, w, Sw, 1e-6)
        within(inv, ri.squeeze(-1), 26 * U * ri.squeeze(-1), "1/rms")
        within(mz, rm, 32 * U * rm.abs(), "mz")
        within(Sz, rS, 64 * U * rS.abs(), "Sz")


def test_add_rmsnorm_equals_the_layer_after_an_addition():
    import triton_tagi as tt
    from triton_tagi.kernels import add_rmsnorm

    ma, Sa, mr, Sr, w, Sw = norm_inputs(40, 512, 3)
    layer = tt.RMSNorm(512, device=DEV)
    layer.mw, layer.Sw = w.clone(), Sw.clone()
    rm, rS = layer.forward(ma + mr, Sa + Sr)
    got = add_rmsnorm(ma, Sa, mr, Sr, w, Sw)
    assert (got[2] - rm).abs().max() <= 64 * U * rm.abs().max()
    assert (got[3] - rS).abs().max() <= 128 * U * rS.abs().max()


def plain_codes(p, top):
    most = p.abs().amax(-1, keepdim=True).float()
    q = torch.where(most > 0, torch.round(top * (p / most.double())), 0.0)
    return q, most.squeeze(-1)


@pytest.mark.parametrize("R,D", ROWS)
@pytest.mark.parametrize("residual", [True, False])
def test_add_rmsnorm_int8(R, D, residual):
    from triton_tagi.kernels import add_rmsnorm_int8

    ma, Sa, mr, Sr, w, Sw = norm_inputs(R, D, R * 5 + D)
    for shift in (False, True):
        a = [shifted(t) if shift else t for t in (ma, Sa, mr, Sr, w, Sw)]
        if not residual:
            a[2] = a[3] = None
        hm, hS, q = add_rmsnorm_int8(*a, eps=1e-6)
        if residual:
            assert torch.equal(hm, ma + mr) and torch.equal(hS, Sa + Sr)
        inv = plain_norm(hm, hS, w, Sw, 1e-6)[2].squeeze(-1)
        W, SW, H = w.double(), Sw.double(), hm.double()
        p = H * W
        t = hS.double() * (W * W + SW) + SW * H * H
        qm, P = plain_codes(p, 127.0)
        qS, T = plain_codes(t, 255.0)
        r = p / P.double().unsqueeze(-1)
        assert torch.equal(q.q_m.double(), qm)
        assert torch.equal(q.q_2.double(), torch.round(255.0 * r * r))
        assert torch.equal(q.q_S.double(), qS)
        P, T = P.double(), T.double()
        for got, ref in zip(q.scales, (inv * P / 127, (inv * P) ** 2 / 255, inv ** 2 * T / 255)):
            within(got, ref, 64 * U * ref, "scales")
        for got, ref, s in zip(q.values(), q[:3], q.scales):
            assert torch.equal(got, ref.float() * s.unsqueeze(-1))


@pytest.mark.parametrize("R,D", ROWS)
@pytest.mark.parametrize("weights", [False, True])
def test_quantize(R, D, weights):
    from triton_tagi.kernels import quantize_moments, quantize_weights

    g = gen(R * 11 + D)
    m, S = randn(g, R, D), rand(g, R, D) * 1e-2
    S[0, 0] = -1.0  # a variance below 0 counts as 0
    if R > 2:
        m[1], S[1] = 0.0, 0.0
        m[2] *= 1e-18
    q = quantize_weights(m.t(), S.t()) if weights else quantize_moments(m, S)
    d, v = m.double(), S.double().clamp_min(0)
    qm, P = plain_codes(d, 127.0)
    qS, T = plain_codes(v, 255.0)
    r = torch.where(P > 0, d.t() / P.double(), 0.0).t()
    if weights:
        q2, U2 = plain_codes((d * d + S.double()).clamp_min(0), 255.0)
        s2 = U2.double() / 255
    else:
        q2, s2 = torch.round(255.0 * r * r), (P * P).double() / 255
    assert torch.equal(q.q_m.double(), qm)
    assert torch.equal(q.q_2.double(), q2)
    assert torch.equal(q.q_S.double(), qS)
    for got, ref in zip(q.scales, (P.double() / 127, s2, T.double() / 255)):
        # 1e-44: results below the normal range are rounded to its grid
        within(got, ref, 4 * U * ref + 1e-44, "scales")


@pytest.mark.parametrize("D", [5, 512, 4096, 9001])
def test_rows_that_are_not_finite_become_nan(D):
    from triton_tagi.kernels import add_rmsnorm_int8, int8_moments_matmul, quantize_moments

    g = gen(D)
    m, S = randn(g, 6, D), rand(g, 6, D)
    m[1, D // 2] = float("nan")
    m[2, D - 1] = float("inf")
    S[3, 0] = float("nan")
    S[4, D - 1] = float("inf")
    bad = torch.tensor([False, True, True, True, True, False], device=DEV)
    w, Sw = torch.ones(D, device=DEV), torch.full((D,), 0.1, device=DEV)
    z = torch.zeros(6, D, device=DEV)
    for q in (quantize_moments(m, S), add_rmsnorm_int8(m, S, z, z, w, Sw)[2]):
        assert torch.equal(q.scales.isnan().all(0), bad) and torch.equal(q.scales.isnan().any(0), bad)
        assert not q.q_m[bad].any() and not q.q_2[bad].any() and not q.q_S[bad].any()
        wq = quantize_moments(randn(g, 4, D), rand(g, 4, D))
        mz, Sz = int8_moments_matmul(q, wq)
        assert torch.equal(mz.isnan().all(1), bad) and torch.equal(Sz.isnan().all(1), bad)
        assert torch.isfinite(mz[~bad]).all() and torch.isfinite(Sz[~bad]).all()


def test_a_row_of_zeros():
    from triton_tagi.kernels import add_rmsnorm, add_rmsnorm_int8

    z, w = torch.zeros(2, 512, device=DEV), torch.ones(512, device=DEV)
    out = add_rmsnorm(z, z, z, z, w, w, eps=1e-6)
    assert not out[2].any() and not out[3].any()
    assert (out[4] - 1e3).abs().max() <= 1e3 * 8 * U + 1e3 * 2e-8  # eps as a float32: 2e-8 off
    q = add_rmsnorm_int8(z, z, z, z, w, w)[2]
    assert not q.q_m.any() and not q.scales.any()


@pytest.mark.parametrize("R,D", ROWS + [(1000, 36), (4100, 516)])
@pytest.mark.parametrize("stream", [True, False])
def test_add_rmsnorm_backward(R, D, stream):
    from triton_tagi.kernels import add_rmsnorm_backward
    from triton_tagi.kernels.norm import add_rmsnorm_backward_sums, add_rmsnorm_backward_update
    from triton_tagi.update.parameters import update_parameters

    g = gen(R * 13 + D)
    dm, dS, h = randn(g, R, D), -rand(g, R, D), randn(g, R, D)
    inv, w, Sw = rand(g, R) + 0.5, 1 + 0.1 * randn(g, D), rand(g, D)
    rm, rS = (randn(g, R, D), -rand(g, R, D)) if stream else (None, None)
    I, W, H = inv.double().unsqueeze(-1), w.double(), h.double()
    a = I * W * dm.double()
    b = (I * W) ** 2 * dS.double()
    e_m, e_S = (a, b) if rm is None else (a + rm.double(), b + rS.double())
    x = I * H * dm.double()
    y = (I * H) ** 2 * dS.double()
    V = Sw.double()
    for shift in (False, True):
        t = [shifted(v) if shift else v for v in (dm, dS, h)]
        d_m, d_S, d_w, d_Sw = add_rmsnorm_backward(*t, inv, w, Sw, rm, rS)
        within(d_m, e_m, U * (4 * a.abs() + e_m.abs()), "d_m")
        within(d_S, e_S, U * (5 * b.abs() + e_S.abs()), "d_S")
        within(d_w, V * x.sum(0), 8 * U * V * x.abs().sum(0), "delta of gamma's mean")
        within(d_Sw, V * V * y.sum(0), 10 * U * V * V * y.abs().sum(0), "delta of gamma's variance")
    sums = torch.empty(2 * D, device=DEV, dtype=torch.float64)
    s_m, s_S = add_rmsnorm_backward_sums(dm, dS, h, inv, w, sums, rm, rS)
    assert torch.equal(s_m, d_m) and torch.equal(s_S, d_S)
    within(sums[:D], x.sum(0), 4 * U * x.abs().sum(0), "sums")
    within(sums[D:], y.sum(0), 5 * U * y.abs().sum(0), "sums")
    w1, S1 = w.clone(), Sw.clone()
    u_m, u_S = add_rmsnorm_backward_update(dm, dS, h, inv, w1, S1, 2.0, rm, rS)
    assert torch.equal(u_m, d_m) and torch.equal(u_S, d_S)
    w2, S2 = w.clone(), Sw.clone()
    update_parameters(w2, S2, d_w, d_Sw, 2.0)
    assert torch.equal(w1, w2) and torch.equal(S1, S2)


def test_no_rows():
    from triton_tagi.kernels import add_rmsnorm, add_rmsnorm_backward, add_rmsnorm_int8

    e, w = torch.empty(0, 3, 64, device=DEV), torch.ones(64, device=DEV)
    hm, hS, mz, Sz, inv = add_rmsnorm(e, e, e, e, w, w)
    assert mz.shape == (0, 3, 64) and inv.shape == (0, 3)
    q = add_rmsnorm_int8(e, e, e, e, w, w)[2]
    assert q.q_m.shape == (0, 64) and q.values()[0].shape == (0, 64)
    d_m, _, d_w, d_Sw = add_rmsnorm_backward(e, e, hm, inv, w, w, e, e)
    assert d_m.shape == e.shape and not d_w.any() and not d_Sw.any()


def test_backward_is_the_derivative_with_the_rms_held():
    """The deltas are J dmz and J^2 dSz with J = d mz / d h_m at a fixed 1/rms, as
    differences of the plain norm give it."""
    from triton_tagi.kernels import add_rmsnorm, add_rmsnorm_backward

    ma, Sa, mr, Sr, w, Sw = norm_inputs(3, 64, 5)
    hm, hS, mz, Sz, inv = add_rmsnorm(ma, Sa, mr, Sr, w, Sw)
    g = gen(9)
    dm, dS = randn(g, 3, 64), -rand(g, 3, 64)
    d_m, d_S, _, _ = add_rmsnorm_backward(dm, dS, hm, inv, w, Sw)
    f = lambda h: inv.double().unsqueeze(-1) * h * w.double()  # noqa: E731
    J = (f(hm.double() + 0.5) - f(hm.double() - 0.5))
    # the map is linear in h, so the difference is the derivative up to 2^-50
    within(d_m, J * dm.double(), 5 * U * (J * dm.double()).abs(), "d_m")
    within(d_S, J * J * dS.double(), 6 * U * (J * J * dS.double()).abs(), "d_S")


# -- 8-bit linear -------------------------------------------------------------------

LINEAR = [(1, 1, 1), (1, 512, 2048), (3, 7, 15), (16, 128, 16), (17, 130, 31), (40, 515, 127),
          (64, 64, 128), (65, 300, 129), (128, 128, 256), (129, 257, 1000), (300, 777, 1001),
          (515, 1030, 640), (2, 5000, 4100)]


def operand(g, rows, K):
    from triton_tagi.kernels import Int8Moments

    ld = (K + 15) // 16 * 16
    q = [torch.randint(lo, hi, (rows, ld), device=DEV, generator=g).to(t)[:, :K]
         for lo, hi, t in ((-127, 128, torch.int8), (0, 256, torch.uint8), (0, 256, torch.uint8))]
    return Int8Moments(*q, rand(g, 3, rows) * 0.01 + 1e-4)


def plain_linear(x, w, mb, Sb):
    xm, x2, xS = (q.double() for q in x[:3])
    wm, w2, wS = (q.double() for q in w[:3])
    a, b = x.scales.double().unsqueeze(-1), w.scales.double().unsqueeze(1)
    mz = (xm @ wm.t()) * a[0] * b[0]
    t1, t2 = (x2 @ wS.t()) * a[1] * b[2], (xS @ w2.t()) * a[2] * b[1]
    bias = lambda t: 0.0 if t is None else t.double()  # noqa: E731
    return mz + bias(mb), t1 + t2 + bias(Sb), mz.abs(), t1 + t2


@pytest.mark.parametrize("M,N,K", LINEAR)
@pytest.mark.parametrize("bias", [True, False])
def test_int8_moments_matmul(M, N, K, bias):
    from triton_tagi._lib import device_status
    from triton_tagi.kernels import int8_moments_matmul

    g = gen(M + N + K)
    x, w = operand(g, M, K), operand(g, N, K)
    mb, Sb = (randn(g, N), rand(g, N)) if bias else (None, None)
    mz, Sz = int8_moments_matmul(x, w, mb, Sb)
    rm, rS, tm, tS = plain_linear(x, w, mb, Sb)
    within(mz, rm, U * (4 * tm + rm.abs()), "mz")
    within(Sz, rS, U * (5 * tS + rS.abs()), "Sz")
    assert device_status() == 0


def test_int8_moments_matmul_largest_sums():
    """Every code at its limit over the longest reduction: 255^2 * 33025 < 2^31."""
    from triton_tagi.kernels import Int8Moments, int8_moments_matmul

    K, ld = 33025, 33040
    full = lambda r, v, t: torch.full((r, ld), v, device=DEV, dtype=t)[:, :K]  # noqa: E731
    one = lambda r: torch.ones(3, r, device=DEV)  # noqa: E731
    x = Int8Moments(full(2, -127, torch.int8), full(2, 255, torch.uint8), full(2, 255, torch.uint8),
                    one(2))
    w = Int8Moments(full(5, 127, torch.int8), full(5, 255, torch.uint8), full(5, 255, torch.uint8),
                    one(5))
    mz, Sz = int8_moments_matmul(x, w)
    assert (mz == float(-127 * 127 * K)).all()
    ref = 2.0 * 255 * 255 * K
    assert ((Sz.double() - ref).abs() <= 4 * U * ref).all()
    with pytest.raises(ValueError, match="33025"):
        big = operand(gen(1), 2, 33026)
        int8_moments_matmul(big, big)


def test_a_token_gives_the_same_result_in_every_batch():
    """1, 20, 40, 200 and 2100 tokens take different tiles and shares of the reduction; the
    integer sums are exact and the rest is rounded alike."""
    from triton_tagi.kernels import Int8Moments, int8_moments_matmul

    g = gen(14)
    x, w = operand(g, 2100, 1500), operand(g, 1300, 1500)
    mb, Sb = randn(g, 1300), rand(g, 1300)
    mz, Sz = int8_moments_matmul(x, w, mb, Sb)
    for n in (1, 20, 40, 200):
        part = Int8Moments(*(q[:n] for q in x[:3]), x.scales[:, :n])
        a, b = int8_moments_matmul(part, w, mb, Sb)
        assert torch.equal(a, mz[:n]) and torch.equal(b, Sz[:n])


def test_int8_operands_of_other_layouts():
    """Codes whose rows do not start on 16-byte boundaries, and column-strided ones."""
    from triton_tagi.kernels import Int8Moments, int8_moments_matmul

    g = gen(4)
    x, w = operand(g, 20, 37), operand(g, 50, 37)
    ref = int8_moments_matmul(x, w)
    tight = Int8Moments(*(q.contiguous() for q in x[:3]), x.scales)
    wide = Int8Moments(*(q.t().contiguous().t() for q in w[:3]), w.scales.t().contiguous().t())
    got = int8_moments_matmul(tight, wide)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    for r in (0, 7, 19):  # one row of a larger operand
        row = Int8Moments(*(q[r:r + 1] for q in x[:3]), x.scales[:, r:r + 1])
        a, b = int8_moments_matmul(row, w)
        assert torch.equal(a, ref[0][r:r + 1]) and torch.equal(b, ref[1][r:r + 1])
    assert torch.equal(tight.values()[0], x.values()[0])


def test_empty_8bit_operands():
    from triton_tagi.kernels import int8_moments_matmul, quantize_moments

    w = operand(gen(5), 6, 32)
    none = quantize_moments(torch.empty(0, 32, device=DEV), torch.empty(0, 32, device=DEV))
    mz, Sz = int8_moments_matmul(none, w)
    assert mz.shape == (0, 6) and Sz.shape == (0, 6)


def test_the_abort_path_releases_its_memory_and_reports():
    """A limit below 1 microsecond makes every tensor-core launch give up its tiles; the
    next launch works as before."""
    from triton_tagi._lib import device_status, set_wait_limit_ns
    from triton_tagi.kernels import int8_moments_matmul

    g = gen(6)
    x, w = operand(g, 200, 640), operand(g, 300, 640)
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
    got = int8_moments_matmul(x, w)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    assert device_status() == 0


# -- together, captured, on other streams ----------------------------------------------


def token_path(ids, mw, Sw, gw, gS, w, mb, Sb, dm, dS):
    """Tokens into a residual stream, their norm through an 8-bit layer, and the deltas
    back into the table's sums."""
    from triton_tagi.kernels import (add_rmsnorm, add_rmsnorm_backward, add_rmsnorm_int8,
                                     embedding_grad, embedding_lookup, int8_moments_matmul)

    mz, Sz = embedding_lookup(ids, mw, Sw, scale=4.0)
    hm, hS, q = add_rmsnorm_int8(mz, Sz, mz, Sz, gw, gS)
    out = int8_moments_matmul(q, w, mb, Sb)
    _, _, zm, zS, inv = add_rmsnorm(mz, Sz, mz, Sz, gw, gS)
    d_m, d_S, d_w, d_Sw = add_rmsnorm_backward(dm, dS, hm, inv, gw, gS, dm, dS)
    return (*out, hm, hS, d_m, d_S, d_w, d_Sw, *embedding_grad(ids, d_m, d_S, mw.shape[0], 4.0),
            zm, zS)


def path_inputs(seed):
    from triton_tagi.kernels import quantize_weights

    g = gen(seed)
    V, D, N, n = 500, 256, 200, 300
    ids = torch.randint(0, V, (n,), device=DEV, generator=g)
    return (ids, randn(g, V, D), rand(g, V, D) * 1e-2, 1 + 0.1 * randn(g, D), rand(g, D) / D,
            quantize_weights(randn(g, D, N) / 16, rand(g, D, N) / 256), randn(g, N), rand(g, N),
            randn(g, n, D), -rand(g, n, D))


def test_the_path_together_matches_32_bits():
    """The 8-bit layer against the float32 contraction of the same norm: a code is off by
    at most half a step of its row."""
    from triton_tagi._lib import device_status

    args = path_inputs(1)
    ids, mw, Sw, gw, gS, w, mb, Sb, dm, dS = args
    mz, Sz, hm, hS, d_m, d_S, _, _, g_m, g_S, zm, zS = token_path(*args)
    assert device_status() == 0
    wm, w2, wS = w.values()
    step = lambda q, i: 0.5 * q.scales[i].double()  # noqa: E731
    x = zm.double()
    # half a step of the token's code (1/254 of the row's largest) times the weights
    slack = (x.abs().amax(-1, keepdim=True) / 254) * wm.double().abs().sum(1)
    ref = x @ wm.double().t() + mb.double()
    within(mz, ref, slack * 1.001 + 1e-5, "mean through 8 bits")
    sq = (x * x).amax(-1, keepdim=True) / 510 * wS.double().sum(1)
    sv = zS.double().amax(-1, keepdim=True) / 510 * w2.double().sum(1)
    ref = (x * x) @ wS.double().t() + zS.double() @ w2.double().t() + Sb.double()
    within(Sz, ref, (sq + sv) * 1.001 + 1e-5, "variance through 8 bits")
    r_m, r_S, t_m, t_S = plain_sums(ids, d_m, d_S, mw.shape[0], -1, 4.0)
    within(g_m, r_m, 34 * U * t_m, "table sums")


def test_the_path_captured_and_replayed():
    a, b = path_inputs(2), path_inputs(3)
    ref_a, ref_b = token_path(*a), token_path(*b)
    static = [t.clone() if isinstance(t, torch.Tensor) else
              type(t)(*(u.clone() for u in t)) for t in a]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token_path(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_path(*static)
    for inputs, ref in ((a, ref_a), (b, ref_b), (a, ref_a)):
        for s, t in zip(static, inputs):
            for u, v in ([(s, t)] if isinstance(s, torch.Tensor) else zip(s, t)):
                u.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, ref):
            assert torch.equal(got, want)


def test_two_streams_at_once():
    a, b = path_inputs(4), path_inputs(5)
    ref_a, ref_b = token_path(*a), token_path(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        with torch.cuda.stream(s1):
            got.append((token_path(*a), ref_a))
        with torch.cuda.stream(s2):
            got.append((token_path(*b), ref_b))
    torch.cuda.synchronize()
    for out, ref in got:
        for x, y in zip(out, ref):
            assert torch.equal(x, y)


# -- through the layers -----------------------------------------------------------------


def small_net(sorted_grad, seed=0, V=50, E=32, S=12, **kw):
    import triton_tagi as tt

    torch.manual_seed(seed)
    d = dict(device=DEV)
    return tt.Sequential([tt.Embedding(V, E, scale=0.25, sorted_grad=sorted_grad, **d, **kw),
                          tt.PositionalEncoding(E, **d), tt.MultiheadAttentionV2(E, 4, S, **d),
                          tt.RMSNorm(E, **d), tt.Linear(E, 64, **d), tt.ReLU(),
                          tt.Linear(64, V, **d)], device=DEV)


def small_batch(V=50, S=12, B=8):
    g = gen(11)
    x = torch.randint(0, V, (B, S), device=DEV, generator=g)
    y = torch.nn.functional.one_hot(x.flip(1), V).float()
    return x.float(), y


@pytest.mark.parametrize("fuse", [True, False])
def test_a_sorted_gradient_trains_as_the_scan_does(fuse):
    """The same step with either gradient: rows sum at most 96 deltas, so the sums differ by
    at most 2 x 96 roundings, and the updates by that share of a capped step."""
    x, y = small_batch()
    nets = [small_net(s) for s in (False, True)]
    for net in nets:
        net.fuse_update = fuse
    for a, b in zip(nets[0].leaves(), nets[1].leaves()):
        for n in ("mw", "Sw"):
            getattr(b, n).copy_(getattr(a, n))
    before = nets[0].layers[0].mw.clone(), nets[0].layers[0].Sw.clone()
    outs = [net.step(x, y, 0.05) for net in nets]
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    a, b = nets[0].layers[0], nets[1].layers[0]
    named = torch.zeros(50, dtype=torch.bool, device=DEV)
    named[x.long()] = True
    assert not torch.equal(a.mw[named], before[0][named])
    assert torch.equal(b.mw[~named], before[0][~named]) and torch.equal(b.Sw[~named], before[1][~named])
    bound = before[1].clamp_min(1e-10).sqrt() / 2.0  # no step is longer
    for got, ref, old in ((b.mw, a.mw, before[0]), (b.Sw, a.Sw, before[1])):
        # a step is a product with Sw and Sw^2 of sums whose terms may cancel: compare
        # with the sums' absolute size through the bound, generously
        assert ((got - ref).abs() <= 1e-3 * bound + 4 * U * old.abs()).all()


def test_a_scaled_embedding_equals_a_scaled_table():
    """Looking up s w is looking up w' = s w: forward outputs match those of a scaled table,
    and the deltas are Sw s sum(dm), Sw^2 s^2 sum(dS)."""
    import triton_tagi as tt

    emb = tt.Embedding(40, 24, device=DEV, out_scale=3.0, padding_idx=2)
    g = gen(12)
    ids = torch.randint(0, 40, (6, 5), device=DEV, generator=g).float()
    mz, Sz = emb.forward(ids, torch.zeros_like(ids))
    i, keep = ids.long(), (ids != 2).unsqueeze(-1)
    assert torch.equal(mz, torch.where(keep, emb.mw[i] * 3.0, 0.0))
    assert torch.equal(Sz, torch.where(keep, emb.Sw[i] * 9.0, 0.0))
    dm, dS = randn(g, 6, 5, 24), -rand(g, 6, 5, 24)
    emb.backward(dm, dS)
    r_m, r_S, t_m, t_S = plain_sums(ids.view(-1), dm.view(-1, 24), dS.view(-1, 24), 40, 2, 3.0)
    W = emb.Sw.double()
    within(emb.delta_mw, W * r_m, 35 * U * W * t_m, "delta_mw")
    within(emb.delta_Sw, W * W * r_S, 36 * U * W * W * t_S, "delta_Sw")


def test_a_sorted_gradient_for_a_reducer():
    """Under data parallelism the raw sums go to the reducer's buffer, and the update is
    applied from there."""
    import triton_tagi as tt

    class Buffers:
        def buffer(self, layer, numel, dtype):
            self.buf = torch.full((numel,), 7.0, dtype=dtype, device=DEV)
            return self.buf

        def ready(self, layer):
            self.told = layer

    emb = tt.Embedding(33, 7, device=DEV, sorted_grad=True)
    g = gen(21)
    ids = torch.randint(0, 33, (4, 9), device=DEV, generator=g).float()
    emb.forward(ids, torch.zeros_like(ids))
    red = Buffers()
    emb._set_param_mode("sums", 2.0, red)
    dm, dS = randn(g, 4, 9, 7), -rand(g, 4, 9, 7)
    emb.backward(dm, dS)
    assert red.told is emb
    r_m, r_S, t_m, t_S = plain_sums(ids.view(-1), dm.view(-1, 7), dS.view(-1, 7), 33, -1, 1.0)
    got = red.buf.view(2, 33, 7)
    within(got[0], r_m, 34 * U * t_m, "sums of the means")
    within(got[1], r_S, 34 * U * t_S, "sums of the variances")
    m0 = emb.mw.clone()
    emb.update(2.0)
    assert torch.equal(emb.mw, m0)  # the reducer applies them
    emb._apply_sums(red.buf, 2.0)
    assert not torch.equal(emb.mw, m0)


@pytest.mark.parametrize("mode", ["deltas", "update", "sums"])
def test_rmsnorm_with_a_residual_equals_addition_and_norm(mode):
    """RMSNorm.forward(residual=) and backward(stream_delta=) against triton_add_shortcut,
    the plain layer and triton_delta_merge, in every parameter mode."""
    import triton_tagi as tt
    from triton_tagi.layers.resblock import triton_add_shortcut

    class Buffers:
        def buffer(self, layer, numel, dtype):
            layer.buf = torch.empty(numel, dtype=dtype, device=DEV)
            return layer.buf

        def ready(self, layer):
            layer.told = True

    D = 96
    ma, Sa, mr, Sr, w, Sw = norm_inputs(60, D, 8)
    shape = (5, 12, D)
    ma, Sa, mr, Sr = (t.view(shape) for t in (ma, Sa, mr, Sr))
    g = gen(13)
    dm, dS, xm, xS = randn(g, *shape), -rand(g, *shape), randn(g, *shape), -rand(g, *shape)
    a, b = tt.RMSNorm(D, device=DEV), tt.RMSNorm(D, device=DEV)
    for layer in (a, b):
        layer.mw, layer.Sw = w.clone(), Sw.clone()
        layer._set_param_mode(mode, 2.0, Buffers())
    hm, hS = mr.clone(), Sr.clone()
    triton_add_shortcut(ma, Sa, hm, hS)
    ref = a.forward(hm, hS)
    got = b.forward(ma, Sa, residual=(mr, Sr))
    assert torch.equal(b.stream[0], hm) and torch.equal(b.stream[1], hS)
    for x, y in zip(got, ref):
        assert (x - y).abs().max() <= 128 * U * y.abs().max()
    r_m, r_S = a.backward(dm, dS)
    triton_add_shortcut(xm, xS, r_m, r_S)
    d_m, d_S = b.backward(dm, dS, stream_delta=(xm, xS))
    assert d_m.shape == shape
    assert (d_m - r_m).abs().max() <= 128 * U * r_m.abs().max()
    assert (d_S - r_S).abs().max() <= 256 * U * r_S.abs().max()
    if mode == "sums":
        assert b.told and (b.buf - a.buf).abs().max() <= 256 * U * a.buf.abs().max()
    elif mode == "deltas":
        for n in ("delta_mw", "delta_Sw"):
            x, y = getattr(b, n), getattr(a, n)
            assert (x - y).abs().max() <= 256 * U * y.abs().max()
        b.update(2.0)
        assert not torch.equal(b.mw, w)
    else:
        assert (b.mw - a.mw).abs().max() <= 256 * U * a.mw.abs().max()
        assert (b.Sw - a.Sw).abs().max() <= 256 * U * a.Sw.abs().max()
    plain = tt.RMSNorm(D, device=DEV)
    plain.forward(ma, Sa)
    with pytest.raises(ValueError, match="stream_delta"):
        plain.backward(dm, dS, stream_delta=(xm, xS))


def test_a_quantized_network_serves_its_predictions():
    """Sequential.quantize(): predictions near the float32 network's, the fused 8-bit norm
    equal to norm and quantization apart, and no training through it."""
    import triton_tagi as tt
    from triton_tagi.layers.int8_linear import Int8Linear

    net = small_net(False, V=48, E=64)
    x, y = small_batch(V=48)
    for _ in range(3):
        net.step(x, y, 0.05)
    mu, var = net.forward(x)
    served = net.quantize()
    twice = served.quantize()
    assert all(a is b for a, b in zip((twice.layers[4], twice.layers[2].q_proj),
                                      (twice.layers[4], served.layers[2].q_proj)))
    assert isinstance(served.layers[4], Int8Linear)
    assert isinstance(served.layers[2].q_proj, Int8Linear)
    assert isinstance(net.layers[4], tt.Linear) and isinstance(net.layers[2].q_proj, tt.Linear)
    q_mu, q_var = served.forward(x)
    # half a step of 127 on both operands of each of five products in a row, the errors
    # of 64 terms adding up at random: a few hundredths of the outputs' own size
    rms = lambda t: t.double().square().mean().sqrt().item()  # noqa: E731
    assert rms(q_mu - mu) <= 0.05 * rms(mu)
    assert rms(q_var - var) <= 0.1 * rms(var)
    assert (q_var > 0).all()
    h = served.layers[2].forward(*served.layers[1].forward(
        *served.layers[0].forward(x, torch.zeros_like(x))))
    fused = served.layers[4].forward_int8(served.layers[3].forward_int8(*h), h[0].shape[:-1])
    apart = served.layers[4].forward(*served.layers[3].forward(*h))
    assert rms(fused[0] - apart[0]) <= 1e-3 * rms(apart[0])
    assert rms(fused[1] - apart[1]) <= 1e-3 * rms(apart[1])
    with pytest.raises(RuntimeError, match="serves forward"):
        served.step(x, y, 0.05)
    with pytest.raises(RuntimeError, match="no backward"):
        served.layers[4].backward(mu, var)
    served.layers[3].forward_int8(*h)
    with pytest.raises(RuntimeError, match="32 bits"):
        served.layers[3].backward(*h)
    # serving in the middle of a pass of the network itself disturbs nothing
    ref = net.layers[3].forward(*h)
    kept = net.layers[3].ma_in
    served.forward(x)
    assert net.layers[3].ma_in is kept and net.layers[2].q_proj.ma_in is not None
    assert torch.equal(net.layers[3].forward(*h)[0], ref[0])
    codes = served.layers[4].weight.q_m.clone()
    net.step(x, y, 0.05)  # it trains on, the served weights stay
    assert torch.equal(codes, served.layers[4].weight.q_m)


def test_a_served_network_replays_from_a_graph():
    net = small_net(False)
    x, _ = small_batch()
    served = net.quantize()
    ref = served.forward(x)
    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        served.forward(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = served.forward(static)
    other = x.flip(0).contiguous()
    for inputs in (x, other, x):
        static.copy_(inputs)
        graph.replay()
        torch.cuda.synchronize()
        want = served.forward(inputs)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert torch.equal(out[0], ref[0])


@pytest.mark.parametrize("kw", [dict(out_scale=4.0), dict(sorted_grad=True)])
def test_the_embedding_step_captured(kw):
    """Sequential(cuda_graph=True) with the sorted gradient: replays equal eager steps."""
    x, y = small_batch()
    sorted_grad = kw.pop("sorted_grad", False)
    nets = [small_net(sorted_grad, **kw) for _ in range(2)]
    nets[1].cuda_graph = True
    for k in range(4):
        xb = x.roll(k, 0).contiguous()
        a = nets[0].step(xb, y, 0.05)
        b = nets[1].step(xb, y, 0.05)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(nets[0].layers[0].mw, nets[1].layers[0].mw)
    assert torch.equal(nets[0].layers[0].Sw, nets[1].layers[0].Sw)
    nets[1].release_graph()
