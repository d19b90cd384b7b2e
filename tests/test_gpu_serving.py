"""Serving and training side by side on a GPU: what a network from Sequential.quantize()
leaves alone, what it answers and what it reports."""

from __future__ import annotations

import pytest
import torch

from test_gpu_token_path import DEV, gen, randn

pytestmark = pytest.mark.gpu


def conv_net(seed=0):
    import triton_tagi as tt

    torch.manual_seed(seed)
    d = dict(device=DEV, gain_w=0.3, gain_b=0.3)
    return tt.Sequential([tt.Conv2D(3, 8, 3, padding=1, **d), tt.ReLU(), tt.BatchNorm2D(8, **d),
                          tt.ResBlock(8, 8, **d), tt.ResBlock(8, 16, stride=2, **d),
                          tt.AvgPool2D(2), tt.Flatten(), tt.Linear(16 * 4 * 4, 10, device=DEV)],
                         device=DEV)


def conv_batch(n, seed):
    g = gen(seed)
    return randn(g, n, 3, 16, 16), randn(g, n, 10)


def everything(net):
    """Parameters and running statistics, in network order."""
    return [getattr(leaf, n) for leaf in net.leaves()
            for n in ("mw", "Sw", "mb", "Sb", "running_mean", "running_var")
            if getattr(leaf, n, None) is not None]


def test_serving_between_the_passes_of_a_network_disturbs_nothing():
    """Forward, a served batch of another size, backward: the deltas and the updates are
    those of a network that nobody served from."""
    from triton_tagi._chain import backward_chain

    x, _ = conv_batch(12, 1)
    other, _ = conv_batch(5, 2)
    g = gen(3)
    dm, dS = randn(g, 12, 10) * 0.1, -randn(g, 12, 10).abs() * 0.1
    out = []
    for serve in (False, True):
        net = conv_net()
        served = net.quantize()
        net.forward(x)
        if serve:
            served.forward(other)
        deltas = backward_chain(net.layers, dm, dS)
        for layer in net.learnable_layers():
            layer.update(2.0)
        out.append([*deltas, *(t for leaf in net.leaves() for t in (leaf.mw, leaf.Sw))])
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_a_network_trains_on_as_if_nobody_had_served_from_it():
    """Served batches between steps, before and after the first one (which initialises the
    BatchNorms): parameters, running statistics and flags are those of a network apart."""
    out = []
    for serve in (False, True):
        net = conv_net()
        served = net.quantize()
        for k in range(3):
            if serve:
                served.forward(conv_batch(5, 10 + k)[0])
                served.eval()
            net.step(*conv_batch(12, k), 0.1)
            served = net.quantize()
        assert all(f for f in net._modes() if f is not None)
        out.append([t.clone() for t in everything(net)])
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_a_served_convolution_network_predicts_as_its_eval_mode_does():
    """The Linear head in 8 bits behind the network's own eval pass; a later step of the
    network moves its running statistics and not the served ones."""
    net = conv_net()
    for k in range(3):
        net.step(*conv_batch(12, k), 0.1)
    served = net.quantize()
    x, _ = conv_batch(6, 20)
    mu, var = served.forward(x)
    net.eval()
    h = net.layers[0].forward(x, torch.zeros_like(x))
    for layer in net.layers[1:-1]:
        h = layer.forward(*h)
    ref_mu, ref_var = net.layers[-1].quantize().forward(*h)
    assert torch.equal(mu, ref_mu) and torch.equal(var, ref_var)
    net.train()
    stats = [t.clone() for leaf in net.leaves() if hasattr(leaf, "running_mean")
             for t in (leaf.running_mean, leaf.running_var)]
    net.step(*conv_batch(12, 3), 0.1)
    now = [t for leaf in net.leaves() if hasattr(leaf, "running_mean")
           for t in (leaf.running_mean, leaf.running_var)]
    assert not any(torch.equal(a, b) for a, b in zip(stats, now))
    own = [t for leaf in served.leaves() if hasattr(leaf, "running_mean")
           for t in (leaf.running_mean, leaf.running_var)]
    assert len(own) == len(stats) and all(torch.equal(a, b) for a, b in zip(stats, own))


def token_net(check_device=None, V=48, E=64, S=12):
    import triton_tagi as tt

    torch.manual_seed(1)
    d = dict(device=DEV)
    return tt.Sequential([tt.Embedding(V, E, scale=0.25, **d), tt.MultiheadAttentionV2(E, 4, S, **d),
                          tt.RMSNorm(E, **d), tt.Linear(E, V, **d)], device=DEV,
                         check_device=check_device)


def tokens(V=48, S=12, B=8):
    return torch.randint(0, V, (B, S), device=DEV, generator=gen(5)).float()


def test_a_served_forward_whose_kernel_gave_up_raises():
    """The host's limit makes the 8-bit kernels give up; with check_device the forward pass
    says so, and the next one is as before. A captured pass is not read (nothing has run)."""
    from triton_tagi._lib import device_status, set_wait_limit_ns

    served = token_net(check_device=True).quantize()
    x = tokens()
    ref = served.forward(x)
    set_wait_limit_ns(500)
    try:
        with pytest.raises(RuntimeError, match="gave up"):
            served.forward(x)
    finally:
        set_wait_limit_ns(0)
    assert device_status() == 0
    got = served.forward(x)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = served.forward(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])


@pytest.mark.parametrize("mode", ["deltas", "update"])
def test_rmsnorm_of_several_rows_per_token(mode):
    """RMSNorm(32) on tokens of 96 norms three rows each: with a residual, and in the
    backward pass, it gives what the same rows give apart."""
    import triton_tagi as tt

    g = gen(7)
    shape = (4, 5, 96)
    ma, mr, dm, xm = (randn(g, *shape) for _ in range(4))
    Sa, Sr, dS, xS = (randn(g, *shape).abs() * 0.1 for _ in range(4))
    a, b = tt.RMSNorm(32, device=DEV), tt.RMSNorm(32, device=DEV)
    rows = lambda t: t.view(-1, 32)  # noqa: E731
    for layer in (a, b):
        layer._set_param_mode(mode, 2.0)
    got = a.forward(ma, Sa, residual=(mr, Sr))
    ref = b.forward(rows(ma), rows(Sa), residual=(rows(mr), rows(Sr)))
    for x, y in zip((*got, *a.stream), (*ref, *b.stream)):
        assert x.shape == shape and torch.equal(rows(x), y)
    got = a.backward(dm, dS, stream_delta=(xm, xS))
    ref = b.backward(rows(dm), rows(dS), stream_delta=(rows(xm), rows(xS)))
    for x, y in zip(got, ref):
        assert x.shape == shape and torch.equal(rows(x), y)
    if mode == "deltas":
        assert torch.equal(a.delta_mw, b.delta_mw) and torch.equal(a.delta_Sw, b.delta_Sw)
    assert torch.equal(a.mw, b.mw) and torch.equal(a.Sw, b.Sw)
    q, p = a.forward_int8(ma, Sa, residual=(mr, Sr)), b.forward_int8(rows(ma), rows(Sa),
                                                                     residual=(rows(mr), rows(Sr)))
    assert all(torch.equal(x, y) for x, y in zip(q, p))
    assert a.stream[0].shape == shape and torch.equal(rows(a.stream[1]), b.stream[1])
    with pytest.raises(ValueError, match="rows of 32"):
        a.forward(ma[..., :50].contiguous(), Sa[..., :50].contiguous(),
                  residual=(mr[..., :50], Sr[..., :50]))
    with pytest.raises(ValueError, match="shape"):  # as many values, other rows
        a.forward(ma, Sa, residual=(mr.view(5, 4, 96), Sr.view(5, 4, 96)))


def test_a_norm_of_several_rows_per_token_is_served():
    """In front of an Int8Linear of the whole token the norm's codes would be rows of
    another width: the served network norms in 32 bits there."""
    import triton_tagi as tt

    torch.manual_seed(2)
    net = tt.Sequential([tt.Linear(16, 96, device=DEV), tt.RMSNorm(32, device=DEV),
                         tt.Linear(96, 10, device=DEV)], device=DEV)
    x = randn(gen(8), 6, 16)
    mu, var = net.forward(x)
    served = net.quantize()
    q_mu, q_var = served.forward(x)
    h = served.layers[1].forward(*served.layers[0].forward(x, torch.zeros_like(x)))
    ref = served.layers[2].forward(*h)
    assert torch.equal(q_mu, ref[0]) and torch.equal(q_var, ref[1])
    rms = lambda t: t.double().square().mean().sqrt().item()  # noqa: E731
    assert rms(q_mu - mu) <= 0.05 * rms(mu) and rms(q_var - var) <= 0.1 * rms(var)


def test_a_stream_changed_in_place_is_refused_by_the_backward():
    """The stream is what the backward pass reads: an addition into it, by this library or
    by torch, would silently change gamma's deltas. A sum of its own is the way."""
    import triton_tagi as tt
    from triton_tagi.layers.resblock import triton_add_shortcut

    g = gen(9)
    ma, mr, dm, xm = (randn(g, 6, 64) for _ in range(4))
    Sa, Sr, dS, xS = (randn(g, 6, 64).abs() * 0.1 for _ in range(4))
    norm = tt.RMSNorm(64, device=DEV)
    norm.forward(ma, Sa, residual=(mr, Sr))
    hm, hS = norm.stream
    kept = hm.clone(), hS.clone()
    out = tt.Add().forward(*norm.stream, xm, xS)
    assert torch.equal(out[0], hm + xm) and torch.equal(hm, kept[0]) and torch.equal(hS, kept[1])
    ref = norm.backward(dm, dS, stream_delta=(xm, xS))
    d_w = norm.delta_mw
    for change in (lambda: triton_add_shortcut(xm, xS, hm, hS), lambda: hm.add_(xm),
                   lambda: hm.view(-1)[:3].zero_()):
        norm.forward(ma, Sa, residual=(mr, Sr))
        hm, hS = norm.stream
        change()
        with pytest.raises(RuntimeError, match="changed in place"):
            norm.backward(dm, dS, stream_delta=(xm, xS))
    norm.forward(ma, Sa, residual=(mr, Sr))
    got = norm.backward(dm, dS, stream_delta=(xm, xS))
    assert all(torch.equal(a, b) for a, b in zip(got, ref)) and torch.equal(norm.delta_mw, d_w)


def test_a_residual_pass_in_inference_mode():
    """Tensors that count no changes are not asked for them."""
    import triton_tagi as tt
    from triton_tagi.layers.resblock import triton_add_shortcut

    g = gen(10)
    norm = tt.RMSNorm(64, device=DEV)
    with torch.inference_mode():
        a, b = randn(g, 4, 64), randn(g, 4, 64).abs()
        norm.forward(a, b, residual=(a, b))
        d_m, _ = norm.backward(a, b)
        triton_add_shortcut(a, b, *norm.stream)
    assert torch.isfinite(d_m).all()


def test_a_transformer_of_width_512_is_served_near_its_own_predictions():
    """Four blocks of attention, norm and a perceptron of 512 - 2048 - 512, head of 64. A
    code is off by 1 / sqrt(12) of a step at random; rows of 512 to 2048 values reach about
    3.5 of their own size, ReLU's 4.5: 0.8 to 1 % per operand, 1.3 % per product, 13
    products in a row and no more gain for an error than for its value: 4.7 % of the
    means' size. Variances take twice that from the means and as much again of their own.
    2.5 times each is allowed."""
    import triton_tagi as tt

    torch.manual_seed(3)
    V, E, S, d = 64, 512, 64, dict(device=DEV)
    layers = [tt.Embedding(V, E, scale=0.25, **d), tt.PositionalEncoding(E, **d)]
    for _ in range(4):
        layers += [tt.MultiheadAttentionV2(E, 8, S, **d), tt.RMSNorm(E, **d),
                   tt.Linear(E, 4 * E, **d), tt.ReLU(), tt.Linear(4 * E, E, **d)]
    net = tt.Sequential(layers + [tt.Linear(E, V, **d)], device=DEV)
    x = tokens(V, S, 4)
    mu, var = net.forward(x)
    q_mu, q_var = net.quantize().forward(x)
    rms = lambda t: t.double().square().mean().sqrt().item()  # noqa: E731
    off_mu, off_var = rms(q_mu - mu) / rms(mu), rms(q_var - var) / rms(var)
    print(f"served means off by {off_mu:.2%}, variances by {off_var:.2%}")
    assert off_mu <= 2.5 * 0.047 and off_var <= 2.5 * 0.14
    assert (q_var > 0).all()
