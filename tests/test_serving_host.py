"""What a network from Sequential.quantize() shares with the network that it was made from,
what it refuses and what it reports: the host side, without a GPU. Weights are laid out by
a kernel, so where a test needs an Int8Linear it stands in empty codes for them."""

from __future__ import annotations

import pytest
import torch

import triton_tagi as tt
from triton_tagi.layers import int8_linear
from triton_tagi.layers.int8_linear import Int8Linear


@pytest.fixture
def codes(monkeypatch):
    """Int8Linear without a GPU: codes of zeros."""
    def zeros(mw, Sw):
        K, N = mw.shape
        z = torch.zeros(N, K, dtype=torch.uint8)
        return int8_linear.Int8Moments(z.to(torch.int8), z, z, torch.zeros(3, N))

    monkeypatch.setattr(int8_linear, "quantize_weights", zeros)


def conv_net():
    d = dict(device="cpu")
    return tt.Sequential([tt.Conv2D(3, 4, 3, padding=1, **d), tt.ReLU(), tt.BatchNorm2D(4, **d),
                          tt.ResBlock(4, 4, **d), tt.ResBlock(4, 8, stride=2, **d)], device="cpu")


def every_layer(net):
    out = []
    for layer in net.layers:
        out.append(layer)
        out += [s for s in vars(layer).values() if isinstance(s, tt.Layer)]
    return out


# -- shared state -------------------------------------------------------------------------


def test_a_served_network_has_layers_of_its_own():
    """No layer, nor any inside a ResBlock, is an object of both networks; what a ResBlock
    walks in its passes is its own too; parameters are shared."""
    net = conv_net()
    served = net.quantize()
    a, b = every_layer(net), every_layer(served)
    assert len(a) == len(b) == 5 + 6 + 9
    assert not {id(x) for x in a} & {id(x) for x in b}
    for block, twin in zip(net.layers[3:], served.layers[3:]):
        own = {id(s) for s in vars(twin).values() if isinstance(s, tt.Layer)}
        assert {id(s) for s in twin._main_layers + twin._proj_layers} == own
        assert {id(s) for s in twin._learnable} < own
        assert [type(s) for s in twin._main_layers] == [type(s) for s in block._main_layers]
        assert twin.conv1.mw is block.conv1.mw and twin.bn2.Sb is block.bn2.Sb


def test_a_served_network_starts_without_what_a_pass_left():
    """Activations that a pass of the network keeps for its backward stay its own."""
    net = conv_net()
    conv, relu, bn = net.layers[:3]
    rms = tt.RMSNorm(4, device="cpu")
    emb = tt.Embedding(5, 4, device="cpu")
    net.layers += [rms, emb]
    t = torch.ones(2)
    conv.input_ma = relu.J = bn.m_hat = rms.ma_in = rms.stream = emb._ids = t
    net.layers[3].relu1.J = net.layers[3].conv2.delta_mw = t
    served = net.quantize()
    assert served.layers[0].input_ma is None and served.layers[1].J is None
    assert served.layers[2].m_hat is None and served.layers[3].relu1.J is None
    assert served.layers[3].conv2.delta_mw is None
    assert served.layers[5].ma_in is None and served.layers[5].stream is None
    assert served.layers[6]._ids is None
    for kept in (conv.input_ma, relu.J, bn.m_hat, rms.ma_in, rms.stream, emb._ids,
                 net.layers[3].relu1.J, net.layers[3].conv2.delta_mw):
        assert kept is t


def test_a_served_network_is_in_eval_mode_with_statistics_of_its_own():
    net = conv_net()
    flags = net._modes()
    for bn in (net.layers[2], net.layers[4].proj_bn):
        bn._stats_allreduce, bn._stats_world = (lambda sums: None), 4
    served = net.quantize()
    served.eval()
    assert net._modes() == flags and all(f for f in flags if f is not None)
    norms = [(a, b) for a, b in zip(every_layer(net), every_layer(served))
             if isinstance(a, tt.BatchNorm2D)]
    assert len(norms) == 6
    for a, b in norms:
        assert a.training and not b.training
        assert b._stats_allreduce is None and b._stats_world == 1
        assert torch.equal(a.running_mean, b.running_mean)
        assert a.running_mean.data_ptr() != b.running_mean.data_ptr()
        assert a.running_var.data_ptr() != b.running_var.data_ptr()
    assert net.layers[2]._stats_allreduce is not None
    assert not any(block.training for block in served.layers[3:])
    with pytest.raises(RuntimeError, match="serves forward"):
        served.train()
    assert not served.layers[2].training
    net.train()
    assert net.layers[2].training and not served.layers[2].training


# -- a served network as a Sequential -----------------------------------------------------


def token_net(E=8, V=12):
    d = dict(device="cpu")
    return tt.Sequential([tt.Embedding(V, E, **d), tt.MultiheadAttentionV2(E, 2, 6, bias=True, **d),
                          tt.RMSNorm(E, **d), tt.Linear(E, V, **d)], device="cpu")


def test_a_served_network_counts_its_parameters(codes):
    net = token_net()
    served = net.quantize()
    assert isinstance(served.layers[1].k_proj, Int8Linear)
    assert served.layers[3].num_parameters == net.layers[3].num_parameters
    assert served.layers[1].num_parameters == net.layers[1].num_parameters
    assert served.num_parameters() == net.num_parameters()
    # what learns: the layers that own parameters in 32 bits
    assert [type(x) for x in served.leaves()] == [tt.Embedding, tt.RMSNorm]
    assert len(net.leaves()) == 6
    for call in (served.layers[1].update, served.layers[3].update):
        with pytest.raises(RuntimeError, match="serves a trained layer"):
            call(2.0)


def test_checkpoints_of_a_served_network_are_refused(codes, tmp_path):
    """A file would lack the 8-bit layers; loading one would write the parameters that the
    served network shares, beside 8-bit weights of before."""
    from triton_tagi.checkpoint import net_state, restore_net_state

    net = token_net()
    served = net.quantize()
    run = tt.RunDir("d", "a", "o", base=str(tmp_path))
    path = run.save_checkpoint(net, 1, {})
    before = [t.clone() for leaf in net.leaves() for t in (leaf.mw, leaf.Sw)]
    for leaf in net.leaves():
        leaf.mw.add_(1.0)
    moved = [t.clone() for leaf in net.leaves() for t in (leaf.mw, leaf.Sw)]
    mixed = tt.Sequential([served.layers[3]], device="cpu")  # built by hand
    for call in (lambda: run.save_checkpoint(served, 2, {}), lambda: net_state(served),
                 lambda: net_state(mixed), lambda: restore_net_state(mixed, {}),
                 lambda: run.load_checkpoint(served, path),
                 lambda: tt.load_model(path, lambda cfg: served, device="cpu")):
        with pytest.raises(RuntimeError, match="8 bits"):
            call()
    assert [p.name for p in run.checkpoints.iterdir()] == [path.name]
    now = [t for leaf in net.leaves() for t in (leaf.mw, leaf.Sw)]
    assert all(torch.equal(a, b) for a, b in zip(now, moved))
    run.load_checkpoint(net, path)  # the network itself
    assert torch.equal(net.layers[0].mw, before[0])


def test_a_linear_too_long_for_8_bits_stays_in_32(codes):
    """More than 33025 inputs: the layer alone refuses, a network serves it in 32 bits."""
    long = tt.Linear(Int8Linear.MAX_IN + 1, 2, device="cpu")
    long.ma_in = torch.ones(1)
    net = tt.Sequential([long, tt.Linear(2, 3, device="cpu"),
                         tt.Linear(Int8Linear.MAX_IN, 1, device="cpu")], device="cpu")
    with pytest.raises(ValueError, match="33025"):
        long.quantize()
    served = net.quantize()
    assert [type(x) for x in served.layers] == [tt.Linear, Int8Linear, Int8Linear]
    assert served.layers[0] is not long and served.layers[0].mw is long.mw
    assert served.layers[0].ma_in is None and long.ma_in is not None
    assert served.num_parameters() == net.num_parameters()


def test_an_attention_too_wide_for_8_bits_stays_in_32(codes, monkeypatch):
    monkeypatch.setattr(Int8Linear, "MAX_IN", 7)
    net = token_net()  # projections of 8 inputs
    served = net.quantize()
    mha, own = served.layers[1], net.layers[1]
    for a, b in zip((mha.q_proj, mha.k_proj, mha.v_proj), (own.q_proj, own.k_proj, own.v_proj)):
        assert type(a) is tt.Linear and a is not b and a.mw is b.mw
    with pytest.raises(RuntimeError, match="serves forward"):
        served.step(None, None, 0.1)


@pytest.mark.parametrize("check", [True, False])
def test_a_served_forward_reads_the_error_word(monkeypatch, check):
    """check_device covers what a served network does, its forward passes: without it a
    kernel that gave up would leave unwritten predictions and no word."""
    from triton_tagi import network

    read = []
    monkeypatch.setattr(network, "check_device_status", lambda: read.append(1))
    net = tt.Sequential([tt.Flatten()], device="cpu", check_device=check)
    x = torch.zeros(2, 3, 4)
    net.forward(x)
    assert not read  # step() reads it for a network that trains
    net.quantize().forward(x)
    assert len(read) == (1 if check else 0)
