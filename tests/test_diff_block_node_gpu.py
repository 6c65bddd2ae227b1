"""GPU: the fused block node with differential attention -- the pairs' weights as inputs of the node."""
import pytest
import torch

from test_diff_block_gpu import _inputs, _net, _run, _status, rel  # noqa: F401

pytestmark = pytest.mark.gpu


def _weights(net):
    return {n: p for n, p in net.named_parameters() if n.endswith("attn_impl.lam")}


def _loss(net, ins):
    from imfvideo_b200.ops.dual import Dual

    x, dx, h, w, lo, hi, y = ins
    out = net.forward_dual(Dual(x, dx), Dual(h, torch.ones_like(h)), w, lo, hi, y)
    return out["u"].p.square().sum() + out["v"].p.square().sum()


@pytest.mark.parametrize("bs", [0, 2])
def test_weights_train_alone(bs):
    net, ins = _net(bs, diff=True), _inputs()
    _, want = _run(net, ins)
    net.zero_grad()
    weights = _weights(net)
    for n, p in net.named_parameters():
        p.requires_grad_(n in weights)
    _loss(net, ins).backward()
    for n, p in net.named_parameters():
        assert (p.grad is not None) == (n in weights), n
        # the same kernels on the same values; dQ adds in arrival order
        assert n not in weights or rel(p.grad, want[n]) < 1e-2, n


def test_gradients_are_returned_and_hooks_run():
    net, ins = _net(diff=True), _inputs()
    _, want = _run(net, ins)
    net.zero_grad()
    weights = _weights(net)
    seen = []
    for n, p in weights.items():
        p.register_hook(lambda g, n=n: seen.append(n))
    got = torch.autograd.grad(_loss(net, ins), list(weights.values()))
    for (n, p), g in zip(weights.items(), got):
        assert rel(g, want[n]) < 1e-2 and p.grad is None, n
    assert sorted(seen) == sorted(weights)


def test_weights_changed_before_the_backward_pass():
    net, ins = _net(diff=True), _inputs()
    loss = _loss(net, ins)
    with torch.no_grad():
        next(iter(_weights(net).values())).mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_frozen_weights_get_no_gradient():
    net, ins = _net(diff=True), _inputs()
    for p in _weights(net).values():
        p.requires_grad_(False)
    _, got = _run(net, ins)
    assert got and not any(n.endswith("attn_impl.lam") for n in got)
