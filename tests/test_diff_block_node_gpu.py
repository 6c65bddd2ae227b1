"""GPU: the fused block node with differential attention and post norms -- the pairs' weights as inputs of the node,
and what the node keeps."""
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


def _kept(act_store, tangent):
    """The storages that a block's node keeps besides its inputs, and the tensors in them."""
    from imfvideo_b200.models.diff_attn import DiffAttentionImpl
    from imfvideo_b200.models.imf_dit_video import TransformerBlock, precompute_axial_rope_3d
    from imfvideo_b200.ops.dual import Dual
    from functools import partial

    torch.manual_seed(0)
    cos, sin = (t.cuda() for t in precompute_axial_rope_3d(16, (3, 5, 9), 20))
    L = cos.shape[0]
    blk = TransformerBlock(256, 4, 128, 128, 48, 16, 64, norm_eps=1e-5,
                           attn_impl=partial(DiffAttentionImpl, seq_len=L, num_heads=4), use_attn_res=True,
                           act_store=act_store, post_norm=True, residual_scale=True).cuda()
    mk = lambda: torch.randn(2, L, 256, device="cuda")
    xs = [Dual(mk().requires_grad_(), mk() if tangent else None) for _ in range(2)]
    saved = []

    def pack(t):
        saved.append(t)
        return t
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = blk.fused_forward(xs[0], xs[1:], False, True, cos, sin, 1e-5)
    assert out.p.grad_fn is not None
    out.p.square().sum().backward()
    inputs = {t.untyped_storage().data_ptr() for t in [x.p for x in xs] + list(blk.parameters()) + [cos, sin]}
    kept = {}
    for t in saved:
        if t.untyped_storage().data_ptr() not in inputs:
            kept.setdefault(t.untyped_storage().data_ptr(), (t.untyped_storage().nbytes(), []))[1].append(t)
    return kept, 2 * L


def test_the_kept_residual_holds_no_tangent():
    kept, rows = _kept("bf16", True)
    mid = [(n, t) for n, ts in kept.values() for t in ts if t.dtype is torch.float32 and t.shape == (rows, 256)]
    assert len(mid) == 1 and mid[0][0] == rows * 256 * 4


def test_8_bit_activations_hold_no_tangents():
    bytes_ = [sum(n for n, _ in _kept("int8", tangent)[0].values()) for tangent in (False, True)]
    assert bytes_[0] == bytes_[1], bytes_


def test_every_residual_scale_moves():
    """Training steps without weight decay: the scales of all residuals but the one that restarts move."""
    from imfvideo_b200.config import apply_overrides, preset
    from imfvideo_b200.train import Trainer

    cfg = apply_overrides(preset("d256"), {
        "model.attn_impl": "diff_jvp", "model.post_norm": True, "model.residual_scale": True, "model.depth": 3,
        "model.aux_head_depth": 1, "optim.warmup_steps": 0, "optim.weight_decay": 0.0})
    cfg.data.latent_frames, cfg.data.latent_size = 4, (32, 32)
    assert cfg.model.attn_res_block_size == 4                # of four blocks only the first begins a residual
    tr = Trainer(cfg, device=torch.device("cuda", 0), verbose=False)
    first = {n: p.detach().clone() for n, p in tr.net.named_parameters() if n.endswith("_keep")}
    g = torch.Generator().manual_seed(7)
    for _ in range(3):
        tr.train_step(torch.randn(1, 16, 4, 32, 32, generator=g).pin_memory(), torch.randint(0, 1000, (1,), generator=g))
    still = [n for n, p in tr.net.named_parameters() if n in first and torch.equal(p, first[n])]
    assert len(first) == 4 * 2 and still == ["shared_blocks.0.attn_keep"], still
