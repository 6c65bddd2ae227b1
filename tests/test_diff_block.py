"""CPU: models with differential attention, post norms and residual scales -- the dual-number pass against
forward-mode AD, reverse mode against the plain forward, names of parameters, configuration."""
import pytest
import torch

from imfvideo_b200.models import IMFDiTVideo
from imfvideo_b200.models.diff_attn import DiffAttentionImpl
from imfvideo_b200.ops.dual import Dual

KW = dict(input_size=16, num_frames=4, hidden_size=64, depth=3, num_heads=4, aux_head_depth=1, kv_lora_rank=32,
          qk_rope_head_dim=8, mlp_ratio=4.0)
MODES = [dict(diff=True), dict(post_norm=True), dict(diff=True, post_norm=True, residual_scale=True)]


def _net(diff=False, **over):
    from functools import partial

    torch.manual_seed(0)
    kw = {**KW, **over}
    if diff:
        kw["attn_impl"] = partial(DiffAttentionImpl, lam_init=0.4)
    net = IMFDiTVideo(**kw)
    with torch.no_grad():
        for p in net.parameters():
            p.add_(torch.randn_like(p) * 0.05)
    return net


def _inputs(B=2):
    g = torch.Generator().manual_seed(1)
    x, dx = (torch.randn(B, 16, 4, 16, 16, generator=g) for _ in range(2))
    t = torch.rand(B, generator=g)
    r = torch.rand(B, generator=g) * t
    w = 1 + 3 * torch.rand(B, generator=g)
    return x, dx, t, r, w, torch.zeros(B), torch.ones(B), torch.randint(0, 1000, (B,), generator=g)


@pytest.mark.parametrize("bs", [0, 2])
@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("mode", MODES)
def test_dual_pass_matches_functorch(mode, bs, ckpt):
    net = _net(attn_res_block_size=bs, grad_checkpoint=ckpt, **mode)
    x, dx, t, r, w, lo, hi, y = _inputs()
    fn = lambda z, tt, rr: net(z, tt, tt - rr, w, lo, hi, y)
    u0, du0, v0 = torch.func.jvp(fn, (x, t, r), (dx, torch.ones_like(t), torch.zeros_like(t)), has_aux=True)
    out = net.forward_dual(Dual(x, dx), Dual(t - r, torch.ones_like(t)), w, lo, hi, y)
    # 32-bit sums in two orders through four blocks: 1e-5 of values of order one, more of the steeper tangent
    assert du0.abs().max() > 1e-3
    assert torch.allclose(out["u"].p, u0, atol=1e-5) and torch.allclose(out["v"].p, v0, atol=1e-5)
    assert torch.allclose(out["u"].t, du0, atol=2e-4) and out["v"].t is None
    net.zero_grad()
    (out["u"].p.square().sum() + out["v"].p.sum()).backward()
    g1 = {n: p.grad.clone() for n, p in net.named_parameters() if p.grad is not None}
    net.zero_grad()
    uu, vv = net(x, t, t - r, w, lo, hi, y)
    (uu.square().sum() + vv.sum()).backward()
    new = [n for n in g1 if n.endswith(("attn_impl.lam", "_post_norm.weight", "_keep"))]
    assert new and all(g1[n].norm() > 0 for n in new if not n.endswith("_keep"))
    for n, p in net.named_parameters():
        if p.grad is not None:
            assert torch.allclose(g1[n], p.grad, atol=1e-5), n


def test_parameters_are_those_of_the_plain_model_and_the_new_ones():
    plain, full = set(_net().state_dict()), set(_net(diff=True, post_norm=True, residual_scale=True).state_dict())
    assert plain < full
    assert {n.split(".", 2)[2] for n in full - plain} == {"attn.attn_impl.lam", "attn_post_norm.weight",
                                                         "mlp_post_norm.weight", "attn_keep", "mlp_keep"}


def test_plain_tensors_take_the_plug_in():
    impl = DiffAttentionImpl(16, 10, 4)
    q, k, v = (torch.randn(2, 10, 4, 16) for _ in range(3))
    o = impl(q, k, v)
    assert isinstance(o, torch.Tensor) and o.shape == v.shape
    assert torch.equal(o, impl(Dual(q), Dual(k), Dual(v)).p)
    assert impl.fused_core is None


def test_configuration_reaches_the_model():
    from imfvideo_b200.config import apply_overrides, preset
    from imfvideo_b200.train import build_model

    cfg = apply_overrides(preset("tiny"), {"model.attn_impl": "diff_jvp", "model.diff_lam_init": 0.3, "model.post_norm": True,
                                           "model.residual_scale": True})
    net, _, _ = build_model(cfg)
    blk = net.shared_blocks[0]
    assert (blk.attn.attn_impl.lam == 0.3).all() and blk.attn.attn_impl.lam.shape == (1,)
    assert blk.attn_post_norm is not None and (blk.mlp_keep == 1).all()
    net, _, _ = build_model(preset("tiny"))
    assert net.shared_blocks[0].attn_post_norm is None and net.shared_blocks[0].attn_keep is None


def test_refusals():
    with pytest.raises(ValueError):
        DiffAttentionImpl(64, 100, 3)
    with pytest.raises(ValueError):
        IMFDiTVideo(**KW, residual_scale=True)


def test_trainer_steps_on_cpu():
    from imfvideo_b200.config import apply_overrides, preset
    from imfvideo_b200.train import Trainer

    cfg = apply_overrides(preset("tiny"), {"model.attn_impl": "diff_jvp", "model.post_norm": True, "model.residual_scale": True,
                                           "optim.warmup_steps": 0})
    tr = Trainer(cfg, device=torch.device("cpu"), verbose=False)
    lam = tr.net.shared_blocks[0].attn.attn_impl.lam
    before = lam.detach().clone()
    g = torch.Generator().manual_seed(0)
    for _ in range(2):
        st = tr.train_step(torch.randn(2, 16, 4, 16, 16, generator=g), torch.randint(0, 1000, (2,), generator=g))
        assert st["loss"] == st["loss"] and not st["skipped"]
    assert lam.grad is not None and lam.shape == before.shape
