"""GPU: differential attention, post norms and residual scales together in the fused block node, against the
op-by-op path on the same kernels, and in a trainer."""
from functools import partial

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
MODES = [dict(diff=True), dict(post_norm=True), dict(diff=True, post_norm=True, residual_scale=True)]


@pytest.fixture(autouse=True)
def _status():
    yield
    from imfvideo_b200.ops import kernels as K

    torch.cuda.synchronize()
    K.check_status()


def _net(bs=2, diff=False, **over):
    from imfvideo_b200.models import IMFDiTVideo, flash_jvp_attention
    from imfvideo_b200.models.diff_attn import DiffAttentionImpl

    torch.manual_seed(0)
    net = IMFDiTVideo(input_size=(16, 32), num_frames=4, depth=3, aux_head_depth=1, attn_res_block_size=bs, hidden_size=256,
                      num_heads=4, kv_lora_rank=128, compute_dtype=BF16,
                      attn_impl=partial(DiffAttentionImpl, lam_init=0.4) if diff else flash_jvp_attention, **over)
    with torch.no_grad():
        for p in net.parameters():
            p.add_(torch.randn_like(p) * 0.03)
    return net.cuda()


def _inputs(B=2):
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dx = (torch.randn(B, 16, 4, 16, 32, device="cuda", generator=g) for _ in range(2))
    h = torch.rand(B, device="cuda", generator=g)
    w = 1 + torch.rand(B, device="cuda", generator=g)
    return x, dx, h, w, torch.zeros(B, device="cuda"), torch.ones(B, device="cuda"), torch.tensor([5, 77], device="cuda")[:B]


def _run(net, ins, zero=True):
    from imfvideo_b200.ops.dual import Dual

    x, dx, h, w, lo, hi, y = ins
    if zero:
        net.zero_grad()
    out = net.forward_dual(Dual(x, dx), Dual(h, torch.ones_like(h)), w, lo, hi, y)
    (out["u"].p.square().sum() + out["v"].p.square().sum()).backward()
    return out, {n: p.grad.clone() for n, p in net.named_parameters() if p.grad is not None}


rel = lambda a, b: ((a.float() - b.float()).norm() / (b.float().norm() + 1e-12)).item()


@pytest.mark.parametrize("bs", [0, 2])
@pytest.mark.parametrize("mode", MODES)
def test_fused_block_matches_generic_composition(mode, bs):
    """Outputs, tangent and every gradient.  Both paths round to bf16 at the same places, 2^-8 of a value each,
    but sum in other orders, so single roundings differ: four blocks of some ten roundings in a chain, each half
    a step at most and independent, are 2^-8 sqrt(40) = 2.5e-2 of a value at the very end at most; gradients go
    through the chain twice."""
    from imfvideo_b200.ops import cuda as cu

    net, ins = _net(bs, **mode), _inputs()
    blk = net.shared_blocks[0]
    assert blk.fused_ok(torch.zeros(1, device="cuda"), BF16)
    out_f, g_f = _run(net, ins)
    cu.disable("block")
    try:
        out_g, g_g = _run(net, ins)
    finally:
        cu.enable("block")
    assert rel(out_f["u"].p, out_g["u"].p) < 2.5e-2 and rel(out_f["v"].p, out_g["v"].p) < 2.5e-2
    assert rel(out_f["u"].t, out_g["u"].t) < 2.5e-2 * 2
    assert set(g_f) >= set(g_g)            # (the node returns zeros for a remix that has nothing to mix yet)
    bad = [(n, rel(g_f[n], g_g[n])) for n in g_g if g_g[n].norm() > 0 and rel(g_f[n], g_g[n]) > 5e-2]
    assert not bad, bad


@pytest.mark.parametrize("bs", [0, 2])
def test_gradients_written_straight_into_existing_buffers(bs):
    """With fp32 ``.grad`` buffers attached the node adds to them: the same as through autograd, twice over."""
    net, ins = _net(bs, diff=True, post_norm=True, residual_scale=True), _inputs()
    _, want = _run(net, ins)
    for p in net.parameters():
        p.grad = torch.zeros_like(p)
    before = {n: p.grad.data_ptr() for n, p in net.named_parameters()}
    assert net.shared_blocks[0].fused_sinks().direct()
    for _ in range(2):
        _run(net, ins, zero=False)
    for n, p in net.named_parameters():
        assert p.grad.data_ptr() == before[n], n
        # the returned matrices are rounded to bf16, 2^-8; dQ adds in arrival order
        assert n not in want or rel(p.grad, 2 * want[n]) < 1e-2, n


def test_recomputed_and_8_bit_activations():
    """The same gradients with blocks that are recomputed (nothing else is rounded), and with activations in 8 bits
    within their error: 1/255 of a group's largest value each, a percent of a gradient."""
    ins = _inputs(1)
    mode = dict(diff=True, post_norm=True, residual_scale=True)
    _, want = _run(_net(**mode), ins)
    _, ckpt = _run(_net(grad_checkpoint=True, **mode), ins)
    _, act8 = _run(_net(act_store="int8", **mode), ins)
    assert set(want) == set(ckpt) == set(act8)
    for n in want:
        if want[n].norm() > 0:
            assert rel(ckpt[n], want[n]) < 1e-2 and rel(act8[n], want[n]) < 5e-2, n


def test_no_gradient_pass_keeps_nothing_and_agrees():
    from imfvideo_b200.ops.dual import Dual

    net, (x, dx, h, w, lo, hi, y) = _net(diff=True, post_norm=True), _inputs()
    a = net.forward_dual(Dual(x), Dual(h), w, lo, hi, y)
    with torch.no_grad():
        b = net.forward_dual(Dual(x), Dual(h), w, lo, hi, y)
    assert torch.equal(a["u"].p.detach(), b["u"].p) and torch.equal(a["v"].p.detach(), b["v"].p)


def test_other_head_dims_take_the_formulas():
    """head_dim 128 has no kernel: the plug-in's formulas run, with gradients."""
    from imfvideo_b200.models.diff_attn import DiffAttentionImpl
    from imfvideo_b200.ops import reference as ref

    impl = DiffAttentionImpl(128, 70, 2).cuda()
    assert impl.fused_core is None
    q, k, v = (torch.randn(1, 70, 2, 128, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    o = impl(q, k, v)
    o.sum().backward()
    assert torch.equal(o, ref.diff_attention(q, k, v, impl.lam)) and impl.lam.grad is not None


def test_trainer_steps():
    """Training steps: finite, bit-identical from run to run with ``run.deterministic``, every new parameter moves."""
    from imfvideo_b200.config import apply_overrides, preset
    from imfvideo_b200.ops import kernels as K
    from imfvideo_b200.train import Trainer

    def run():
        cfg = apply_overrides(preset("d256"), {
            "model.attn_impl": "diff_jvp", "model.post_norm": True, "model.residual_scale": True, "model.depth": 3,
            "model.aux_head_depth": 1, "optim.warmup_steps": 0, "run.deterministic": True})
        cfg.data.latent_frames, cfg.data.latent_size = 4, (32, 32)
        tr = Trainer(cfg, device=torch.device("cuda", 0), verbose=False)
        first = {n: p.detach().clone() for n, p in tr.net.named_parameters()}
        g = torch.Generator().manual_seed(7)
        out = []
        for _ in range(3):
            x = torch.randn(1, 16, 4, 32, 32, generator=g).pin_memory()
            out.append(tr.train_step(x, torch.randint(0, 1000, (1,), generator=g)))
        return out, first, {n: p.detach().clone() for n, p in tr.net.named_parameters()}

    try:
        (s1, first, p1), (s2, _, p2) = run(), run()
    finally:
        K.set_deterministic(False)
    assert all(s["loss"] == s["loss"] and not s["skipped"] and s["grad_norm"] > 0 for s in s1)
    assert [s["loss"] for s in s1] == [s["loss"] for s in s2] and all(torch.equal(p1[n], p2[n]) for n in p1)
    new = [n for n in p1 if n.endswith(("attn_impl.lam", "_post_norm.weight"))]
    assert len(new) == 4 * 3 and all(not torch.equal(first[n], p1[n]) for n in new), \
        [n for n in new if torch.equal(first[n], p1[n])]
