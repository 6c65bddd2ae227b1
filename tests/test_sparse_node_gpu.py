"""GPU: the fused block node with block-sparse attention -- the mixing logits as inputs of the node."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _net(kind):
    from imfvideo_b200.config import preset
    from imfvideo_b200.train import build_model

    cfg = preset("d256")
    cfg.model.depth, cfg.model.aux_head_depth = 2, 1
    cfg.model.attn_impl = kind
    cfg.model.sla2_topk, cfg.model.sla2_bq, cfg.model.sla2_bk = 0.25, 128, 64
    cfg.model.sla2_tile = (4, 4, 4)
    cfg.data.latent_frames, cfg.data.latent_size = 8, (16, 32)      # grid (8, 8, 16) -> 16 tiles
    torch.manual_seed(0)
    net = build_model(cfg)[0].cuda()
    net.compute_dtype = torch.bfloat16
    with torch.no_grad():
        for p in net.parameters():
            p.add_(torch.randn_like(p) * 0.03)
    return net, {n: p for n, p in net.named_parameters() if n.endswith("alpha_logit")}


def _loss(net):
    from imfvideo_b200.ops.dual import Dual

    g = torch.Generator(device="cuda").manual_seed(1)
    x, dx = (torch.randn(1, 16, 8, 16, 32, device="cuda", generator=g) for _ in range(2))
    one, zero = torch.ones(1, device="cuda"), torch.zeros(1, device="cuda")
    out = net.forward_dual(Dual(x, dx), Dual(0.4 * one, one), 1.5 * one, zero, one, torch.tensor([7], device="cuda"))
    return out["u"].p.square().sum() + out["v"].p.square().sum()


rel = lambda a, b: ((a - b).norm() / b.norm()).item()


@pytest.mark.parametrize("linear_kernels", [True, False])
@pytest.mark.parametrize("kind", ["sla2_jvp", "sla2_cube_qat"])
def test_mixing_logits(kind, linear_kernels, monkeypatch):
    """Returned by ``torch.autograd.grad``; trained alone; added in place to a buffer that is there; a change between
    the passes is noticed."""
    from imfvideo_b200.ops import linattn as LA

    assert LA.AVAILABLE
    monkeypatch.setattr(LA, "AVAILABLE", linear_kernels)
    net, alphas = _net(kind)
    assert net.shared_blocks[0].fused_ok(torch.zeros(1, device="cuda"), torch.bfloat16)
    _loss(net).backward()
    want = {n: p.grad.clone() for n, p in alphas.items()}
    net.zero_grad()
    # the same kernels on the same values; dQ adds in arrival order
    for (n, p), g in zip(alphas.items(), torch.autograd.grad(_loss(net), list(alphas.values()))):
        assert want[n].norm() > 0 and rel(g, want[n]) < 1e-2 and p.grad is None, n
    for n, p in net.named_parameters():
        p.requires_grad_(n in alphas)
    buffers = {n: torch.ones_like(p) for n, p in alphas.items()}
    for n, p in alphas.items():
        p.grad = buffers[n]
    _loss(net).backward()
    for n, p in alphas.items():
        assert p.grad is buffers[n] or p.grad.data_ptr() == buffers[n].data_ptr(), n
        assert rel(p.grad - 1, want[n]) < 1e-2 + 2.0 ** -23 * p.numel() ** 0.5 / want[n].norm().item(), n
    loss = _loss(net)
    with torch.no_grad():
        next(iter(alphas.values())).add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
