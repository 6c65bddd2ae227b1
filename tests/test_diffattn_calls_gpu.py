"""GPU: tangents of another type than their primal's; outputs over inputs."""
import pytest
import torch

from test_diffattn_gpu import _inputs, _status  # noqa: F401

pytestmark = pytest.mark.gpu


def test_tangents_of_another_type_of_diff_attention():
    from imfvideo_b200.ops import dual as D

    q, k, v, lam, tan = _inputs(1, 90, 2, seed=8, tangent=True)
    want = D.diff_attention(*(D.Dual(*z) for z in zip((q, k, v), tan)), lam)
    for dt in (torch.float32, torch.float64):
        got = D.diff_attention(*(D.Dual(a, b.to(dt)) for a, b in zip((q, k, v), tan)), lam)
        assert torch.equal(got.p, want.p) and torch.equal(got.t, want.t)


@pytest.mark.parametrize("dres,dy", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
def test_tangents_of_another_type_of_norm_add_norm(dres, dy):
    """As on the CPU, where the formulas take them as they are."""
    from imfvideo_b200.ops import dual as D

    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    res, y = D.Dual(rnd(5, 64), rnd(5, 64).to(dres)), D.Dual(rnd(5, 64).bfloat16(), rnd(5, 64).to(dy))
    vec = [rnd(64) for _ in range(4)]
    call = lambda r, y, w: D.norm_add_norm(r, y, w[0], w[1], 1e-5, w[2], w[3])
    x, n = call(res, y, vec)
    xc, nc = call(res.map(torch.Tensor.cpu), y.map(torch.Tensor.cpu), [w.cpu() for w in vec])
    assert x.t.dtype == torch.float32 and n.t.dtype == torch.bfloat16
    for a, b in ((x.p, xc.p), (x.t, xc.t)):
        assert (a.cpu() - b).abs().max() < 1e-5 * (1 + b.abs().max())       # 32-bit sums of 64 terms
    for a, b in ((n.p, nc.p), (n.t, nc.t)):                                 # one step of bf16 where those fall apart
        assert (a.cpu().float() - b.float()).abs().max() <= 2.0 ** -7 * b.float().abs().max()


def test_dv_over_the_weights():
    """The weights are read while dv is written: refused.  The forward pass's results are read before: the same gradients."""
    from imfvideo_b200.ops import diffattn as DA

    q, k, v, lam, go = _inputs(1, 40, 2)
    o, _, saved = DA.diff_attn_fwd(q, k, v, lam)
    want = DA.diff_attn_bwd(q, k, v, lam, o, saved, go)
    out = torch.empty_like(q)
    for inside in (out.view(-1)[640:642], out.view(torch.float32).view(-1)[100:102]):
        inside.copy_(lam)
        with pytest.raises(ValueError, match="over an input"):
            DA.diff_attn_bwd(q, k, v, inside, o, saved, go, gv_out=out)
    wide = torch.empty(1, 40, 4, 72, device="cuda", dtype=torch.bfloat16)
    wide[0, 3, 1, 64:68] = lam.view(torch.bfloat16)          # between two rows of the output
    got = DA.diff_attn_bwd(q, k, v, wide[0, 3, 1, 64:68].view(torch.float32), o, saved, go, gv_out=wide[..., :64])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(DA.diff_attn_bwd(q, k, v, lam, o, saved, go, gv_out=o), want):
        assert torch.equal(a, b)                             # (one K/V tile)
