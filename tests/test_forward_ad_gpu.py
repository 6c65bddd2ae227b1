"""GPU: forward-mode AD (``torch.autograd.forward_ad``) through differential attention and the norms around a branch.
The kernels know no dual tensors of torch: a call that gets one has to take the formulas, with or without gradients
asked for, and any other call the kernels."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from test_diffattn_gpu import _forward64, _inputs, _tangent64, _wide, _within

pytestmark = pytest.mark.gpu
F32 = torch.float32


@pytest.fixture(autouse=True)
def _level():
    """A failure must not leave the level open for other tests."""
    yield
    assert fwAD.unpack_dual(torch.zeros(1)).tangent is None


@pytest.mark.parametrize("grad,asked", [(False, False), (True, False), (True, True)])
def test_diff_attention(grad, asked):
    from imfvideo_b200.ops import dual as D

    q, k, v, lam, tan = _inputs(1, 90, 2, seed=4, tangent=True)
    lam.requires_grad_(asked)
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        args = [D.Dual(fwAD.make_dual(a, b)) for a, b in zip((q, k, v), tan)]
        o, do = fwAD.unpack_dual(D.diff_attention(*args, lam).p)
        assert do is not None
        o, do = o.detach().clone(), do.detach().clone()
    lam = lam.detach()
    _within(_wide(o), *_forward64(q, k, v, lam)[2:4], "o")
    _within(_wide(do), *_tangent64(q, k, v, lam, tan), "do")


def test_diff_attention_of_a_dual_weight():
    from imfvideo_b200.ops import dual as D

    q, k, v, lam, _ = _inputs(1, 70, 2, seed=5)
    step = torch.tensor([1.0, -2.0], device="cuda")
    with torch.no_grad(), fwAD.dual_level():
        o = D.diff_attention(D.Dual(q), D.Dual(k), D.Dual(v), fwAD.make_dual(lam, step)).p
        do = fwAD.unpack_dual(o).tangent
        assert do is not None
        do = do.clone()
    O2 = _forward64(q, k, v, lam)[1][:, :, 1]
    want = -step.double()[None, :, None, None] * O2
    # one rounding to bf16, and 32-bit sums
    _within(_wide(do), want, 2.0 ** -8 * want.abs() + 1e-5, "do")


@pytest.mark.parametrize("grad,asked", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("which", ["res", "y", "gate"])
def test_norm_add_norm(which, grad, asked):
    from imfvideo_b200.ops import dual as D

    g = torch.Generator(device="cuda").manual_seed(6)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    t = dict(res=rnd(5, 64), y=rnd(5, 64), post=rnd(64), gate=rnd(64), scale=rnd(64), pre=rnd(64))
    step = rnd(*t[which].shape)
    t["post"].requires_grad_(asked)

    def f(a):
        x, n = D.norm_add_norm(D.Dual(a["res"]), D.Dual(a["y"]), a["post"], a["gate"], 1e-5, a["scale"], a["pre"])
        return x.p, n.p
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        got = [fwAD.unpack_dual(z).tangent for z in f({**t, which: fwAD.make_dual(t[which], step)})]
        assert all(z is not None for z in got)
        got = [z.detach().clone() for z in got]
    cpu = {n: z.detach().cpu().double() for n, z in t.items()}
    h = 1e-6 * step.cpu().double()
    up, down = f({**cpu, which: cpu[which] + h}), f({**cpu, which: cpu[which] - h})
    for a, b, c in zip(got, up, down):
        want = (b - c) / 2e-6
        # 32-bit sums of 64 terms, and differences of 64-bit values 2e-6 apart
        assert (a.cpu().double() - want).abs().max() < 1e-5 * (1 + want.abs().max())


def test_other_calls_take_the_kernels():
    from imfvideo_b200.ops import dual as D, kernels as K

    q, k, v, lam, _ = _inputs(1, 70, 2, seed=7)
    y, w = torch.ones(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with torch.no_grad(), fwAD.dual_level():
        fwAD.make_dual(torch.ones(2), torch.ones(2))
        for f in (lambda: D.diff_attention(D.Dual(q), D.Dual(k), D.Dual(v), lam),
                  lambda: D.norm_add_norm(None, D.Dual(y), w, w, 1e-5)):
            before = K.LAUNCHES.count
            f()
            assert K.LAUNCHES.count > before
