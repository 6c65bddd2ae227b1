"""CPU: norms around a branch -- the formulas against the definition, autograd and differences in 64 bits, and
the refusals."""
import itertools

import pytest
import torch

from imfvideo_b200.ops import dual as D

F64 = torch.float64
EPS = 1e-5
FORMS = list(itertools.product([True, False], [True, False], [True, False]))


def _inputs(has_res, has_scale, has_pre, R=(2, 3), width=8, dtype=F64):
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=dtype)
    v = dict(res=rnd(*R, width) if has_res else None, y=rnd(*R, width), post=1 + 0.3 * rnd(width), gate=0.5 * rnd(width),
             res_scale=1 + 0.2 * rnd(width) if has_res and has_scale else None, pre=1 + 0.3 * rnd(width) if has_pre else None)
    return v, rnd(*R, width) if has_res else None, rnd(*R, width)


def _call(v, dres=None, dy=None):
    res = None if v["res"] is None else D.Dual(v["res"], dres)
    return D.norm_add_norm(res, D.Dual(v["y"], dy), v["post"], v["gate"], EPS, res_scale=v["res_scale"], pre=v["pre"])


def _definition(v):
    rms = lambda t: ((t * t).mean(-1, keepdim=True) + EPS) ** 0.5
    x = v["gate"] * v["post"] * v["y"] / rms(v["y"])
    if v["res"] is not None:
        x = x + v["res"] * (1 if v["res_scale"] is None else v["res_scale"])
    return x, None if v["pre"] is None else v["pre"] * x / rms(x)


@pytest.mark.parametrize("form", FORMS)
def test_against_the_definition_and_differences(form):
    v, _, _ = _inputs(*form)
    x, n = _call(v)
    wx, wn = _definition(v)
    assert torch.allclose(x.p, wx, atol=1e-13) and x.t is None
    assert (n is None) == (wn is None) and (n is None or torch.allclose(n.p, wn, atol=1e-13))
    names = [k for k in v if v[k] is not None]

    def f(*ts):
        a, b = _call({**v, **dict(zip(names, ts))})
        return a.p if b is None else (a.p, b.p)
    assert torch.autograd.gradcheck(f, [v[k].requires_grad_() for k in names])


@pytest.mark.parametrize("form", FORMS)
def test_tangent_against_forward_mode(form):
    v, dres, dy = _inputs(*form)
    x, n = _call(v, dres, dy)
    moving = [("y", dy)] + ([("res", dres)] if dres is not None else [])
    f = lambda *ts: tuple(t for t in _definition({**v, **dict(zip([m for m, _ in moving], ts))}) if t is not None)
    val, tan = torch.func.jvp(f, tuple(v[m] for m, _ in moving), tuple(t for _, t in moving))
    assert torch.allclose(x.t, tan[0], atol=1e-12) and (n is None or torch.allclose(n.t, tan[1], atol=1e-12))


def test_residual_that_stands_still_and_branch_that_does():
    v, dres, dy = _inputs(True, True, True)
    zero = torch.zeros_like(dy)
    for a, b in ((_call(v, None, dy), _call(v, zero, dy)), (_call(v, dres, None), _call(v, dres, zero))):
        assert torch.equal(a[0].t, b[0].t) and torch.equal(a[1].t, b[1].t)


def test_types():
    v, _, _ = _inputs(True, False, True, dtype=torch.float32)
    v["y"] = v["y"].bfloat16()
    x, n = _call(v)
    assert x.p.dtype == torch.float32 and n.p.dtype == torch.bfloat16
    v["res"] = None
    assert _call(v)[0].p.dtype == torch.float32


def test_refusals():
    v, _, _ = _inputs(True, True, True)
    for bad in (dict(res=None), dict(post=v["post"][:4]), dict(gate=v["gate"][None]), dict(pre=v["pre"][:1]),
                dict(res=v["res"][:1]), dict(res_scale=torch.ones((), dtype=F64))):
        with pytest.raises(ValueError):
            _call({**v, **bad})


def test_row_numbers_have_32_bits():
    from imfvideo_b200.ops import postnorm as PN

    w = torch.empty(8, device="meta")
    with pytest.raises(ValueError, match="2\\^30"):
        PN.norm_add_norm_fwd(None, torch.empty(1 << 30, 8, device="meta"), w, w, 1e-5)
