"""CPU: differential attention -- the formulas against the definition, against autograd and differences in 64
bits, and the refusals."""
import pytest
import torch

from imfvideo_b200.ops import dual as D
from imfvideo_b200.ops import reference as ref

F64 = torch.float64


def _inputs(B=2, L=7, H=2, d=8, seed=0, dtype=F64):
    g = torch.Generator().manual_seed(seed)
    q, k, v, dq, dk, dv = (torch.randn(B, L, 2 * H, d, generator=g, dtype=dtype) for _ in range(6))
    return q, k, v, torch.tensor([0.4, -1.3], dtype=dtype)[:H], dq, dk, dv


def _definition(q, k, v, lam, scale):
    """One row at a time."""
    B, L, H2, d = q.shape
    o = torch.zeros_like(v)
    for b in range(B):
        for j in range(H2 // 2):
            V = torch.cat([v[b, :, 2 * j], v[b, :, 2 * j + 1]], -1)
            for i in range(L):
                a = [torch.softmax(k[b, :, 2 * j + m] @ q[b, i, 2 * j + m] * scale, 0) for m in (0, 1)]
                r = (a[0] - lam[j] * a[1]) @ V
                o[b, i, 2 * j], o[b, i, 2 * j + 1] = r[:d], r[d:]
    return o


@pytest.mark.parametrize("L", [1, 2, 7])
@pytest.mark.parametrize("scale", [None, 0.3])
def test_against_the_definition(L, scale):
    q, k, v, lam, *_ = _inputs(L=L)
    got = D.diff_attention(D.Dual(q), D.Dual(k), D.Dual(v), lam, scale)
    assert got.t is None
    assert torch.allclose(got.p, _definition(q, k, v, lam, 8 ** -0.5 if scale is None else scale), atol=1e-13)


def test_gradients_against_differences():
    q, k, v, lam, *_ = _inputs(L=5)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    f = lambda a, b, c, w: D.diff_attention(D.Dual(a), D.Dual(b), D.Dual(c), w).p
    assert torch.autograd.gradcheck(f, leaves)


def test_tangent_against_forward_mode_and_differences():
    q, k, v, lam, dq, dk, dv = _inputs()
    f = lambda a, b, c: ref.diff_attention(a, b, c, lam)
    o, do = torch.func.jvp(f, (q, k, v), (dq, dk, dv))
    got = D.diff_attention(D.Dual(q, dq), D.Dual(k, dk), D.Dual(v, dv), lam)
    assert torch.allclose(got.p, o, atol=1e-13) and torch.allclose(got.t, do, atol=1e-12)
    h = 1e-6
    diff = (f(q + h * dq, k + h * dk, v + h * dv) - f(q - h * dq, k - h * dk, v - h * dv)) / (2 * h)
    assert torch.allclose(got.t, diff, atol=1e-7)


def test_tangent_is_detached_and_missing_ones_are_zero():
    q, k, v, lam, dq, _, _ = _inputs()
    q.requires_grad_()
    a = D.diff_attention(D.Dual(q, dq), D.Dual(k), D.Dual(v), lam)
    b = D.diff_attention(D.Dual(q, dq), D.Dual(k, torch.zeros_like(k)), D.Dual(v, torch.zeros_like(v)), lam)
    assert a.p.requires_grad and not a.t.requires_grad and torch.equal(a.t, b.t)


def test_one_weight_for_all_pairs():
    q, k, v, *_ = _inputs()
    lam = torch.tensor(0.6, dtype=F64, requires_grad=True)
    o = D.diff_attention(D.Dual(q), D.Dual(k), D.Dual(v), lam).p
    assert torch.equal(o, D.diff_attention(D.Dual(q), D.Dual(k), D.Dual(v), lam.detach().expand(2)).p)
    g, = torch.autograd.grad(o.sum(), lam)
    assert g.shape == ()


def test_bf16_result_is_rounded_once():
    q, k, v, lam, *_ = _inputs(dtype=torch.float32)
    q, k, v = (t.bfloat16() for t in (q, k, v))
    got = D.diff_attention(D.Dual(q), D.Dual(k), D.Dual(v), lam).p
    want = _definition(q.double(), k.double(), v.double(), lam.double(), 8 ** -0.5)
    # half a step of bf16, and 32-bit sums of some ten terms
    assert got.dtype == torch.bfloat16 and ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()


def test_refusals():
    q, k, v, lam, *_ = _inputs()
    dual = lambda *t, **kw: D.diff_attention(*(D.Dual(x) for x in t[:3]), t[3], **kw)
    for f in (lambda: dual(q[:, :, :3], k[:, :, :3], v[:, :, :3], lam), lambda: dual(q, k[:, :3], v, lam),
              lambda: dual(q, k, v[..., :4], lam), lambda: dual(q, k, v, torch.ones(3, dtype=F64)),
              lambda: dual(q[0], k[0], v[0], lam), lambda: dual(q, k, v, lam, impl="sdpa")):
        with pytest.raises(ValueError):
            f()
