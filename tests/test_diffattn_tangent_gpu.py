"""GPU: the forward-mode kernel of differential attention on the paths that ``test_diffattn_gpu.py`` does not take.
Bounds are that file's."""
import pytest
import torch

from test_diffattn_gpu import (SLACK, U, _check_grads, _forward64, _inputs, _own, _pairs, _status,  # noqa: F401
                               _tangent64, _wide, _within)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,L,H", [(1, 1, 1), (2, 33, 3), (1, 64, 2), (4, 64, 80), (1, 532, 2)])
def test_walks_of_one_tile_are_the_same_every_time(B, L, H):
    """A CTA that begins with one K/V tile (all of them up to 64 rows, five of 45 at 1 x 532, 2 pairs): the group without
    a step goes on to the next walk's queries."""
    q, k, v, lam, tan = _inputs(B, L, H, seed=L, tangent=True)
    first = _own(q, k, v, lam, tan)
    _within(_wide(first[0]), *_forward64(q, k, v, lam)[2:4], "o")
    _within(_wide(first[1]), *_tangent64(q, k, v, lam, tan), "do")
    for _ in range(300):
        o, do, saved = _own(q, k, v, lam, tan)
        assert torch.equal(o, first[0]) and torch.equal(do, first[1])
        assert all(torch.equal(a, b) for a, b in zip(saved, first[2]))


def _joined(saved, o):
    """(o, O_2) with the bytes that their rounding dropped: 1/256 of bf16's last place each."""
    o2, low, _ = saved
    B, L, H2, D = o.shape
    low = low.view(B, L, H2, D // 8, 2, 8)
    join = lambda t, c: ((t.view(torch.int16).int() << 16) + (c.reshape(t.shape).int() << 8)).view(torch.float32)
    return join(o, low[..., 0, :]), join(o2, low[..., 1, :])


def _scores(q, k, scale):
    return _pairs(q) @ _pairs(k).transpose(-1, -2) * scale


def _score_error(q, k, scale):
    """What the 32-bit sums of a score are off by at most: 2^-20 of the products' sum."""
    return (_scores(q.abs(), k.abs(), scale).amax() * 2.0 ** -20).item()


def _tangent_and_bound(q, k, v, lam, tan, scale):
    """do, and its bound from the roundings of A and A dS (U of each), errors s of the scores (A is off by 2 s of its value,
    its own and its row sum's) and 2^-20 of the products' sum of dS."""
    A, O, *_ = _forward64(q, k, v, lam, scale)
    dq, dk, dv = tan
    dS = _scores(dq, k, scale) + _scores(q, dk, scale)
    edS = (_scores(dq.abs(), k.abs(), scale) + _scores(q.abs(), dk.abs(), scale)) * 2.0 ** -20
    V, dV = _wide(v)[:, :, None], _wide(dv)[:, :, None]
    T = A * dS
    mu = T.sum(-1, keepdim=True)
    dO = T @ V + A @ dV - mu * O
    s = 2 * _score_error(q, k, scale)
    AV = A @ V.abs()
    b = (SLACK * U + s) * (T.abs() @ V.abs() + A @ dV.abs() + mu.abs() * AV) + (A * edS) @ V.abs() + \
        ((s + 2.0 ** -18) * T.abs().sum(-1, keepdim=True) + (A * edS).sum(-1, keepdim=True)) * O.abs()
    w = lam.double()[None, :, None, None]
    want = dO[:, :, 0] - w * dO[:, :, 1]
    return want, b[:, :, 0] + w.abs() * b[:, :, 1] + U * want.abs() + 1e-6


def _check(q, k, v, lam, tan, scale):
    """o, do and all that is kept for the backward pass."""
    o, do, saved = _own(q, k, v, lam, tan, scale=scale)
    A, O, want, e, e2 = _forward64(q, k, v, lam, scale)
    s = _score_error(q, k, scale)
    more = 1 + 2 * s / U
    _within(_wide(o), want, e * more, "o")
    _within(_wide(saved[0]), O[:, :, 1], e2 * more, "o2")
    # 16 bits: half of 1/256 of bf16's last place, a whole one at the largest
    jo, j2 = _joined(saved, o)
    _within(_wide(jo), want, (e - U * want.abs()) * more + 2.0 ** -15 * want.abs(), "o in 16 bits")
    _within(_wide(j2), O[:, :, 1], (e2 - U * O[:, :, 1].abs()) * more + 2.0 ** -15 * O[:, :, 1].abs(), "o2 in 16 bits")
    lse = torch.logsumexp(_scores(q, k, scale), -1)
    B, L, H2, _ = q.shape
    assert (saved[2].view(B, H2 // 2, 2, L) - lse).abs().max() < 1e-4 + s
    _within(_wide(do), *_tangent_and_bound(q, k, v, lam, tan, scale), "do")
    return o, do, saved


# 1,100 and 1,500 rows: fewer items than SMs, in shares that a second launch merges; 640 x 8: whole items
PLACES = [(1, 1, 1), (1, 65, 1), (2, 129, 2), (1, 532, 2), (1, 1100, 2), (1, 1500, 3), (2, 640, 8), (1, 2061, 3)]


@pytest.mark.parametrize("scale", [0.125, 0.1, 0.3, 0.25])
@pytest.mark.parametrize("B,L,H", PLACES)
def test_scales_and_what_is_kept(B, L, H, scale):
    """Scales that are no power of two multiply every T, the others the queries."""
    q, k, v, lam, tan = _inputs(B, L, H, seed=L, tangent=True)
    _check(q, k, v, lam, tan, scale)


@pytest.mark.parametrize("scale", [0.125, 0.11])
@pytest.mark.parametrize("B,L,H", [(1, 700, 2), (1, 1100, 2), (2, 640, 8)])
def test_rows_that_outgrow_their_reference(B, L, H, scale):
    """O, dO and the sums move to a new reference, many times a row."""
    q, k, v, lam, tan = _inputs(B, L, H, seed=3, std=4.0, tangent=True)
    k = k * torch.linspace(0.2, 2.0, L, device="cuda")[None, :, None, None].bfloat16()
    tops = torch.stack([t.amax(-1) for t in _scores(q, k, scale).split(64, -1)], -1) * 1.4426950408889634
    ref, moves = tops[..., 0], 0
    for t in tops.unbind(-1)[1:]:
        ref, moves = torch.where(t > ref + 8, t, ref), moves + (t > ref + 8).sum().item()
    assert moves > 2 * ref.numel()
    _check(q, k, v, lam, tan, scale)


def test_backward_of_what_the_tangent_kernel_kept():
    """A training step's pair of calls: forward with tangent that keeps its state, then the gradients."""
    from imfvideo_b200.ops import diffattn as DA

    for B, L, H in ((1, 64, 2), (1, 1100, 2), (2, 640, 8)):
        q, k, v, lam, tan = _inputs(B, L, H, seed=L + 1, tangent=True)
        go = tan[2]
        o, _, saved = _own(q, k, v, lam, tan)
        _check_grads(q, k, v, lam, go, DA.diff_attn_bwd(q, k, v, lam, o, saved, go))
