"""GPU: out-of-bounds writes of differential attention and of the norms around a branch.  Every tensor that their calls
allocate, results and workspaces, lies between two guard regions filled with a sentinel, which must be intact afterwards;
sizes are ragged on purpose."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
SENTINEL = {BF16: -7.75, F32: -12345.5, torch.int8: 77, torch.uint8: 173}


class Guards:
    """Stands in for the calls' allocations."""

    def __init__(self, monkeypatch, *modules):
        self.made = []
        for m in modules:
            monkeypatch.setattr(m, "_new", self.new)
        self.empty_like = torch.empty_like
        monkeypatch.setattr(torch, "empty_like", self.like)

    def new(self, shape, dtype, dev):
        n, pad = math.prod(shape) if not isinstance(shape, int) else shape, 16384
        buf = torch.full((n + 2 * pad,), SENTINEL[dtype], dtype=dtype, device=dev)
        self.made.append((buf, pad, n))
        return buf[pad:pad + n].view(shape)

    def like(self, t, dtype=None):
        return self.new(t.shape, dtype or t.dtype, t.device) if t.is_cuda else self.empty_like(t, dtype=dtype or t.dtype)

    def check(self):
        torch.cuda.synchronize()
        for buf, pad, n in self.made:
            s = SENTINEL[buf.dtype]
            assert (buf[:pad] == s).all() and (buf[pad + n:] == s).all(), (buf.dtype, n)
        made, self.made = len(self.made), []
        return made


# one item; whole items; shares of few items (a second launch merges them); split K/V tiles of the backward pass; short rows
# of many heads
@pytest.mark.parametrize("scale", [0.125, 0.1])
@pytest.mark.parametrize("B,L,H", [(1, 1, 1), (1, 65, 1), (3, 300, 2), (1, 1100, 2), (1, 1500, 3), (1, 2061, 3), (1, 4116, 1),
                                   (2, 33, 40), (4, 63, 80)])
def test_diff_attention(B, L, H, scale, monkeypatch):
    from imfvideo_b200.ops import diffattn as DA
    from imfvideo_b200.ops import kernels as K

    g = torch.Generator(device="cuda").manual_seed(L)
    q, k, v, dq, dk, dv = (torch.randn(B, L, 2 * H, 64, device="cuda", generator=g).bfloat16() for _ in range(6))
    lam = torch.rand(H, device="cuda", generator=g)

    def run():
        for order in (False, True):
            monkeypatch.setattr(K, "DETERMINISTIC", order)
            o, _, saved = DA.diff_attn_fwd(q, k, v, lam, scale=scale)
            yield (o, *saved, *DA.diff_attn_bwd(q, k, v, lam, o, saved, dq, scale)[1:])
            yield DA.diff_attn_fwd(q, k, v, lam, need_bwd=False, scale=scale)[:1]
            o, do, saved = DA.diff_attn_fwd(q, k, v, lam, dq, dk, dv, scale=scale)
            yield (o, do, *saved, *DA.diff_attn_bwd(q, k, v, lam, o, saved, dq, scale)[1:])
            yield DA.diff_attn_fwd(q, k, v, lam, dq, dk, dv, need_bwd=False, scale=scale)[:2]
    want = list(run())
    guards = Guards(monkeypatch, DA)
    for a, b in zip(run(), want):
        assert guards.check() >= len(b)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    K.check_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,D", [(1, 8), (33, 264), (257, 520), (129, 1000), (300, 1280), (9, 1800), (5, 2056), (3, 8192),
                                    (2500, 768)])
def test_norms_around_a_branch(rows, D, dtype, monkeypatch):
    from imfvideo_b200.ops import kernels as K, postnorm as PN

    g = torch.Generator(device="cuda").manual_seed(D)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    res, dres, gx = (rnd(rows, D) for _ in range(3))
    y, dy, gn = (rnd(rows, D).to(dtype) for _ in range(3))
    post, gate, keep, pre = (rnd(D) for _ in range(4))

    def run():
        yield PN.norm_add_norm_fwd(res, y, post, gate, 1e-5, keep, pre)
        yield PN.norm_add_norm_fwd(res, y, post, gate, 1e-5, keep, pre, dres, dy)
        yield PN.norm_add_norm_fwd(None, y, post, gate, 1e-5, None, None, None, dy)
        yield PN.norm_add_norm_bwd(res, y, post, gate, 1e-5, keep, pre, gx, gn)
        yield PN.norm_add_norm_bwd(res, y, post, gate, 1e-5, None, None, gx, None)
    want = list(run())
    guards = Guards(monkeypatch, PN)
    for a, b in zip(run(), want):
        assert guards.check() > 1
        for s, t in zip(a, b):
            assert s is None and t is None or torch.equal(s, t)
    K.check_status()
