"""GPU: differential attention against the formulas in 64 bits.

Tolerances hold element by element and are sums of the roundings that the kernels make.  A rounding to bf16
is off by at most U = 2^-8 of the value.  Forward: the probabilities are rounded (U of A |V|), then the result;
scores, exponentials and sums are in 32 bits, for which every bound gets 1/8 more (scores of a few tens are
off by 1e-5, exponentials by as much of their value).  The tangent rounds A and A dS.  Backward: A and dS are
rounded, delta comes from o and O_2 as they were kept."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = torch.finfo(torch.bfloat16).eps / 2
SLACK = 1.125
BF16, F64 = torch.bfloat16, torch.float64


@pytest.fixture(autouse=True)
def _status():
    yield
    from imfvideo_b200.ops import kernels as K

    torch.cuda.synchronize()
    K.check_status()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(B, L, H, seed=0, std=1.0, offset=0.5, tangent=False):
    g = _gen(seed)
    rnd = lambda: torch.randn(B, L, 2 * H, 64, device="cuda", generator=g)
    off = offset * torch.randn(2 * H, 64, device="cuda", generator=g)
    q, k, v = (std * rnd()).bfloat16(), (std * rnd()).bfloat16(), (rnd() + off).bfloat16()
    lam = torch.rand(H, device="cuda", generator=g) * 1.2 - 0.2
    go = rnd().bfloat16()
    if not tangent:
        return q, k, v, lam, go
    return q, k, v, lam, tuple((0.5 * rnd()).bfloat16() for _ in range(3))


def _pairs(t):
    """(B, H, 2, L, 64) in 64 bits"""
    B, L, H2, D = t.shape
    return t.double().view(B, L, H2 // 2, 2, D).permute(0, 2, 3, 1, 4)


def _wide(t):
    B, L, H2, D = t.shape
    return t.double().reshape(B, L, H2 // 2, 2 * D).transpose(1, 2)


def _unwide(t, like):
    return t.transpose(1, 2).reshape(like.shape)


def _unpair(t, like):
    return t.permute(0, 3, 1, 2, 4).reshape(like.shape)


def _forward64(q, k, v, lam, scale=0.125):
    """A (B, H, 2, L, L), O_m, o and the bounds of o and of O_2."""
    A = torch.softmax(_pairs(q) @ _pairs(k).transpose(-1, -2) * scale, -1)
    V = _wide(v)
    O = A @ V[:, :, None]
    w = lam.double()[None, :, None, None]
    o = O[:, :, 0] - w * O[:, :, 1]
    AV = A @ V.abs()[:, :, None]
    e = SLACK * U * (AV[:, :, 0] + w.abs() * AV[:, :, 1]) + U * o.abs() + 1e-6
    e2 = SLACK * U * AV[:, :, 1] + U * O[:, :, 1].abs() + 1e-6
    return A, O, o, e, e2


def _within(got, want, bound, what):
    over = (got.double() - want).abs() - bound
    assert not torch.isnan(got).any(), what
    assert over.max().item() <= 0, (what, over.max().item(), ((got.double() - want).abs() / bound).max().item())


def _own(q, k, v, lam, tangents=(None,) * 3, **kw):
    from imfvideo_b200.ops import diffattn as DA

    return DA.diff_attn_fwd(q, k, v, lam, *tangents, **kw)


SHAPES = [(1, 1, 1), (1, 2, 2), (2, 63, 1), (1, 64, 3), (1, 65, 1), (2, 127, 2), (1, 128, 1), (1, 129, 2), (3, 300, 2),
          (1, 532, 2), (1, 1025, 1), (2, 640, 8), (1, 2061, 3)]


@pytest.mark.parametrize("B,L,H", SHAPES)
def test_forward(B, L, H):
    q, k, v, lam, _ = _inputs(B, L, H, seed=L)
    o, do, saved = _own(q, k, v, lam)
    A, O, want, e, e2 = _forward64(q, k, v, lam)
    assert do is None
    _within(_wide(o), want, e, "o")
    o2, low, lse = saved
    _within(_wide(o2), O[:, :, 1], e2, "o2")
    s = torch.logsumexp(_pairs(q) @ _pairs(k).transpose(-1, -2) * 0.125, -1)
    assert (lse.view(B, H, 2, L) - s).abs().max() < 1e-4
    o_only = _own(q, k, v, lam, need_bwd=False)
    assert torch.equal(o_only[0], o) and o_only[1:] == (None, ())


def _tangent64(q, k, v, lam, tan):
    """do and its bound."""
    A, O, *_ = _forward64(q, k, v, lam)
    dq, dk, dv = tan
    dS = (_pairs(dq) @ _pairs(k).transpose(-1, -2) + _pairs(q) @ _pairs(dk).transpose(-1, -2)) * 0.125
    V, dV = _wide(v)[:, :, None], _wide(dv)[:, :, None]
    T = A * dS
    mu = T.sum(-1, keepdim=True)
    dO = T @ V + A @ dV - mu * O
    b = T.abs() @ V.abs() + A @ dV.abs() + mu.abs() * (A @ V.abs())
    w = lam.double()[None, :, None, None]
    dwant = dO[:, :, 0] - w * dO[:, :, 1]
    return dwant, SLACK * U * (b[:, :, 0] + w.abs() * b[:, :, 1]) + U * dwant.abs() + 1e-6


@pytest.mark.parametrize("B,L,H", SHAPES)
def test_tangent(B, L, H):
    q, k, v, lam, tan = _inputs(B, L, H, seed=L, tangent=True)
    o, do, saved = _own(q, k, v, lam, tan)
    A, O, want, e, e2 = _forward64(q, k, v, lam)
    _within(_wide(o), want, e, "o")
    _within(_wide(saved[0]), O[:, :, 1], e2, "o2")
    _within(_wide(do), *_tangent64(q, k, v, lam, tan), "do")


def _backward64(q, k, v, lam, go, scale=0.125):
    """Gradients and their bounds."""
    A, O, o, e, e2 = _forward64(q, k, v, lam, scale)
    # o and O_2 are kept to half of 1/256 of bf16's last place (a whole one at the largest), 2^-15 of the value
    e, e2 = (x - U * y.abs() + 2.0 ** -15 * y.abs() for x, y in ((e, o), (e2, O[:, :, 1])))
    V, G, w = _wide(v), _wide(go), lam.double()[None, :, None, None]
    wm = torch.stack([torch.ones_like(w), -w], 2)                                # (1, H, 2, 1, 1)
    dP = (G @ V.transpose(-1, -2))[:, :, None]
    delta = (G[:, :, None] * O).sum(-1, keepdim=True)
    ed2 = (G.abs() * e2).sum(-1, keepdim=True)
    ed = torch.stack([(G.abs() * e).sum(-1, keepdim=True) + w.abs() * ed2, ed2], 2)
    P = wm * A
    dS = P * (dP - delta)
    edS = SLACK * (U * dS.abs() + P.abs() * (ed + 2e-5 * (dP.abs() + delta.abs())))
    Q, K = _pairs(q), _pairs(k)
    want = {"dq": (dS @ K * scale, edS @ K.abs() * scale), "dk": (dS.mT @ Q * scale, edS.mT @ Q.abs() * scale),
            "dv": ((P.mT @ G[:, :, None]).sum(2), SLACK * U * (P.abs().mT @ G.abs()[:, :, None]).sum(2)),
            "dlam": (-delta[:, :, 1].sum((0, 2, 3)), SLACK * ed2.sum((0, 2, 3)))}
    return {n: (x, b + U * x.abs() + 1e-6) for n, (x, b) in want.items()}


def _check_grads(q, k, v, lam, go, got, scale=0.125):
    want = _backward64(q, k, v, lam, go, scale)
    _within(_pairs(got[0]), *want["dq"], "dq")
    _within(_pairs(got[1]), *want["dk"], "dk")
    _within(_wide(got[2]), *want["dv"], "dv")
    _within(got[3], *want["dlam"], "dlam")


@pytest.mark.parametrize("B,L,H", SHAPES)
def test_backward(B, L, H):
    from imfvideo_b200.ops import diffattn as DA

    q, k, v, lam, go = _inputs(B, L, H, seed=L)
    o, _, saved = _own(q, k, v, lam)
    _check_grads(q, k, v, lam, go, DA.diff_attn_bwd(q, k, v, lam, o, saved, go))


@pytest.mark.parametrize("std,scale", [(4.0, 0.125), (0.05, 0.125), (1.0, 1.0), (1.0, 0.01)])
def test_peaked_and_flat_maps(std, scale):
    """Rows that outgrow their reference maximum many times (scores of some hundreds), and maps so flat that the two
    are nearly equal."""
    from imfvideo_b200.ops import diffattn as DA

    q, k, v, lam, go = _inputs(1, 700, 2, seed=3, std=std)
    k = k * torch.linspace(0.2, 2.0, 700, device="cuda")[None, :, None, None].bfloat16()
    o, _, saved = _own(q, k, v, lam, scale=scale)
    A, O, want, e, e2 = _forward64(q, k, v, lam, scale)
    # scores of a few hundred are off by their 32-bit rounding, 2^-20 of the products' sum at most
    s = (_pairs(q).abs() @ _pairs(k).abs().transpose(-1, -2) * scale).amax() * 2.0 ** -20
    more = 1 + (s / U).item() * 2
    _within(_wide(o), want, e * more, "o")
    got = DA.diff_attn_bwd(q, k, v, lam, o, saved, go, scale)
    for n, t in (("dq", _pairs(got[0])), ("dk", _pairs(got[1])), ("dv", _wide(got[2])), ("dlam", got[3])):
        x, b = _backward64(q, k, v, lam, go, scale)[n]
        _within(t, x, b * more, n)


def test_weights_of_every_sign_and_type():
    from imfvideo_b200.ops import diffattn as DA

    q, k, v, _, go = _inputs(1, 200, 4, seed=5)
    for lam in (torch.tensor([0.0, -1.5, 1.0, 3.0], device="cuda"),
                torch.tensor([0.0, -1.5, 1.0, 3.0], device="cuda").bfloat16(),
                torch.tensor([0.7], device="cuda").expand(4),
                torch.tensor([0.1, 9.0, 0.2, 9.0, 0.3, 9.0, 0.4, 9.0], device="cuda")[::2]):
        o, _, saved = _own(q, k, v, lam)
        A, O, want, e, e2 = _forward64(q, k, v, lam)
        _within(_wide(o), want, e, "o")
        _within(_wide(saved[0]), O[:, :, 1], e2, "o2")
        got = DA.diff_attn_bwd(q, k, v, lam, o, saved, go)
        assert got[3].dtype == lam.dtype
        _check_grads(q, k, v, lam, go, got)


def test_strides_and_broadcasts():
    """Bands of wider rows as the block hands them over, transposed, broadcast and unaligned tensors."""
    from imfvideo_b200.ops import diffattn as DA

    B, L, H = 2, 150, 2
    q, k, v, lam, go = _inputs(B, L, H, seed=7)
    want_o, _, want_saved = _own(q, k, v, lam)
    want = DA.diff_attn_bwd(q, k, v, lam, want_o, want_saved, go)
    wide = torch.randn(B, L, 2 * H, 48 + 64, device="cuda").bfloat16()
    wide[..., 48:] = v
    band = wide[..., 48:]
    odd = torch.empty(B * L * 2 * H * 64 + 1, device="cuda", dtype=BF16)[1:].view(q.shape).copy_(q)
    swapped = k.transpose(1, 2).contiguous().transpose(1, 2)
    o, _, saved = _own(odd, swapped, band, lam)
    assert torch.equal(o, want_o) and all(torch.equal(a, b) for a, b in zip(saved, want_saved))
    out = torch.full((B, L, 2 * H, 48 + 64), 7.0, device="cuda", dtype=BF16)
    got = DA.diff_attn_bwd(odd, swapped, band, lam, o, saved, go, gv_out=out[..., 48:])
    assert got[2].data_ptr() == out[..., 48:].data_ptr() and (out[..., :48] == 7).all()
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a, b)
    one = q[:, :, :1].expand(-1, -1, 2 * H, -1)                   # all heads the same query
    o, *_ = _own(one, k, v, lam)
    assert torch.equal(o, _own(one.contiguous(), k, v, lam)[0])
    g1 = go[:1].expand(B, -1, -1, -1)
    a = DA.diff_attn_bwd(q, k, v, lam, want_o, want_saved, g1)
    b = DA.diff_attn_bwd(q, k, v, lam, want_o, want_saved, g1.contiguous())
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    single = q[:1].as_strided((1, L, 2 * H, 64), (1, 2 * H * 64, 64, 1))        # the stride of a single batch counts for nothing
    assert torch.equal(_own(single, k[:1], v[:1], lam)[0], want_o[:1])


def test_rows_behind_the_last_one_stay():
    """Neighbours of the dv output keep their values at a ragged length."""
    from imfvideo_b200.ops import diffattn as DA

    B, L, H = 1, 77, 1
    q, k, v, lam, go = _inputs(B, L, H, seed=1)
    o, _, saved = _own(q, k, v, lam)
    buf = torch.full((L + 60, 2 * H, 64), 3.0, device="cuda", dtype=BF16)
    DA.diff_attn_bwd(q, k, v, lam, o, saved, go, gv_out=buf[:L].unsqueeze(0))
    assert (buf[L:] == 3).all()


def test_infinite_and_nan_values_stay_in_their_row():
    """A NaN in one query reaches that query's row alone; lse of rows far below zero leaves the others finite."""
    q, k, v, lam, _ = _inputs(1, 300, 1, seed=2)
    clean = _own(q, k, v, lam)[0]
    bad = q.clone()
    bad[0, 17, 1, 5] = float("nan")
    o = _own(bad, k, v, lam)[0]
    rows = torch.ones(300, dtype=torch.bool, device="cuda")
    rows[17] = False
    assert torch.equal(o[0, rows], clean[0, rows]) and o[0, 17].isnan().all()


def test_nan_keys_give_nan_gradients_to_their_pair_alone():
    from imfvideo_b200.ops import diffattn as DA

    q, k, v, lam, go = _inputs(1, 100, 2, seed=2)            # one K/V tile: dq has one order
    clean = DA.diff_attn_bwd(q, k, v, lam, *_own(q, k, v, lam)[::2], go)
    bad = k.clone()
    bad[0, 17, 0, 5] = float("nan")
    got = DA.diff_attn_bwd(q, bad, v, lam, *_own(q, bad, v, lam)[::2], go)
    for a, b in zip(got[:3], clean[:3]):
        assert a[:, :, 0].isnan().all() and torch.equal(a[:, :, 2:], b[:, :, 2:])
    assert got[3][1] == clean[3][1]


def _room(gb):
    free = torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved() - torch.cuda.memory_allocated()
    if free < gb * 1e9:
        pytest.skip(f"{gb} GB of device memory")


@pytest.mark.parametrize("dim", [0, 1])
def test_strides_past_32_bits(dim):
    """Bands of one buffer whose batches (or rows) are so far apart that offsets need 64 bits."""
    from imfvideo_b200.ops import diffattn as DA

    B, L, H = 2, 70, 1
    ins = _inputs(B, L, H, seed=3)
    n = (B, L)[dim] - 1
    far = (2 ** 31 + 640) // n // 8 * 8 + 8                  # n strides of it pass 2^31 elements
    _room(6 * far * n / 2 ** 31)
    near = 640                                               # 2H heads of five tensors
    buf = torch.empty(n * far + near * max(B, L) + 640, device="cuda", dtype=BF16)
    st = (far, near) if dim == 0 else (near, far)
    bands = [buf[i * 128:].as_strided((B, L, 2 * H, 64), (*st, 64, 1)) for i in range(5)]
    q, k, v, go = (b.copy_(t) for b, t in zip(bands, (*ins[:3], ins[4])))
    lam = ins[3]
    o, _, saved = _own(q, k, v, lam)
    want, _, want_saved = _own(*ins[:4])
    assert torch.equal(o, want) and all(torch.equal(a, b) for a, b in zip(saved, want_saved))
    got = DA.diff_attn_bwd(q, k, v, lam, o, saved, go, gv_out=bands[4])
    assert got[2].data_ptr() == bands[4].data_ptr()
    for a, b in zip(got, DA.diff_attn_bwd(*ins[:4], want, want_saved, ins[4])):
        assert torch.equal(a, b)                             # (one K/V tile)


def test_tensors_past_32_bits():
    """More than 2^31 elements: the last batches agree with the formulas."""
    from imfvideo_b200.ops import diffattn as DA

    B, L, H = 65540, 128, 2
    _room(70)
    g = _gen(5)
    q, k, v, go = (torch.randn(B, L, 2 * H, 64, device="cuda", dtype=BF16, generator=g) for _ in range(4))
    lam = torch.tensor([0.4, 0.7], device="cuda")
    tail = [t[-3:].clone() for t in (q, k, v)]
    o, do, _ = _own(q, k, v, lam, (go, go, go), need_bwd=False)
    _within(_wide(o[-3:]), *_forward64(*tail, lam)[2:4], "o")
    _within(_wide(do[-3:]), *_tangent64(*tail, lam, (go[-3:],) * 3), "do")
    del do
    o, _, saved = _own(q, k, v, lam)
    dq, dk, dv, _ = DA.diff_attn_bwd(q, k, v, lam, o, saved, go)
    dlam = DA.diff_attn_bwd(*tail, lam, o[-3:], (saved[0][-3:], saved[1][-3:], saved[2][-3:]), go[-3:])[3]
    _check_grads(*tail, lam, go[-3:], (dq[-3:], dk[-3:], dv[-3:], dlam))


def test_two_graphs_at_once():
    """Two captured calls of different sizes, with tangents, split items and gradients, replayed on two streams."""
    from imfvideo_b200.ops import diffattn as DA

    calls, graphs = [], []
    for L, H in ((1100, 2), (1500, 1)):
        q, k, v, lam, tan = _inputs(1, L, H, seed=L, tangent=True)
        o, _, saved = _own(q, k, v, lam)

        def call(q=q, k=k, v=v, lam=lam, tan=tan, o=o, saved=saved):
            return (*_own(q, k, v, lam, tan, need_bwd=False)[:2], *DA.diff_attn_bwd(q, k, v, lam, o, saved, tan[0])[1:])
        want = call()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            out = call()
        calls.append((call, want, out))              # (call keeps its inputs alive)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for _, want, got in calls:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_far_negative_scores():
    """lse of -400: the rows behind the last key must not turn infinite in the backward pass."""
    from imfvideo_b200.ops import diffattn as DA

    g = _gen(0)
    base = torch.randn(1, 1, 2, 64, device="cuda", generator=g)
    q = (base + 0.05 * torch.randn(1, 100, 2, 64, device="cuda", generator=g)).bfloat16()
    k = (-50 * base / base.norm(dim=-1, keepdim=True) + 0.05 * torch.randn(1, 100, 2, 64, device="cuda", generator=g)).bfloat16()
    v = torch.randn(1, 100, 2, 64, device="cuda", generator=g).bfloat16()
    go = torch.randn(1, 100, 2, 64, device="cuda", generator=g).bfloat16()
    lam = torch.tensor([0.5], device="cuda")
    o, _, saved = _own(q, k, v, lam, scale=1.0)
    assert saved[2].max() < -200
    for t in DA.diff_attn_bwd(q, k, v, lam, o, saved, go, 1.0):
        assert t.isfinite().all()


def test_fixed_order_is_bit_identical(monkeypatch):
    from imfvideo_b200.ops import diffattn as DA
    from imfvideo_b200.ops import kernels as K

    q, k, v, lam, go = _inputs(1, 1700, 2, seed=4)
    o, _, saved = _own(q, k, v, lam)
    free = DA.diff_attn_bwd(q, k, v, lam, o, saved, go)
    monkeypatch.setattr(K, "DETERMINISTIC", True)
    a = DA.diff_attn_bwd(q, k, v, lam, o, saved, go)
    b = DA.diff_attn_bwd(q, k, v, lam, o, saved, go)
    for x, y, z in zip(a, b, free):
        assert torch.equal(x, y)
    for x, z in zip(a[1:], free[1:]):
        assert torch.equal(x, z)                  # everything but dq has one order anyway
    _check_grads(q, k, v, lam, go, a)


def test_autograd_streams_and_graph_replay():
    """Gradients through the dual function; the same on another stream, beside another call, and from a captured graph
    on new inputs."""
    from imfvideo_b200.ops import dual as D

    def step(q, k, v, lam, go):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
        o = D.diff_attention(*(D.Dual(t) for t in leaves[:3]), leaves[3]).p
        return (o.detach(),) + torch.autograd.grad(o, leaves, go)

    # 128 rows of keys: one K/V tile, so dq has one order too
    ins = [_inputs(2, 128, 2, seed=s) for s in (1, 2)]
    want = [step(*i) for i in ins]
    _check_grads(*ins[0], want[0][1:])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = []
    for i, s in zip(ins, streams):
        with torch.cuda.stream(s):
            got.append(step(*i))
    torch.cuda.synchronize()
    for g_, w_ in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g_, w_))
    static = [t.clone() for t in ins[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for t, n in zip(static, ins[1]):
        t.copy_(n)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want[1]))


def test_scalar_weight_gradient_sums_over_pairs():
    from imfvideo_b200.ops import dual as D

    q, k, v, _, go = _inputs(1, 130, 3, seed=9)
    lam = torch.tensor(0.4, device="cuda", requires_grad=True)
    o = D.diff_attention(D.Dual(q), D.Dual(k), D.Dual(v), lam).p
    g, = torch.autograd.grad(o, lam, go)
    per = torch.full((3,), 0.4, device="cuda", requires_grad=True)
    gp, = torch.autograd.grad(D.diff_attention(D.Dual(q), D.Dual(k), D.Dual(v), per).p, per, go)
    assert g.shape == () and abs(g.item() - gp.sum().item()) <= 1e-5 * gp.abs().sum().item()


def test_partial_tangents_count_as_zero():
    from imfvideo_b200.ops import dual as D

    q, k, v, lam, (dq, dk, dv) = _inputs(1, 90, 1, seed=11, tangent=True)
    zero = torch.zeros_like(q)
    a = D.diff_attention(D.Dual(q, dq), D.Dual(k), D.Dual(v), lam)
    b = D.diff_attention(D.Dual(q, dq), D.Dual(k, zero), D.Dual(v, zero), lam)
    assert torch.equal(a.t, b.t) and not a.t.requires_grad


def test_empty():
    from imfvideo_b200.ops import diffattn as DA

    for shape in ((0, 5, 2, 64), (2, 0, 2, 64), (2, 5, 0, 64)):
        z = torch.zeros(shape, device="cuda", dtype=BF16)
        lam = torch.ones(shape[2] // 2, device="cuda")
        o, do, saved = DA.diff_attn_fwd(z, z, z, lam, z, z, z)
        assert o.shape == do.shape == z.shape
        dq, dk, dv, dlam = DA.diff_attn_bwd(z, z, z, lam, o, saved, z)
        assert dq.shape == z.shape and (dlam == 0).all() and dlam.shape == lam.shape


def _dv_over_sliding_rows(lam, o, saved, go):
    """q's rows lie over one another, and dv over them"""
    from imfvideo_b200.ops import diffattn as DA

    buf = torch.zeros(1, 100, 4, 64, device="cuda", dtype=BF16)
    q = buf.as_strided(go.shape, (100 * 256, 64, 64, 1))
    return DA.diff_attn_bwd(q, go, go, lam, o, saved, go, gv_out=buf[:, :40])


def test_refusals():
    from imfvideo_b200.ops import diffattn as DA

    q, k, v, lam, go = _inputs(1, 40, 2)
    o, _, saved = _own(q, k, v, lam)
    o2, low, lse = saved
    bad = [lambda: _own(q.float(), k, v, lam), lambda: _own(q[:, :, :3], k, v, lam),
           lambda: _own(q[..., :32], k[..., :32], v[..., :32], lam), lambda: _own(q, k[:, :39], v, lam),
           lambda: _own(q, k, v, lam[:1]), lambda: _own(q, k, v, lam.double()), lambda: _own(q, k, v, lam.cpu()),
           lambda: _own(q, k, v, lam, scale=0.0), lambda: _own(q, k, v, lam, scale=-1.0),
           lambda: _own(q, k, v, lam, scale=math.nan), lambda: _own(q, k, v, lam, scale=math.inf),
           lambda: _own(q, k, v, lam, (q, None, None)),
           lambda: DA.diff_attn_bwd(q, k, v, lam, o, (o2, low, lse[:, :1]), go),
           lambda: DA.diff_attn_bwd(q, k, v, lam, o, (o2, low[..., :64], lse), go),
           lambda: DA.diff_attn_bwd(q, k, v, lam, o, (o2.float(), low, lse), go),
           lambda: DA.diff_attn_bwd(q, k, v, lam, o, saved, go, gv_out=q[:, :1].expand_as(q)),
           lambda: DA.diff_attn_bwd(q, k, v, lam, o, saved, go, gv_out=v),
           lambda: _dv_over_sliding_rows(lam, o, saved, go),
           lambda: DA.diff_attn_bwd(q, k, v, lam, o, saved, go, gv_out=torch.empty(
               1, 40, 4, 66, device="cuda", dtype=BF16)[..., :64])]
    for f in bad:
        with pytest.raises(ValueError):
            f()
