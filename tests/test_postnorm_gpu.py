"""GPU: norms around a branch against the formulas in 64 bits.

fp32 results: sums of up to 8,192 terms of one sign as a tree of chains of at most 64 and a few dozen additions,
so a row's norm is off by 100 * 2^-24 at the very most; with the reciprocal root's and the products' roundings
the bound is 1e-5 of the magnitude of the terms that are added.  Column sums add a row a step in chains of at
most rows / CTAs: 2e-5 of the sum of magnitudes.  bf16 results add half a step, 2^-8 of the value."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U = {BF16: torch.finfo(BF16).eps / 2, F32: torch.finfo(F32).eps / 2}
EPS, REL = 1e-5, 1e-5
FORMS = [f for f in itertools.product([True, False], [True, False], [True, False]) if f[0] or not f[1]]
SIZES = [(1, 8), (3, 64), (7, 256), (532, 256), (33, 264), (300, 512), (257, 520), (129, 1000), (64, 1024), (65, 1536),
         (20, 2048), (9, 2056), (5, 4096), (5, 8192), (2500, 768),
         (450, 1032), (300, 1280), (450, 1288), (299, 1792), (20, 1800)]


def _inputs(R, D, has_res, has_scale, has_pre, dtype=BF16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    v = dict(res=3 * rnd(R, D) if has_res else None, y=(rnd(R, D) * torch.exp(0.5 * rnd(D))).to(dtype),
             post=1 + 0.2 * rnd(D), gate=0.5 * rnd(D), r=1 + 0.2 * rnd(D) if has_scale else None,
             pre=1 + 0.2 * rnd(D) if has_pre else None)
    t = dict(dres=rnd(R, D) if has_res else None, dy=rnd(R, D).to(dtype))
    go = dict(gx=rnd(R, D), gn=rnd(R, D).to(dtype) if has_pre else None)
    return v, t, go


def _d(v):
    return {k: None if t is None else t.double() for k, t in v.items()}


def _mean(t):
    return t.mean(-1, keepdim=True)


def _forward64(v, t=None):
    """Results and the magnitudes of the terms that make them."""
    v = _d(v)
    w, r = v["gate"] * v["post"], 1.0 if v["r"] is None else v["r"]
    iy = (_mean(v["y"] ** 2) + EPS).rsqrt()
    yh = v["y"] * iy
    res = 0.0 if v["res"] is None else v["res"] * r
    x = w * yh + res
    ax = (w * yh).abs() + abs(res)
    ix = (_mean(x ** 2) + EPS).rsqrt()
    out = {"x": (x, ax)}
    if v["pre"] is not None:
        out["n"] = (x * ix * v["pre"], ax * ix * v["pre"].abs())
    if t is not None:
        t = _d(t)
        dres = 0.0 if t["dres"] is None else t["dres"] * r
        inner = t["dy"] - yh * _mean(yh * t["dy"])
        dx = w * iy * inner + dres
        adx = w.abs() * iy * (t["dy"].abs() + yh.abs() * _mean((yh * t["dy"]).abs())) + abs(dres)
        out["dx"] = (dx, adx)
        if v["pre"] is not None:
            xh, axh = x * ix, ax * ix
            out["dn"] = (v["pre"] * ix * (dx - xh * _mean(xh * dx)),
                         v["pre"].abs() * ix * (adx + axh * _mean(axh * adx)))
    return out


def _within(got, want, mag, rel, what):
    over = (got.double() - want).abs() - (rel * mag + U[got.dtype] * want.abs() + 1e-30)
    assert not got.isnan().any() and over.max().item() <= 0, (what, over.max().item())


def _check_forward(v, t, got):
    want = _forward64(v, t)
    for name, g in zip(("x", "n", "dx", "dn"), got):
        assert (g is None) == (name not in want)
        if g is not None:
            _within(g, *want[name], REL, name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("R,D", SIZES)
def test_forward_and_tangent(R, D, form, dtype):
    from imfvideo_b200.ops import postnorm as PN

    v, t, _ = _inputs(R, D, *form, dtype=dtype)
    args = (v["res"], v["y"], v["post"], v["gate"], EPS, v["r"], v["pre"])
    got = PN.norm_add_norm_fwd(*args)
    _check_forward(v, None, got)
    both = PN.norm_add_norm_fwd(*args, t["dres"], t["dy"])
    _check_forward(v, t, both)
    assert torch.equal(both[0], got[0])


def _backward64(v, go):
    v, go = _d(v), _d(go)
    w, r = v["gate"] * v["post"], 1.0 if v["r"] is None else v["r"]
    iy = (_mean(v["y"] ** 2) + EPS).rsqrt()
    yh = v["y"] * iy
    res = 0.0 if v["res"] is None else v["res"]
    x, ax = w * yh + res * r, (w * yh).abs() + abs(res * r)
    ix = (_mean(x ** 2) + EPS).rsqrt()
    xh, axh = x * ix, ax * ix
    g, ag = go["gx"], go["gx"].abs()
    out = {}
    if v["pre"] is not None:
        a = v["pre"] * go["gn"]
        g = g + ix * (a - xh * _mean(a * xh))
        ag = ag + ix * (a.abs() + axh * _mean(a.abs() * axh))
        out["g_pre"] = ((go["gn"] * xh).sum(0), (go["gn"].abs() * axh).sum(0))
    if v["res"] is not None:
        out["g_res"] = (g * r, ag * abs(r))
    if v["r"] is not None:
        out["g_r"] = ((g * res).sum(0), (ag * abs(res)).sum(0))
    s, sa = (g * yh).sum(0), (ag * yh.abs()).sum(0)
    out["g_gate"], out["g_post"] = (s * v["post"], sa * v["post"].abs()), (s * v["gate"], sa * v["gate"].abs())
    b, ab = g * w, ag * w.abs()
    out["g_y"] = (iy * (b - yh * _mean(b * yh)), iy * (ab + yh.abs() * _mean(ab * yh.abs())))
    return out


def _check_backward(v, go, got):
    want = _backward64(v, go)
    for name, g in zip(("g_res", "g_y", "g_pre", "g_r", "g_gate", "g_post"), got):
        assert (g is None) == (name not in want), name
        if g is not None:
            _within(g, *want[name], REL if name in ("g_res", "g_y") else 2e-5, name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("R,D", SIZES)
def test_backward(R, D, form, dtype):
    from imfvideo_b200.ops import postnorm as PN

    v, _, go = _inputs(R, D, *form, dtype=dtype, seed=1)
    _check_backward(v, go, PN.norm_add_norm_bwd(v["res"], v["y"], v["post"], v["gate"], EPS, v["r"], v["pre"],
                                                go["gx"], go["gn"]))


@pytest.mark.parametrize("which", ["x", "n"])
def test_gradient_of_one_output(which):
    """Only x or only n is used; also what autograd asks for when some inputs need no gradient."""
    from imfvideo_b200.ops import dual as D

    v, _, go = _inputs(70, 256, True, True, True)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items()}
    x, n = D.norm_add_norm(D.Dual(leaves["res"]), D.Dual(leaves["y"]), leaves["post"], leaves["gate"], EPS,
                           res_scale=leaves["r"], pre=leaves["pre"])
    if which == "x":
        grads = torch.autograd.grad(x.p, [leaves[k] for k in ("res", "y", "r", "gate", "post")], go["gx"])
        go = dict(gx=go["gx"], gn=torch.zeros_like(go["gn"]))
        names = ("g_res", "g_y", "g_r", "g_gate", "g_post")
    else:
        grads = torch.autograd.grad(n.p, [leaves[k] for k in ("y", "pre", "post")], go["gn"])
        go = dict(gx=torch.zeros_like(go["gx"]), gn=go["gn"])
        names = ("g_y", "g_pre", "g_post")
    want = _backward64(v, go)
    for name, g in zip(names, grads):
        _within(g, *want[name], 2e-5, name)


def test_duals_strides_and_leading_dimensions():
    from imfvideo_b200.ops import dual as D

    v, t, _ = _inputs(60, 128, True, False, True)
    call = lambda v, t: D.norm_add_norm(D.Dual(v["res"], t["dres"]), D.Dual(v["y"], t["dy"]), v["post"], v["gate"], EPS,
                                        pre=v["pre"])
    want = call(v, t)
    band = lambda z: torch.cat([z, z], -1)[:, 128:]                            # rows of a wider tensor
    off = torch.empty(60 * 128 + 1, device="cuda", dtype=BF16)[1:].view(60, 128).copy_(v["y"])      # unaligned
    vec = torch.stack([v["post"], v["gate"]], 1)
    got = call(dict(v, res=band(v["res"]), y=off, post=vec[:, 0]), dict(t, dy=band(t["dy"])))
    three = lambda d: {k: z.view(3, 20, 128) if z is not None and z.dim() == 2 else z for k, z in d.items()}
    got3 = call(three(v), three(t))
    for a, b, c in zip(want, got, got3):
        assert torch.equal(a.p, b.p) and torch.equal(a.t, b.t)
        assert c.p.shape == (3, 20, 128) and torch.equal(a.p, c.p.view(60, 128)) and torch.equal(a.t, c.t.view(60, 128))


def test_rows_of_zeros_and_nan_rows():
    """A row of zeros has a norm of sqrt(eps); a NaN stays in its row."""
    from imfvideo_b200.ops import postnorm as PN

    v, t, go = _inputs(40, 512, True, True, True)
    v["y"][3] = 0
    v["y"][4], v["res"][4] = 0, 0
    args = lambda v: (v["res"], v["y"], v["post"], v["gate"], EPS, v["r"], v["pre"])
    clean = PN.norm_add_norm_fwd(*args(v), t["dres"], t["dy"])
    _check_forward(v, t, clean)
    back = PN.norm_add_norm_bwd(*args(v), go["gx"], go["gn"])
    _check_backward(v, go, back)
    bad = dict(v, y=v["y"].clone())
    bad["y"][17, 100] = float("nan")
    got = PN.norm_add_norm_fwd(*args(bad), t["dres"], t["dy"])
    rows = torch.arange(40, device="cuda") != 17
    for a, b in zip(got, clean):
        assert torch.equal(a[rows], b[rows]) and a[17].isnan().all()


def test_streams_and_graph_replay():
    from imfvideo_b200.ops import dual as D

    def step(res, y, post, gate, r, pre, gx, gn):
        leaves = [z.detach().requires_grad_() for z in (res, y, post, gate, r, pre)]
        x, n = D.norm_add_norm(D.Dual(leaves[0]), D.Dual(leaves[1]), leaves[2], leaves[3], EPS, res_scale=leaves[4],
                               pre=leaves[5])
        return (x.p.detach(), n.p.detach()) + torch.autograd.grad([x.p, n.p], leaves, [gx, gn])

    ins = []
    for s in (0, 1):
        v, _, go = _inputs(900, 384, True, True, True, seed=s)
        ins.append([*v.values(), *go.values()])
    want = [step(*i) for i in ins]
    torch.cuda.synchronize()
    got = []
    for i in ins:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(step(*i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    static = [z.clone() for z in ins[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for z, n in zip(static, ins[1]):
        z.copy_(n)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want[1]))


def test_tensors_past_32_bits():
    """More than 2^31 elements: the last rows agree with the formulas."""
    from imfvideo_b200.ops import postnorm as PN

    R, D = 262160, 8192
    if torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved() - torch.cuda.memory_allocated() < 60e9:
        pytest.skip("60 GB of device memory")
    v, t, go = _inputs(20, D, True, True, True, seed=3)
    big = lambda z: torch.zeros(R, D, device="cuda", dtype=z.dtype)
    res, y, gx, gn = (big(z) for z in (v["res"], v["y"], go["gx"], go["gn"]))
    for b, z in zip((res, y, gx, gn), (v["res"], v["y"], go["gx"], go["gn"])):
        b[-20:] = z
    args = (res, y, v["post"], v["gate"], EPS, v["r"], v["pre"])
    x, n, _, _ = PN.norm_add_norm_fwd(*args)
    _check_forward(v, None, (x[-20:], n[-20:], None, None))
    assert not x[:-20].any() and not n[:-20].any()
    del x, n
    got = PN.norm_add_norm_bwd(*args, gx, gn)
    _check_backward(v, go, (got[0][-20:], got[1][-20:], *got[2:]))


def test_two_graphs_at_once():
    """Two captured calls of different widths replayed on two streams."""
    from imfvideo_b200.ops import postnorm as PN

    calls, graphs = [], []
    for R, D in ((700, 256), (300, 1536)):
        v, t, go = _inputs(R, D, True, True, True, seed=D)
        args = (v["res"], v["y"], v["post"], v["gate"], EPS, v["r"], v["pre"])

        def call(args=args, t=t, go=go):
            return (*PN.norm_add_norm_fwd(*args, t["dres"], t["dy"]), *PN.norm_add_norm_bwd(*args, go["gx"], go["gn"]))
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


def test_types_that_have_no_kernel_take_the_formulas():
    from imfvideo_b200.ops import dual as D

    v, _, _ = _inputs(5, 64, True, False, True)
    x, n = D.norm_add_norm(D.Dual(v["res"].double()), D.Dual(v["y"].double()), v["post"], v["gate"], EPS, pre=v["pre"])
    assert x.p.dtype == n.p.dtype == torch.float64
    y = torch.randn(5, 12, device="cuda")                                      # 12 channels: no multiple of 8
    x, _ = D.norm_add_norm(None, D.Dual(y), torch.ones(12, device="cuda"), torch.ones(12, device="cuda"), EPS)
    assert torch.allclose(x.p, y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS), rtol=1e-5)


def test_empty_and_refusals():
    from imfvideo_b200.ops import postnorm as PN

    v, t, go = _inputs(6, 64, True, True, True)
    a = lambda **kw: [{**v, **kw}[k] for k in ("res", "y", "post", "gate")] + [EPS] + [{**v, **kw}[k] for k in ("r", "pre")]
    z = dict(res=v["res"][:0], y=v["y"][:0])
    assert all(o.shape == (0, 64) for o in PN.norm_add_norm_fwd(*a(**z), t["dres"][:0], t["dy"][:0]))
    back = PN.norm_add_norm_bwd(*a(**z), go["gx"][:0], go["gn"][:0])
    assert back[0].shape == back[1].shape == (0, 64) and all((g == 0).all() and g.shape == (64,) for g in back[2:])
    bad = [lambda: PN.norm_add_norm_fwd(*a(y=v["y"].half())), lambda: PN.norm_add_norm_fwd(*a(post=v["post"].double())),
           lambda: PN.norm_add_norm_fwd(*a(res=v["res"][:5])), lambda: PN.norm_add_norm_fwd(*a(res=v["res"].bfloat16())),
           lambda: PN.norm_add_norm_fwd(*a(res=None)), lambda: PN.norm_add_norm_fwd(*a(gate=v["gate"].cpu())),
           lambda: PN.norm_add_norm_fwd(*a(), t["dres"], None), lambda: PN.norm_add_norm_fwd(*a(pre=v["pre"][:8])),
           lambda: PN.norm_add_norm_fwd(*a(), t["dres"], t["dy"].float()),
           lambda: PN.norm_add_norm_bwd(*a(), go["gx"], None), lambda: PN.norm_add_norm_bwd(*a(pre=None), go["gx"], go["gn"]),
           lambda: PN.norm_add_norm_fwd(None, torch.zeros(2, 8200, device="cuda"), torch.ones(8200, device="cuda"),
                                        torch.ones(8200, device="cuda"), EPS),
           lambda: PN.norm_add_norm_fwd(None, torch.zeros(2, 12, device="cuda"), torch.ones(12, device="cuda"),
                                        torch.ones(12, device="cuda"), EPS)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
