"""GPU: activations in 8 bits and the backward operators on them, against the formulas in 64 bits."""
import math

import pytest
import torch

from imfvideo_b200.ops import reference as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
TANH = 2.0 ** -10.9          # relative error of the hardware's hyperbolic tangent (PTX ISA: 2^-11)


@pytest.fixture(scope="module")
def A():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from imfvideo_b200.ops import cuda as cu

    assert cu.available(), "kernel library must load on a GPU box"
    from imfvideo_b200.ops import act8

    return act8


@pytest.fixture(scope="module")
def K(A):
    from imfvideo_b200.ops import kernels

    return kernels


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, s=1.0, dtype=BF16):
    return (torch.randn(*shape, device="cuda", generator=g) * s).to(dtype)


def _activations(g, rows, C, dtype=BF16):
    """Channels of different size, some of them far above the rest."""
    s = torch.exp(torch.randn(C, device="cuda", generator=g))
    return (torch.randn(rows, C, device="cuda", generator=g) * s).to(dtype)


def _same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def _check_store(A, x, p=None):
    p = A.store8(x) if p is None else p
    flat = x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    codes, steps = ref.store8(flat)
    assert torch.equal(p.codes, codes) and torch.equal(p.steps, steps)
    v = A.restore8(p)
    want = ref.values8(codes, steps, x.shape[-1]).to(x.dtype).view(x.shape)
    assert v.dtype == x.dtype and v.shape == x.shape and _same(v, want)
    return p


# ------------------------------------------------------------- store, restore ---
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,C", [(1, 1), (1, 32), (3, 7), (5, 33), (2, 64), (77, 48), (130, 528), (31, 1021),
                                    (2068, 682), (4099, 1376), (9000, 2064), (9000, 2048), (6000, 1021), (90000, 64)])
def test_store_and_restore(A, dtype, rows, C):
    _check_store(A, _activations(_gen(rows + C), rows, C, dtype))


def test_edges_of_the_format(A):
    from test_act8 import edge_rows

    for dtype in (BF16, F32):
        _check_store(A, edge_rows().cuda().to(dtype))
    top = torch.full((2, 64), torch.finfo(F32).max, device="cuda")
    top[1] = -top[1]
    _check_store(A, top)
    every = torch.arange(-127, 128, device="cuda").to(F32)              # every code, at every step
    x = torch.zeros(249, 9, 32, device="cuda")
    x.view(249, -1)[:, :255] = every
    x[:, :, 31] = 127.0                                                 # so that the step is one
    x = x * torch.exp2(torch.arange(249, device="cuda").double() - 127).to(F32)[:, None, None]
    p = _check_store(A, x.view(249, -1))
    assert torch.equal(p.steps[:, :8].long(), torch.arange(249, device="cuda")[:, None].expand(249, 8))
    assert torch.equal(A.restore8(p), x.view(249, -1))


def test_strides_alignment_and_many_tensors(A):
    g = _gen(5)
    wide = _randn(g, 2, 50, 3, 112)
    odd = _randn(g, 40, 203)
    f = _randn(g, 6, 5, 4, 3, 40, dtype=F32)
    xs = [wide[..., 48:], wide.transpose(1, 2), wide[:, ::3], odd[:, 3:], odd[:, 1:70], odd.t()[:, :33],
          wide[:, :, 1], f[..., 4:], f.permute(0, 2, 1, 3, 4), f.permute(3, 1, 0, 2, 4)[::2, :, :, ::3], odd[7],
          odd[:, 5], torch.empty(0, 40, device="cuda"), _randn(g, 9, 1, 8).expand(9, 4, 8)]
    xs += [_randn(g, 3 + i, 40 + i) for i in range(25)]                 # more than one launch takes
    ps = A.store8(xs)
    for x, p in zip(xs, ps):
        _check_store(A, x, p)
    for p, v in zip(ps, A.restore8(ps)):
        assert _same(v, p.restore())


def test_restore_into_views_leaves_the_rest(A):
    g = _gen(6)
    p, q = A.store8([_randn(g, 2, 33, 3, 45), _randn(g, 66, 77, dtype=F32)])
    a = torch.full((2, 33, 3, 64), -7.75, dtype=BF16, device="cuda")
    b = torch.full((66, 100), -7.75, device="cuda")
    out = A.restore8([p, q], [a[..., 11:56], b[:, 23:]])
    assert _same(a[..., 11:56], p.restore()) and _same(b[:, 23:], q.restore())
    assert (a[..., :11] == -7.75).all() and (a[..., 56:] == -7.75).all() and (b[:, :23] == -7.75).all()
    assert out[0].data_ptr() == a[..., 11:56].data_ptr()
    with pytest.raises(ValueError):
        A.restore8(q, torch.empty(77, 66, device="cuda").t())
    with pytest.raises(ValueError):
        A.restore8([p], [torch.empty(2, 33, 3, 45, dtype=BF16)])         # on the CPU
    with pytest.raises(ValueError):
        A.restore8(p, torch.empty(2, 1, 3, 45, dtype=BF16, device="cuda").expand(2, 33, 3, 45))
    with pytest.raises(ValueError):
        A.restore8(q, torch.empty(1, 77, device="cuda").expand(66, 77))


def test_offsets_beyond_32_bits(A):
    """Rows 2^30 elements apart, and a tensor of more than 2^32 bytes of codes."""
    buf = torch.zeros(2 * 2 ** 30 + 128, dtype=BF16, device="cuda")
    x = buf.as_strided((3, 80), (2 ** 30, 1))
    x.copy_(_randn(_gen(7), 3, 80))
    _check_store(A, x)
    y = torch.zeros_like(buf).as_strided((3, 80), (2 ** 30, 1))
    A.restore8(A.store8(x), y)
    assert _same(y, A.store8(x).restore())
    del buf, x, y
    rows = 2 ** 32 // 4096 + 3
    big = torch.ones(rows, 4096, dtype=BF16, device="cuda")
    big[-1] = torch.arange(4096, device="cuda") % 61
    p = A.store8(big)
    v = A.restore8(p)
    assert torch.equal(v[-2:], A.store8(big[-2:]).restore()) and bool((v[:-1] == 1).all())
    del big, p, v
    torch.cuda.empty_cache()


# ------------------------------------------------------------- weight gradient ---
def _wgrad_check(got, dy, p, base=None):
    x = ref.values8(p.codes, p.steps, p.cols)
    want = dy.double().t() @ x.double()
    size = dy.double().abs().t() @ x.double().abs()
    if base is not None:
        want, size = want + base.double(), size + base.double().abs()
    # every addition may drop 2^-23 of a running sum that is at most `size`
    assert ((got.double() - want).abs() <= (dy.shape[0] + 4) * 2.0 ** -23 * size).all()
    assert (got.double() - want).norm() <= 1e-5 * want.norm()


@pytest.mark.parametrize("rows,N,C", [(1, 8, 1), (1, 136, 300), (7, 16, 31), (63, 128, 128), (64, 8, 64),
                                      (65, 264, 77), (130, 528, 256), (532, 528, 257), (1000, 144, 512),
                                      (4099, 40, 1021), (2068, 1376, 256), (29140, 256, 128), (16500, 72, 40),
                                      (70, 5400, 1000), (8300, 10000, 500), (300, 20000, 130)])
def test_weight_gradient(A, K, rows, N, C):
    g = _gen(rows)
    dy, p = _randn(g, rows, N), A.store8(_activations(g, rows, C))
    got = A.gemm_wgrad8(dy, p)
    assert got.dtype == F32 and got.shape == (N, C)
    _wgrad_check(got, dy, p)
    assert torch.equal(A.gemm_wgrad8(dy, p), got)                        # fixed order
    base = torch.randn(N, C, device="cuda", generator=g)
    acc = base.clone()
    assert A.gemm_wgrad8(dy, p, out=acc, accumulate=True) is acc
    _wgrad_check(acc, dy, p, base)
    K.check_status()


def test_weight_gradient_views(A, K):
    """A band of a wider dY, a result inside a guarded wider buffer at aligned and at odd pitches."""
    g = _gen(11)
    dy = _randn(g, 777, 400)[:, 8:8 + 203]
    p = A.store8(_randn(g, 3, 259, 100))                                 # rows from two dimensions
    for ld, c0 in ((160, 32), (163, 5)):
        for accumulate in (False, True):
            buf = torch.full((203, ld), 3.5, device="cuda")
            out = buf[:, c0:c0 + 100]
            A.gemm_wgrad8(dy, p, out=out, accumulate=accumulate)
            _wgrad_check(out, dy, p, torch.full((203, 100), 3.5, device="cuda") if accumulate else None)
            assert (buf[:, :c0] == 3.5).all() and (buf[:, c0 + 100:] == 3.5).all()
    assert torch.equal(A.gemm_wgrad8(dy[:0], A.store8(_randn(g, 0, 100))), torch.zeros(203, 100, device="cuda"))
    with pytest.raises(ValueError):
        A.gemm_wgrad8(_randn(g, 777, 203), p)                            # rows 406 bytes apart
    with pytest.raises(ValueError):
        A.gemm_wgrad8(_randn(g, 777, 208)[:, 1:], p)
    with pytest.raises(ValueError):
        A.gemm_wgrad8(_randn(g, 208, 777).t(), p)
    with pytest.raises(ValueError):
        A.gemm_wgrad8(dy, p, out=torch.empty(1, 100, device="cuda").expand(203, 100))
    K.check_status()


@pytest.mark.parametrize("rows,N,C", [(1, 406, 78), (63, 607, 738), (129, 82, 625), (127, 338, 486), (700, 40, 99)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_weight_gradient_leaves_what_is_beside_it(A, K, rows, N, C, accumulate):
    """Widths that are no whole 16 bytes, in front of a wider buffer's other columns and rows."""
    g = _gen(13)
    dy, p = _randn(g, rows, (N + 7) // 8 * 8)[:, :N], A.store8(_randn(g, rows, C))
    for pitch in (C + 1, (C + 3) // 4 * 4, (C + 7) // 4 * 4):
        buf = torch.randn(N + 2, pitch, device="cuda", generator=g)
        was = buf.clone()
        A.gemm_wgrad8(dy, p, out=buf[:N, :C], accumulate=accumulate)
        _wgrad_check(buf[:N, :C], dy, p, was[:N, :C] if accumulate else None)
        assert torch.equal(buf[:N, C:], was[:N, C:]) and torch.equal(buf[N:], was[N:])
    K.check_status()


@pytest.mark.parametrize("N,C", [(9216, 1024), (18800, 256), (18800, 128)])
@pytest.mark.parametrize("blocks", [1, 2, 3, 4, 5, 6, 7, 8, 9, 17])
def test_weight_gradient_of_walks_about_the_rings(A, K, N, C, blocks):
    """One tile a pair of CTAs (of 512, 256 and 128 columns), of fewer k-blocks than a ring has stages, as many
    and more, launch after launch: an arrival left over from one would disturb the next.  Whole numbers, so
    that every sum is exact."""
    g, rows = _gen(blocks), 64 * blocks - 5
    dy = torch.randint(-2, 3, (rows, N), device="cuda", generator=g).to(BF16)
    x = torch.randint(-60, 61, (rows, C), device="cuda", generator=g).to(BF16)
    x[:, ::32] = 100.0                                                   # so that the step is one
    p = A.store8(x)
    assert torch.equal(p.restore(), x)
    want = (dy.double().t() @ x.double()).float()
    outs = [A.gemm_wgrad8(dy, p) for _ in range(12)]
    assert want.abs().max() < 2 ** 24 and all(torch.equal(o, want) for o in outs)
    K.check_status()


@pytest.mark.parametrize("rows,N,C,bound", [(32780, 5472, 1024, 2e-6), (29140, 1376, 256, 5.5e-7)])
def test_weight_gradient_sums_in_chains(A, K, rows, N, C, bound):
    """The tensor core drops what is below 2^-25 of a running sum, half of that on average and always towards zero.  The
    sums of a random walk of n steps add up to n / sqrt(3) times its end, so a chain of n products of 16 rows
    loses 0.5 x 0.72 (the mean of a number's unit over it) x 2^-25 n / sqrt(3) = 6.2e-9 n of the result: 0.87e-6 for
    the 35 x 4 products of a chain at 1,024 columns (2.6e-6 for a slice of 103 x 4 in one chain), 4.7e-7 for the 19 x 4 at
    256 (9.4e-7 for a slice of 38 x 4).  Sums of chains and slices in 32 bits add 2^-24 each."""
    g = _gen(rows)
    dy, p = _randn(g, rows, N, s=0.02), A.store8(_activations(g, rows, C))
    want = dy.double().t() @ p.restore().double()
    base = torch.randn(N, C, device="cuda", generator=g) * want.std().float()
    out = base.clone()
    A.gemm_wgrad8(dy, p, out=out, accumulate=True)
    assert (A.gemm_wgrad8(dy, p).double() - want).norm() <= bound * want.norm()
    assert (out.double() - want - base.double()).norm() <= bound * (want + base.double()).norm()
    K.check_status()


@pytest.mark.parametrize("rows,N,C", [(16384, 2048, 1024), (29140, 1376, 256), (9000, 1000, 100)])
def test_weight_gradient_repeats(A, K, rows, N, C):
    """Two hundred launches, several chains of products each, give the same bits, which are the exact sums."""
    g = _gen(rows)
    dy = torch.randint(-2, 3, (rows, N), device="cuda", generator=g).to(BF16)
    x = torch.randint(-60, 61, (rows, C), device="cuda", generator=g).to(BF16)
    x[:, ::32] = 100.0                                                   # so that the step is one
    p = A.store8(x)
    want = dy.double().t() @ x.double()
    assert want.abs().max() < 2 ** 24 and (dy.double().abs().t() @ x.double().abs()).max() < 2 ** 24
    want, same = want.float(), torch.ones((), dtype=torch.bool, device="cuda")
    for _ in range(200):
        same &= (A.gemm_wgrad8(dy, p) == want).all()
    assert bool(same)
    K.check_status()


def test_weight_gradient_bad_values(A, K):
    """A group with an infinity makes NaN of its own 32 columns, an infinity of dY of its own row."""
    g = _gen(12)
    x, dy = _randn(g, 300, 96), _randn(g, 300, 64)
    x[17, 40] = float("inf")
    bad = torch.isnan(A.gemm_wgrad8(dy, A.store8(x)))
    assert bad[:, 32:64].all() and not bad[:, :32].any() and not bad[:, 64:].any()
    x[17, 40], dy[5, 9] = 1.0, float("nan")
    bad = torch.isnan(A.gemm_wgrad8(dy, A.store8(x)))
    assert bad[9].all() and bad.sum() == 96
    K.check_status()


# ------------------------------------------------------------- gated activation ---
@pytest.mark.parametrize("lbeta", [25.0, None])
@pytest.mark.parametrize("rows,F", [(1, 1), (1, 8), (3, 21), (77, 688), (130, 24), (2068, 682), (5000, 1000)])
def test_gated_activation(A, rows, F, lbeta):
    g = _gen(rows + F)
    gu, gout = _randn(g, rows, 2 * F, s=2.0), _randn(g, rows, F)
    p = A.store8(gu)
    grad, y = A.situ_bwd8(p, gout, 4.0, lbeta)
    v = ref.values8(p.codes, p.steps, 2 * F).double()
    gate, up, go = v[:, :F], v[:, F:], gout.double()
    dg, du, want_y = (t.double() for t in ref.situ_mul_grad(gate, up, gout, 4.0, lbeta))
    up_ = up.abs() if lbeta is None else (lbeta * torch.tanh(up / lbeta)).abs()
    # a = beta th sg with sg = (1 + tanh(gate / 2)) / 2: TANH |th| on th, TANH / 2 on sg (both below 1), so
    # 1.5 beta TANH on a; (1 - th^2) sg is 2.5 TANH off, beta th sg (1 - sg) at most 2 beta TANH; up' and
    # its derivative 1 - tu^2 TANH and 2 TANH; then one rounding to bf16
    a_err, da_err, u_err = 6.0 * TANH, (2.5 + 8.0) * TANH, TANH if lbeta else 0.0
    half = 2.0 ** -8
    assert ((y.double() - want_y).abs() <= half * want_y.abs() + 1.01 * (a_err + 4 * u_err) * up_ + 1e-30).all()
    assert ((grad[:, :F].double() - dg).abs() <= half * dg.abs() + 1.01 * go.abs() * up_ * (da_err + 2 * u_err)
            + 1e-30).all()
    assert ((grad[:, F:].double() - du).abs() <= half * du.abs() + 1.01 * go.abs() * (a_err + 8 * u_err) + 1e-30).all()
    wide = torch.full((rows, F + 24), 1e4, dtype=BF16, device="cuda")    # a band of a wider gradient
    wide[:, 8:8 + F] = gout
    again, y2 = A.situ_bwd8(p, wide[:, 8:8 + F], 4.0, lbeta)
    assert torch.equal(again, grad) and torch.equal(y2, y)


def test_gated_activation_refuses_scattered_columns(A):
    p = A.store8(torch.zeros(4, 64, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError):
        A.situ_bwd8(p, torch.zeros(32, 4, dtype=BF16, device="cuda").t(), 4.0, 25.0)


# ------------------------------------------------------------- attention ---
def _attention(A, K, B, L, H, hd, seed, s=1.0):
    g = _gen(seed)
    q, k, v, go = (_randn(g, B, L, H, hd, s=x) for x in (s, 1.0, 1.0, 1.0))
    o, _, lse = K.attn_fwd(q, k, v)
    return A.store8([q, k, v, o]), lse, go, o


def _oracle(ps, lse, go, scale=None):
    v = [p.restore().double() for p in ps]
    q, k, v, o, go = (t.transpose(1, 2) for t in (*v, go.double()))
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    P = torch.exp(q @ k.transpose(-1, -2) * scale - lse.double()[..., None])
    ds = P * (go @ v.transpose(-1, -2) - (go * o).sum(-1, keepdim=True))
    out = (ds @ k * scale, ds.transpose(-1, -2) @ q * scale, P.transpose(-1, -2) @ go)
    return [t.transpose(1, 2) for t in out]


def _near(got, want, what):
    # q times a constant, the probabilities, dS and the result are each rounded to bf16, 2^-8 at most and
    # unrelated from element to element: 4 roundings of 2^-8 / sqrt(3) each add up to 2 2^-8 / sqrt(3) = 4.6e-3
    # of the norm at the very most of their range; twice that
    for a, b, name in zip(got, want, ("dq", "dk", "dv")):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel < 1e-2, (what, name, rel)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B,L,H", [(1, 2, 1), (2, 65, 3), (1, 128, 4), (3, 333, 2), (1, 1025, 5), (1, 2049, 1)])
def test_attention(A, K, B, L, H, hd):
    ps, lse, go, o = _attention(A, K, B, L, H, hd, L + H)
    got = A.attn_bwd8(*ps, lse, go)
    _near(got, _oracle(ps, lse, go), (B, L, H, hd))
    # a bf16 v and o in the place of packed ones, dv into a band
    v, o_ = ps[2].restore(), ps[3].restore()
    wide = torch.full((B, L, H, hd + 48), 3.0, dtype=BF16, device="cuda")
    dq, dk, dv = A.attn_bwd8(ps[0], ps[1], v, o_, lse, go, gv_out=wide[..., 48:])
    assert dv.data_ptr() == wide[..., 48:].data_ptr() and (wide[..., :48] == 3).all()
    _near((dq, dk, dv), [t.double() for t in got], "mixed")
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_one_token(A, K, hd):
    """dQ and dK of a single token are zero but for the rounding of delta (2^-17 of |go| |o|)."""
    ps, lse, go, o = _attention(A, K, 2, 1, 3, hd, 3)
    dq, dk, dv = A.attn_bwd8(*ps, lse, go)
    _, _, want = _oracle(ps, lse, go)
    q, k, v, _ = (p.restore().double() for p in ps)
    # dv = P go: the kernel rounds q times a constant to bf16 before the score product, each factor off by
    # 2^-8 at most, so the exponent is off by 2^-8 scale sum |q k| at most and P by expm1 of that (the
    # score's own fp32 rounding is in the 1e-5); then P and dv are rounded to bf16, 2^-8 each
    exponent = 2.0 ** -8 * hd ** -0.5 * (q * k).abs().sum(-1, keepdim=True) + 1e-5
    rel = (1 + torch.expm1(exponent)) * (1 + 2.0 ** -8) ** 2 - 1
    assert ((dv.double() - want).abs() <= rel * want.abs() + 1e-30).all()
    size = (go.double().norm(dim=-1) * v.norm(dim=-1))[..., None] * 2.0 ** -15 * hd ** -0.5
    assert (dq.double().abs() <= size * k.abs() * 1.2 + 1e-12).all()
    assert (dk.double().abs() <= size * q.abs() * 1.2 + 1e-12).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_fixed_order_and_views(A, K, hd):
    ps, lse, go, o = _attention(A, K, 1, 1500, 3, hd, 21)
    wide = torch.empty(1, 1500, 3, hd + 32, dtype=BF16, device="cuda")
    wide[..., 32:] = go
    was = K.DETERMINISTIC
    try:
        K.set_deterministic(True)
        a = A.attn_bwd8(*ps, lse, wide[..., 32:])
        b = A.attn_bwd8(*ps, lse, go)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    finally:
        K.set_deterministic(was)
    got = A.attn_bwd8(*ps, lse, go.transpose(1, 2).contiguous().transpose(1, 2))
    _near(got, [t.double() for t in a], "order of go")
    _near(A.attn_bwd8(*ps, lse, go, scale=0.05), _oracle(ps, lse, go, 0.05), "scale")
    low = torch.logsumexp(-0.1 * torch.einsum("blhd,bmhd->bhlm", *(p.restore().float() for p in ps[:2])), -1)
    _near(A.attn_bwd8(*ps, low, go, scale=-0.1), _oracle(ps, low, go, -0.1), "a scale below zero")
    # bf16 v and o that are not laid out for TMA: copied first
    v, o_ = ps[2].restore(), ps[3].restore()
    odd = torch.empty(1, 1500, 3, hd + 4, dtype=BF16, device="cuda")[..., 4:]
    odd.copy_(v)
    K.set_deterministic(True)
    try:
        a = A.attn_bwd8(ps[0], ps[1], v, o_, lse, go)
        b = A.attn_bwd8(ps[0], ps[1], odd, o_.transpose(1, 3).contiguous().transpose(1, 3), lse, go)
        c = A.attn_bwd8(*ps, lse, go)
    finally:
        K.set_deterministic(was)
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))
    flat = torch.full_like(lse, math.log(1500))                          # scale 0: P = 1 / L, dQ = dK = 0
    dq, dk, dv = A.attn_bwd8(*ps, flat, go, scale=0.0)
    assert (dq == 0).all() and (dk == 0).all()
    _near((dv,), _oracle(ps, flat, go, 0.0)[2:], "a scale of zero")
    none = torch.empty(0, 5, 2, hd, dtype=BF16, device="cuda")
    assert A.attn_bwd8(*A.store8([none] * 4), torch.empty(0, 2, 5, device="cuda"), none)[0].shape == none.shape
    with pytest.raises(ValueError):
        A.attn_bwd8(*ps, lse.transpose(1, 2).contiguous().transpose(1, 2), go)
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B", [1, 2])
def test_attention_of_broadcast_tensors(A, K, hd, B):
    """Output gradients that are one row for all (of a mean), V and O shared by the heads: as their copies."""
    g, (L, H) = _gen(31), (150, 3)
    q8, k8 = A.store8([_randn(g, B, L, H, hd), _randn(g, B, L, H, hd)])
    lse = torch.full((B, H, L), math.log(L) + 1.0, device="cuda")
    v, o = (_randn(g, B, L, 1, hd).expand(B, L, H, hd) for _ in range(2))
    was = K.DETERMINISTIC
    K.set_deterministic(True)
    try:
        for go in (_randn(g, B, 1, H, hd), _randn(g, 1, 1, 1, hd), _randn(g, 1, L, H, hd)):
            go = go.expand(B, L, H, hd)
            a = A.attn_bwd8(q8, k8, v, o, lse, go)
            b = A.attn_bwd8(q8, k8, v.contiguous(), o.contiguous(), lse, go.contiguous())
            assert all(torch.equal(x, y) for x, y in zip(a, b))
        with pytest.raises(ValueError):
            A.attn_bwd8(q8, k8, v, o, lse, go, gv_out=torch.empty(B, 1, H, hd, dtype=BF16, device="cuda").expand(B, L, H, hd))
    finally:
        K.set_deterministic(was)
    with pytest.raises(ValueError):
        A.gemm_wgrad8(_randn(g, 1, 64).expand(96, 64), A.store8(_randn(g, 96, 40)))
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("L", [1, 65, 128, 200, 333])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_scores_far_below_zero(A, K, hd, L, sign):
    """All scores near -100: exp(-lse) of the rows behind the last key is no number of 32 bits."""
    g, H = _gen(50 + L), 2
    q, k, v, go = (_randn(g, 1, L, H, hd) for _ in range(4))
    q[..., 0], k[..., 0] = 16.0, -100.0 * sign * hd ** 0.5 / 16      # the scores; the other channels tell them apart
    k[..., 0] = k[..., 0].float().round().to(BF16)
    scale = sign * hd ** -0.5
    q8, k8, v8 = A.store8([q, k, v])
    z = [p.restore().double() for p in (q8, k8, v8)]
    s = torch.einsum("blhd,bmhd->bhlm", z[0], z[1]) * scale
    lse = torch.logsumexp(s, -1).float()
    assert (lse < -89).all()
    o8 = A.store8(torch.einsum("bhlm,bmhd->blhd", torch.softmax(s, -1), z[2]).to(BF16))
    got = A.attn_bwd8(q8, k8, v8, o8, lse, go, scale=scale)
    want = _oracle((q8, k8, v8, o8), lse, go, scale)
    assert all(torch.isfinite(t).all() for t in got)
    # P, dS and the results are rounded to bf16 (1.6e-3 of the norm each); the exponent is off by the (hi, lo) pair of
    # lse / scale, 2^-16 of 110 at most, and 32-bit sums of scores, 2^-23 of a few 110: 2e-3
    if L > 1:             # (one token: dQ and dK are nothing but roundings; channel 0 of k is one value, its dQ too)
        _near((got[0][..., 1:], got[1], got[2]), [want[0][..., 1:], want[1], want[2]], (hd, L, sign))
    else:
        _near((got[2],) * 3, [want[2]] * 3, (hd, L, sign))
    gq, gk, gv = K.attn_bwd(q, k, v, o8.restore(), lse, go, scale=scale)
    assert torch.isfinite(gq).all() and torch.isfinite(gk).all() and torch.isfinite(gv).all()
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("L", [333, 1025, 2049])
def test_attention_rounds_twice_on_the_way(A, K, hd, L):
    """What is rounded to bf16 is P or dS and then the result, 1.66e-3 of the norm each (half a unit, evenly spread,
    over normally distributed values), together 2.35e-3.  A q multiplied by a constant and rounded too would
    make it 3.0e-3 to 3.6e-3."""
    ps, lse, go, o = _attention(A, K, 1, L, 3, hd, L)
    for a, b, name in zip(A.attn_bwd8(*ps, lse, go), _oracle(ps, lse, go), ("dq", "dk", "dv")):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel < 2.7e-3, (name, rel)
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_one_token_exponent(A, K, hd):
    """dV = P go of a single token, where P is the exponential of a difference: off by the (hi, lo) pair of bf16 that
    holds lse, 2^-16 of it, and by 32-bit sums; then P and dV are rounded to bf16, 2^-8 each."""
    ps, lse, go, o = _attention(A, K, 3, 1, 5, hd, 4, s=2.0)
    _, _, want = _oracle(ps, lse, go)
    q, k = (p.restore().double() for p in ps[:2])
    size = lse.double().abs().transpose(1, 2)[..., None]
    exponent = 2.0 ** -16 * size + 8 * 2.0 ** -23 * (size + hd ** -0.5 * (q * k).abs().sum(-1, keepdim=True))
    rel = (1 + torch.expm1(exponent)) * (1 + 2.0 ** -22) * (1 + 2.0 ** -8) ** 2 - 1
    dv = A.attn_bwd8(*ps, lse, go)[2]
    assert ((dv.double() - want).abs() <= rel * want.abs() + 1e-30).all()
    K.check_status()


@pytest.mark.parametrize("hd,L,B,H", [(64, 2100, 1, 40), (64, 2100, 3, 25), (64, 9000, 1, 9), (128, 2100, 1, 20),
                                      (128, 2100, 2, 19), (128, 5000, 1, 7)])
def test_attention_of_more_heads_than_are_worked_on_at_once(A, K, hd, L, B, H):
    """Heads go in groups (34 MB of what they read and add to), the last of them smaller, whose tiles are split;
    every head against the formula, from 8 bits and in bf16, and against the fixed order, which has one group."""
    group = 34000000 // (L * hd * 8)
    assert 1 <= group < B * H and B * H % group
    ps, lse, go, o = _attention(A, K, B, L, H, hd, L + H)
    q, k, v, o8 = (p.restore() for p in ps)
    got, got16 = A.attn_bwd8(*ps, lse, go), K.attn_bwd(q, k, v, o8, lse, go)
    was = K.DETERMINISTIC
    K.set_deterministic(True)
    try:
        fixed, fixed16 = A.attn_bwd8(*ps, lse, go), K.attn_bwd(q, k, v, o8, lse, go)
    finally:
        K.set_deterministic(was)
    K.check_status()
    cut = lambda t, b, h: t[b:b + 1, :, h:h + 1]
    for b in range(B):
        for h in range(H):
            one = [cut(t, b, h).double().transpose(1, 2) for t in (q, k, v, o8, go)]
            s = one[0] @ one[1].transpose(-1, -2) * hd ** -0.5
            P = torch.exp(s - lse[b:b + 1, h:h + 1, :, None].double())
            dS = P * (one[4] @ one[2].transpose(-1, -2) - (one[4] * one[3]).sum(-1, keepdim=True))
            want = [(dS @ one[1] * hd ** -0.5), (dS.transpose(-1, -2) @ one[0] * hd ** -0.5), P.transpose(-1, -2) @ one[4]]
            want = [t.transpose(1, 2) for t in want]
            for res in (got, got16, fixed, fixed16):
                _near([cut(t, b, h) for t in res], want, (b, h))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [500, 2000])
def test_attention_of_large_scores(A, K, hd, size):
    """Scores near 500 and 2,000, and delta of that size: P and dS are exponentials and products of differences of numbers
    that large, which 16 bits (a pair of bf16) would get wrong by 2^-17 of them: 0.8 and 3 % of P."""
    B, L, H = 1, 300, 2
    g = _gen(70)
    q, k, v, go = (_randn(g, B, L, H, hd) for _ in range(4))
    q[..., 0], k[..., 0] = 16.0, round(size * hd ** 0.5 / 16 / 4) * 4.0
    v[..., 0], go[..., 0] = 64.0, size / 64
    q8, k8, v8 = A.store8([q, k, v])
    z = [p.restore().double() for p in (q8, k8, v8)]
    s = torch.einsum("blhd,bmhd->bhlm", z[0], z[1]) * hd ** -0.5
    lse = torch.logsumexp(s, -1).float()
    o8 = A.store8(torch.einsum("bhlm,bmhd->blhd", torch.softmax(s, -1), z[2]).to(BF16))
    assert lse.min() > 0.9 * size and (o8.restore()[..., 0] == 64).all()
    got = A.attn_bwd8(q8, k8, v8, o8, lse, go)
    want = _oracle((q8, k8, v8, o8), lse, go)
    # two roundings to bf16 (2.35e-3, see test_attention_rounds_twice_on_the_way); lse in 32 bits, 2^-25 of it on the
    # average, is the oracle's too; what the tensor core drops of sums of `size`, 2^-25 of the sum in each of 5 (9)
    # steps and its conversion by scale, less than 2^-21 size = 1e-3 at 2,000.  (Channel 0 of k is one value: its
    # dQ is a sum that cancels.)
    for a, b, name in zip((got[0][..., 1:], got[1], got[2]), (want[0][..., 1:], want[1], want[2]), ("dq", "dk", "dv")):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel < 4e-3, (name, rel)
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_scores_beyond_the_exponents_of_32_bits(A, K, hd, sign):
    """Scores near +-25,000, where lse is beyond 2^15 in powers of two."""
    B, L, H = 1, 200, 2
    g = _gen(71)
    q, k, v, go = (_randn(g, B, L, H, hd) for _ in range(4))
    q[..., 0], k[..., 0] = 512.0, sign * round(25000 * hd ** 0.5 / 512 / 4) * 4.0
    q8, k8, v8 = A.store8([q, k, v])
    z = [p.restore().double() for p in (q8, k8, v8)]
    s = torch.einsum("blhd,bmhd->bhlm", z[0], z[1]) * hd ** -0.5
    lse = torch.logsumexp(s, -1).float()
    assert (lse.abs() > 22000).all()
    o8 = A.store8(torch.einsum("bhlm,bmhd->blhd", torch.softmax(s, -1), z[2]).to(BF16))
    got = A.attn_bwd8(q8, k8, v8, o8, lse, go)
    want = _oracle((q8, k8, v8, o8), lse, go)
    # two roundings to bf16, 2.4e-3; lse log2 e and the scale are each rounded, 2^-24 of 36,000 = 2.2e-3; sums of 2^18 in the
    # tensor core drop up to 2^-7 a step (with a bit or two below 32 bits' last), 5 or 9 steps over a scale of 1 / 8 or
    # 1 / 11: 6e-3; all together 1.3e-2, mostly of one sign
    for a, b, name in zip((got[0][..., 1:], got[1], got[2]), (want[0][..., 1:], want[1], want[2]), ("dq", "dk", "dv")):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel < 1.3e-2, (name, rel)
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_strides_of_single_dimensions(A, K, hd):
    """The stride of a dimension of one element is anything: no address depends on it."""
    for shape, strides in (((1, 65, 2, hd), (1, 2 * hd, hd, 1)), ((1, 65, 1, hd), (3, hd, 5, 1)),
                           ((2, 1, 3, hd), (3 * hd, 7, hd, 1)), ((1, 1, 1, hd), (1, 1, 1, 1))):
        B, L, H, _ = shape
        ps, lse, go, _ = _attention(A, K, B, L, H, hd, 60)
        buf = torch.full((B * L * H * hd + 64,), 3.0, dtype=BF16, device="cuda")
        got = A.attn_bwd8(*ps, lse, go, gv_out=buf.as_strided(shape, strides))[2]
        assert torch.equal(got, A.attn_bwd8(*ps, lse, go)[2])
        assert torch.equal(buf[:-64].view(shape), got) and (buf[-64:] == 3).all()
        with pytest.raises(ValueError):
            A.attn_bwd8(*ps, lse, go, gv_out=buf[1:].as_strided(shape, strides, 1))
    with pytest.raises(ValueError):
        A.attn_bwd8(*ps, lse, go, gv_out=buf.new_empty(2 * hd)[::2].view(shape))
    K.check_status()


@pytest.mark.parametrize("hd,L", [(64, 67001), (128, 34001)])
def test_attention_of_one_head_at_a_time(A, K, hd, L):
    """Sequences so long that a single head is more than a group: as in the fixed order, which has one group.  The two
    differ in the order of 32-bit sums, which moves a result across a rounding to bf16 (2^-8) now and then."""
    assert 34000000 // (L * hd * 8) == 0
    ps, lse, go, o = _attention(A, K, 1, L, 2, hd, 8)
    got = A.attn_bwd8(*ps, lse, go)
    was = K.DETERMINISTIC
    K.set_deterministic(True)
    try:
        fixed = A.attn_bwd8(*ps, lse, go)
    finally:
        K.set_deterministic(was)
    K.check_status()
    for h in range(2):
        for a, b in zip(got, fixed):
            a, b = a[:, :, h].double(), b[:, :, h].double()
            assert (a - b).norm() <= 1e-3 * b.norm() and (a - b).abs().max() <= 2.0 ** -7 * b.abs().max()
    # rows of dQ in the first, a middle and the last tile, and the same of dK and dV, against the formula
    q, k, v, o8 = (p.restore() for p in ps)
    rows = torch.tensor([0, 1, 127, L // 2, L - 2, L - 1], device="cuda")
    for h in range(2):
        Q, Kk, V, O, G = (t[0, :, h].double() for t in (q, k, v, o8, go))
        stat, delta = lse[0, h].double(), (G * O).sum(1)
        P = torch.exp(Q[rows] @ Kk.t() * hd ** -0.5 - stat[rows, None])
        dq = (P * (G[rows] @ V.t() - delta[rows, None])) @ Kk * hd ** -0.5
        P = torch.exp(Kk[rows] @ Q.t() * hd ** -0.5 - stat)
        want = (dq, (P * (V[rows] @ G.t() - delta)) @ Q * hd ** -0.5, P @ G)
        _near([t[0, rows, h] for t in got], want, h)


def test_attention_gradient_is_a_difference_quotient(A, K):
    """Along a random direction of q, k and v the loss changes as the gradients say (64-bit differences)."""
    B, L, H, hd = 1, 40, 2, 64
    g = _gen(30)
    q, k, v, go = (_randn(g, B, L, H, hd, s=0.5) for _ in range(4))
    ps = A.store8([q, k, v])
    z = [p.restore().double() for p in ps]

    def fwd(q, k, v):
        s = torch.einsum("blhd,bmhd->bhlm", q, k) / math.sqrt(hd)
        return torch.einsum("bhlm,bmhd->blhd", torch.softmax(s, -1), v), torch.logsumexp(s, -1)

    o, lse = fwd(*z)
    grads = A.attn_bwd8(*ps, o.bfloat16(), lse.float(), go)
    for i in range(3):
        d = torch.randn(z[i].shape, device="cuda", generator=g, dtype=torch.float64)
        up, down = list(z), list(z)
        up[i], down[i] = z[i] + 1e-4 * d, z[i] - 1e-4 * d
        want = ((fwd(*up)[0] - fwd(*down)[0]) * go.double()).sum() / 2e-4
        got = (grads[i].double() * d).sum()
        # 2-norm of the roundings of one gradient (see _near) against a unit direction
        assert (got - want).abs() <= 1e-2 * grads[i].double().norm() * 3


# ------------------------------------------------------------- streams, graphs, together ---
def _linear_step(A, x, gu, dy, gout):
    """What a block does: keep, then gradients from what was kept."""
    x8, gu8 = A.store8([x, gu])
    grad, act = A.situ_bwd8(gu8, gout, 4.0, 25.0)
    return A.gemm_wgrad8(dy, x8), grad, act, A.restore8(x8)


def test_another_stream_and_two_graphs(A, K):
    g = _gen(40)
    mk = lambda: (_randn(g, 600, 256), _randn(g, 600, 2 * 344), _randn(g, 600, 528), _randn(g, 600, 344))
    a, b = mk(), mk()
    want = [_linear_step(A, *t) for t in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _linear_step(A, *a)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want[0]))
    graphs, outs = [], []
    for t in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_linear_step(A, *t))
        graphs.append(graph)
    for t, s in zip(a + b, mk() + mk()):
        t.copy_(s)
    want = [_linear_step(A, *t) for t in (a, b)]
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(got, w))
    K.check_status()


def test_threads_at_once(A, K):
    """Two host threads, a stream each: every call has its own workspace."""
    import threading

    g = _gen(42)
    mk = lambda: (_randn(g, 3000, 256), _randn(g, 3000, 2 * 344), _randn(g, 3000, 528), _randn(g, 3000, 344))
    data = [mk(), mk()]
    want = [_linear_step(A, *t) for t in data]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = _linear_step(A, *data[i])
                torch.cuda.current_stream().synchronize()
        except Exception as exc:      # noqa: BLE001
            errors.append(exc)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in range(2):
        assert all(torch.equal(x, y) for x, y in zip(got[i], want[i]))
    K.check_status()


def test_attention_in_a_graph(A, K):
    g = _gen(41)
    q, k, v, go = (_randn(g, 1, 700, 2, 64) for _ in range(4))

    def step():
        o, _, lse = K.attn_fwd(q, k, v)
        return A.attn_bwd8(*A.store8([q, k, v, o]), lse, go)

    was = K.DETERMINISTIC
    try:
        K.set_deterministic(True)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for t in (q, k, v, go):
            t.copy_(_randn(g, *t.shape))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    finally:
        K.set_deterministic(was)
    K.check_status()
