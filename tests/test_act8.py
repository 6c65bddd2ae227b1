"""CPU: activations in 8 bits -- the format against its definition, the formulas against autograd in
64 bits, and every refusal."""
import math

import pytest
import torch

from imfvideo_b200.ops import act8
from imfvideo_b200.ops import reference as ref

BF16, F32 = torch.bfloat16, torch.float32
BF16_MAX = torch.finfo(BF16).max


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def definition(x):
    """(codes, steps) from the words of the format, a group at a time, in Python numbers."""
    rows, C = x.shape
    G = -(-C // 32)
    codes, steps = torch.zeros(rows, G * 32, dtype=torch.int8), torch.zeros(rows, (G + 3) // 4 * 4, dtype=torch.uint8)
    for r in range(rows):
        for g in range(G):
            v = x[r, 32 * g:32 * g + 32].double().tolist()
            if not all(math.isfinite(e) for e in v):
                steps[r, g] = 255
                continue
            amax = max(abs(e) for e in v)
            s = 0
            while s < 248 and amax / 2.0 ** (s - 127) >= 127.5:
                s += 1
            steps[r, g] = s
            for i, e in enumerate(v):
                codes[r, 32 * g + i] = max(-127, min(127, round(e / 2.0 ** (s - 127))))
    return codes, steps


def edge_rows(C=70):
    """Rows where the format can go wrong: zeros, the carry at 127.5 steps, ties, the type's largest and
    smallest values, infinities and NaN."""
    g = _gen(0)
    x = torch.randn(12, C, generator=g)
    x[0] = 0.0
    x[1, :32] = torch.arange(32) * 0.5                       # ties: 0.5 of a step and so on
    x[1, 31] = 64.0
    x[2, 0], x[2, 1] = 127.5, 127.25                         # 127.5 steps carry, 127.25 would not
    x[3, :32] = 0.1
    x[3, 5] = -127.25
    x[4] = BF16_MAX
    x[4, 1] = -BF16_MAX
    x[5] *= 1e-38                                            # subnormal steps
    x[6] = 1e-41
    x[7, 3] = float("inf")
    x[8, 40] = float("nan")
    x[9, 69] = float("-inf")
    x[10] = x[10].bfloat16().float() * 2.0 ** 100
    return x


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_format_is_its_definition(dtype):
    x = edge_rows().to(dtype)
    p = act8.store8(x)
    codes, steps = definition(x.float())
    assert torch.equal(p.steps, steps) and torch.equal(p.codes, codes)
    assert p.shape == x.shape and p.dtype == dtype and p.nbytes == 12 * (96 + 4)


def test_values_are_exact_in_bf16_and_half_a_step_off():
    x = torch.randn(64, 200, generator=_gen(1)) * torch.exp(3 * torch.randn(64, 200, generator=_gen(2)))
    p = act8.store8(x)
    v = act8.restore8(p)
    assert v.dtype == F32 and torch.equal(v.bfloat16().float(), v)
    step = 2.0 ** (p.steps[:, :7].double() - 127)
    err = torch.nn.functional.pad((v.double() - x.double()).abs(), (0, 24)).view(64, 7, 32)
    assert (err <= step[..., None] / 2).all()
    amax = torch.nn.functional.pad(x.abs(), (0, 24)).view(64, 7, 32).amax(-1).double()
    assert (step <= amax / 63.75).all() and (step * 127.5 > amax).all()


def test_bad_groups_read_as_nan_and_no_others():
    x = edge_rows()
    v = act8.restore8(act8.store8(x))
    bad = torch.zeros(12, 96, dtype=torch.bool)
    bad[7, :32] = bad[8, 32:64] = bad[9, 64:] = True
    assert torch.equal(torch.isnan(v), bad[:, :70]) and torch.isfinite(v[4]).all()


def test_several_tensors_shapes_and_outputs():
    g = _gen(3)
    wide = torch.randn(2, 5, 3, 80, generator=g).bfloat16()
    xs = [torch.randn(7, 33, generator=g), wide[..., 16:], torch.randn(40, generator=g).bfloat16(),
          wide.transpose(1, 2)[:, :, ::2], torch.empty(0, 8), torch.randn(4, 0)]
    ps = act8.store8(xs)
    for x, p, v in zip(xs, ps, act8.restore8(ps)):
        assert p.shape == x.shape and v.shape == x.shape and v.dtype == x.dtype
        assert torch.equal(v, act8.store8(x.contiguous()).restore())
    band = torch.full((2, 5, 3, 70), 7.0, dtype=BF16)
    out = act8.restore8(ps[1], band[..., 6:])
    assert out.data_ptr() == band[..., 6:].data_ptr() and (band[..., :6] == 7).all()
    assert torch.equal(out, ps[1].restore())
    assert ps[0].view(7, 1, 33).restore().shape == (7, 1, 33)
    assert act8.store8([]) == [] and act8.restore8([]) == []


def test_weight_gradient_formula():
    g = _gen(4)
    x, dy = torch.randn(50, 45, generator=g).bfloat16(), torch.randn(50, 24, generator=g).bfloat16()
    p = act8.store8(x)
    want = dy.double().t() @ p.restore().double()
    got = act8.gemm_wgrad8(dy, p)
    # 50 products and sums in 32 bits
    assert got.dtype == F32 and (got - want).abs().max() <= 50 * 2.0 ** -24 * (dy.double().abs().t() @ x.double().abs()).max()
    base = torch.randn(24, 45, generator=g)
    acc = base.clone()
    assert act8.gemm_wgrad8(dy, p, out=acc, accumulate=True) is acc
    assert torch.allclose(acc, base + got, atol=1e-5)
    assert torch.equal(act8.gemm_wgrad8(dy[:0], act8.store8(x[:0])), torch.zeros(24, 45))


@pytest.mark.parametrize("lbeta", [25.0, None])
def test_gated_activation_formula(lbeta):
    g = _gen(5)
    gu, gout = (torch.randn(9, 2 * 21, generator=g) * 3).bfloat16(), torch.randn(9, 21, generator=g).bfloat16()
    p = act8.store8(gu)
    grad, y = act8.situ_bwd8(p, gout, 4.0, lbeta)
    z = p.restore().double().requires_grad_()
    up = z[:, 21:] if lbeta is None else lbeta * torch.tanh(z[:, 21:] / lbeta)
    want_y = 4.0 * torch.tanh(z[:, :21] / 4.0) * torch.sigmoid(z[:, :21]) * up
    want, = torch.autograd.grad(want_y, z, gout.double())
    # one rounding to bf16, some 32-bit operations (1 - th^2 loses up to 2^-22 absolute before the product)
    near = lambda a, b: (a.double() - b).abs() <= 2.0 ** -8 * b.abs() + 2.0 ** -18
    assert near(y, want_y.detach()).all() and near(grad, want).all()


@pytest.mark.parametrize("B,L,H", [(1, 1, 1), (2, 7, 3)])
def test_attention_formula(B, L, H):
    g = _gen(6)
    q, k, v, go = (torch.randn(B, L, H, 64, generator=g).bfloat16() for _ in range(4))
    q8, k8, v8 = act8.store8([q, k, v])
    z = [p.restore().double().requires_grad_() for p in (q8, k8, v8)]
    s = torch.einsum("blhd,bmhd->bhlm", z[0], z[1]) / 8
    o = torch.einsum("bhlm,bmhd->blhd", torch.softmax(s, -1), z[2])
    want = torch.autograd.grad(o, z, go.double())
    # with the exact output the recomputed form is the gradient itself
    got = ref.attention_grad(*(t.detach() for t in z), o.detach(), torch.logsumexp(s, -1).detach().float(), go)
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= 2.0 ** -14
    lse = torch.logsumexp(s, -1).float().detach()
    got = act8.attn_bwd8(q8, k8, v8, o.detach().bfloat16(), lse, go, gv_out=torch.empty(B, L, H, 64, dtype=BF16))
    assert (got[2].double() - want[2]).abs().max() <= 2.0 ** -8 * want[2].abs().max() + 2.0 ** -14


def test_refusals():
    x = torch.randn(4, 64).bfloat16()
    p = act8.store8(x)
    no = lambda: pytest.raises(ValueError)
    for bad in (x.half(), x.double(), x.int(), torch.tensor(1.0)):
        with no():
            act8.store8(bad)
    for codes, steps, shape in ((p.codes[:, :32], p.steps, (4, 64)), (p.codes.int(), p.steps, (4, 64)),
                                (p.codes, p.steps[:, :2], (4, 64)), (p.codes, p.steps.int(), (4, 64)),
                                (p.codes, p.steps, (5, 64)), (p.codes.t().contiguous().t(), p.steps, (4, 64)),
                                (p.codes, p.steps, (4, 65)), (p.codes, p.steps, ())):
        with no():
            act8.Packed8(codes, steps, shape)
    with no():
        act8.Packed8(p.codes, p.steps, (4, 64), torch.float16)
    with no():
        p.view(4, 32)
    with no():
        act8.restore8(p, torch.empty(4, 64))                 # type
    with no():
        act8.restore8(p, torch.empty(4, 65, dtype=BF16))
    with no():
        act8.restore8([p], [None, None])
    dy = torch.randn(4, 8).bfloat16()
    for a, b, out in ((dy.float(), p, None), (dy[:3], p, None), (dy, act8.store8(x.float()), None), (dy, x, None),
                      (dy, p, torch.zeros(8, 63)), (dy, p, torch.zeros(8, 64, dtype=BF16)),
                      (dy, p, torch.zeros(64, 8).t())):
        with no():
            act8.gemm_wgrad8(a, b, out)
    gout = torch.randn(4, 32).bfloat16()
    for a, b, beta, lb in ((p, gout.float(), 4.0, 25.0), (p, gout[:, :31], 4.0, 25.0), (p, gout, 0.0, 25.0),
                           (p, gout, 4.0, 0.0), (act8.store8(x[:, :63]), gout, 4.0, 25.0), (x, gout, 4.0, 25.0),
                           (p, gout, float("nan"), 25.0)):
        with no():
            act8.situ_bwd8(a, b, beta, lb)
    q = act8.store8(torch.randn(1, 4, 2, 64).bfloat16())
    go, lse = torch.randn(1, 4, 2, 64).bfloat16(), torch.zeros(1, 2, 4)
    for args in ((q, q, q, go, lse, go.float()), (q, q, q, go, lse[:, :1], go), (q, q, q, go, lse.double(), go),
                 (q, q, q.view(1, 2, 4, 64), go, lse, go), (p.view(1, 4, 1, 64), q, q, go, lse, go),
                 (q.view(4, 2, 64), q, q, go, lse, go), (go, q, q, go, lse, go), (q, q, q, go[:, :3], lse, go),
                 (q, q, q, go, lse, go, None, go[..., :32])):
        with no():
            act8.attn_bwd8(*args)
    small = act8.store8(torch.randn(1, 4, 2, 32).bfloat16())
    with no():
        act8.attn_bwd8(small, small, small, go[..., :32], lse, go[..., :32])


def test_outputs_that_share_memory():
    """Elements of one output, or of two, in one place are refused; bands and rows that interleave are not."""
    a, b = act8.store8([torch.randn(6, 40).bfloat16(), torch.randn(6, 24).bfloat16()])
    f = act8.store8(torch.randn(6, 20))
    c = act8.store8(torch.randn(3, 2, 8).bfloat16())
    flat = lambda n=2000, dt=BF16: torch.full((n,), 7.0, dtype=dt)
    buf = flat()
    row = lambda p, o, s: buf.as_strided(p.shape, (s, 1), o)
    for ps, outs in (([a], [row(a, 0, 39)]), ([a], [row(a, 0, 1)]), ([a], [row(a, 0, 0)]),
                     ([a], [buf[:40].expand(6, 40)]), ([c], [buf.as_strided((3, 2, 8), (16, 12, 1))]),
                     ([c], [buf.as_strided((3, 2, 8), (8, 16, 1))]),
                     ([a, a], [row(a, 0, 40), row(a, 0, 40)]), ([a, b], [row(a, 0, 64), row(b, 39, 64)]),
                     ([a, b], [row(a, 24, 63), row(b, 0, 63)]), ([b, a], [row(b, 0, 24), row(a, 143, 40)]),
                     ([a, b], [row(a, 0, 80), row(b, 60, 81)])):
        with pytest.raises(ValueError):
            act8.restore8(ps, outs)
    assert (buf == 7).all()
    for ps, outs in (([a, b], [row(a, 0, 64), row(b, 40, 64)]), ([a, b], [row(a, 24, 64), row(b, 0, 64)]),
                     ([a, b], [row(a, 0, 40), row(b, 240, 24)]), ([c], [buf.as_strided((3, 2, 8), (16, 24, 1))]),
                     ([c], [buf.as_strided((3, 2, 8), (8, 24, 1))]), ([a, b], [row(a, 0, 80), row(b, 40, 160)][:2]),
                     ([a], [row(a, 5, 40)]), ([b, a, b], [None, row(a, 0, 64), row(b, 40, 64)])):
        buf.fill_(7.0)
        for p, o in zip(ps, act8.restore8(ps, outs)):
            assert torch.equal(o, p.restore())
    out = flat(6 * 20, F32).view(6, 20)
    assert torch.equal(act8.restore8([f, a], [out, None])[0], f.restore())


@pytest.mark.parametrize("seed", range(40))
def test_sharing_of_memory_is_found(seed):
    """Two or three random outputs of a small buffer: refused exactly where two of their elements have one place."""
    import random

    rng = random.Random(seed)
    refused = taken = 0
    for _ in range(30):
        buf, ps, outs, places = torch.zeros(400, dtype=BF16), [], [], []
        for _ in range(rng.choice([1, 2, 3])):
            shape = [rng.choice([1, 1, 2, 3]) for _ in range(rng.choice([1, 2]))] + [rng.choice([1, 2, 5, 8])]
            strides = [rng.choice([0, 1, 3, 8, 8, 16, 16, 24, 40]) for _ in shape[:-1]] + [1]
            out = buf.as_strided(shape, strides, rng.choice([0, 5, 8, 16, 100, 200, 200 + rng.randrange(60)]))
            ps.append(act8.store8(torch.randn(shape).bfloat16()))
            outs.append(out)
            places += torch.arange(400).as_strided(shape, strides, out.storage_offset()).flatten().tolist()
        if len(set(places)) == len(places):
            for p, o in zip(ps, act8.restore8(ps, outs)):
                assert torch.equal(o, p.restore())
            taken += 1
        else:
            with pytest.raises(ValueError):
                act8.restore8(ps, outs)
            refused += 1
    assert refused and taken


def test_attention_outputs_that_share_memory():
    q = act8.store8(torch.randn(2, 4, 2, 64).bfloat16())
    go, lse = torch.randn(2, 4, 2, 64).bfloat16(), torch.zeros(2, 2, 4)
    buf = torch.zeros(4096, dtype=BF16)
    for strides in ((512, 128, 32, 1), (512, 128, 0, 1), (0, 128, 64, 1), (512, 64, 64, 1), (448, 128, 64, 1)):
        with pytest.raises(ValueError):
            act8.attn_bwd8(q, q, q, go, lse, go, gv_out=buf.as_strided((2, 4, 2, 64), strides))
    want = act8.attn_bwd8(q, q, q, go, lse, go)[2]
    for strides in ((512, 128, 64, 1), (128, 256, 64, 1), (64, 128, 512, 1)):
        got = act8.attn_bwd8(q, q, q, go, lse, go, gv_out=buf.as_strided((2, 4, 2, 64), strides))[2]
        assert torch.equal(got, want)


def test_views_of_packed_tensors():
    p = act8.store8(torch.randn(4, 64).bfloat16())
    for shape in ((-2, -2, 64), (-1, 64), (64,), (), (4, -64)):
        with pytest.raises(ValueError):
            p.view(*shape)
    v = p.view(2, 1, 2, 64)
    assert v.shape == (2, 1, 2, 64) and torch.equal(v.restore().view(4, 64), p.restore())


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39, 3e38])
def test_scales_that_are_no_number_of_32_bits(scale):
    q = act8.store8(torch.randn(1, 4, 2, 64).bfloat16())
    go, lse = torch.randn(1, 4, 2, 64).bfloat16(), torch.zeros(1, 2, 4)
    with pytest.raises(ValueError):
        act8.attn_bwd8(q, q, q, go, lse, go, scale)


@pytest.mark.parametrize("bad", [math.inf, math.nan, 1e39, 1e-39, 1e-60, 0.0, -4.0])
def test_betas_that_are_no_positive_number_of_32_bits(bad):
    """(their reciprocals, or products with a tanh of zero, would be NaN where the formula has a value)"""
    gu, gout = act8.store8(torch.zeros(2, 16).bfloat16()), torch.ones(2, 8).bfloat16()
    for beta, lbeta in ((bad, 25.0), (4.0, bad), (bad, None)):
        with pytest.raises(ValueError):
            act8.situ_bwd8(gu, gout, beta, lbeta)
    for t in act8.situ_bwd8(gu, gout, 2.0 ** -126, 3.4e38):
        assert torch.isfinite(t).all()


def test_option_of_the_model():
    from imfvideo_b200.config import apply_overrides, preset
    from imfvideo_b200.models import IMFDiTVideo
    from imfvideo_b200.train import build_model

    cfg = apply_overrides(preset("tiny"), {"model.act_store": "int8"})
    net = build_model(cfg)[0]
    assert all(b.act_store == "int8" for b in net.shared_blocks) and preset("tiny").model.act_store == "bf16"
    with pytest.raises(ValueError):
        IMFDiTVideo(input_size=8, num_frames=1, hidden_size=64, depth=2, num_heads=2, aux_head_depth=1,
                    act_store="int4")


def test_option_with_block_recomputation_warns():
    import warnings

    from imfvideo_b200.config import apply_overrides, preset
    from imfvideo_b200.train import build_model

    def build(**model):
        return build_model(apply_overrides(preset("tiny"), {"model." + k: v for k, v in model.items()}))

    with pytest.warns(UserWarning, match="saves no memory"):
        build(act_store="int8", grad_checkpoint=True)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        build(act_store="int8", grad_checkpoint=False)
        build(act_store="bf16", grad_checkpoint=True)
