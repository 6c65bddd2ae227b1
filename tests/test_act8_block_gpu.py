"""GPU: transformer blocks that keep their activations in 8 bits (``act_store="int8"``)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def kernels():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from imfvideo_b200.ops import cuda as cu

    assert cu.available()
    from imfvideo_b200.ops import kernels as K

    return K


GRID, PREFIX = (3, 5, 9), 20


def _block(act_store, gate=True, wide=False):
    from imfvideo_b200.models import flash_jvp_attention
    from imfvideo_b200.models.imf_dit_video import TransformerBlock

    torch.manual_seed(0)
    d, H = (384, 3) if wide else (256, 4)
    hd = d // H
    rope = hd // 4
    blk = TransformerBlock(d, H, d // 2, 128, hd - rope, rope, hd, weight_init_constant=0.5, norm_eps=1e-5,
                           attn_impl=flash_jvp_attention, use_attn_res=True, situ_beta=4.0, situ_linear_beta=25.0,
                           mla_use_output_gate=gate, act_store=act_store).cuda()
    with torch.no_grad():
        for p in blk.parameters():
            p.add_(torch.randn_like(p) * 0.05)
        blk.attn_scale.add_(0.5)
        blk.mlp_scale.add_(0.5)
    return blk


def _inputs(blk, B=2, tangent=True):
    from imfvideo_b200.models.imf_dit_video import precompute_axial_rope_3d
    from imfvideo_b200.ops.dual import Dual

    a = blk.attn
    d, rope = a.hidden_size, a.qk_rope_head_dim
    g = torch.Generator(device="cuda").manual_seed(5)
    cos, sin = precompute_axial_rope_3d(rope, GRID, PREFIX)
    L = cos.shape[0]
    mk = lambda: torch.randn(B, L, d, device="cuda", generator=g)
    prim = [mk().requires_grad_() for _ in range(2)]
    tang = [mk() if tangent else None for _ in range(2)]
    return [Dual(p, t) for p, t in zip(prim, tang)], cos.cuda(), sin.cuda(), mk()


def _run(blk, xs, cos, sin, go, fresh):
    out = blk.fused_forward(xs[0], xs[1:], fresh, True, cos, sin, 1e-5)
    out.p.backward(go)
    grads = [x.p.grad for x in xs] + [p.grad for p in blk.parameters()]
    for x in xs:
        x.p.grad = None
    for p in blk.parameters():
        p.grad = None
    return out, grads


class _Core:
    """The dense core whose backward pass reads q, k and o in 8 bits."""

    def __init__(self):
        from imfvideo_b200.ops.block import DENSE_CORE

        self.fwd = DENSE_CORE.fwd

    def bwd(self, q, k, v, o, saved, go, gv_out=None):
        from imfvideo_b200.ops import act8

        return act8.attn_bwd8(act8.store8(q), act8.store8(k), v, o, saved[0], go, gv_out=gv_out)


class _RoundTrip:
    """Makes a block that keeps bf16 activations see, in its backward pass, what the 8-bit one would: the
    last fifteen tensors it saves are its activations, each goes through store8 / restore8, and the
    gate's product and the activation are made again from those."""

    NAMES = ("n1", "a", "qlat", "kvlat", "qb", "kvb", "q", "k", "o", "og", "a_out", "n2", "gu", "act", "m")

    def __init__(self, blk):
        self.blk, self.saved = blk, []

    def pack(self, t):
        self.saved.append(t)
        return len(self.saved) - 1

    def unpack(self, i):
        from imfvideo_b200.ops import act8, rowops as R

        first = len(self.saved) - len(self.NAMES)
        if i < first:
            return self.saved[i]
        get = lambda name: act8.store8(self.saved[first + self.NAMES.index(name)]).restore()
        name, g = self.NAMES[i - first], self.blk.fused_geom()
        if name == "og":
            o = get("o").view(-1, g.H * g.dv)
            if not g.gate:
                return o
            a, out = get("a"), torch.empty_like(o)
            R.outgate_fwd(o, None, a[:, g.dq + g.dc + g.dr:], None, out, None, o.shape[0], o.shape[1], o.shape[1], g.na)
            return out
        if name == "act":
            gu = get("gu")
            out = torch.empty(gu.shape[0], g.fp, dtype=BF16, device="cuda")
            R.situ_fwd(gu, None, out, None, gu.shape[0], g.fp, 4.0, 25.0)
            return out
        return get(name)


@pytest.mark.parametrize("gate,wide,fresh,tangent", [(True, False, False, True), (False, False, True, True),
                                                     (True, True, True, False)])
def test_block_from_8_bit_activations(kernels, monkeypatch, gate, wide, fresh, tangent):
    """Forward: the same bits as with bf16 activations.  Gradients: those that the bf16 backward pass gives
    for the stored values -- data gradients bit for bit (the same kernels on the same numbers),
    weight gradients but for the order of their fp32 sums (2e-5 of the norm) and one rounding to bf16."""
    kernels.set_deterministic(True)
    try:
        blk8, blk = _block("int8", gate, wide), _block("bf16", gate, wide)
        xs, cos, sin, go = _inputs(blk, tangent=tangent)
        out8, got = _run(blk8, xs, cos, sin, go, fresh)
        _, plain = _run(blk, xs, cos, sin, go, fresh)
        rt = _RoundTrip(blk)
        monkeypatch.setattr("imfvideo_b200.ops.block.DENSE_CORE", _Core())
        with torch.autograd.graph.saved_tensors_hooks(rt.pack, rt.unpack):
            out, want = _run(blk, xs, cos, sin, go, fresh)
    finally:
        kernels.set_deterministic(False)
    kernels.check_status()
    assert torch.equal(out8.p, out.p) and (not tangent or torch.equal(out8.t, out.t))
    names = ["prefix", "snap"] + [n for n, _ in blk.named_parameters()]
    for n, a, b, c in zip(names, got, want, plain):
        if b is None:
            assert a is None
            continue
        a, b, c = a.double(), b.double(), c.double()
        if n in ("prefix", "snap") or b.dim() == 1 or "res_proj" in n:
            assert torch.equal(a, b), n
        else:
            assert (a - b).norm() <= (2e-5 + 2.0 ** -8) * b.norm(), n
        # and near the gradients without 8 bits: a code is half a step of amax / 63.75 off at most, with amax up to
        # 4.5 of the group's rms values 2 % rms; five such factors meet in a gradient at most
        assert (a - c).norm() <= 0.1 * c.norm(), n


@pytest.mark.parametrize("own", ["bwd", "both"])
def test_cores_derived_from_the_dense_one(kernels, monkeypatch, own):
    """A core that overrides the dense one's methods runs its own backward pass, from q, k and o as they are."""
    from imfvideo_b200.ops.block import DenseCore

    calls = []

    class Core(DenseCore):
        scale = 0.2 if own == "both" else None

        def fwd(self, q, k, v, dq, dk, dv, need_bwd):
            o, do, lse = kernels.attn_fwd(q, k, v, dq, dk, dv, scale=self.scale, need_lse=need_bwd)
            return o, do, (lse,)

        def bwd(self, q, k, v, o, saved, go, gv_out=None):
            calls.append((q, k, o))
            dq, dk, dv = kernels.attn_bwd(q, k, v, o, saved[0], go, scale=self.scale, gv_out=gv_out)
            return dq * 0.5, dk, dv

    kernels.set_deterministic(True)
    monkeypatch.setattr("imfvideo_b200.ops.block.DENSE_CORE", Core())
    try:
        grads = []
        for store in ("int8", "bf16"):
            blk = _block(store)
            xs, cos, sin, go = _inputs(blk)
            grads.append(_run(blk, xs, cos, sin, go, False)[1])
    finally:
        kernels.set_deterministic(False)
    kernels.check_status()
    assert len(calls) == 2 and all(torch.equal(a, b) for a, b in zip(*calls))
    for a, b in zip(*grads):
        # (see test_block_from_8_bit_activations)
        assert (a is None) == (b is None) and (a is None or (a - b).norm() <= 0.1 * b.norm())


def test_straight_into_gradient_buffers(kernels):
    """Weight gradients accumulated into existing fp32 buffers equal those returned to autograd."""
    kernels.set_deterministic(True)
    try:
        blk = _block("int8")
        xs, cos, sin, go = _inputs(blk)
        _, want = _run(blk, xs, cos, sin, go, False)
        for p in blk.parameters():
            p.grad = torch.ones_like(p)
        assert blk.fused_sinks().direct()
        out = blk.fused_forward(xs[0], xs[1:], False, True, cos, sin, 1e-5)
        out.p.backward(go)
    finally:
        kernels.set_deterministic(False)
    for (n, p), w in zip(blk.named_parameters(), want[2:]):
        if w is not None:
            a, b = p.grad.double() - 1, w.double()
            # one rounding to bf16 in the returned form, 2^-23 of the buffer's 1 in the other
            assert (a - b).norm() <= 2.0 ** -8 * b.norm() + 2.0 ** -22 * b.numel() ** 0.5, n
    kernels.check_status()


def test_what_a_block_keeps(kernels):
    """Bytes that live between forward and backward: at most 0.45 of the bf16 block's (33/32 bytes a
    channel for thirteen tensors against two for fifteen, and the fp32 input in both)."""
    kept = {}
    for mode in ("bf16", "int8"):
        blk = _block(mode)
        xs, cos, sin, go = _inputs(blk, B=8, tangent=False)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = blk.fused_forward(xs[0], xs[1:], False, True, cos, sin, 1e-5)
        torch.cuda.synchronize()
        kept[mode] = torch.cuda.memory_allocated() - before - out.p.numel() * 4
        weights = sum(p.numel() for p in blk.parameters()) * 2      # bf16 copies of the matrices
        kept[mode] -= weights
        out.p.backward(go)
    assert kept["int8"] <= 0.45 * kept["bf16"], kept


@pytest.mark.parametrize("name", ["d256", "d256_sla2"])
def test_trainer_steps(kernels, name):
    """Training steps with 8-bit activations: finite, repeatable bit for bit with ``run.deterministic``,
    loss of the first step equal to the bf16 trainer's (the forward pass is the same)."""
    from imfvideo_b200.config import apply_overrides, preset
    from imfvideo_b200.train import Trainer

    def run(store):
        cfg = apply_overrides(preset(name), {"model.act_store": store, "model.depth": 3, "model.aux_head_depth": 1,
                                             "optim.warmup_steps": 0, "run.deterministic": True})
        cfg.data.latent_frames, cfg.data.latent_size = 4, (32, 32)
        tr = Trainer(cfg, device=torch.device("cuda", 0), verbose=False)
        g = torch.Generator().manual_seed(7)
        out = []
        for _ in range(2):
            x = torch.randn(1, 16, 4, 32, 32, generator=g).pin_memory()
            out.append(tr.train_step(x, torch.randint(0, 1000, (1,), generator=g)))
        return out, torch.cat([p.detach().float().flatten() for p in tr.net.parameters()])

    try:
        (s1, p1), (s2, p2), (s0, _) = run("int8"), run("int8"), run("bf16")
    finally:
        kernels.set_deterministic(False)
    kernels.check_status()
    assert all(s["loss"] == s["loss"] and not s["skipped"] and s["grad_norm"] > 0 for s in s1)
    assert [s["loss"] for s in s1] == [s["loss"] for s in s2] and torch.equal(p1, p2)
    assert s1[0]["loss"] == s0[0]["loss"]
    assert abs(s1[0]["grad_norm"] - s0[0]["grad_norm"]) <= 0.1 * s0[0]["grad_norm"]


def test_with_block_recomputation(kernels):
    """Together with ``grad_checkpoint`` (pointless, but allowed)."""
    from imfvideo_b200.models import IMFDiTVideo, flash_jvp_attention
    from imfvideo_b200.ops.dual import Dual

    def grads(ckpt):
        torch.manual_seed(0)
        net = IMFDiTVideo(input_size=(16, 32), num_frames=2, depth=2, aux_head_depth=1, hidden_size=256, num_heads=4,
                          kv_lora_rank=128, attn_res_block_size=2, attn_impl=flash_jvp_attention, compute_dtype=BF16,
                          act_store="int8", grad_checkpoint=ckpt)
        with torch.no_grad():
            for p in net.parameters():
                p.add_(torch.randn_like(p) * 0.03)
        net = net.cuda()
        g = torch.Generator(device="cuda").manual_seed(1)
        x, dx = (torch.randn(1, 16, 2, 16, 32, device="cuda", generator=g) for _ in range(2))
        one = torch.ones(1, device="cuda")
        out = net.forward_dual(Dual(x, dx), Dual(one * 0.4, one), one * 2, one * 0, one, torch.tensor([3], device="cuda"))
        (out["u"].p.square().mean() + out["v"].p.square().mean()).backward()
        return [p.grad for p in net.parameters()]

    kernels.set_deterministic(True)
    try:
        for a, b in zip(grads(False), grads(True)):
            assert (a is None) == (b is None)
            if a is not None:
                assert (a - b).norm() <= 2.0 ** -7 * a.norm() + 1e-12
    finally:
        kernels.set_deterministic(False)
    kernels.check_status()
