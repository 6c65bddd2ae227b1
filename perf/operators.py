"""What the operators on 8-bit activation checkpoints are measured on.

A training step keeps the activations of every transformer block for its backward pass.  These
operators keep them as 8-bit codes with a power-of-two step for each 32 channels of a row, and run the
backward pass from them (``imfvideo_b200.ops.act8``).

Kinds of case
  store    activations into checkpoints and back: one tensor, or what a whole block keeps, at once
  restore  checkpoints back into activations, as the backward pass of a block does first
  wgrad    weight gradient dY^T X of a linear layer whose input X is a checkpoint
  situ     reverse mode of the gated activation from the checkpoint of its input [gate | up]; the
           activation itself comes along for the next weight gradient
  attn     reverse mode of dense attention from checkpoints of q, k, v and o

Rows are tokens.  The sizes are those of the d=256 and d=1024 models and of the 12 x 128-head model
of this repository, on their own clips and on short ones.
"""

import math

import torch

own = False

GROUP = 32
BETA, LBETA = 4.0, 25.0


def listed():
    return [
        # everything a block of the d=256 model keeps of the smoke run's clip (4 x 8 x 16 patches + 20):
        # many small tensors, latency counts
        dict(name="store_smoke", kind="store", whole=True, rows=532, d=256, H=4, lora=128),
        # everything a block of the d=1024 model keeps of a full clip
        dict(name="store_d1024", kind="store", whole=True, rows=32780, d=1024, H=16, lora=512),
        # one fp32 tensor of odd width, a band of a wider one: a residual stream
        dict(name="store_odd_fp32", kind="store", whole=False, rows=2068, cols=1021, more=3, fp32=True),
        # the backward pass of a d=256 block begins: checkpoints of a full clip back to bf16
        dict(name="restore_d256", kind="restore", whole=True, rows=29140, d=256, H=4, lora=128),
        # a narrow tensor of a short clip
        dict(name="restore_short", kind="restore", whole=False, rows=276, cols=528, more=0, fp32=False),
        # gate / up weights of the d=256 model on a full clip
        dict(name="wgrad_d256", kind="wgrad", rows=29140, n_out=1376, n_in=256),
        # the same of the d=1024 model: a large product
        dict(name="wgrad_d1024", kind="wgrad", rows=32780, n_out=5472, n_in=1024),
        # the fused q / kv / gate projection of the smoke run
        dict(name="wgrad_smoke", kind="wgrad", rows=532, n_out=528, n_in=256),
        # the MLP of the d=1024 model and of a short clip on the d=256 model
        dict(name="situ_d1024", kind="situ", rows=32780, F=2736),
        dict(name="situ_clip", kind="situ", rows=2068, F=688),
        # attention of the d=256 model on a full clip, and of the 12 x 128-head model on five frames
        dict(name="attn_d256", kind="attn", B=1, L=29140, H=4, hd=64),
        dict(name="attn_hd128_5f", kind="attn", B=1, L=7820, H=12, hd=128),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: one token to some 33 thousand, narrow to wide, odd sizes among them."""
    most = {}
    for c in listed():
        w = work(c)
        for m in w:
            most[c["kind"], m] = max(most.get((c["kind"], m), 0), w[m])
    while True:
        kind = rng.choice(["store", "restore", "wgrad", "situ", "attn", "attn"])
        if kind in ("store", "restore"):
            if rng.random() < 0.5:
                d, H, lora = rng.choice([(256, 4, 128), (384, 6, 96), (1024, 16, 512), (1536, 12, 384)])
                c = dict(kind=kind, whole=True, rows=_logint(rng, 20, 32780), d=d, H=H, lora=lora)
            else:
                c = dict(kind=kind, whole=False, rows=_logint(rng, 1, 32780), cols=_logint(rng, 1, 6000),
                         more=rng.choice([0, 0, 1, 8, 40]), fp32=kind == "store" and rng.random() < 0.4)
        elif kind == "wgrad":
            c = dict(kind=kind, rows=_logint(rng, 1, 32780), n_out=8 * _logint(rng, 1, 684),
                     n_in=rng.choice([1, 8, 8]) * _logint(rng, 8, 190))
        elif kind == "situ":
            c = dict(kind=kind, rows=_logint(rng, 1, 32780), F=8 * _logint(rng, 1, 342))
        else:
            # (a sequence of one token attends to itself alone: its dQ and dK are zero, all noise)
            c = dict(kind=kind, B=rng.choice([1, 1, 2, 3]), L=_logint(rng, 2, 32780),
                     H=rng.choice([1, 2, 3, 4, 6, 12, 16]), hd=rng.choice([64, 64, 128]))
        if all(work(c)[m] <= most[kind, m] for m in ("bytes", "flops")):
            return c


def _widths(c):
    """Widths of the tensors a case stores: one, or all that a block of d channels keeps."""
    if not c["whole"]:
        return [c["cols"]]
    d, H, lora = c["d"], c["H"], c["lora"]
    hd = d // H
    rope = max(2, hd // 4)
    F = (int(d * 8 / 3) + 7) // 8 * 8
    return [d, d // 2 + lora + rope + d, d // 2, lora, d, H * (2 * hd - rope), d, d, d, d, d, 2 * F, d]


# ------------------------------------------------------------------ the format ---
def _power(e, bits, bias):
    """2^e in 32 or 64 bits, exactly, from the bits of the number (e = -127 in 32 is half the smallest normal one)."""
    whole, mant = (torch.int32, 23) if bits == 32 else (torch.int64, 52)
    n = e.to(whole) + bias
    n = torch.where(n <= 0, torch.full_like(n, 1 << (mant - 1)), n << mant)
    return n.view(torch.float32 if bits == 32 else torch.float64)


def _store(x):
    """(codes (R, pitch) int8, steps (R, spitch) uint8) of x (R, C): groups of 32 channels, the pitches
    rounded up to 32 channels and 4 groups."""
    R, C = x.shape
    G = (C + GROUP - 1) // GROUP
    g = torch.zeros(R, G * GROUP, dtype=torch.float32, device=x.device)
    g[:, :C] = x
    g = g.view(R, G, GROUP)
    amax = g.abs().amax(-1)
    mant, exp = torch.frexp(amax)                                   # amax = mant 2^exp, mant in [1/2, 1)
    e = exp - 7 + (mant >= 127.5 / 128).to(exp.dtype)               # the largest is 64 to 127 steps
    e = torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(-127, 121)
    bad = ~torch.isfinite(amax)
    codes = torch.round(g * _power(-e, 32, 127)[..., None]).clamp(-127, 127)
    codes = torch.where(bad[..., None], torch.zeros_like(codes), codes)
    steps = torch.zeros(R, (G + 3) // 4 * 4, dtype=torch.uint8, device=x.device)
    steps[:, :G] = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return codes.to(torch.int8).view(R, G * GROUP), steps


def _values(p, C):
    """fp32 values (R, C) of codes and steps."""
    codes, steps = p
    R, W = codes.shape
    e = steps[:, :W // GROUP].to(torch.int32) - 127
    step = torch.where(e == 128, torch.full_like(e, 0x7fc00000).view(torch.float32), _power(e, 32, 127))
    return (codes.view(R, W // GROUP, GROUP).float() * step[..., None]).view(R, W)[:, :C]


# ------------------------------------------------------------------ inputs ---
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, R, C, more=0, dtype=torch.bfloat16):
    """Activations of a network: channels of different size, a few of them far above the rest."""
    scale = torch.exp(0.5 * torch.randn(C + more, device="cuda", generator=g))
    scale = scale * torch.where(torch.rand(C + more, device="cuda", generator=g) < 0.01, 12.0, 1.0)
    x = torch.randn(R, C + more, device="cuda", generator=g) * scale
    return x.to(dtype)[:, more:]


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["kind"] in ("store", "restore"):
        dt = torch.bfloat16 if c["whole"] or not c["fp32"] else torch.float32
        xs = [_activations(g, c["rows"], w, 0 if c["whole"] else c["more"], dt) for w in _widths(c)]
        if c["kind"] == "store":
            return dict(c, xs=xs)
        return dict(c, widths=_widths(c), packed=[_store(x) for x in xs])
    if c["kind"] == "wgrad":
        dy = (torch.randn(c["rows"], c["n_out"], device="cuda", generator=g) * 0.02).bfloat16()
        return dict(c, dy=dy, x=_store(_activations(g, c["rows"], c["n_in"])))
    if c["kind"] == "situ":
        gu = _activations(g, c["rows"], 2 * c["F"])
        gout = (torch.randn(c["rows"], c["F"], device="cuda", generator=g) * 0.05).bfloat16()
        return dict(c, gu=_store(gu), gout=gout)
    B, L, H, hd = c["B"], c["L"], c["H"], c["hd"]
    q, k, v, go = (torch.randn(B, L, H, hd, device="cuda", generator=g).bfloat16() for _ in range(4))
    o = torch.empty(B, L, H, hd, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(B, H, L, device="cuda")
    for b in range(B):                                 # a head at a time, for memory
        for h in range(H):
            s = q[b, :, h].float() @ k[b, :, h].float().t() * hd ** -0.5
            lse[b, h] = torch.logsumexp(s, -1)
            o[b, :, h] = (torch.exp(s - lse[b, h][:, None]) @ v[b, :, h].float()).bfloat16()
    return dict(c, packed=[_store(t.reshape(B * L * H, hd)) for t in (q, k, v, o)], lse=lse, go=go)


# ------------------------------------------------------------------ one pass ---
def _situ(gate, up, gout):
    """Gradients of gate and up of y = beta tanh(gate/beta) sigmoid(gate) lbeta tanh(up/lbeta), and y."""
    th, sg, tu = torch.tanh(gate / BETA), 1 / (1 + torch.exp(-gate)), torch.tanh(up / LBETA)
    a, u = BETA * th * sg, LBETA * tu
    da = (1 - th * th) * sg + BETA * th * sg * (1 - sg)
    return gout * da * u, gout * a * (1 - tu * tu), a * u


def _attention(q, k, v, o, lse, go, scale):
    """dQ, dK, dV of (B, H, L, hd) tensors; the probabilities come back from the scores and lse."""
    p = torch.exp(q @ k.transpose(-1, -2) * scale - lse[..., None])
    dv = p.transpose(-1, -2) @ go
    ds = p * (go @ v.transpose(-1, -2) - (go * o).sum(-1)[..., None])
    return ds @ k * scale, ds.transpose(-1, -2) @ q * scale, dv


def _plain(st):
    kind = st["kind"]
    if kind == "store":
        return [_values(_store(x), x.shape[1]).to(x.dtype) for x in st["xs"]]
    if kind == "restore":
        return [_values(p, w).bfloat16() for p, w in zip(st["packed"], st["widths"])]
    if kind == "wgrad":
        return st["dy"].float().t() @ _values(st["x"], st["n_in"])
    if kind == "situ":
        gu, F = _values(st["gu"], 2 * st["F"]), st["F"]
        gg, gu_, y = _situ(gu[:, :F], gu[:, F:], st["gout"].float())
        return torch.cat([gg, gu_], 1).bfloat16(), y.bfloat16()
    B, L, H, hd = st["B"], st["L"], st["H"], st["hd"]
    heads = lambda t: t.reshape(B, L, H, hd).transpose(1, 2)
    q, k, v, o = (heads(_values(p, hd)) for p in st["packed"])
    out = _attention(q, k, v, o, st["lse"], heads(st["go"].float()), hd ** -0.5)
    return tuple(t.transpose(1, 2).contiguous().bfloat16() for t in out)


def _own(st):
    from imfvideo_b200.ops import act8

    kind = st["kind"]
    made = lambda p, shape: act8.Packed8(p[0], p[1], shape)
    if kind == "store":
        return act8.restore8(act8.store8(st["xs"]))
    if kind == "restore":
        return act8.restore8([made(p, (st["rows"], w)) for p, w in zip(st["packed"], st["widths"])])
    if kind == "wgrad":
        return act8.gemm_wgrad8(st["dy"], made(st["x"], (st["rows"], st["n_in"])))
    if kind == "situ":
        return act8.situ_bwd8(made(st["gu"], (st["rows"], 2 * st["F"])), st["gout"], BETA, LBETA)
    shape = (st["B"], st["L"], st["H"], st["hd"])
    q8, k8, v8, o8 = (made(p, shape) for p in st["packed"])
    return act8.attn_bwd8(q8, k8, v8, o8, st["lse"], st["go"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ work and oracle ---
def work(case):
    c = case
    if c["kind"] in ("store", "restore"):
        n = c["rows"] * sum(_widths(c))
        size = 2 if c["whole"] or not c["fp32"] else 4
        byte8 = n * 33 / 32
        if c["kind"] == "restore":
            return {"bytes": byte8 + 2 * n, "flops": n}
        return {"bytes": 2 * size * n + 2 * byte8, "flops": 4 * n}      # in; checkpoint written and read; out
    if c["kind"] == "wgrad":
        R, N, K = c["rows"], c["n_out"], c["n_in"]
        return {"bytes": 2 * R * N + R * K * 33 / 32 + 4 * N * K, "flops": 2 * R * N * K}
    if c["kind"] == "situ":
        n = c["rows"] * c["F"]
        return {"bytes": 2 * n * 33 / 32 + 2 * n + 4 * n + 2 * n, "flops": 25 * n}
    B, L, H, hd = c["B"], c["L"], c["H"], c["hd"]
    n = B * L * H * hd
    return {"bytes": 4 * n * 33 / 32 + 2 * n + 6 * n + 4 * B * H * L, "flops": 10 * B * H * L * L * hd}


def _exact_store(x):
    """Values in 64 bits of x stored in 8: a step is the smallest power of two that the group's largest
    magnitude rounds to at most 127 of (127.5 of them round to 128)."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c0 in range(0, x.shape[1], GROUP):
        v = x[:, c0:c0 + GROUP].double()
        e = torch.frexp(v.abs().amax(1, keepdim=True) / 127.5)[1]          # the smallest with 2^e above it
        step = _power(e.clamp(-127, 121), 64, 1023)
        out[:, c0:c0 + GROUP] = torch.round(v / step).clamp(-127, 127) * step
    return out


def _exact_values(p, C):
    codes, steps = p
    step = _power(steps.int() - 127, 64, 1023).repeat_interleave(GROUP, 1)[:, :C]
    return codes[:, :C].double() * step


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "store":
        return [_exact_store(x) for x in st["xs"]]
    if kind == "restore":
        return [_exact_values(p, w) for p, w in zip(st["packed"], st["widths"])]
    if kind == "wgrad":
        return st["dy"].double().t() @ _exact_values(st["x"], st["n_in"])
    if kind == "situ":
        gu, F = _exact_values(st["gu"], 2 * st["F"]), st["F"]
        with torch.enable_grad():
            z = gu.requires_grad_()
            y = BETA * torch.tanh(z[:, :F] / BETA) * torch.sigmoid(z[:, :F]) * LBETA * torch.tanh(z[:, F:] / LBETA)
            grad, = torch.autograd.grad(y, z, st["gout"].double())
        return grad, y.detach()
    B, L, H, hd = st["B"], st["L"], st["H"], st["hd"]
    q, k, v, o = (_exact_values(p, hd).view(B, L, H, hd) for p in st["packed"])
    go, lse = st["go"].double(), st["lse"].double()
    dq, dk, dv = (torch.empty_like(q) for _ in range(3))
    for b in range(B):
        for h in range(H):
            qh, kh, vh, oh, gh = (t[b, :, h] for t in (q, k, v, o, go))
            w = qh @ kh.t()
            w = w.mul_(hd ** -0.5).sub_(lse[b, h][:, None]).exp_()
            dv[b, :, h] = w.t() @ gh
            w *= gh @ vh.t() - (gh * oh).sum(1, keepdim=True)
            dq[b, :, h] = w @ kh * hd ** -0.5
            dk[b, :, h] = w.t() @ qh * hd ** -0.5
    return dq, dk, dv
