"""What differential attention and the norms around a block's branch are measured on.

Both belong to one variant of this repository's transformer block: attention whose second softmax map
is subtracted with a learned weight for each pair of heads, and a residual update that norms what a
branch returns before it is gated and added (``imfvideo_b200.ops.dual.diff_attention`` and
``norm_add_norm``).

Kinds of case
  attn_fwd    o alone, as the sampler evaluates the network
  attn_jvp    o and its forward-mode tangent, as a training step's first pass
  attn_train  o, then the gradients of q, k, v and of the pairs' weights
  norm_fwd, norm_jvp, norm_train  the same three for
              x = r * res + gate * post * y / rms(y),  n = pre * x / rms(x)

Tokens, heads and widths are those of the d=256, d=384, d=1024 and d=1536 models of this repository, on
their own clips and on short ones.  L counts tokens, H pairs of heads of 64 channels.
"""

import math

import torch

own = False

HD = 64
EPS = 1e-5


def listed():
    return [
        # the smoke run's clip (4 x 8 x 16 patches + 20 tokens) in the d=256 model's sampler: latency counts
        dict(name="attn_fwd_smoke", kind="attn_fwd", B=1, L=532, H=2),
        # five frames in the d=1024 model's sampler
        dict(name="attn_fwd_d1024_5f", kind="attn_fwd", B=1, L=7820, H=8),
        # two odd clips at once in the d=384 model, with tangent
        dict(name="attn_jvp_odd", kind="attn_jvp", B=2, L=2061, H=3),
        # a full clip of the d=256 model, with tangent: the largest
        dict(name="attn_jvp_d256", kind="attn_jvp", B=1, L=29140, H=2),
        # training on the smoke run's clip
        dict(name="attn_train_smoke", kind="attn_train", B=1, L=532, H=2),
        # training on five frames, d=1024
        dict(name="attn_train_d1024_5f", kind="attn_train", B=1, L=7820, H=8),
        # training on a full clip, d=256
        dict(name="attn_train_d256", kind="attn_train", B=1, L=29140, H=2),
        # attention branch of the smoke run
        dict(name="norm_train_smoke", kind="norm_train", rows=532, D=256, res=True, scale=True, pre=True),
        # a full clip of the d=1024 model: first pass with tangent, and training
        dict(name="norm_jvp_d1024", kind="norm_jvp", rows=32780, D=1024, res=True, scale=True, pre=True),
        dict(name="norm_train_d1024", kind="norm_train", rows=32780, D=1024, res=True, scale=True, pre=True),
        # the end of a block (no norm follows) at an odd width, in the sampler
        dict(name="norm_fwd_odd", kind="norm_fwd", rows=2061, D=1000, res=True, scale=False, pre=False),
        # a residual stream that begins anew (no res), 12 x 128-head model on five frames
        dict(name="norm_train_fresh", kind="norm_train", rows=7820, D=1536, res=False, scale=False, pre=True),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: one token to some 33 thousand, odd lengths and widths among them."""
    most = {}
    for c in listed():
        for m, w in work(c).items():
            most[c["kind"], m] = max(most.get((c["kind"], m), 0), w)
    most["norm_fwd", "bytes"], most["norm_fwd", "flops"] = most["norm_jvp", "bytes"], most["norm_jvp", "flops"]
    while True:
        kind = rng.choice(["attn_fwd", "attn_jvp", "attn_train", "attn_train", "norm_fwd", "norm_jvp", "norm_train"])
        if kind.startswith("attn"):
            # (a sequence of one token attends to itself alone: its dQ and dK are zero, all noise)
            c = dict(kind=kind, B=rng.choice([1, 1, 2, 3]), L=_logint(rng, 2 if kind == "attn_train" else 1, 32780),
                     H=rng.choice([1, 2, 3, 6, 8]))
        else:
            c = dict(kind=kind, rows=_logint(rng, 1, 40000), D=8 * _logint(rng, 4, 256), res=rng.random() < 0.8,
                     scale=rng.random() < 0.5, pre=rng.random() < 0.7)
            c["scale"] = c["scale"] and c["res"]
        if all(w <= most[kind, m] for m, w in work(c).items()):
            return c


# ------------------------------------------------------------------ inputs ---
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    rnd = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    if c["kind"].startswith("attn"):
        B, L, H = c["B"], c["L"], c["H"]
        shape = (B, L, 2 * H, HD)
        # queries and keys come normed per head; values have an offset in each channel, and the gradient
        # that comes back leans on what all tokens have in common
        offset = 0.5 * rnd(2 * H, HD)
        c["q"], c["k"], c["v"] = rnd(*shape).bfloat16(), rnd(*shape).bfloat16(), (rnd(*shape) + offset).bfloat16()
        c["lam"] = (0.2 + 0.6 * torch.rand(H, device="cuda", generator=g)).bfloat16()
        if c["kind"] == "attn_jvp":
            c["dq"], c["dk"], c["dv"] = ((0.3 * rnd(*shape)).bfloat16() for _ in range(3))
        if c["kind"] == "attn_train":
            c["go"] = (0.02 * (rnd(*shape) + offset)).bfloat16()
        return c
    R, D = c["rows"], c["D"]
    # a residual stream that has grown, a branch's output with channels of different size
    chan = torch.exp(0.5 * rnd(D))
    c["y"] = (rnd(R, D) * chan).bfloat16()
    c["resid"] = 3 * rnd(R, D) if c["res"] else None
    c["post"], c["gate"] = 1 + 0.2 * rnd(D), 0.5 + 0.2 * rnd(D)
    c["r"] = 0.9 + 0.1 * rnd(D) if c["scale"] else None
    c["gain"] = 1 + 0.2 * rnd(D) if c["pre"] else None
    if c["kind"] == "norm_jvp":
        c["dy"] = (0.3 * rnd(R, D) * chan).bfloat16()
        c["dres"] = rnd(R, D) if c["res"] else None
    if c["kind"] == "norm_train":
        c["gx"] = 0.02 * rnd(R, D)
        c["gn"] = (0.02 * rnd(R, D)).bfloat16() if c["pre"] else None
    return c


# ------------------------------------------------------------------ one pass, plain ---
def _maps(t, m):
    """(B, H, L, 64) in 32 bits: the queries or keys of map m of every pair."""
    return t[:, :, m::2].transpose(1, 2).float()


def _wide(t):
    """(B, H, L, 128) in 32 bits: both heads of a pair side by side."""
    return t.reshape(*t.shape[:2], t.shape[2] // 2, 2 * HD).transpose(1, 2).float()


def _back(t, like):
    return t.transpose(1, 2).reshape(like.shape).to(like.dtype)


def _softmax(s):
    s = torch.exp(s - s.amax(-1, keepdim=True))
    return s / s.sum(-1, keepdim=True)


def _attn_map(st, m):
    """O_m, and its tangent where there is one."""
    scale = HD ** -0.5
    q, k, v = _maps(st["q"], m), _maps(st["k"], m), _wide(st["v"])
    a = _softmax(q @ k.transpose(-1, -2) * scale)
    if st["kind"] != "attn_jvp":
        return a @ v, None
    ds = (_maps(st["dq"], m) @ k.transpose(-1, -2) + q @ _maps(st["dk"], m).transpose(-1, -2)) * scale
    t = a * (ds - (a * ds).sum(-1, keepdim=True))
    return a @ v, t @ v + a @ _wide(st["dv"])


def _attn_grads(st, m, weight, delta, dp):
    """Gradients of q_m and k_m, and of V through this map, which enters with `weight`."""
    scale = HD ** -0.5
    q, k = _maps(st["q"], m), _maps(st["k"], m)
    a = weight * _softmax(q @ k.transpose(-1, -2) * scale)
    gv = a.transpose(-1, -2) @ _wide(st["go"])
    a *= dp - delta
    return a @ k * scale, a.transpose(-1, -2) @ q * scale, gv


def _pairs(t1, t2, like):
    return torch.stack([t1, t2], 2).flatten(1, 2).transpose(1, 2).reshape(like.shape).to(like.dtype)


def _attn(st):
    lam = st["lam"].float()[:, None, None]
    (o1, t1), (o2, t2) = _attn_map(st, 0), _attn_map(st, 1)
    o = _back(o1 - lam * o2, st["q"])
    if st["kind"] == "attn_fwd":
        return o
    if st["kind"] == "attn_jvp":
        return o, _back(t1 - lam * t2, st["q"])
    go = _wide(st["go"])
    dp = go @ _wide(st["v"]).transpose(-1, -2)
    d1, d2 = (go * o1).sum(-1, keepdim=True), (go * o2).sum(-1, keepdim=True)
    gq1, gk1, gv1 = _attn_grads(st, 0, 1.0, d1, dp)
    gq2, gk2, gv2 = _attn_grads(st, 1, -lam, d2, dp)
    glam = -d2.sum((0, 2, 3)).to(st["lam"].dtype)
    return o, _pairs(gq1, gq2, st["q"]), _pairs(gk1, gk2, st["k"]), _back(gv1 + gv2, st["v"]), glam


def _norm(st):
    y, R, gate, post = st["y"].float(), st["resid"], st["gate"], st["post"]
    r = 1.0 if st["r"] is None else st["r"]
    iy = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    yh = y * iy
    x = yh * (gate * post) + (0 if R is None else R * r)
    ix = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    xh = x * ix
    n = None if st["gain"] is None else (xh * st["gain"]).to(st["y"].dtype)
    if st["kind"] == "norm_fwd":
        return {"x": x, "n": n}
    if st["kind"] == "norm_jvp":
        dy = st["dy"].float()
        dx = iy * (dy - yh * (yh * dy).mean(-1, keepdim=True)) * (gate * post) + (0 if R is None else st["dres"] * r)
        dn = None if n is None else (ix * (dx - xh * (xh * dx).mean(-1, keepdim=True)) * st["gain"]).to(st["y"].dtype)
        return {"x": x, "n": n, "dx": dx, "dn": dn}
    gx, out = st["gx"], {"x": x, "n": n}
    if n is not None:
        gn = st["gn"].float()
        out["g_gain"] = (gn * xh).sum(0)
        gn = gn * st["gain"]
        gx = gx + ix * (gn - xh * (gn * xh).mean(-1, keepdim=True))
    if R is not None:
        out["g_res"] = gx * r
    if st["r"] is not None:
        out["g_r"] = (gx * R).sum(0)
    s = (gx * yh).sum(0)
    out["g_gate"], out["g_post"] = s * post, s * gate
    gy = gx * (gate * post)
    out["g_y"] = (iy * (gy - yh * (gy * yh).mean(-1, keepdim=True))).to(st["y"].dtype)
    return out


# ------------------------------------------------------------------ one pass, the framework ---
def _own(st):
    from imfvideo_b200.ops import dual as D

    kind = st["kind"]
    if kind == "attn_fwd":
        return D.diff_attention(D.Dual(st["q"]), D.Dual(st["k"]), D.Dual(st["v"]), st["lam"]).p
    if kind == "attn_jvp":
        return tuple(D.diff_attention(D.Dual(st["q"], st["dq"]), D.Dual(st["k"], st["dk"]),
                                      D.Dual(st["v"], st["dv"]), st["lam"]))
    if kind == "attn_train":
        leaves = [st[n].detach().requires_grad_() for n in ("q", "k", "v", "lam")]
        with torch.enable_grad():
            o = D.diff_attention(*(D.Dual(t) for t in leaves[:3]), leaves[3]).p
        return (o.detach(), *torch.autograd.grad(o, leaves, st["go"]))
    if kind == "norm_train":
        names = {"resid": "g_res", "y": "g_y", "post": "g_post", "gate": "g_gate", "r": "g_r", "gain": "g_gain"}
        leaf = {n: None if st[n] is None else st[n].detach().requires_grad_() for n in names}
        with torch.enable_grad():
            x, n = D.norm_add_norm(None if leaf["resid"] is None else D.Dual(leaf["resid"]), D.Dual(leaf["y"]),
                                   leaf["post"], leaf["gate"], EPS, res_scale=leaf["r"], pre=leaf["gain"])
        have = [m for m in names if leaf[m] is not None]
        outs = [(x.p, st["gx"])] + ([] if n is None else [(n.p, st["gn"])])
        grads = torch.autograd.grad([o for o, _ in outs], [leaf[m] for m in have], [g for _, g in outs])
        return {"x": x.p.detach(), "n": None if n is None else n.p.detach(), **{names[m]: g for m, g in zip(have, grads)}}
    x, n = D.norm_add_norm(None if st["resid"] is None else D.Dual(st["resid"], st.get("dres")),
                           D.Dual(st["y"], st.get("dy")), st["post"], st["gate"], EPS, res_scale=st["r"], pre=st["gain"])
    out = {"x": x.p, "n": None if n is None else n.p}
    return out if kind == "norm_fwd" else {**out, "dx": x.t, "dn": None if n is None else n.t}


def run(state):
    if own:
        out = _own(state)
    else:
        out = _attn(state) if state["kind"].startswith("attn") else _norm(state)
    return {k: out[k] for k in sorted(out) if out[k] is not None} if isinstance(out, dict) else out


# ------------------------------------------------------------------ work and oracle ---
def work(case):
    c = case
    if c["kind"].startswith("attn"):
        n = c["B"] * c["L"] * c["H"] * 2 * HD                       # elements of q
        pairs = c["B"] * c["H"] * c["L"] ** 2
        fwd = 2 * 2 * pairs * (HD + 2 * HD)                        # two maps: scores and product with V
        if c["kind"] == "attn_fwd":
            return {"bytes": 2 * 4 * n, "flops": fwd}
        if c["kind"] == "attn_jvp":                                # two products make dS, two make do
            return {"bytes": 2 * 8 * n, "flops": fwd + 2 * 2 * pairs * (2 * HD + 2 * 2 * HD)}
        # reverse: scores again, dP once for both maps, dV once, dQ and dK of both
        return {"bytes": 2 * 8 * n, "flops": fwd + 2 * pairs * (2 * HD + 2 * HD + 2 * HD + 2 * 2 * HD)}
    n, t = c["rows"] * c["D"], 2 if c["kind"] == "norm_jvp" else 1
    moved = 2 + 4 + (4 if c["res"] else 0) + (2 if c["pre"] else 0)
    if c["kind"] == "norm_train":                                  # g_x, g_n in; g_y, g_res out
        moved += 4 + (2 if c["pre"] else 0) + 2 + (4 if c["res"] else 0)
    return {"bytes": t * moved * n, "flops": t * (30 if c["kind"] == "norm_train" else 12) * n}


def _exact_attn(st):
    B, L, H = st["B"], st["L"], st["H"]
    lam64 = st["lam"].double()
    o = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    more = [torch.zeros_like(o) for _ in range({"attn_fwd": 0, "attn_jvp": 1, "attn_train": 3}[st["kind"]])]
    glam = torch.zeros_like(lam64)
    for b in range(B):
        for j in range(H):
            pair = slice(2 * j, 2 * j + 2)
            v = st["v"][b, :, pair].double().reshape(L, 2 * HD)
            total, dtotal, parts = 0, 0, []
            for m in (0, 1):
                w = 1.0 if m == 0 else -lam64[j]
                q, k = st["q"][b, :, 2 * j + m].double(), st["k"][b, :, 2 * j + m].double()
                a = torch.softmax((q @ k.t()).mul_(1 / math.sqrt(HD)), -1)
                om = a @ v
                total = total + w * om
                if st["kind"] == "attn_jvp":
                    ds = st["dq"][b, :, 2 * j + m].double() @ k.t()
                    ds = ds.addmm_(q, st["dk"][b, :, 2 * j + m].double().t()).mul_(1 / math.sqrt(HD)).mul_(a)
                    dom = a @ st["dv"][b, :, pair].double().reshape(L, 2 * HD) + ds @ v
                    dtotal = dtotal + w * (dom - ds.sum(-1, keepdim=True) * om)
                if st["kind"] == "attn_train":
                    go = st["go"][b, :, pair].double().reshape(L, 2 * HD)
                    more[2][b, :, pair] += (w * (a.t() @ go)).view(L, 2, HD)
                    ds = (go @ v.t()).sub_((go * om).sum(-1, keepdim=True)).mul_(a).mul_(w / math.sqrt(HD))
                    more[0][b, :, 2 * j + m], more[1][b, :, 2 * j + m] = ds @ k, ds.t() @ q
                    if m == 1:
                        glam[j] -= (go * om).sum()
            o[b, :, pair] = total.view(L, 2, HD)
            if st["kind"] == "attn_jvp":
                more[0][b, :, pair] = dtotal.view(L, 2, HD)
    return o if st["kind"] == "attn_fwd" else (o, *more) if st["kind"] == "attn_jvp" else (o, *more, glam)


def _exact_norm(st):
    names = ("resid", "y", "post", "gate", "r", "gain")
    leaf = {n: None if st[n] is None else st[n].double() for n in names}

    def f(v):
        rms = lambda t: (t.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        x = v["y"] / rms(v["y"]) * v["post"] * v["gate"]
        if v["resid"] is not None:
            x = x + (v["resid"] if v["r"] is None else v["resid"] * v["r"])
        return x, None if v["gain"] is None else x / rms(x) * v["gain"]

    if st["kind"] == "norm_fwd":
        x, n = f(leaf)
        return {"x": x, "n": n}
    if st["kind"] == "norm_jvp":
        moving = [n for n in ("resid", "y") if leaf[n] is not None]
        tang = tuple(st["d" + ("res" if n == "resid" else n)].double() for n in moving)
        outs = lambda *a: tuple(t for t in f({**leaf, **dict(zip(moving, a))}) if t is not None)
        val, dval = torch.func.jvp(outs, tuple(leaf[n] for n in moving), tang)
        return {"x": val[0], "dx": dval[0], "n": val[1] if len(val) > 1 else None, "dn": dval[1] if len(dval) > 1 else None}
    with torch.enable_grad():
        have = [n for n in names if leaf[n] is not None]
        for n in have:
            leaf[n].requires_grad_()
        x, n = f(leaf)
        loss = (x * st["gx"].double()).sum() + (0 if n is None else (n * st["gn"].double()).sum())
        grads = torch.autograd.grad(loss, [leaf[m] for m in have])
    out = {"x": x.detach(), "n": None if n is None else n.detach()}
    return {**out, **{"g_" + ("res" if m == "resid" else m): g for m, g in zip(have, grads)}}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"].startswith("attn"):
        return _exact_attn(st)
    out = _exact_norm(st)
    return {k: out[k] for k in sorted(out) if out[k] is not None}
