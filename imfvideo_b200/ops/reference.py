"""Plain-PyTorch formulas for every dual-number (primal, tangent) op.

These are the CPU path, the oracle for every CUDA kernel test, and the
numerics contract of the framework.  Each ``*_jvp`` function returns
``(y, dy)`` for inputs ``(x, dx)``; parameters carry no tangent (the iMF
loss differentiates w.r.t. time only, reference ``imf_video.py:485-533``).

All math is done in fp32 regardless of the storage dtype, matching the
reference modules (``models/imf_dit_video.py:121-165``, ``:266-320``).
"""

from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch

Tensor = torch.Tensor


# --------------------------------------------------------------------------
# RMSNorm
# --------------------------------------------------------------------------
def rmsnorm(x: Tensor, weight: Optional[Tensor], eps: float) -> Tensor:
    xf = x.float()
    r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    y = (xf * r).to(x.dtype)
    return y if weight is None else y * weight


def rmsnorm_jvp(x: Tensor, dx: Tensor, weight: Optional[Tensor], eps: float
                ) -> Tuple[Tensor, Tensor]:
    """y = x r g with r = rsqrt(mean x^2 + eps);
    dy = g (r dx - x r^3 mean(x dx))."""
    xf, dxf = x.float(), dx.float()
    r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    y = xf * r
    dy = dxf * r - xf * (r.pow(3) * (xf * dxf).mean(-1, keepdim=True))
    if weight is not None:
        w = weight.float()
        y, dy = y * w, dy * w
    return y.to(x.dtype), dy.to(dx.dtype)


# --------------------------------------------------------------------------
# SituAndMul: beta tanh(g/beta) sigmoid(g) * (lbeta tanh(up/lbeta))
# --------------------------------------------------------------------------
def situ_mul(gate: Tensor, up: Tensor, beta: float,
             linear_beta: Optional[float]) -> Tensor:
    g, u = gate.float(), up.float()
    a = beta * torch.tanh(g / beta) * torch.sigmoid(g)
    if linear_beta is not None:
        u = linear_beta * torch.tanh(u / linear_beta)
    return (a * u).to(gate.dtype)


def situ_mul_jvp(gate: Tensor, up: Tensor, dgate: Tensor, dup: Tensor,
                 beta: float, linear_beta: Optional[float]
                 ) -> Tuple[Tensor, Tensor]:
    """Includes the ``linear_beta`` clamp on the up branch in the tangent
    (the reference's Triton tangent kernel omits it,
    ``models/triton_mla_block_jvp.py:437-471``; the module applies it,
    ``models/imf_dit_video.py:163-164``)."""
    g, u = gate.float(), up.float()
    dg, du = dgate.float(), dup.float()
    th = torch.tanh(g / beta)
    sg = torch.sigmoid(g)
    a = beta * th * sg
    da = ((1 - th * th) * sg + beta * th * sg * (1 - sg)) * dg
    if linear_beta is not None:
        tu = torch.tanh(u / linear_beta)
        du = (1 - tu * tu) * du
        u = linear_beta * tu
    return (a * u).to(gate.dtype), (da * u + a * du).to(dgate.dtype)


# --------------------------------------------------------------------------
# Rotary embedding on adjacent (even, odd) channel pairs
# --------------------------------------------------------------------------
def rope(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    """x: (b, l, H, dr); cos/sin: (l, dr/2). Linear in x, so the tangent of
    rope(x) is rope(dx)."""
    xf = x.float()
    xr, xi = xf[..., 0::2], xf[..., 1::2]
    c, s = cos[None, :, None, :], sin[None, :, None, :]
    out = torch.stack([xr * c - xi * s, xr * s + xi * c], dim=-1).flatten(-2)
    return out.to(x.dtype)


# --------------------------------------------------------------------------
# Dense attention (b, l, H, d) layout, softmax scale 1/sqrt(dk)
# --------------------------------------------------------------------------
def _q_chunk(l: int, s: int, bh: int, budget_bytes: int = 1 << 30) -> int:
    per_row = max(1, s * bh * 4 * 4)
    return max(16, min(l, budget_bytes // per_row))


def attention(q: Tensor, k: Tensor, v: Tensor, scale: Optional[float] = None
              ) -> Tensor:
    """softmax(q k^T * scale) v, fp32 softmax; einsum form so forward-mode
    and reverse-mode AD both work on every backend."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    s = torch.einsum("blhd,bshd->bhls", q.float(), k.float()) * scale
    p = torch.softmax(s, dim=-1)
    return torch.einsum("bhls,bshd->blhd", p, v.float()).to(v.dtype)


def attention_lse(q: Tensor, k: Tensor, scale: Optional[float] = None) -> Tensor:
    """Natural-log LSE of the scaled scores: (b, H, l)."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    s = torch.einsum("blhd,bshd->bhls", q.float(), k.float()) * scale
    return torch.logsumexp(s, dim=-1)


@torch.no_grad()
def attention_jvp(q: Tensor, k: Tensor, v: Tensor, dq: Tensor, dk: Tensor,
                  dv: Tensor, scale: Optional[float] = None,
                  chunk: Optional[int] = None) -> Tuple[Tensor, Tensor]:
    """(o, do) with
        ds = (dq k^T + q dk^T) scale,  dp = p (ds - rowsum(p ds)),
        do = dp v + p dv.
    Chunked over query rows so the (l, s) score matrix never exceeds ~1 GB."""
    b, l, H, _ = q.shape
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    kf, vf, dkf, dvf = k.float(), v.float(), dk.float(), dv.float()
    step = chunk or _q_chunk(l, k.shape[1], b * H)
    o = torch.empty(b, l, H, v.shape[-1], dtype=v.dtype, device=v.device)
    do = torch.empty_like(o)
    for i in range(0, l, step):
        qf, dqf = q[:, i:i + step].float(), dq[:, i:i + step].float()
        s = torch.einsum("blhd,bshd->bhls", qf, kf) * scale
        ds = (torch.einsum("blhd,bshd->bhls", dqf, kf)
              + torch.einsum("blhd,bshd->bhls", qf, dkf)) * scale
        p = torch.softmax(s, dim=-1)
        dp = p * (ds - (p * ds).sum(-1, keepdim=True))
        o[:, i:i + step] = torch.einsum("bhls,bshd->blhd", p, vf).to(o.dtype)
        do[:, i:i + step] = (torch.einsum("bhls,bshd->blhd", dp, vf)
                             + torch.einsum("bhls,bshd->blhd", p, dvf)).to(o.dtype)
    return o, do


# --------------------------------------------------------------------------
# Differential attention: heads 2j and 2j + 1 are a pair whose values lie side by side,
# o = (softmax(q_2j k_2j^T) - lam_j softmax(q_2j+1 k_2j+1^T)) [v_2j | v_2j+1]
# --------------------------------------------------------------------------
def _pair_maps(t: Tensor) -> Tensor:
    """(b, l, 2H, d) -> (b, l, H, 2, d): the two heads of a pair"""
    return t.reshape(*t.shape[:2], t.shape[2] // 2, 2, t.shape[3])


def diff_attention(q: Tensor, k: Tensor, v: Tensor, lam: Tensor, scale: Optional[float] = None) -> Tensor:
    """(b, l, 2H, d) tensors, lam (H,) or one weight for all; einsum form, so that forward- and
    reverse-mode AD both work."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    up = lambda t: t if t.dtype == torch.float64 else t.float()
    qp, kp = _pair_maps(up(q)), _pair_maps(up(k))
    vp = up(v).reshape(*v.shape[:2], v.shape[2] // 2, 2 * v.shape[3])
    p = torch.softmax(torch.einsum("blhmd,bshmd->bhmls", qp, kp) * scale, dim=-1)
    w = up(lam).expand(v.shape[2] // 2)[None, :, None, None]
    # each map times V first: flat maps are nearly equal, and their difference would be rounded
    o = torch.einsum("bhmls,bshd->bhmld", p, vp)
    o = o[:, :, 0] - w * o[:, :, 1]
    return o.transpose(1, 2).reshape(v.shape).to(v.dtype)


@torch.no_grad()
def diff_attention_jvp(q: Tensor, k: Tensor, v: Tensor, lam: Tensor, dq: Tensor, dk: Tensor, dv: Tensor,
                       scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """(o, do); the weights carry no tangent."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    up = lambda t: t if t.dtype == torch.float64 else t.float()
    qp, kp, dqp, dkp = (_pair_maps(up(t)) for t in (q, k, dq, dk))
    wide = lambda t: up(t).reshape(*t.shape[:2], t.shape[2] // 2, 2 * t.shape[3])
    vp, dvp = wide(v), wide(dv)
    score = lambda a, b: torch.einsum("blhmd,bshmd->bhmls", a, b) * scale
    p = torch.softmax(score(qp, kp), dim=-1)
    ds = score(dqp, kp) + score(qp, dkp)
    t = p * (ds - (p * ds).sum(-1, keepdim=True))
    w = up(lam).expand(v.shape[2] // 2)[None, :, None, None]
    prod = lambda a, b: torch.einsum("bhmls,bshd->bhmld", a, b)
    back = lambda z: (z[:, :, 0] - w * z[:, :, 1]).transpose(1, 2).reshape(v.shape).to(v.dtype)
    return back(prod(p, vp)), back(prod(t, vp) + prod(p, dvp))


# --------------------------------------------------------------------------
# Norms around a branch: x = r res + gate post y / rms(y),  n = pre x / rms(x)
# --------------------------------------------------------------------------
def norm_add_norm(res: Optional[Tensor], y: Tensor, post: Tensor, gate: Tensor, eps: float,
                  res_scale: Optional[Tensor] = None, pre: Optional[Tensor] = None
                  ) -> Tuple[Tensor, Optional[Tensor]]:
    """(x, n or None) in 32 bits or more, unrounded."""
    up = lambda t: t if t is None or t.dtype == torch.float64 else t.float()
    unit = lambda t: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps)
    x = unit(up(y)) * (up(gate) * up(post))
    if res is not None:
        x = x + (up(res) if res_scale is None else up(res) * up(res_scale))
    return x, None if pre is None else unit(x) * up(pre)


@torch.no_grad()
def norm_add_norm_jvp(res: Optional[Tensor], dres: Optional[Tensor], y: Tensor, dy: Tensor, post: Tensor,
                      gate: Tensor, eps: float, res_scale: Optional[Tensor] = None, pre: Optional[Tensor] = None
                      ) -> Tuple[Tensor, Optional[Tensor]]:
    """(dx, dn or None): parameters carry no tangent; without ``dres`` the residual stands still."""
    up = lambda t: t if t is None or t.dtype == torch.float64 else t.float()

    def unit_jvp(t, dt):
        r = torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps)
        return r * (dt - t * r * r * (t * dt).mean(-1, keepdim=True))
    dx = unit_jvp(up(y), up(dy)) * (up(gate) * up(post))
    if dres is not None:
        dx = dx + (up(dres) if res_scale is None else up(dres) * up(res_scale))
    if pre is None:
        return dx, None
    x, _ = norm_add_norm(res, y, post, gate, eps, res_scale)
    return dx, unit_jvp(x, dx) * up(pre)


# --------------------------------------------------------------------------
# Attention residual (Kimi-style per-token softmax over residual history)
# --------------------------------------------------------------------------
def attn_res(cands: Sequence[Tensor], w: Tensor, eps: float) -> Tensor:
    """cands: J tensors (..., d), the LAST one is the current prefix sum.
    w: (d,) fused score direction (norm gain * projection weight)."""
    v = torch.stack([c.float() for c in cands], dim=-2)          # (..., J, d)
    r = torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + eps)
    s = ((v * r) * w.float()).sum(-1)                             # (..., J)
    p = torch.softmax(s, dim=-1)
    return (p.unsqueeze(-1) * v).sum(-2).to(cands[-1].dtype)


@torch.no_grad()
def attn_res_jvp(cands: Sequence[Tensor], dcands: Sequence[Tensor], w: Tensor,
                 eps: float) -> Tuple[Tensor, Tensor]:
    v = torch.stack([c.float() for c in cands], dim=-2)
    dv = torch.stack([c.float() for c in dcands], dim=-2)
    d = v.shape[-1]
    wf = w.float()
    r = torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + eps)       # (..., J, 1)
    vw = (v * wf).sum(-1, keepdim=True)
    dvw = (dv * wf).sum(-1, keepdim=True)
    vdv = (v * dv).sum(-1, keepdim=True) / d
    s = (r * vw).squeeze(-1)
    ds = (r * dvw - r.pow(3) * vw * vdv).squeeze(-1)
    p = torch.softmax(s, dim=-1)
    dp = p * (ds - (p * ds).sum(-1, keepdim=True))
    out = (p.unsqueeze(-1) * v).sum(-2)
    dout = (dp.unsqueeze(-1) * v).sum(-2) + (p.unsqueeze(-1) * dv).sum(-2)
    return out.to(cands[-1].dtype), dout.to(dcands[-1].dtype)


# --------------------------------------------------------------------------
# Newton-Schulz (used by the optimizer tests as the oracle of the kernel)
# --------------------------------------------------------------------------
def newton_schulz(G: Tensor, coeffs: Tuple[float, float, float], steps: int = 5,
                  eps: float = 1e-7, dtype: Optional[torch.dtype] = None) -> Tensor:
    a, b, c = coeffs
    X = G.to(dtype or torch.float32)
    X = X / (X.norm() + eps)
    tr = G.shape[0] > G.shape[1]
    if tr:
        X = X.T
    for _ in range(steps):
        A = X @ X.T
        B = b * A + c * (A @ A)
        X = a * X + B @ X
    return X.T if tr else X


# --------------------------------------------------------------------------
# Activations in 8 bits (``ops/act8.py``, ``csrc/act8.cuh``)
# --------------------------------------------------------------------------
def store8(x: Tensor) -> Tuple[Tensor, Tensor]:
    """(codes (rows, pitch) int8, steps (rows, spitch) uint8) of a (rows, C) tensor: for each 32
    channels a power of two 2^(s-127) so that the largest of them is 64 to 127 steps (s = 255:
    a NaN or an infinity among them); pitches rounded up to 32 channels and 4 groups."""
    rows, C = x.shape
    G = -(-C // 32)
    g = x.new_zeros(rows, G * 32, dtype=torch.float32)
    g[:, :C] = x
    g = g.view(rows, G, 32)
    amax = g.abs().amax(-1)
    s = ((amax.view(torch.int32) + 0x10000) >> 23) - 6
    s = s.clamp(0, 248)
    inv = ((254 - s) << 23).view(torch.float32)
    bad = ~torch.isfinite(amax)
    codes = torch.round(g * inv[..., None]).clamp(-127, 127).masked_fill(bad[..., None], 0)
    steps = torch.zeros(rows, (G + 3) // 4 * 4, dtype=torch.uint8, device=x.device)
    steps[:, :G] = s.masked_fill(bad, 255).to(torch.uint8)
    return codes.to(torch.int8).view(rows, G * 32), steps


def values8(codes: Tensor, steps: Tensor, C: int) -> Tensor:
    """fp32 (rows, C) values code * 2^(s-127) of ``store8``'s outputs (s = 255: NaN)."""
    rows, pitch = codes.shape
    s = steps[:, :pitch // 32].to(torch.int32)
    bits = torch.where(s == 0, 0x00400000, torch.where(s == 255, 0x7fc00000, s << 23)).to(torch.int32)
    step = bits.view(torch.float32)
    return (codes.view(rows, pitch // 32, 32).float() * step[..., None]).view(rows, pitch)[:, :C]


def situ_mul_grad(gate: Tensor, up: Tensor, gout: Tensor, beta: float, linear_beta: Optional[float]
                  ) -> Tuple[Tensor, Tensor, Tensor]:
    """(d gate, d up, y) of y = situ_mul(gate, up) for the output gradient ``gout``, in fp32."""
    g, u, go = gate.float(), up.float(), gout.float()
    th, sg = torch.tanh(g / beta), torch.sigmoid(g)
    a = beta * th * sg
    da = (1 - th * th) * sg + a * (1 - sg)
    if linear_beta is None:
        up_, dup = u, torch.ones_like(u)
    else:
        tu = torch.tanh(u / linear_beta)
        up_, dup = linear_beta * tu, 1 - tu * tu
    return go * da * up_, go * a * dup, a * up_


def attention_grad(q: Tensor, k: Tensor, v: Tensor, o: Tensor, lse: Tensor, go: Tensor,
                   scale: Optional[float] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """(dq, dk, dv) in fp32 of softmax attention on (B, L, H, d) tensors; the probabilities are
    recomputed from the scores and ``lse`` (B, H, L)."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    q, k, v, o, go = (t.float().transpose(1, 2) for t in (q, k, v, o, go))
    p = torch.exp(q @ k.transpose(-1, -2) * scale - lse[..., None])
    ds = p * (go @ v.transpose(-1, -2) - (go * o).sum(-1, keepdim=True))
    out = (ds @ k * scale, ds.transpose(-1, -2) @ q * scale, p.transpose(-1, -2) @ go)
    return tuple(t.transpose(1, 2) for t in out)
