"""Differential attention plug-in (``model.attn_impl = "diff_jvp"``): heads 2j and 2j + 1 are a pair whose
second softmax map is subtracted with a learned weight, both multiplying the pair's values side by side

    o = (softmax(q_2j k_2j^T / sqrt(d)) - lam_j softmax(q_2j+1 k_2j+1^T / sqrt(d))) [v_2j | v_2j+1]

What both maps give to tokens that matter to neither cancels.  Projections, shapes and checkpoints are those of
dense attention with the same number of heads, plus one vector of weights a block.  The reference has no such
attention; the module is a plug-in like its SLA2 family (reference ``models/sla2_attention.py:23-61``)."""

from __future__ import annotations

import warnings
from typing import Optional

import torch
import torch.nn as nn

from ..ops import dual as D
from ..ops.dual import Dual

Tensor = torch.Tensor


class DiffAttentionImpl(nn.Module):
    """attn_impl with one weight for each pair of heads; (b, l, H, hd) duals or tensors in and out.  CUDA kernels
    take bf16 and head_dim 64, everything else the formulas."""

    def __init__(self, head_dim: int, seq_len: int, num_heads: int, lam_init: float = 0.5):
        super().__init__()
        if num_heads % 2:
            raise ValueError(f"differential attention pairs heads: {num_heads} is odd")
        maps = 4 * num_heads * seq_len ** 2                 # bytes of a batch entry's
        if head_dim != 64 and maps > 1 << 30:
            warnings.warn(f"differential attention has kernels for head_dim 64 only: with {head_dim} the formulas run, whose "
                          f"softmax maps take {maps / 1e9:.1f} GB a batch entry and tensor", stacklevel=2)
        self.head_dim = head_dim
        self.lam = nn.Parameter(torch.full((num_heads // 2,), float(lam_init)))

    def forward(self, q, k, v):
        plain = not isinstance(q, Dual)
        q, k, v = (D.lift(x) for x in (q, k, v))
        kernels = q.p.dtype == torch.bfloat16 and q.p.shape[-1] == 64
        out = D.diff_attention(q, k, v, self.lam, impl="auto" if kernels else "math")
        return out.p if plain else out


class DiffCore:
    """Attention core for ``ops.block``: the forward and backward kernels, with the pairs' weights as an input of the
    block's node."""

    def __init__(self, mod: DiffAttentionImpl):
        self.params = (mod.lam,)

    def fwd(self, q, k, v, dq, dk, dv, need_bwd: bool):
        from ..ops import diffattn as DA

        lam, = self.params
        o, do, saved = DA.diff_attn_fwd(q, k, v, lam, dq, dk, dv, need_bwd=need_bwd)
        return o, do, (lam, *saved)

    def bwd(self, q, k, v, o, saved, go, gv_out: Optional[Tensor] = None):
        from ..ops import diffattn as DA

        lam, *saved = saved
        return DA.diff_attn_bwd(q, k, v, lam, o, saved, go, gv_out=gv_out)


def _fused_core(self):
    """The core where the fused block can use it, else None."""
    if not self.lam.is_cuda or self.head_dim != 64 or self.lam.dtype != torch.float32:
        return None
    from ..ops import cuda as cu

    return DiffCore(self) if cu.available() else None


DiffAttentionImpl.fused_core = property(_fused_core)
