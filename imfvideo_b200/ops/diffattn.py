"""Differential attention on the sm_100a kernels (``csrc/attn_diff_fwd.cu``, ``csrc/attn_diff_bwd.cu``).

Heads 2j and 2j + 1 of q, k, v (B, L, 2H, 64) are a pair.  Both heads' values lie side by side, and the
second softmax map is subtracted with the pair's learned weight:

    A_m = softmax(scale q_m k_m^T),  V = [v_2j | v_2j+1],  o = (A_1 - lam_j A_2) V

so the tensors are those of ordinary attention with 2H heads and nothing is copied to form pairs.
``ops.dual.diff_attention`` is the entry point for models (dual numbers, any device);
``diff_attn_fwd`` / ``diff_attn_bwd`` are the launches.  bf16, head_dim 64, any length from one token on,
any number of pairs; lam is fp32 or bf16 and its gradient has its type.  Launches go to the current
stream of the tensors' device; workspaces belong to the call.  The reference has no such attention.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import cuda as _cuda
from .act8 import _apart, _elsewhere, _in_one_place, _new, _places, _same_device, _span
from .dual import Dual

Tensor = torch.Tensor
BF16, F32 = torch.bfloat16, torch.float32
HEAD_DIM = 64
_KERNELS = None


def _kernels():
    """``ops.kernels`` with the argument types of this module's launchers set (loads the library)."""
    global _KERNELS
    if _KERNELS is None:
        if not _cuda.available():
            raise RuntimeError("differential attention on a GPU needs the kernel library")
        from . import kernels as K

        vp, ci, cl, i64, cf = (ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_int64,
                               ctypes.c_float)
        lib = K._lib
        for name, n in (("imf_attn_diff_fwd_scratch_bytes", 4), ("imf_attn_diff_bwd_scratch_bytes", 3)):
            getattr(lib, name).restype = cl
            getattr(lib, name).argtypes = [ci] * n
        lib.imf_attn_diff_fwd.restype = ci
        lib.imf_attn_diff_fwd.argtypes = [vp] * 7 + [i64, ci] + [vp] * 5 + [ci] * 3 + [vp, vp, cf, vp, cl, vp, vp]
        lib.imf_attn_diff_bwd.restype = ci
        lib.imf_attn_diff_bwd.argtypes = [vp] * 9 + [i64, ci] + [vp] * 4 + [ci] * 3 + [vp] * 4 + [cf, vp, cl, ci, vp, vp]
        _KERNELS = K
    return _KERNELS


def _check(what: str, shape, lam: Tensor, scale: Optional[float], names: str, *tensors) -> Tuple[torch.device, float]:
    if len(shape) != 4 or shape[3] != HEAD_DIM or shape[2] % 2:
        raise ValueError(f"{what} takes (B, L, an even number of heads, {HEAD_DIM}), not {tuple(shape)}")
    dev = lam.device
    for i, t in enumerate(tensors):
        if t is not None and (t.dtype is not BF16 or t.shape != shape or t.device != dev):
            raise ValueError(f"{what}: {names.split()[i]} is {t.dtype} {tuple(t.shape)} on {t.device}, bf16 {tuple(shape)} on "
                             f"{dev} (where lam is) expected")
    if (lam.dtype is not F32 and lam.dtype is not BF16) or lam.dim() != 1 or lam.shape[0] != shape[2] // 2:
        raise ValueError(f"{what}: lam is {lam.dtype} {tuple(lam.shape)}, fp32 or bf16 ({shape[2] // 2},) expected")
    scale = HEAD_DIM ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"{what}: scale {scale} is not a positive number between 1e-30 and 1e30")
    return dev, scale


@lru_cache(maxsize=64)
def _rows(shape: Tuple[int, ...]):
    """(batch, row, head) strides of a contiguous tensor, as a tuple and for one and for six tensors as the
    launchers take them."""
    B, L, H, D = shape
    row = (L * H * D, H * D, D)
    return row, (ctypes.c_int64 * 3)(*row), (ctypes.c_int64 * 18)(*row * 6)


@lru_cache(maxsize=64)
def _scratch_bytes(which: str, device: int, *sizes: int) -> int:
    """Of a launch on the current device, whose index is ``device``: they go by its SMs."""
    return getattr(_kernels()._lib, f"imf_attn_diff_{which}_scratch_bytes")(*sizes)


def _operands(tensors, row, six):
    """(the tensors, or copies of those without 16-byte aligned rows; their strides as the launchers take
    them).  Strides of single dimensions are replaced: no address depends on them."""
    out, strides = [], None
    for i, t in enumerate(tensors):
        st = row
        if not t.is_contiguous():
            s = [x if n > 1 else r for n, x, r in zip(t.shape, t.stride(), row)]
            if t.stride(3) == 1 and t.data_ptr() % 16 == 0 and not any(x % 8 or x == 0 for x in s):
                st = s
            else:
                t = t.contiguous()             # a broadcast, transposed or unaligned tensor
        if t.data_ptr() % 16:
            t = t.clone()
        out.append(t)
        if st is not row:
            strides = strides or list(row) * 6
            strides[3 * i:3 * i + 3] = st
    return out, six if strides is None else (ctypes.c_int64 * 18)(*strides)


def _like(t: Tensor) -> Tensor:
    """An uninitialised contiguous tensor of the same shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else _new(t.shape, t.dtype, t.device)


def _meet(a: Tensor, b: Tensor) -> bool:
    """Whether the stretches of memory from the first to the last byte of two tensors meet."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def diff_attn_fwd(q: Tensor, k: Tensor, v: Tensor, lam: Tensor, dq: Optional[Tensor] = None,
                  dk: Optional[Tensor] = None, dv: Optional[Tensor] = None, scale: Optional[float] = None,
                  need_bwd: bool = True) -> Tuple[Tensor, Optional[Tensor], tuple]:
    """(o, do | None, saved) of (B, L, 2H, 64) bf16 CUDA tensors at any strides; lam (H,).  With tangents
    dq, dk, dv (all or none) also do.  ``need_bwd``: saved is what ``diff_attn_bwd`` takes, O_2 in bf16, the
    bytes that o and O_2 lost when they were rounded (int8, o's shape with twice the channels) and the log-sum-exp
    (B, 2H, L) of both maps; otherwise it is empty."""
    shape, tang = q.shape, dq is not None
    if (dk is None) == tang or (dv is None) == tang:
        raise ValueError("diff_attn_fwd: tangents of q, k and v come together")
    dev, scale = _check("diff_attn_fwd", shape, lam, scale, "q k v dq dk dv", q, k, v, dq, dk, dv)
    if dev.type != "cuda":
        raise ValueError("diff_attn_fwd launches on a GPU; dual.diff_attention also takes CPU tensors")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return diff_attn_fwd(q, k, v, lam, dq, dk, dv, scale, need_bwd)
    B, L, H2, D = shape
    o = _like(q)
    do = _like(q) if tang else None
    o2, low, lse = saved = (_like(q), _new((B, L, H2, 2 * D), torch.int8, dev), _new((B, H2, L), F32, dev)) if need_bwd else (None,) * 3
    saved = saved if need_bwd else ()
    if 0 in shape:
        return o, do, saved
    K = _kernels()
    row, row3, row18 = _rows(shape)
    ts, strides = _operands((q, k, v, dq, dk, dv) if tang else (q, k, v), row, row18)
    ptr = [t.data_ptr() for t in ts]
    nscr = _scratch_bytes("fwd", dev.index, B, L, H2 // 2, tang)
    scr = _new(nscr, torch.uint8, dev) if nscr else None
    p = K._ptr
    K._check(K._lib.imf_attn_diff_fwd(
        *(ptr if tang else (*ptr, None, None, None)), lam.data_ptr(), lam.stride(0), lam.dtype is BF16, o.data_ptr(), p(do),
        p(o2), p(low), p(lse), B, L, H2 // 2, strides, row3, scale, p(scr), nscr,
        K.status_word(dev).data_ptr(), K._stream()), "imf_attn_diff_fwd")
    K.LAUNCHES.count += 1
    return o, do, saved


def diff_attn_bwd(q: Tensor, k: Tensor, v: Tensor, lam: Tensor, o: Tensor, saved: tuple, go: Tensor,
                  scale: Optional[float] = None, gv_out: Optional[Tensor] = None
                  ) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """(dq, dk, dv, dlam) from what ``diff_attn_fwd`` returned and the output gradient ``go``.  ``gv_out``
    takes dv (16-byte aligned rows, no two elements in one place, apart from q, k, v, lam and go; what the forward
    pass returned is read before dv is written), as in ``kernels.attn_bwd``, whose fixed-order mode holds here
    too."""
    shape = q.shape
    o2, low, lse = saved
    dev, scale = _check("diff_attn_bwd", shape, lam, scale, "q k v o o2 go gv_out", q, k, v, o, o2, go, gv_out)
    _same_device("diff_attn_bwd", q, low, lse)
    if dev.type != "cuda":
        raise ValueError("diff_attn_bwd launches on a GPU; dual.diff_attention also takes CPU tensors")
    B, L, H2, D = shape
    if lse.dtype is not F32 or lse.shape != (B, H2, L) or not lse.is_contiguous():
        raise ValueError(f"diff_attn_bwd: lse has to be contiguous fp32 {(B, H2, L)}")
    if low.dtype is not torch.int8 or low.shape != (B, L, H2, 2 * D) or not (low.is_contiguous() and o2.is_contiguous()):
        raise ValueError("diff_attn_bwd: saved has to be what diff_attn_fwd returned")
    row = _rows(shape)[0]
    dv_strides = None
    if gv_out is not None and 0 not in shape:
        st = [s if n > 1 else r for n, s, r in zip(shape, gv_out.stride(), row)]
        dv_strides = (ctypes.c_int64 * 3)(*st)
        if gv_out.stride(3) != 1 or gv_out.data_ptr() % 16 or any(s % 8 for s in st):
            raise ValueError("diff_attn_bwd: the dv output needs 16-byte aligned rows")
        if not _apart(*_places(gv_out)):
            raise ValueError("diff_attn_bwd: no two elements of the dv output in one place")
        if any(_in_one_place(gv_out, t) if _apart(*_places(t)) else _meet(gv_out, t) for t in (q, k, v, lam, go)):
            raise ValueError("diff_attn_bwd: the dv output lies over an input")
    return _backward(q, k, v, lam, o, saved, go, scale, gv_out, dv_strides)


def _backward(q, k, v, lam, o, saved, go, scale, gv_out, dv_strides):
    """``diff_attn_bwd`` of checked tensors; dv_strides None: those of a contiguous one."""
    shape, dev = q.shape, q.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _backward(q, k, v, lam, o, saved, go, scale, gv_out, dv_strides)
    B, L, H2, D = shape
    o2, low, lse = saved
    dq, dk = _like(o2), _like(o2)
    dv = _like(o2) if gv_out is None else gv_out
    dlam = _new((H2 // 2,), lam.dtype, dev)
    if 0 in shape:
        return dq, dk, dv, dlam.zero_()
    K = _kernels()
    row, row3, row18 = _rows(shape)
    (q_, k_, v_, g_), strides = _operands((q, k, v, go), row, row18)
    o = o.contiguous()
    nscr = _scratch_bytes("bwd", dev.index, B, L, H2 // 2)
    scr = _new(nscr, torch.uint8, dev)
    K._check(K._lib.imf_attn_diff_bwd(
        q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), o.data_ptr(), o2.data_ptr(), low.data_ptr(), g_.data_ptr(),
        lse.data_ptr(), lam.data_ptr(), lam.stride(0), lam.dtype is BF16, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
        dlam.data_ptr(), B, L, H2 // 2, strides, row3, row3, dv_strides or row3, scale, scr.data_ptr(), nscr,
        bool(K.DETERMINISTIC), K.status_word(dev).data_ptr(), K._stream()), "imf_attn_diff_bwd")
    K.LAUNCHES.count += 3
    return dq, dk, dv, dlam


class _DiffAttnFn(torch.autograd.Function):
    """o and the detached tangent do; reverse mode through the primal only."""

    @staticmethod
    def forward(ctx, q, k, v, lam, dq, dk, dv, scale):
        need_bwd = any(ctx.needs_input_grad[:4])
        o, do, saved = diff_attn_fwd(q, k, v, lam, dq, dk, dv, scale, need_bwd)
        if need_bwd:
            ctx.save_for_backward(q, k, v, lam, o, *saved)
            ctx.scale = HEAD_DIM ** -0.5 if scale is None else float(scale)
            ctx.set_materialize_grads(False)
        if do is not None:
            ctx.mark_non_differentiable(do)
        return o, do

    @staticmethod
    @once_differentiable
    def backward(ctx, go, _gdo):
        if go is None:
            return (None,) * 8
        # (the forward pass has checked these, autograd gives a gradient of o's shape and type)
        q, k, v, lam, o, *saved = ctx.saved_tensors
        return (*_backward(q, k, v, lam, o, saved, go, ctx.scale, None, None), None, None, None, None)


def diff_attention_dual(q: Dual, k: Dual, v: Dual, lam: Tensor, scale: Optional[float] = None) -> Dual:
    """``ops.dual.diff_attention`` on CUDA tensors; lam (H,).  Tangents of another type are rounded to their primal's:
    the tensor core multiplies both with the same operands."""
    t = (q.t, k.t, v.t)
    if any(x is not None for x in t):
        t = tuple(torch.zeros_like(p.p) if x is None else x.to(p.p.dtype) for p, x in zip((q, k, v), t))
    if torch.is_grad_enabled() and (q.p.requires_grad or k.p.requires_grad or v.p.requires_grad or lam.requires_grad):
        o, do = _DiffAttnFn.apply(q.p, k.p, v.p, lam, *t, scale)
        return Dual(o, do)
    return Dual(*diff_attn_fwd(q.p, k.p, v.p, lam, *t, scale, need_bwd=False)[:2])
