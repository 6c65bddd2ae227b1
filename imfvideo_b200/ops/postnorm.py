"""Norms around a block's branch on the sm_100a kernels (``csrc/rowops_postnorm.cu``):

    x = res_scale * res + gate * post * y / rms(y),    n = pre * x / rms(x)

``ops.dual.norm_add_norm`` is the entry point for models (dual numbers, any device);
``norm_add_norm_fwd`` / ``norm_add_norm_bwd`` are the launches.  Rows are all leading dimensions, fewer than
2^30; D a multiple of 8 up to 8,192; y and n bf16 or fp32 (one type), the residual stream and the learned vectors
fp32.  Launches go to the current stream of the tensors' device; workspaces belong to the call.  The
reference norms a branch's input only (reference ``models/imf_dit_video.py:909-972``).
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import cuda as _cuda
from .act8 import _elsewhere, _new
from .dual import Dual

Tensor = torch.Tensor
BF16, F32 = torch.bfloat16, torch.float32
MAX_WIDTH, MAX_ROWS = 8192, 1 << 30
_PTRS = ctypes.c_void_p * 18
_KERNELS = None


def _kernels():
    """``ops.kernels`` with the argument types of this module's launchers set (loads the library)."""
    global _KERNELS
    if _KERNELS is None:
        if not _cuda.available():
            raise RuntimeError("norm_add_norm on a GPU needs the kernel library")
        from . import kernels as K

        vp, ci = ctypes.c_void_p, ctypes.c_int
        K._lib.imf_norm_add_norm_grid.restype = ci
        K._lib.imf_norm_add_norm_grid.argtypes = [ci, ci]
        K._lib.imf_norm_add_norm.restype = ci
        K._lib.imf_norm_add_norm.argtypes = [vp, ci, ci, ctypes.c_float, ci, ci, vp, vp]
        _KERNELS = K
    return _KERNELS


def supported(y: Tensor, x_dtype: torch.dtype, n_dtype: Optional[torch.dtype], post: Tensor, gate: Tensor,
              res_scale: Optional[Tensor], pre: Optional[Tensor], dy: Optional[Tensor] = None,
              dres: Optional[Tensor] = None) -> bool:
    """Whether the kernels take these types and this width."""
    yt, D = y.dtype, y.shape[-1] if y.dim() else 0
    return ((yt is BF16 or yt is F32) and x_dtype is F32 and (n_dtype is None or n_dtype is yt) and D % 8 == 0
            and 0 < D <= MAX_WIDTH and post.dtype is F32 and gate.dtype is F32
            and (res_scale is None or res_scale.dtype is F32) and (pre is None or pre.dtype is F32)
            and (dy is None or dy.dtype is yt) and (dres is None or dres.dtype is F32))


def _aligned(t: Optional[Tensor]) -> Optional[Tensor]:
    """Contiguous, 16-byte aligned rows of a tensor (the tensor itself where it has them)."""
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _prepare(what: str, y, vectors, streams, likes):
    """Checks and aligns the operands: learned ``vectors`` and fp32 ``streams`` and others of y's type (``likes``),
    of y's shape."""
    shape, yt, dev = y.shape, y.dtype, y.device
    if (yt is not BF16 and yt is not F32) or not shape or shape[-1] % 8 or not 0 < shape[-1] <= MAX_WIDTH or \
            y.numel() // shape[-1] >= MAX_ROWS:
        raise ValueError(f"{what}: y bf16 or fp32 with a multiple of 8 up to {MAX_WIDTH} channels and fewer than 2^30 "
                         f"rows, not {yt} {tuple(shape)}")
    for want, dtype, ts in ((shape[-1:], F32, vectors), (shape, F32, streams), (shape, yt, likes)):
        for t in ts:
            if t is not None and (t.dtype is not dtype or t.shape != want or t.device != dev):
                raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)} on {t.device} where {dtype} {tuple(want)} on {dev} is expected")
    if dev.type != "cuda":
        raise ValueError(f"{what} launches on a GPU; dual.norm_add_norm also takes CPU tensors")
    return [_aligned(t) for t in (y, *vectors, *streams, *likes)]


def _like(y: Tensor, dtype: torch.dtype) -> Tensor:
    """An uninitialised tensor of a contiguous one's shape."""
    return torch.empty_like(y) if y.dtype is dtype else torch.empty_like(y, dtype=dtype)


def norm_add_norm_fwd(res: Optional[Tensor], y: Tensor, post: Tensor, gate: Tensor, eps: float,
                      res_scale: Optional[Tensor] = None, pre: Optional[Tensor] = None,
                      dres: Optional[Tensor] = None, dy: Optional[Tensor] = None
                      ) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor], Optional[Tensor]]:
    """(x, n | None, dx | None, dn | None) of CUDA tensors; with ``dy`` the tangents too (``dres`` None: the
    residual stands still)."""
    what = "norm_add_norm_fwd"
    if (dres is not None and (dy is None or res is None)) or (res_scale is not None and res is None):
        raise ValueError(f"{what}: dres without dy or res, or res_scale without res")
    y, post, gate, res_scale, pre, res, dres, dy = _prepare(what, y, (post, gate, res_scale, pre), (res, dres), (dy,))
    dev, yt = y.device, y.dtype
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return norm_add_norm_fwd(res, y, post, gate, eps, res_scale, pre, dres, dy)
    x = _like(y, F32)
    n = None if pre is None else torch.empty_like(y)
    dx = None if dy is None else _like(y, F32)
    dn = None if dy is None or pre is None else torch.empty_like(y)
    D = y.shape[-1]
    rows = y.numel() // D
    if rows:
        K = _kernels()
        ptrs = _PTRS(*[0 if t is None else t.data_ptr() for t in (res, dres, y, dy, post, gate, res_scale, pre, x, dx, n, dn)])
        K._check(K._lib.imf_norm_add_norm(ptrs, rows, D, eps, yt is F32, dy is not None,
                                          K.status_word(dev).data_ptr(), K._stream()), "imf_norm_add_norm")
        K.LAUNCHES.count += 1
    return x, n, dx, dn


def norm_add_norm_bwd(res: Optional[Tensor], y: Tensor, post: Tensor, gate: Tensor, eps: float,
                      res_scale: Optional[Tensor], pre: Optional[Tensor], gx: Optional[Tensor], gn: Optional[Tensor],
                      want_g_res: bool = True, raw: bool = False):
    """(g_res | None, g_y, g_pre | None, g_r | None, g_gate, g_post) from the gradients of x and n (None: zero;
    ``gn`` together with ``pre``).  With ``raw`` the last four are replaced by the [g, 4, D] buffer of their
    partial sums (columns pre, r, gate, post) for a later ``rowops.ColSums`` reduction; columns of vectors that
    are not there are not written.  g_res may be ``gx`` itself."""
    what = "norm_add_norm_bwd"
    if (gn is None) != (pre is None) or (res_scale is not None and res is None):
        raise ValueError(f"{what}: gn and pre come together, res_scale with res")
    y, post, gate, res_scale, pre, res, gx, gn = _prepare(what, y, (post, gate, res_scale, pre), (res, gx), (gn,))
    return _backward(res, y, post, gate, eps, res_scale, pre, gx, gn, want_g_res, raw)


def _backward(res, y, post, gate, eps, res_scale, pre, gx, gn, want_g_res, raw):
    """``norm_add_norm_bwd`` of checked and aligned tensors."""
    dev, yt, D = y.device, y.dtype, y.shape[-1]
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _backward(res, y, post, gate, eps, res_scale, pre, gx, gn, want_g_res, raw)
    rows = y.numel() // D
    want_g_res = want_g_res and res is not None
    # without a second norm and a scale the residual's gradient is x's
    passed = want_g_res and pre is None and res_scale is None and gx is not None
    g_res = gx if passed else _like(y, F32) if want_g_res else None
    g_y = torch.empty_like(y)
    if rows:
        K = _kernels()
        part = _new((_partial_rows(rows, D), 4, D), F32, dev)
        sums = None if raw else _new((4, D), F32, dev)
        ptrs = _PTRS(*[0 if t is None else t.data_ptr() for t in (
            res, None, y, None, post, gate, res_scale, pre, None, None, None, None, gx, gn, None if passed else g_res, g_y,
            part, sums)])
        K._check(K._lib.imf_norm_add_norm(ptrs, rows, D, eps, yt is F32, 2, K.status_word(dev).data_ptr(), K._stream()),
                 "imf_norm_add_norm")
        K.LAUNCHES.count += 1 if raw else 2
    else:
        part, sums = torch.zeros(1, 4, D, dtype=F32, device=dev), torch.zeros(4, D, dtype=F32, device=dev)
    if raw:
        return g_res, g_y, part
    g_pre, g_r, g_gate, g_post = sums.unbind(0)
    return g_res, g_y, None if pre is None else g_pre, None if res_scale is None else g_r, g_gate, g_post


@lru_cache(maxsize=64)
def _partial_rows(rows: int, D: int) -> int:
    return _kernels()._lib.imf_norm_add_norm_grid(rows, D)


class _NormAddNormFn(torch.autograd.Function):
    """x, n and their detached tangents; reverse mode through the primal only."""

    @staticmethod
    def forward(ctx, res, y, post, gate, res_scale, pre, dres, dy, eps):
        x, n, dx, dn = norm_add_norm_fwd(res, y, post, gate, eps, res_scale, pre, dres, dy)
        ctx.set_materialize_grads(False)
        if any(ctx.needs_input_grad[:6]):
            ctx.save_for_backward(res, y, post, gate, res_scale, pre)
            ctx.eps = eps
        if dx is not None:
            ctx.mark_non_differentiable(*((dx,) if dn is None else (dx, dn)))
        return x, n, dx, dn

    @staticmethod
    @once_differentiable
    def backward(ctx, gx, gn, _gdx, _gdn):
        if gx is None and gn is None:
            return (None,) * 9
        # (the forward pass has checked these, autograd gives gradients of the outputs' shapes and types)
        res, y, post, gate, res_scale, pre = map(_aligned, ctx.saved_tensors)
        gn = None if pre is None else torch.zeros_like(y) if gn is None else _aligned(gn)
        g_res, g_y, g_pre, g_r, g_gate, g_post = _backward(
            res, y, post, gate, ctx.eps, res_scale, pre, _aligned(gx), gn, ctx.needs_input_grad[0], False)
        return g_res, g_y, g_post, g_gate, g_r, g_pre, None, None, None


def norm_add_norm_dual(res: Optional[Dual], y: Dual, post: Tensor, gate: Tensor, eps: float,
                       res_scale: Optional[Tensor], pre: Optional[Tensor]):
    """``ops.dual.norm_add_norm`` on CUDA tensors of the kernels' types."""
    rp, rt = (None, None) if res is None else res
    dy = y.t
    if dy is None and rt is not None:
        dy = torch.zeros_like(y.p)
    if torch.is_grad_enabled() and (y.p.requires_grad or post.requires_grad or gate.requires_grad or
                                    any(t is not None and t.requires_grad for t in (rp, res_scale, pre))):
        x, n, dx, dn = _NormAddNormFn.apply(rp, y.p, post, gate, res_scale, pre, rt, dy, eps)
    else:
        x, n, dx, dn = norm_add_norm_fwd(rp, y.p, post, gate, eps, res_scale, pre, rt, dy)
    return Dual(x, dx), None if n is None else Dual(n, dn)
