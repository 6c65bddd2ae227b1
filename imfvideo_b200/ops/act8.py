"""Activations kept in 8 bits for the backward pass, and the backward operators that read them
(``csrc/act8.cu``, ``csrc/act8.cuh``).

What a training step keeps of every transformer block is most of its memory.  ``store8`` writes
activations as one signed byte a channel and one step byte for each 32 channels of a row; the value
is code * 2^(step - 127), at most half a step off: 1/127.5 of the group's largest magnitude, or 2^-128
in groups below 2^-121 or so, and up to a step for fp32 above the largest bf16.  The step is a
power of two, so the values are exact in bf16 and the tensor cores multiply what was stored.  A
group that holds a NaN or an infinity reads as NaN throughout.

    packed = store8([x, y, z])                # one launch, one allocation
    x, y, z = restore8(packed)                # back to their types
    gemm_wgrad8(dy, packed[0])                # weight gradient dY^T X
    situ_bwd8(gu8, gout, beta, lbeta)         # gated activation, backward (and forward again)
    attn_bwd8(q8, k8, v8, o8, lse, go)        # dense attention, probabilities recomputed

``model.act_store = "int8"`` keeps the activations of the fused blocks this way
(``ops/block.py``); blocks off the fused path (CPU, fp32) keep theirs as they are.  These are
operators of a backward pass: none of them is differentiable.  CPU tensors take the formulas of
``ops/reference.py``.  All launches go to the current stream of the tensors' device; workspaces
belong to the call.  There is no counterpart in the reference, which recomputes blocks instead
(reference ``models/imf_dit_video.py:909-972``).
"""

from __future__ import annotations

import ctypes
import math
import struct
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import cuda as _cuda
from . import reference as ref

Tensor = torch.Tensor
BF16, F32 = torch.bfloat16, torch.float32
GROUP = 32
_F32_MIN, _F32_MAX = torch.finfo(F32).tiny, torch.finfo(F32).max
_MAX_RECS = 16                 # tensors a launch takes
# n records x, codes, steps, n0, n1, n2, s0, s1, s2, cols, fp32
_RECS = [struct.Struct("<" + 11 * n * "q") for n in range(_MAX_RECS + 1)]
_KERNELS = None


def _kernels():
    """``ops.kernels`` with the argument types of this module's launchers set (loads the library)."""
    global _KERNELS
    if _KERNELS is None:
        if not _cuda.available():
            raise RuntimeError("8-bit activations on a GPU need the kernel library")
        from . import kernels as K

        vp, ci, cl, i64, cf = (ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_int64,
                               ctypes.c_float)
        for name in ("imf_store8", "imf_restore8"):
            getattr(K._lib, name).restype = ci
            getattr(K._lib, name).argtypes = [vp, ci, vp]
        K._lib.imf_wgrad8_work.restype = i64
        K._lib.imf_wgrad8_work.argtypes = [ci] * 3 + [vp, i64]
        K._lib.imf_wgrad8.restype = ci
        K._lib.imf_wgrad8.argtypes = [vp, i64, vp, vp, ci, ci, ci, vp, i64, ci, vp, i64, vp, vp]
        K._lib.imf_attn_bwd8.restype = ci
        K._lib.imf_attn_bwd8.argtypes = [vp] * 10 + [ci] * 4 + [vp] * 4 + [cf, vp, cl, ci, vp, vp]
        K._lib.imf_situ_bwd8.restype = ci
        K._lib.imf_situ_bwd8.argtypes = [vp] * 5 + [cl, ci] + [i64] * 3 + [cf, cf, ci, vp]
        _KERNELS = K
    return _KERNELS


_PROTO: dict = {}


def _new(shape, dtype: torch.dtype, dev: torch.device) -> Tensor:
    """``torch.empty`` from an empty tensor of the device and type: a third of the host time less."""
    proto = _PROTO.get((dev, dtype))
    if proto is None:
        proto = _PROTO[dev, dtype] = torch.empty(0, dtype=dtype, device=dev)
    return proto.new_empty(shape)


def _pitches(cols: int) -> Tuple[int, int]:
    """Channels and groups that a row of codes and of steps is rounded up to."""
    groups = (cols + GROUP - 1) // GROUP
    return groups * GROUP, (groups + 3) // 4 * 4


class Packed8:
    """A tensor of ``shape`` in 8 bits: ``codes`` int8 (rows, channels rounded up to 32) and ``steps``
    uint8 (rows, groups rounded up to 4), rows being all leading dimensions; ``dtype`` is what
    ``restore8`` returns (bf16, or fp32 for a tensor that was fp32).  Of one ``store8`` call all
    share one buffer, which lives until the last of them is gone."""

    __slots__ = ("shape", "dtype", "rows", "cols", "device", "_codes", "_steps", "_arena", "_at")

    def __init__(self, codes: Tensor, steps: Tensor, shape: Sequence[int], dtype: torch.dtype = BF16):
        self.shape = shape = torch.Size(shape)
        if len(shape) < 1 or min(shape) < 0:
            raise ValueError(f"not the shape of an activation: {tuple(shape)}")
        if dtype is not BF16 and dtype is not F32:
            raise ValueError(f"8-bit activations are bf16 or fp32, not {dtype}")
        self.cols = cols = shape[-1]
        self.rows = rows = math.prod(shape[:-1])
        self.dtype, self.device = dtype, codes.device
        pitch, spitch = _pitches(cols)
        if codes.dtype is not torch.int8 or codes.shape != (rows, pitch) or not codes.is_contiguous():
            raise ValueError(f"codes of {tuple(shape)}: contiguous int8 ({rows}, {pitch}) expected, got "
                             f"{codes.dtype} {tuple(codes.shape)}")
        if steps.dtype is not torch.uint8 or steps.shape != (rows, spitch) or not steps.is_contiguous():
            raise ValueError(f"steps of {tuple(shape)}: contiguous uint8 ({rows}, {spitch}) expected, got "
                             f"{steps.dtype} {tuple(steps.shape)}")
        if steps.device != self.device:
            raise ValueError("codes and steps are on different devices")
        if codes.data_ptr() % 16 or steps.data_ptr() % 4:
            raise ValueError("codes need a 16-byte, steps a 4-byte aligned address")
        self._codes, self._steps, self._arena, self._at = codes, steps, None, None

    @classmethod
    def _in(cls, arena: Tensor, at: Tuple[int, int], shape, dtype, rows: int) -> "Packed8":
        """In the buffer ``arena`` at byte offsets ``at`` of codes and steps."""
        p = cls.__new__(cls)
        p.shape, p.dtype, p.device = shape, dtype, arena.device
        p.rows, p.cols = rows, shape[-1]
        p._codes = p._steps = None
        p._arena, p._at = arena, at
        return p

    @property
    def codes(self) -> Tensor:
        if self._codes is None:
            pitch, o = _pitches(self.cols)[0], self._at[0]
            self._codes = self._arena[o:o + self.rows * pitch].view(torch.int8).view(self.rows, pitch)
        return self._codes

    @property
    def steps(self) -> Tensor:
        if self._steps is None:
            spitch, o = _pitches(self.cols)[1], self._at[1]
            self._steps = self._arena[o:o + self.rows * spitch].view(self.rows, spitch)
        return self._steps

    def _ptrs(self) -> Tuple[int, int]:
        if self._arena is not None:
            base = self._arena.data_ptr()
            return base + self._at[0], base + self._at[1]
        return self._codes.data_ptr(), self._steps.data_ptr()

    @property
    def nbytes(self) -> int:
        return self.rows * sum(_pitches(self.cols))

    def view(self, *shape: int) -> "Packed8":
        """The same rows under other leading dimensions."""
        if not shape or shape[-1] != self.cols or math.prod(shape[:-1]) != self.rows or min(shape) < 0:
            raise ValueError(f"{tuple(self.shape)} cannot be seen as {tuple(shape)}")
        p = Packed8.__new__(Packed8)
        p.shape, p.dtype, p.device, p.rows, p.cols = torch.Size(shape), self.dtype, self.device, self.rows, self.cols
        p._codes, p._steps, p._arena, p._at = self._codes, self._steps, self._arena, self._at
        return p

    def restore(self) -> Tensor:
        return restore8(self)

    def __repr__(self) -> str:
        return f"Packed8({tuple(self.shape)}, {self.dtype}, {self.nbytes} bytes, {self.device})"


def buffer(ps: Sequence[Packed8]) -> Tensor:
    """The buffer that the tensors of one ``store8`` call share (what an autograd node saves)."""
    return ps[0]._arena


def layout(ps: Sequence[Packed8]) -> list:
    """Where in it they are; with the buffer, ``in_buffer`` makes them again."""
    return [(p._at, p.shape, p.dtype, p.rows) for p in ps]


def in_buffer(arena: Tensor, where: list) -> List[Packed8]:
    return [Packed8._in(arena, *w) for w in where]


def _row_dims(t: Tensor, rows: int) -> Optional[Tuple[int, ...]]:
    """(n0, n1, n2, s0, s1, s2) of a tensor's rows (all dimensions but the last, merged where the
    strides allow it), or None where more than three remain or the channels are not adjacent."""
    if t.is_contiguous():
        return 1, 1, rows, 0, 0, t.shape[-1]
    shape, strides = t.shape, t.stride()
    if shape[-1] > 1 and strides[-1] != 1:
        return None
    dims: List[List[int]] = []
    for n, s in zip(shape[:-1], strides[:-1]):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * s:
            dims[-1] = [dims[-1][0] * n, s]
        else:
            dims.append([n, s])
    if len(dims) > 3:
        return None
    dims = [[1, 0]] * (3 - len(dims)) + dims
    return tuple(d[0] for d in dims) + tuple(d[1] for d in dims)


def _places(t: Tensor) -> Tuple[List[Tuple[int, int]], int]:
    """((stride, n) of the dimensions that count but adjacent channels, smallest first; how many those are)."""
    dims = sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1)
    return (dims[1:], dims[0][1]) if dims and dims[0][0] == 1 else (dims, 1)


def _starts(dims: List[Tuple[int, int]]) -> Tensor:
    at = torch.zeros(1, dtype=torch.int64)
    for s, n in dims:
        at = (at[:, None] + torch.arange(n) * s).flatten()
    return at


def _apart(dims: List[Tuple[int, int]], run: int) -> bool:
    """Whether runs of ``run`` elements at these strides lie in different places."""
    reach = run
    for s, n in dims:
        if s < reach:
            break
        reach += s * (n - 1)
    else:
        return True
    return dims[0][0] > 0 and bool((_starts(dims).sort().values.diff() >= run).all())      # strides that interleave


def _span(t: Tensor) -> Tuple[int, int]:
    """First and last byte + 1 of a tensor."""
    at, n = t.data_ptr(), t.numel()
    if n and not t.is_contiguous():
        n = 1 + sum(s * (m - 1) for m, s in zip(t.shape, t.stride()))
    return at, at + n * t.element_size()


def _in_one_place(a: Tensor, b: Tensor) -> bool:
    """Whether two tensors, each of elements apart, share memory."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0 or a0 == a1 or b0 == b1:
        return False
    if a0 > b0:
        a, b, a0, b0 = b, a, b0, a0
    (da, ra), (db, rb), es, d = _places(a), _places(b), a.element_size(), b0 - a0
    if da == db and b.element_size() == es and d % es == 0 and d >= ra * es and _apart(da, d // es + rb):
        return False                           # two bands of one buffer
    at = torch.cat([_starts(da) * es, _starts(db) * b.element_size() + d])
    end = at + torch.tensor([ra * es, rb * b.element_size()]).repeat_interleave(
        torch.tensor([a.numel() // ra, b.numel() // rb]))
    at, order = at.sort()
    return bool((at[1:] < end[order][:-1]).any())


def _share(ts: Sequence[Tensor]) -> bool:
    """Whether any two of several tensors share memory."""
    if len(ts) < 2:
        return False
    spans = sorted((*_span(t), i) for i, t in enumerate(ts))
    if all(a[1] <= b[0] for a, b in zip(spans, spans[1:])):
        return False
    return any(_in_one_place(a, b) for i, a in enumerate(ts) for b in ts[:i])


def _launch(fn_name: str, recs: List[int]) -> None:
    """``recs``: eleven numbers for each tensor."""
    K = _kernels()
    fn = getattr(K._lib, fn_name)
    for i in range(0, len(recs), 11 * _MAX_RECS):
        part = recs[i:i + 11 * _MAX_RECS]
        n = len(part) // 11
        K._check(fn(_RECS[n].pack(*part), n, K._stream()), fn_name)
        K.LAUNCHES.count += 1


def _elsewhere(device: torch.device) -> bool:
    """Whether the launches need another current device."""
    return device.index != torch._C._cuda_getDevice()


def _same_device(what: str, *ts) -> torch.device:
    dev = ts[0].device
    for t in ts:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on different devices")
    return dev


def store8(xs: Union[Tensor, Sequence[Tensor]]) -> Union[Packed8, List[Packed8]]:
    """8-bit form of one tensor or of several (bf16 or fp32, one device; last dimension = channels,
    any number of leading ones, rows at any strides).  Several share one launch and one buffer."""
    if isinstance(xs, Tensor):
        return store8([xs])[0]
    xs = list(xs)
    if not xs:
        return []
    dev = xs[0].device
    for x in xs:
        if (x.dtype is not BF16 and x.dtype is not F32) or x.dim() < 1:
            raise ValueError(f"store8 takes bf16 or fp32 activations, not {x.dtype} of {x.dim()} dimensions")
        if x.device != dev:
            raise ValueError("store8: tensors on different devices")
    if dev.type != "cuda":
        out = []
        for x in xs:
            codes, steps = ref.store8(x.detach().reshape(math.prod(x.shape[:-1]), x.shape[-1]))
            out.append(Packed8(codes, steps, x.shape, x.dtype))
        return out
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return store8(xs)
    geo, total = [], 0
    for x in xs:
        shape = x.shape
        cols = shape[-1]
        rows = x.numel() // cols if cols else math.prod(shape[:-1])
        groups = (cols + GROUP - 1) // GROUP
        steps = total + (rows * groups * GROUP + 127) // 128 * 128
        geo.append((total, steps, shape, rows, cols))
        total = steps + (rows * ((groups + 3) // 4 * 4) + 127) // 128 * 128
    arena = _new(total, torch.uint8, dev)
    base = arena.data_ptr()
    out, recs, hold = [], [], []
    for x, (codes, steps, shape, rows, cols) in zip(xs, geo):
        out.append(Packed8._in(arena, (codes, steps), shape, x.dtype, rows))
        if rows == 0 or cols == 0:
            continue
        dims = _row_dims(x, rows)
        if dims is None:                       # channels apart, or rows that are no three strides
            x = x.detach().contiguous()
            hold.append(x)
            dims = _row_dims(x, rows)
        recs += (x.data_ptr(), base + codes, base + steps, *dims, cols, x.dtype is F32)
    if recs:
        _launch("imf_store8", recs)
    return out


def restore8(ps: Union[Packed8, Sequence[Packed8]], outs=None) -> Union[Tensor, List[Tensor]]:
    """The values of one packed tensor or of several, in one launch; ``outs``: where they go (one
    tensor, or a list with None for a new one), of the packed shape and type, rows at any three
    strides, channels adjacent, no two elements in one place."""
    if isinstance(ps, Packed8):
        return restore8([ps], None if outs is None else [outs])[0]
    ps = list(ps)
    if not ps:
        return []
    outs = [None] * len(ps) if outs is None else list(outs)
    if len(outs) != len(ps):
        raise ValueError(f"{len(ps)} packed tensors and {len(outs)} outputs")
    dev = _same_device("restore8", *ps, *outs)
    for p, o in zip(ps, outs):
        if o is not None and (o.shape != p.shape or o.dtype != p.dtype):
            raise ValueError(f"output {o.dtype} {tuple(o.shape)} for packed {p.dtype} {tuple(p.shape)}")
    given = [o for o in outs if o is not None]
    if not all(o.is_contiguous() or _apart(*_places(o)) for o in given) or _share(given):
        raise ValueError("restore8 output: no two elements in one place, of one output or of two")
    if dev.type != "cuda":
        for i, p in enumerate(ps):
            v = ref.values8(p.codes, p.steps, p.cols).to(p.dtype).view(p.shape)
            outs[i] = v if outs[i] is None else outs[i].copy_(v)
        return outs
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return restore8(ps, outs)
    recs = []
    for i, p in enumerate(ps):
        o = outs[i]
        if o is None:
            o = outs[i] = _new(p.shape, p.dtype, dev)
        if p.rows == 0 or p.cols == 0:
            continue
        dims = _row_dims(o, p.rows)
        if dims is None:
            raise ValueError("restore8 output: the channels have to be adjacent, the rows at three strides at most")
        recs += (o.data_ptr(), *p._ptrs(), *dims, p.cols, p.dtype is F32)
    if recs:
        _launch("imf_restore8", recs)
    return outs


def gemm_wgrad8(dy: Tensor, x8: Packed8, out: Optional[Tensor] = None, accumulate: bool = False) -> Tensor:
    """Weight gradient ``out[n_out, n_in] (+)= dy^T x`` of a linear layer whose input (rows, n_in) is
    kept in 8 bits; ``dy`` (rows, n_out) bf16 with 16-byte aligned rows, fp32 result, slices of
    the rows summed in a fixed order (see ``kernels.gemm_wgrad``)."""
    if not isinstance(x8, Packed8) or x8.dtype != BF16:
        raise ValueError("gemm_wgrad8 takes a bf16 activation packed by store8")
    if dy.dtype != BF16 or dy.dim() != 2 or dy.shape[0] != x8.rows:
        raise ValueError(f"dy {dy.dtype} {tuple(dy.shape)} does not go with packed rows {x8.rows}")
    N, C = dy.shape[1], x8.cols
    if out is None:
        accumulate = False
    elif out.dtype != F32 or tuple(out.shape) != (N, C) or (C > 1 and out.stride(1) != 1) \
            or (N > 1 and out.stride(0) < C):
        raise ValueError(f"out has to be fp32 ({N}, {C}) with adjacent columns and rows apart")
    dev = _same_device("gemm_wgrad8", dy, x8, out)
    if out is None:
        out = _new((N, C), F32, dev)
    if dy.numel() == 0 or C == 0:
        return out if accumulate else out.zero_()
    if dev.type != "cuda":
        g = dy.float().t() @ ref.values8(x8.codes, x8.steps, C)
        return out.add_(g) if accumulate else out.copy_(g)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return gemm_wgrad8(dy, x8, out, accumulate)
    rows = x8.rows
    ld = dy.stride(0) if rows > 1 else (N + 7) // 8 * 8
    if dy.stride(1) != 1 and N > 1 or ld % 8 or ld < N or dy.data_ptr() % 16:
        raise ValueError("dy needs adjacent columns and 16-byte aligned rows that do not overlap")
    if max(rows, N, C) >= 2 ** 31 - 512:
        raise ValueError(f"gemm_wgrad8: sizes of 2^31 and more ({rows}, {N}, {C})")
    K = _kernels()
    ldo = out.stride(0) if N > 1 else (C + 3) // 4 * 4
    floats = K._lib.imf_wgrad8_work(rows, N, C, out.data_ptr(), ldo)
    work = _new(floats, F32, dev) if floats else None
    codes, steps = x8._ptrs()
    K._check(K._lib.imf_wgrad8(dy.data_ptr(), ld, codes, steps, rows, N, C, out.data_ptr(), ldo, int(accumulate),
                               None if work is None else work.data_ptr(), floats,
                               K.status_word(dev).data_ptr(), K._stream()), "imf_wgrad8")
    K.LAUNCHES.count += 2 if floats else 1
    return out


def situ_bwd8(gu8: Packed8, gout: Tensor, beta: float, lbeta: Optional[float]) -> Tuple[Tensor, Tensor]:
    """Reverse mode of y = situ(gate) up' from the packed [gate | up] (rows, 2F): returns (its
    gradient (rows, 2F), y (rows, F)), bf16 -- y is what the next layer's weight gradient multiplies, so
    it need not be kept.  ``gout`` (rows, F) bf16, adjacent columns; the betas are positive normal numbers of
    32 bits."""
    if not isinstance(gu8, Packed8) or gu8.dtype != BF16 or gu8.cols % 2:
        raise ValueError("situ_bwd8 takes a bf16 [gate | up] packed by store8")
    rows, F = gu8.rows, gu8.cols // 2
    if gout.dtype != BF16 or gout.dim() != 2 or tuple(gout.shape) != (rows, F):
        raise ValueError(f"gout {gout.dtype} {tuple(gout.shape)}: bf16 ({rows}, {F}) expected")
    if not _F32_MIN <= beta <= _F32_MAX or (lbeta is not None and not _F32_MIN <= lbeta <= _F32_MAX):
        raise ValueError(f"beta {beta} and linear beta {lbeta} have to be positive normal numbers of 32 bits")
    dev = _same_device("situ_bwd8", gu8, gout)
    g_gu, act = _new((rows, 2 * F), BF16, dev), _new((rows, F), BF16, dev)
    if rows == 0 or F == 0:
        return g_gu, act
    if dev.type != "cuda":
        gu = ref.values8(gu8.codes, gu8.steps, 2 * F)
        a, b, y = ref.situ_mul_grad(gu[:, :F], gu[:, F:], gout, beta, lbeta)
        return g_gu.copy_(torch.cat([a, b], 1)), act.copy_(y)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return situ_bwd8(gu8, gout, beta, lbeta)
    if F > 1 and gout.stride(1) != 1:
        raise ValueError("gout needs adjacent columns")
    K = _kernels()
    codes, steps = gu8._ptrs()
    K._check(K._lib.imf_situ_bwd8(codes, steps, gout.data_ptr(), g_gu.data_ptr(), act.data_ptr(), rows, F,
                                  gout.stride(0), 2 * F, F, float(beta), float(lbeta or 0.0),
                                  int(lbeta is not None), K._stream()), "imf_situ_bwd8")
    K.LAUNCHES.count += 1
    return g_gu, act


def attn_bwd8(q8: Packed8, k8: Packed8, v8: Union[Packed8, Tensor], o8: Union[Packed8, Tensor], lse: Tensor,
              go: Tensor, scale: Optional[float] = None, gv_out: Optional[Tensor] = None
              ) -> Tuple[Tensor, Tensor, Tensor]:
    """(dq, dk, dv) of dense attention on (B, L, H, head_dim 64 or 128) from checkpoints of q, k, v and
    the output o, the forward's log-sum-exp (B, H, L) and the output gradient ``go`` (bf16):

        P = exp(scale q k^T - lse),  dV = P^T go,  dS = P * (go v^T - rowsum(go * o)),
        dQ = scale dS k,  dK = scale dS^T q

    v and o may also be bf16 tensors (a band of a wider buffer that is restored anyway).  ``gv_out``
    takes dv (16-byte aligned rows, no two elements in one place), as in ``kernels.attn_bwd``, whose
    fixed-order mode holds here too.  ``scale`` is finite, of either sign."""
    for name, t in (("q", q8), ("k", k8)):
        if not isinstance(t, Packed8):
            raise ValueError(f"attn_bwd8: {name} has to be packed by store8")
    shape = q8.shape
    if len(shape) != 4 or shape[3] not in (64, 128):
        raise ValueError(f"attn_bwd8 takes (B, L, H, 64 or 128), not {tuple(shape)}")
    B, L, H, hd = shape
    for name, t in (("q", q8), ("k", k8), ("v", v8), ("o", o8), ("go", go), ("gv_out", gv_out)):
        if t is not None and (t.shape != shape or t.dtype != BF16):
            raise ValueError(f"attn_bwd8: {name} is {t.dtype} {tuple(t.shape)}, q is bf16 {tuple(shape)}")
    if lse.dtype != F32 or tuple(lse.shape) != (B, H, L) or not lse.is_contiguous():
        raise ValueError(f"attn_bwd8: lse has to be contiguous fp32 {(B, H, L)}")
    dev = _same_device("attn_bwd8", q8, k8, v8, o8, lse, go, gv_out)
    if 0 in shape:
        new = lambda: _new(shape, BF16, dev)
        return new(), new(), new() if gv_out is None else gv_out
    scale = hd ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _F32_MAX / 2:         # the kernels multiply it by log2 e
        raise ValueError(f"attn_bwd8: scale {scale}")
    if gv_out is not None and not _apart(*_places(gv_out)):
        raise ValueError("attn_bwd8: no two elements of the dv output in one place")
    if dev.type != "cuda":
        plain = lambda t: t.restore() if isinstance(t, Packed8) else t
        dq, dk, dv = ref.attention_grad(*(plain(t) for t in (q8, k8, v8, o8)), lse, go, scale)
        dv = dv.to(BF16) if gv_out is None else gv_out.copy_(dv)
        return dq.to(BF16), dk.to(BF16), dv
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return attn_bwd8(q8, k8, v8, o8, lse, go, scale, gv_out)
    K = _kernels()
    lib, stream = K._lib, K._stream()
    dq, dk = _new(shape, BF16, dev), _new(shape, BF16, dev)
    dv = _new(shape, BF16, dev) if gv_out is None else gv_out
    row = (L * H * hd, H * hd, hd)
    dv_strides = [s if m > 1 else r for m, s, r in zip(shape, dv.stride(), row)]      # no address depends on the others
    if dv.stride(3) != 1 or dv.data_ptr() % 16 or any(s % 8 for s in dv_strides):
        raise ValueError("attn_bwd8: the dv output needs 16-byte aligned rows")
    # what is packed but o gets its values in bf16 in front of the kernel's own scratch, in the call's first launch.
    # (head_dim 64 at a scale of zero: the kernel's form for an exact Q divides by it, so the other one runs)
    first = hd == 128 or abs(scale) >= 1e-30
    n, rows = 2 * B * L * H * hd, B * L * H
    size = (n + 255) // 256 * 256
    nscr = lib.imf_attn_bwd_scratch_bytes_hd(B, L, H, hd)
    space = sum(isinstance(t, Packed8) for t in ((q8, k8, v8) if first else (q8, k8, v8, o8))) * size
    work = _new(space + nscr, torch.uint8, dev)
    at = base = work.data_ptr()
    codes, recs, ptrs, strides, hold = [], [], [], [], []
    for t in (q8, k8, v8, o8, go):
        if not isinstance(t, Packed8):
            t = K._tma_ok(t)
            if 0 in t.stride():                # a broadcast gradient, shared heads
                t = t.contiguous()
            strides.append(row if t.is_contiguous() else t.stride()[:3])
            ptrs.append(t.data_ptr())
            hold.append(t)                     # a copy lives until the launch
            codes += (None, None)
            continue
        pair = t._ptrs()
        codes += pair
        strides.append(row)
        if first and len(ptrs) == 3:           # o stays as it is
            ptrs.append(None)
            continue
        recs += (at, *pair, 1, 1, rows, 0, 0, hd, hd, 0)
        ptrs.append(at)
        at += size
    i64 = ctypes.c_int64
    q_, k_, v_, o_, g_ = strides
    common = (*ptrs, lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, L, H, hd,
              (i64 * 12)(*q_, *k_, *v_, *g_), (i64 * 3)(*o_), (i64 * 3)(*row), (i64 * 3)(*dv_strides), scale,
              base + space, nscr)
    fixed, status = int(K.DETERMINISTIC), K.status_word(dev).data_ptr()
    if first:
        K._check(lib.imf_attn_bwd8((ctypes.c_void_p * 8)(*codes[:8]), *common, fixed, status, stream), "imf_attn_bwd8")
    else:
        _launch("imf_restore8", recs)
        K._check(lib.imf_attn_bwd(*common, None, None, None, 0, 0, fixed, None, status, stream), "imf_attn_bwd")
    K.LAUNCHES.count += 3
    return dq, dk, dv
