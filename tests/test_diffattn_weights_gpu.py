"""GPU: the gradient of differential attention's weights, against what the kernel sums.

dlam = -sum dO . O_2.  O_2 is what the forward pass kept (its error has a test of its own): what is left are 32-bit sums over a
row's 128 channels, eight in a chain and sixteen in a tree, 12 * 2^-24 of the magnitudes at most, then
64-bit sums over rows, and dlam's own rounding.  With a gradient that is correlated with O_2 the sum stands far above
that bound, so a batch entry, a half of the channels or a tail of rows that is left out shows."""
import pytest
import torch

from test_diffattn_gpu import SHAPES, _inputs, _own, _status, _wide  # noqa: F401
from test_diffattn_tangent_gpu import _joined

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0.0, 0.5])
@pytest.mark.parametrize("B,L,H", SHAPES + [(2, 2061, 2)])
def test_weight_gradient(B, L, H, offset, dtype):
    """``offset``: a gradient that the values' own offset is correlated with."""
    from imfvideo_b200.ops import diffattn as DA

    q, k, v, lam, go = _inputs(B, L, H, seed=L)
    lam = lam.to(dtype)
    o, _, saved = _own(q, k, v, lam)
    O2 = _joined(saved, o)[1]
    go = (go.float() + offset * O2.sign()).bfloat16()
    got = DA.diff_attn_bwd(q, k, v, lam, o, saved, go)[3]
    terms = _wide(go) * _wide(O2)                            # (B, H, L, 128)
    want, size = -terms.sum((0, 2, 3)), terms.abs().sum((0, 2, 3))
    bound = 1e-6 * size + torch.finfo(dtype).eps / 2 * want.abs()
    assert got.dtype == dtype and ((got.double() - want).abs() <= bound).all()
    if offset and dtype is torch.float32:
        # what any part of it is worth (with a correlated gradient; a random sum can be near zero): every batch entry, half
        # of the channels, the last rows
        parts = torch.stack([*terms[:, :, :, :64].sum((2, 3)), *terms.sum((2, 3)), terms[:, :, -1].sum((0, 2))])
        assert (parts.abs() > 4 * bound).all()
