"""GPU: the forward-mode kernel of differential attention on the paths that ``test_diffattn_gpu.py`` does not take.
Bounds are that file's."""
import pytest
import torch

from test_diffattn_gpu import _forward64, _inputs, _own, _status, _tangent64, _wide, _within  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,L,H", [(1, 1, 1), (2, 33, 3), (1, 64, 2), (4, 64, 80), (1, 532, 2)])
def test_walks_of_one_tile_are_the_same_every_time(B, L, H):
    """A CTA that begins with one K/V tile (all of them up to 64 rows, five of 45 at 1 x 532, 2 pairs): the group without
    a step goes on to the next walk's queries."""
    q, k, v, lam, tan = _inputs(B, L, H, seed=L, tangent=True)
    first = _own(q, k, v, lam, tan)
    _within(_wide(first[0]), *_forward64(q, k, v, lam)[2:4], "o")
    _within(_wide(first[1]), *_tangent64(q, k, v, lam, tan), "do")
    for _ in range(300):
        o, do, saved = _own(q, k, v, lam, tan)
        assert torch.equal(o, first[0]) and torch.equal(do, first[1])
        assert all(torch.equal(a, b) for a, b in zip(saved, first[2]))
