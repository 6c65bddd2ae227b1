"""CPU: what differential attention's calls keep, and what its module says of sizes that no kernel takes."""
import warnings

import pytest


def test_scratch_sizes_are_kept_by_device(monkeypatch):
    """The launchers ask their device for its SMs: a size asked for on one device says nothing of another."""
    from imfvideo_b200.ops import diffattn as DA

    calls = []

    class Lib:
        def imf_attn_diff_fwd_scratch_bytes(self, *sizes):
            calls.append(sizes)
            return 1000 * len(calls)

    class Kernels:
        _lib = Lib()
    monkeypatch.setattr(DA, "_kernels", lambda: Kernels)
    DA._scratch_bytes.cache_clear()
    try:
        got = [DA._scratch_bytes("fwd", dev, 1, 700, 2, True) for dev in (0, 1, 0, 1)]
    finally:
        DA._scratch_bytes.cache_clear()
    assert got == [1000, 2000, 1000, 2000] and calls == [(1, 700, 2, True)] * 2


def test_head_dims_without_a_kernel_are_named():
    """Long sequences of another head_dim than 64: the formulas' maps are named with their size."""
    from imfvideo_b200.models.diff_attn import DiffAttentionImpl

    with pytest.warns(UserWarning, match="head_dim 64.*51.6 GB"):
        DiffAttentionImpl(128, 32780, 12)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        DiffAttentionImpl(64, 32780, 12)
        DiffAttentionImpl(16, 100, 4)
