"""Contracts of the layer operators that need no GPU: what the C ABI refuses before a device is touched."""

from __future__ import annotations

import pytest

from serron_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("mean,rstd", [(8, None), (None, 8)])
def test_one_statistic_alone_is_refused(lib, mean, rstd):
    """A forward pass writes both where it writes one."""
    for outer in (0, 2):
        rc = lib.serron_layer_norm(8, outer, 3, 4, 0, None, None, 0, 1e-5, 8, mean, rstd, 256, 1 << 20, 0, None)
        assert rc == _lib.ERR_INVALID
        assert "serron::layer_norm: mean and rstd are given both or not at all" in lib.serron_last_error().decode()
        rc = lib.serron_dropout_add_layer_norm(8, 8, outer, 3, 4, 0, None, None, 0, 0.5, 1, None, 0, 1e-5, 8, 8, mean,
                                               rstd, 256, 1 << 20, 0, None)
        assert rc == _lib.ERR_INVALID
        assert "serron::dropout_add_layer_norm: mean and rstd" in lib.serron_last_error().decode()


def test_sizes_at_the_top_of_the_range(lib):
    """What is accepted has a workspace that 64 bits hold; the rest is refused with a message."""
    size = lib.serron_layer_norm_workspace_bytes
    top = (1 << 31) - 1
    for dtype in range(4):
        for backward in (0, 1):
            for outer, length, inner in ((1, top, 1), (1, top, 2), (3, top - 255, 1), (1 << 20, 5, top), (1 << 56, 1, 1)):
                got = size(outer, length, inner, dtype, backward)
                assert 0 < got < 1 << 62 and got % 256 == 0
            for outer, length, inner in ((1 << 59, 1, 1), ((1 << 59) - 1, 1, 1), (1 << 28, top, 1), (1, top, 1 << 27)):
                if outer * length * inner > ((1 << 63) - 1) // 64:
                    assert size(outer, length, inner, dtype, backward) == -1
                    assert "too many elements" in lib.serron_last_error().decode()
