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
