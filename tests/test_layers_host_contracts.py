"""Contracts of the layer operators that need no GPU: what the C ABI refuses before a device is touched."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from serron_b200 import _lib


PACKAGE = os.path.dirname(os.path.abspath(_lib.__file__))


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


def test_addresses_off_their_elements_are_refused(lib):
    """A kernel that read them would fault; nothing is launched."""
    def refused(rc, *patterns):
        assert rc == _lib.ERR_INVALID
        assert all(p in lib.serron_last_error().decode() for p in patterns)

    elements = "tensors must start on a boundary of their elements"
    space = 1 << 20
    for size, dtype in ((4, 0), (8, 1), (2, 2), (2, 3)):
        stat = 8 if dtype == 1 else 4
        for k in range(6):
            t = [64 + (size // 2 if i == k else 0) for i in range(4)] + [64 + (stat // 2 if i == k else 0) for i in (4, 5)]
            refused(lib.serron_layer_norm(t[0], 2, 3, 4, dtype, t[1], t[2], dtype, 1e-5, t[3], t[4], t[5], 256, space, 0,
                                          None), "serron::layer_norm: ", elements)
            refused(lib.serron_layer_norm_backward(t[0], t[1], t[4], t[5], 2, 3, 4, dtype, t[2], dtype, t[3], None, None,
                                                   256, space, 0, None), "serron::layer_norm_backward: ", elements)
            refused(lib.serron_dropout_add_layer_norm(t[0], t[1], 2, 3, 4, dtype, None, None, dtype, 0.5, 1, None, 0, 1e-5,
                                                      t[2], t[3], t[4], t[5], 256, space, 0, None),
                    "serron::dropout_add_layer_norm: ", elements)
            refused(lib.serron_dropout_add_layer_norm_backward(t[0], t[1], t[2], t[4], t[5], 2, 3, 4, dtype, t[3], dtype,
                                                               0.5, 1, None, 0, 64, 64, None, None, 256, space, 0, None),
                    "serron::dropout_add_layer_norm_backward: ", elements)
        for k in range(3):
            t = [64 + (size // 2 if i == k else 0) for i in range(3)]
            refused(lib.serron_dropout(t[0], t[1], 12, 1, dtype, 0.5, 1, None, 0, t[2], 0, None), "serron::dropout: ",
                    elements)
    for k in range(2):  # gradients of float32 parameters beside 16-bit activations
        t = [64 + (2 if i == k else 0) for i in range(2)]
        refused(lib.serron_layer_norm_backward(64, 64, 64, 64, 2, 3, 4, 3, None, 0, 64, t[0], t[1], 256, space, 0, None),
                elements)
    refused(lib.serron_dropout(64, None, 12, 1, 0, 0.5, 1, 68, 0, 64, 0, None), "seed in device memory", "8 bytes")
    # rows beyond the register kernels need a workspace
    refused(lib.serron_layer_norm(64, 1, 300000, 1, 0, None, None, 0, 1e-5, 64, None, None, 264, 1 << 30, 0, None),
            "serron::layer_norm: the workspace must be aligned to 256 bytes")


@pytest.mark.skipif(shutil.which("readelf") is None, reason="needs binutils")
def test_binding_shares_the_cpp_runtime():
    """A copy of its own beside torch's crashes where a number goes into an error message."""
    out = subprocess.run(["readelf", "-d", os.path.join(PACKAGE, "_layers.so")], check=True, capture_output=True, text=True)
    assert "[libstdc++.so.6]" in out.stdout


@pytest.mark.skipif(shutil.which("make") is None, reason="needs make")
def test_library_builds_without_torch(tmp_path):
    """The C library has no torch symbols, and whoever builds it need have no torch."""
    target = str(tmp_path / "_layers.so")
    library = os.path.join(PACKAGE, "libserron_b200.so")
    out = subprocess.run(["make", "-s", "-C", os.path.join(PACKAGE, "csrc"), "-o", library, f"LAYERS={target}",
                          "PYTHON=false", target], capture_output=True, text=True)
    assert out.returncode == 0 and not os.path.exists(target)
    assert "_layers.so is not built: false has no torch" in out.stderr
