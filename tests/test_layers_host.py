"""The layer operators' checks that need no GPU: refusals of the public functions and of the C ABI, the oracle's
generator against its published vectors, modules and workspace sizes."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import serron_b200 as serron
from serron_b200 import _lib
from tests import layer_oracle


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_generator_against_published_vectors():
    """The known answers of Philox4x32-10: counter and key of zeros, of ones, and of the digits of pi."""
    ones = (1 << 64) - 1
    for block, sequence, seed, want in [
        (0, 0, 0, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
        (ones, ones, ones, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
        (0x85A308D3243F6A88, 0x0370734413198A2E, 0x299F31D0A4093822, (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
    ]:
        got = layer_oracle.philox(np.array([block], dtype=np.uint64), sequence, seed)[0]
        assert tuple(int(v) for v in got) == want


def test_oracle_gradients_against_autograd():
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(3, 5, 4, generator=gen, dtype=torch.float64, requires_grad=True)
    w = torch.randn(5, generator=gen, dtype=torch.float64, requires_grad=True)
    b = torch.randn(5, generator=gen, dtype=torch.float64, requires_grad=True)
    gy = torch.randn(3, 5, 4, generator=gen, dtype=torch.float64)
    y = torch.nn.functional.layer_norm(x.transpose(1, 2), (5,), w, b, 1e-3).transpose(1, 2)
    want = torch.autograd.grad(y, (x, w, b), gy)
    norm = layer_oracle.Norm(x.detach(), w.detach(), b.detach(), 1, 1e-3)
    torch.testing.assert_close(norm.y, y.detach(), rtol=1e-12, atol=1e-12)
    for (got, _), exact in zip(norm.backward(gy), want):
        torch.testing.assert_close(got, exact, rtol=1e-11, atol=1e-11)


def test_names_are_public():
    for name in ("layer_norm", "dropout", "dropout_add_layer_norm", "LayerNorm2d", "Dropout", "DropoutAddLayerNorm2d",
                 "DropoutUnit"):
        assert hasattr(serron, name)
    for name in ("layer_norm", "dropout", "dropout_add_layer_norm"):
        assert getattr(serron.functional, name) is getattr(serron, name)


def test_no_cpu_path():
    x = torch.rand(1, 2, 3, 3)
    with pytest.raises(RuntimeError, match="serron::layer_norm: input must be a CUDA tensor"):
        serron.layer_norm(x)
    with pytest.raises(RuntimeError, match="serron::dropout: input must be a CUDA tensor"):
        serron.dropout(x, seed=1)
    with pytest.raises(RuntimeError, match="serron::dropout_add_layer_norm: input must be a CUDA tensor"):
        serron.dropout_add_layer_norm(x, x, seed=1)


class _Cuda:
    """A tensor that says it is on a GPU: what is refused before any kernel is refused for it too."""

    def __init__(self, t):
        self._t = t
        self.is_cuda = True

    def __getattr__(self, name):
        return getattr(self._t, name)


@pytest.mark.parametrize("kwargs,error,pattern", [
    (dict(dim=4), ValueError, "dim 4 is out of range for a 4-D input"),
    (dict(dim=-5), ValueError, "dim -5 is out of range"),
    (dict(eps=-1.0), ValueError, "eps must be finite and not negative"),
    (dict(eps=float("nan")), ValueError, "eps must be finite"),
    (dict(eps=float("inf")), ValueError, "eps must be finite"),
    (dict(weight=torch.ones(4)), RuntimeError, r"weight must have the shape \(3,\)"),
    (dict(weight=torch.ones(3, 1)), RuntimeError, r"weight must have the shape \(3,\)"),
    (dict(bias=torch.ones(2)), RuntimeError, r"bias must have the shape \(3,\)"),
    (dict(weight=torch.ones(3, dtype=torch.float64)), RuntimeError, "weight must be float32 or have the input's dtype"),
    (dict(weight=torch.ones(3), bias=torch.ones(3, dtype=torch.bfloat16)), RuntimeError,
     "bias must be float32 or have the input's dtype"),
])
def test_layer_norm_refusals(kwargs, error, pattern):
    with pytest.raises(error, match=pattern):
        serron.layer_norm(_Cuda(torch.rand(2, 3, 4, 5)), **kwargs)


def test_layer_norm_refuses_mixed_parameters_and_empty_rows():
    x = _Cuda(torch.rand(2, 3, 4, 5).half())
    with pytest.raises(RuntimeError, match="weight and bias must share a dtype"):
        serron.layer_norm(x, torch.ones(3), torch.ones(3).half())
    with pytest.raises(ValueError, match="dimension 1 of the input is empty"):
        serron.layer_norm(_Cuda(torch.rand(2, 0, 4)))
    with pytest.raises(ValueError, match="out of range for a 0-D input"):
        serron.layer_norm(_Cuda(torch.tensor(1.0)), dim=0)
    with pytest.raises(RuntimeError, match="unsupported dtype torch.int32"):
        serron.layer_norm(_Cuda(torch.ones(2, 3, dtype=torch.int32)))


@pytest.mark.parametrize("kwargs,error,pattern", [
    (dict(p=-0.1), ValueError, "p must be between 0 and 1, got -0.1"),
    (dict(p=1.5), ValueError, "p must be between 0 and 1"),
    (dict(p=float("nan")), ValueError, "p must be between 0 and 1, got nan"),
    (dict(seed=-1), ValueError, "seed must be in"),
    (dict(seed=1 << 64), ValueError, "seed must be in"),
    (dict(seed=1.5), TypeError, "integer"),
    (dict(sequence=-1), ValueError, "sequence must be in"),
    (dict(sequence=1 << 64), ValueError, "sequence must be in"),
    (dict(seed=torch.zeros(2, dtype=torch.int64)), ValueError, "one int64, got 2"),
    (dict(seed=torch.zeros(1, dtype=torch.int32)), ValueError, "one int64, got 1 of torch.int32"),
])
@pytest.mark.parametrize("joined", [False, True])
def test_dropout_refusals(kwargs, error, pattern, joined):
    x = _Cuda(torch.rand(2, 3))
    kwargs = {"seed": 1, **kwargs}
    with pytest.raises(error, match=pattern):
        if joined:
            serron.dropout_add_layer_norm(x, x, **kwargs)
        else:
            serron.dropout(x, **kwargs)


@pytest.mark.parametrize("residual,pattern", [
    (torch.rand(2, 4), "residual and input must share a shape"),
    (torch.rand(3), "residual and input must share a shape"),
    (torch.rand(2, 3).double(), "residual and input must share a dtype"),
])
def test_residual_refusals(residual, pattern):
    x = _Cuda(torch.rand(2, 3))
    with pytest.raises(RuntimeError, match=pattern):
        serron.dropout(x, seed=1, residual=residual)
    with pytest.raises(RuntimeError, match=pattern):
        serron.dropout_add_layer_norm(x, residual, seed=1)


def test_dropout_units():
    with pytest.raises(ValueError, match="unit 'channel' needs an input of at least 2 dimensions, got 1"):
        serron.dropout(_Cuda(torch.rand(4)), seed=1, unit=serron.DropoutUnit.CHANNEL)
    with pytest.raises(ValueError, match="unit 'sample' needs an input of at least 1 dimensions, got 0"):
        serron.dropout(_Cuda(torch.tensor(1.0)), seed=1, unit=serron.DropoutUnit.SAMPLE)
    with pytest.raises(ValueError, match="'pixel' is not a valid DropoutUnit"):
        serron.dropout(_Cuda(torch.rand(4, 4)), seed=1, unit="pixel")


def test_modules():
    norm = serron.LayerNorm2d(5, dtype=torch.bfloat16)
    assert list(norm.state_dict()) == ["weight", "bias"]
    assert torch.equal(norm.weight, torch.ones(5, dtype=torch.bfloat16)) and not norm.bias.any()
    assert serron.LayerNorm2d(5, affine=False).state_dict() == {}
    x, r = torch.rand(2, 3), torch.rand(2, 3)
    drop = serron.Dropout(0.3).eval()  # outside training nothing runs but the sum
    assert drop(x) is x and torch.equal(drop(x, r), x + r)
    assert serron.Dropout(0.0)(x) is x
    assert list(serron.DropoutAddLayerNorm2d(4, 0.1).state_dict()) == ["weight", "bias"]


def test_c_abi_refusals(lib):
    def message():
        return lib.serron_last_error().decode()

    def norm(outer=2, length=3, inner=4, dtype=0, weight=None, param=0, eps=1e-5, nbytes=0):
        return lib.serron_layer_norm(None, outer, length, inner, dtype, weight, None, param, eps, None, None, None, None,
                                     nbytes, 0, None)

    assert norm(length=0) == _lib.ERR_INVALID and "must not be empty" in message()
    assert norm(outer=-1) == _lib.ERR_INVALID and "must be non-negative" in message()
    assert norm(length=1 << 31) == _lib.ERR_INVALID and "below 2^31" in message()
    assert norm(outer=1 << 40, length=1 << 30, inner=1 << 30) == _lib.ERR_INVALID and "too many" in message()
    assert norm(dtype=4) == _lib.ERR_INVALID and "unsupported dtype code 4" in message()
    assert norm(dtype=1, weight=8, param=0) == _lib.ERR_INVALID and "must be float32 or have" in message()
    assert norm(eps=-1.0) == _lib.ERR_INVALID and "eps must be finite" in message()
    assert norm() == _lib.ERR_INVALID and "must not be null" in message()
    assert norm(outer=0) == _lib.OK  # nothing to do, no device needed
    rc = lib.serron_layer_norm(8, 2, 300000, 1, 0, None, None, 0, 1e-5, 8, None, None, None, 0, 0, None)
    assert rc == _lib.ERR_WORKSPACE and "serron::layer_norm: workspace of 0 bytes" in message()
    rc = lib.serron_layer_norm_backward(8, 8, 8, 8, 2, 3, 4, 0, None, 0, 8, 8, 8, None, 0, 0, None)
    assert rc == _lib.ERR_WORKSPACE and "serron::layer_norm_backward: workspace" in message()
    assert lib.serron_layer_norm_backward(None, None, None, None, 0, 3, 4, 0, None, 0, None, None, None, None, 0, 0,
                                          None) == _lib.OK

    def drop(numel=4, span=1, dtype=0, p=0.5):
        return lib.serron_dropout(None, None, numel, span, dtype, p, 1, None, 0, None, 0, None)

    assert drop(p=1.1) == _lib.ERR_INVALID and "serron::dropout: p must be between 0 and 1" in message()
    assert drop(p=float("nan")) == _lib.ERR_INVALID and "p must be between" in message()
    assert drop(span=0) == _lib.ERR_INVALID and "at least one element" in message()
    assert drop(numel=-1) == _lib.ERR_INVALID and "non-negative" in message()
    assert drop(dtype=-1) == _lib.ERR_INVALID and "unsupported dtype code -1" in message()
    assert drop() == _lib.ERR_INVALID and "must not be null" in message()
    assert drop(numel=0) == _lib.OK


def test_c_abi_workspace_sizes(lib):
    size = lib.serron_layer_norm_workspace_bytes
    assert size(0, 5, 1, 0, 0) == 0
    assert size(2, 0, 1, 0, 1) == -1 and size(2, 3, 4, 9, 1) == -1
    for args in [(3, 50001, 1), (5, 67, 5917), (8192, 1024, 1), (1, 4000, 49)]:
        for dtype in range(4):
            for backward in (0, 1):
                got = size(*args, dtype, backward)
                assert got >= 0 and got % 256 == 0
    assert isinstance(ctypes.c_int64(size(1 << 20, 1024, 1, 3, 1)).value, int)
