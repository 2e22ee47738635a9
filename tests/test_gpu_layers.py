"""Layer norm, dropout and their join on the GPU, against 64-bit oracles with derived bounds (layer_oracle.py), against
differences, and bit for bit where the operator is exact (masks, dropout, what must not depend on layout or order)."""

from __future__ import annotations

import math

import pytest
import torch

from tests import layer_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float64]
IDS = [str(d).split(".")[-1] for d in DTYPES]
EPS = 1e-5


@pytest.fixture(scope="module")
def serron():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import serron_b200

    return serron_b200


def _rand(shape, dtype, seed, scale=1.0, level=0.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64) * scale + level).to(dtype)


def _params(length, dtype, params, seed):
    if params == "none":
        return None, None
    pdtype = dtype if params in ("same", "weight", "bias") or dtype == torch.float64 else torch.float32
    w = _rand((length,), pdtype, seed + 1, 0.3, 1.0)
    b = _rand((length,), pdtype, seed + 2, 0.3)
    return (None if params == "bias" else w), (None if params == "weight" else b)


def _normed(y, h, w=None, b=None, dim=1):
    ref = oracle.Norm(h, w, b, dim, EPS)
    oracle.within(y, ref.y, ref.y_bound(), "norm of h")


def _check_norm(serron, x, dim, params="f32", seed=0, gy=None):
    """Forward and backward of one call against the oracle; returns y and the gradients."""
    length = x.shape[dim]
    w, b = _params(length, x.dtype, params, seed)
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = serron.layer_norm(x, w, b, dim=dim, eps=EPS)
    assert y.dtype == x.dtype and y.shape == x.shape
    gy = _rand(x.shape, x.dtype, seed + 3) if gy is None else gy
    grads = list(torch.autograd.grad(y, leaves, gy))
    with torch.no_grad():
        again = serron.layer_norm(x, w, b, dim=dim, eps=EPS)
        assert torch.equal(again, y), "without a backward to follow"
        ref = oracle.Norm(x, w, b, dim, EPS)
        oracle.within(y, ref.y, ref.y_bound(), "y")
        wanted = ref.backward(gy)
        names = ["dx"] + ["dw"] * (w is not None) + ["db"] * (b is not None)
        pairs = [wanted[0]] + [wanted[1]] * (w is not None) + [wanted[2]] * (b is not None)
        for name, got, (want, bound) in zip(names, grads, pairs):
            oracle.within(got, want, bound, name)
    return y.detach(), grads


# rows of every kind: one element, odd, around warps, vectors, threads and chunks, long and very long ones
ROWS = [(1, 1), (5, 1), (3, 2), (7, 3), (2, 7), (1000, 8), (33, 9), (5, 31), (6, 32), (3, 33), (9, 63), (17, 100),
        (4, 255), (70, 256), (3, 257), (300, 511), (2, 768), (129, 1000), (40, 1024), (3, 1025), (9, 2047), (5, 2048),
        (3, 4096), (2, 5003), (5, 8192), (3, 8193), (1, 16384), (2, 16385), (2, 32767), (3, 32768), (1, 50001),
        (2, 65536), (1, 65537), (1, 131075), (2, 262144), (1, 300001), (1, 1048576)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,length", ROWS)
def test_norm_rows(serron, rows, length, dtype):
    _check_norm(serron, _rand((rows, length), dtype, length, 1.5, 0.7), -1, "f32" if length % 2 else "same", length)


MAPS = [(1, 1, 1, 1), (1, 1, 3, 5), (2, 3, 5, 7), (1, 2, 1, 2), (3, 8, 4, 4), (2, 32, 16, 16), (1, 5, 1, 1), (2, 16, 31, 33),
        (1, 67, 9, 61), (5, 64, 7, 7), (2, 128, 14, 14), (2, 129, 6, 10), (1, 255, 5, 13), (1, 512, 8, 8),
        (3, 1000, 3, 3), (1, 1024, 4, 6), (1, 1025, 3, 3), (2, 2053, 7, 5), (1, 4100, 2, 2), (300, 12, 3, 2), (1, 32, 128, 130),
        (2, 3, 200, 333)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", MAPS)
def test_norm_maps(serron, shape, dtype):
    _check_norm(serron, _rand(shape, dtype, sum(shape), 1.5, 0.7), 1, "same" if shape[1] % 2 else "f32", sum(shape))


@pytest.mark.parametrize("params", ["none", "weight", "bias", "same", "f32"])
@pytest.mark.parametrize("shape,dim", [((6, 96), 1), ((2, 24, 5, 6), 1), ((2, 24, 5, 6), -1), ((3, 4, 10), 0)])
def test_norm_params(serron, shape, dim, params):
    for dtype in (torch.float32, torch.bfloat16):
        _check_norm(serron, _rand(shape, dtype, 5), dim, params)


@pytest.mark.parametrize("rows,length", [(150000, 16), (40000, 72), (70001, 8), (9000, 1024), (600, 9001)])
def test_norm_many_rows(serron, rows, length):
    """The gradients of the parameters stay sums of a tree however many rows there are."""
    _check_norm(serron, _rand((rows, length), torch.bfloat16, 9, 1.0, 2.0), 1, "f32", 9)


def test_norm_many_pixels(serron):
    _check_norm(serron, _rand((7, 24, 250, 252), torch.float16, 9, 1.0, 2.0), 1, "f32", 9)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_norm_layouts(serron, dtype):
    """Any dense order is read as it lies and gives the values of the contiguous copy; so do strided views, expanded
    inputs and tensors that start off a vector's boundary."""
    base = _rand((3, 20, 6, 10), dtype, 4)
    w, b = _params(20, dtype, "f32", 4)
    gy = _rand(base.shape, dtype, 8)
    norm = oracle.Norm(base, w, b, 1, EPS)
    (dx, dx_bound), *_ = norm.backward(gy)
    wide = torch.empty((3, 20, 6, 20), dtype=dtype, device="cuda")

    def shifted(t, by):
        return torch.empty(t.numel() + by, dtype=dtype, device="cuda")[by:].view(t.shape).copy_(t)

    views = {
        "channels_last": base.to(memory_format=torch.channels_last),
        "transposed": base.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0),
        "strided": wide[..., ::2].copy_(base),
        **{f"offset{k}": shifted(base, k) for k in (1, 2, 3, 4)},
    }
    for name, x in views.items():
        x = x.detach().requires_grad_()
        y = serron.layer_norm(x, w, b, eps=EPS)
        oracle.within(y, norm.y, norm.y_bound(), name)
        if name in ("channels_last", "transposed"):
            assert y.stride() == x.stride()
        for grad in (gy, gy.to(memory_format=torch.channels_last), shifted(gy, 1)):
            oracle.within(torch.autograd.grad(y, x, grad, retain_graph=True)[0], dx, dx_bound, name)
    x = base.detach().requires_grad_()
    ones = torch.autograd.grad(serron.layer_norm(x, w, b, eps=EPS).sum(), x)[0]  # an expanded gradient
    (want, bound), *_ = norm.backward(torch.ones_like(base))
    oracle.within(ones, want, bound, "sum")
    row = _rand((1, 20), dtype, 5).requires_grad_()  # a broadcast input: its gradient is the rows' sum
    y = serron.layer_norm(row.expand(4, 20), w, b, dim=1, eps=EPS)
    ref = oracle.Norm(row.detach().expand(4, 20), w, b, 1, EPS)
    oracle.within(y, ref.y, ref.y_bound(), "expanded")
    strided = torch.empty((20, 2), dtype=w.dtype, device="cuda")  # parameters that are columns of something
    strided[:, 0], strided[:, 1] = w, b
    y = serron.layer_norm(base, strided[:, 0], strided[:, 1], eps=EPS)
    oracle.within(y, norm.y, norm.y_bound(), "strided parameters")


@pytest.mark.parametrize("shape,dim", [((4, 96), 1), ((4, 97), 1), ((1, 40000), 1), ((2, 12, 5, 7), 1), ((1, 12, 8, 8), 1),
                                       ((1, 1500, 2, 4), 1)])
def test_norm_rows_stand_alone(serron, shape, dim):
    """NaN, infinities and values that are all alike touch their own row only."""
    clean = _rand(shape, torch.float32, 6)
    x = clean.clone()
    rows = x.movedim(dim, -1).reshape(-1, shape[dim])
    count = rows.shape[0]
    bad = {0: float("nan")}
    if count > 2:
        bad[1] = float("inf")
        bad[2] = float("-inf")
    rows = rows.clone()
    for r, v in bad.items():
        rows[r, shape[dim] // 2] = v
    if count > 3:
        rows[3] = 5.0  # no spread: xhat is zero, y the bias
    moved = [s for d, s in enumerate(shape) if d != dim % len(shape)]
    x = rows.view(*moved, shape[dim]).movedim(-1, dim).contiguous()
    w, b = _params(shape[dim], torch.float32, "f32", 3)
    y = serron.layer_norm(x, w, b, dim=dim).movedim(dim, -1).reshape(-1, shape[dim])
    want = serron.layer_norm(clean, w, b, dim=dim).movedim(dim, -1).reshape(-1, shape[dim])
    for r in range(count):
        if r in bad:
            assert bool(y[r].isnan().all())
        elif r == 3:
            assert torch.equal(y[r], b)
        else:
            assert torch.equal(y[r], want[r]), r


def test_norm_of_large_level(serron):
    """A level far above the spread: two passes over the row keep what one pass of squares would lose."""
    for shape, dim in [((4, 512), 1), ((2, 64, 8, 8), 1), ((1, 30000), 1)]:
        _check_norm(serron, _rand(shape, torch.float32, 3, 1.0, 1000.0), dim)


def test_norm_eps_zero_and_extremes(serron):
    x = torch.tensor([[1.0, 3.0], [2.0**60, -(2.0**60)], [2.0**-60, -(2.0**-60)]], device="cuda")
    y = serron.layer_norm(x, dim=1, eps=0.0)
    assert torch.equal(y, torch.tensor([[-1.0, 1.0], [1.0, -1.0], [1.0, -1.0]], device="cuda"))
    ones = serron.layer_norm(torch.ones(2, 4, device="cuda"), dim=1, eps=0.0)
    assert bool(ones.isnan().all())  # 0 / 0, as the formula says


@pytest.mark.parametrize("shape,dim", [((0, 7), 1), ((3, 7, 0), 1), ((0, 7, 4, 4), 1)])
def test_norm_of_nothing(serron, shape, dim):
    x = torch.empty(shape, device="cuda").requires_grad_()
    w, b = torch.ones(7, device="cuda").requires_grad_(), torch.ones(7, device="cuda").requires_grad_()
    y = serron.layer_norm(x, w, b, dim=dim)
    grads = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == x.shape and grads[0].shape == x.shape
    assert not grads[1].any() and not grads[2].any()
    y, h = serron.dropout_add_layer_norm(x, x, w, b, dim=dim, seed=1)
    assert y.shape == h.shape == x.shape
    assert serron.dropout(x, seed=1).shape == x.shape


@pytest.mark.parametrize("shape,dim", [((3, 40), 1), ((2, 33, 5, 7), 1), ((2, 3000), 1)])
@pytest.mark.parametrize("joined", [False, True])
def test_gradients_against_differences(serron, shape, dim, joined):
    """Directional derivatives in float64.  With h = 1e-4 the central difference is off by h^2 / 6 times a third derivative
    of order one per element (1.7e-9) and by rounding 2^-53 / h (1.1e-12): 1e-6 of the sum's scale is far above both
    and far below any wrong term."""
    length, h = shape[dim], 1e-4
    t = [_rand(shape, torch.float64, 1), _rand(shape, torch.float64, 2), _rand((length,), torch.float64, 3, 0.3, 1.0),
         _rand((length,), torch.float64, 4)]
    if not joined:
        del t[1]
    gy, gh = _rand(shape, torch.float64, 5), _rand(shape, torch.float64, 6)

    def f(args):
        if not joined:
            return (serron.layer_norm(*args, dim=dim) * gy).sum()
        y, s = serron.dropout_add_layer_norm(*args, p=0.3, seed=11, dim=dim)
        return (y * gy).sum() + (s * gh).sum()

    grads = torch.autograd.grad(f([v.requires_grad_() for v in t]), t)
    for k, g in enumerate(grads):
        for seed in range(3):
            d = _rand(t[k].shape, torch.float64, 20 + seed)
            with torch.no_grad():
                up, down = ([v + sign * h * d if i == k else v for i, v in enumerate(t)] for sign in (1, -1))
                want = (f(up) - f(down)) / (2 * h)
            assert abs(float((g * d).sum() - want)) <= 1e-6 * math.sqrt(gy.numel()), (k, seed)


def test_partial_gradients_and_no_second_ones(serron):
    """Only what is asked for is computed, and it is the same; a second derivative is refused, not wrong."""
    for shape in ((6, 50), (2, 10, 4, 4)):
        x, w, b = _rand(shape, torch.float32, 1), *_params(shape[1], torch.float32, "f32", 2)
        gy = _rand(shape, torch.float32, 3)

        def grads(needs):
            leaves = [t.clone().requires_grad_(n) for t, n in zip((x, w, b), needs)]
            y = serron.layer_norm(*leaves)
            return dict(zip([i for i, n in enumerate(needs) if n],
                            torch.autograd.grad(y, [t for t in leaves if t.requires_grad], gy)))

        full = grads((True, True, True))
        for needs in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
            for i, g in grads(needs).items():
                assert torch.equal(g, full[i]), (needs, i)
    x = _rand((3, 8), torch.float32, 1).requires_grad_()
    g = torch.autograd.grad(serron.layer_norm(x).square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


# ------------------------------------------------------------------------------------------------
# dropout: exact
# ------------------------------------------------------------------------------------------------
SIZES = [1, 2, 3, 4, 5, 7, 8, 9, 31, 255, 1023, 1024, 1025, 4097, 65537, 1000003]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", SIZES)
def test_dropout_elements(serron, n, dtype):
    x = _rand((n,), dtype, n).requires_grad_()
    r = _rand((n,), dtype, n + 1).requires_grad_()
    gy = _rand((n,), dtype, n + 2)
    for p, seed, sequence in [(0.1, 5, 0), (0.5, (1 << 64) - 1, (1 << 64) - 1), (0.9, 1 << 33, 1 << 40)]:
        y = serron.dropout(x, p, seed=seed, sequence=sequence)
        assert torch.equal(y, oracle.dropout(x.detach(), p, seed, sequence))
        z = serron.dropout(x, p, seed=seed, sequence=sequence, residual=r)
        assert torch.equal(z, oracle.dropout(x.detach(), p, seed, sequence, residual=r.detach()))
        gx, gr = torch.autograd.grad(z, (x, r), gy)
        assert torch.equal(gx, oracle.dropout(gy, p, seed, sequence)) and torch.equal(gr, gy)
        assert torch.equal(torch.autograd.grad(y, x, gy)[0], gx)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(3, 5), (2, 3, 1), (4, 6, 2), (5, 3, 3), (3, 7, 5, 1), (2, 9, 4, 8), (6, 5, 7, 9), (2, 16, 32, 33),
                                   (1, 3, 100, 100), (40, 33, 7, 7), (8, 64, 14, 14), (3, 1001, 13), (5, 1700, 8), (2, 3, 8191),
                                   (2, 3, 8192), (1, 2, 70001)])
def test_dropout_units(serron, shape, dtype):
    x, r = _rand(shape, dtype, 1), _rand(shape, dtype, 2)
    for unit, lead in ((serron.DropoutUnit.CHANNEL, 2), (serron.DropoutUnit.SAMPLE, 1)):
        span = math.prod(shape[lead:])
        for residual in (None, r):
            y = serron.dropout(x, 0.4, seed=77, sequence=3, unit=unit, residual=residual)
            assert torch.equal(y, oracle.dropout(x, 0.4, 77, 3, span, residual)), (unit, residual is None)
        leaf = x.clone().requires_grad_()
        g = torch.autograd.grad(serron.dropout(leaf, 0.4, seed=77, sequence=3, unit=unit), leaf, r)[0]
        assert torch.equal(g, oracle.dropout(r, 0.4, 77, 3, span))


def test_dropout_probabilities(serron):
    x = _rand((4099,), torch.float32, 1)
    assert torch.equal(serron.dropout(x, 0.0, seed=1), x)
    assert torch.equal(serron.dropout(x, 1.0, seed=1), torch.zeros_like(x))
    assert torch.equal(serron.dropout(x, 1.0, seed=1, residual=x), x)
    assert torch.equal(serron.dropout(x, 1 - 2.0**-40, seed=1), torch.zeros_like(x))  # rounds to one
    assert torch.equal(serron.dropout(x, 1 - 2.0**-31, seed=1), oracle.dropout(x, 1 - 2.0**-31, 1, 0))
    assert torch.equal(serron.dropout(x, 2.0**-33, seed=1), x * (1 / (1 - 2.0**-33)))  # rounds to none
    # of 2^22 decisions with p = 1/4 the number dropped has a deviation of 887: five of them
    kept = int(serron.dropout(torch.ones(1 << 22, device="cuda"), 0.25, seed=9).count_nonzero())
    assert abs(kept - 3 * (1 << 20)) < 5 * 887


def test_dropped_values_leave_nothing(serron):
    x = torch.full((4096,), float("nan"), device="cuda")
    x[1::2] = float("inf")
    keep = oracle.kept(0, 4096, 0.5, 3, 0).cuda()
    for unit_shape, unit in (((4096,), serron.DropoutUnit.ELEMENT), ((16, 256), serron.DropoutUnit.SAMPLE)):
        y = serron.dropout(x.view(unit_shape), 0.5, seed=3, unit=unit).flatten()
        k = keep if unit is serron.DropoutUnit.ELEMENT else oracle.kept(0, 16, 0.5, 3, 0).cuda().repeat_interleave(256)
        assert not y[~k].any() and not bool(y[k].isfinite().any())


def test_dropout_views(serron):
    """Decisions go by the row-major index whatever the strides and the start."""
    base = _rand((6, 10, 7), torch.float16, 1)
    want = oracle.dropout(base, 0.3, 4, 0)
    for x in (base.transpose(0, 2).contiguous().transpose(0, 2), torch.stack((base, base), -1)[..., 1]):
        assert torch.equal(serron.dropout(x, 0.3, seed=4), want)
    flat, other = _rand((3000,), torch.bfloat16, 2), _rand((3000,), torch.bfloat16, 3)
    for a in range(9):
        x = flat[a:a + 2900]
        assert torch.equal(serron.dropout(x, 0.3, seed=4), oracle.dropout(x, 0.3, 4, 0))
        r = other[2 * a:2 * a + 2900]  # another start than the input's
        assert torch.equal(serron.dropout(x, 0.3, seed=4, residual=r), oracle.dropout(x, 0.3, 4, 0, residual=r))
        z = flat[a:a + 2888].view(8, 361)
        got = serron.dropout(z, 0.3, seed=4, unit=serron.DropoutUnit.SAMPLE)
        assert torch.equal(got, oracle.dropout(z, 0.3, 4, 0, 361))
    row = _rand((1, 7), torch.float32, 5).requires_grad_()  # a broadcast input
    g = torch.autograd.grad(serron.dropout(row.expand(5, 7), 0.3, seed=4).sum(), row)[0]
    assert torch.equal(g, oracle.dropout(torch.ones(5, 7, device="cuda"), 0.3, 4, 0).sum(0, keepdim=True))


def test_dropout_past_32_bits(serron):
    """Elements whose index and whose block's index pass 2^32 and 2^31."""
    n = (1 << 32) + 1029
    x = torch.ones(n, dtype=torch.float16, device="cuda")
    y = serron.dropout(x, 0.5, seed=6)
    for first in (0, (1 << 31) - 500, (1 << 32) - 500, n - 1000):
        assert torch.equal(y[first:first + 1000].cpu() != 0, oracle.kept(first, 1000, 0.5, 6, 0))
    del y
    z = serron.dropout(x.view(-1, 1029 + (1 << 32)), 0.5, seed=8, unit=serron.DropoutUnit.SAMPLE)
    assert bool((z != 0).all()) == bool(oracle.kept(0, 1, 0.5, 8, 0)[0]) and bool((z[0, -9:] == z[0, 0]).all())


def test_join_past_32_bits(serron):
    """Offsets past 2^31 elements in each layout."""
    n = (1 << 31) + 4096
    x = torch.zeros(n, dtype=torch.float16, device="cuda")
    x[-4096:] = _rand((4096,), torch.float16, 1)
    for shape, dim in (((n // 1024, 1024), 1), ((2, 16, n // 32), 1)):
        y, h = serron.dropout_add_layer_norm(x.view(shape), x.view(shape), p=0.5, seed=2, dim=dim)
        tail = h.view(-1)[-1024:]
        keep = oracle.kept(n - 1024, 1024, 0.5, 2, 0).cuda()
        assert torch.equal(tail, torch.where(keep, 3 * x[-1024:].float(), x[-1024:].float()).half())
        y, h = (t[-1:, ..., -1024:] for t in (y, h))
        _normed(y, h)


def test_seed_in_a_tensor(serron):
    x = _rand((1000,), torch.float32, 1)
    for value in (0, 12345, (1 << 63) - 1):
        seed = torch.tensor([value], device="cuda")
        assert torch.equal(serron.dropout(x, 0.5, seed=seed), serron.dropout(x, 0.5, seed=value))
    seed = torch.tensor(-1, device="cuda")  # the bits count
    assert torch.equal(serron.dropout(x, 0.5, seed=seed), serron.dropout(x, 0.5, seed=(1 << 64) - 1))
    leaf = x.clone().requires_grad_()
    y = serron.dropout(leaf, 0.5, seed=seed)
    seed.add_(1)  # the backward would draw another mask
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_graph_replays_under_new_seeds(serron):
    x, r = _rand((64, 40), torch.float32, 1), _rand((64, 40), torch.float32, 2)
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serron.dropout_add_layer_norm(x, r, p=0.5, seed=seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = serron.dropout_add_layer_norm(x, r, p=0.5, seed=seed)
    for value in (3, 4):
        seed.fill_(value)
        graph.replay()
        assert torch.equal(h, oracle.dropout(x, 0.5, value, 0, residual=r))
        _normed(y, h)


# ------------------------------------------------------------------------------------------------
# the join
# ------------------------------------------------------------------------------------------------
def _check_join(serron, shape, dim, dtype, p, params="f32", seed=0):
    x, r = _rand(shape, dtype, seed, 1.5, 0.5), _rand(shape, dtype, seed + 1)
    w, b = _params(shape[dim], dtype, params, seed)
    leaves = [t.requires_grad_() for t in (x, r, w, b) if t is not None]
    y, h = serron.dropout_add_layer_norm(x, r, w, b, p=p, seed=seed + 9, sequence=2, dim=dim, eps=EPS)
    gy, gh = _rand(shape, dtype, seed + 3), _rand(shape, dtype, seed + 4)
    grads = list(torch.autograd.grad((y, h), leaves, (gy, gh), retain_graph=True))
    with torch.no_grad():
        assert torch.equal(h, oracle.dropout(x, p, seed + 9, 2, residual=r))
        ref = oracle.Norm(h, w, b, dim, EPS)
        oracle.within(y, ref.y, ref.y_bound(), "y")
        (dh, bound), *params_wanted = ref.backward(gy, gh)
        oracle.within(grads[1], dh, bound, "dresidual")
        keep = oracle.kept(0, x.numel(), p, seed + 9, 2).view(shape).cuda()
        scale = 1 / (1 - p) if p < 1 else 0.0
        dx = torch.where(keep, ref.dx_exact * scale, 0.0)
        dx_bound = (ref.dx_off + 4 * ref.u * ref.dx_exact.abs()) * scale + oracle.ROUNDOFF[dtype] * dx.abs() + oracle.STEP[dtype]
        oracle.within(grads[0], dx, dx_bound, "dx")
        wanted = params_wanted[:1] * (w is not None) + params_wanted[1:] * (b is not None)
        for name, got, (want, bound) in zip(("dw", "db"), grads[2:], wanted):
            oracle.within(got, want, bound, name)
    return y, h, leaves, (gy, gh), grads


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,length", [(1, 1), (3, 2), (5, 31), (40, 64), (9, 257), (33, 1000), (70, 1024), (4, 4096),
                                         (3, 8191), (2, 16384), (1, 50001), (2, 65536), (1, 140000), (1, 600000)])
def test_join_rows(serron, rows, length, dtype):
    _check_join(serron, (rows, length), 1, dtype, 0.3, "same" if length % 2 else "f32", length)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (2, 3, 5, 7), (3, 8, 4, 4), (2, 32, 16, 16), (1, 67, 9, 61), (2, 128, 14, 14),
                                   (2, 129, 6, 10), (1, 512, 8, 8), (1, 1024, 4, 6), (1, 1025, 3, 3), (1, 2053, 7, 2)])
def test_join_maps(serron, shape, dtype):
    _check_join(serron, shape, 1, dtype, 0.3, "f32" if shape[1] % 2 else "same", sum(shape))


@pytest.mark.parametrize("shape", [(12, 96), (3, 1001), (2, 10, 6, 6), (2, 10, 5, 5), (1, 3000, 3, 3)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_join_with_its_seed_in_a_tensor(serron, shape, dtype):
    x, r, gy, gh = (_rand(shape, dtype, k) for k in range(4))
    leaves = [x.requires_grad_(), r.requires_grad_()]
    out = []
    for seed in (77, torch.tensor(77, device="cuda")):
        y, h = serron.dropout_add_layer_norm(x, r, p=0.3, seed=seed, sequence=5)
        out.append([y, h, *torch.autograd.grad((y, h), leaves, (gy, gh))])
    for a, c in zip(*out):
        assert torch.equal(a, c)


@pytest.mark.parametrize("p", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("params", ["none", "weight", "bias", "f32"])
def test_join_probabilities_and_params(serron, p, params):
    for shape in ((12, 96), (2, 10, 6, 6)):
        _check_join(serron, shape, 1, torch.bfloat16, p, params)


@pytest.mark.parametrize("shape", [(12, 96), (2, 10, 6, 6), (2, 1500, 3, 3)])
def test_join_partial_gradients(serron, shape):
    """One output's gradient alone, one input's alone: what the whole backward gives with zeros for the other."""
    y, h, leaves, (gy, gh), _ = _check_join(serron, shape, 1, torch.float32, 0.3)
    zero = torch.zeros_like(gy)
    want = torch.autograd.grad((y, h), leaves, (gy, zero), retain_graph=True)
    for a, c in zip(torch.autograd.grad(y, leaves, gy, retain_graph=True), want):
        assert torch.equal(a, c)
    want = torch.autograd.grad((y, h), leaves, (zero, gh), retain_graph=True)
    got = torch.autograd.grad(h, leaves, gh, retain_graph=True, allow_unused=True)
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    assert torch.equal(got[1], gh)
    full = torch.autograd.grad((y, h), leaves, (gy, gh), retain_graph=True)
    for k in range(4):
        others = [t.detach().requires_grad_(i == k) for i, t in enumerate(leaves)]
        outs = serron.dropout_add_layer_norm(*others, p=0.3, seed=9, sequence=2, eps=EPS)
        outs, given = (outs, (gy, gh)) if k < 2 else (outs[:1], (gy,))
        assert torch.equal(torch.autograd.grad(outs, others[k], given)[0], full[k]), k


def test_join_views_and_layouts(serron):
    base, r = _rand((2, 12, 5, 6), torch.float16, 1), _rand((2, 12, 5, 6), torch.float16, 2)
    want = serron.dropout_add_layer_norm(base, r, p=0.3, seed=5)
    last = torch.channels_last
    padded = torch.empty(2 * base.numel() + 3, dtype=torch.float16, device="cuda")
    shifted = padded[1:1 + base.numel()].view(base.shape).copy_(base)
    for a, c in ((base.to(memory_format=last), r), (base, r.to(memory_format=last)), (shifted, r)):
        got = serron.dropout_add_layer_norm(a, c, p=0.3, seed=5)
        assert torch.equal(got[1], want[1])
        _normed(got[0], want[1])


# ------------------------------------------------------------------------------------------------
# the same again: run to run, on other streams, as layers
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(500, 1024), (6, 40, 33, 35), (16, 30001)])
def test_same_bits_every_time(serron, shape):
    first = _check_join(serron, shape, 1, torch.bfloat16, 0.2)[-1]
    for _ in range(3):
        for a, c in zip(first, _check_join(serron, shape, 1, torch.bfloat16, 0.2)[-1]):
            assert torch.equal(a, c)


def test_other_streams(serron):
    x, r = _rand((64, 32, 40, 40), torch.float32, 1), _rand((64, 32, 40, 40), torch.float32, 2)
    want = serron.dropout_add_layer_norm(x, r, p=0.5, seed=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(10_000_000)
        late = x * 2  # what follows reads it in the order of this stream
        got = serron.dropout_add_layer_norm(late * 0.5, r, p=0.5, seed=3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_modules(serron):
    torch.manual_seed(5)
    x, r = _rand((2, 6, 9, 9), torch.float32, 1), _rand((2, 6, 9, 9), torch.float32, 2)
    drop = serron.Dropout(0.5)
    a, b = drop(x), drop(x)
    assert not torch.equal(a, b)
    torch.manual_seed(5)
    assert torch.equal(drop(x), a) and torch.equal(drop(x), b)
    channels = serron.Dropout(0.5, unit=serron.DropoutUnit.CHANNEL)(x)
    assert set((channels != 0).flatten(2).float().mean(-1).flatten().tolist()) <= {0.0, 1.0}
    norm = serron.LayerNorm2d(6, device="cuda")
    join = serron.DropoutAddLayerNorm2d(6, 0.5, device="cuda")
    y, h = join(x, r)
    _normed(y, h)
    _normed(norm(h), h)
    assert not torch.equal(h, x + r)
    y, h = join.eval()(x, r)
    assert torch.equal(h, x + r)
    _normed(y, h)


def test_autocast_leaves_them_alone(serron):
    x = _rand((2, 6, 9, 9), torch.float16, 1)
    w, b = _params(6, torch.float16, "f32", 1)
    want = serron.layer_norm(x, w, b)
    with torch.autocast("cuda"):
        assert torch.equal(serron.layer_norm(x, w, b), want)
        assert serron.dropout(x.float(), seed=1).dtype == torch.float32


def test_example_learns(serron):
    """The operators together, as a network uses them: the example's loss falls, every parameter gets a gradient, and
    evaluation drops nothing."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "residual_denoiser.py")
    spec = importlib.util.spec_from_file_location("residual_denoiser", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    model, losses = example.train(60)
    assert losses[-1] < 0.5 * losses[0] and all(math.isfinite(v) for v in losses)
    model.eval()
    noisy, _ = example.batch(2, 32, torch.Generator("cuda").manual_seed(3))
    with torch.no_grad():
        assert torch.equal(model(noisy), model(noisy))
    for p in model.parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all())
