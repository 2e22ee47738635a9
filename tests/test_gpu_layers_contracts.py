"""Contracts of the layer operators on the GPU: the top of the index range, tiny spreads, what autograd may hand back,
captured graphs.  Bounds: layer_oracle.py."""

from __future__ import annotations

import pytest
import torch

from tests import layer_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def serron():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import serron_b200

    return serron_b200


def _signs(n, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    out = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    for part in out.split(1 << 27):
        part.copy_(torch.randint(0, 2, part.shape, generator=gen, device="cuda", dtype=torch.int8) * 2 - 1)
    return out


def _total(*factors):
    parts = zip(*(f.split(1 << 27) for f in factors))
    return sum(float(torch.stack(p).float().prod(0).sum(dtype=torch.float64)) for p in parts)


def _near(got, want, bound):
    """``want`` and ``got`` in pieces; bfloat16 results are rounded once more (2^-8 of values below 4)."""
    for k, part in enumerate(got.split(1 << 27)):
        off = (part.float() - want(slice(k << 27, (k << 27) + part.numel()))).abs().amax()
        assert float(off) <= bound + 2.0**-6, (k, float(off))


@pytest.mark.parametrize("inner", [1, 2])
def test_longest_dimension(serron, inner):
    """A dimension within a block's stride of 2^31: the index that ends a row's loop does not fit in 31 bits.

    x and grad_output are signs, so |x|, |xhat|, X of the bound are 1 and G is |w| = 1.  The longest chain is the join of
    65535 chunks, three roundings each, and about 200 within a chunk: K u = 0.012, three times that on y, nine on dx
    and (for one row) the formula's own product on dw."""
    length = (1 << 31) - 3
    chain = (3 * 65535 + 200) * 2.0**-24
    x = _signs(length * inner, 1)
    gy = _signs(length * inner, 2)
    shape = (1, length) if inner == 1 else (1, length, inner)
    # the columns of inner = 2 are rows of their own
    columns = [slice(i, None, inner) for i in range(inner)]
    sums = [(_total(x[c]) / length, _total(gy[c]) / length, _total(gy[c], x[c]) / length) for c in columns]
    leaves = [x.view(shape).requires_grad_()]
    if inner == 1:
        leaves += [torch.ones(length, dtype=torch.bfloat16, device="cuda").requires_grad_(),
                   torch.zeros(length, dtype=torch.bfloat16, device="cuda").requires_grad_()]
    y = serron.layer_norm(*leaves, dim=1, eps=0.0)
    grads = torch.autograd.grad(y, leaves, gy.view(shape))
    with torch.no_grad():
        for c, (m, g, gx) in zip(columns, sums):
            rstd = (1 - m * m) ** -0.5
            g_xhat = (gx - m * g) * rstd
            xc, gc = x[c], gy[c]
            _near(y.view(-1)[c], lambda s: (xc[s].float() - m) * rstd, 3 * chain)
            _near(grads[0].view(-1)[c], lambda s: rstd * (gc[s].float() - g - (xc[s].float() - m) * rstd * g_xhat), 9 * chain)
            if inner == 1:
                _near(grads[1], lambda s: gc[s].float() * (xc[s].float() - m) * rstd, 3 * chain)
                assert torch.equal(grads[2], gc)


def _rand(shape, dtype, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["rows", "channels_last", "transposed"])
def test_saved_tensors_kept_on_the_host(serron, name, dtype):
    """save_on_cpu packs into row-major memory; gradients are those without it, to the bit."""
    base = _rand((3, 24, 6, 10), dtype, 1)
    x = {"rows": base, "channels_last": base.to(memory_format=torch.channels_last),
         "transposed": base.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0)}[name]
    w, b, r, gy, gh = _rand((24,), torch.float32, 2), _rand((24,), torch.float32, 3), *(_rand(x.shape, dtype, k) for k in (4, 5, 6))
    leaves = [t.requires_grad_() for t in (x, r, w, b)]
    calls = [lambda: (serron.layer_norm(x, w, b),), lambda: (serron.dropout(x, 0.3, seed=torch.tensor(5, device="cuda")),),
             lambda: serron.dropout_add_layer_norm(x, r, w, b, p=0.3, seed=5)]
    for call in calls:
        want = torch.autograd.grad(call(), leaves, (gy, gh)[:len(call())], allow_unused=True)
        with torch.autograd.graph.save_on_cpu(pin_memory=True):
            outputs = call()
        got = torch.autograd.grad(outputs, leaves, (gy, gh)[:len(outputs)], allow_unused=True)
        for a, c in zip(got, want):
            assert a is c is None or torch.equal(a, c)


@pytest.mark.parametrize("shape", [(12, 96), (3, 1001), (2, 10, 6, 6), (2, 10, 5, 5)])
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.float16])
def test_an_unused_norm_has_no_part_in_gradients(serron, shape, dtype):
    """Rows that hold NaN or an infinity, and rows without spread at eps = 0, have no norm; the sum's gradient passes by."""
    x, r, gh = (_rand(shape, dtype, k) for k in (1, 2, 3))
    x.view(-1)[5], r.view(-1)[-1] = float("inf"), float("nan")
    leaves = [x.requires_grad_(), r.requires_grad_(), *(_rand((shape[1],), dtype, k).requires_grad_() for k in (4, 5))]
    _, h = serron.dropout_add_layer_norm(*leaves, p=0.3, seed=7, sequence=2, eps=0.0)
    gx, gr, gw, gb = torch.autograd.grad(h, leaves, gh)
    assert torch.equal(gx, oracle.dropout(gh, 0.3, 7, 2)) and torch.equal(gr, gh)
    assert not gw.any() and not gb.any()


def _scaled_signs(shape, dim, dtype, scale):
    """Signs of equal number in every row (a zero beside them where the length is odd), times a power of two."""
    length = shape[dim]
    row = torch.cat((torch.ones(length // 2), -torch.ones(length // 2), torch.zeros(length % 2))).double()
    moved = [s for d, s in enumerate(shape) if d != dim]
    return (row * scale).expand(*moved, length).movedim(-1, dim).contiguous().to("cuda", dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [2.0**-65, 2.0**-63, 2.0**50])
@pytest.mark.parametrize("shape,dim", [((9, 96), 1), ((9, 97), 1), ((40, 1024), 1), ((3, 20001), 1), ((2, 70000), 1),
                                       ((2, 24, 6, 6), 1), ((2, 24, 5, 7), 1), ((1, 1500, 2, 4), 1), ((1, 2100, 3, 3), 1)])
def test_gradients_of_any_spread(serron, shape, dim, scale, dtype):
    """rstd is up to 2^65, its square beyond float32; no term of the formula is.  Sums and squares of the signs are exact; the
    variance, 2^-130, is rounded to a multiple of 2^-149, which takes 2^-20 of it and 2^-21 of rstd, a 64th of the bounds'
    K u.  So those hold as at any scale."""
    x, r = _scaled_signs(shape, dim, dtype, scale), torch.zeros(shape, dtype=dtype, device="cuda")
    w, b = 1 + 0.3 * _rand((shape[dim],), torch.float32, 1), _rand((shape[dim],), torch.float32, 2)
    gy, gh = _rand(shape, dtype, 3), _rand(shape, torch.float32, 4) / scale
    leaves = [t.requires_grad_() for t in (x, r, w, b)]
    ref = oracle.Norm(x.detach(), w.detach(), b.detach(), dim, 0.0)
    y = serron.layer_norm(x, w, b, dim=dim, eps=0.0)
    with torch.no_grad():
        oracle.within(y, ref.y, ref.y_bound(), "y")
    grads = torch.autograd.grad(y, (x, w, b), gy)
    for name, got, (want, bound) in zip(("dx", "dw", "db"), grads, ref.backward(gy)):
        oracle.within(got, want, bound, name)
    gh = gh.to(dtype)
    outputs = serron.dropout_add_layer_norm(x, r, w, b, p=0.0, seed=0, dim=dim, eps=0.0)
    grads = torch.autograd.grad(outputs, leaves, (gy, gh))
    (want, bound), *_ = ref.backward(gy, gh)
    for got in grads[:2]:
        oracle.within(got, want, bound, "dx of the join")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("shape,dim", [((9, 96), 1), ((9, 97), 1), ((40, 1024), 1), ((2, 20000), 1), ((2, 140000), 1),
                                       ((2, 24, 6, 6), 1), ((2, 24, 5, 7), 1), ((1, 2100, 3, 3), 1)])
def test_statistics_of_no_variance(serron, shape, dim, dtype):
    """eps = 0: rstd is 1 / 0, an infinity, of every kernel; what is off the mean by less than squares can hold becomes an
    infinity with its sign, what is not off it is 0 / 0.  With eps it is finite."""
    tiny = 2.0**-80 if dtype != torch.float64 else 2.0**-600
    x = _scaled_signs(shape, dim, dtype, tiny)
    y = serron.layer_norm(x, dim=dim, eps=0.0)
    assert torch.equal(y.nan_to_num(0.0, posinf=1.0, neginf=-1.0), (x / tiny)) and torch.equal(y.isnan(), x == 0)
    level = torch.full(shape, 3.0, dtype=dtype, device="cuda")
    assert bool(serron.layer_norm(level, dim=dim, eps=0.0).isnan().all())
    assert not serron.layer_norm(level, dim=dim).any()
    _, stats = torch.ops.serron._layer_norm(level, None, None, dim, 0.0, True)
    assert bool((stats[0] == 3.0).all()) and bool((stats[1] == float("inf")).all())
    huge = _scaled_signs(shape, dim, dtype, 2.0**70 if dtype != torch.float64 else 2.0**600)  # an infinite variance: rstd 0
    assert not serron.layer_norm(huge, dim=dim, eps=0.0).any()


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.float16, torch.bfloat16])
def test_everything_is_dropped_whatever_the_words(serron, dtype):
    """The first word of this seed is 2^32 - 1, which no threshold in 32 bits is above."""
    seed = 1352247272
    assert oracle.philox(oracle.np.zeros(1, dtype="uint64"), 0, seed)[0, 0] == 0xFFFFFFFF
    for n in (1, 2, 7, 300):
        x = torch.full((n,), float("nan"), dtype=dtype, device="cuda")
        r = _rand((n,), dtype, 1)
        for given in (seed, torch.tensor(seed, device="cuda")):
            for unit in ("element", "sample"):
                assert not serron.dropout(x, 1.0, seed=given, unit=serron.DropoutUnit(unit)).any()
                assert torch.equal(serron.dropout(x, 1.0, seed=given, residual=r, unit=serron.DropoutUnit(unit)), r)
            assert torch.equal(serron.dropout_add_layer_norm(x, r, p=1.0, seed=given, dim=0)[1], r)


def test_layers_take_their_seed_from_memory_in_a_graph(serron):
    """Replays drop what the seed in the tensor says, forward and backward, as the functions do without a graph."""
    x, r, gy, gh = (_rand((2, 6, 9, 9), torch.float32, k) for k in range(4))
    leaves = [t.requires_grad_() for t in (x, r)]
    drop = serron.Dropout(0.5, unit=serron.DropoutUnit.CHANNEL)
    join = serron.DropoutAddLayerNorm2d(6, 0.5, device="cuda")
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step(seed):
        y, h = join(drop(x, seed=seed, sequence=1), r, seed=seed, sequence=2)
        return y, h, *torch.autograd.grad((y, h), (*leaves, join.weight, join.bias), (gy, gh))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(seed)
        with pytest.raises(RuntimeError, match="every replay"):
            drop(x)
        with pytest.raises(RuntimeError, match="every replay"):
            join(x, r)
    seen = []
    for value in (3, 4):
        seed.fill_(value)
        graph.replay()
        for a, c in zip(out, step(value)):
            assert torch.equal(a, c)
        seen.append(out[1].clone())
    assert not torch.equal(*seen)


@pytest.mark.parametrize("p", [0.0, 2.0**-32, 1 - 2.0**-32, 1.0])
@pytest.mark.parametrize("shape", [(2, 10, 5, 5), (1, 67, 3, 7), (3, 1001)])
def test_join_of_odd_sizes_at_the_ends_of_p(serron, shape, p):
    """One element an access on maps of 25 and 21 pixels, shifted vectors on rows of 1001."""
    for dtype in (torch.float32, torch.float16):
        x, r, gy, gh = (_rand(shape, dtype, k) for k in range(4))
        w, b = (_rand((shape[1],), torch.float32, k) for k in (5, 6))
        leaves = [t.requires_grad_() for t in (x, r, w, b)]
        y, h = serron.dropout_add_layer_norm(*leaves, p=p, seed=8, sequence=3)
        grads = torch.autograd.grad((y, h), leaves, (gy, gh))
        with torch.no_grad():
            assert torch.equal(h, oracle.dropout(x, p, 8, 3, residual=r))
            ref = oracle.Norm(h, w, b, 1, 1e-5)
            oracle.within(y, ref.y, ref.y_bound(), "y")
            (dh, bound), *others = ref.backward(gy, gh)
            oracle.within(grads[1], dh, bound, "dresidual")
            for got, (want, off) in zip(grads[2:], others):
                oracle.within(got, want, off, "dw, db")
            if p in (0.0, 2.0**-32):  # with 2^-32 the only word below the threshold is 0: none of these
                assert torch.equal(grads[0], grads[1])
            if p == 1.0:
                assert not grads[0].any()


def test_operators_are_as_torch_wants_them(serron):
    """Schemas, fake kernels and autograd registrations against the real kernels."""
    ops = torch.ops.serron
    for shape, dim in (((2, 6, 4, 5), 1), ((7, 24), -1)):
        x = _rand(shape, torch.float32, 1).requires_grad_()
        if len(shape) == 4:
            x = x.detach().to(memory_format=torch.channels_last).requires_grad_()
        w, b = (_rand((shape[dim],), torch.float32, k).requires_grad_() for k in (2, 3))
        utils = ("test_schema", "test_autograd_registration", "test_faketensor")
        seed = torch.tensor(5, device="cuda")
        torch.library.opcheck(ops.layer_norm, (x, w, b, dim, 1e-5), test_utils=utils)
        torch.library.opcheck(ops.layer_norm, (x, None, None, dim, 1e-5), test_utils=utils)
        torch.library.opcheck(ops.dropout, (x, x, 1, 0.3, 7, seed, 2), test_utils=utils)
        torch.library.opcheck(ops.dropout_add_layer_norm, (x, x, w, b, 0.3, 7, None, 2, dim, 1e-5), test_utils=utils)


def test_traced_calls_compute(serron):
    """What a tracer recorded gives another input its own outputs."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def f(x, r, w, b):
        y, h = serron.dropout_add_layer_norm(serron.layer_norm(x, w, b), r, w, b, p=0.3, seed=5)
        return serron.dropout(y, 0.2, seed=6, residual=h)

    args, others = ([*(_rand((2, 6, 9, 9), torch.float32, s + k) for k in (1, 2)),
                     *(_rand((6,), torch.float32, s + k) for k in (3, 4))] for s in (0, 10))
    for traced in (make_fx(f)(*args), torch.jit.trace(f, tuple(args))):
        assert torch.equal(traced(*others), f(*others))


def test_function_transforms_and_tangents(serron):
    x, w, b = _rand((5, 8), torch.float32, 1), _rand((8,), torch.float32, 2), _rand((8,), torch.float32, 3)

    def f(v):
        return serron.dropout(serron.layer_norm(v, w, b, dim=0), 0.3, seed=5).square().sum()

    got = torch.func.vmap(torch.func.grad(f))(x)
    for row, g in zip(x, got):
        leaf = row.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(f(leaf), leaf)[0], g)
    with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
        torch.func.jvp(f, (x[0],), (x[1],))


def test_backward_follows_its_stream_and_runs_in_threads(serron):
    """A node runs on the stream of its forward pass, and nodes of other graphs at the same time."""
    import threading

    x, r, gy, gh = (_rand((8, 32, 40, 40), torch.float32, k) for k in range(4))
    w, b = (_rand((32,), torch.float32, k) for k in (5, 6))
    leaves = [t.requires_grad_() for t in (x, r, w, b)]

    def step():
        outputs = serron.dropout_add_layer_norm(*leaves, p=0.3, seed=5)
        return torch.autograd.grad(outputs, leaves, (gy, gh))

    want = step()
    torch.cuda.synchronize()
    results = {}

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                results[k] = step()
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(4):
        for a, c in zip(results[k], want):
            assert torch.equal(a, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = [t.detach().clone().requires_grad_() for t in leaves]
        outputs = serron.dropout_add_layer_norm(*late, p=0.3, seed=5)
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(torch.autograd.grad(outputs, late, (gy, gh)), want):  # from the default stream
        assert torch.equal(a, c)


def test_recomputed_layers_draw_the_same_mask(serron):
    from torch.utils.checkpoint import checkpoint

    x, r = (_rand((2, 6, 9, 9), torch.float32, k).requires_grad_() for k in (1, 2))
    join = serron.DropoutAddLayerNorm2d(6, 0.5, device="cuda")
    grads = []
    for again in (False, True):
        torch.manual_seed(3)
        y, h = checkpoint(join, x, r, use_reentrant=False) if again else join(x, r)
        grads.append(torch.autograd.grad((y * 2 + h).square().sum(), (x, r, join.weight)))
    for a, c in zip(*grads):
        assert torch.equal(a, c)
