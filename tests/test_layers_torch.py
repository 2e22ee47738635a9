"""The layer operators as torch sees them, without a GPU: what tracers, fake tensors, function transforms and autograd
make of them.  Plain kernels for CPU tensors stand in for the CUDA ones while a test runs; like those, they walk the
memory of their tensors, and keep statistics in its order."""

from __future__ import annotations

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import serron_b200 as serron
from serron_b200 import _layer_ops
from tests import layer_oracle

EPS = 1e-5


def _dense(x):
    return torch.empty_like(x).stride() == x.stride()


def _rows(t, like, dim):
    """The rows along ``dim`` of ``t``, read through the strides of ``like`` from the memory of ``t``."""
    order = sorted(range(like.dim()), key=lambda d: -like.stride(d))
    memory = t.as_strided((t.numel(),), (1,))
    return memory.view([like.shape[d] for d in order]).movedim(order.index(dim), -1)


def _stand_in_norm(x, w, b, dim, eps, stats):
    x = x if _dense(x) else x.contiguous()
    rows = _rows(x, x, dim)
    mean = rows.mean(-1, keepdim=True)
    rstd = ((rows - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    y = torch.empty_like(x)
    _rows(y, x, dim).copy_((rows - mean) * rstd * (1 if w is None else w) + (0 if b is None else b))
    return y, torch.stack((mean.flatten(), rstd.flatten())) if stats else None


def _stand_in_norm_backward(gy, x, stats, w, dim, params, wanted):
    x = x if _dense(x) else x.contiguous()
    gy = torch.empty_like(x).copy_(gy)
    rows, g0 = _rows(x, x, dim), _rows(gy, x, dim)
    mean, rstd = (s.view(rows.shape[:-1]).unsqueeze(-1) for s in stats)
    xhat = (rows - mean) * rstd
    g = g0 if w is None else g0 * w
    dx = torch.empty_like(x)
    _rows(dx, x, dim).copy_(rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True)))
    lead = list(range(rows.dim() - 1))
    return (dx if wanted[0] else None, (g0 * xhat).sum(lead).to(params) if wanted[1] else None,
            g0.sum(lead).to(params) if wanted[2] else None)


def _stand_in_dropout(x, residual, span, p, seed, seed_tensor, sequence):
    seed = (int(seed_tensor) if seed_tensor is not None else seed) % (1 << 64)
    y = layer_oracle.dropout(x.contiguous(), p, seed, sequence % (1 << 64), span)
    return y if residual is None else y + residual


def _stand_in_join(x, r, w, b, p, seed, seed_tensor, sequence, dim, eps, stats):
    h = _stand_in_dropout(x, r.contiguous(), 1, p, seed, seed_tensor, sequence)
    y, s = _stand_in_norm(h, w, b, dim, eps, stats)
    return y, h, s


def _stand_in_join_backward(gy, gh, h, stats, w, dim, params, p, seed, seed_tensor, sequence, wanted):
    dh, dw, db = _stand_in_norm_backward(gy, h.contiguous(), stats, w, dim, params, (True, *wanted[2:]))
    dh = dh if gh is None else dh + gh
    dx = _stand_in_dropout(dh, None, 1, p, seed, seed_tensor, sequence)
    return dx if wanted[0] else None, dh if wanted[1] else None, dw, db


@pytest.fixture
def layers():
    """The compiled binding, with kernels for CPU tensors."""
    binding = _layer_ops.binding()
    library = torch.library.Library("serron", "IMPL")
    for name, kernel in (("_layer_norm", _stand_in_norm), ("_layer_norm_backward", _stand_in_norm_backward),
                         ("dropout", _stand_in_dropout), ("_dropout_add_layer_norm", _stand_in_join),
                         ("_dropout_add_layer_norm_backward", _stand_in_join_backward)):
        library.impl(name, kernel, "CPU")
    yield binding
    library._destroy()


def _tensors(shape, dim, seed=1):
    gen = torch.Generator().manual_seed(seed)
    draw = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    return draw(*shape), draw(*shape), 1 + 0.3 * draw(shape[dim]), draw(shape[dim])


def _plain_norm(x, w, b, dim):
    along = [-1 if d == dim else 1 for d in range(x.dim())]
    d = x - x.mean(dim, keepdim=True)
    return d * (d.square().mean(dim, keepdim=True) + EPS).rsqrt() * w.view(along) + b.view(along)


def _plain_drop(x, p=0.3, seed=7, sequence=2):
    keep = layer_oracle.kept(0, x.numel(), p, seed, sequence).view(x.shape)
    return torch.where(keep, x / (1 - p), torch.zeros((), dtype=x.dtype))


def _functions(layers, dim=1):
    """(operator, plain form) pairs of the arguments x, r, w, b."""
    def join(x, r, w, b):
        y, h = layers.dropout_add_layer_norm(x, r, w, b, 0.3, 7, None, 2, dim, EPS)
        return y * 2 + h

    def plain_join(x, r, w, b):
        h = r + _plain_drop(x)
        return _plain_norm(h, w, b, dim) * 2 + h

    return {
        "layer_norm": (lambda x, r, w, b: layers.layer_norm(x, w, b, dim, EPS) + r,
                       lambda x, r, w, b: _plain_norm(x, w, b, dim) + r),
        "dropout": (lambda x, r, w, b: layers.dropout(x, r, 1, 0.3, 7, None, 2), lambda x, r, w, b: _plain_drop(x) + r),
        "join": (join, plain_join),
    }


NAMES = ["layer_norm", "dropout", "join"]


def _close(a, b):
    torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-11)


@pytest.mark.parametrize("name", NAMES)
def test_gradients(layers, name):
    args = [t.requires_grad_() for t in _tensors((3, 5, 4), 1)]
    f, plain = _functions(layers)[name]
    y, want = f(*args), plain(*args)
    _close(y, want)
    gy = torch.randn_like(y)
    got = torch.autograd.grad(y, args, gy, allow_unused=True)
    want = torch.autograd.grad(want, args, gy, allow_unused=True)
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        if a is not None:
            _close(a, b)


@pytest.mark.parametrize("name", NAMES)
def test_jit_trace_records_the_operator(layers, name):
    f, _ = _functions(layers)[name]
    traced = torch.jit.trace(f, _tensors((3, 5, 4), 1), check_trace=False)
    assert "serron::" in str(traced.graph)
    other = _tensors((3, 5, 4), 1, seed=2)
    _close(traced(*other), f(*other))


@pytest.mark.parametrize("name", NAMES)
def test_fx_trace_records_the_operator_and_its_gradient(layers, name):
    f, plain = _functions(layers)[name]

    def step(*args):
        leaves = [t.detach().requires_grad_() for t in args]
        y = f(*leaves)
        return [y, *(g for g in torch.autograd.grad(y.sum(), leaves, allow_unused=True) if g is not None)]

    traced = make_fx(step)(*_tensors((3, 5, 4), 1))
    assert "serron" in str(traced.graph)
    other = _tensors((3, 5, 4), 1, seed=2)
    for a, b in zip(traced(*other), step(*other), strict=True):
        _close(a, b)


def test_fake_tensors_have_the_shapes_and_strides(layers):
    """A fake tensor says that it is on a GPU, and no GPU is needed (but for autograd's engine, which asks the driver)."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.serron
    with FakeTensorMode():
        for dtype, params in ((torch.bfloat16, torch.float32), (torch.float16, torch.float16)):
            x = torch.empty(2, 6, 4, 5, dtype=dtype, device="cuda").to(memory_format=torch.channels_last)
            w = torch.empty(6, dtype=params, device="cuda")
            y = serron.layer_norm(x.requires_grad_(), w, w)
            assert y.shape == x.shape and y.dtype == dtype and y.stride() == x.stride() and y.device.type == "cuda"
            assert y.requires_grad
            assert serron.layer_norm(x[..., ::2]).is_contiguous()
            assert serron.dropout(x, 0.3, seed=1).is_contiguous()
            y, h = serron.dropout_add_layer_norm(x, x, w, None, p=0.3, seed=1)
            assert y.shape == h.shape == x.shape and y.is_contiguous() and h.dtype == dtype
            x = x.detach()
            _, stats = ops._layer_norm(x, w, w, 1, EPS, True)
            assert stats.shape == (2, 40) and stats.dtype == torch.float32
            for wanted in ((True, True, True), (False, True, False)):
                dx, dw, db = ops._layer_norm_backward(y, x, stats, w, 1, params, wanted)
                assert (dx is not None) == wanted[0] and (db is not None) == wanted[2]
                assert dw.shape == w.shape and dw.dtype == params
                assert dx is None or dx.stride() == x.stride()
            dx, dr, dw, db = ops._dropout_add_layer_norm_backward(y, None, h, stats, w, 1, params, 0.3, 1, None, 0,
                                                                  (True, True, True, False))
            assert dx.shape == dr.shape == x.shape and dw.dtype == params and db is None


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms(layers, name):
    """Gradients of functions, and many of them at once (the mask then being each sample's own call's)."""
    f, plain = _functions(layers, dim=0)[name]
    args = _tensors((5, 4), 0)
    got = torch.func.grad(lambda *a: f(*a).sin().sum(), argnums=(0, 1))(*args)
    want = torch.func.grad(lambda *a: plain(*a).sin().sum(), argnums=(0, 1))(*args)
    for a, b in zip(got, want):
        _close(a, b)
    xs = torch.stack([args[0], 2 * args[1], args[0] + args[1]])
    per_sample = torch.func.vmap(torch.func.grad(lambda x: f(x, *args[1:]).sin().sum()))(xs)
    for x, g in zip(xs, per_sample):
        _close(g, torch.func.grad(lambda x: plain(x, *args[1:]).sin().sum())(x))


@pytest.mark.parametrize("name", ["layer_norm", "join"])
def test_second_derivatives_are_refused(layers, name):
    """However they are asked for: neither zero nor part of one comes back."""
    f, _ = _functions(layers)[name]
    if name == "layer_norm":
        f = lambda x, r, w, b: layers.layer_norm(x, w, b, 1, EPS)  # noqa: E731
    x, r, w, b = _tensors((3, 5, 4), 1)
    leaf = x.clone().requires_grad_()
    g = torch.autograd.grad(f(leaf, r, w, b).square().sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.func.grad(lambda v: torch.func.grad(lambda x: f(x, r, w, b).sin().sum())(v).sin().sum())(x)
    for leaf in (x.clone().requires_grad_(), x.transpose(0, 1)[..., ::2].requires_grad_()):  # the second one is copied
        v = r if leaf.shape == r.shape else r.transpose(0, 1)[..., ::2]
        g = torch.autograd.grad(f(leaf, v, None, None).sum(), leaf, create_graph=True)[0]
        with pytest.raises(RuntimeError, match="once_differentiable"):
            torch.autograd.grad((g * leaf).sum(), leaf)  # it reaches the leaf by another way too
    y = f(x, r, w.requires_grad_(), b)
    gy = torch.ones_like(y, requires_grad=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(torch.autograd.grad(y, w, gy, create_graph=True)[0].sum(), gy)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("which", range(4))
def test_forward_mode_is_refused(layers, name, which):
    """There are no forward-mode derivatives, and an output without a tangent would pass for a constant."""
    f, _ = _functions(layers)[name]
    args = list(_tensors((3, 5, 4), 1))
    if (name, which) in (("layer_norm", 1), ("dropout", 2), ("dropout", 3)):
        return  # not an argument of the operator
    with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
        torch.func.jvp(lambda v: f(*args[:which], v, *args[which + 1:]), (args[which],), (torch.ones_like(args[which]),))
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        args[which] = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            f(*args)


@pytest.mark.parametrize("name", NAMES)
def test_tangents_of_gradients_are_refused(layers, name):
    """Forward over reverse: the gradient that comes to a node carries the tangent."""
    f, _ = _functions(layers)[name]
    x, r, w, b = (t.requires_grad_() for t in _tensors((3, 5, 4), 1))
    y = f(x, r, w, b)
    with torch.autograd.forward_ad.dual_level():
        gy = torch.autograd.forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            torch.autograd.grad(y, x, gy)


def test_dropout_is_linear_in_its_gradient(layers):
    """Its backward pass is dropout again, with all of its derivatives."""
    x, r, *_ = _tensors((3, 5, 4), 1)
    x.requires_grad_()
    r.requires_grad_()
    g = torch.autograd.grad((layers.dropout(x, None, 1, 0.3, 7, None, 2) * r).square().sum(), x, create_graph=True)[0]
    want = torch.autograd.grad((_plain_drop(x) * r).square().sum(), x, create_graph=True)[0]
    _close(g, want)
    for a, b in zip(torch.autograd.grad(g.sum(), (x, r)), torch.autograd.grad(want.sum(), (x, r))):
        _close(a, b)


def test_views_with_a_pending_sign_or_conjugation(layers):
    """torch negates such a view when it is read; the operators read the negated values."""
    x, r, w, b = _tensors((3, 5, 4), 1)
    for view in (torch._neg_view(x), torch.complex(r, x).conj().imag):
        assert view.is_neg()
        leaf = view.detach().requires_grad_()
        y = layers.layer_norm(leaf, w, b, 1, EPS)
        _close(y, _plain_norm(-x, w, b, 1))
        _close(layers.dropout(view, view, 1, 0.3, 7, None, 2), _plain_drop(-x) - x)
        gy = torch._neg_view(r)
        want = torch.autograd.grad(_plain_norm(leaf, w, b, 1), leaf, -r)[0]
        _close(torch.autograd.grad(y, leaf, gy)[0], want)


@pytest.mark.parametrize("call,pattern", [
    (lambda o, x, w: o.layer_norm(x, w[:3], None, 1, EPS), "must have the shape"),
    (lambda o, x, w: o.layer_norm(x, w, w.float(), 1, EPS), "share a dtype"),
    (lambda o, x, w: o.layer_norm(x, w, None, 3, EPS), "out of range"),
    (lambda o, x, w: o.layer_norm(x, torch.ones(5, dtype=x.dtype), None, 1, EPS), "one device"),
    (lambda o, x, w: o._layer_norm_backward(x[:1], x, w, None, 1, w.dtype, [True] * 3), "shape and dtype"),
    (lambda o, x, w: o._layer_norm_backward(x, x, w, None, 1, w.dtype, [True] * 3), "statistics of another input"),
    (lambda o, x, w: o._layer_norm_backward(x, x, x.new_empty(2, 12), w.float(), 1, w.dtype, [True] * 3), "weight of"),
    (lambda o, x, w: o._dropout_add_layer_norm_backward(x, None, x, x.new_empty(2, 12), w, 1, torch.float32, 0.3, 7, None,
                                                        2, [True] * 4), "weight of"),
    (lambda o, x, w: o.dropout(x, x[:1], 1, 0.3, 7, None, 2), "shape and dtype"),
    (lambda o, x, w: o.dropout(x, None, 1, 0.3, 7, w, 2), "one int64"),
    (lambda o, x, w: o.dropout_add_layer_norm(x, x.float(), None, None, 0.3, 7, None, 2, 1, EPS), "shape and dtype"),
    (lambda o, x, w: o.dropout_add_layer_norm(x, x, None, w[1:], 0.3, 7, None, 2, 1, EPS), "must have the shape"),
])
def test_the_operators_refuse_what_leaves_their_tensors(call, pattern):
    """torch.ops is open to all: the checks that memory depends on are the operators' own (here of tensors without memory)."""
    _layer_ops.binding()
    x, w = (torch.empty(s, dtype=torch.float64, device="meta") for s in ((3, 5, 4), (5,)))
    with pytest.raises(RuntimeError, match=pattern):
        call(torch.ops.serron, x, w)


def test_no_kernel_for_cpu_tensors():
    _layer_ops.binding()
    x = torch.rand(2, 3)
    with pytest.raises(NotImplementedError, match="CPU"):
        torch.ops.serron.layer_norm(x, None, None, 1, EPS)
    with pytest.raises(NotImplementedError, match="CPU"):
        torch.ops.serron.dropout(x, None, 1, 0.3, 7, None, 2)


HOOKS = {
    "contiguous": lambda t: t.contiguous(),
    "reversed": lambda t: t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim()))),
    "strided": lambda t: torch.stack((t, t + 1), -1)[..., 0],
}


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("order", [(0, 1, 2, 3), (0, 2, 3, 1), (3, 0, 1, 2)])
def test_hooks_may_bring_saved_tensors_back_in_another_order(layers, order, hook):
    """What a hook returns has the values of what it was given, and not its strides (torch's save_on_cpu packs into
    row-major memory)."""
    shape = (2, 3, 4, 5)
    memory, other, w, b = _tensors([shape[d] for d in order], order.index(1))
    x = memory.permute(*[order.index(d) for d in range(4)])
    r = other.reshape(shape)
    assert x.shape == shape
    for name in NAMES:
        f, _ = _functions(layers)[name]
        leaves = [t.detach().requires_grad_() for t in (x, r, w, b)]
        want = torch.autograd.grad(f(*leaves).sin().sum(), leaves, allow_unused=True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, HOOKS[hook]):
            y = f(*leaves).sin().sum()
        for a, c in zip(torch.autograd.grad(y, leaves, allow_unused=True), want):
            assert (a is None) == (c is None)
            if a is not None:
                _close(a, c)


@pytest.mark.parametrize("change", [lambda t: t.float(), lambda t: t[:1]])
def test_hooks_that_change_a_saved_tensor_are_refused(layers, change):
    """Another dtype or size would be read past its end."""
    x, r, w, b = _tensors((3, 5, 4), 1)
    leaf, w = x.to("meta").requires_grad_(), w.to("meta")
    for f in (lambda: layers.layer_norm(leaf, w, None, 1, EPS),
              lambda: layers.dropout_add_layer_norm(leaf, leaf, w, None, 0.3, 7, None, 2, 1, EPS)[0]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y = f()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaf, torch.empty_like(y))


def test_an_unused_norm_has_no_part_in_gradients(layers):
    """A row that holds an infinity has no norm, and the sum's gradient passes it by where only the sum is used."""
    x, r, w, b = _tensors((3, 5, 4), 1)
    x[0, 2, 1], r[1, 0, 0] = float("inf"), float("nan")
    leaves = [t.requires_grad_() for t in (x, r, w, b)]
    _, h = layers.dropout_add_layer_norm(*leaves, 0.3, 7, None, 2, 1, EPS)
    gh = torch.randn_like(h)
    gx, gr, gw, gb = torch.autograd.grad(h, leaves, gh, create_graph=True)
    assert torch.equal(gx, layer_oracle.dropout(gh, 0.3, 7, 2)) and torch.equal(gr, gh)
    assert not gw.any() and not gb.any()


def test_layers_do_not_draw_seeds_for_a_graph(monkeypatch):
    """A capture would freeze the drawn seed; the layers say so before anything runs."""
    class OnGpu:
        is_cuda, dtype, device, shape = True, torch.float32, torch.device("cuda"), (2, 3)

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="every replay"):
        serron.Dropout(0.3)(OnGpu())
    with pytest.raises(RuntimeError, match="every replay"):
        serron.DropoutAddLayerNorm2d(3, 0.3)(OnGpu(), OnGpu())
    assert isinstance(serron.Dropout(0.3).eval()(OnGpu()), OnGpu)


@pytest.mark.parametrize("name", NAMES)
def test_inference_mode(layers, name):
    """Below autograd altogether, with tensors from inside and from outside."""
    f, _ = _functions(layers)[name]
    outside = _tensors((3, 5, 4), 1)
    want = f(*outside)
    with torch.inference_mode():
        _close(f(*outside), want)
        _close(f(*(t.clone() for t in outside)), want)
        assert not f(*outside).requires_grad
