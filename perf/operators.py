"""Workloads of the layer operators: layer norm, dropout, and the two joined with a residual sum.

``listed()`` names the cases and ``draw()`` gives more of the same ranges.  ``run()`` makes one pass, either in
plain torch arithmetic (``own`` false) or through the package's public functions (``own`` true); ``exact()``
computes the same outputs in 64 bits.

The operators, for a tensor x of which one dimension of length L is normalised:

* layer norm: m = mean(x), v = mean((x - m)^2), y = (x - m) / sqrt(v + eps) * weight + bias;
* dropout: element (or unit) j is kept when u_j >= round(p * 2^32), u_j being word j % 4 of the Philox4x32-10
  block with key ``seed`` and counter (j // 4, sequence), both 64 bits wide, low word first;
  y = x / (1 - p) where kept, 0 elsewhere, plus the residual where there is one;
* the join: h = residual + dropout(x), a 32-bit sum rounded to the type of x, and y = layer norm of that h.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _case(op, shape, dim, dtype, *, train, params="f32", affine=True, p=0.0, unit="element", residual=False, name=None):
    case = {"op": op, "shape": "x".join(str(s) for s in shape), "dim": dim, "dtype": dtype, "train": train,
            "params": params, "affine": affine, "p": p, "unit": unit, "residual": residual}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # one token answered by a served model: latency alone
        _case("layer_norm", (1, 1024), -1, "bf16", train=False, name="norm one token"),
        # feature maps of the learnable-layer workload, normalised over their channels at every pixel
        _case("layer_norm", (64, 32, 256, 256), 1, "bf16", train=True, name="norm maps"),
        # a training batch of tokens, parameters in the activations' type
        _case("layer_norm", (8192, 1024), -1, "bf16", train=True, params="same", name="norm tokens"),
        # maps with odd sides and an odd number of channels
        _case("layer_norm", (5, 67, 97, 61), 1, "f32", train=True, name="norm ragged maps"),
        # few rows of great and odd length: whole images flattened before the norm
        _case("layer_norm", (33, 50001), -1, "f16", train=True, name="norm long rows"),
        # the small map of a unit test or a single image: latency
        _case("dropout", (1, 32, 16, 16), 1, "f32", train=True, p=0.1, name="drop small map"),
        # the end of a residual branch on the learnable-layer workload's maps
        _case("dropout", (64, 32, 256, 256), 1, "bf16", train=True, p=0.1, residual=True, name="drop maps"),
        # whole channels dropped, as convolutional networks do
        _case("dropout", (16, 64, 128, 128), 1, "f16", train=True, p=0.25, unit="channel", name="drop channels"),
        # an odd number of elements
        _case("dropout", (31, 333, 1021), 1, "f32", train=True, p=0.5, name="drop odd"),
        # one token answered by a served model: nothing dropped, residual sum and norm
        _case("join", (1, 2048), -1, "bf16", train=False, name="join one token"),
        # a residual block of a network on maps
        _case("join", (32, 64, 128, 128), 1, "bf16", train=True, p=0.1, name="join maps"),
        # a residual block of a network on tokens
        _case("join", (2048, 4096), -1, "f16", train=True, p=0.1, name="join tokens"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("layer_norm", "dropout", "join"))
    most = 1 << 25  # elements: an eighth of the largest listed case and more steps per element at most
    if rng.random() < 0.5:
        length = _log_int(rng, 8, 100000)
        shape, dim = (_log_int(rng, 1, max(1, min(100000, most // length))), length), -1
    else:
        channels = _log_int(rng, 8, 1024)
        h, w = _log_int(rng, 1, 256), _log_int(rng, 1, 256)
        shape, dim = (_log_int(rng, 1, max(1, min(64, most // (channels * h * w)))), channels, h, w), 1
        while math.prod(shape) > most:
            shape = (shape[0], shape[1], max(1, shape[2] // 2), shape[3])
    train = rng.random() < 0.75  # dropout without: an ensemble of masked passes, as for uncertainty
    p = 0.0 if op == "layer_norm" or (op == "join" and not train) else rng.choice((0.1, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)))
    unit = rng.choice(("element", "element", "channel", "sample")) if op == "dropout" else "element"
    # whole samples are dropped from a residual branch (stochastic depth); a few units alone may all be dropped
    residual = op == "dropout" and (unit == "sample" or shape[0] * shape[1] < 64 or rng.random() < 0.5)
    return _case(op, shape, dim, rng.choice(("f32", "f16", "bf16")), train=train, params=rng.choice(("f32", "same")),
                 affine=op == "dropout" or rng.random() < 0.8, p=p, unit=unit, residual=residual)


def _shape(case):
    return tuple(int(s) for s in case["shape"].split("x"))


def work(case):
    shape = _shape(case)
    n, length = math.prod(shape), shape[case["dim"]]
    size = 2 if case["dtype"] != "f32" else 4
    psize = 4 if case["params"] == "f32" else size
    params = 2 * length * psize if case["affine"] and case["op"] != "dropout" else 0
    if case["op"] == "layer_norm":
        # x in, y out; training: grad_output in, grad_input and the parameters' gradients out
        return {"bytes": (4 if case["train"] else 2) * n * size + (2 if case["train"] else 1) * params,
                "flops": (20 if case["train"] else 8) * n}
    if case["op"] == "dropout":
        # x (and the residual) in, y out; training: grad_output in, grad_input out
        return {"bytes": ((4 if case["train"] else 2) + int(case["residual"])) * n * size,
                "flops": (4 if case["train"] else 2) * n}
    # x and the residual in, h and y out; training: both outputs' gradients in, both inputs' gradients out
    return {"bytes": (8 if case["train"] else 4) * n * size + (2 if case["train"] else 1) * params,
            "flops": (26 if case["train"] else 10) * n}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    shape, dtype = _shape(case), _DTYPES[case["dtype"]]
    pdtype = torch.float32 if case["params"] == "f32" else dtype
    dim = case["dim"] % len(shape)
    length = shape[dim]
    along = [length if d == dim else 1 for d in range(len(shape))]

    def randn(s, to):
        return torch.randn(s, generator=gen, device=dev).to(to)

    def grad(t):
        return t.requires_grad_(case["train"])

    # activations: each channel with a level and a spread of its own
    level, spread = randn(along, torch.float32), 0.5 + torch.rand(along, generator=gen, device=dev)
    state = {"case": case, "dim": dim, "seed": (seed * 0x9E3779B97F4A7C15 + 1) % (1 << 62), "sequence": seed % 1000}
    state["x"] = grad((torch.randn(shape, generator=gen, device=dev) * spread + level).to(dtype))
    if case["residual"] or case["op"] == "join":
        state["residual"] = grad(randn(shape, dtype))
    if case["op"] != "dropout" and case["affine"]:
        state["weight"] = grad((1 + 0.2 * torch.randn(length, generator=gen, device=dev)).to(pdtype))
        state["bias"] = grad((0.2 * torch.randn(length, generator=gen, device=dev)).to(pdtype))
    if case["train"]:
        state["grad_y"] = randn(shape, dtype)
        if case["op"] == "join":
            state["grad_h"] = randn(shape, dtype)
    return state


def _span(case):
    """Elements that share one decision."""
    shape = _shape(case)
    return {"element": 1, "channel": math.prod(shape[2:]), "sample": math.prod(shape[1:])}[case["unit"]]


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import serron_b200 as serron

    case = state["case"]
    inputs = [state[k] for k in ("x", "residual", "weight", "bias") if k in state]
    weight, bias = state.get("weight"), state.get("bias")
    if case["op"] == "layer_norm":
        outputs = (serron.layer_norm(state["x"], weight, bias, dim=state["dim"], eps=_EPS),)
    elif case["op"] == "dropout":
        outputs = (serron.dropout(state["x"], case["p"], seed=state["seed"], sequence=state["sequence"],
                                  unit=serron.DropoutUnit(case["unit"]), residual=state.get("residual")),)
    else:
        outputs = serron.dropout_add_layer_norm(state["x"], state["residual"], weight, bias, p=case["p"],
                                                seed=state["seed"], sequence=state["sequence"], dim=state["dim"],
                                                eps=_EPS)
    if not case["train"]:
        return list(outputs)
    grads = [state[k] for k in ("grad_y", "grad_h") if k in state]
    return [*outputs, *torch.autograd.grad(outputs, inputs, grads)]


_M32 = 0xFFFFFFFF


def _philox(seed, sequence, blocks, device):
    """The Philox4x32-10 blocks 0 .. blocks-1 as an int64 tensor (blocks, 4) of 32-bit words."""
    j = torch.arange(blocks, device=device)
    c0, c1 = j & _M32, j >> 32
    c2, c3 = torch.full_like(j, sequence & _M32), torch.full_like(j, sequence >> 32)
    k0, k1 = seed & _M32, seed >> 32
    for _ in range(10):
        # products of 32-bit words: their 64 bits come out whole, though the sign may be set
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _M32) ^ c1 ^ k0, b & _M32, ((a >> 32) & _M32) ^ c3 ^ k1, a & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack((c0, c1, c2, c3), 1)


def _kept(state):
    """Which elements of x are kept."""
    case, x = state["case"], state["x"]
    span = _span(case)
    units = x.numel() // span
    words = _philox(state["seed"], state["sequence"], -(-units // 4), x.device).view(-1)[:units]
    kept = words >= round(case["p"] * 2**32)
    return kept.view(-1, 1).expand(units, span).reshape(x.shape)


def _along(v, x, dim):
    return v.float().view([-1 if d == dim else 1 for d in range(x.dim())])


def _norm_plain(state, x, residual_grad=None):
    """y, and in training the gradients of x (plus ``residual_grad``), weight and bias, in 32 bits."""
    dim, train = state["dim"], state["case"]["train"]
    others = [d for d in range(x.dim()) if d != dim]
    centred = x - x.mean(dim, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim, keepdim=True) + _EPS)
    normed = centred * rstd
    y = normed
    if "weight" in state:
        y = normed * _along(state["weight"], x, dim) + _along(state["bias"], x, dim)
    if not train:
        return y, None, []
    g = grad_y = state["grad_y"].float()
    grads = []
    if "weight" in state:
        g = grad_y * _along(state["weight"], x, dim)
        grads = [(grad_y * normed).sum(others).to(state["weight"].dtype), grad_y.sum(others).to(state["bias"].dtype)]
    grad_x = rstd * (g - g.mean(dim, keepdim=True) - normed * (g * normed).mean(dim, keepdim=True))
    return y, grad_x if residual_grad is None else grad_x + residual_grad, grads


@torch.no_grad()
def _run_plain(state):
    case, x = state["case"], state["x"]
    dtype, train = x.dtype, case["train"]
    scale = 1 / (1 - case["p"])
    if case["op"] == "layer_norm":
        y, grad_x, grads = _norm_plain(state, x.float())
        return [y.to(dtype), grad_x.to(dtype), *grads] if train else [y.to(dtype)]
    kept = _kept(state) if case["p"] > 0 else torch.ones_like(x, dtype=torch.bool)
    dropped = torch.where(kept, x.float() * scale, 0.0)
    if case["op"] == "dropout":
        y = dropped + state["residual"].float() if "residual" in state else dropped
        if not train:
            return [y.to(dtype)]
        grad_x = torch.where(kept, state["grad_y"].float() * scale, 0.0)
        return [y.to(dtype), grad_x.to(dtype), *([state["grad_y"]] if "residual" in state else [])]
    h = (state["residual"].float() + dropped).to(dtype)
    if not train:
        return [_norm_plain(state, h.float())[0].to(dtype), h]
    y, grad_h, grads = _norm_plain(state, h.float(), state["grad_h"].float())
    return [y.to(dtype), h, torch.where(kept, grad_h * scale, 0.0).to(dtype), grad_h.to(dtype), *grads]


# ------------------------------------------------------------------------------------------------
# the same in 64 bits
# ------------------------------------------------------------------------------------------------
def _mul_exact(c, m):
    """High and low 32-bit words of c * m, by 16-bit halves, so that no product passes 48 bits."""
    low, high = c * (m & 0xFFFF), c * (m >> 16)
    mid = (low >> 16) + (high & 0xFFFFFFFFFFFF)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _kept_exact(case, seed, sequence, numel, device):
    span = _span(case)
    units = numel // span
    counter = [torch.zeros(-(-units // 4), dtype=torch.int64, device=device) for _ in range(4)]
    counter[0] += torch.arange(-(-units // 4), device=device) % (1 << 32)
    counter[1] += torch.arange(-(-units // 4), device=device) // (1 << 32)
    counter[2] += sequence % (1 << 32)
    counter[3] += sequence // (1 << 32)
    for r in range(10):
        key = [(seed + r * 0x9E3779B9) % (1 << 32), ((seed >> 32) + r * 0xBB67AE85) % (1 << 32)]
        hi0, lo0 = _mul_exact(counter[0], 0xD2511F53)
        hi1, lo1 = _mul_exact(counter[2], 0xCD9E8D57)
        counter = [hi1 ^ counter[1] ^ key[0], lo1, hi0 ^ counter[3] ^ key[1], lo0]
    u = torch.stack(counter, 1).reshape(-1)[:units]
    return (u >= round(case["p"] * 2**32)).repeat_interleave(span)


def exact(case, seed):
    state = prepare(case, seed)
    names = [k for k in ("x", "residual", "weight", "bias") if k in state]
    wide = {k: state[k].detach().double().requires_grad_(case["train"]) for k in names}
    dim, x = state["dim"], wide["x"]

    def norm(t):
        t = t.movedim(dim, -1)
        d = t - t.sum(-1, keepdim=True) / t.shape[-1]
        y = d / (d.pow(2).sum(-1, keepdim=True) / t.shape[-1] + _EPS).sqrt()
        if "weight" in wide:
            y = y * wide["weight"] + wide["bias"]
        return y.movedim(-1, dim)

    if case["op"] != "layer_norm":
        kept = _kept_exact(case, state["seed"], state["sequence"], x.numel(), x.device).view(x.shape)
        x = torch.where(kept, x / (1 - case["p"]), torch.zeros((), dtype=torch.float64, device=x.device))
        if "residual" in wide:
            x = x + wide["residual"]
    if case["op"] == "join":
        # the norm is of h as it is returned, a 32-bit sum rounded to its type, with the gradient passed on as it is
        scaled = state["x"].detach().float() * (1 / (1 - case["p"]))
        rounded = (state["residual"].detach().float() + torch.where(kept.view(x.shape), scaled, 0.0)).to(state["x"].dtype)
        outputs = [norm(x + (rounded.double() - x.detach())), x]
    else:
        outputs = [norm(x) if case["op"] == "layer_norm" else x]
    if not case["train"]:
        return [o.detach() for o in outputs]
    grads = [state[k].double() for k in ("grad_y", "grad_h") if k in state]
    return [*(o.detach() for o in outputs), *torch.autograd.grad(outputs, [wide[k] for k in names], grads)]
