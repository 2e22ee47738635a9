"""Autograd functions over the compiled operators.

Contract as packages/serron/torch-ext/serron/autograd.py:32-123: the input and the structuring
element are promoted to their common dtype and saved; the backward casts ``grad_output`` to that dtype
and returns grads only for the inputs that want them.

B200 difference: the forward also writes one winner record per output, and the backward gathers
straight from those records instead of searching every window again.  Without autocast the records come
from the forward itself.  Under CUDA autocast the value is computed on float16 casts while the backward
works in the promoted dtype, exactly like the reference; for odd square windows of 3 to 15 with a
float32 structuring element one kernel computes the float16 value and the promoted (float32) winners in
the same pass (so the promoted copy of the input is never made); other autocast calls keep no records
and the backward searches the windows itself.  After the autocast forward the backward reads the float16
``grad_output`` and writes ``grad_input`` in the input's dtype directly (float32 sums in between), which
gives the values of the reference's casts up and down without making the copies.

The layer operators at the end (layer norm, dropout and their join) have no reference counterpart.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _flatness, _layer_ops, _lib, _ops
from ._autotune import ensure_loaded, select_algorithm
from ._ops import add_op_namespace_prefix, ops
from .enums import Algorithm

__all__ = ["_DilateFunction", "_ErodeFunction", "add_op_namespace_prefix", "ops"]


def _match_dtype(input_: torch.Tensor, kernel: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(input_, kernel)`` cast to ``torch.promote_types`` of their dtypes."""
    dtype = torch.promote_types(input_.dtype, kernel.dtype)
    return input_.to(dtype), kernel.to(dtype)


def _autocast_cast(t: torch.Tensor) -> torch.Tensor:
    """The cast CUDA autocast applies to serron::erode/dilate arguments (float16; float64 untouched)."""
    if t.is_cuda and t.is_floating_point() and t.dtype is not torch.float64:
        return t.to(torch.float16)
    return t


def _forward(ctx, op: int, input_: torch.Tensor, kernel: torch.Tensor, border: int, algo: int) -> torch.Tensor:
    ensure_loaded(input_.device)
    flat = _flatness.is_flat(kernel)
    ctx.border = border
    ctx.flat = flat
    ctx.algo = int(algo)
    ctx.op = op
    ctx.winners = None
    ctx.winners_format = 0
    ctx.widened = False
    ctx.input_dtype = input_.dtype
    # grad mode is off inside Function.forward; needs_input_grad says whether a backward can follow
    wants_grad = any(ctx.needs_input_grad[:2])
    ctx.dtype = torch.promote_types(input_.dtype, kernel.dtype)
    if (wants_grad and int(algo) == 0 and input_.is_cuda and torch.is_autocast_enabled("cuda")
            and ctx.dtype == torch.float32 and _ops.autocast_fused_ok(input_, kernel.to(ctx.dtype))):
        kernel = kernel.to(ctx.dtype)
        ctx.save_for_backward(kernel)
        y, ctx.winners, ctx.winners_format = _ops.forward_autocast(op, input_, kernel, border)
        ctx.widened = True
        return y
    input_, kernel = _match_dtype(input_, kernel)
    ctx.save_for_backward(kernel, input_)
    algo = int(algo) or select_algorithm(input_, kernel, flat, backward=False)
    x, k = input_, kernel
    if input_.is_cuda and torch.is_autocast_enabled("cuda"):
        x, k = _autocast_cast(input_), _autocast_cast(kernel)
    if wants_grad and x.dtype == input_.dtype and input_.is_cuda and kernel.is_cuda:
        y, ctx.winners, ctx.winners_format = _ops.forward_with_winners(op, x, k, border, flat, algo)
        return y
    return _ops.forward(op, x, k, border, flat, algo)


def _backward(ctx, grad_output: torch.Tensor):
    needs_input, needs_kernel = ctx.needs_input_grad[:2]
    if not (needs_input or needs_kernel):
        return None, None, None, None
    kernel = ctx.saved_tensors[0]
    if ctx.widened and grad_output.dtype in (torch.float16, torch.bfloat16, torch.float32):
        # the casts of grad_output up to float32 and of grad_input down to the input's dtype happen inside
        # the gather (the same values, without the two copies)
        grad_input, grad_kernel = _ops.backward_from_winners_widened(
            ctx.op, grad_output, ctx.winners, ctx.winners_format, kernel, ctx.border, needs_kernel, ctx.input_dtype)
        return (grad_input if needs_input else None), (grad_kernel if needs_kernel else None), None, None
    grad_output = grad_output.to(ctx.dtype).contiguous()
    if ctx.winners is not None:
        grad_input, grad_kernel = _ops.backward_from_winners(ctx.op, grad_output, ctx.winners, ctx.winners_format,
                                                             kernel, ctx.border, needs_kernel)
    else:
        input_ = ctx.saved_tensors[1]
        algo = ctx.algo or select_algorithm(input_, kernel, ctx.flat, backward=True)
        grad_input, grad_kernel = _ops.backward(ctx.op, grad_output, input_, kernel, ctx.border, ctx.flat,
                                                needs_kernel, algo)
    return (grad_input if needs_input else None), (grad_kernel if needs_kernel else None), None, None


class _ErodeFunction(torch.autograd.Function):
    """Autograd binding of ``serron::erode`` / ``serron::erode_backward``."""

    @staticmethod
    def forward(ctx, input_: torch.Tensor, kernel: torch.Tensor, border: int, algo: int = Algorithm.AUTO):
        return _forward(ctx, _lib.ERODE, input_, kernel, border, algo)

    @staticmethod
    def backward(ctx, grad_output: torch.Tensor):
        return _backward(ctx, grad_output)


class _DilateFunction(torch.autograd.Function):
    """Autograd binding of ``serron::dilate`` / ``serron::dilate_backward``."""

    @staticmethod
    def forward(ctx, input_: torch.Tensor, kernel: torch.Tensor, border: int, algo: int = Algorithm.AUTO):
        return _forward(ctx, _lib.DILATE, input_, kernel, border, algo)

    @staticmethod
    def backward(ctx, grad_output: torch.Tensor):
        return _backward(ctx, grad_output)


class _DerivedFunction(torch.autograd.Function):
    """A derived operation in one launch (``serron_derived_forward``), with the backward of the reference's
    composition (packages/serron/torch-ext/serron/functional.py:40-92) from the two stages' records:

    * gradient ``D(x) - E(x)``: grad_x = D'(go) - E'(go), grad_w = Dw(go) - Ew(go);
    * opening ``D(E(x))``: h = D'(go) over the intermediate, grad_x = E'(h), grad_w = Dw(go) + Ew(h);
    * closing ``E(D(x))``: the same with the operations swapped;
    * top_hat ``x - opening(x)``: grad_x = go - E'(D'(go)), grad_w = -(Dw(go) + Ew(h));
    * black_hat ``closing(x) - x``: grad_x = D'(E'(go)) - go, grad_w = Ew(go) + Dw(h).

    A gather of -g is the negated gather of g bit for bit (each sum is negated exactly), so these are the
    reference's autograd results: its sums of two gradient contributions are the same two values, and a
    sum of two values does not depend on their order.
    """

    @staticmethod
    def forward(ctx, input_: torch.Tensor, kernel: torch.Tensor, border: int, mode: int):
        y, win_a, win_b, fmt = _ops.derived_forward(mode, input_, kernel, border)
        ctx.save_for_backward(kernel)
        ctx.records = (win_a, win_b, fmt)
        ctx.border = border
        ctx.mode = mode
        return y

    @staticmethod
    def backward(ctx, grad_output: torch.Tensor):
        needs_input, needs_kernel = ctx.needs_input_grad[:2]
        if not (needs_input or needs_kernel):
            return None, None, None, None
        (kernel,) = ctx.saved_tensors
        win_a, win_b, fmt = ctx.records
        go = grad_output.to(kernel.dtype).contiguous()
        mode, border = ctx.mode, ctx.border

        def gather(op, g, records):
            return _ops.backward_from_winners(op, g, records, fmt, kernel, border, needs_kernel)

        if mode == _ops.DERIVED_GRADIENT:
            g_d, k_d = gather(_lib.DILATE, go, win_a)
            g_e, k_e = gather(_lib.ERODE, go, win_b)
            grad_input, grad_kernel = g_d - g_e, k_d - k_e
        else:
            first = _lib.ERODE if mode in (_ops.DERIVED_OPENING, _ops.DERIVED_TOP_HAT) else _lib.DILATE
            second = _lib.DILATE if first == _lib.ERODE else _lib.ERODE
            h, k_2 = gather(second, go, win_b)
            g_1, k_1 = gather(first, h, win_a)
            if mode == _ops.DERIVED_TOP_HAT:
                grad_input, grad_kernel = go - g_1, -(k_2 + k_1)
            elif mode == _ops.DERIVED_BLACK_HAT:
                grad_input, grad_kernel = g_1 - go, k_2 + k_1
            else:
                grad_input, grad_kernel = g_1, k_2 + k_1
        return (grad_input if needs_input else None), (grad_kernel if needs_kernel else None), None, None


# ------------------------------------------------------------------------------------------------
# layer operators: statistics (layer norm) or nothing but the seed (dropout) are kept between the passes
# ------------------------------------------------------------------------------------------------
def _param_dtype(*params: torch.Tensor | None) -> torch.dtype | None:
    return next((p.dtype for p in params if p is not None), None)


class _LayerNormFunction(torch.autograd.Function):
    """``serron_layer_norm`` and its backward, for arguments that are already checked."""

    @staticmethod
    def forward(ctx, input_: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, dim: int,
                eps: float):
        y, x, mean, rstd = _layer_ops.layer_norm(input_, weight, bias, dim, eps, True)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.dim = dim
        ctx.param_dtype = _param_dtype(weight, bias) or x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output: torch.Tensor):
        x, mean, rstd, weight = ctx.saved_tensors
        return (*_layer_ops.layer_norm_backward(grad_output, x, mean, rstd, weight, ctx.param_dtype, ctx.dim,
                                                ctx.needs_input_grad[:3]), None, None)


class _DropoutFunction(torch.autograd.Function):
    """``serron_dropout``; the backward draws the same mask again."""

    @staticmethod
    def forward(ctx, input_: torch.Tensor, residual: torch.Tensor | None, span: int, p: float,
                seed: int | torch.Tensor, sequence: int):
        ctx.save_for_backward(seed if isinstance(seed, torch.Tensor) else None)
        ctx.rule = (span, p, seed if isinstance(seed, int) else None, sequence)
        return _layer_ops.dropout(input_, residual, span, p, seed, sequence)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output: torch.Tensor):
        span, p, seed, sequence = ctx.rule
        (seed_tensor,) = ctx.saved_tensors
        grad_input = None
        if ctx.needs_input_grad[0]:
            grad_input = _layer_ops.dropout(grad_output, None, span, p, seed if seed_tensor is None else seed_tensor,
                                            sequence)
        return grad_input, (grad_output if ctx.needs_input_grad[1] else None), None, None, None, None


class _DropoutAddLayerNormFunction(torch.autograd.Function):
    """``serron_dropout_add_layer_norm`` and its backward, for arguments that are already checked."""

    @staticmethod
    def forward(ctx, input_: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None,
                bias: torch.Tensor | None, p: float, seed: int | torch.Tensor, sequence: int, dim: int, eps: float):
        y, h, mean, rstd = _layer_ops.dropout_add_layer_norm(input_, residual, weight, bias, p, seed, sequence, dim,
                                                             eps, True)
        ctx.save_for_backward(h, mean, rstd, weight, seed if isinstance(seed, torch.Tensor) else None)
        ctx.set_materialize_grads(False)
        ctx.rule = (p, seed if isinstance(seed, int) else None, sequence)
        ctx.dim = dim
        ctx.param_dtype = _param_dtype(weight, bias) or h.dtype
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output: torch.Tensor | None, grad_sum: torch.Tensor | None):
        h, mean, rstd, weight, seed_tensor = ctx.saved_tensors
        p, seed, sequence = ctx.rule
        if grad_output is None:
            if grad_sum is None:
                return (None,) * 9
            grad_output = torch.zeros_like(h)
        grads = _layer_ops.dropout_add_layer_norm_backward(
            grad_output, grad_sum, h, mean, rstd, weight, ctx.param_dtype, p, seed if seed_tensor is None else seed_tensor,
            sequence, ctx.dim, ctx.needs_input_grad[:4])
        return (*grads, None, None, None, None, None)
