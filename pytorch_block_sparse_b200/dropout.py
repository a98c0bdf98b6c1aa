"""Dropout with the residual add behind it, from a counter-based generator: the mask is a function of a seed, a counter and
the element's index, so it is never stored -- backward draws it again.

The reference leaves both to the model (a ``torch.nn.Dropout`` and an addition after the layer); here they stand behind the
output projection of a block-sparse layer (``BlockSparseLinear(dropout=p)``) and by themselves.
"""
import torch

from . import native


def new_rng_state(device, seed=None):
    """int64 ``[2]`` (seed, counter) on ``device``; the seed is drawn from torch's default generator unless given."""
    if seed is None:
        seed = int(torch.randint(1 << 62, (1,)).item())
    return torch.tensor([seed, 0], dtype=torch.int64, device=device)


def rate_units(p):
    """The rate in units of 2^-16, the resolution of the mask."""
    cut = round(p * 65536) if 0.0 <= p < 1.0 else 65536
    if cut >= 65536:
        raise ValueError("dropout rate %r: expected 0 <= p < 1 (rounded to a multiple of 2^-16)" % (p,))
    return cut


class DropoutResidualFunction(torch.autograd.Function):
    """``apply(x, residual, cut, rng)``; both gradients come from the output's: the residual's is the same tensor."""

    @staticmethod
    def forward(ctx, x, residual, cut, rng):
        ctx.cut = cut
        ctx.save_for_backward(rng)
        return native.dropout(x.contiguous(), residual.contiguous() if residual is not None else None, cut, rng)

    @staticmethod
    def backward(ctx, grad):
        (rng,) = ctx.saved_tensors
        want_x, want_residual, _, _ = ctx.needs_input_grad
        dx = None
        if want_x and torch.is_grad_enabled():  # a gradient of this gradient is wanted: the operator is linear in x
            dx = DropoutResidualFunction.apply(grad, None, ctx.cut, rng)
        elif want_x:
            dx = native.dropout(grad.contiguous(), None, ctx.cut, rng)
        return dx, grad if want_residual else None, None, None


def dropout_residual(x, p, rng=None, residual=None):
    """``dropout(x, p) + residual`` in one kernel, mask never stored.

    ``x``: fp32 or bf16 CUDA tensor; ``residual`` (optional): same shape and type.  ``rng``: int64 ``[2]`` CUDA tensor (seed,
    counter) -- equal values give equal masks; it is read when the kernel runs, so a captured call draws anew in every
    replay if the graph moves the counter on (:func:`next_rng`), and it must not change between forward and backward.
    Without one both numbers are drawn from torch's generator of ``x``'s device: seeds, activation checkpointing and captured
    graphs then behave as with torch's own dropout.
    Element ``i`` (of the contiguous tensor) is kept when its 16-bit number of Philox4x32-10 is at least ``round(p * 65536)``;
    kept values are scaled by the inverse of the exact share kept.  A dropped value leaves exactly the residual, also where
    ``x`` is infinite or NaN."""
    cut = rate_units(p)
    if not x.is_cuda:
        raise native.NativeError("x must be a CUDA tensor (got %s); there is no CPU path" % x.device)
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("dropout_residual takes float32 or bfloat16 tensors, got %s" % x.dtype)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("residual must match x: %s %s %s, got %s %s %s" % (
            tuple(x.shape), x.dtype, x.device, tuple(residual.shape), residual.dtype, residual.device))
    if rng is None:
        rng = torch.randint(1 << 62, (2,), device=x.device)
    elif rng.dtype != torch.int64 or tuple(rng.shape) != (2,) or rng.device != x.device or not rng.is_contiguous():
        raise ValueError("rng must be a contiguous int64 tensor of 2 elements (seed, counter) on %s" % x.device)
    return DropoutResidualFunction.apply(x, residual, cut, rng)


def next_rng(state):
    """The (seed, counter) of one draw from ``state`` as a tensor of its own; the state's counter moves on, on the device."""
    if state.dtype != torch.int64 or tuple(state.shape) != (2,) or not state.is_contiguous():
        raise ValueError("state must be a contiguous int64 tensor of 2 elements (seed, counter)")
    return native.rng_next(state)
