"""The gated feed-forward block on block-sparse weights: ``h = act(x @ Wg.T + bg) * (x @ Wu.T + bu)``.

Both projections live in ONE :class:`BlockSparseMatrix` of ``2 * hidden`` rows whose block-rows alternate -- block-row ``2j`` is
the gate's block-row ``j``, ``2j + 1`` the up projection's -- so that one product computes both, the two halves of a hidden unit
meet in the same tile, and each gradient is one product too.  The pattern, the sparsity optimizer and checkpoints see
an ordinary block-sparse matrix.  The reference has no gated layer: its user builds two ``BlockSparseLinear`` and multiplies
(``block_sparse_linear.py:157-233`` is the layer this one stands beside).
"""
import math

import numpy
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import native
from .block_sparse import BlockSparseMatrix

# Up to this many tokens inference computes from the stored blocks directly (``bsmm_gated_small``).  us, few-token kernel / weight
# images and tensor-core kernel, on one B200: bf16, 4096 -> 8192 at density 0.25, 16 tokens 21 / 44, 32 tokens 26 / 44, 48 tokens
# 42 / 44, 64 tokens 44 / 44; 4096 -> 16384 at 0.1, 32 tokens 29 / 32, 48 tokens 46 / 32; 1024 -> 2048 at 0.5, 32 tokens 8 / 15.
# fp32, 4096 -> 8192: 8 tokens 23 / 88, 16 tokens 39 / 86, 32 tokens 68 / 75, 48 tokens 99 / 75; 1024 -> 4096 at 0.5, 16 tokens 14 / 31,
# 32 tokens 24 / 23.
SMALL_TOKENS = 32


def interleave_rows(gate, up):
    """``[hidden, ...]`` of the gate and of the up projection -> ``[2 * hidden, ...]``, 32 rows of each in turn."""
    tail = gate.shape[1:]
    return torch.stack([gate.reshape(-1, 32, *tail), up.reshape(-1, 32, *tail)], 1).reshape(-1, *tail)


def split_rows(both):
    """Inverse of :func:`interleave_rows`: ``(gate, up)``."""
    tail = both.shape[1:]
    parts = both.reshape(-1, 2, 32, *tail)
    return parts[:, 0].reshape(-1, *tail), parts[:, 1].reshape(-1, *tail)


class BlockSparseGatedFunction(torch.autograd.Function):
    """``apply(input, weight_data, weight, bias, activation, precision)`` with ``input [m, k]``."""

    @staticmethod
    def forward(ctx, input, weight_data, weight, bias, activation, precision):
        assert weight_data.is_contiguous()
        ctx.weight, ctx.activation = weight, activation
        ctx.precision = prec = native.resolve_precision(precision)
        # The weights are packed in every pass, never cached (writes through ``.data`` do not bump version counters).
        if _fused(input, prec):
            # g and u are kept in bf16, the type of every other tensor that this mode keeps for backward
            h, pre = native.gated_forward(input, _gated_plan(weight), weight_data, bias, activation, True)
            ctx.packed = native.pack_weights(weight_data, prec).images if ctx.needs_input_grad[0] else None
        else:
            x = input if input.dtype is torch.float32 else input.float()
            h, pre, ctx.packed = _gated_pass(weight).forward(x, weight_data, bias, activation, prec, _out_dtype(input, prec))
        ctx.save_for_backward(input, pre, weight_data)
        return h

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():  # create_graph: the gradients are handed out, a second differentiation raises
            return _gradients_once(ctx, grad)
        return _gradients(ctx, grad)


def _gradients(ctx, grad):
    input, pre, data = ctx.saved_tensors
    weight, (want_x, want_w, _, want_bias, _, _) = ctx.weight, ctx.needs_input_grad
    grad = grad.contiguous()
    if grad.dtype is torch.bfloat16 and (grad.shape[0] < 32 or data.shape[0] == 0):
        # the products of bf16 tensors start at 32 tokens: fewer go through the fp32 ones
        grad, pre = grad.float(), pre.float()
    x = input if input.dtype is grad.dtype else input.to(grad.dtype)
    dx, dw, dbias, sumsq = _gated_pass(weight).backward(
        x, pre, grad, data, ctx.packed, ctx.activation, ctx.precision, want_x, want_w, want_bias)
    if want_w:
        weight.last_grad_block_sumsq = sumsq
    return dx if dx is None or dx.dtype is input.dtype else dx.to(input.dtype), dw, None, dbias, None, None


_gradients_once = once_differentiable(_gradients)


def _out_dtype(x, prec):
    """bf16 tensors stay bf16 in the 'bf16' precision; every other combination computes fp32 (as BlockSparseLinear)."""
    return torch.bfloat16 if x.dtype is torch.bfloat16 and prec == native.PREC_BF16 else torch.float32


def _fused(x, prec):
    """Whether the one-kernel forward runs: bf16 tensors in the 'bf16' precision."""
    return prec == native.PREC_BF16 and x.dtype is torch.bfloat16 and x.shape[0] > 0 and x.shape[1] <= native.GATED_MAX_K


def _cached_plan(weight, kind, buffers, build):
    """``build(*buffers)`` kept beside the matrix's other plans while its index buffers are these.  What is built while a
    stream is captured belongs to the graph and is not kept."""
    key = (kind, *[v for t in buffers for v in (t.data_ptr(), t._version)])
    plan = weight._plan_cache.get(key)
    if plan is None:
        plan = build(*buffers)
        if not native.capturing():
            weight._plan_cache = {k: v for k, v in weight._plan_cache.items() if k[0] != kind}
            weight._plan_cache[key] = plan
    return plan


def _gated_plan(weight):
    """Plan of the one-kernel forward."""
    return _cached_plan(weight, "gated", (weight.row_start_ends_a, weight.cols_a),
                        lambda ptr, idx: native.GatedPlan(ptr, idx, weight.shape[0] // 2, weight.shape[1]))


def _gated_pass(weight):
    """Plans of the passes through the matrix's products."""
    return _cached_plan(weight, "gated pass", (weight.row_start_ends_a, weight.cols_a, weight.col_start_ends_b, weight.rows_b,
                                               weight.blocks), native.GatedPass)


class BlockSparseGatedLinear(nn.Module):
    """``act(gate(x)) * up(x)`` with block-sparse projections ``in_features -> hidden_features`` (multiples of 32).

    ``density``: share of the 32x32 blocks stored, ``int(density * in * hidden / 1024)`` positions drawn at random, the same for
    both projections (a hidden block reads the same inputs through both).  ``weight`` hands in the matrix instead,
    ``[2 * hidden, in]`` with alternating block-rows and any pattern.  ``activation``: ``"silu"`` or ``"gelu"`` (erf form).
    ``bias``: fp32 ``[2 * hidden]``, laid out like the weight's rows.  ``precision``: as ``set_default_precision``; ``None`` follows the
    default at each call.  Input: fp32 or bf16 ``[..., in]``; the output is bf16 for bf16 input in the ``"bf16"`` precision, else
    fp32.  Without gradients and up to ``SMALL_TOKENS`` tokens the products are exact fp32 in every precision.  In the fp32-class
    precisions (``"tf32x3"``, ``"bf16x3"``) a pass needs a workspace of 6 bytes per input value, backward 12 more per hidden unit
    and token."""

    def __init__(self, in_features, hidden_features, bias=True, density=0.5, activation="silu", weight=None, precision=None):
        super().__init__()
        if in_features <= 0 or in_features % 32 != 0:
            raise Exception(f"BlockSparseGatedLinear invalid in_features={in_features}, should be multiple of 32")
        if hidden_features <= 0 or hidden_features % 32 != 0:
            raise Exception(f"BlockSparseGatedLinear invalid hidden_features={hidden_features}, should be multiple of 32")
        if activation not in ("silu", "gelu"):
            raise Exception(f"BlockSparseGatedLinear invalid activation={activation}, expected 'silu' or 'gelu'")
        if precision is not None and precision not in native.PRECISIONS:
            raise ValueError("unknown precision %r, expected one of %s" % (precision, sorted(native.PRECISIONS)))
        self.in_features, self.hidden_features = in_features, hidden_features
        self.activation, self.precision = activation, precision
        if weight is None:
            if density < 0 or density > 1:
                raise Exception(f"BlockSparseGatedLinear invalid density={density}")
            rows, cols = hidden_features // 32, in_features // 32
            cells = numpy.random.choice(rows * cols, size=int(density * rows * cols), replace=False)
            weight = self._matrix(cells, rows, cols, "cuda")
            with torch.no_grad():
                weight.data.normal_()
        elif not isinstance(weight, BlockSparseMatrix) or tuple(weight.block_shape) != (32, 32):
            raise Exception("BlockSparseGatedLinear weight should be a BlockSparseMatrix with 32x32 blocks")
        elif tuple(weight.shape) != (2 * hidden_features, in_features):
            raise Exception("BlockSparseGatedLinear weight should be of shape (%d, %d), not %s" % (
                2 * hidden_features, in_features, tuple(weight.shape)))
        self.weight = weight
        if bias:
            self.bias = nn.Parameter(torch.zeros(2 * hidden_features, device=weight.data.device))
        else:
            self.register_parameter("bias", None)

    @staticmethod
    def _matrix(cells, rows, cols, device):
        """Matrix of zeros with both projections' blocks at the positions ``cells`` of the ``rows`` x ``cols`` grid."""
        mask = torch.zeros(rows * cols, dtype=torch.bool, device=device)
        mask[torch.as_tensor(cells, dtype=torch.int64, device=device)] = True
        mask = mask.view(rows, cols).repeat_interleave(2, 0)
        data = torch.zeros((2 * len(cells) * 32, 32), dtype=torch.float32, device=device)
        return BlockSparseMatrix((2 * rows * 32, cols * 32), mask, data)

    @classmethod
    def from_linears(cls, gate, up, density=1.0, activation="silu", precision=None):
        """From two dense ``nn.Linear`` of one shape: ``density`` of their blocks, drawn at random, scaled by
        ``1 / sqrt(density)`` as ``BlockSparseLinear`` does."""
        if gate.weight.shape != up.weight.shape or (gate.bias is None) != (up.bias is None):
            raise Exception("gate and up should be two linear layers of one shape, both with a bias or both without")
        hidden, inner = gate.weight.shape
        if hidden % 32 != 0 or inner % 32 != 0:
            raise Exception(f"BlockSparseGatedLinear invalid layer {hidden}x{inner}, should be multiples of 32")
        if density <= 0 or density > 1:
            raise Exception(f"BlockSparseGatedLinear invalid density={density}")
        rows, cols = hidden // 32, inner // 32
        cells = numpy.random.choice(rows * cols, size=int(density * rows * cols), replace=False)
        with torch.no_grad():
            weight = cls._matrix(cells, rows, cols, "cuda")
            BlockSparseMatrix.from_dense(interleave_rows(gate.weight.detach().float().cuda(), up.weight.detach().float().cuda()),
                                         out=weight)
            weight.multiply_(1.0 / math.sqrt(density))
            layer = cls(inner, hidden, bias=gate.bias is not None, activation=activation, weight=weight, precision=precision)
            if gate.bias is not None:
                layer.bias.copy_(interleave_rows(gate.bias.detach().float().cuda(), up.bias.detach().float().cuda()))
        return layer

    def to_dense(self):
        """``(gate, up)``: the two weights as dense ``[hidden, in]`` matrices."""
        return split_rows(self.weight.to_dense())

    def forward(self, x):
        weight, bias = self.weight, self.bias
        data = weight.get_differentiable_data()
        shape = x.shape
        if len(shape) < 2:
            raise Exception(f"Invalid dimensions for x {tuple(shape)} : x should have at least 2 dimensions.")
        if shape[-1] != self.in_features:
            raise Exception("Invalid matrices sizes (%d, %d) x (%d, %d)" % (
                x.numel() // max(1, shape[-1]), shape[-1], self.in_features, 2 * self.hidden_features))
        if x.dtype is not torch.float32 and x.dtype is not torch.bfloat16:
            raise ValueError("BlockSparseGatedLinear takes float32 or bfloat16 tensors, got %s" % x.dtype)
        if not data.is_cuda:
            weight._require_cuda()
        if data.dtype is not torch.float32:
            raise Exception("BlockSparseGatedLinear weights should be float32, not of type %s" % data.dtype)
        if bias is not None and bias.dtype is not torch.float32:
            bias = bias.float()
        if x.device != data.device:
            raise native.NativeError("x is on %s, the layer on %s" % (x.device, data.device))
        flat = (x if len(shape) == 2 else x.reshape(-1, shape[-1])).contiguous()
        if torch.is_grad_enabled() and (x.requires_grad or data.requires_grad or (bias is not None and bias.requires_grad)):
            h = BlockSparseGatedFunction.apply(flat, data, weight, bias, self.activation, self.precision)
        else:
            h = self._infer(flat, weight, bias, data)
        return h if len(shape) == 2 else h.reshape(*shape[:-1], self.hidden_features)

    def _infer(self, flat, weight, bias, data):
        prec = native.resolve_precision(self.precision)
        if flat.shape[0] <= SMALL_TOKENS:
            return native.gated_small(flat, weight.row_start_ends_a, weight.cols_a, data, self.hidden_features, bias,
                                      self.activation, _out_dtype(flat, prec))
        if _fused(flat, prec):
            return native.gated_forward(flat, _gated_plan(weight), data, bias, self.activation, False)[0]
        x = flat if flat.dtype is torch.float32 else flat.float()
        return _gated_pass(weight).forward(x, data, bias, self.activation, prec, _out_dtype(flat, prec), keep=False)[0]

    def extra_repr(self):
        return "in_features={}, hidden_features={}, bias={}, activation={}, block_count={}".format(
            self.in_features, self.hidden_features, self.bias is not None, self.activation, self.weight.blocks.shape[0] // 2)
