"""Low-rank adapters of many requests at once beside a shared projection (serving).

A batch holds the tokens of several requests back to back; each request may bring an adapter of its own, a pair of thin
matrices ``D [rank, in]`` and ``U [out, rank]`` with a scale.  One call adds ``s * (x @ D.T) @ U.T`` of each token's adapter to
the output of the projection that all requests share (``BlockSparseLinear(x, adapters=...)``), whatever mix of prompts and
single tokens the batch is.  The reference has no counterpart.
"""
import torch
import torch.nn as nn

from . import native


class AdapterRequests:
    """Which tokens belong to which request, and which adapter each request uses.

    ``offsets``: int32 ``[n + 1]``, request ``i`` owns tokens ``offsets[i] .. offsets[i + 1] - 1`` (non-decreasing); ``adapters``:
    int32 ``[n]``, ``-1`` for none.  Both CUDA tensors, read when the kernels run: a captured graph may be replayed with new
    contents.  Tokens outside every request keep the projection's output.  :meth:`from_lengths` builds and checks them
    from host lists."""

    def __init__(self, offsets, adapters):
        for name, t in (("offsets", offsets), ("adapters", adapters)):
            if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise ValueError("%s must be a contiguous one-dimensional int32 tensor" % name)
        if offsets.shape[0] != adapters.shape[0] + 1:
            raise ValueError("offsets must have one element more than adapters, got %d and %d"
                             % (offsets.shape[0], adapters.shape[0]))
        if offsets.device != adapters.device:
            raise ValueError("offsets and adapters must be on one device")
        self.offsets, self.adapters = offsets, adapters

    @classmethod
    def from_lengths(cls, lengths, adapters, device="cuda"):
        if len(lengths) != len(adapters):
            raise ValueError("%d lengths for %d adapters" % (len(lengths), len(adapters)))
        offsets = [0]
        for n in lengths:
            if n < 0:
                raise ValueError("negative length %d" % n)
            offsets.append(offsets[-1] + n)
        return cls(torch.tensor(offsets, dtype=torch.int32, device=device),
                   torch.tensor([-1 if a is None else a for a in adapters], dtype=torch.int32, device=device))


class LowRankAdapters(nn.Module):
    """``count`` adapters of rank up to ``rank`` for one projection ``in_features -> out_features`` (multiples of 32).

    They are kept as the kernels read them: ``down [count, R, in]``, ``up [count, out, R]`` with ``R`` the rank padded by zeros to
    16, 32 or a multiple of 64 (up to 256), ``scaling [count]`` fp32.  Adapters that were not loaded are zero.  They serve:
    buffers without gradients."""

    def __init__(self, in_features, out_features, count, rank, dtype=torch.float32, device="cuda"):
        super().__init__()
        if in_features <= 0 or in_features % 32 != 0 or out_features <= 0 or out_features % 32 != 0:
            raise Exception("LowRankAdapters invalid sizes %d, %d: should be multiples of 32" % (in_features, out_features))
        if count < 1 or not 1 <= rank <= 256:
            raise Exception("LowRankAdapters invalid count=%d or rank=%d (1 to 256)" % (count, rank))
        if dtype not in (torch.float32, torch.bfloat16):
            raise Exception("LowRankAdapters invalid dtype=%s, expected float32 or bfloat16" % dtype)
        padded = 16 if rank <= 16 else 32 if rank <= 32 else (rank + 63) // 64 * 64
        self.in_features, self.out_features, self.count, self.rank = in_features, out_features, count, rank
        self.register_buffer("down", torch.zeros((count, padded, in_features), dtype=dtype, device=device))
        self.register_buffer("up", torch.zeros((count, out_features, padded), dtype=dtype, device=device))
        self.register_buffer("scaling", torch.zeros(count, dtype=torch.float32, device=device))

    @torch.no_grad()
    def load(self, index, down, up, scaling=1.0):
        """Adapter ``index``: ``down [r, in]``, ``up [out, r]`` with ``r <= rank``; what it held before is gone."""
        if not 0 <= index < self.count:
            raise IndexError("adapter %d of %d" % (index, self.count))
        r = down.shape[0]
        if r > self.rank or tuple(down.shape) != (r, self.in_features) or tuple(up.shape) != (self.out_features, r):
            raise ValueError("adapter shapes %s, %s do not fit [r, %d], [%d, r] with r <= %d" % (
                tuple(down.shape), tuple(up.shape), self.in_features, self.out_features, self.rank))
        self.down[index].zero_()
        self.up[index].zero_()
        self.down[index, :r].copy_(down)
        self.up[index, :, :r].copy_(up)
        self.scaling[index] = scaling

    @torch.no_grad()
    def load_all(self, down, up, scaling):
        """All adapters at once: ``down [count, r, in]``, ``up [count, out, r]``, ``scaling [count]``."""
        r = down.shape[1]
        if (r > self.rank or tuple(down.shape) != (self.count, r, self.in_features)
                or tuple(up.shape) != (self.count, self.out_features, r) or tuple(scaling.shape) != (self.count,)):
            raise ValueError("adapter shapes %s, %s, %s do not fit" % (tuple(down.shape), tuple(up.shape), tuple(scaling.shape)))
        self.down.zero_()
        self.up.zero_()
        self.down[:, :r].copy_(down)
        self.up[:, :, :r].copy_(up)
        self.scaling.copy_(scaling)

    def forward(self, x, requests, base=None, inplace=False, dtype=None):
        """``base + s_a * (x @ D_a.T) @ U_a.T`` for each token's adapter ``a`` (``base`` alone where it has none; ``base=None``:
        zeros).  ``x [..., in]`` in the adapters' type, its leading dimensions flattened to the batch's tokens;
        ``base [..., out]`` in the same type or fp32.  ``inplace`` adds into ``base`` (contiguous) and returns it.  ``dtype``: the
        output's type where there is no base, ``x``'s (the default) or fp32."""
        if (x.requires_grad or (base is not None and base.requires_grad)) and torch.is_grad_enabled():
            raise native.NativeError("LowRankAdapters serve and have no gradients: call them under torch.no_grad()")
        buffers = self._buffers
        down, up, scaling = buffers["down"], buffers["up"], buffers["scaling"]
        lead, kind = x.shape[:-1], x.dtype
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise Exception("Invalid input %s for adapters of %d features" % (tuple(x.shape), self.in_features))
        if kind is not down.dtype or kind is not up.dtype or (kind is not torch.float32 and kind is not torch.bfloat16):
            raise ValueError("x is %s, the adapters are %s: expected one type, float32 or bfloat16" % (kind, down.dtype))
        if scaling.dtype is not torch.float32:  # (the module was cast as a whole)
            scaling = scaling.float()
        device = down.device
        if x.device != device or requests.offsets.device != device or (base is not None and base.device != device):
            raise native.NativeError("x, the requests, the base and the adapters must be on one device, got %s, %s, %s, %s" % (
                x.device, requests.offsets.device, base.device if base is not None else None, device))
        if base is not None:
            if base.shape != lead + (self.out_features,):
                raise ValueError("base must be %s, got %s" % (tuple(lead) + (self.out_features,), tuple(base.shape)))
            kind = base.dtype
        elif dtype is not None:
            kind = dtype
        if kind is not x.dtype and kind is not torch.float32:
            raise ValueError("the output's type is %s: expected %s or float32" % (kind, x.dtype))
        if inplace:
            if base is None or not base.is_contiguous() or base.data_ptr() % 16 != 0:
                raise ValueError("inplace wants a contiguous, 16-byte aligned base")
            out = base
        elif base is not None:
            base = native._aligned(base.contiguous())
            out = torch.empty_like(base)
        else:
            out = x.new_empty(lead + (self.out_features,), dtype=kind)
        if x.dim() != 2:
            x = x.reshape(-1, self.in_features)
        native.adapters(x.contiguous(), requests.offsets, requests.adapters, native._aligned(down), native._aligned(up), scaling,
                        base, out)
        return out

    def extra_repr(self):
        return "in_features={}, out_features={}, count={}, rank={}".format(
            self.in_features, self.out_features, self.count, self.rank)
