"""The gated feed-forward block: the activation kernels elementwise, the layer in every precision against 64 bits (values and
gradients), few tokens, odd patterns, graphs and streams, and a feed-forward block built of it."""
import copy
import io
import math

import numpy as np
import pytest
import torch

from pytorch_block_sparse_b200 import (AdapterRequests, BlockSparseGatedLinear, BlockSparseLinear, BlockSparseMatrix,
                                       LowRankAdapters, SparseOptimizer, native)
from pytorch_block_sparse_b200 import gated_linear
from pytorch_block_sparse_b200.gated_linear import SMALL_TOKENS, interleave_rows, split_rows

from .gpu_util import TOL, assert_device_healthy, randn

pytestmark = pytest.mark.gpu


def act64(g, kind):
    """Value and slope of the gate's activation in 64 bits."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def columns(pre):
    g, u = pre.reshape(pre.shape[0], -1, 2, 32).unbind(2)
    return g.reshape(pre.shape[0], -1), u.reshape(pre.shape[0], -1)


def make(inner, hidden, density=0.5, bias=True, act="silu", precision=None, seed=0, mask=None, bf16_values=False):
    """A layer whose pre-activations have about unit size."""
    np.random.seed(seed)
    torch.manual_seed(seed)
    weight = None
    if mask is not None:
        weight = BlockSparseMatrix((2 * hidden, inner), mask.cuda(), torch.zeros((int(mask.sum()) * 32, 32), device="cuda"))
    layer = BlockSparseGatedLinear(inner, hidden, bias=bias, density=density, activation=act, weight=weight, precision=precision)
    with torch.no_grad():
        per_row = max(1.0, layer.weight.data.shape[0] / 32 / (2 * hidden / 32) * 32)
        d = randn(tuple(layer.weight.data.shape), seed + 1) / per_row ** 0.5
        layer.weight.data.copy_(d.bfloat16().float() if bf16_values else d)
        if bias:
            layer.bias.copy_(randn((2 * hidden,), seed + 2) * 0.3)
    return layer


def reference(layer, x, dh=None):
    """h, and with dh the gradients (dx, dW dense, db), in 64 bits on the host."""
    w = layer.weight.to_dense().detach().cpu().double()
    b = layer.bias.detach().cpu().double() if layer.bias is not None else 0.0
    x = x.cpu().double().reshape(-1, x.shape[-1])
    g, u = columns(x @ w.t() + b)
    a, slope = act64(g, layer.activation)
    h = a * u
    if dh is None:
        return h
    dh = dh.cpu().double().reshape(h.shape)
    dpre = interleave_rows((dh * u * slope).t(), (dh * a).t()).t()
    return h, dpre @ w, dpre.t() @ x, dpre.sum(0)


def rel(got, want):
    return float(torch.linalg.norm(got.detach().cpu().double() - want) / (torch.linalg.norm(want) + 1e-300))


def in_data_layout(layer, dense):
    """The stored blocks of a dense [2 * hidden, in] matrix in ``data`` layout."""
    blocks = layer.weight.blocks.view(-1, 2).cpu().long()
    grid = dense.reshape(dense.shape[0] // 32, 32, dense.shape[1] // 32, 32)
    return grid[blocks[:, 1], :, blocks[:, 0], :].transpose(1, 2).reshape(-1, 32)


# A product of precision p is within TOL[p] of its norm (the bar of every product in this package).  With pre-activations of
# unit size |act'| <= 1.13 and rms(act(g)) >= 0.6, so h = act(g) u is within (1.13 / 0.6 + 1) < 3 times that, dpre likewise
# (|act''| <= 1), and the two products of the backward pass add one each: 4.  bf16 outputs add half a step, 2^-8, and
# bf16 dpre another.
def bound(precision, products, out=torch.float32, roundings=0):
    return products * TOL[precision] + (2.0 ** -8 if out == torch.bfloat16 else 0.0) + roundings * 2.0 ** -8


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,hidden", [(1, 32), (3, 96), (255, 64), (257, 32), (700, 544)])
@pytest.mark.parametrize("types", ["fp32", "bf16", "all bf16"])
def test_activation_kernels_elementwise(act, m, hidden, types):
    pre = randn((m, 2 * hidden), 1) * 3
    pre[0, :8] = torch.tensor([0.0, -0.0, 30.0, -30.0, 1e-30, 88.0, -88.0, 100.0])
    dh = randn((m, hidden), 2)
    if types != "fp32":
        dh = dh.bfloat16()
    if types == "all bf16":
        pre = pre.bfloat16()
    out_dtype = dh.dtype
    g, u = columns(pre.double())
    a, slope = act64(g, act)
    h = native.gated_act(pre.cuda(), act, out_dtype)
    half = 2.0 ** -8 * (1 + 2.0 ** -7) if out_dtype == torch.bfloat16 else 0.0
    # exp and erf to a few units in the last place (2^-23), of a value of at most |g u|; denormal results vanish
    assert ((h.cpu().double() - a * u).abs() <= 1e-6 * (g * u).abs() + half * (a * u).abs() + 1e-37).all()
    dpre, db = native.gated_act_backward(pre.cuda(), dh.cuda(), act, True)
    assert dpre.dtype == out_dtype and db.dtype == torch.float32
    want_g, want_u = dh.double() * u * slope, dh.double() * a
    got_g, got_u = columns(dpre.cpu().double())
    assert ((got_g - want_g).abs() <= 3e-6 * (1 + g.abs()) * (dh.double() * u).abs() + half * want_g.abs() + 1e-37).all()
    assert ((got_u - want_u).abs() <= 1e-6 * (dh.double() * g).abs() + half * want_u.abs() + 1e-37).all()
    want_db = interleave_rows(want_g.sum(0), want_u.sum(0))
    size = interleave_rows(((1 + g.abs()) * dh.double().abs() * (u.abs() + 1)).sum(0), (dh.double() * g).abs().sum(0))
    assert ((db.cpu().double() - want_db).abs() <= (3e-6 + (m / 32 + 40) * 2.0 ** -24) * size + 1e-37).all()
    again = native.gated_act_backward(pre.cuda(), dh.cuda(), act, True)
    assert torch.equal(again[0], dpre) and torch.equal(again[1], db)
    assert native.gated_act_backward(pre.cuda(), dh.cuda(), act, False)[1] is None


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype,precision", [(torch.float32, None), (torch.bfloat16, "bf16"), (torch.bfloat16, "tf32x3"), (torch.float32, "bf16")])
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 16, 17, SMALL_TOKENS])
@pytest.mark.parametrize("sizes", [(32, 32), (96, 160), (1056, 544), (64, 2080)])
def test_few_tokens(act, dtype, precision, tokens, sizes):
    layer = make(*sizes, density=0.4 if sizes[0] > 32 else 1.0, act=act, precision=precision, seed=tokens)
    x = randn((tokens, sizes[0]), 5).to(dtype)
    with torch.no_grad():
        h = layer(x.cuda())
    out = torch.bfloat16 if dtype == torch.bfloat16 and precision == "bf16" else torch.float32
    assert h.dtype == out and h.shape == (tokens, sizes[1])
    # exact fp32 products in every precision: the bar of fp32
    assert rel(h, reference(layer, x)) <= bound("fp32", 3, out)
    with torch.no_grad():
        assert torch.equal(layer(x.cuda()), h)


@pytest.mark.parametrize("precision", ["fp32", "tf32x3", "bf16x3", "tf32", "bf16"])
@pytest.mark.parametrize("tokens,inner,hidden,density,bias,act", [
    (33, 32, 32, 1.0, True, "silu"), (100, 96, 160, 0.5, False, "gelu"), (129, 544, 1056, 0.3, True, "silu"),
    (300, 2080, 96, 0.2, True, "gelu"), (1000, 256, 512, 0.1, False, "silu"),
])
def test_inference_in_every_precision(precision, tokens, inner, hidden, density, bias, act):
    for dtype in (torch.float32, torch.bfloat16):
        layer = make(inner, hidden, density, bias, act, precision, seed=tokens)
        x = randn((tokens, inner), 6).to(dtype)
        with torch.no_grad():
            h = layer(x.cuda())
        out = torch.bfloat16 if dtype == torch.bfloat16 and precision == "bf16" else torch.float32
        assert h.dtype == out
        assert rel(h, reference(layer, x)) <= bound(precision, 3, out)
        assert_device_healthy()


@pytest.mark.parametrize("precision", ["fp32", "tf32x3", "bf16x3", "tf32", "bf16"])
@pytest.mark.parametrize("tokens,inner,hidden,density,bias,act", [
    (1, 64, 96, 0.5, True, "silu"), (31, 96, 160, 0.5, True, "gelu"), (129, 544, 1056, 0.3, True, "silu"),
    (500, 1056, 96, 0.2, False, "gelu"),
])
def test_training_in_every_precision(precision, tokens, inner, hidden, density, bias, act):
    for dtype in (torch.float32, torch.bfloat16):
        layer = make(inner, hidden, density, bias, act, precision, seed=tokens)
        x = randn((tokens, inner), 6).to(dtype)
        out = torch.bfloat16 if dtype == torch.bfloat16 and precision == "bf16" else torch.float32
        dh = randn((tokens, hidden), 7).to(out)
        xg = x.cuda().requires_grad_()
        h = layer(xg)
        assert h.dtype == out
        h.backward(dh.cuda())
        want_h, want_dx, want_dw, want_db = reference(layer, x, dh)
        rounded = 1 if out == torch.bfloat16 else 0
        assert rel(h, want_h) <= bound(precision, 3, out)
        assert xg.grad.dtype == dtype and rel(xg.grad, want_dx) <= bound(precision, 4, dtype, rounded)
        assert rel(layer.weight.data.grad, in_data_layout(layer, want_dw)) <= bound(precision, 4, roundings=rounded)
        if bias:
            assert rel(layer.bias.grad, want_db) <= bound(precision, 4, roundings=rounded)
        assert_device_healthy()


def test_the_gradient_agrees_with_differences():
    layer = make(96, 64, 0.7, precision="fp32", seed=3)
    x, w = randn((40, 96), 1).cuda(), randn((40, 64), 2).cuda()
    xg = x.clone().requires_grad_()
    leaves = [xg, layer.weight.data, layer.bias]
    grads = torch.autograd.grad(layer(xg), leaves, w)
    step = 2.0 ** -7
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        v = randn(tuple(leaf.shape), 10 + i).cuda()
        values = []
        with torch.no_grad():
            for s in (step, -step):
                leaf += s * v
                values.append((native_forward(layer, xg) * w.double()).sum().item())
                leaf -= s * v
        diff = (values[0] - values[1]) / (2 * step)
        want = (grad.double() * v).sum().item()
        # central differences: step^2 / 6 of a third derivative of the size of the loss, and fp32 noise over the step
        size = float(torch.linalg.norm(grad.double()) * torch.linalg.norm(v.double())) + float(torch.linalg.norm(w.double())) * 8
        assert abs(diff - want) <= (step ** 2 + 2.0 ** -20 / step) * size * 4


def native_forward(layer, x):
    return layer(x.detach()).double()


def test_patterns_that_differ_between_gate_and_up():
    """Rows without blocks on one or both sides, blocks that only one side has, and a matrix without any."""
    rows, cols = 7, 5
    g = torch.Generator().manual_seed(4)
    mask = torch.rand((2 * rows, cols), generator=g) < 0.4
    mask[4] = False        # the gate of hidden block 2 reads nothing: act(bias)
    mask[7] = False        # the up projection of hidden block 3
    mask[12:14] = False    # both of hidden block 6
    for precision in (None, "bf16"):
        dtype = torch.bfloat16 if precision else torch.float32
        layer = make(cols * 32, rows * 32, precision=precision, mask=mask, seed=5)
        for tokens in (3, 150):
            x, dh = randn((tokens, cols * 32), 1).to(dtype), randn((tokens, rows * 32), 2).to(dtype)
            xg = x.cuda().requires_grad_()
            h = layer(xg)
            got = torch.autograd.grad(h, [xg, layer.weight.data, layer.bias], dh.cuda())
            want = reference(layer, x, dh)
            p = precision or "tf32x3"
            assert rel(h, want[0]) <= bound(p, 3, dtype)
            assert rel(got[0], want[1]) <= bound(p, 4, dtype, 1 if precision else 0)
            assert rel(got[1], in_data_layout(layer, want[2])) <= bound(p, 4, roundings=1 if precision else 0)
            assert rel(got[2], want[3]) <= bound(p, 4, roundings=1 if precision else 0)
            with torch.no_grad():
                assert rel(layer(x.cuda()), want[0]) <= bound(p, 3, dtype)
    empty = make(64, 64, mask=torch.zeros((4, 2), dtype=torch.bool), seed=1)
    for tokens in (2, 70):
        x = randn((tokens, 64), 3)
        with torch.no_grad():
            assert rel(empty(x.cuda()), reference(empty, x)) <= bound("fp32", 3)
        xg = x.cuda().requires_grad_()
        empty(xg).sum().backward()
        assert (xg.grad == 0).all()
    assert_device_healthy()


def test_patterns_moved_by_the_sparsity_optimizer():
    layer = make(256, 192, 0.5, seed=6)
    x = randn((100, 256), 1)
    layer(x.cuda()).sum().backward()
    n = layer.weight.blocks.shape[0] // 2
    slots = torch.arange(0, n, 3, dtype=torch.int32, device="cuda")
    layer.weight.move_blocks_(slots, layer.weight.sample_free_positions(slots.shape[0], 5))
    assert layer.weight.pattern_status() == 0
    for tokens in (5, 100):
        with torch.no_grad():
            assert rel(layer(x[:tokens].cuda()), reference(layer, x[:tokens])) <= bound("tf32x3", 3)


def test_shapes_strides_streams_and_empty_batches():
    layer = make(64, 96, 0.6, seed=7)
    wide = randn((3, 40, 70), 1).cuda()
    x = wide[:, :, 1:65]
    for rows in (slice(0, 2), slice(0, 40)):
        with torch.no_grad():
            want = layer(x[:, rows].contiguous())
            assert want.shape == (3, rows.stop, 96)
            assert torch.equal(layer(x[:, rows]), want)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got = layer(x[:, rows])
            side.synchronize()
            assert torch.equal(got, want)
    with torch.no_grad():
        assert layer(x[:, :0]).shape == (3, 0, 96)
        flat = wide.reshape(-1)[1:65].view(1, 64)  # contiguous, not on a 16-byte boundary
        assert torch.equal(layer(flat), layer(flat.clone()))
    empty = torch.empty((0, 64), device="cuda", requires_grad=True)
    h = layer(empty)
    g = torch.autograd.grad(h, [empty, layer.weight.data, layer.bias], torch.empty((0, 96), device="cuda"))
    assert g[0].shape == (0, 64) and (g[1] == 0).all() and (g[2] == 0).all()
    # an expanded output gradient
    xg = x[0].detach().clone().requires_grad_()
    layer(xg).sum().backward()
    want = reference(layer, xg.detach(), torch.ones(40, 96))
    assert rel(xg.grad, want[1]) <= bound("tf32x3", 4)


@pytest.mark.parametrize("tokens", [4, 200])
def test_captured_inference_follows_its_inputs_and_weights(tokens):
    layer = make(128, 64, 0.6, precision="bf16", seed=8)
    x = randn((tokens, 128), 1).bfloat16().cuda()
    with torch.no_grad():
        layer(x)  # the first call per device, and the plans, before the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x)
        for seed in (2, 3):
            x.copy_(randn((tokens, 128), seed))
            layer.weight.data.mul_(-0.5)
            graph.replay()
            assert torch.equal(out, layer(x))
    assert_device_healthy()


def test_a_captured_training_step():
    layer = make(128, 64, 0.6, seed=9)
    x, dh = randn((64, 128), 1).cuda().requires_grad_(), randn((64, 64), 2).cuda()
    leaves = [x, layer.weight.data, layer.bias]

    def step():
        h = layer(x)
        return [h.detach(), *torch.autograd.grad(h, leaves, dh)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        x.copy_(randn((64, 128), 3))
        layer.weight.data.mul_(1.5)
    graph.replay()
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("precision", [None, "bf16"])
def test_a_first_call_under_capture_leaves_nothing_behind(precision):
    """Plans built while capturing are the graph's: an eager call before any replay must build its own."""
    layer = make(128, 96, 0.5, precision=precision, seed=11)
    dtype = torch.bfloat16 if precision else torch.float32
    x = randn((200, 128), 1).to(dtype).cuda()
    with torch.no_grad():
        make(128, 96, 0.5, precision=precision, seed=12)(x)  # the device's first call, with another layer
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x)
        eager = layer(x)
        assert rel(eager, reference(layer, x)) <= bound(precision or "tf32x3", 3, dtype)
        graph.replay()
        assert torch.equal(out, eager)
        side = torch.cuda.Stream()
        layer.weight._plan_cache = {}
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x)  # builds on the side stream
        assert torch.equal(layer(x), eager)
    torch.cuda.synchronize()
    assert_device_healthy()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("tokens,inner,hidden,density,same", [
    (33, 32, 32, 1.0, True), (128, 64, 128, 1.0, True), (129, 544, 160, 0.5, True), (400, 1056, 1184, 0.15, False),
    (300, 4096, 96, 0.6, True), (1500, 256, 4000, 0.3, False), (2049, 96, 2080, 0.05, False),
])
def test_the_bf16_kernel_alone(act, tokens, inner, hidden, density, same):
    """Weights that bf16 holds: only the sums and the output round, so the bar is the output's type (half a step)."""
    hidden = hidden // 32 * 32
    g = torch.Generator().manual_seed(tokens)
    mask = torch.rand((hidden // 16, inner // 32), generator=g) < density
    if same:
        mask[1::2] = mask[0::2]
    layer = make(inner, hidden, act=act, precision="bf16", mask=mask, seed=tokens, bf16_values=True)
    x, dh = randn((tokens, inner), 6).bfloat16(), randn((tokens, hidden), 7).bfloat16()
    want = reference(layer, x, dh)
    with torch.no_grad():
        h = layer(x.cuda())
    # each sum of K terms in fp32 is within K 2^-23 of the magnitudes, here far below the output's half step: 1.1 of it
    assert rel(h, want[0]) <= 1.1 * 2.0 ** -8
    assert torch.isfinite(h).all()
    xg = x.cuda().requires_grad_()
    got = layer(xg)
    assert torch.equal(got, h)
    got.backward(dh.cuda())
    assert rel(xg.grad, want[1]) <= bound("bf16", 4, torch.bfloat16, 1)
    assert rel(layer.weight.data.grad, in_data_layout(layer, want[2])) <= bound("bf16", 4, roundings=1)
    assert rel(layer.bias.grad, want[3]) <= bound("bf16", 4, roundings=1)
    assert_device_healthy()


@pytest.mark.parametrize("tokens,inner,hidden,density,same", [
    (32, 32, 32, 1.0, True), (63, 64, 96, 1.0, True), (64, 32, 32, 1.0, True), (65, 64, 96, 1.0, True), (100, 544, 160, 0.5, False), (1024, 1056, 96, 0.4, True),
    (1025, 96, 1184, 0.3, False), (2500, 2080, 64, 0.7, True), (6001, 256, 512, 0.2, True), (4096, 64, 4096, 0.6, False),
])
def test_the_fp32_weight_gradient(tokens, inner, hidden, density, same):
    """Three bf16 parts of every value: what is dropped is 2^-24 of a term, the sums drift by 2e-8 per addition over segments
    of 64: 2e-6 of the norm, far inside the 1e-5 of the precision's products."""
    g = torch.Generator().manual_seed(tokens)
    mask = torch.rand((hidden // 16, inner // 32), generator=g) < density
    if same:
        mask[1::2] = mask[0::2]
    layer = make(inner, hidden, mask=mask, seed=tokens)
    passes = gated_linear._gated_pass(layer.weight)
    x, pre, dh = randn((tokens, inner), 1).cuda(), randn((tokens, 2 * hidden), 2).cuda(), randn((tokens, hidden), 3).cuda()
    data = layer.weight.data.detach()
    got = passes.backward(x, pre, dh, data, None, "silu", native.PREC_TF32X3, False, True, True)
    dpre, _ = native.gated_act_backward(pre, dh, "silu", False)  # the product alone is on trial
    want = in_data_layout(layer, dpre.cpu().double().t() @ x.cpu().double())
    assert got[0] is None and torch.isfinite(got[1]).all()
    assert rel(got[1], want) <= 2e-6
    assert torch.allclose(got[3].cpu().double(), want.view(-1, 1024).square().sum(1), rtol=2e-5, atol=1e-12)
    assert rel(got[2], dpre.cpu().double().sum(0)) <= 1e-6
    again = passes.backward(x, pre, dh, data, None, "silu", native.PREC_TF32X3, False, True, True)
    assert torch.equal(again[1], got[1]) and torch.equal(again[3], got[3])
    assert_device_healthy()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("tokens,inner,hidden,density,same", [
    (1, 32, 32, 1.0, True), (33, 64, 96, 1.0, True), (128, 544, 160, 0.5, False), (129, 1056, 96, 0.4, True),
    (256, 96, 1184, 0.3, False), (257, 2080, 64, 0.7, True), (1000, 4096, 96, 0.9, True), (700, 64, 4096, 0.6, False),
])
def test_the_fp32_kernel_alone(act, tokens, inner, hidden, density, same):
    """g and u to 2e-6 of their norm (three bf16 parts: 2^-24 of a term is dropped; the sums drift by 2e-8 per addition over
    segments of 64), rows longer than a segment among them; h by 3 times that, the same with and without g and u kept."""
    g = torch.Generator().manual_seed(tokens)
    mask = torch.rand((hidden // 16, inner // 32), generator=g) < density
    if same:
        mask[1::2] = mask[0::2]
    mask[:2] = True
    layer = make(inner, hidden, act=act, mask=mask, seed=tokens)
    x = randn((tokens, inner), 1)
    passes = gated_linear._gated_pass(layer.weight)
    data, bias = layer.weight.data.detach(), layer.bias.detach()
    h, pre, packed = passes.forward(x.cuda(), data, bias, act, native.PREC_TF32X3, torch.float32)
    assert packed is None and torch.isfinite(pre).all()
    want = x.double() @ layer.weight.to_dense().detach().cpu().double().t() + bias.cpu().double()
    assert rel(pre, want) <= 2e-6
    assert rel(h, reference(layer, x)) <= 6e-6
    alone = passes.forward(x.cuda(), data, bias, act, native.PREC_TF32X3, torch.float32, keep=False)
    assert alone[1] is None and torch.equal(alone[0], h)
    assert torch.equal(native.gated_act(pre, act, torch.float32), h)
    assert_device_healthy()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("tokens,inner,hidden,density,same", [
    (1, 32, 32, 1.0, True), (33, 96, 64, 1.0, True), (64, 160, 544, 0.5, False), (129, 96, 1056, 0.4, True), (257, 2080, 64, 0.3, False),
    (1000, 96, 4096, 0.9, True), (700, 4096, 64, 0.6, False), (2500, 1056, 1184, 0.2, True), (300, 64, 32 * 1100, 0.05, False),
    (128 * 149 + 1, 32, 64, 1.0, True), (5000, 4096, 96, 0.02, False),
])
def test_the_fp32_input_gradient(act, tokens, inner, hidden, density, same):
    """Three bf16 parts of every value, as the weight gradient: 2e-6 of the norm.  Columns without a block get zeros."""
    g = torch.Generator().manual_seed(tokens)
    mask = torch.rand((hidden // 16, inner // 32), generator=g) < density
    if same:
        mask[1::2] = mask[0::2]
    mask[0, 0] = True
    layer = make(inner, hidden, act=act, mask=mask, seed=tokens)
    passes = gated_linear._gated_pass(layer.weight)
    x, pre, dh = randn((tokens, inner), 1).cuda(), randn((tokens, 2 * hidden), 2).cuda(), randn((tokens, hidden), 3).cuda()
    data = layer.weight.data.detach()
    got = passes.backward(x, pre, dh, data, None, act, native.PREC_TF32X3, True, False, False)
    dpre, _ = native.gated_act_backward(pre, dh, act, False)
    want = dpre.cpu().double() @ layer.weight.to_dense().detach().cpu().double()
    assert got[1] is None and got[2] is None and torch.isfinite(got[0]).all()
    assert rel(got[0], want) <= 2e-6
    assert (got[0].cpu()[want == 0] == 0).all()
    again = passes.backward(x, pre, dh, data, None, act, native.PREC_BF16X3, True, True, True)
    assert torch.equal(again[0], got[0])
    assert_device_healthy()


@pytest.mark.parametrize("precision", ["tf32x3", "fp32", "bf16"])
def test_no_tokens_with_gradients(precision):
    layer = make(64, 96, precision=precision)
    x = torch.empty((2, 0, 64), device="cuda", dtype=torch.bfloat16 if precision == "bf16" else torch.float32, requires_grad=True)
    h = layer(x)
    assert h.shape == (2, 0, 96)
    got = torch.autograd.grad(h.sum(), [x, layer.weight.data, layer.bias])
    assert got[0].shape == x.shape and not got[1].any() and not got[2].any()
    assert_device_healthy()


@pytest.mark.parametrize("precision,dtype", [("tf32x3", torch.float32), ("bf16", torch.bfloat16), ("fp32", torch.float32)])
@pytest.mark.parametrize("tokens", [3, 20, 300])
def test_non_finite_tokens_stay_alone(precision, dtype, tokens):
    """A token with a NaN or an infinity loses its own h and dx, every other token's stay bit for bit."""
    layer = make(160, 96, density=0.6, precision=precision)
    x, dh = randn((tokens, 160), 1).cuda().to(dtype), randn((tokens, 96), 2).cuda().to(dtype)
    broken = x.clone()
    broken[1, ::7] = float("nan")
    broken[tokens - 1, 3] = float("inf")
    rest = [t for t in range(tokens) if t not in (1, tokens - 1)]
    with torch.no_grad():
        assert torch.equal(layer(broken)[rest], layer(x)[rest])
        assert torch.isnan(layer(broken)[1]).any()
    got = []
    for v in (x, broken):
        v = v.clone().requires_grad_()
        h = layer(v)
        got.append((h.detach(), torch.autograd.grad(h, v, dh)[0]))
    for a, b in zip(*got):
        assert torch.equal(a[rest], b[rest])
    assert_device_healthy()


@pytest.mark.parametrize("precision,dtype", [("tf32x3", torch.float32), ("bf16", torch.bfloat16)])
def test_offsets_past_32_bits(precision, dtype):
    """g and u of more than 2^31 values: the first and last tokens' h and dx, and the weight gradient of a gradient that only they
    have, against a call on those tokens alone."""
    tokens, inner, hidden = 270001, 64, 4096
    layer = make(inner, hidden, density=0.5, precision=precision)
    x = torch.randn((tokens, inner), device="cuda").to(dtype).requires_grad_()
    ends = torch.cat([torch.arange(200), torch.arange(tokens - 200, tokens)]).cuda()
    h = layer(x)
    dh = torch.zeros_like(h)
    dh[ends] = torch.randn((400, hidden), device="cuda").to(dtype)
    dx, dw, db = torch.autograd.grad(h, [x, layer.weight.data, layer.bias], dh)
    xs = x.detach()[ends].requires_grad_()
    hs = layer(xs)
    want = torch.autograd.grad(hs, [xs, layer.weight.data, layer.bias], dh[ends])
    assert torch.equal(h.detach()[ends], hs.detach()) and torch.equal(dx[ends], want[0])
    assert not dx[1000:-1000].any()
    tolerance = 4e-6 if precision == "tf32x3" else 2e-2  # sums in another order (bf16: of rounded terms)
    assert rel(dw, want[1].cpu().double()) <= tolerance and rel(db, want[2].cpu().double()) <= tolerance
    assert_device_healthy()
    del h, dh, x, dx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("precision,dtype", [("tf32x3", torch.float32), ("bf16", torch.bfloat16)])
def test_steps_on_two_streams_at_once(precision, dtype):
    """The first steps of a layer, whose plans the first call builds, on two streams that do not wait for one another."""
    xs = [randn((700, 1024), i).cuda().to(dtype) for i in range(2)]
    dh = randn((700, 512), 5).cuda().to(dtype)

    def step(layer, x):
        x = x.clone().requires_grad_()
        h = layer(x)
        return (h.detach(), *torch.autograd.grad(h, [x, layer.weight.data, layer.bias], dh))

    want = [step(make(1024, 512, precision=precision), x) for x in xs]
    layer = make(1024, 512, precision=precision)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for stream, x in zip(streams, xs):
        with torch.cuda.stream(stream):
            got.append([step(layer, x) for _ in range(4)])
    torch.cuda.synchronize()
    for rounds, expected in zip(got, want):
        for values in rounds:
            assert all(torch.equal(a, b) for a, b in zip(values, expected))
    assert_device_healthy()


def test_a_second_differentiation_raises():
    layer = make(64, 96)
    x = randn((40, 64), 1).cuda().requires_grad_()
    want = torch.autograd.grad(layer(x).square().sum(), [x, layer.weight.data])
    got = torch.autograd.grad(layer(x).square().sum(), [x, layer.weight.data], create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got[0].sum().backward()


def test_copies_and_pickles_leave_the_plans_behind():
    layer = make(96, 64)
    x = randn((70, 96), 1).cuda()
    layer(x.requires_grad_()).sum().backward()
    want = layer(x)
    buffer = io.BytesIO()
    torch.save(layer, buffer)
    buffer.seek(0)
    for other in (copy.deepcopy(layer), torch.load(buffer, weights_only=False)):
        assert torch.equal(other(x), want)


def test_the_sparsity_optimizer_moves_blocks_of_the_layer():
    layer = make(128, 256, density=0.25)
    x, dh = randn((100, 128), 1).cuda(), randn((100, 256), 2).cuda()
    sparse = SparseOptimizer(SparseOptimizer.sparse_objects(layer), lr=0.25, new_coefficients_scale=1.0, seed=1)
    adam = torch.optim.Adam(layer.parameters(), lr=1e-3)
    sparse.attach_optimizer(adam)
    layer(x).backward(dh)  # plans exist before the pattern changes
    before = layer.weight.to_dense().detach().clone()
    adam.step()
    sparse.step()
    assert not torch.equal(before != 0, layer.weight.to_dense().detach() != 0)
    xs = x.clone().requires_grad_()
    h = layer(xs)
    dx, dw = torch.autograd.grad(h, [xs, layer.weight.data], dh)
    want = reference(layer, x, dh)
    assert rel(h, want[0]) <= 1e-5 and rel(dx, want[1]) <= 1e-5 and rel(dw, in_data_layout(layer, want[2])) <= 1e-5


def test_from_linears_and_state_dict():
    torch.manual_seed(0)
    gate, up = torch.nn.Linear(96, 64), torch.nn.Linear(96, 64)
    layer = BlockSparseGatedLinear.from_linears(gate, up)
    dense = layer.to_dense()
    assert torch.equal(dense[0].cpu(), gate.weight) and torch.equal(dense[1].cpu(), up.weight)
    x = randn((50, 96), 1)
    want = torch.nn.functional.silu(gate.double()(x.double())) * up.double()(x.double())
    with torch.no_grad():
        assert rel(layer(x.cuda()), want.detach()) <= bound("tf32x3", 3)
        assert rel(layer(x[:3].cuda()), want[:3].detach()) <= bound("fp32", 3)
    np.random.seed(1)
    half = BlockSparseGatedLinear.from_linears(gate.float(), up.float(), density=0.5, activation="gelu")
    stored = half.weight.to_dense(data_replace=torch.ones_like(half.weight.data)) == 1
    full = interleave_rows(gate.weight.detach(), up.weight.detach()).cuda()
    assert torch.allclose(half.weight.to_dense(), torch.where(stored, full / math.sqrt(0.5), 0.0))
    np.random.seed(2)
    other = BlockSparseGatedLinear(96, 64, density=0.5, activation="gelu")
    other.load_state_dict(half.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x.cuda()), half(x.cuda()))
    a, b = split_rows(interleave_rows(gate.weight, up.weight))
    assert torch.equal(a, gate.weight) and torch.equal(b, up.weight)


def test_a_feed_forward_block_trains_and_serves():
    """Gated projections, output projection with dropout, residual and per-request adapters together, against 64 bits."""
    np.random.seed(3)
    torch.manual_seed(3)
    up = make(128, 256, 0.5, seed=10)
    down = BlockSparseLinear(256, 128, density=0.5, dropout=0.2)
    with torch.no_grad():
        down.weight.data.normal_(0, 128 ** -0.5)
        down.bias.normal_(0, 0.1)
    x, dy = randn((2, 35, 128), 1), randn((2, 35, 128), 2)
    xg = x.cuda().requires_grad_()
    torch.manual_seed(4)
    seed, counter = torch.randint(1 << 62, (2,), device="cuda").tolist()
    torch.manual_seed(4)
    out = down(up(xg), residual=xg)
    leaves = [xg, up.weight.data, up.bias, down.weight.data, down.bias]
    got = torch.autograd.grad(out, leaves, dy.cuda())
    # 64 bits, by autograd on the host
    from .test_dropout_gpu import philox_halves

    keep = torch.from_numpy(philox_halves(out.numel(), seed, counter) >= round(0.2 * 65536)).view(70, 128)
    host = [x.double().reshape(-1, 128), up.weight.to_dense().detach().cpu().double(), up.bias.detach().cpu().double(),
            down.weight.to_dense().detach().cpu().double(), down.bias.detach().cpu().double()]
    host = [t.requires_grad_() for t in host]
    g, u = columns(host[0] @ host[1].t() + host[2])
    h = g * torch.sigmoid(g) * u
    y = torch.where(keep, (h @ host[3].t() + host[4]) * (65536 / (65536 - round(0.2 * 65536))), 0.0) + host[0]
    want = torch.autograd.grad(y, host, dy.double().reshape(-1, 128))
    assert rel(out.reshape(-1, 128), y.detach()) <= bound("tf32x3", 4)
    assert rel(got[0].reshape(-1, 128), want[0]) <= bound("tf32x3", 6)
    assert rel(got[1], in_data_layout(up, want[1])) <= bound("tf32x3", 6)
    assert rel(got[2], want[2]) <= bound("tf32x3", 6)
    blocks = down.weight.blocks.view(-1, 2).cpu().long()
    grid = want[3].reshape(4, 32, 8, 32)
    assert rel(got[3], grid[blocks[:, 1], :, blocks[:, 0], :].transpose(1, 2).reshape(-1, 32)) <= bound("tf32x3", 5)
    assert rel(got[4], want[4]) <= bound("tf32x3", 2)
    # serving: no dropout, an adapter for one of the two requests
    up.eval(), down.eval()
    ad = LowRankAdapters(256, 128, 2, 8)
    ad.load(1, randn((8, 256), 5).cuda() / 16, randn((128, 8), 6).cuda())
    requests = AdapterRequests.from_lengths([35, 35], [None, 1])
    with torch.no_grad():
        served = down(up(x.cuda()), residual=x.cuda(), adapters=(ad, requests))
    y = (h @ host[3].t() + host[4] + host[0]).detach()
    y[35:] += h.detach()[35:] @ (randn((8, 256), 5).double() / 16).t() @ randn((128, 8), 6).double().t()
    assert rel(served.reshape(-1, 128), y) <= bound("tf32x3", 6)
    assert_device_healthy()
