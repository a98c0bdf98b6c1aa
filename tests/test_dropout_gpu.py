"""Dropout from the counter-based generator with the residual add: the mask against a numpy statement of Philox4x32-10
bit by bit, values against 64 bits, the gradient, streams, graphs and the layer that carries it."""
import copy

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

from pytorch_block_sparse_b200 import BlockSparseLinear, dropout_residual, new_rng_state, next_rng

from .gpu_util import randn

pytestmark = pytest.mark.gpu


def philox_halves(count, seed, counter):
    """The first ``count`` 16-bit numbers of the stream: words of Philox4x32-10 with counter (i, counter) and key seed."""
    mask = 0xFFFFFFFF
    i = np.arange((count + 7) // 8, dtype=np.uint64)
    c = [i & np.uint64(mask), i >> np.uint64(32), np.full_like(i, counter & mask), np.full_like(i, (counter >> 32) & mask)]
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & np.uint64(mask),
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & np.uint64(mask)]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = np.stack(c, 1)
    return np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)[:count]


def rng_of(seed, counter):
    return torch.tensor([seed, counter], dtype=torch.int64, device="cuda")


def expected(x, residual, p, seed, counter):
    cut = round(p * 65536)
    keep = torch.from_numpy(philox_halves(x.numel(), seed, counter) >= cut).view(x.shape)
    kept = torch.where(keep, x.double() * (65536 / (65536 - cut)), torch.zeros((), dtype=torch.float64))
    return kept + (residual.double() if residual is not None else 0), keep, kept


# The published known answers of Philox4x32-10 for the all-zero and the all-one counter and key.
def test_the_statement_of_the_generator_gives_the_published_words():
    def words(seed, counter, index):
        h = philox_halves(8, seed, counter) if index == 0 else None
        return h[0::2] | (h[1::2] << np.uint64(16))

    assert [int(w) for w in words(0, 0, 0)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (1, 1), (3, 5, 11), (257, 1003), (64, 4096)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999])
@pytest.mark.parametrize("with_residual", [False, True])
def test_values_mask_and_gradient(dtype, shape, p, with_residual):
    x = randn(shape, 1).to(dtype)
    residual = randn(shape, 2).to(dtype) if with_residual else None
    dout = randn(shape, 3).to(dtype)
    seed, counter = (1 << 61) + 12345678901, (1 << 33) + 7
    want, keep, kept = expected(x, residual, p, seed, counter)
    xg = x.cuda().requires_grad_()
    rg = residual.cuda().requires_grad_() if with_residual else None
    out = dropout_residual(xg, p, rng_of(seed, counter), residual=rg)
    assert out.dtype == dtype and out.shape == x.shape
    # fp32: the scale, the product and the sum round once each (half a step, 2^-24); bf16 output: half a step, 2^-8
    half = torch.finfo(torch.float32).eps / 2
    out_half = torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 0.0
    tol = 3 * half * (kept.abs() + want.abs()) + out_half * want.abs() * (1 + 2 ** -7)
    assert ((out.detach().cpu().double() - want).abs() <= tol).all()
    out.backward(dout.cuda())
    dx, _, dkept = expected(dout, None, p, seed, counter)
    got = xg.grad.cpu().double()
    assert ((got - dx).abs() <= 3 * half * dkept.abs() + out_half * dx.abs() * (1 + 2 ** -7)).all()
    assert (got[~keep] == 0).all()
    if with_residual:
        assert torch.equal(rg.grad.cpu(), dout)


def test_the_gradient_agrees_with_differences():
    x, v, w = (randn((33, 95), s).cuda() for s in (4, 5, 6))
    rng = rng_of(9, 9)
    x.requires_grad_()
    (g,) = torch.autograd.grad(dropout_residual(x, 0.3, rng), x, w)
    with torch.no_grad():  # linear in x: the difference is exact up to the rounding of its two terms
        up, down = (dropout_residual(x + s * v, 0.3, rng).double() for s in (0.5, -0.5))
        diff = ((up - down) * w).sum().item()
        size = ((up.abs() + down.abs()) * w.abs()).sum().item()
    assert abs(diff - (g.double() * v).sum().item()) <= 8 * 2.0 ** -24 * size


def test_a_gradient_of_the_gradient():
    x, v = randn((16, 40), 4).cuda().requires_grad_(), randn((16, 40), 5).cuda().requires_grad_()
    rng = rng_of(9, 9)
    (g,) = torch.autograd.grad(dropout_residual(x * x, 0.3, rng), x, v, create_graph=True)  # 2 x v keep / (1 - p)
    gx, gv = torch.autograd.grad(g.sum(), [x, v])
    keep = torch.from_numpy(philox_halves(x.numel(), 9, 9) >= round(0.3 * 65536)).view(x.shape).cuda()
    scale = keep * (65536 / (65536 - round(0.3 * 65536)))
    assert torch.allclose(gx, 2 * v * scale, rtol=1e-6) and torch.allclose(gv, 2 * x * scale, rtol=1e-6)


def test_non_finite_values():
    x = randn((64, 64), 7)
    x[::3, ::2] = float("inf")
    x[1::3, 1::2] = float("nan")
    x[2::3] = -float("inf")
    residual = randn((64, 64), 8)
    out = dropout_residual(x.cuda(), 0.5, rng_of(1, 2), residual=residual.cuda()).cpu()
    keep = torch.from_numpy(philox_halves(x.numel(), 1, 2) >= 32768).view(x.shape)
    assert torch.equal(out[~keep], residual[~keep])  # nothing of a dropped value is left
    assert torch.isnan(out[keep & torch.isnan(x)]).all()
    assert (out[keep & torch.isinf(x)] == x[keep & torch.isinf(x)]).all()


def test_strides_views_streams_and_empty_tensors():
    base = randn((48, 130), 10).cuda()
    rng = rng_of(3, 4)
    want = dropout_residual(base[:, 1:129].contiguous(), 0.25, rng, residual=base[:, :128].contiguous())
    assert torch.equal(dropout_residual(base[:, 1:129], 0.25, rng, residual=base[:, :128]), want)
    flat = base.view(-1)[1:1001]  # contiguous, but not on a 16-byte boundary
    assert torch.equal(dropout_residual(flat, 0.25, rng), dropout_residual(flat.clone(), 0.25, rng))
    assert dropout_residual(torch.empty((0, 5), device="cuda"), 0.25, rng).shape == (0, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dropout_residual(base[:, 1:129], 0.25, rng, residual=base[:, :128])
    side.synchronize()
    assert torch.equal(got, want)
    # an expanded residual gradient: a broadcast input sums its gradient
    row = randn((1, 128), 11).cuda().requires_grad_()
    dropout_residual(base[:, :128].contiguous(), 0.25, rng, residual=row.expand(48, 128)).sum().backward()
    assert torch.equal(row.grad, torch.full_like(row, 48.0))


def test_large_element_indices():
    """Groups beyond 2^32 elements would take 8 GB; the counter's carry is checked through the generator, the element
    index here past 2^31."""
    n = (1 << 31) + 24
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    out = dropout_residual(x, 0.5, rng_of(5, 6))
    tail = out[-40:].float().cpu().numpy()
    # the last 40 elements are groups (n - 40) / 8 ... : draw those alone
    first = (n - 40) // 8
    i = np.arange(first, first + 5, dtype=np.uint64)
    mask = np.uint64(0xFFFFFFFF)
    c = [i & mask, i >> np.uint64(32), np.full_like(i, 6), np.zeros_like(i)]
    k0, k1 = 5, 0
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & mask, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & mask]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = np.stack(c, 1)
    halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)
    assert np.array_equal(tail, np.where(halves >= 32768, 2.0, 0.0))


def test_a_state_moves_on_and_a_captured_call_draws_anew():
    state = new_rng_state("cuda", seed=42)
    first, second = next_rng(state), next_rng(state)
    assert first.tolist() == [42, 0] and second.tolist() == [42, 1] and state.tolist() == [42, 2]
    x = torch.ones((128, 256), device="cuda")
    out = torch.empty_like(x)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out.copy_(dropout_residual(x, 0.5, next_rng(state)))
    masks = []
    for counter in (2, 3):
        graph.replay()
        torch.cuda.synchronize()
        keep = philox_halves(x.numel(), 42, counter) >= 32768
        assert np.array_equal(out.cpu().numpy().reshape(-1) != 0, keep)
        masks.append(keep)
    assert not np.array_equal(*masks)
    assert new_rng_state("cuda").tolist()[0] != new_rng_state("cuda").tolist()[0]


def test_the_layer_drops_its_output_in_training_only():
    np.random.seed(0)
    torch.manual_seed(0)
    lin = BlockSparseLinear(128, 96, density=0.5, dropout=0.25)
    with torch.no_grad():
        lin.weight.data.normal_(0, 0.1)
        lin.bias.normal_()
    x, residual, dy = randn((4, 9, 128), 1).cuda(), randn((4, 9, 96), 2).cuda(), randn((4, 9, 96), 3).cuda()
    assert sorted(lin.state_dict()) == sorted(BlockSparseLinear(128, 96, density=0.5).state_dict())
    plain = BlockSparseLinear(128, 96, density=0.5)
    plain.weight, plain.bias = lin.weight, lin.bias
    torch.manual_seed(3)
    seed, counter = torch.randint(1 << 62, (2,), device="cuda").tolist()
    torch.manual_seed(3)
    xa, ra = x.clone().requires_grad_(), residual.clone().requires_grad_()
    out = lin(xa, residual=ra)
    keep = torch.from_numpy(philox_halves(out.numel(), seed, counter) >= 16384).view(out.shape).cuda()
    xb = x.clone().requires_grad_()
    y = plain(xb)
    want = torch.where(keep, y * (65536 / 49152), 0.0) + residual
    assert torch.allclose(out, want, rtol=1e-6, atol=1e-6)
    got = torch.autograd.grad(out, [xa, ra, lin.weight.data, lin.bias], dy)
    ref = torch.autograd.grad(y, [xb, lin.weight.data, lin.bias], torch.where(keep, dy * (65536 / 49152), 0.0))
    assert torch.equal(got[1], dy)
    for a, b in zip((got[0], got[2], got[3]), ref):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
    lin.eval()
    assert torch.equal(lin(x, residual=residual), plain(x, residual=residual))


def test_checkpointed_copied_and_captured_layers():
    """What torch's own dropout does: a recomputed forward pass draws the same mask again, a copy of a layer draws others than
    the layer, a captured step draws anew in every replay."""
    np.random.seed(0)
    torch.manual_seed(0)
    lin = BlockSparseLinear(64, 64, density=1.0, dropout=0.5)
    with torch.no_grad():
        lin.weight.data.normal_(0, 0.1)
    x = randn((100, 64), 1).cuda().requires_grad_()
    torch.manual_seed(7)
    (want,) = torch.autograd.grad(lin(x).square().sum(), x)
    torch.manual_seed(7)
    (got,) = torch.autograd.grad(torch.utils.checkpoint.checkpoint(lin, x, use_reentrant=False).square().sum(), x)
    assert torch.equal(got, want)
    torch.manual_seed(7)
    assert not torch.equal(lin(x) == 0, copy.deepcopy(lin)(x) == 0)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(stream):
        lin(x)
    torch.cuda.synchronize()
    with torch.no_grad(), torch.cuda.graph(graph, stream=stream):
        out = lin(x)
    masks = []
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        masks.append((out == 0).cpu())
    assert not torch.equal(*masks) and 0.4 < masks[0].float().mean().item() < 0.6
