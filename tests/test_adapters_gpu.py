"""Low-rank adapters of many requests against 64-bit arithmetic: request mixes, ranks, types, padding, graphs, streams, and the
shared projection they stand beside."""
import numpy as np
import pytest
import torch

from pytorch_block_sparse_b200 import AdapterRequests, BlockSparseLinear, LowRankAdapters

from .gpu_util import assert_device_healthy, randn

pytestmark = pytest.mark.gpu


def make(inner, outer, count, rank, dtype, seed=0):
    """Adapters with values of ``dtype``; returns them and their (down, up, scaling) in 64 bits."""
    down = randn((count, rank, inner), seed).div_(inner ** 0.5).to(dtype)
    up = randn((count, outer, rank), seed + 1).div_(rank ** 0.5).to(dtype)
    scaling = torch.linspace(0.5, 2.0, count)
    ad = LowRankAdapters(inner, outer, count, rank, dtype=dtype)
    ad.load_all(down.cuda(), up.cuda(), scaling.cuda())
    return ad, (down.double(), up.double(), scaling.double())


def reference(x, lengths, ids, weights, base):
    """``(y, bound)``: the result in 64 bits, and the sum of the magnitudes of its terms' factors that rounding acts on."""
    down, up, scaling = weights
    y = base.double().clone()
    s1 = torch.zeros_like(y)  # |scale| (|x| |D|^T) |U|^T
    at = 0
    for n, a in zip(lengths, ids):
        if a is not None and a >= 0 and n > 0:
            rows = slice(at, at + n)
            xr = x[rows].double()
            y[rows] += scaling[a] * (xr @ down[a].t()) @ up[a].t()
            s1[rows] = scaling[a] * (xr.abs() @ down[a].abs().t()) @ up[a].abs().t()
        at += n
    return y, s1


def tolerance(y, s1, dtype, out_dtype, inner, rank):
    """Elementwise: fp32 sums in the tensor core (at most one step, 2^-23, of the sum of magnitudes per addition, one
    addition per 16 products and one per partial sum), the split into bf16 hi and lo parts (2^-16 of an operand is dropped,
    twice for fp32 inputs in each product, once for v with bf16 ones), and the output's own rounding (half a step)."""
    adds = inner / 16 + rank / 16 + 40
    split = 6 * 2.0 ** -16 if dtype == torch.float32 else 2.0 ** -16
    out_half = torch.finfo(out_dtype).eps / 2
    return (adds * 2.0 ** -23 + split) * s1 + out_half * y.abs() * (1 + 2.0 ** -7) + 2.0 ** -23 * y.abs()


def check(got, x, lengths, ids, weights, base, dtype, inner, rank):
    y, s1 = reference(x, lengths, ids, weights, base)
    got = got.cpu()
    assert torch.isfinite(got).all()
    off = (got.double() - y).abs()
    assert (off <= tolerance(y, s1, dtype, got.dtype, inner, rank)).all(), float((off / (s1 + 1e-30)).max())
    if got.dtype == torch.float32:  # fp32 class: each of the two products within 1e-5 of its norm
        delta = y - base.double()
        assert torch.linalg.norm(got.double() - y) <= 2e-5 * torch.linalg.norm(delta) + 2.0 ** -24 * torch.linalg.norm(y)


MIXES = {
    "one token": ([1], [0]),
    "single tokens": ([1] * 37, [i % 5 for i in range(37)]),
    "single tokens, one adapter": ([1] * 20, [2] * 20),
    "prompts": ([50, 3, 0, 129, 16, 0, 17], [0, 1, 2, 3, 4, 0, 2]),
    "some without": ([5, 7, 0, 40, 1], [None, 3, 1, None, 0]),
    "none at all": ([4, 9], [None, None]),
    "a prompt among tokens": ([1, 1, 1, 200, 1, 1], [4, 3, 2, 1, 0, 4]),
    "a prompt of many clusters": ([300, 7], [1, 3]),
    "more requests than a warp asks for at once": ([1, 0, 2] * 60, [i % 5 for i in range(180)]),
}


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("types", ["fp32", "bf16", "bf16 in fp32"])
@pytest.mark.parametrize("sizes", [(32, 32, 1), (96, 160, 8), (1056, 544, 16), (256, 96, 24), (160, 2080, 64), (64, 64, 100)])
def test_mixes_ranks_and_types(mix, types, sizes):
    run_mix(*MIXES[mix], types, sizes)


def run_mix(lengths, ids, types, sizes):
    inner, outer, rank = sizes
    dtype = torch.float32 if types == "fp32" else torch.bfloat16
    out_dtype = torch.bfloat16 if types == "bf16" else torch.float32
    ad, weights = make(inner, outer, 5, rank, dtype, seed=3)
    tokens = sum(lengths)
    x, base = randn((tokens, inner), 5).to(dtype), randn((tokens, outer), 6).to(out_dtype)
    requests = AdapterRequests.from_lengths(lengths, ids)
    with torch.no_grad():
        got = ad(x.cuda(), requests, base=base.cuda())
        assert got.dtype == out_dtype
        check(got, x, lengths, ids, weights, base, dtype, inner, rank)
        again = base.cuda()
        assert ad(x.cuda(), requests, base=again, inplace=True) is again
        assert torch.equal(again, got)  # in place, and the same bits a second time
        alone = ad(x.cuda(), requests, dtype=out_dtype)
        check(alone, x, lengths, ids, weights, torch.zeros_like(base), dtype, inner, rank)
    assert_device_healthy()


PROMPTS = {  # long enough for the form that owns 128 tokens at a time
    "one": ([769], [1]),
    "odd": ([577, 130, 0, 1, 3, 129], [0, 3, 1, 2, None, 4]),
    "many adapters near one another": ([700, 5, 1, 7, 2, 30, 1, 60], [0, 1, 2, 3, 4, 0, 1, 2]),
    "none but one": ([400, 20, 400], [None, 4, None]),
    "more requests than a warp asks for at once": ([40] * 70, [i % 6 - 1 for i in range(70)]),
}


@pytest.mark.parametrize("mix", PROMPTS)
@pytest.mark.parametrize("types", ["fp32", "bf16", "bf16 in fp32"])
@pytest.mark.parametrize("sizes", [(32, 32, 1), (96, 160, 16), (1056, 544, 24), (544, 2080, 64), (64, 96, 200), (64, 64, 64),
                                   (4128, 288, 48), (160, 4128, 128), (96, 32, 100)])
def test_prompts(mix, types, sizes):
    run_mix(*PROMPTS[mix], types, sizes)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rank", [128, 256, 200])
def test_large_ranks(dtype, rank):
    ad, weights = make(320, 192, 3, rank, dtype, seed=9)
    lengths, ids = [33, 1, 20], [2, 0, 1]
    x, base = randn((54, 320), 5).to(dtype), randn((54, 192), 6).to(dtype)
    with torch.no_grad():
        got = ad(x.cuda(), AdapterRequests.from_lengths(lengths, ids), base=base.cuda())
    check(got, x, lengths, ids, weights, base, dtype, 320, rank)


def test_tokens_outside_every_request_keep_their_base():
    ad, weights = make(64, 64, 2, 16, torch.float32)
    x, base = randn((50, 64), 1), randn((50, 64), 2)
    x[40:] = float("nan")  # padding behind the last request
    x[:3] = float("inf")   # before the first
    requests = AdapterRequests(torch.tensor([3, 10, 40], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    with torch.no_grad():
        got = ad(x.cuda(), requests, base=base.cuda()).cpu()
        assert torch.equal(got[:3], base[:3]) and torch.equal(got[40:], base[40:])
        check(got[3:40], x[3:40], [7, 30], [0, 1], weights, base[3:40], torch.float32, 64, 16)
        alone = ad(x.cuda(), requests).cpu()
        assert (alone[:3] == 0).all() and (alone[40:] == 0).all()
        # the same for long prompts
        xl, bl = randn((900, 64), 3), randn((900, 64), 4)
        xl[:3], xl[870:] = float("inf"), float("nan")
        long = AdapterRequests(torch.tensor([3, 300, 870], dtype=torch.int32, device="cuda"), torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
        got = ad(xl.cuda(), long, base=bl.cuda()).cpu()
        assert torch.equal(got[:3], bl[:3]) and torch.equal(got[870:], bl[870:])
        check(got[3:870], xl[3:870], [297, 570], [1, 0], weights, bl[3:870], torch.float32, 64, 16)
        # a token's NaN stays its own
        x2 = randn((50, 64), 1)
        x2[20] = float("nan")
        rows = ad(x2.cuda(), requests, base=base.cuda()).cpu().isnan().any(1)
        assert rows.nonzero().flatten().tolist() == [20]
        # ids outside the adapters, offsets beyond the tokens and no request at all: handled, not followed
        wild = AdapterRequests(torch.tensor([0, 10, 70], dtype=torch.int32, device="cuda"), torch.tensor([7, 1], dtype=torch.int32, device="cuda"))
        got = ad(x2.cuda()[:15], wild, base=base.cuda()[:15]).cpu()
        assert torch.equal(got[:10], base[:10])
        check(got[10:], x2[10:15], [5], [1], weights, base[10:15], torch.float32, 64, 16)
        none = AdapterRequests.from_lengths([], [])
        assert torch.equal(ad(x2.cuda(), none, base=base.cuda()).cpu(), base)
        assert ad(torch.empty((0, 64), device="cuda"), none).shape == (0, 64)


def test_loading_replaces_an_adapter():
    ad, _ = make(64, 96, 3, 16, torch.float32)
    down, up = randn((5, 64), 7), randn((96, 5), 8)
    ad.load(1, down.cuda(), up.cuda(), scaling=0.25)
    x = randn((6, 64), 9)
    with torch.no_grad():
        got = ad(x.cuda(), AdapterRequests.from_lengths([6], [1])).cpu().double()
    want = 0.25 * (x.double() @ down.double().t()) @ up.double().t()
    assert torch.linalg.norm(got - want) <= 2e-5 * torch.linalg.norm(want)


def test_shapes_strides_streams_and_graphs():
    ad, weights = make(96, 64, 4, 8, torch.bfloat16)
    wide = randn((2, 12, 130), 1).to(torch.bfloat16).cuda()
    x = wide[:, :, 1:97]  # neither contiguous nor aligned
    requests = AdapterRequests.from_lengths([10, 14], [3, 0])
    base = randn((2, 12, 64), 2).to(torch.bfloat16).cuda()
    with torch.no_grad():
        want = ad(x.contiguous(), requests, base=base)
        assert want.shape == (2, 12, 64)
        assert torch.equal(ad(x, requests, base=base), want)
        assert torch.equal(ad(x, requests, base=base.transpose(0, 1).contiguous().transpose(0, 1)), want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = ad(x, requests, base=base)
        side.synchronize()
        assert torch.equal(got, want)
        # captured: replayed with other tokens, other requests and other adapters
        static_x, static_base = x.contiguous().clone(), base.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ad(static_x, requests, base=static_base)
        graph.replay()
        assert torch.equal(out, want)
        static_x.copy_(x.flip(0))
        requests.offsets.copy_(torch.tensor([0, 1, 20], dtype=torch.int32))
        requests.adapters.copy_(torch.tensor([2, 1], dtype=torch.int32))
        graph.replay()
        other = AdapterRequests.from_lengths([1, 19], [2, 1])
        assert torch.equal(out, ad(static_x, other, base=static_base))


def test_results_do_not_depend_on_neighbours():
    """A request's rows are the same bits whatever else is in the batch at the same place."""
    ad, _ = make(512, 256, 4, 16, torch.bfloat16)
    x, base = randn((64, 512), 1).to(torch.bfloat16).cuda(), randn((64, 256), 2).to(torch.bfloat16).cuda()
    with torch.no_grad():
        a = ad(x, AdapterRequests.from_lengths([8, 24, 32], [0, 1, 2]), base=base)
        b = ad(x, AdapterRequests.from_lengths([8, 24, 32], [3, 1, 0]), base=base)
    assert torch.equal(a[8:32], b[8:32]) and not torch.equal(a[:8], b[:8])


@pytest.mark.parametrize("activation", [None, "gelu"])
@pytest.mark.parametrize("with_residual", [False, True])
def test_beside_the_shared_projection(activation, with_residual):
    np.random.seed(1)
    torch.manual_seed(1)
    lin = BlockSparseLinear(128, 192, density=0.5, activation=activation).eval()
    with torch.no_grad():
        lin.weight.data.normal_(0, 0.1)
        lin.bias.normal_()
    ad, weights = make(128, 192, 3, 16, torch.float32, seed=4)
    lengths, ids = [20, 1, 0, 1, 30], [1, 0, 2, None, 2]
    x, residual = randn((52, 128), 1), randn((52, 192), 2) if with_residual else None
    with torch.no_grad():
        got = lin(x.cuda(), residual=residual.cuda() if with_residual else None,
                  adapters=(ad, AdapterRequests.from_lengths(lengths, ids))).cpu().double()
    base = x.double() @ lin.weight.to_dense().detach().cpu().double().t() + lin.bias.detach().cpu().double()
    if with_residual:
        base = base + residual.double()
    want, _ = reference(x, lengths, ids, weights, base)
    if activation == "gelu":
        want = torch.nn.functional.gelu(want)
    assert torch.linalg.norm(got - want) <= 3e-5 * torch.linalg.norm(want)  # three products of the 1e-5 class
    with pytest.raises(Exception, match="no_grad"):
        lin(x.cuda().requires_grad_(), adapters=(ad, AdapterRequests.from_lengths(lengths, ids)))


def test_offsets_past_32_bits():
    """Element offsets beyond 2^31: the last tokens of a batch of 2^31 / in + some."""
    inner, outer, tokens = 8192, 32, (1 << 31) // 8192 + 40
    ad, weights = make(inner, outer, 2, 16, torch.bfloat16)
    x = torch.zeros((tokens, inner), dtype=torch.bfloat16, device="cuda")
    tail = randn((20, inner), 3).to(torch.bfloat16)
    x[-20:] = tail.cuda()
    with torch.no_grad():
        got = ad(x, AdapterRequests.from_lengths([tokens - 20, 20], [0, 1]))
    assert (got[:-20] == 0).all()
    check(got[-20:], tail, [20], [1], weights, torch.zeros((20, outer), dtype=torch.bfloat16), torch.bfloat16, inner, 16)
