"""What the gated block, dropout and the adapters refuse, without a GPU: the library's entry points by status code before
anything is launched, the Python layer by exceptions."""
import ctypes

import pytest
import torch

from pytorch_block_sparse_b200 import (AdapterRequests, BlockSparseGatedLinear, BlockSparseLinear, BlockSparseMatrix, LowRankAdapters,
                                       dropout_residual, native, next_rng)
from pytorch_block_sparse_b200.dropout import rate_units
from pytorch_block_sparse_b200.gated_linear import interleave_rows, split_rows

OK, INVALID, UNSUPPORTED, TOO_LARGE = 0, 1, 2, 4
fake, odd, null = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1004), None


def test_gated_entry_points():
    lib = native.load()
    act = lib.bsmm_gated_act
    assert act(fake, 4, 33, fake, 0, null) == INVALID          # hidden not a multiple of 32
    assert act(fake, -1, 32, fake, 0, null) == INVALID
    assert act(null, 4, 32, fake, 0, null) == INVALID
    assert act(odd, 4, 32, fake, 0, null) == INVALID           # misaligned
    assert act(fake, 4, 32, fake, native.GATED_PRE_BF16, null) == UNSUPPORTED  # bf16 pre only with bf16 tensors
    assert act(fake, 4, 32, fake, 0x100, null) == UNSUPPORTED
    assert act(fake, 1 << 32, 32, fake, 0, null) == TOO_LARGE
    assert act(null, 0, 32, null, 0, null) == OK               # nothing to do
    assert lib.bsmm_gated_act_workspace_bytes(-1, 32) == -1
    assert lib.bsmm_gated_act_workspace_bytes(257, 64) == 2 * 128 * 4
    back = lib.bsmm_gated_act_backward
    assert back(fake, fake, 4, 32, fake, fake, null, 0, null) == INVALID  # a bias gradient without its workspace
    assert back(fake, null, 4, 32, fake, null, null, 0, null) == INVALID
    assert back(fake, fake, 4, 48, fake, null, null, 0, null) == INVALID
    small = lib.bsmm_gated_small
    assert small(fake, 4, 40, fake, fake, 1, fake, 32, null, fake, 0, null) == INVALID
    assert small(fake, 4, 32, null, fake, 1, fake, 32, null, fake, 0, null) == INVALID
    assert small(fake, 4, 32, fake, odd, 1, fake, 32, null, fake, 0, null) == INVALID
    assert small(fake, 1 << 20, 32, fake, fake, 1, fake, 32, null, fake, 0, null) == TOO_LARGE
    assert small(fake, 4, 32, fake, fake, 1, fake, 32, null, fake, native.GATED_PRE_BF16 | native.GATED_IO_BF16, null) == UNSUPPORTED
    assert small(null, 0, 32, fake, null, 0, null, 32, null, fake, 0, null) == OK


def test_gated_kernel_entry_points():
    lib = native.load()
    both = native.GATED_IO_BF16 | native.GATED_PRE_BF16
    assert lib.bsmm_gated_plan_bytes(64, 100, 4) == -1
    assert lib.bsmm_gated_plan_bytes(32, 32, 1) > 0
    assert lib.bsmm_gated_images_bytes(3) == 3 * 4096 and lib.bsmm_gated_images_bytes(-1) == -1
    assert lib.bsmm_build_gated_plan(null, fake, 32, 32, 1, fake, null) == INVALID
    assert lib.bsmm_build_gated_plan(fake, fake, 32, 32, 1, odd, null) == INVALID
    assert lib.bsmm_build_gated_plan(fake, fake, 32, native.GATED_MAX_K + 32, 1, fake, null) == TOO_LARGE
    assert lib.bsmm_gated_pack(fake, fake, 32, 32, 1, odd, null) == INVALID
    run = lib.bsmm_gated_forward
    assert run(fake, 4, 0, fake, fake, 1, 32, null, fake, null, both, null) == INVALID
    assert run(fake, 4, 32, fake, fake, 1, 32, null, fake, null, 0, null) == UNSUPPORTED  # bf16 tensors only
    assert run(fake, 4, 32, fake, null, 1, 32, null, fake, null, both, null) == INVALID
    assert run(fake, 4, 32, fake, odd, 1, 32, null, fake, null, both, null) == INVALID
    assert run(fake, 4, native.GATED_MAX_K + 32, fake, fake, 1, 32, null, fake, null, both, null) == TOO_LARGE
    assert run(null, 0, 32, null, null, 0, 32, null, null, null, both, null) == OK
    assert lib.bsmm_build_gated_f32_plan(fake, fake, fake, fake, 32, 48, 1, fake, null) == INVALID
    passes = lib.bsmm_gated_pass_forward
    x3 = native.PREC_TF32X3
    assert passes(fake, 4, 32, fake, fake, 1, fake, null, null, null, 32, null, fake, fake, null, 1 << 30, null) == UNSUPPORTED
    assert passes(fake, 4, 48, fake, fake, 1, fake, null, null, null, 32, null, fake, fake, null, 0, null) == INVALID
    assert passes(fake, 4, 32, fake, fake, 1, fake, null, null, null, 32, null, null, fake, null, 0, null) == INVALID  # no pre
    assert passes(fake, 4, 32, fake, fake, 1, fake, null, null, fake, 32, null, null, fake, null, x3, null) == INVALID  # no workspace
    assert passes(fake, 4, 32, fake, fake, 1, fake, null, null, fake, 32, odd, null, fake, fake, x3, null) == INVALID
    assert passes(fake, 4, native.GATED_MAX_K + 32, fake, fake, 1, fake, null, null, fake, 32, null, null, fake, fake, x3, null) == TOO_LARGE
    assert lib.bsmm_gated_forward_workspace_bytes(-1, 32, 32, 1, x3) == -1
    assert lib.bsmm_gated_forward_workspace_bytes(4, 32, 32, 1, 0) == 0
    back = lib.bsmm_gated_pass_backward
    args = [fake, fake, fake, 64, 32, fake, fake, fake, fake, 1, fake, fake, fake, fake, fake, 32, fake, null, fake, null, null, fake]
    assert back(*args[:-1], null, native.PREC_TF32X3, null) == INVALID                     # no workspace
    assert back(*args, native.PREC_TF32X3 | (native.GATED_X_BF16 << 16), null) == UNSUPPORTED
    assert back(*args, native.PREC_TF32X3 | (native.GATED_IO_BF16 << 16), null) == UNSUPPORTED  # bf16 tensors: BF16 precision
    args[4] = 48
    assert back(*args, native.PREC_TF32X3, null) == INVALID


def test_dropout_entry_points():
    lib = native.load()
    drop = lib.bsmm_dropout
    assert drop(fake, null, fake, 8, 65536, fake, 0, null) == INVALID  # everything dropped
    assert drop(fake, null, fake, -1, 0, fake, 0, null) == INVALID
    assert drop(fake, null, fake, 8, 0, null, 0, null) == INVALID
    assert drop(fake, odd, fake, 8, 0, fake, 0, null) == INVALID
    assert drop(fake, null, fake, 8, 0, fake, 2, null) == UNSUPPORTED
    assert drop(null, null, null, 0, 0, null, 0, null) == OK
    assert lib.bsmm_rng_next(null, fake, null) == INVALID
    assert lib.bsmm_rng_next(odd, fake, null) == INVALID


def test_adapter_entry_points():
    lib = native.load()

    def run(tokens=4, inner=32, outer=32, requests=1, count=1, rank=16, x=fake, offsets=fake, down=fake, base=null, out=fake, ws=fake, flags=0):
        return lib.bsmm_adapters(x, tokens, inner, outer, offsets, fake, requests, count, rank, down, fake, fake, base, out, ws, flags, null)

    for bad in (dict(tokens=-1), dict(inner=40), dict(outer=40), dict(inner=0), dict(rank=8), dict(rank=24), dict(rank=320), dict(rank=0),
                dict(x=null), dict(offsets=null), dict(down=null), dict(out=null), dict(ws=null), dict(base=odd), dict(x=odd)):
        assert run(**bad) == INVALID, bad
    assert run(flags=native.ADAPTERS_OUT_BF16) == UNSUPPORTED  # a bf16 output of fp32 adapters
    assert run(flags=4) == UNSUPPORTED
    assert run(tokens=1 << 32) == TOO_LARGE
    assert run(tokens=0) == OK and run(outer=0) == OK
    assert lib.bsmm_adapters_workspace_bytes(10, 64, 16) >= 640
    assert lib.bsmm_adapters_workspace_bytes(10, 65, 16) == -1


def test_dropout_arguments():
    assert rate_units(0.0) == 0 and rate_units(0.5) == 32768
    for p in (-0.1, 1.0, 1.5, 1 - 1e-9, float("nan")):
        with pytest.raises(ValueError, match="rate"):
            rate_units(p)
    x = torch.zeros(4)
    rng = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(native.NativeError, match="CUDA"):
        dropout_residual(x, 0.1, rng)
    with pytest.raises(ValueError, match="state"):
        next_rng(torch.zeros(3, dtype=torch.int64))
    with pytest.raises(native.NativeError, match="CUDA"):
        next_rng(rng)
    with pytest.raises(ValueError, match="rate"):
        BlockSparseLinear(32, 32, dropout=1.0)
    with pytest.raises(Exception, match="activation"):
        BlockSparseLinear(32, 32, activation="gelu", dropout=0.1)


def test_adapter_arguments():
    i32 = dict(dtype=torch.int32)
    for offsets, ids in ((torch.zeros(2, dtype=torch.int64), torch.zeros(1, **i32)), (torch.zeros(2, **i32), torch.zeros(2, **i32)),
                         (torch.zeros((2, 1), **i32), torch.zeros(1, **i32)), (torch.zeros(4, **i32)[::2], torch.zeros(1, **i32))):
        with pytest.raises(ValueError):
            AdapterRequests(offsets, ids)
    with pytest.raises(ValueError, match="lengths"):
        AdapterRequests.from_lengths([1, 2], [0], device="cpu")
    with pytest.raises(ValueError, match="negative"):
        AdapterRequests.from_lengths([1, -2], [0, 0], device="cpu")
    requests = AdapterRequests.from_lengths([3, 0, 2], [1, None, -1], device="cpu")
    assert requests.offsets.tolist() == [0, 3, 3, 5] and requests.adapters.tolist() == [1, -1, -1]
    for bad in (dict(in_features=40), dict(out_features=0), dict(count=0), dict(rank=0), dict(rank=257), dict(dtype=torch.float16)):
        with pytest.raises(Exception, match="LowRankAdapters"):
            LowRankAdapters(**{**dict(in_features=32, out_features=64, count=2, rank=8, device="cpu"), **bad})
    ad = LowRankAdapters(32, 64, 2, 8, device="cpu")
    assert tuple(ad.down.shape) == (2, 16, 32) and tuple(ad.up.shape) == (2, 64, 16)
    assert [LowRankAdapters(32, 64, 1, r, device="cpu").down.shape[1] for r in (1, 16, 17, 33, 65, 200)] == [16, 16, 32, 64, 128, 256]
    ad.load(1, torch.ones(3, 32), torch.ones(64, 3), 2.0)
    assert ad.down[1, :3].eq(1).all() and ad.down[1, 3:].eq(0).all() and ad.scaling.tolist() == [0.0, 2.0]
    with pytest.raises(IndexError):
        ad.load(2, torch.ones(3, 32), torch.ones(64, 3))
    for down, up in ((torch.ones(9, 32), torch.ones(64, 9)), (torch.ones(3, 31), torch.ones(64, 3)), (torch.ones(3, 32), torch.ones(64, 4))):
        with pytest.raises(ValueError, match="fit"):
            ad.load(0, down, up)
    with pytest.raises(ValueError, match="fit"):
        ad.load_all(torch.ones(3, 4, 32), torch.ones(3, 64, 4), torch.ones(3))
    x = torch.zeros(5, 32)
    with pytest.raises(native.NativeError, match="no_grad"):
        ad(x.clone().requires_grad_(), requests)
    with torch.no_grad():
        with pytest.raises(Exception, match="features"):
            ad(torch.zeros(5, 64), requests)
        with pytest.raises(ValueError, match="bfloat16"):
            ad(x.bfloat16(), requests)
        with pytest.raises(ValueError, match="base"):
            ad(x, requests, base=torch.zeros(5, 32))
        with pytest.raises(ValueError, match="type"):
            ad(x, requests, base=torch.zeros(5, 64, dtype=torch.bfloat16))
        with pytest.raises(ValueError, match="type"):
            ad(x, requests, dtype=torch.bfloat16)
        with pytest.raises(ValueError, match="inplace"):
            ad(x, requests, inplace=True)
        with pytest.raises(ValueError, match="inplace"):
            ad(x, requests, base=torch.zeros(64, 5).t(), inplace=True)
        with pytest.raises(native.NativeError, match="CUDA"):
            ad(x, requests)


def cpu_layer(**kwargs):
    mask = torch.zeros((4, 3), dtype=torch.bool)
    mask[0, 1] = mask[1, 1] = True
    return BlockSparseGatedLinear(96, 64, weight=BlockSparseMatrix((128, 96), mask, torch.zeros(64, 32)), **kwargs)


def test_gated_arguments():
    for bad in (dict(in_features=40), dict(hidden_features=0), dict(activation="relu"), dict(density=1.5)):
        with pytest.raises(Exception, match="BlockSparseGatedLinear"):
            BlockSparseGatedLinear(**{**dict(in_features=32, hidden_features=32), **bad})
    with pytest.raises(ValueError, match="precision"):
        cpu_layer(precision="fp64")
    mask = torch.ones((4, 3), dtype=torch.bool)
    with pytest.raises(Exception, match="shape"):
        BlockSparseGatedLinear(96, 32, weight=BlockSparseMatrix((128, 96), mask, torch.zeros(12 * 32, 32)))
    with pytest.raises(Exception, match="32x32"):
        BlockSparseGatedLinear(128, 64, weight=BlockSparseMatrix((128, 128), torch.ones((2, 2), dtype=torch.bool), torch.zeros(256, 64), (64, 64)))
    layer = cpu_layer()
    with pytest.raises(Exception, match="at least 2"):
        layer(torch.zeros(96))
    with pytest.raises(Exception, match="Invalid matrices sizes"):
        layer(torch.zeros(4, 64))
    with pytest.raises(ValueError, match="float16"):
        layer(torch.zeros(4, 96, dtype=torch.float16))
    with pytest.raises(Exception, match="CUDA"):
        layer(torch.zeros(4, 96))
    with pytest.raises(Exception, match="one shape"):
        BlockSparseGatedLinear.from_linears(torch.nn.Linear(32, 64), torch.nn.Linear(32, 32))
    gate, up = layer.to_dense()
    assert tuple(gate.shape) == tuple(up.shape) == (64, 96)
    both = torch.arange(128 * 3).view(128, 3)
    assert torch.equal(interleave_rows(*split_rows(both)), both)
    assert torch.equal(split_rows(both)[0][:32], both[:32]) and torch.equal(split_rows(both)[1][:32], both[32:64])
