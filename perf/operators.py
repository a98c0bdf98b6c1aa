"""The operators that stand around a block-sparse projection, as cases to be measured.

gated     the gated feed-forward block: h = act(x Wg^T + bg) * (x Wu^T + bu) with both weights in one block-sparse matrix
          whose block-rows alternate (gate, up); inference on bf16 and fp32 tensors, training (forward and gradients) on fp32 ones
dropout   dropout from a counter-based generator (Philox4x32-10) with the residual add behind it, forward and gradient
adapters  low-rank adapters of many requests beside a shared projection's output

`own` false: elementary torch operations in 32 bits.  `own` true: the calls a user makes of pytorch_block_sparse_b200.
"""
import math

import torch

own = False

BF16, FP32 = "bf16", "fp32"
DTYPES = {BF16: torch.bfloat16, FP32: torch.float32}


def listed():
    return [
        # one token of a small model being generated: latency
        dict(name="gated_token", op="gated", train=False, dtype=BF16, tokens=1, inner=1024, hidden=2048, density=0.5, act="silu", bias=False),
        # a step of generation for a small batch, weights far larger than a cache line's worth of work per token
        dict(name="gated_batch", op="gated", train=False, dtype=BF16, tokens=8, inner=4096, hidden=8192, density=0.25, act="silu", bias=True),
        # a ragged prompt through a large layer
        dict(name="gated_prompt", op="gated", train=False, dtype=BF16, tokens=4001, inner=4096, hidden=8192, density=0.25, act="silu", bias=False),
        # a short prompt in fp32, layer sizes that are odd multiples of the block
        dict(name="gated_prompt_fp32", op="gated", train=False, dtype=FP32, tokens=517, inner=1056, hidden=2720, density=0.35, act="gelu", bias=True),
        # a training step of a base-size feed-forward block (8 x 128 tokens less a ragged rest), odd token count
        dict(name="gated_train", op="gated", train=True, dtype=FP32, tokens=1001, inner=768, hidden=2048, density=0.5, act="gelu", bias=True),
        # a training step of a large layer
        dict(name="gated_train_large", op="gated", train=True, dtype=FP32, tokens=8192, inner=4096, hidden=4096, density=0.25, act="silu", bias=True),
        # dropout and residual of a small fine-tuning batch: latency
        dict(name="dropout_small", op="dropout", dtype=FP32, rows=256, cols=768, p=0.1, residual=True),
        # odd row length, no residual, a high rate
        dict(name="dropout_odd", op="dropout", dtype=BF16, rows=4099, cols=1003, p=0.5, residual=False),
        # the hidden states of a large training batch
        dict(name="dropout_large", op="dropout", dtype=BF16, rows=16384, cols=4096, p=0.1, residual=True),
        # one request generating on its adapter
        dict(name="adapters_token", op="adapters", dtype=FP32, tokens=1, requests=1, count=1, rank=8, inner=1024, outer=1024),
        # many requests generating at once, each a single token
        dict(name="adapters_batch", op="adapters", dtype=BF16, tokens=64, requests=64, count=32, rank=16, inner=4096, outer=4096),
        # prompts of ragged lengths, some without an adapter, some empty
        dict(name="adapters_prompts", op="adapters", dtype=BF16, tokens=6001, requests=24, count=8, rank=64, inner=4096, outer=4096),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = max(_flops(c) for c in listed())
    op = rng.choice(["gated", "gated", "dropout", "adapters"])
    if op == "dropout":
        case = dict(op=op, dtype=rng.choice([BF16, FP32]), rows=_log_int(rng, 1, 16384), cols=_log_int(rng, 8, 4096),
                    p=rng.choice([0.05, 0.1, 0.2, 0.3, 0.5]), residual=rng.random() < 0.6)
        if case["dtype"] == FP32:
            case["rows"] = max(1, case["rows"] // 2)
        return case
    if op == "adapters":
        tokens = _log_int(rng, 1, 6000)
        return dict(op=op, dtype=rng.choice([BF16, BF16, FP32]), tokens=tokens, requests=min(_log_int(rng, 1, 64), tokens),
                    count=_log_int(rng, 1, 32), rank=rng.choice([4, 8, 16, 24, 32, 64]), inner=32 * _log_int(rng, 8, 128),
                    outer=32 * _log_int(rng, 8, 128))
    while True:
        train = rng.random() < 0.5
        case = dict(op=op, train=train, dtype=FP32 if train else rng.choice([BF16, BF16, FP32]), tokens=_log_int(rng, 1, 8192), inner=32 * _log_int(rng, 4, 128),
                    hidden=32 * _log_int(rng, 8, 256), density=round(rng.uniform(0.1, 0.6), 2), act=rng.choice(["silu", "gelu"]),
                    bias=rng.random() < 0.5)
        if _flops(case) <= most:
            return case


def _pairs(case):
    """Stored (gate, up) pairs of blocks of a gated layer."""
    return max(1, int(case["density"] * (case["hidden"] // 32) * (case["inner"] // 32)))


def _adapters_in_use(case):
    return min(case["count"], max(1, case["requests"]))


def _flops(case):
    if case["op"] == "gated":
        return (3 if case["train"] else 1) * 2 * case["tokens"] * 2 * _pairs(case) * 1024
    if case["op"] == "dropout":
        return 4 * case["rows"] * case["cols"]
    return 2 * case["tokens"] * case["rank"] * (case["inner"] + case["outer"])


def work(case):
    size = 2 if case["dtype"] == BF16 else 4
    if case["op"] == "gated":
        m, h, f, blocks = case["tokens"], case["inner"], case["hidden"], 2 * _pairs(case)
        moved = m * (h + f) * size + blocks * 4096 + (8 * f if case["bias"] else 0)
        if case["train"]:  # dh read, dx, dW and db written
            moved += m * (h + f) * size + blocks * 4096 + (8 * f if case["bias"] else 0)
    elif case["op"] == "dropout":  # x and the residual read, out written; dout read, dx written
        moved = (5 if case["residual"] else 4) * case["rows"] * case["cols"] * size
    else:
        moved = (case["tokens"] * (case["inner"] + 2 * case["outer"]) + _adapters_in_use(case) * case["rank"] * (case["inner"] + case["outer"])) * size
    return {"bytes": moved, "flops": _flops(case)}


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(to)

    if case["op"] == "gated":
        m, inner, hidden = case["tokens"], case["inner"], case["hidden"]
        rows, cols = hidden // 32, inner // 32
        pick = torch.randperm(rows * cols, device="cuda", generator=gen)[: _pairs(case)]
        mask = torch.zeros(rows * cols, dtype=torch.bool, device="cuda")
        mask[pick] = True
        mask = mask.view(rows, cols).repeat_interleave(2, 0)  # gate and up of a hidden unit read the same inputs
        # weights of a bf16 checkpoint for bf16 tensors, fp32 ones for fp32; the layer keeps them in fp32
        data = randn(2 * _pairs(case) * 32, 32, scale=1.0 / math.sqrt(case["density"] * inner)).float()
        state = dict(case=case, x=randn(m, inner), mask=mask, data=data, bias=randn(2 * hidden, scale=0.1, to=torch.float32) if case["bias"] else None)
        if case["train"]:
            state["dh"] = randn(m, hidden)
        if own:
            from pytorch_block_sparse_b200 import BlockSparseGatedLinear, BlockSparseMatrix

            layer = BlockSparseGatedLinear(
                inner, hidden, bias=case["bias"], activation=case["act"], weight=BlockSparseMatrix((2 * hidden, inner), mask, data),
                precision="bf16" if case["dtype"] == BF16 else None)
            if case["bias"]:
                with torch.no_grad():
                    layer.bias.copy_(state["bias"])
            state["layer"] = layer
            state["x"].requires_grad_(case["train"])
        return state
    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        rng = torch.tensor([seed * 0x9E3779B9 + 12345, seed % 1000 + (1 << 33)], dtype=torch.int64, device="cuda")  # seed and counter
        return dict(case=case, x=randn(*shape), residual=randn(*shape) if case["residual"] else None, dout=randn(*shape), rng=rng)
    tokens, n = case["tokens"], case["requests"]
    # ragged prompts: cuts at random places (equal ones leave an empty request); one token for each while generating
    if n == tokens:
        offsets = torch.arange(n + 1, device="cuda")
    else:
        cuts = torch.randint(0, tokens + 1, (n - 1,), device="cuda", generator=gen).sort().values
        offsets = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), tokens)])
    ids = torch.arange(n, device="cuda") % case["count"]
    if n > 4:
        ids[3] = -1  # a request without an adapter
    state = dict(case=case, x=randn(tokens, case["inner"]), base=randn(tokens, case["outer"]), offsets=offsets.int(), ids=ids.int(),
                 down=randn(case["count"], case["rank"], case["inner"], scale=1.0 / math.sqrt(case["inner"])),
                 up=randn(case["count"], case["outer"], case["rank"], scale=1.0 / math.sqrt(case["rank"])),
                 scaling=torch.rand(case["count"], device="cuda", generator=gen) + 0.5)
    if own:
        from pytorch_block_sparse_b200 import AdapterRequests, LowRankAdapters

        adapters = LowRankAdapters(case["inner"], case["outer"], case["count"], case["rank"], dtype=dtype)
        adapters.load_all(state["down"], state["up"], state["scaling"])
        state["adapters"], state["requests"] = adapters, AdapterRequests(state["offsets"], state["ids"])
    return state


# ------------------------------------------------------------------------------------------------------- plain forms
def _dense(mask, data):
    """The dense matrix of a block-sparse one: slot s, in row-major order of the pattern, holds its block transposed."""
    at = mask.nonzero()
    grid = torch.zeros(mask.shape[0], mask.shape[1], 32, 32, device=data.device, dtype=data.dtype)
    grid[at[:, 0], at[:, 1]] = data.view(-1, 32, 32).transpose(1, 2)
    return grid.permute(0, 2, 1, 3).reshape(mask.shape[0] * 32, mask.shape[1] * 32)


def _act(g, kind):
    if kind == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))


def _act_grad(g, kind):
    if kind == "silu":
        s = 1 / (1 + torch.exp(-g))
        return s * (1 + g * (1 - s))
    return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))


def _gated(state):
    case, mask = state["case"], state["mask"]
    x = state["x"].detach().float()
    weight = _dense(mask, state["data"])
    pre = x @ weight.t()
    if case["bias"]:
        pre = pre + state["bias"]
    g, u = pre.view(x.shape[0], -1, 2, 32).unbind(2)  # block-rows alternate: gate, up
    a = _act(g, case["act"])
    h = (a * u).reshape(x.shape[0], -1)
    if not case["train"]:
        return h.to(state["x"].dtype)
    dh = state["dh"].float().view_as(g)
    dpre = torch.stack([dh * u * _act_grad(g, case["act"]), dh * a], 2).reshape(x.shape[0], -1)
    dx = dpre @ weight
    at = mask.nonzero()
    blocks = (dpre.t() @ x).view(mask.shape[0], 32, mask.shape[1], 32).permute(0, 2, 3, 1)
    dw = blocks[at[:, 0], at[:, 1]].reshape(-1, 32)
    out = [h, dx, dw]
    return out + [dpre.sum(0)] if case["bias"] else out


def _multiply(a, b):
    """High and low 32 bits of the product of 32-bit numbers held in int64 (the product itself wraps, its bits are right)."""
    product = a * b
    return (product >> 32) & 0xFFFFFFFF, product & 0xFFFFFFFF


def _philox(index, rng):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): counter (index, rng[1]), key rng[0]; four 32-bit numbers for each index."""
    low = 0xFFFFFFFF
    c0, c1 = index & low, (index >> 32) & low
    c2, c3 = (rng[1] & low).expand_as(index), ((rng[1] >> 32) & low).expand_as(index)
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    for _ in range(10):
        h0, l0 = _multiply(c0, 0xD2511F53)
        h1, l1 = _multiply(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], -1)


def _keep(count, p, rng):
    """keep[i]: the i-th 16-bit number of the generator's stream (8 for each counter value, the low half of each word first) is
    not below p in units of 2^-16, and the scale of the values kept."""
    words = _philox(torch.arange((count + 7) // 8, device=rng.device), rng)
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:count]
    cut = round(p * 65536)
    return halves >= cut, 65536 / (65536 - cut)


def _dropout(state):
    x, residual = state["x"], state["residual"]
    keep, scale = _keep(x.numel(), state["case"]["p"], state["rng"])
    factor = keep.view_as(x).float() * scale
    out = x.float() * factor
    if residual is not None:
        out = out + residual.float()
    return out.to(x.dtype), (state["dout"].float() * factor).to(x.dtype)


def _adapters(state):
    x, down, up = state["x"].float(), state["down"].float(), state["up"].float()
    count, rank = down.shape[:2]
    # the adapter of each token: of the request whose tokens it is among
    token = torch.arange(x.shape[0], device=x.device, dtype=torch.int32)
    mine = state["ids"].long()[torch.searchsorted(state["offsets"], token, right=True) - 1]
    # every token with every adapter, all but its own struck out
    v = (x @ down.view(count * rank, -1).t()).view(-1, count, rank)
    own_one = mine[:, None] == torch.arange(count, device=x.device)
    v = v * (own_one * state["scaling"])[:, :, None]
    y = state["base"].float() + v.view(-1, count * rank) @ up.permute(0, 2, 1).reshape(count * rank, -1)
    return y.to(state["base"].dtype)


# ----------------------------------------------------------------------------------------------------------- one pass
def _own(state):
    case = state["case"]
    if case["op"] == "gated":
        layer, x = state["layer"], state["x"]
        if not case["train"]:
            with torch.no_grad():
                return layer(x)
        h = layer(x)
        leaves = [x, layer.weight.data] + ([layer.bias] if case["bias"] else [])
        return [h.detach(), *torch.autograd.grad(h, leaves, state["dh"])]
    if case["op"] == "dropout":
        from pytorch_block_sparse_b200 import dropout_residual

        x = state["x"].requires_grad_()
        out = dropout_residual(x, case["p"], state["rng"], residual=state["residual"])
        return out.detach(), torch.autograd.grad(out, x, state["dout"])[0]
    with torch.no_grad():
        return state["adapters"](state["x"], state["requests"], base=state["base"])


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"gated": _gated, "dropout": _dropout, "adapters": _adapters}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------- values in 64 bits
def _exact_gated(state):
    case = state["case"]
    x, mask = state["x"].detach().double(), state["mask"]
    rows, cols = mask.shape
    # dense weights by scattering every stored value to its place: slot s, value (c, r) -> W[32 R + r, 32 C + c]
    r_block, c_block = torch.nonzero(mask, as_tuple=True)
    inner = torch.arange(32, device=x.device)
    at_row = (r_block[:, None, None] * 32 + inner[None, None, :]).expand(-1, 32, 32)
    at_col = (c_block[:, None, None] * 32 + inner[None, :, None]).expand(-1, 32, 32)
    weight = torch.zeros(rows * 32, cols * 32, dtype=torch.float64, device=x.device)
    weight[at_row, at_col] = state["data"].double().view(-1, 32, 32)
    unit = torch.arange(rows * 16, device=x.device)
    gate_rows = unit // 32 * 64 + unit % 32
    wg, wu = weight[gate_rows], weight[gate_rows + 32]
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        b = state["bias"].double()
        g, u = g + b[gate_rows], u + b[gate_rows + 32]
    if case["act"] == "silu":
        sig = torch.sigmoid(g)
        a, slope = g * sig, sig + g * sig * (1 - sig)
    else:
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
        a, slope = g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    h = a * u
    if not case["train"]:
        return h
    dh = state["dh"].double()
    dg, du = dh * u * slope, dh * a
    dx = dg @ wg + du @ wu
    dw = torch.zeros_like(weight)
    dw[gate_rows], dw[gate_rows + 32] = dg.t() @ x, du.t() @ x
    out = [h, dx, dw[at_row, at_col].reshape(-1, 32)]
    if case["bias"]:
        db = torch.zeros(rows * 32, dtype=torch.float64, device=x.device)
        db[gate_rows], db[gate_rows + 32] = dg.sum(0), du.sum(0)
        out.append(db)
    return out


def _exact_dropout(state):
    import numpy as np

    x = state["x"]
    seed, counter = (int(v) for v in state["rng"].cpu())
    groups = np.arange((x.numel() + 7) // 8, dtype=np.uint64)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [groups & low, groups >> half, np.full_like(groups, counter & 0xFFFFFFFF), np.full_like(groups, (counter >> 32) & 0xFFFFFFFF)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2**32, (k[1] + 0xBB67AE85) % 2**32]
    words = np.stack(c, 1).astype(np.uint32)
    drawn = torch.from_numpy(np.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[: x.numel()].astype(np.int32)).to(x.device)
    cut = round(state["case"]["p"] * 2**16)
    kept = torch.where(drawn < cut, 0.0, 1.0).double().view(x.shape) / (1 - cut / 2**16)
    out = x.detach().double() * kept
    if state["residual"] is not None:
        out = out + state["residual"].double()
    return out, state["dout"].double() * kept


def _exact_adapters(state):
    x, y = state["x"].double(), state["base"].double().clone()
    offsets, ids = state["offsets"].tolist(), state["ids"].tolist()
    for first, last, a in zip(offsets[:-1], offsets[1:], ids):
        if a >= 0:
            y[first:last] += float(state["scaling"][a]) * (x[first:last] @ state["down"][a].double().t()) @ state["up"][a].double().t()
    return y


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"gated": _exact_gated, "dropout": _exact_dropout, "adapters": _exact_adapters}[case["op"]](state)
