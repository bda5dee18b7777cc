"""The products of a mixture-of-experts layer and of 8-bit serving, as cases to measure: inputs, the
operators' plain forms, this library's calls, and their values in 64 bits.

Five paths. ``T`` rows of ``x`` are sorted by expert; expert ``e`` owns the rows from
``group_ends[e - 1]`` to ``group_ends[e]``.

``experts``   y[t] = x[t] W[e(t)]                                (inference: one product)
``train``     y, dx[t] = dy[t] W[e(t)]^T, dW[e] = x[e]^T dy[e]   (a training step's three products)
``quantize``  q, s of x [rows, K] with one scale for 128 consecutive values of a row, or of a
              weight [N, K] with one for each 128 x 128 tile: s = amax / 448, q = e4m3(x * (448 / amax))
``scaled``    y = (qa sa) (qb sb)^T with such operands
``scaled`` with experts: the same over rows sorted by expert, with one weight for each
"""

from __future__ import annotations

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0**-100
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One token sent to two of eight experts: two weights of 117 MB are streamed for two rows.
        {"name": "experts decode", "path": "experts", "rows": 2, "experts": 8, "active": 2, "k": 4096, "n": 14336, "type": "bf16", "layout": "kn", "skew": 0.0},
        # A decode batch of 48 tokens with six of 64 small experts each: about five rows an expert.
        {"name": "experts batch", "path": "experts", "rows": 288, "experts": 64, "active": 60, "k": 2048, "n": 1408, "type": "fp16", "layout": "nk", "skew": 1.0},
        # A prefill of 4097 tokens with two of eight experts each.
        {"name": "experts prefill", "path": "experts", "rows": 8194, "experts": 8, "active": 8, "k": 4096, "n": 14336, "type": "bf16", "layout": "kn", "skew": 0.5},
        # Fine-tuning a small layer: ragged groups of tens of rows, one expert without any.
        {"name": "train small", "path": "train", "rows": 421, "experts": 8, "active": 7, "k": 520, "n": 1000, "type": "fp16", "layout": "kn", "skew": 1.0},
        # A pretraining micro-batch: 16384 rows over 32 experts, weights stored as nn.Linear does.
        {"name": "train large", "path": "train", "rows": 16384, "experts": 32, "active": 32, "k": 2048, "n": 2816, "type": "bf16", "layout": "nk", "skew": 0.7},
        # The activations of a decode batch before an 8-bit projection.
        {"name": "quantize rows batch", "path": "quantize", "rows": 31, "k": 4096, "type": "bf16", "tiles": False},
        # The activations of a prefill before the down projection.
        {"name": "quantize rows prefill", "path": "quantize", "rows": 8192, "k": 14336, "type": "bf16", "tiles": False},
        # A projection's weight, once for each checkpoint or after each update.
        {"name": "quantize weight", "path": "quantize", "rows": 18944, "k": 3584, "type": "fp16", "tiles": True},
        # One token through a down projection.
        {"name": "scaled decode", "path": "scaled", "rows": 1, "experts": 0, "active": 0, "k": 18944, "n": 3584, "type": "bf16", "skew": 0.0},
        # A mixed batch of 257 rows through an up projection.
        {"name": "scaled mixed", "path": "scaled", "rows": 257, "experts": 0, "active": 0, "k": 4096, "n": 12800, "type": "fp16", "skew": 0.0},
        # A prefill through an up projection.
        {"name": "scaled prefill", "path": "scaled", "rows": 8192, "experts": 0, "active": 0, "k": 4096, "n": 14336, "type": "bf16", "skew": 0.0},
        # Experts served in 8 bits: 4099 rows over 32 of them.
        {"name": "scaled experts", "path": "scaled", "rows": 4099, "experts": 32, "active": 31, "k": 2048, "n": 2816, "type": "bf16", "skew": 0.7},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def _extent(rng, low, high):
    """A hidden size: a multiple of 8, and one time in six any number."""
    v = _spread(rng, low, high)
    return v if rng.random() < 1 / 6 else (v + 7) // 8 * 8


def draw(rng):
    path = rng.choice(("experts", "train", "quantize", "scaled", "scaled experts"))
    kind = rng.choice(("bf16", "fp16"))
    if path == "quantize":
        tiles = rng.random() < 0.4
        return {"path": path, "rows": _spread(rng, 1, 8192), "k": _extent(rng, 128, 14336), "type": kind, "tiles": tiles}
    k, n = _extent(rng, 256, 4096), _extent(rng, 256, 8192)
    if path == "scaled":
        return {"path": path, "rows": _spread(rng, 1, 8192), "experts": 0, "active": 0, "k": k, "n": n, "type": kind, "skew": 0.0}
    experts = _spread(rng, 2, 64)
    rows = _spread(rng, 1, 8192)
    active = max(1, min(rows, experts, round(experts * (0.3 + rng.random()))))
    n = min(n, max(256, 14336 * 8 // experts))
    case = {"path": path.split()[0], "rows": rows, "experts": experts, "active": active, "k": k, "n": n, "type": kind, "skew": round(rng.random() * 1.5, 2)}
    if path != "scaled experts":
        case["layout"] = rng.choice(("kn", "nk"))
    return case


def _sizes(case, g):
    """Rows of each expert: `active` of the experts have one at least, and the others follow weights that fall off with the expert's rank."""
    experts, active, rows = case["experts"], case["active"], case["rows"]
    order = torch.randperm(experts, generator=g)[:active]
    counts = torch.zeros(experts, dtype=torch.int64)
    counts[order] = 1
    left = rows - active
    if left > 0:
        weights = torch.arange(1, active + 1, dtype=torch.float64) ** -case["skew"]
        picked = torch.multinomial(weights, left, replacement=True, generator=g)
        counts[order] += torch.bincount(picked, minlength=active)
    return counts


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    kind = TYPES[case["type"]]
    rows, k = case["rows"], case["k"]

    def normal(*shape, scale=1.0):
        return torch.empty(shape, device="cuda", dtype=kind).normal_(0.0, scale, generator=g)

    state = {"path": case["path"], "kind": kind}
    if case["path"] == "quantize":
        state["tiles"] = case["tiles"]
        # Activations have rows and channels of very different size.
        x = normal(rows, k, scale=0.02 if case["tiles"] else 1.0)
        state["x"] = x if case["tiles"] else x * torch.exp(normal(rows, 1))
        return state
    n = case["n"]
    if case["experts"]:
        counts = _sizes(case, host)
        ends = torch.cumsum(counts, 0)
        # What a program with its router on the host has in hand; the calls take the ends on the GPU.
        state["bounds"] = [(e, int(end - count), int(end)) for e, (end, count) in enumerate(zip(ends, counts))]
        state["ends"] = ends.to(torch.int32).cuda()
    if case["path"] == "scaled":
        lead = (case["experts"],) if case["experts"] else ()
        a = normal(rows, k) * torch.exp(normal(rows, 1))
        w = normal(*lead, n, k, scale=k**-0.5)
        state["a"], state["sa"] = _quantize_plain(a, False)
        state["b"], state["sb"] = _quantize_plain(w, True)
        return state
    shape = (k, n) if case["layout"] == "kn" else (n, k)
    w = normal(case["experts"], *shape, scale=k**-0.5)
    state["x"] = normal(rows, k)
    state["w"] = w if case["layout"] == "kn" else w.transpose(1, 2)
    if case["path"] == "train":
        state["dy"] = normal(rows, n)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["path"] == "train":
        state["x"].requires_grad_()
        state["w"] = state["w"].detach().requires_grad_()
    return state


def _blocks(k):
    return (k + BLOCK - 1) // BLOCK


def _quantize_plain(x, tiles):
    """q in e4m3 and its scales: one for 128 values of a row, or for 128 x 128 values of a matrix."""
    lead, (rows, k) = x.shape[:-2], x.shape[-2:]
    high = BLOCK if tiles else 1
    padded = torch.nn.functional.pad(x.float(), (0, _blocks(k) * BLOCK - k, 0, -rows % high))
    cells = padded.view(*lead, padded.shape[-2] // high, high, _blocks(k), BLOCK)
    amax = cells.abs().amax(dim=(-3, -1)).clamp(min=AMAX_FLOOR)
    most = torch.full_like(amax, E4M3_MAX)  # a tensor: a quotient with a number is a product with its inverse
    q = (cells * (most / amax)[..., :, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    q = q.view(padded.shape)[..., :rows, :k].to(torch.float8_e4m3fn).contiguous()
    return q, amax / most


def _dequantize(q, s, tiles, kind=torch.float32):
    s = s.to(kind).repeat_interleave(BLOCK, dim=-1)[..., : q.shape[-1]]
    if tiles:
        s = s.repeat_interleave(BLOCK, dim=-2)[..., : q.shape[-2], :]
    return q.to(kind) * s


def _run_own(state):
    from heliostune_b200 import blockscale, grouped

    if state["path"] == "experts":
        return grouped.grouped_matmul(state["x"], state["w"], state["ends"])
    if state["path"] == "train":
        y = grouped.grouped_matmul(state["x"], state["w"], state["ends"])
        dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if state["path"] == "quantize":
        q, s = (blockscale.quantize_tiles if state["tiles"] else blockscale.quantize_rows)(state["x"])
        return {"q": q, "s": s}
    return blockscale.matmul_blockscaled(state["a"], state["sa"], state["b"], state["sb"], state.get("ends"), out_dtype=state["kind"])


def _run_plain(state):
    kind = state["kind"]
    if state["path"] == "quantize":
        q, s = _quantize_plain(state["x"], state["tiles"])
        return {"q": q, "s": s}
    if state["path"] == "scaled":
        a = _dequantize(state["a"], state["sa"], False)
        if "ends" not in state:
            return (a @ _dequantize(state["b"], state["sb"], True).T).to(kind)
        y = torch.zeros(a.shape[0], state["b"].shape[1], device=a.device)
        for e, start, end in state["bounds"]:
            if end > start:
                torch.mm(a[start:end], _dequantize(state["b"][e], state["sb"][e], True).T, out=y[start:end])
        return y.to(kind)
    x, w = state["x"].detach(), state["w"].detach()
    y = torch.zeros(x.shape[0], w.shape[2], device=x.device)
    train = state["path"] == "train"
    if train:
        dy, dx, dw = state["dy"].float(), torch.zeros(x.shape, device=x.device), torch.zeros(w.shape, device=x.device)
    x = x.float()
    for e, start, end in state["bounds"]:
        if end > start:
            weight = w[e].float()
            torch.mm(x[start:end], weight, out=y[start:end])
            if train:
                torch.mm(dy[start:end], weight.T, out=dx[start:end])
                torch.mm(x[start:end].T, dy[start:end], out=dw[e])
    if train:
        return {"y": y.to(kind), "dx": dx.to(kind), "dw": dw.to(kind)}
    return y.to(kind)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    rows, k = case["rows"], case["k"]
    if case["path"] == "quantize":
        scales = (_blocks(rows) if case["tiles"] else rows) * _blocks(k)
        return {"bytes": rows * k * 3 + scales * 4, "flops": 2 * rows * k}
    n, weights = case["n"], case["active"] if case["experts"] else 1
    flops = 2 * rows * k * n
    if case["path"] == "scaled":
        scales = rows * _blocks(k) + weights * _blocks(n) * _blocks(k)
        return {"bytes": rows * k + weights * k * n + 2 * rows * n + 4 * scales, "flops": flops}
    product = rows * k + rows * n
    if case["path"] == "experts":
        return {"bytes": 2 * (product + weights * k * n), "flops": flops}
    # x, dy and the weights read once; y, dx and every expert's gradient written once.
    return {"bytes": 2 * (2 * product + (weights + case["experts"]) * k * n), "flops": 3 * flops}


def _e4m3_64(v):
    """The nearest e4m3 value of each 64-bit number: 3 bits after the leading one, steps of 2^-9 below 2^-6, ties to even."""
    _, exponent = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), exponent.clamp(min=-5) - 4)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    state = _inputs(case, seed)
    if case["path"] == "quantize":
        x = state["x"].double()
        rows, k = x.shape
        high = BLOCK if case["tiles"] else 1
        row = torch.arange(rows, device=x.device) // high
        column = torch.arange(k, device=x.device) // BLOCK
        amax = torch.full((int(row[-1]) + 1, k), AMAX_FLOOR, device=x.device, dtype=torch.float64)
        amax = amax.scatter_reduce(0, row[:, None].expand(rows, k), x.abs(), "amax")
        cells = torch.full((amax.shape[0], _blocks(k)), AMAX_FLOOR, device=x.device, dtype=torch.float64)
        cells = cells.scatter_reduce(1, column[None].expand(amax.shape[0], k), amax, "amax")
        return {"q": _e4m3_64(x * E4M3_MAX / cells[row][:, column]), "s": cells / E4M3_MAX}
    if case["path"] == "scaled":
        a, b = state["a"].double(), state["b"].double()
        column = torch.arange(a.shape[1], device=a.device) // BLOCK
        line = torch.arange(b.shape[-2], device=a.device) // BLOCK
        a = a * state["sa"].double()[:, column]
        if not case["experts"]:
            return a @ (b * state["sb"].double()[line][:, column]).T
        parts = [a[start:end] @ (b[e] * state["sb"][e].double()[line][:, column]).T for e, start, end in state["bounds"]]
        return torch.cat(parts)
    x, w = state["x"].double(), state["w"]
    y = torch.cat([x[start:end] @ w[e].double() for e, start, end in state["bounds"]])
    if case["path"] == "experts":
        return y
    dy = state["dy"].double()
    dx = torch.cat([dy[start:end] @ w[e].double().T for e, start, end in state["bounds"]])
    dw = torch.stack([x[start:end].T @ dy[start:end] for e, start, end in state["bounds"]])
    return {"y": y, "dx": dx, "dw": dw}
