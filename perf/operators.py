"""The operators of a learned LayerStack router, as a user's program calls them.

A LayerStack net evaluates a position with one of S small dense stacks.  A
router that learns which one is a token model over the feature rows the net
already reads: every feature of a position is looked up in a table (`lookup`),
dropped out in training (`dropout`), multiplied with the router's weights -- in
8-bit integers when it evaluates (`int8`) -- and the resulting logits choose a
stack, with a balance loss that keeps all stacks in use (`router`).

`run` computes one pass of one operator: in plain torch operations in 32 bits
where `own` is false, by the framework's kernels where it is true.  Rows are
positions or tokens, columns features; a feature row is padded with -1.
"""
import math

import numpy as np
import torch

own = False

F32, BF16 = "f32", "bf16"
_TYPES = {F32: torch.float32, BF16: torch.bfloat16}
_BYTES = {F32: 4, BF16: 2}

HALFKA_ROWS = 73305   # HalfKA_hm2 feature rows
HALFKP_ROWS = 125388  # HalfKP feature rows
PIECE_ROWS = 1629     # piece rows of one king block


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # serving one position: its 40 features are looked up, latency only
        {"name": "lookup one position", "op": "lookup", "vocab": HALFKA_ROWS, "tokens": 40, "width": 256, "type": F32},
        # a training batch of 16384 positions with 40 features each
        {"name": "lookup batch 16384", "op": "lookup", "vocab": HALFKA_ROWS, "tokens": 16384 * 40, "width": 256,
         "type": BF16},
        # the table's gradient for a ragged last batch and an odd width: piece rows, every row hit often
        {"name": "lookup grad ragged", "op": "lookup_grad", "vocab": PIECE_ROWS, "tokens": 1801 * 38, "width": 257,
         "type": F32},
        # the table's gradient for a training batch of 32768 positions
        {"name": "lookup grad batch 32768", "op": "lookup_grad", "vocab": HALFKA_ROWS, "tokens": 32768 * 40,
         "width": 256, "type": F32},
        # dropout on a few positions' tokens (fine-tuning on single games)
        {"name": "dropout small", "op": "dropout", "rows": 40, "cols": 256, "pad": 0, "p": 0.1, "type": F32,
         "residual": False},
        # dropout's gradient for a ragged batch of an odd width inside a wider matrix
        {"name": "dropout grad ragged", "op": "dropout_grad", "rows": 20011, "cols": 769, "pad": 31, "p": 0.25,
         "type": F32, "residual": False},
        # dropout of a training batch's tokens with the residual added
        {"name": "dropout batch 16384", "op": "dropout", "rows": 16384 * 40, "cols": 256, "pad": 0, "p": 0.1,
         "type": BF16, "residual": True},
        # choosing among the 9 stacks of a k3k3 net for one small engine batch
        {"name": "router serve k3k3", "op": "router", "rows": 64, "experts": 9, "k": 1, "pad": 0, "normalize": False,
         "type": F32, "train": False},
        # training the router of an 81-stack k9k9 net at the global batch of 262144 positions
        {"name": "router train k9k9", "op": "router", "rows": 262144, "experts": 81, "k": 2, "pad": 0,
         "normalize": True, "type": F32, "train": True},
        # one position through a dense layer: bound by reading the 8-bit weights
        {"name": "int8 one position", "op": "int8", "rows": 1, "inner": 1536, "outer": 2048, "pad": 0, "bias": True,
         "type": F32, "out": F32},
        # a ragged search batch through a layer of odd sizes
        {"name": "int8 ragged batch", "op": "int8", "rows": 301, "inner": 1537, "outer": 1001, "pad": 3, "bias": True,
         "type": BF16, "out": F32},
        # a validation batch of 16384 positions through a wide dense layer
        {"name": "int8 batch 16384", "op": "int8", "rows": 16384, "inner": 4096, "outer": 4096, "pad": 0,
         "bias": False, "type": BF16, "out": BF16},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ranges: sizes spread over their logarithm, odd ones among them."""
    op = rng.choice(["lookup", "lookup_grad", "dropout", "dropout_grad", "router", "int8"])
    kind = rng.choice([F32, BF16])
    while True:
        if op in ("lookup", "lookup_grad"):
            case = {"op": op, "vocab": _log(rng, 64, HALFKP_ROWS), "tokens": _log(rng, 1, 32768 * 40),
                    "width": rng.choice([_log(rng, 8, 2048), 8 * _log(rng, 1, 256)]), "type": kind}
            cost, most = case["tokens"] * case["width"], 16384 * 40 * 256 * (1 if op == "lookup" else 2)
            cost += case["vocab"] * case["width"] if op == "lookup_grad" else 0
        elif op in ("dropout", "dropout_grad"):
            case = {"op": op, "rows": _log(rng, 1, 16384 * 40), "cols": rng.choice([_log(rng, 1, 4096), 8 * _log(rng, 1, 512)]),
                    "pad": rng.choice([0, 0, 8, rng.randrange(1, 40)]), "p": round(rng.uniform(0.0, 0.6), 3), "type": kind,
                    "residual": op == "dropout" and rng.random() < 0.5}
            cost, most = case["rows"] * (case["cols"] + case["pad"]), 16384 * 40 * 256
        elif op == "router":
            experts = _log(rng, 2, 512)
            case = {"op": op, "rows": _log(rng, 1, 262144), "experts": experts, "k": rng.randint(1, min(8, experts)),
                    "pad": rng.choice([0, 0, rng.randrange(1, 9)]), "normalize": rng.random() < 0.5, "type": kind,
                    "train": rng.random() < 0.6}
            cost, most = case["rows"] * (experts + case["pad"]), 262144 * 81
        else:
            case = {"op": op, "rows": _log(rng, 1, 16384), "inner": rng.choice([_log(rng, 16, 8192), 16 * _log(rng, 1, 512)]),
                    "outer": rng.choice([_log(rng, 1, 8192), 16 * _log(rng, 1, 512)]), "pad": rng.choice([0, 0, rng.randrange(1, 20)]),
                    "bias": rng.random() < 0.5, "type": kind, "out": rng.choice([F32, BF16])}
            cost, most = case["rows"] * case["inner"] * case["outer"], 16384 * 4096 * 4096
        if cost <= most:
            return case


def work(case):
    """Bytes that have to be read and written, and operations, of one pass."""
    op, s = case["op"], _BYTES[case["type"]]
    if op in ("lookup", "lookup_grad"):
        n, d, v = case["tokens"], case["width"], case["vocab"]
        if op == "lookup":  # the rows that are named (at most the table), the tokens, the output
            return {"bytes": min(n, v) * d * s + 4 * n + n * d * s, "flops": n * d}
        return {"bytes": n * d * s + 4 * n + v * d * 4, "flops": n * d + v * d}
    if op in ("dropout", "dropout_grad"):
        e = case["rows"] * case["cols"]
        return {"bytes": e * s * (3 if case["residual"] else 2), "flops": 2 * e}
    if op == "router":
        t, e, k = case["rows"], case["experts"], case["k"]
        forward = t * e * s + 8 * t * k + 8 * e
        return {"bytes": forward + (t * e * s + 4 * t * k if case["train"] else 0),
                "flops": t * e * (12 if case["train"] else 6)}
    m, k, n = case["rows"], case["inner"], case["outer"]
    return {"bytes": m * k * s + n * k + 4 * n + (4 * n if case["bias"] else 0) + m * n * _BYTES[case["out"]],
            "flops": 2 * m * k * n}


# --------------------------------------------------------------------------- inputs
def _normal(g, rows, cols, kind, pad=0, scale=1.0):
    """rows x cols values; with `pad`, a slice of a wider matrix."""
    wide = torch.randn(rows, cols + pad, generator=g, device="cuda")
    return (wide * scale).to(_TYPES[kind])[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op in ("lookup", "lookup_grad"):
        n, v, d = case["tokens"], case["vocab"], case["width"]
        # a few feature rows are named by many positions, most by few; one in 32 slots is padding
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        tokens = (u.pow(3) * v).to(torch.int64).clamp_(max=v - 1) * 7919 % v
        tokens = torch.where(torch.rand(n, generator=g, device="cuda") < 1 / 32, -1, tokens).to(torch.int32)
        state = {"case": case, "tokens": tokens, "scale": 1.0 / math.sqrt(40.0)}
        if op == "lookup":
            state["table"] = _normal(g, v, d, case["type"], scale=0.05)
        else:
            state["grad"] = _normal(g, n, d, case["type"], scale=1e-3)
        return state
    if op in ("dropout", "dropout_grad"):
        state = {"case": case, "x": _normal(g, case["rows"], case["cols"], case["type"], case["pad"]),
                 "seed": seed * 0x9E3779B97F4A7C15 % 2**64, "offset": seed % 1000 + 2**32}
        if case["residual"]:
            state["residual"] = _normal(g, case["rows"], case["cols"], case["type"])
        return state
    if op == "router":
        t, e, k = case["rows"], case["experts"], case["k"]
        wide = torch.randn(t, e + case["pad"], generator=g, device="cuda") * 1.5
        wide += torch.randn(e + case["pad"], generator=g, device="cuda")  # some stacks are liked more
        # stacks that a position may not take, and padding rows that may take none
        wide.masked_fill_(torch.rand(t, e + case["pad"], generator=g, device="cuda") < 0.05, -math.inf)
        wide.masked_fill_((torch.rand(t, 1, generator=g, device="cuda") < 0.01), -math.inf)
        state = {"case": case, "logits": wide.to(_TYPES[case["type"]])[:, :e], "balance": 0.01}
        if case["train"]:
            state["gate_grad"] = torch.randn(t, k, generator=g, device="cuda") / t
            state["loss_grad"] = torch.ones(1, device="cuda")
        return state
    m, k, n = case["rows"], case["inner"], case["outer"]
    channel = torch.exp(0.5 * torch.randn(k + case["pad"], generator=g, device="cuda"))  # some inputs are larger
    x = (torch.randn(m, k + case["pad"], generator=g, device="cuda") * channel).to(_TYPES[case["type"]])[:, :k]
    state = {"case": case, "x": x,
             "weight": (torch.randn(n, k, generator=g, device="cuda") * 40).round().clamp(-127, 127).to(torch.int8),
             "weight_scale": 0.002 * (0.5 + torch.rand(n, generator=g, device="cuda"))}
    if case["bias"]:
        state["bias"] = torch.randn(n, generator=g, device="cuda")
    return state


# --------------------------------------------------------------------------- plain forms
_MASK32 = 0xFFFFFFFF
_PHILOX_MUL = (0xD2511F53, 0xCD9E8D57)
_PHILOX_WEYL = (0x9E3779B9, 0xBB67AE85)


def _plain_keep(elements, p, seed, offset):
    """Which elements dropout keeps, and the factor of those: element i is lane i % 8 (16 bits each) of the
    Philox4x32-10 block with counter (i / 8, offset) and key `seed`, kept where the lane is not below p * 2^16."""
    threshold = int(math.floor(p * 65536 + 0.5))
    block = torch.arange((elements + 7) // 8, device="cuda", dtype=torch.int64)
    c0, c1 = block & _MASK32, (block >> 32) & _MASK32
    c2, c3 = torch.full_like(block, offset & _MASK32), torch.full_like(block, (offset >> 32) & _MASK32)
    k0, k1 = seed & _MASK32, (seed >> 32) & _MASK32
    for _ in range(10):
        a, b = c0 * _PHILOX_MUL[0], c2 * _PHILOX_MUL[1]  # the low 64 bits: a product that wraps keeps them
        c0, c1, c2, c3 = ((b >> 32) & _MASK32) ^ c1 ^ k0, b & _MASK32, ((a >> 32) & _MASK32) ^ c3 ^ k1, a & _MASK32
        k0, k1 = (k0 + _PHILOX_WEYL[0]) & _MASK32, (k1 + _PHILOX_WEYL[1]) & _MASK32
    words = torch.stack([c0, c1, c2, c3], 1)
    lanes = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:elements]
    return lanes >= threshold, 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0


def _plain_dropout(state, x, residual):
    case = state["case"]
    keep, factor = _plain_keep(x.numel(), case["p"], state["seed"], state["offset"])
    y = torch.where(keep.view(x.shape), x.float() * factor, 0.0)
    return (y if residual is None else y + residual.float()).to(x.dtype)


def _plain_router(state):
    case, z = state["case"], state["logits"].float()
    e, k = case["experts"], case["k"]
    top = z.amax(1, keepdim=True)
    live = (top > -math.inf) & (top < math.inf)
    weight = torch.exp(z - torch.where(live, top, 0.0))
    p = torch.where(live, weight / weight.sum(1, keepdim=True), torch.where(top == -math.inf, 0.0, math.nan))
    value, order = torch.sort(z, dim=1, descending=True, stable=True)
    chosen = live & (value[:, :k] > -math.inf)
    experts = torch.where(chosen, order[:, :k], -1)
    slot = experts.clamp(min=0)
    gates = torch.where(chosen, p.gather(1, slot), 0.0)
    if case["normalize"]:
        gates = torch.where(chosen, gates / gates.sum(1, keepdim=True), 0.0)
    counts = torch.zeros(e + 1, dtype=torch.int32, device=z.device)
    counts.index_add_(0, torch.where(chosen, experts, e).reshape(-1), torch.ones_like(experts, dtype=torch.int32).reshape(-1))
    counts[e] = live.sum()
    rows = counts[e].clamp(min=1).float()
    share = counts[:e].float() / counts[:e].sum().clamp(min=1).float()
    mean = p.sum(0) / rows
    loss = state["balance"] * e * (share * mean).sum().reshape(1)
    out = {"experts": experts.to(torch.int32), "gates": gates, "counts": counts, "mean": mean, "loss": loss}
    if case["train"]:
        pull = state["balance"] * e * share / rows * state["loss_grad"]
        given = torch.where(chosen, state["gate_grad"], 0.0)
        spread = torch.zeros_like(p)
        if case["normalize"]:
            spread.scatter_add_(1, slot, gates * (given - (gates * given).sum(1, keepdim=True)))
            grad = spread + p * (pull - (p * pull).sum(1, keepdim=True))
        else:
            a = spread.scatter_add_(1, slot, given) + pull
            grad = p * (a - (p * a).sum(1, keepdim=True))
        out["grad"] = grad.to(state["logits"].dtype)
    return out


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "lookup":
        tokens, table = state["tokens"].long(), state["table"]
        inside = (tokens >= 0) & (tokens < case["vocab"])
        rows = table[torch.where(inside, tokens, 0)].float() * state["scale"]
        return torch.where(inside[:, None], rows, 0.0).to(table.dtype)
    if op == "lookup_grad":
        tokens = state["tokens"].long()
        inside = (tokens >= 0) & (tokens < case["vocab"])
        sums = torch.zeros(case["vocab"], case["width"], device=tokens.device)
        sums.index_add_(0, torch.where(inside, tokens, 0), torch.where(inside[:, None], state["grad"].float(), 0.0))
        return sums * state["scale"]
    if op in ("dropout", "dropout_grad"):
        return _plain_dropout(state, state["x"], state.get("residual"))
    if op == "router":
        return _plain_router(state)
    x = state["x"].float()
    top = x.abs().amax(1, keepdim=True)
    top = torch.where(top < math.inf, top, math.nan)
    some = ~(top < 2.0**-100)
    q = torch.where(some, torch.round(x * (127.0 / top)), 0.0)
    scale = torch.where(some, top / 127.0, 0.0)
    y = (q @ state["weight"].float().T) * (scale * state["weight_scale"])
    if case["bias"]:
        y = y + state["bias"]
    return y.to(_TYPES[case["out"]])


# --------------------------------------------------------------------------- the framework's calls
_contexts = {}


def _context():
    """The program's context on torch's current stream."""
    import bulletou_b200 as bo

    stream = torch.cuda.current_stream()
    ctx = _contexts.get(stream.cuda_stream)
    if ctx is None:
        ctx = _contexts[stream.cuda_stream] = bo.Context(stream.device_index, stream=stream.cuda_stream)
    return bo, ctx


def _framework(state):
    bo, ctx = _context()
    case = state["case"]
    op = case["op"]
    if op == "lookup":
        table = state["table"]
        out = torch.empty(case["tokens"], case["width"], dtype=table.dtype, device="cuda")
        bo.embedding_forward(ctx, table, state["tokens"], out, scale=state["scale"])
        return out
    if op == "lookup_grad":
        out = torch.empty(case["vocab"], case["width"], device="cuda")
        bo.embedding_backward(ctx, state["tokens"], state["grad"], out, scale=state["scale"])
        return out
    if op in ("dropout", "dropout_grad"):
        x = state["x"]
        out = torch.empty(case["rows"], case["cols"], dtype=x.dtype, device="cuda")
        if op == "dropout":
            bo.dropout(ctx, x, out, probability=case["p"], seed=state["seed"], offset=state["offset"],
                       residual=state.get("residual"))
        else:
            bo.dropout_backward(ctx, x, out, probability=case["p"], seed=state["seed"], offset=state["offset"])
        return out
    if op == "router":
        t, e, k = case["rows"], case["experts"], case["k"]
        logits = state["logits"]
        experts = torch.empty(t, k, dtype=torch.int32, device="cuda")
        gates = torch.empty(t, k, device="cuda")
        counts = torch.empty(e + 1, dtype=torch.int32, device="cuda")
        mean = torch.empty(e, device="cuda")
        loss = torch.empty(1, device="cuda")
        bo.router_forward(ctx, logits, experts, gates, counts, mean, loss, balance=state["balance"],
                          normalize_gates=case["normalize"])
        out = {"experts": experts, "gates": gates, "counts": counts, "mean": mean, "loss": loss}
        if case["train"]:
            out["grad"] = torch.empty(t, e, dtype=logits.dtype, device="cuda")
            bo.router_backward(ctx, logits, experts, counts, state["gate_grad"], state["loss_grad"], out["grad"],
                               balance=state["balance"], normalize_gates=case["normalize"])
        return out
    out = torch.empty(case["rows"], case["outer"], dtype=_TYPES[case["out"]], device="cuda")
    bo.int8_linear(ctx, state["x"], state["weight"], state["weight_scale"], out, bias=state.get("bias"))
    return out


def run(state):
    return _framework(state) if own else _plain(state)


# --------------------------------------------------------------------------- 64 bits
def _philox_lanes(blocks, seed, offset):
    """16-bit lanes [blocks, 8] of Philox4x32-10, in unsigned 64-bit products."""
    low = np.uint64(_MASK32)
    half = np.uint64(32)
    i = np.arange(blocks, dtype=np.uint64)
    x = [i & low, i >> half, np.full(blocks, offset & _MASK32, np.uint64), np.full(blocks, offset >> 32, np.uint64)]
    key = [seed & _MASK32, seed >> 32]
    for _ in range(10):
        first, second = np.uint64(_PHILOX_MUL[0]) * x[0], np.uint64(_PHILOX_MUL[1]) * x[2]
        x = [(second >> half) ^ x[1] ^ np.uint64(key[0]), second & low, (first >> half) ^ x[3] ^ np.uint64(key[1]), first & low]
        key = [(k + w) % 2**32 for k, w in zip(key, _PHILOX_WEYL)]
    lanes = np.empty((blocks, 8), np.uint16)
    for j in range(4):
        lanes[:, 2 * j] = (x[j] & np.uint64(0xFFFF)).astype(np.uint16)
        lanes[:, 2 * j + 1] = (x[j] >> np.uint64(16)).astype(np.uint16)
    return lanes.reshape(-1)


def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits."""
    state = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        table = torch.cat([state["table"].double() * state["scale"], torch.zeros(1, case["width"], device="cuda", dtype=torch.float64)])
        return table[state["tokens"].long()]  # -1 names the row of zeros
    if op == "lookup_grad":
        # each row's gradients are neighbours once sorted: differences of running sums, in blocks of columns
        order = torch.sort(state["tokens"].long(), stable=True)
        edges = torch.searchsorted(order.values, torch.arange(case["vocab"] + 1, device="cuda"))
        out = torch.empty(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
        for c in range(0, case["width"], 64):
            part = state["grad"][:, c:c + 64].double()[order.indices]
            run_sum = torch.cat([torch.zeros_like(part[:1]), part.cumsum(0)])
            out[:, c:c + 64] = (run_sum[edges[1:]] - run_sum[edges[:-1]]) * state["scale"]
        return out
    if op in ("dropout", "dropout_grad"):
        n = case["rows"] * case["cols"]
        dropped = round(math.floor(case["p"] * 65536 + 0.5))
        lanes = torch.from_numpy(_philox_lanes((n + 7) // 8, state["seed"], state["offset"])[:n].astype(np.int32)).cuda()
        y = state["x"].double() * (65536 / (65536 - dropped)) if dropped < 65536 else torch.zeros_like(state["x"].double())
        y = y.masked_fill((lanes < dropped).view(case["rows"], case["cols"]), 0.0)
        return y + state["residual"].double() if case["residual"] else y
    if op == "router":
        z = state["logits"].double()
        none = (z == -math.inf).all(1)
        p = torch.softmax(z.masked_fill(none[:, None], 0.0), 1).masked_fill(none[:, None], 0.0)
        # the k largest, lowest index first among equals: push the chosen ones down one by one
        left, picked = z.clone(), []
        for _ in range(case["k"]):
            best = left.amax(1, keepdim=True)
            first = ((left == best).long().cumsum(1) == 0).sum(1, keepdim=True).clamp(max=case["experts"] - 1)
            picked.append(torch.where(best > -math.inf, first, -1))
            left.scatter_(1, first, -math.inf)
        index = torch.cat(picked, 1)
        hot = torch.zeros(case["rows"], case["experts"] + 1, dtype=torch.float64, device="cuda")
        hot.scatter_(1, torch.where(index < 0, case["experts"], index), 1.0)
        hot = hot[:, :-1]
        gate = p * hot
        if case["normalize"]:
            gate = torch.where(hot > 0, gate / gate.sum(1, keepdim=True), 0.0)
        gates = torch.where(index < 0, 0.0, gate.gather(1, index.clamp(min=0)))
        alive = max(1, int((~none).sum()))
        share = hot.sum(0) / max(1.0, float(hot.sum()))
        mean = p.sum(0) / alive
        balance = state["balance"] * case["experts"]
        out = {"experts": None, "gates": gates, "counts": None, "mean": mean, "loss": balance * (share @ mean).reshape(1)}
        if case["train"]:
            upstream = torch.zeros_like(hot).scatter_add_(1, index.clamp(min=0), torch.where(index < 0, 0.0, state["gate_grad"].double()))
            pull = balance * share / alive * float(state["loss_grad"])
            if case["normalize"]:
                out["grad"] = gate * (upstream - (gate * upstream).sum(1, keepdim=True)) + p * (pull - p @ pull[:, None])
            else:
                out["grad"] = p * (upstream + pull - (p * (upstream + pull)).sum(1, keepdim=True))
        return out
    x = state["x"].double()
    top = x.abs().max(1, keepdim=True).values
    levels = torch.round(x / top * 127) if x.numel() else x
    levels = torch.where(top > 0, levels, 0.0)
    y = levels @ state["weight"].double().T * (top / 127) * state["weight_scale"].double()
    return y + state["bias"].double() if case["bias"] else y
