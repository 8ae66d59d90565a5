"""Plain 64-bit forms of the token-layer operators, for the tests."""
import numpy as np

U32 = 2.0 ** -24   # half an ulp of 1 in f32
UBF = 2.0 ** -8    # a bf16 rounding, relative (8 significant bits: 2^-9, and room for a tie)


def philox(counter, key):
    """Philox4x32-10 of counters [n, 4] under key (2,), both of 32-bit words."""
    x = [np.asarray(counter[:, i], np.uint64) for i in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> half) ^ x[1] ^ np.uint64(k0), b & low, (a >> half) ^ x[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) % 2**32, (k1 + 0xBB67AE85) % 2**32
    return np.stack(x, 1).astype(np.uint32)


def dropout_keep(first, n, p, seed, offset):
    """Kept elements [first, first + n), and the factor."""
    threshold = int(np.floor(p * 65536 + 0.5))
    blocks = np.arange(first // 8, (first + n + 7) // 8, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    counter = np.stack([blocks & low, blocks >> np.uint64(32), np.full(blocks.size, offset % 2**32, np.uint64),
                        np.full(blocks.size, offset >> 32, np.uint64)], 1)
    words = philox(counter, (seed % 2**32, seed >> 32))
    lanes = np.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)
    lanes = lanes[first - 8 * int(blocks[0] if blocks.size else 0):][:n]
    return lanes >= threshold, (65536 / (65536 - threshold) if threshold < 65536 else 0.0)


def embedding(table, tokens, scale):
    t = np.asarray(tokens, np.int64).reshape(-1)
    inside = (t >= 0) & (t < table.shape[0])
    rows = np.zeros((t.size, table.shape[1]))
    rows[inside] = scale * table.astype(np.float64)[t[inside]]
    return rows


def embedding_grad(tokens, grad, vocab, scale):
    """The gradient, and the sum of magnitudes and the number of terms behind each row."""
    t = np.asarray(tokens, np.int64).reshape(-1)
    inside = (t >= 0) & (t < vocab)
    out, mag, terms = np.zeros((vocab, grad.shape[1])), np.zeros((vocab, grad.shape[1])), np.zeros(vocab)
    np.add.at(out, t[inside], grad.astype(np.float64)[inside])
    np.add.at(mag, t[inside], np.abs(grad.astype(np.float64))[inside])
    np.add.at(terms, t[inside], 1)
    return scale * out, abs(scale) * mag, terms


def router(logits, k, balance, normalize):
    z = logits.astype(np.float64)
    rows, experts = z.shape
    top = z.max(1) if rows else np.zeros(0)
    broken = np.isnan(z).any(1) | (top == np.inf)
    alive = ~broken & (top > -np.inf)
    p = np.zeros_like(z)
    e = np.exp(z[alive] - top[alive, None])
    p[alive] = e / e.sum(1, keepdims=True)
    p[broken] = np.nan
    index = np.full((rows, k), -1, np.int32)
    gates = np.zeros((rows, k))
    for t in np.nonzero(alive)[0]:
        order = np.argsort(-z[t], kind="stable")[:k]
        order = order[z[t, order] > -np.inf]
        index[t, : order.size] = order
        g = p[t, order]
        gates[t, : order.size] = g / g.sum() if normalize else g
    counts = np.bincount(index[index >= 0], minlength=experts)[:experts]
    live = int(alive.sum())
    mean = p.sum(0) / max(live, 1)
    share = counts / max(counts.sum(), 1)
    return {"p": p, "alive": alive, "experts": index, "gates": gates, "counts": np.append(counts, live), "mean": mean,
            "loss": balance * experts * float((share * mean).sum())}


def router_objective(logits, index, share, live, gate_grad, loss_grad, balance, normalize):
    """The scalar whose gradient the backward pass is, the choices and shares held fixed."""
    z = logits.astype(np.float64)
    alive = z.max(1) > -np.inf
    e = np.where(alive[:, None], np.exp(z - np.where(alive, z.max(1), 0.0)[:, None]), 0.0)
    p = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
    total = loss_grad * balance * z.shape[1] * float((share * p.sum(0) / max(live, 1)).sum())
    for t in range(z.shape[0]):
        picked = index[t][index[t] >= 0]
        g = p[t, picked]
        if normalize and picked.size:
            g = g / g.sum()
        total += float((g * gate_grad[t, : picked.size]).sum())
    return total


def router_grad(logits, r, gate_grad, loss_grad, balance, normalize):
    p, index = np.nan_to_num(r["p"]), r["experts"]
    rows, experts = p.shape
    share = r["counts"][:-1] / max(r["counts"][:-1].sum(), 1)
    h = balance * experts * share / max(r["counts"][-1], 1) * loss_grad
    u = np.zeros_like(p)
    g = np.zeros_like(p)
    for t in range(rows):
        picked = index[t][index[t] >= 0]
        u[t, picked] = gate_grad[t, : picked.size]
        g[t, picked] = r["gates"][t, : picked.size]
    if normalize:
        out = p * (h - (p * h).sum(1, keepdims=True)) + g * (u - (g * u).sum(1, keepdims=True))
    else:
        out = p * (h + u - (p * (h + u)).sum(1, keepdims=True))
    return out


def quantize_rows(x):
    """The 8-bit rows and scales, with the definition's f32 arithmetic."""
    x = np.asarray(x, np.float32)
    rows, cols = x.shape
    top = np.abs(x).max(1) if cols else np.zeros(rows, np.float32)
    bad = ~np.isfinite(x).all(1) if cols else np.zeros(rows, bool)
    some = ~bad & (top >= np.float32(2.0 ** -100))
    q = np.zeros((rows, cols), np.int8)
    with np.errstate(all="ignore"):
        inverse = np.float32(127) * (np.float32(1) / top)
        q[some] = np.rint((x[some] * inverse[some, None]).astype(np.float32)).astype(np.int8)
        scales = np.where(bad, np.float32(np.nan), np.where(some, top * (np.float32(1) / np.float32(127)), np.float32(0)))
    return q, scales.astype(np.float32)


def int8_product(q, scales, w, w_scales, bias):
    """The product, and the magnitude its roundings scale with."""
    acc = q.astype(np.float64) @ w.astype(np.float64).T  # exact: below 2^53
    y = acc * scales.astype(np.float64)[:, None] * w_scales.astype(np.float64)
    size = np.abs(y)
    if bias is not None:
        y = y + bias.astype(np.float64)
    return y, size
