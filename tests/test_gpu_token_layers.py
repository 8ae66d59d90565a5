"""GPU: the token-layer operators (lookup and its gradient, dropout, router,
8-bit product) against plain forms in 64 bits, at the sizes, types, strides and
masks where they can go wrong, and their refusals.

Tolerances: u = 2^-24.  One f32 rounding is u relative; a sum of n terms in any
order is off by at most n u times the sum of magnitudes; a result in bf16 adds
one rounding of 2^-8 relative.
"""
import numpy as np
import pytest

import bulletou_b200 as bo
from tests.token_layer_cases import (U32, UBF, dropout_keep, embedding, embedding_grad, int8_product, quantize_rows,
                                     router, router_grad, router_objective)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16 = "f32", "bf16"


@pytest.fixture(scope="module")
def tctx():
    c = bo.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def kind(t):
    return torch.float32 if t == F32 else torch.bfloat16


def device(a, t=F32, pad=0, shift=0):
    """`a` on the GPU in type t: a slice of a matrix `pad` columns wider that starts `shift` elements into its memory."""
    a = np.atleast_2d(np.asarray(a))
    rows, cols = a.shape
    dt = {np.dtype(np.int32): torch.int32, np.dtype(np.int8): torch.int8}.get(a.dtype, kind(t))
    memory = torch.full((shift + rows * (cols + pad) + pad + 1,), 77, device="cuda", dtype=dt)
    view = torch.as_strided(memory, (rows, cols), (max(cols + pad, 1), 1), shift)
    view.copy_(torch.from_numpy(np.ascontiguousarray(a)).to("cuda").to(dt))
    return view


def host(t):
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def rounding(t):
    return UBF if t == BF16 else 0.0


# --------------------------------------------------------------------------- lookup
LOOKUPS = [  # vocab, tokens, width, pad, shift
    (1, 1, 1, 0, 0), (5, 1, 8, 0, 0), (7, 40, 256, 0, 0), (100, 33, 257, 0, 0), (100, 33, 24, 8, 0), (64, 129, 31, 1, 1),
    (300, 70, 64, 0, 1), (300, 70, 64, 3, 0), (1629, 513, 1536, 0, 0), (9, 0, 16, 0, 0), (9, 5, 0, 0, 0), (0, 6, 16, 0, 0),
]


@pytest.mark.parametrize("vocab,n,width,pad,shift", LOOKUPS)
@pytest.mark.parametrize("t_in,t_out", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)])
def test_lookup(tctx, vocab, n, width, pad, shift, t_in, t_out):
    rng = np.random.default_rng(vocab * 1000 + n)
    table = device(rng.standard_normal((vocab, width)), t_in, pad, shift)
    tokens = rng.integers(-2, vocab + 2, n).astype(np.int32)
    out = device(np.full((n, width), 9.0), t_out, pad, shift)
    bo.embedding_forward(tctx, table, device(tokens), out, scale=0.37)
    want = embedding(host(table), tokens, float(np.float32(0.37)))
    assert (np.abs(host(out) - want) <= (2 * U32 + rounding(t_out)) * np.abs(want)).all()
    inside = (tokens >= 0) & (tokens < vocab)
    assert (host(out)[~inside] == 0).all()


def test_lookup_of_strided_token_matrix(tctx):
    rng = np.random.default_rng(5)
    table, tokens = rng.standard_normal((50, 16)), rng.integers(-1, 50, (13, 7)).astype(np.int32)
    out = device(np.zeros((91, 16)))
    bo.embedding_forward(tctx, device(table), device(tokens, pad=5), out, scale=2.0)
    assert np.array_equal(host(out), embedding(host(device(table)), tokens, 2.0))
    grad = rng.standard_normal((91, 16))
    got = device(np.ones((50, 16)))
    bo.embedding_backward(tctx, device(tokens, pad=5), device(grad), got, scale=2.0)
    want, mag, terms = embedding_grad(tokens, host(device(grad)), 50, 2.0)
    assert (np.abs(host(got) - want) <= (terms[:, None] + 2) * U32 * mag).all()


def test_lookup_of_infinities_and_nan(tctx):
    """What a row holds comes through; a padded token never reads one."""
    table = np.array([[np.inf, -np.inf, np.nan, 1.0], [2.0, 3.0, 4.0, 5.0]], np.float32)
    out = device(np.zeros((3, 4)))
    bo.embedding_forward(tctx, device(table), device(np.array([0, -1, 1], np.int32)), out, scale=0.5)
    got = host(out)
    assert got[0, 0] == np.inf and got[0, 1] == -np.inf and np.isnan(got[0, 2]) and got[0, 3] == 0.5
    assert (got[1] == 0).all() and np.array_equal(got[2], [1.0, 1.5, 2.0, 2.5])


def test_lookup_beyond_32_bit_offsets(tctx):
    stride = 2**30 + 8  # row 2 starts past 2^31 elements
    memory = torch.zeros(2 * stride + 64, device="cuda", dtype=torch.bfloat16)
    table = torch.as_strided(memory, (3, 64), (stride, 1))
    table.copy_(torch.arange(192, device="cuda").view(3, 64))
    out = torch.empty(4, 64, device="cuda", dtype=torch.bfloat16)
    bo.embedding_forward(tctx, table, torch.tensor([2, 0, -1, 1], dtype=torch.int32, device="cuda"), out)
    assert torch.equal(out[0], table[2]) and torch.equal(out[1], table[0]) and torch.equal(out[3], table[1])
    assert not out[2].any()


GRADS = [  # vocab, tokens, width, pad, shift
    (1, 1, 1, 0, 0), (3, 4000, 5, 0, 0), (40, 33, 257, 0, 0), (1000, 50, 24, 8, 0), (64, 129, 31, 1, 1), (2, 9001, 64, 0, 0),
    (513, 20001, 16, 0, 1), (70000, 300, 8, 0, 0), (1629, 5000, 136, 0, 0), (11, 0, 16, 0, 0), (11, 5, 0, 0, 0),
    (300, 2048, 32, 4, 0), (300, 2049, 1030, 0, 0), (1, 70000, 12, 0, 0),
]


@pytest.mark.parametrize("vocab,n,width,pad,shift", GRADS)
@pytest.mark.parametrize("t_in,t_out", [(F32, F32), (BF16, F32), (BF16, BF16), (F32, BF16)])
def test_lookup_gradient(tctx, vocab, n, width, pad, shift, t_in, t_out):
    rng = np.random.default_rng(vocab + 7 * n)
    tokens = (vocab * rng.random(n) ** 3).astype(np.int32)
    tokens[rng.random(n) < 0.1] = -1
    tokens[rng.random(n) < 0.02] = vocab
    grad = device(rng.standard_normal((n, width)), t_in, pad, shift)
    got = device(np.full((vocab, width), 9.0), t_out, pad, shift)
    bo.embedding_backward(tctx, device(tokens), grad, got, scale=-1.7)
    want, mag, terms = embedding_grad(tokens, host(grad), vocab, float(np.float32(-1.7)))
    bound = (terms[:, None] + 2) * U32 * mag + rounding(t_out) * np.abs(want)
    assert (np.abs(host(got) - want) <= bound).all()
    again = device(np.full((vocab, width), 3.0), t_out, pad, shift)
    bo.embedding_backward(tctx, device(tokens), grad, again, scale=-1.7)
    assert torch.equal(got, again)


def test_lookup_gradient_against_differences(tctx):
    """The lookup is linear, so a step of one in a table value moves the loss by exactly its gradient."""
    rng = np.random.default_rng(8)
    tokens = rng.integers(-1, 6, 30).astype(np.int32)
    table, up = rng.standard_normal((6, 4)), rng.standard_normal((30, 4)).astype(np.float32)
    got = device(np.zeros((6, 4)))
    bo.embedding_backward(tctx, device(tokens), device(up), got, scale=0.5)
    base = (embedding(table, tokens, 0.5) * up).sum()
    for v in range(6):
        for c in range(4):
            moved = table.copy()
            moved[v, c] += 1.0
            diff = (embedding(moved, tokens, 0.5) * up).sum() - base
            assert abs(host(got)[v, c] - diff) <= 40 * U32 * np.abs(up).sum()


def test_lookup_gradient_of_padded_tokens_is_not_read(tctx):
    """NaN and infinities in the gradients of tokens outside the table reach no row."""
    rng = np.random.default_rng(9)
    for n in (40, 5000):
        tokens = rng.integers(0, 30, n).astype(np.int32)
        outside = rng.random(n) < 0.3
        tokens[outside] = rng.choice([-1, 30, 2**31 - 1, -2**31], outside.sum())
        grad = rng.standard_normal((n, 24)).astype(np.float32)
        grad[outside] = np.where(rng.random((outside.sum(), 24)) < 0.5, np.nan, np.inf)
        got = device(np.full((30, 24), 5.0))
        bo.embedding_backward(tctx, device(tokens), device(grad), got)
        want, mag, terms = embedding_grad(tokens, grad, 30, 1.0)
        assert (np.abs(host(got) - want) <= (terms[:, None] + 2) * U32 * mag).all()


@pytest.mark.parametrize("n", [1, 31, 4097, 100003])
def test_lookup_gradient_of_one_token(tctx, n):
    """Every entry in one row: the longest sum, far from the other rows' sizes."""
    got = device(np.full((1000, 8), 5.0))
    bo.embedding_backward(tctx, device(np.full(n, 777, np.int32)), device(np.ones((n, 8))), got)
    want = np.zeros((1000, 8))
    want[777] = n  # sums of ones are exact below 2^24
    assert np.array_equal(host(got), want)


# --------------------------------------------------------------------------- dropout
DROPS = [(1, 1, 0, 0), (1, 7, 0, 0), (3, 8, 0, 0), (5, 9, 0, 0), (17, 256, 0, 0), (17, 256, 8, 0), (17, 256, 3, 0), (9, 264, 0, 1),
         (33, 129, 31, 0), (1, 100001, 0, 0), (4000, 3, 1, 2), (0, 5, 0, 0), (5, 0, 0, 0)]


@pytest.mark.parametrize("rows,cols,pad,shift", DROPS)
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("p,residual", [(0.1, False), (0.5, True), (0.0, True), (1.0, False)])
def test_dropout(tctx, rows, cols, pad, shift, t, p, residual):
    rng = np.random.default_rng(rows * 31 + cols)
    x = device(rng.standard_normal((rows, cols)), t, pad, shift)
    r = device(rng.standard_normal((rows, cols)), t, 2 * pad) if residual else None
    out = device(np.full((rows, cols), 9.0), t, pad, shift)
    seed, offset = 0xFEDCBA9876543210, 2**33 + 5
    bo.dropout(tctx, x, out, probability=p, seed=seed, offset=offset, residual=r)
    keep, factor = dropout_keep(0, rows * cols, p, seed, offset)
    keep = keep.reshape(rows, cols)
    scaled = np.where(keep, host(x) * factor, 0.0)
    want = scaled + (host(r) if residual else 0.0)
    got = host(out)
    assert (np.abs(got - want) <= 3 * U32 * (np.abs(scaled) + np.abs(want)) + rounding(t) * np.abs(want)).all()
    if not residual:
        assert (got[~keep] == 0).all()


def test_dropout_mask_does_not_depend_on_layout_or_type(tctx):
    shape = (37, 41)
    masks = []
    for t, pad, shift in [(F32, 0, 0), (F32, 7, 0), (BF16, 0, 0), (BF16, 7, 3)]:
        out = device(np.zeros(shape), t, pad, shift)
        bo.dropout(tctx, device(np.ones(shape), t), out, probability=0.3, seed=3, offset=9)
        masks.append(host(out) != 0)
    assert all(np.array_equal(masks[0], m) for m in masks[1:])
    assert 0.2 < 1 - masks[0].mean() < 0.4
    other = device(np.zeros(shape))
    bo.dropout(tctx, device(np.ones(shape)), other, probability=0.3, seed=3, offset=10)
    assert not np.array_equal(host(other) != 0, masks[0])


def test_dropped_elements_are_zero_whatever_they_hold(tctx):
    x = np.full((8, 16), np.nan, np.float32)
    x[::2] = np.inf
    out = device(np.ones((8, 16)))
    bo.dropout(tctx, device(x), out, probability=0.5, seed=1)
    keep, _ = dropout_keep(0, 128, 0.5, 1, 0)
    got = host(out)
    assert (got[~keep.reshape(8, 16)] == 0).all() and not np.isfinite(got[keep.reshape(8, 16)]).any()


@pytest.mark.parametrize("cols,pad", [(64, 0), (63, 2)])
def test_dropout_in_place_and_backward(tctx, cols, pad):
    rng = np.random.default_rng(2)
    a = rng.standard_normal((11, cols))
    x, apart = device(a, pad=pad), device(np.zeros((11, cols)))
    bo.dropout_backward(tctx, x, apart, probability=0.4, seed=17, offset=4)
    bo.dropout(tctx, x, x, probability=0.4, seed=17, offset=4)
    assert torch.equal(x, apart)
    # dropout is linear in x: its differences are its gradient
    keep, factor = dropout_keep(0, 11 * cols, 0.4, 17, 4)
    ones = device(np.zeros((11, cols)))
    bo.dropout_backward(tctx, device(np.ones((11, cols))), ones, probability=0.4, seed=17, offset=4)
    assert np.array_equal(host(ones), np.where(keep.reshape(11, cols), np.float32(factor), 0.0))


def test_dropout_beyond_32_bit_elements(tctx):
    rows, cols = 2**20 + 3, 4096  # the last rows are past 2^32 elements
    x = torch.ones(rows, cols, device="cuda", dtype=torch.bfloat16)
    bo.dropout(tctx, x, x, probability=0.25, seed=5, offset=6)
    for row in (0, 2**20 - 1, 2**20, rows - 1):
        keep, factor = dropout_keep(row * cols, cols, 0.25, 5, 6)
        want = torch.where(torch.from_numpy(keep).cuda(), torch.tensor(factor, device="cuda").bfloat16(), 0.0)
        assert torch.equal(x[row].float(), want.float())


# --------------------------------------------------------------------------- router
def logits_of(rng, rows, experts, masked=True):
    z = rng.standard_normal((rows, experts)) * 2
    if masked and rows:
        z[rng.random((rows, experts)) < 0.2] = -np.inf
        z[rng.random(rows) < 0.1] = -np.inf
    return z


def run_router(ctx, z, k, balance, normalize, pad=0):
    rows, experts = z.shape
    out = {"experts": device(np.full((rows, k), 9, np.int32), pad=pad), "gates": device(np.full((rows, k), 9.0), pad=pad),
           "counts": device(np.full(experts + 1, 9, np.int32)), "mean": device(np.full(experts, 9.0)), "loss": device([9.0])}
    bo.router_forward(ctx, z, out["experts"], out["gates"], out["counts"], out["mean"], out["loss"], balance=balance,
                      normalize_gates=normalize)
    return out


ROUTERS = [(1, 1, 1), (1, 9, 1), (64, 9, 1), (65, 9, 2), (33, 2, 2), (301, 81, 1), (300, 81, 3), (7, 512, 8), (40, 511, 4),
           (2000, 33, 2), (5000, 16, 1), (3, 64, 8), (129, 4, 4), (257, 3, 1), (0, 9, 1)]


def router_tolerance(z, experts):
    """Relative error of a probability: the rounded difference to the largest logit enters the exponential, whose own
    error and the quotient's are a few u, and the sum's at most experts u."""
    finite = np.abs(z[np.isfinite(z)])
    return (2 * (finite.max() if finite.size else 0.0) + experts + 8) * U32


@pytest.mark.parametrize("rows,experts,k", ROUTERS)
@pytest.mark.parametrize("t,pad,normalize", [(F32, 0, False), (F32, 5, True), (BF16, 0, True), (BF16, 3, False)])
def test_router(tctx, rows, experts, k, t, pad, normalize):
    rng = np.random.default_rng(rows * 7 + experts)
    z = device(logits_of(rng, rows, experts), t, pad)
    out = run_router(tctx, z, k, 0.02, normalize, pad)
    want = router(host(z), k, 0.02, normalize)
    assert np.array_equal(host(out["experts"]), want["experts"])
    assert np.array_equal(host(out["counts"])[0], want["counts"])
    rel = router_tolerance(host(z), experts)
    assert (np.abs(host(out["gates"]) - want["gates"]) <= (2 * rel + 9 * U32) * want["gates"]).all()
    many = rel + (rows + 2) * U32
    assert (np.abs(host(out["mean"])[0] - want["mean"]) <= many * want["mean"]).all()
    assert abs(host(out["loss"])[0, 0] - want["loss"]) <= (many + (experts + 4) * U32) * want["loss"]
    # gradient against the formula
    gg = rng.standard_normal((rows, k)).astype(np.float32)
    got = device(np.full((rows, experts), 9.0), t, pad)
    bo.router_backward(tctx, z, out["experts"], out["counts"], device(gg, pad=pad), device([1.5]), got, balance=0.02,
                       normalize_gates=normalize)
    grad = router_grad(host(z), want, gg, 1.5, 0.02, normalize)
    # each term is a product of a few rounded factors with differences of numbers up to max |u| + max h
    size = (np.abs(gg).max(initial=0.0) + 0.02 * experts * 1.5) * 2
    p = np.nan_to_num(want["p"])
    g = np.zeros_like(p)
    for i in range(rows):
        picked = want["experts"][i][want["experts"][i] >= 0]
        g[i, picked] = want["gates"][i, : picked.size]
    bound = (4 * rel + (experts + 16) * U32) * size * (p + g) + rounding(t) * np.abs(grad)
    assert (np.abs(host(got) - grad) <= bound).all()
    again = run_router(tctx, z, k, 0.02, normalize, pad)
    for name in out:
        assert torch.equal(out[name], again[name])


@pytest.mark.parametrize("counts", [[500, 500], [12800, 12754], [3, 4, 3, 4, 3], [2**31 - 1, 2**31 - 2], [7] * 128])
def test_router_balance_gradient_of_experts_nearly_in_balance(tctx, counts):
    # what all experts' pulls share cancels: the error is measured by how far they differ
    rng = np.random.default_rng(len(counts))
    experts = len(counts)
    z = rng.uniform(-3, 3, (301, experts)).astype(np.float32).astype(np.float64)
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    pull = 0.5 * np.float32(0.9) / 301 * ((experts * np.array(counts, np.int64) - sum(counts)) / sum(counts))
    want = p * (pull - (p * pull).sum(1, keepdims=True))
    got = device(np.full((301, experts), 9.0))
    bo.router_backward(tctx, device(z), device(np.zeros((301, 1), np.int32)), device(np.array([counts + [301]], np.int32)), None,
                       device([np.float32(0.9)]), got, balance=0.5)
    # a probability: the rounding of its exponent (6 log2 e) and of its operations and the sum's; then the pull's and the dot's
    bound = (2 * 6 * 1.4427 + 64 + experts) * U32 * p * np.abs(pull).max() + 1e-45
    assert (np.abs(host(got) - want) <= bound).all()


@pytest.mark.parametrize("normalize", [False, True])
def test_router_gradient_formula_against_differences(tctx, normalize):
    rng = np.random.default_rng(4)
    z = logits_of(rng, 6, 5).astype(np.float32).astype(np.float64)
    r = router(z, 2, 0.3, normalize)
    gg = rng.standard_normal((6, 2)).astype(np.float32)
    share, live = r["counts"][:-1] / r["counts"][:-1].sum(), int(r["counts"][-1])
    want = router_grad(z, r, gg, 0.7, 0.3, normalize)
    zd = device(z)
    out = run_router(tctx, zd, 2, 0.3, normalize)
    got = device(np.zeros((6, 5)))
    bo.router_backward(tctx, zd, out["experts"], out["counts"], device(gg), device([np.float32(0.7)]), got, balance=0.3,
                       normalize_gates=normalize)
    h = 1e-5
    for t in range(6):
        for e in range(5):
            if not np.isfinite(z[t, e]):
                assert want[t, e] == 0 and host(got)[t, e] == 0
                continue
            up, down = z.copy(), z.copy()
            up[t, e] += h
            down[t, e] -= h
            f = [router_objective(v, r["experts"], share, live, gg, 0.7, 0.3, normalize) for v in (up, down)]
            diff = (f[0] - f[1]) / (2 * h)
            assert abs(diff - want[t, e]) <= 1e-8  # h^2 of the third derivative (~1) and the cancellation, 1e-16 / h
            assert abs(host(got)[t, e] - diff) <= 1e-8 + 100 * U32 * (np.abs(gg).max() + 1)


def test_router_ties_take_the_lowest_index(tctx):
    z = np.zeros((3, 40))
    z[1, 7:] = 1.0
    z[2] = -np.finfo(np.float32).max  # the type's lowest value is a logit like any other
    out = run_router(tctx, device(z), 3, 1.0, False)
    assert np.array_equal(host(out["experts"]), [[0, 1, 2], [7, 8, 9], [0, 1, 2]])
    assert np.allclose(host(out["gates"])[2], 1 / 40, rtol=50 * U32)
    assert host(out["counts"])[0, -1] == 3


def test_router_of_masked_and_broken_rows(tctx):
    inf, nan = np.inf, np.nan
    z = np.array([[-inf, -inf, -inf], [1.0, -inf, -inf], [-inf, 0.0, 0.0]])
    out = run_router(tctx, device(z), 2, 1.0, True)
    assert np.array_equal(host(out["experts"]), [[-1, -1], [0, -1], [1, 2]])
    assert np.array_equal(host(out["gates"]), [[0, 0], [1, 0], [0.5, 0.5]])
    assert np.array_equal(host(out["counts"])[0], [1, 1, 1, 2])
    assert np.allclose(host(out["mean"])[0], [0.5, 0.25, 0.25])
    got = device(np.full((3, 3), 9.0))
    bo.router_backward(tctx, device(z), out["experts"], out["counts"], device(np.ones((3, 2))), device([1.0]), got,
                       balance=1.0, normalize_gates=True)
    assert (host(got)[0] == 0).all() and (host(got)[1] == 0).all() and np.isfinite(host(got)).all()
    # nothing alive at all: no loss, no gradient
    out = run_router(tctx, device(np.full((4, 3), -inf)), 1, 1.0, False)
    assert (host(out["experts"]) == -1).all() and (host(out["counts"]) == 0).all()
    assert (host(out["mean"]) == 0).all() and host(out["loss"])[0, 0] == 0
    # NaN and +inf choose nothing and show in the loss; the other rows keep their choices
    z = np.array([[0.0, nan, 1.0], [inf, 0.0, 0.0], [3.0, 2.0, 1.0]])
    out = run_router(tctx, device(z), 1, 1.0, False)
    assert np.array_equal(host(out["experts"])[:, 0], [-1, -1, 0])
    assert np.array_equal(host(out["counts"])[0], [1, 0, 0, 1])
    assert np.isnan(host(out["mean"])).all() and np.isnan(host(out["loss"])).all()
    bo.router_backward(tctx, device(z), out["experts"], out["counts"], None, device([1.0]), got, balance=1.0)
    assert np.isnan(host(got)[:2]).all() and np.isfinite(host(got)[2]).all()


def test_router_gradient_in_place_and_without_parts(tctx):
    rng = np.random.default_rng(12)
    z = device(logits_of(rng, 50, 20))
    out = run_router(tctx, z, 2, 0.5, False)
    gg = device(rng.standard_normal((50, 2)))
    parts = []
    for g, l in ((gg, None), (None, device([2.0])), (gg, device([2.0])), (None, None)):
        d = device(np.zeros((50, 20)))
        bo.router_backward(tctx, z, out["experts"], out["counts"], g, l, d, balance=0.5)
        parts.append(host(d))
    assert np.abs(parts[0] + parts[1] - parts[2]).max() <= 32 * U32 * (np.abs(host(gg)).max() + 20)
    assert (parts[3] == 0).all()
    bo.router_backward(tctx, z, out["experts"], out["counts"], gg, device([2.0]), z, balance=0.5)
    assert np.array_equal(host(z), parts[2])


@pytest.mark.parametrize("experts", [2, 9, 81, 300])
def test_router_single_normalised_gate_is_one_and_adds_nothing(tctx, experts):
    """softmax over one choice: the gate is 1, and however large its gradient, the logits' is the balance loss's alone."""
    rng = np.random.default_rng(experts)
    z = device(rng.standard_normal((70, experts)))
    out = run_router(tctx, z, 1, 0.1, True)
    assert (host(out["gates"]) == 1).all()
    got, alone = device(np.ones((70, experts))), device(np.ones((70, experts)))
    bo.router_backward(tctx, z, out["experts"], out["counts"], device(np.full((70, 1), 1e6)), device([1.0]), got, balance=0.1,
                       normalize_gates=True)
    bo.router_backward(tctx, z, out["experts"], out["counts"], None, device([1.0]), alone, balance=0.1, normalize_gates=True)
    # the chosen logit goes through its own product: one rounding of the difference apart
    assert np.abs(host(got) - host(alone)).max() <= 4 * U32 * 0.1 * experts / 70


def test_router_gradient_skips_foreign_experts(tctx):
    """Expert indexes outside the range (a caller's own padding) take no gradient and read nothing."""
    z = device(np.zeros((2, 4)))
    got = device(np.ones((2, 4)))
    counts = device(np.array([1, 1, 0, 0, 2], np.int32))
    bo.router_backward(tctx, z, device(np.array([[-5], [1000]], np.int32)), counts, device(np.ones((2, 1))), None, got,
                       balance=1.0)
    assert (host(got) == 0).all()


# --------------------------------------------------------------------------- 8-bit product
INT8 = [  # rows, inner, outer
    (1, 1, 1), (1, 16, 8), (1, 1536, 2048), (2, 1000, 9), (3, 333, 77), (8, 128, 130), (9, 4096, 33), (16, 64, 257), (17, 100, 16),
    (64, 256, 128), (65, 257, 129), (128, 2560, 9), (129, 512, 300), (300, 1537, 1001), (513, 96, 520), (1025, 144, 257),
    (2, 0, 5), (9, 0, 5), (0, 8, 5), (4, 8, 0), (5, 8192, 3), (33, 20001, 7), (2000, 96, 1300), (4700, 200, 1100), (300, 260, 20000), (130, 200, 7000), (5, 5000, 70),
]


def int8_bound(size, want, t_out):
    """The scales' product, its product with the sum, the sum's conversion and the bias: four roundings."""
    return 4 * U32 * (size + np.abs(want)) + rounding(t_out) * np.abs(want)


@pytest.mark.parametrize("rows,inner,outer", INT8)
@pytest.mark.parametrize("t_in,t_out,bias,pad,shift", [(F32, F32, True, 0, 0), (BF16, BF16, False, 0, 0), (BF16, F32, True, 5, 1),
                                                       (F32, BF16, False, 16, 0)])
def test_int8(tctx, rows, inner, outer, t_in, t_out, bias, pad, shift):
    rng = np.random.default_rng(rows * 100 + inner + outer)
    x = device(rng.standard_normal((rows, inner)) * np.exp(rng.standard_normal((1, inner))), t_in, pad, shift)
    w = rng.integers(-128, 128, (outer, inner)).astype(np.int8)
    ws = (0.01 * (0.5 + rng.random(outer))).astype(np.float32)
    b = rng.standard_normal(outer).astype(np.float32) if bias else None
    q, scales = device(np.full((rows, inner), 5, np.int8), pad=pad, shift=shift), device(np.full(rows, 9.0))
    bo.int8_quantize_rows(tctx, x, q, scales)
    want_q, want_s = quantize_rows(host(x))
    assert np.array_equal(host(q), want_q) and np.array_equal(host(scales)[0], want_s.astype(np.float64))
    want, size = int8_product(want_q, want_s, w, ws, b)
    wd = device(w, pad=pad, shift=shift)
    out = device(np.full((rows, outer), 9.0), t_out, pad, shift)
    bo.int8_matmul(tctx, q, scales, wd, device(ws), out, bias=None if b is None else device(b))
    assert (np.abs(host(out) - want) <= int8_bound(size, want, t_out)).all()
    fused = device(np.full((rows, outer), 7.0), t_out, pad, shift)
    bo.int8_linear(tctx, x, wd, device(ws), fused, bias=None if b is None else device(b))
    assert torch.equal(fused, out)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_int8_extreme_sums_are_exact(tctx, rows):
    """The largest products of the longest rows: sums up to 2^31 that f32 could not hold on the way."""
    inner = 131071
    q = np.full((rows, inner), -128, np.int8)
    w = np.full((4, inner), -128, np.int8)
    w[1] = 127
    w[2, ::2] = 127
    w[3] = 0
    w[3, 5] = 1
    out = device(np.zeros((rows, 4)))
    bo.int8_matmul(tctx, device(q), device(np.ones(rows)), device(w), device(np.ones(4)), out)
    acc = q[:1].astype(np.int64) @ w.astype(np.int64).T
    assert acc.max() == 2**31 - 16384
    assert np.array_equal(host(out), np.broadcast_to(acc.astype(np.float32).astype(np.float64), (rows, 4)))


def test_int8_rows_of_zeros_infinities_and_nan(tctx):
    x = np.ones((6, 24), np.float32)
    x[0] = 0.0
    x[1, 5] = np.inf
    x[2, 23] = np.nan
    x[3] = 1e-35     # below 2^-100
    x[4] = 1e-42     # subnormal
    x[5] = -3.0e38   # near the largest
    q, s = device(np.full((6, 24), 5, np.int8)), device(np.zeros(6))
    bo.int8_quantize_rows(tctx, device(x), q, s)
    assert (host(q)[:5] == 0).all() and (host(q)[5] == -127).all()
    got = host(s)[0]
    assert got[0] == 0 and np.isnan(got[1:3]).all() and (got[3:5] == 0).all() and got[5] == np.float32(3.0e38) * (np.float32(1) / np.float32(127))
    out = device(np.zeros((6, 7)))
    bias = np.arange(7.0)
    bo.int8_linear(tctx, device(x), device(np.ones((7, 24), np.int8)), device(np.full(7, 1e-3)), out, bias=device(bias))
    y = host(out)
    assert (y[[0, 3, 4]] == bias).all() and np.isnan(y[1:3]).all() and np.isfinite(y[5]).all()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("pad", [0, 8, 1])  # results that leave in blocks, into padded rows, and element by element
def test_int8_of_many_tiles_of_long_rows(tctx, t, pad):
    rows, inner, outer = 4700, 2100, 3990
    g = torch.Generator(device="cuda").manual_seed(7)
    q = torch.randint(-127, 128, (rows, inner), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (outer, inner), generator=g, device="cuda", dtype=torch.int8)
    scales, ws = torch.rand(rows, generator=g, device="cuda"), torch.rand(outer, generator=g, device="cuda")
    wide = torch.full((rows, outer + 10 + pad), 9.0, device="cuda", dtype=kind(t))
    bo.int8_matmul(tctx, q, scales, w, ws, wide[:, :outer])
    assert (wide[:, outer:] == 9.0).all()
    want = (q.double() @ w.double().T) * scales.double()[:, None] * ws.double()
    # the sum's, the scales' product's and the result's rounding, and bf16's
    assert ((wide[:, :outer].double() - want).abs() <= (4 * U32 + (2.0 ** -8 if t == BF16 else 0.0)) * want.abs()).all()


def test_int8_beyond_32_bit_offsets(tctx):
    stride = 2**30 + 16  # row 2 of the weights starts past 2^31 bytes
    memory = torch.zeros(2 * stride + 64, device="cuda", dtype=torch.int8)
    w = torch.as_strided(memory, (3, 64), (stride, 1))
    w.copy_(torch.tensor([[1], [2], [3]], device="cuda", dtype=torch.int8).expand(3, 64))
    for rows in (1, 50):
        out = torch.empty(rows, 3, device="cuda")
        bo.int8_matmul(tctx, torch.ones(rows, 64, device="cuda", dtype=torch.int8), torch.ones(rows, device="cuda"), w,
                       torch.ones(3, device="cuda"), out)
        assert torch.equal(out, torch.tensor([64.0, 128.0, 192.0], device="cuda").expand(rows, 3))


# --------------------------------------------------------------------------- streams, graphs, buffers
def test_library_buffers_streams_and_graphs():
    """The operators on the library's own buffers and stream, and replayed from a captured graph."""
    ctx = bo.Context(0)
    rng = np.random.default_rng(21)
    table = rng.standard_normal((30, 12)).astype(np.float32)
    tokens = rng.integers(-1, 30, 50).astype(np.int32)
    tb, kb = bo.F32Buffer.from_host(ctx, table), bo.I32Buffer.from_host(ctx, tokens)
    out, grad = bo.F32Buffer(ctx, 50 * 12), bo.F32Buffer(ctx, 30 * 12)
    m_table, m_out, m_grad = bo.DeviceMatrix(tb, 30, 12), bo.DeviceMatrix(out, 50, 12), bo.DeviceMatrix(grad, 30, 12)

    def both():
        bo.embedding_forward(ctx, m_table, kb, m_out, scale=3.0)
        bo.embedding_backward(ctx, kb, m_out, m_grad, scale=1.0)

    both()
    first = grad.download()
    want, mag, terms = embedding_grad(tokens, out.download().reshape(50, 12), 30, 1.0)
    assert np.array_equal(out.download().reshape(50, 12), embedding(table, tokens, 3.0).astype(np.float32))
    assert (np.abs(first.reshape(30, 12) - want) <= (terms[:, None] + 2) * U32 * mag).all()
    bo.GraphExec.begin_capture(ctx)
    both()
    graph = bo.GraphExec.end_capture(ctx)
    grad.fill(0.0)
    tokens2 = rng.integers(-1, 30, 50).astype(np.int32)
    kb.upload(tokens2)
    graph.launch(ctx)
    got = grad.download().reshape(30, 12)
    want, mag, terms = embedding_grad(tokens2, out.download().reshape(50, 12), 30, 1.0)
    assert (np.abs(got - want) <= (terms[:, None] + 2) * U32 * mag).all()
    graph.close()
    ctx.close()


def test_all_operators_in_one_graph():
    """Captured once after their sizes have run; the replay reads what the buffers hold then."""
    stream = torch.cuda.Stream()
    ctx = bo.Context(0, stream=stream.cuda_stream)
    with torch.cuda.stream(stream):
        rng = np.random.default_rng(6)
        tokens = device(rng.integers(-1, 40, 3000).astype(np.int32))
        table, weights = device(rng.standard_normal((40, 32))), device(rng.integers(-127, 128, (9, 32)).astype(np.int8))
        hidden, d_table = device(np.zeros((3000, 32))), device(np.zeros((40, 32)))
        logits, d_logits = device(np.zeros((3000, 9))), device(np.zeros((3000, 9)))
        out = {"experts": device(np.zeros((3000, 2), np.int32)), "gates": device(np.zeros((3000, 2))),
               "counts": device(np.zeros(10, np.int32)), "mean": device(np.zeros(9)), "loss": device([0.0])}
        scales, one, gate_grad = device(np.full(9, 0.01)), device([1.0]), device(rng.standard_normal((3000, 2)))

        def everything():
            bo.embedding_forward(ctx, table, tokens, hidden, scale=0.5)
            bo.dropout(ctx, hidden, hidden, probability=0.2, seed=8)
            bo.int8_linear(ctx, hidden, weights, scales, logits)
            bo.router_forward(ctx, logits, out["experts"], out["gates"], out["counts"], out["mean"], out["loss"], balance=0.1)
            bo.router_backward(ctx, logits, out["experts"], out["counts"], gate_grad, one, d_logits, balance=0.1)
            bo.embedding_backward(ctx, tokens, hidden, d_table, scale=2.0)

        everything()
        bo.GraphExec.begin_capture(ctx)
        everything()
        graph = bo.GraphExec.end_capture(ctx)
        tokens.copy_(device(rng.integers(-1, 40, 3000).astype(np.int32)))
        table.mul_(-0.75)
        everything()
        want = [t.clone() for t in (hidden, logits, d_logits, d_table, *out.values())]
        for t in (hidden, logits, d_logits, d_table, *out.values()):
            t.fill_(3)
        graph.launch(ctx)
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (hidden, logits, d_logits, d_table, *out.values())))
    graph.close()
    ctx.close()


def test_tensors_of_another_stream_are_ordered_by_events():
    """The context has a stream of its own: torch's work and the library's wait for one another by events."""
    import ctypes

    ctx = bo.Context(0)
    p = ctypes.c_void_p()
    ctx.lib.call("bulletou_b200_context_stream", ctx.as_ptr(), ctypes.byref(p))
    theirs, ours = torch.cuda.current_stream(), torch.cuda.ExternalStream(p.value)
    x, y = torch.zeros(2048, 4096, device="cuda"), torch.zeros(2048, 4096, device="cuda")
    for round_ in range(1, 6):
        for _ in range(20):
            x.add_(1.0)  # work that the library has to wait for
        ours.wait_stream(theirs)
        bo.dropout(ctx, x, y, probability=0.0, seed=1)
        theirs.wait_stream(ours)
        assert bool((y == 20.0 * round_).all())
    ctx.close()


def test_scratch_grows_between_sizes(tctx):
    """Small, large, small again: scratch that grew in between changes nothing."""
    rng = np.random.default_rng(3)

    def once(n):
        g = np.random.default_rng(n)
        tokens, grad = g.integers(0, 20, n).astype(np.int32), g.standard_normal((n, 16))
        got = device(np.zeros((20, 16)))
        bo.embedding_backward(tctx, device(tokens), device(grad), got)
        x, w = device(g.standard_normal((n, 40))), device(g.integers(-127, 128, (6, 40)).astype(np.int8))
        y = device(np.zeros((n, 6)))
        bo.int8_linear(tctx, x, w, device(np.ones(6)), y)
        return host(got), host(y)

    del rng
    small = once(50)
    once(30000)
    again = once(50)
    assert all(np.array_equal(a, b) for a, b in zip(small, again))


# --------------------------------------------------------------------------- columns of one matrix
def test_operands_that_are_columns_of_one_matrix(tctx):
    """Slices of a wider matrix share its memory's span, but no element."""
    rng = np.random.default_rng(31)
    wide = torch.from_numpy(rng.standard_normal((20, 48)).astype(np.float32)).cuda()
    before = wide.clone()
    for x, out in ((wide[:, :16], wide[:, 16:32]), (wide[:, 32:], wide[:, 16:32])):
        bo.dropout(tctx, x, out, probability=0.5, seed=4)
        keep, factor = dropout_keep(0, 320, 0.5, 4, 0)
        assert np.array_equal(host(out), np.where(keep.reshape(20, 16), host(x) * factor, 0.0))
    assert torch.equal(wide[:, :16], before[:, :16]) and torch.equal(wide[:, 32:], before[:, 32:])
    for x, out in ((wide[:, :16], wide[:, 8:24]), (wide[1:, :16], wide[:-1, 15:31])):  # they share a column
        with pytest.raises(bo.CudaCppError, match="overlap"):
            bo.dropout(tctx, x, out, probability=0.5, seed=4)


# --------------------------------------------------------------------------- refusals
def test_refusals(tctx):
    f, i8, i32 = (lambda *s: torch.zeros(*s, device="cuda")), (lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int8)), \
                 (lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32))
    bf = f(4, 8).bfloat16()
    same = f(8, 8)
    cases = [
        ("expected", lambda: bo.embedding_forward(tctx, f(5, 8), i32(4), f(4, 7))),
        ("expected", lambda: bo.embedding_forward(tctx, f(5, 8), i32(4), f(3, 8))),
        ("does not take", lambda: bo.embedding_forward(tctx, f(5, 8), f(4), f(4, 8))),
        ("does not take", lambda: bo.embedding_forward(tctx, i32(5, 8), i32(4), f(4, 8))),
        ("must not be null", lambda: bo.embedding_forward(tctx, None, i32(4), f(4, 8))),
        ("overlap", lambda: bo.embedding_forward(tctx, same[:5], i32(4), same[4:])),
        ("expected", lambda: bo.embedding_backward(tctx, i32(4), f(4, 8), f(5, 9))),
        ("overlap", lambda: bo.embedding_backward(tctx, i32(4), same[:4], same[3:])),
        ("probability", lambda: bo.dropout(tctx, f(4, 8), f(4, 8), probability=1.5, seed=1)),
        ("probability", lambda: bo.dropout(tctx, f(4, 8), f(4, 8), probability=-0.1, seed=1)),
        ("probability", lambda: bo.dropout(tctx, f(4, 8), f(4, 8), probability=float("nan"), seed=1)),
        ("does not take", lambda: bo.dropout(tctx, f(4, 8), bf, probability=0.5, seed=1)),
        ("expected", lambda: bo.dropout(tctx, f(4, 8), f(4, 8), probability=0.5, seed=1, residual=f(4, 9))),
        ("overlap", lambda: bo.dropout(tctx, same[:4], same[1:5], probability=0.5, seed=1)),
        ("experts", lambda: run_router(tctx, f(4, 513), 1, 1.0, False)),
        ("top_k", lambda: run_router(tctx, f(4, 20), 9, 1.0, False)),
        ("top_k", lambda: run_router(tctx, f(4, 3), 4, 1.0, False)),
        ("router counts", lambda: bo.router_forward(tctx, f(4, 3), i32(4, 1), f(4, 1), i32(3), f(3), f(1), balance=1.0)),
        ("router loss", lambda: bo.router_forward(tctx, f(4, 3), i32(4, 1), f(4, 1), i32(4), f(3), f(2), balance=1.0)),
        ("logit gradients", lambda: bo.router_backward(tctx, f(4, 8), i32(4, 1), i32(9), None, None, bf, balance=1.0)),
        ("at most", lambda: bo.int8_matmul(tctx, i8(1, 131072), f(1), i8(1, 131072), f(1), f(1, 1))),
        ("expected", lambda: bo.int8_linear(tctx, f(4, 8), i8(3, 9), f(3), f(4, 3))),
        ("expected", lambda: bo.int8_linear(tctx, f(4, 8), i8(3, 8), f(4), f(4, 3))),
        ("expected", lambda: bo.int8_linear(tctx, f(4, 8), i8(3, 8), f(3), f(4, 4))),
        ("does not take", lambda: bo.int8_linear(tctx, f(4, 8), f(3, 8), f(3), f(4, 3))),
        ("does not take", lambda: bo.int8_quantize_rows(tctx, f(4, 8), f(4, 8), f(4))),
        ("overlap", lambda: bo.int8_linear(tctx, same[:4], i8(8, 8), f(8), same[2:6])),
        # the Python side
        ("contiguous", lambda: bo.dropout(tctx, f(8, 4).t(), f(4, 8), probability=0.5, seed=1)),
        ("dimensions", lambda: bo.dropout(tctx, f(2, 2, 8), f(4, 8), probability=0.5, seed=1)),
        ("not supported", lambda: bo.dropout(tctx, f(4, 8).double(), f(4, 8), probability=0.5, seed=1)),
        ("tensor is on", lambda: bo.dropout(tctx, torch.zeros(4, 8), f(4, 8), probability=0.5, seed=1)),
        ("a matrix is expected", lambda: bo.dropout(tctx, np.zeros((4, 8)), f(4, 8), probability=0.5, seed=1)),
        ("row stride", lambda: bo.dropout(tctx, f(8).expand(4, 8), f(4, 8), probability=0.5, seed=1)),
    ]
    for message, call in cases:
        with pytest.raises(bo.CudaCppError, match=message):
            call()
    # a refused call leaves the context usable
    out = f(4, 8)
    bo.dropout(tctx, torch.ones(4, 8, device="cuda"), out, probability=0.0, seed=1)
    assert bool((out == 1).all())


def test_device_matrix_refusals(ctx):
    b, i = bo.F32Buffer(ctx, 100), bo.I32Buffer(ctx, 10)
    for bad in (lambda: bo.DeviceMatrix(b, 10, 11), lambda: bo.DeviceMatrix(b, 10, 10, offset=1),
                lambda: bo.DeviceMatrix(b, 2, 10, row_stride=9), lambda: bo.DeviceMatrix(b, 10, 10, "i8"),
                lambda: bo.DeviceMatrix(i, 5, 9, "i8"), lambda: bo.DeviceMatrix(i, 1, 21, "bf16"),
                lambda: bo.DeviceMatrix(i, 1, 4, "f32"), lambda: bo.DeviceMatrix(b, -1, 4)):
        with pytest.raises(bo.CudaCppError):
            bad()
    assert bo.DeviceMatrix(i, 4, 10, "i8").row_stride == 10
    assert bo.DeviceMatrix(b, 9, 10, row_stride=11).data == b.device_ptr()
