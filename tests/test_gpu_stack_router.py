"""GPU: the learned LayerStack router (lookup, dropout, logits, routing and back; 8-bit evaluation) against plain 64-bit
arithmetic, and its example."""
import sys

import numpy as np
import pytest

import bulletou_b200 as bo
from tests.conftest import ROOT
from tests.token_layer_cases import U32, dropout_keep, embedding, embedding_grad, int8_product, quantize_rows, router, router_grad

pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

VOCAB, ACTIVE, WIDTH, STACKS, BATCH, TOP = 60, 7, 12, 5, 33, 2


def make(ctx, drop):
    rng = np.random.default_rng(7)
    table = rng.standard_normal((VOCAB, WIDTH)).astype(np.float32)
    weights = (rng.standard_normal((STACKS, ACTIVE * WIDTH)) * 0.3).astype(np.float32)
    tokens = rng.integers(-1, VOCAB, (BATCH, ACTIVE)).astype(np.int32)
    tokens[4] = -1  # a position without tokens
    costs = rng.random((BATCH, STACKS)).astype(np.float32)
    r = bo.StackRouter(ctx, VOCAB, ACTIVE, WIDTH, STACKS, BATCH, top_k=TOP, balance=0.05, drop_probability=drop, seed=3,
                       table=table, weights=weights)
    return r, table, weights, tokens, costs


@pytest.mark.parametrize("drop", [0.0, 0.25])
def test_train_step_gradients(drop):
    ctx = bo.Context(0)
    r, table, weights, tokens, costs = make(ctx, drop)
    r.gradients(bo.I32Buffer.from_host(ctx, tokens), bo.F32Buffer.from_host(ctx, costs))
    keep, factor = dropout_keep(0, BATCH * ACTIVE * WIDTH, drop, 3, 0)
    mask = keep.reshape(-1, WIDTH) * factor
    hidden = embedding(table, tokens, float(np.float32(r.scale))) * mask
    z = hidden.reshape(BATCH, -1) @ weights.astype(np.float64).T
    got_z = r.logits.download().reshape(BATCH, STACKS)
    n = ACTIVE * WIDTH
    assert np.abs(got_z - z).max() <= (n + 6) * U32 * np.abs(hidden.reshape(BATCH, -1)).max() * np.abs(weights).sum(1).max()
    want = router(got_z, TOP, 0.05, True)  # the choices follow the logits in hand
    experts = r.experts.download().reshape(BATCH, TOP)
    assert np.array_equal(experts, want["experts"]) and np.array_equal(r.read_counts(), want["counts"][:-1])
    picked = np.take_along_axis(costs, experts, 1) / BATCH
    cost, balance = r.read_losses()
    assert abs(cost - (want["gates"] * picked).sum()) <= 1e-5 and abs(balance - want["loss"]) <= 1e-5 * want["loss"]
    d_z = router_grad(got_z, want, picked, 1.0, 0.05, True)
    d_weights = d_z.T @ hidden.reshape(BATCH, -1)
    d_hidden = (d_z @ weights.astype(np.float64)).reshape(-1, WIDTH) * mask
    d_table, mag, _ = embedding_grad(tokens, d_hidden, VOCAB, r.scale)
    # f32 chains of at most a few hundred terms: 1e-5 of the largest magnitude is above 150 u
    for got, exact in ((r.weight_gradients, d_weights), (r.table_gradients, d_table)):
        assert np.abs(got.download().reshape(exact.shape) - exact).max() <= 1e-5 * max(np.abs(exact).max(), mag.max())
    r.update(bo.RangerUpdateParams(radam=bo.RAdamUpdateParams(step=1)))
    assert not np.array_equal(r.table.download().reshape(VOCAB, WIDTH), table)  # Ranger has moved them
    assert not np.array_equal(r.weights.download().reshape(weights.shape), weights)
    ctx.close()


def test_choices_in_eight_bits():
    ctx = bo.Context(0)
    r, table, weights, tokens, _ = make(ctx, 0.0)
    buckets = bo.I32Buffer(ctx, BATCH)
    r.choose(bo.I32Buffer.from_host(ctx, tokens), buckets)
    hidden = (np.float32(r.scale) * np.where(tokens.reshape(-1, 1) >= 0, table[tokens.reshape(-1)], np.float32(0))).reshape(BATCH, -1)
    q, s = quantize_rows(hidden)
    w, ws = quantize_rows(weights)
    z, size = int8_product(q, s, w, ws, None)
    got = r.logits.download().reshape(BATCH, STACKS)
    assert (np.abs(got - z) <= 4 * U32 * size).all()
    assert np.array_equal(buckets.download(), got.argmax(1)) and buckets.download()[4] == 0
    with pytest.raises(bo.CudaCppError, match="buckets have"):
        r.choose(bo.I32Buffer.from_host(ctx, tokens), bo.I32Buffer(ctx, BATCH + 1))
    with pytest.raises(bo.CudaCppError, match="invalid stack router"):
        bo.StackRouter(ctx, 10, 4, 8, 3, 16, top_k=4)
    ctx.close()


def test_example_learns_the_rule_and_feeds_an_sfnn_step():
    sys.path.insert(0, str(ROOT / "examples"))
    try:
        import learned_stacks
    finally:
        sys.path.pop(0)
    out = learned_stacks.main(steps=40, batch=1024)
    assert out["after"] > 0.6 > out["before"]
    assert np.isfinite(out["loss"]) and out["choices"].min() >= 0 and out["choices"].max() < 9
