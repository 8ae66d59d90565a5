"""GPU: the token layers at the edges of what they take: empty inner sizes,
limits of shared memory and of 32-bit indexes, operands that begin and end inside
16 bytes, graphs that outlive a larger call, and the router model's evaluation.
"""
import numpy as np
import pytest

import bulletou_b200 as bo
from tests.token_layer_cases import U32, UBF, int8_product, quantize_rows

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tctx():
    c = bo.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# --------------------------------------------------------------------------- lookup
@pytest.mark.parametrize("width,pad", [(8, 0), (256, 0), (257, 0), (63, 1)])
@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -2.0])
def test_padded_tokens_are_zeros_at_any_scale(tctx, width, pad, scale):
    table = torch.ones(5, width + pad, device="cuda")[:, :width]
    tokens = torch.tensor([-1, 4, 5, 0, -1, 2, 2**31 - 1], device="cuda", dtype=torch.int32)
    for t in (torch.float32, torch.bfloat16):
        out = torch.full((7, width), 9.0, device="cuda", dtype=t)
        bo.embedding_forward(tctx, table, tokens, out, scale=scale)
        inside = torch.tensor([False, True, False, True, False, True, False], device="cuda")
        assert not out[~inside].any() and torch.equal(out[inside].nan_to_num(7.0), torch.full((3, width), scale, device="cuda", dtype=t).nan_to_num(7.0))


# --------------------------------------------------------------------------- 8-bit product
@pytest.mark.parametrize("rows,outer", [(1, 5), (2, 300), (40, 70), (300, 20000), (4096, 4096), (4700, 1100), (70000, 65)])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [True, False])
def test_int8_of_no_inner_columns_is_the_bias(tctx, rows, outer, t, bias):
    """At few tiles and at many, whichever kernel they go to: an empty sum is 0, so the results are exact."""
    g = torch.Generator(device="cuda").manual_seed(rows + outer)
    b = torch.randn(outer, generator=g, device="cuda") if bias else None
    want = (torch.zeros(outer, device="cuda") if b is None else b).to(t).expand(rows, outer)
    scales, ws = torch.rand(rows, generator=g, device="cuda"), torch.rand(outer, generator=g, device="cuda")
    w = torch.empty(outer, 0, device="cuda", dtype=torch.int8)
    out = torch.full((rows, outer), 9.0, device="cuda", dtype=t)
    bo.int8_linear(tctx, torch.empty(rows, 0, device="cuda"), w, ws, out, bias=b)
    assert torch.equal(out, want)
    out.fill_(9.0)
    bo.int8_matmul(tctx, torch.empty(rows, 0, device="cuda", dtype=torch.int8), scales, w, ws, out, bias=b)
    assert torch.equal(out, want)


@pytest.mark.parametrize("rows", [1, 2, 3])
@pytest.mark.parametrize("inner", [24543, 24544, 24545, 24560, 24561, 24576, 24577, 49152, 49153])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_int8_around_the_shared_memory_of_few_rows(tctx, rows, inner, t):
    """Two rows fill a launch's 48 KB of shared memory, with the kernel's own 64 bytes, at 24544 columns."""
    rng = np.random.default_rng(inner + rows)
    x = cuda(rng.standard_normal((rows, inner)).astype(np.float32))
    w = rng.integers(-128, 128, (11, inner)).astype(np.int8)
    ws = (0.01 * (0.5 + rng.random(11))).astype(np.float32)
    want_q, want_s = quantize_rows(x.cpu().numpy())
    want, size = int8_product(want_q, want_s, w, ws, None)
    # the scales' product, its product with the sum, the sum's conversion and the last operation; bf16's
    bound = 4 * U32 * (size + np.abs(want)) + (UBF if t == torch.bfloat16 else 0.0) * np.abs(want)
    out = torch.full((rows, 11), 9.0, device="cuda", dtype=t)
    bo.int8_linear(tctx, x, cuda(w), cuda(ws), out)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
    out.fill_(9.0)
    bo.int8_matmul(tctx, cuda(want_q), cuda(want_s), cuda(w), cuda(ws), out)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,gap", [(1, 1, 0), (1, 15, 0), (1, 16, 0), (1, 33, 0), (3, 7, 0), (3, 40, 1), (2, 255, 9), (4, 1031, 3)])
def test_quantise_rows_that_begin_and_end_inside_16_bytes(tctx, t, rows, cols, gap):
    """At every alignment, from the first element of the memory to its last; what lies beside the rows is not looked at."""
    rng = np.random.default_rng(cols)
    for shift in range(8):
        memory = torch.full((shift + rows * (cols + gap) - gap,), float("nan"), device="cuda", dtype=t)
        x = torch.as_strided(memory, (rows, cols), (cols + gap, 1), shift)
        x.copy_(cuda(rng.standard_normal((rows, cols)).astype(np.float32)))
        q, s = torch.full((rows, cols), 5, device="cuda", dtype=torch.int8), torch.zeros(rows, device="cuda")
        bo.int8_quantize_rows(tctx, x, q, s)
        want_q, want_s = quantize_rows(x.float().cpu().numpy())
        assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(s.cpu().numpy(), want_s)


@pytest.mark.parametrize("t,cols", [(torch.float32, 2**29 + 9), (torch.bfloat16, 2**30 + 9)])
@pytest.mark.parametrize("shift", [0, 1])  # a row on 16 bytes and off them
def test_quantise_rows_of_more_than_31_bits_of_bytes(tctx, t, cols, shift):
    memory = torch.zeros(cols + shift, device="cuda", dtype=t)
    x = memory[shift:].view(1, cols)
    at = torch.tensor([0, 1, 17, 4095, 4096, 8191, 2**20 + 3, 2**28 + 1, cols - 2**20, cols - 17, cols - 1], device="cuda")
    x[0, at] = torch.linspace(-1.0, 2.0, 11, device="cuda").to(t)
    q, s = torch.full((1, cols), 5, device="cuda", dtype=torch.int8), torch.zeros(1, device="cuda")
    bo.int8_quantize_rows(tctx, x, q, s)
    want_q, want_s = quantize_rows(x[:, at].float().cpu().numpy())  # they hold the largest; the rest are zeros
    assert np.array_equal(q[:, at].cpu().numpy(), want_q) and s.item() == want_s[0]
    q[0, at] = 0
    assert not q.view(-1)[: cols // 8 * 8].view(torch.int64).any() and not q[0, cols // 8 * 8 :].any()


# --------------------------------------------------------------------------- graphs
def scratch_bytes(ctx):
    import ctypes

    n = ctypes.c_size_t(0)
    ctx.lib.call("bulletou_b200_context_scratch_bytes", ctx.as_ptr(), ctypes.byref(n))
    return n.value


class Calls:
    """The three operators that use scratch, on tensors for up to `n` tokens."""

    def __init__(self, n, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.n, self.g = n, g
        self.tokens = torch.randint(-1, 700, (n,), generator=g, device="cuda", dtype=torch.int32)
        self.grad = torch.randn(n, 40, generator=g, device="cuda")
        self.logits = torch.randn(n, 9, generator=g, device="cuda")
        self.weights = torch.randint(-127, 128, (70, 40), generator=g, device="cuda", dtype=torch.int8)
        self.scales = torch.rand(70, generator=g, device="cuda")
        self.out = {"table": torch.zeros(700, 40, device="cuda"), "experts": torch.zeros(n, 2, device="cuda", dtype=torch.int32),
                    "gates": torch.zeros(n, 2, device="cuda"), "counts": torch.zeros(10, device="cuda", dtype=torch.int32),
                    "mean": torch.zeros(9, device="cuda"), "loss": torch.zeros(1, device="cuda"), "y": torch.zeros(n, 70, device="cuda")}

    def run(self, ctx):
        o = self.out
        bo.embedding_backward(ctx, self.tokens, self.grad, o["table"])
        bo.router_forward(ctx, self.logits, o["experts"], o["gates"], o["counts"], o["mean"], o["loss"], balance=0.1)
        bo.int8_linear(ctx, self.grad, self.weights, self.scales, o["y"])


def test_graph_replays_after_larger_calls():
    """Scratch that a graph was captured with stays its own when larger calls outgrow it."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx, plain = (bo.Context(0, stream=stream.cuda_stream) for _ in range(2))
        small, sizes = Calls(6000, 1), (20000, 90000)
        small.run(ctx)
        held = scratch_bytes(ctx)
        bo.GraphExec.begin_capture(ctx)
        small.run(ctx)
        graph = bo.GraphExec.end_capture(ctx)
        for n in sizes:
            large = Calls(n, n)
            large.run(ctx)
            large.run(plain)
            # the captured blocks are kept once; those of the first larger size are not
            assert scratch_bytes(ctx) == scratch_bytes(plain) + held
            junk = torch.full((1 << 26,), float("nan"), device="cuda")  # whatever was freed holds something else by now
            small.tokens.copy_(torch.randint(-1, 700, (6000,), generator=small.g, device="cuda", dtype=torch.int32))
            small.grad.normal_(generator=small.g)
            small.logits.normal_(generator=small.g)
            small.run(ctx)
            want = {k: v.clone() for k, v in small.out.items()}
            for v in small.out.values():
                v.fill_(3)
            graph.launch(ctx)
            stream.synchronize()
            assert all(torch.equal(want[k], small.out[k]) for k in want)
            del junk
        graph.close()
        ctx.close()
        plain.close()


# --------------------------------------------------------------------------- the router model
VOCAB, ACTIVE, WIDTH, STACKS, BATCH = 50, 6, 8, 5, 40


@pytest.fixture
def model():
    ctx = bo.Context(0)
    rng = np.random.default_rng(11)
    r = bo.StackRouter(ctx, VOCAB, ACTIVE, WIDTH, STACKS, BATCH, top_k=2, balance=0.05, drop_probability=0.2, seed=5)
    tokens = rng.integers(-1, VOCAB, (BATCH, ACTIVE)).astype(np.int32)
    costs = bo.F32Buffer.from_host(ctx, rng.random((BATCH, STACKS)).astype(np.float32))
    yield ctx, r, tokens, bo.I32Buffer.from_host(ctx, tokens), costs, bo.I32Buffer(ctx, BATCH)
    ctx.close()


def eight_bit_choices(r, tokens):
    """The choices of the parameters that the model holds now, and whether a position's two best logits are apart."""
    table, weights = r.table.download().reshape(VOCAB, WIDTH), r.weights.download().reshape(STACKS, -1)
    hidden = (np.float32(r.scale) * np.where(tokens.reshape(-1, 1) >= 0, table[tokens.reshape(-1)], np.float32(0))).reshape(BATCH, -1)
    z, size = int8_product(*quantize_rows(hidden), *quantize_rows(weights), None)
    order = np.sort(z, 1)
    return z.argmax(1), order[:, -1] - order[:, -2] > 8 * U32 * size.max()


def test_choice_leaves_the_last_steps_losses(model):
    ctx, r, tokens, on_device, costs, buckets = model
    r.gradients(on_device, costs)
    losses = r.read_losses()
    r.choose(on_device, buckets)
    assert r.read_losses() == losses


def test_choices_follow_the_weights(model):
    """After a step and after new values in the parameters' buffers; weights are kept from before only where that is asked."""
    ctx, r, tokens, on_device, costs, buckets = model

    def check():
        want, apart = eight_bit_choices(r, tokens)
        assert apart.any() and np.array_equal(buckets.download()[apart], want[apart])
        return want

    r.choose(on_device, buckets)
    first = check()
    r.train_step(bo.RangerUpdateParams(radam=bo.RAdamUpdateParams(step=1, learning_rate=0.5)), on_device, costs)
    r.choose(on_device, buckets, keep_weights=True)  # kept weights end with an update
    check()
    rng = np.random.default_rng(13)
    r.table.upload(rng.standard_normal((VOCAB, WIDTH)).astype(np.float32))
    r.weights.upload(rng.standard_normal((STACKS, ACTIVE * WIDTH)).astype(np.float32))
    r.choose(on_device, buckets)
    assert not np.array_equal(check(), first)
    r.choose(on_device, buckets, keep_weights=True)
    check()
    r.weights.upload(-r.weights.download())
    before = buckets.download()
    r.choose(on_device, buckets, keep_weights=True)
    assert np.array_equal(buckets.download(), before)
    r.choose(on_device, buckets)
    check()


def test_position_that_is_not_finite_has_no_choice(model):
    """-1, a bucket that belongs to no stack; the others choose as before."""
    ctx, r, tokens, on_device, costs, buckets = model
    r.choose(on_device, buckets)
    before = buckets.download()
    table = r.table.download().reshape(VOCAB, WIDTH)
    broken = int(tokens[0][tokens[0] >= 0][0])
    table[broken, 3] = np.nan
    r.table.upload(table)
    r.choose(on_device, buckets)
    hit = (tokens == broken).any(1)
    got = buckets.download()
    assert (got[hit] == -1).all() and np.array_equal(got[~hit], before[~hit])
    assert r.read_counts().sum() == BATCH - hit.sum()


# --------------------------------------------------------------------------- router
def test_gates_of_equal_logits_are_rounded_once(tctx):
    """One of n alike: the exponentials and their sum are exact, so the gate is 1 / n to half a unit in its last place
    (and 2^-45 for the iteration behind it)."""
    for n in range(1, 513):
        z = torch.full((1, n), -3.25, device="cuda")
        experts, gates = torch.zeros(1, 1, device="cuda", dtype=torch.int32), torch.zeros(1, 1, device="cuda")
        counts, mean, loss = torch.zeros(n + 1, device="cuda", dtype=torch.int32), torch.zeros(n, device="cuda"), torch.zeros(1, device="cuda")
        bo.router_forward(tctx, z, experts, gates, counts, mean, loss, balance=1.0)
        half_unit = 2.0 ** (np.floor(np.log2(1 / n)) - 24)
        assert abs(gates.item() - 1 / n) <= half_unit + 2.0 ** -45 / n, n
