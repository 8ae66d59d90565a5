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
