"""CPU: the plain forms behind the token-layer tests, and refusals that need no GPU."""
import ctypes

import numpy as np
import pytest

from tests.token_layer_cases import dropout_keep, philox, quantize_rows, router, router_grad, router_objective


def test_philox_known_answers():
    """The generator's published known-answer vectors (zeros, ones, digits of pi)."""
    cases = [((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
             ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
             ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
              (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]
    for counter, key, want in cases:
        assert tuple(int(v) for v in philox(np.array([counter], np.uint64), key)[0]) == want


def test_dropout_keep_is_a_window_of_one_sequence():
    whole, factor = dropout_keep(0, 1000, 0.25, 7, 2**40)
    part, _ = dropout_keep(133, 500, 0.25, 7, 2**40)
    assert np.array_equal(whole[133:633], part) and factor == 4 / 3
    assert dropout_keep(0, 100, 1.0, 7, 0)[0].sum() == 0 and dropout_keep(0, 100, 0.0, 7, 0)[0].all()


@pytest.mark.parametrize("normalize", [False, True])
def test_router_gradient_is_the_objectives(normalize):
    rng = np.random.default_rng(1)
    z = rng.standard_normal((5, 7))
    z[1, 3], z[2] = -np.inf, -np.inf
    r = router(z, 3, 0.1, normalize)
    gg = rng.standard_normal((5, 3))
    want = router_grad(z, r, gg, 1.3, 0.1, normalize)
    share, live = r["counts"][:-1] / r["counts"][:-1].sum(), int(r["counts"][-1])
    for t in range(5):
        for e in range(7):
            if np.isfinite(z[t, e]):
                f = []
                for s in (1e-5, -1e-5):
                    moved = z.copy()
                    moved[t, e] += s
                    f.append(router_objective(moved, r["experts"], share, live, gg, 1.3, 0.1, normalize))
                assert abs((f[0] - f[1]) / 2e-5 - want[t, e]) < 1e-8


def test_balance_loss_is_least_where_experts_are_used_alike():
    even = router(np.eye(4) * 3, 1, 1.0, False)
    assert abs(even["loss"] - 1.0) < 1e-12
    assert router(np.tile([3.0, 0, 0, 0], (4, 1)), 1, 1.0, False)["loss"] > 1.5


def test_quantised_rows_reach_127():
    q, s = quantize_rows(np.array([[0.5, -1.0, 0.25], [0, 0, 0]], np.float32))
    assert q.tolist() == [[64, -127, 32], [0, 0, 0]] and s[1] == 0


def test_entries_refuse_a_null_context(lib):
    from bulletou_b200._lib import SIGNATURES

    for name in ("embedding_forward", "embedding_backward", "dropout", "router_forward", "router_backward",
                 "int8_quantize_rows", "int8_matmul", "int8_linear"):
        full = f"bulletou_b200_{name}_device"
        values = (ctypes.c_float, ctypes.c_double, ctypes.c_int, ctypes.c_uint64)
        args = [a(0) if a in values else None for a in SIGNATURES[full]]
        assert lib.fn(full)(*args) == -1
        assert "context must not be null" in lib.last_error()
