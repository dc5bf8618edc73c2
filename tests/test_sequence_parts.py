"""The f32 inputs of the cross entropy's three bf16 parts on the CPU: the parts
themselves, and that the bounds used on the device find a part that is lost."""
import numpy as np
import pytest

import sequence_parts as sp
import sequence_ref as ref


def test_parts_hold_24_bits():
    x = ref.rounded(np.random.default_rng(1).normal(size=10000), "f32")
    assert (np.abs(sum(sp.parts(x)) - x) <= 2.0 ** -24 * np.abs(x)).all()
    p = sp.parts(sp.pattern(50, 50, 2))
    assert (p[0] == 1).all() and (p[1] == 2.0 ** -9).all() and (p[2] >= 2.0 ** -18).all() and (p[2] < 2.0 ** -17).all()


LOST = [[(2, 0)], [(0, 2)], [(1, 1)], [(1, 0)], [(0, 1)], [(0, 0)]]


def test_logit_bound_finds_a_lost_product():
    x, w = sp.logit_inputs(12, 300, 3)
    z = x @ w.T
    assert (np.abs(sp.product(x, w) - z) <= sp.U * z).all()
    for without in LOST:
        off = np.abs(sp.product(x, w, without) - z)
        # (A1 B1 is 2^-18 = 64 U of the sum)
        assert (off > 2 * sp.LOGIT * z).all(), without


@pytest.mark.parametrize("turn", [False, True])
def test_gradient_bounds_find_a_lost_part(turn):
    x, w, targets, g = sp.gradient_inputs(200, 40, 4)
    lse = ref.loss(x, w, targets, "f32")[1]
    p = np.exp(x @ w.T - lse[:, None])
    dz = g[:, None].astype(np.float64) * (p - [1, 0])
    if turn:  # one token counts: dw = dz^T x
        for n in range(12):
            only = np.zeros_like(g)
            only[n] = g[n]
            _, want, _, bound = ref.loss_backward(x, w, targets, lse, only, "f32")
            a, b = ref.rounded(dz[n:n + 1], "f32").T, x[n:n + 1].T
            assert (np.abs(sp.product(a, b) - want) <= bound / 8).all()
            assert (np.abs(sp.product(a, b, [(0, 2)]) - want) > bound).any()
    else:
        want, _, bound, _ = ref.loss_backward(x, w, targets, lse, g, "f32")
        a, b = ref.rounded(dz, "f32"), w.T
        assert (np.abs(sp.product(a, b) - want) <= bound / 8).all()
        for without in LOST[:2]:
            assert (np.abs(sp.product(a, b, without) - want) > bound).any(), without


def test_lost_third_parts_of_dz_show_in_dw():
    """Over the tokens taken one at a time, some lose more than the bound."""
    x, w, targets, g = sp.gradient_inputs(64, 40, 5)
    lse = ref.loss(x, w, targets, "f32")[1]
    dz = g[:, None].astype(np.float64) * (np.exp(x @ w.T - lse[:, None]) - [1, 0])
    found = 0
    for n in range(64):
        only = np.zeros_like(g)
        only[n] = g[n]
        _, want, _, bound = ref.loss_backward(x, w, targets, lse, only, "f32")
        a, b = ref.rounded(dz[n:n + 1], "f32").T, x[n:n + 1].T
        found += (np.abs(sp.product(a, b, [(2, 0)]) - want) > bound).any()
    assert found >= 5
