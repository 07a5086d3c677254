"""trs_cross_attention and its gradient at the ends of the f32 range: finite
inputs whose scores, values or gradients are far from 1, and infinite keys
(tests/_cross.py holds the bounds and their reasons)."""
from __future__ import annotations

import numpy as np
import pytest

from _cross import Truth, check
from _gpu import to_host
from test_cross_attention_gpu import backward, both, cuda, draw, forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", range(1, 10))
@pytest.mark.parametrize("D", [32, 64, 128])
def test_a_key_of_minus_infinity_takes_no_gradient(rows, D):
    """Every query's score with one key is -inf: the key has no weight, its dk and dv are 0, and the other keys'
    gradients are those without it (a row that only fills up a block of rows adds nothing)."""
    q, k, v, g = draw(1, rows, 40, 1, 1, D, seed=rows)
    q[..., 0] = 1.0
    keep = np.arange(40) != 11
    t = Truth(q, k[:, keep], v[:, keep], 0.125, None, g)
    k[0, 11, 0, 0] = -np.inf
    tq, tk, tv, tg = cuda(q), cuda(k), cuda(v), cuda(g)
    out, lse = forward(tq, tk, tv, 0.125)
    check(to_host(out), t.out, t.out_tol, "out")
    check(to_host(lse), t.lse, t.lse_tol, "lse")
    dq, dk, dv = map(to_host, backward(tg, tq, tk, tv, out, lse, 0.125))
    assert (dk[0, 11] == 0).all() and (dv[0, 11] == 0).all()
    check(dk[:, keep], t.dk, t.dk_tol, "dk")
    check(dv[:, keep], t.dv, t.dv_tol, "dv")
    check(dq[..., 1:], t.dq[..., 1:], t.dq_tol[..., 1:], "dq")  # its element 0 is 0 * inf


# B, Tq, Tk, Hq, Hk, D: both sides of the row limits, two row tiles, a walk in parts
RANGE = [(1, 3, 100, 1, 1, 64), (1, 16, 100, 1, 1, 64), (1, 17, 100, 1, 1, 64), (1, 130, 200, 2, 1, 64), (1, 20, 1000, 1, 1, 64),
         (1, 8, 100, 1, 1, 128), (1, 9, 100, 1, 1, 128), (1, 300, 200, 1, 1, 128), (1, 40, 100, 1, 1, 80), (1, 20, 100, 1, 1, 160)]


@pytest.mark.parametrize("size", RANGE, ids=str)
@pytest.mark.parametrize("vs", [1e34, 5e35])
def test_large_values(size, vs):
    """Values up to 2e36, whose weighted sums (weights of 1 at most, less than 100 of them in all) stay in range."""
    q, k, v, g = draw(*size, seed=21)
    both(q, k, v * np.float32(vs), g * np.float32(1 / vs), size[-1] ** -0.5)
