"""trs_cross_attention and its gradient at the ends of the f32 range: finite
inputs whose scores, values or gradients are far from 1, and infinite keys
(tests/_cross.py holds the bounds and their reasons)."""
from __future__ import annotations

import numpy as np
import pytest

from _cross import U, Truth, check, near
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


@pytest.mark.parametrize("size", RANGE, ids=str)
@pytest.mark.parametrize("amplitude", [1e3, 3e3, 1e4, 1e7])
def test_large_scores(size, amplitude):
    """Scores of 1e6 and more: where a row's two largest are further apart than their errors, all of the weight is the
    largest's, and the output its value, held in 22 bits (2^-40 of the tile's largest) and rounded a few times.  The
    gradient's P = exp(S - lse) is off by more than itself there, but it stays a weight: finite and at most 1 (the
    exponential's 2 units and the roundings of the sum beside it), so that |dv| <= sum |grad|."""
    f = np.float32
    q, k, v, g = draw(*size, seed=22)
    q, k = q * f(amplitude), k * f(amplitude)
    scale = size[-1] ** -0.5
    tq, tk, tv, tg = cuda(q), cuda(k), cuda(v), cuda(g)
    out, lse = forward(tq, tk, tv, scale)
    t = Truth(q, k, v, scale, None, g)
    check(to_host(out), t.out, t.out_tol, "out")
    check(to_host(lse), t.lse, t.lse_tol, "lse")
    peaked = 0
    for h in range(size[3]):
        j = h // (size[3] // size[4])
        S = scale * q[0, :, h].astype(np.float64) @ k[0, :, j].T.astype(np.float64)
        first = S.argmax(-1)
        gap = np.sort(S, -1)[:, -1] - np.sort(S, -1)[:, -2]
        clear = gap > 4 * t.lse_tol[0, h] + 200
        peaked += clear.sum()
        want = v[0, first, j].astype(np.float64)
        far = np.abs(to_host(out)[0, :, h] - want)[clear]
        assert (far <= 2.0**-20 * np.abs(want[clear]) + 2.0**-38 * np.abs(v).max()).all()
    assert peaked > 0.9 * size[1] * size[3]
    dq, dk, dv = map(to_host, backward(tg, tq, tk, tv, out, lse, scale))
    assert np.isfinite(dq).all() and np.isfinite(dk).all() and np.isfinite(dv).all()
    most = np.abs(g).astype(np.float64).sum((0, 1)).reshape(size[4], -1, size[5]).sum(1)
    assert (np.abs(dv[0]) <= most * (1 + 2.0**-10)).all()


@pytest.mark.parametrize("rows,D", [(3, 64), (130, 64), (40, 128), (20, 160)])
def test_scores_beyond_f32(rows, D):
    """Finite inputs, scores of +-1e50.  A row with one of +inf has no defined weights: NaN, not the 0 of a row without
    keys.  Rows of -inf alone count as empty, and such keys beside others take nothing."""
    _, _, v, g = draw(1, rows, 200, 1, 1, D, seed=23)
    f = np.float32
    q, k = np.full((1, rows, 1, D), 1e25, f), np.full((1, 200, 1, D), 1e25, f)
    for last in (0, 199):  # one such score is enough, in the first tile or the last
        some = -k
        some[0, last] *= -1
        for x in (k, some):
            out, lse = (to_host(y) for y in forward(cuda(q), cuda(x), cuda(v), 0.125))
            assert np.isnan(out).all() and not (lse < 0).any()
    out, lse = forward(cuda(q), cuda(-k), cuda(v), 0.125)
    assert (to_host(out) == 0).all() and (to_host(lse) == -np.inf).all()
    for d in backward(cuda(g), cuda(q), cuda(-k), cuda(v), out, lse, 0.125):
        assert (to_host(d) == 0).all()
    for there in (slice(0, 64), slice(128, 200)):  # whole tiles of the other kind: scores of 0
        some = -k
        some[0, there] = 0
        out, _ = forward(cuda(q), cuda(some), cuda(v), 0.125)
        want = v[0, there].astype(np.float64).mean(0)
        tol = 2.0**-18 * np.abs(v[0, there]).mean(0) + 2.0**-38 * np.abs(v).max()
        assert (np.abs(to_host(out)[0] - want) <= tol).all()
    # a query of zeros among them
    q[0, 1] = 0
    out, lse = (to_host(y) for y in forward(cuda(q), cuda(-k), cuda(v), 0.125))
    assert (out[0, 0] == 0).all() and abs(lse[0, 0, 1] - np.log(200)) < 1e-5
    assert (np.abs(out[0, 1] - v[0].astype(np.float64).mean(0)) <= 2.0**-18 * np.abs(v[0]).mean(0) + 2.0**-38 * np.abs(v).max()).all()


@pytest.mark.parametrize("size", [(1, 6, 90, 1, 1, 64), (1, 130, 200, 1, 1, 64), (1, 40, 100, 1, 1, 128)], ids=str)
@pytest.mark.parametrize("gs,vs", [(1e8, 1e8), (1e30, 1e3)])
def test_zero_rows_beside_large_ones(size, gs, vs):
    """Queries that take no part in the loss, values that are 0, next to large ones."""
    f = np.float32
    q, k, v, g = draw(*size, seed=26)
    g[:, ::3] = 0
    v[:, ::4] = 0
    both(q, k, v * f(vs), g * f(gs), 0.125)


@pytest.mark.parametrize("size", [(1, 6, 100, 1, 1, 80), (1, 40, 100, 1, 1, 80), (1, 150, 100, 2, 1, 64), (1, 40, 300, 1, 1, 96),
                                  (1, 12, 100, 1, 1, 128), (1, 20, 60, 1, 1, 160)], ids=str)
@pytest.mark.parametrize("gs,vs,ks", [(1e-34, 1.0, 1.0), (1e-32, 1.0, 1e-3), (1e-16, 1e-18, 1.0), (1e-36, 1e20, 1e-18)])
def test_small_gradients(size, gs, vs, ks):
    """Gradients near the smallest normal number (2^-126) keep their bits: sums of some dozen terms of about 1e-35, each
    off by half of 2^-149 where a product falls below 2^-126, 1e-10 of the sum."""
    f = np.float32
    q, k, v, g = draw(*size, seed=24)
    both(q * f(1 / ks), k * f(ks), v * f(vs), g * f(gs), size[-1] ** -0.5)


@pytest.mark.parametrize("size", [(1, 3, 90, 1, 1, 64), (1, 130, 200, 1, 1, 64), (1, 40, 100, 1, 1, 128)], ids=str)
def test_operands_at_both_ends_of_the_range(size):
    """Small queries on large keys under a small scale: the scores are of order 1, whatever the scale and one operand
    make by themselves."""
    f = np.float32
    q, k, v, g = draw(*size, seed=25)
    q, k = q * f(2.0**-116), k * f(2.0**124)
    tq, tk, tv, tg = cuda(q), cuda(k), cuda(v), cuda(g)
    out, lse = forward(tq, tk, tv, 1e-3)
    dq = backward(tg, tq, tk, tv, out, lse, 1e-3)[0]
    t = Truth(q, k, v, 1e-3, None, g)
    for got, want, tol, name, terms in ((out, t.out, t.out_tol, "out", None), (lse, t.lse, t.lse_tol, "lse", None),
                                        (dq, t.dq, t.dq_tol, "dq", t.dq_terms)):
        check(to_host(got), want, tol, name)
        near(to_host(got), want, name, t.s_max, terms)


@pytest.mark.parametrize("size", [(1, 3, 100, 1, 1, 64), (1, 16, 100, 1, 1, 64), (1, 17, 100, 1, 1, 64), (1, 130, 200, 2, 1, 64),
                                  (1, 7, 300, 1, 1, 33), (1, 40, 100, 1, 1, 128), (1, 20, 60, 1, 1, 160)], ids=str)
@pytest.mark.parametrize("qs,ks,vs,gs,scale", [(1e19, 1e19, 1.0, 1.0, 1.25e-38), (1e18, 1e8, 1e-20, 1.0, 1e-27),
                                               (1e-10, 1e-8, 1e18, 1e3, 1e17)])
def test_scales_far_from_1(size, qs, ks, vs, gs, scale):
    """Large or small queries and keys under a scale that makes up for them: neither q k nor scale dS has to be an f32
    for S and the gradients to be.  Where a gradient lies below 2^-126 (dq of 1e-39 in the second case), each of its n
    terms is rounded to a multiple of 2^-149, off by half of that: n 2^-150 of an element besides."""
    f = np.float32
    q, k, v, g = draw(*size, seed=27)
    q, k, v, g = q * f(qs), k * f(ks), v * f(vs), g * f(gs)
    out, _, *grads = both(q, k, v, g, scale, norm=False)
    t = Truth(q, k, v, scale, None, g)
    near(to_host(out), t.out, "out", t.s_max)
    for got, want, n, terms in zip(grads, (t.dq, t.dk, t.dv), (size[2], size[1] * size[3], size[1] * size[3]),
                                   (t.dq_terms, t.dk_terms, np.zeros(()))):
        far = np.linalg.norm(to_host(got) - want)
        norm = np.linalg.norm(want) + np.linalg.norm(terms)
        assert far <= (32 + 4 * t.s_max) * U * norm + np.sqrt(want.size) * n * 2.0**-150, far / norm
