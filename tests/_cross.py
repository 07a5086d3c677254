"""The definition of cross attention and of its gradients in 64 bits, with the
bounds that the tests hold f32 results to.

u = 2^-24.  Every product of two operands is off by less than 12 u of itself
(two 22-bit operands and the dropped product of their low parts; the CUDA-core
path: 1 u) and a sum of D of them inside the tensor core by less than 64 u of
the terms (at most 24 additions in a chain, each cut by 2^-23, and 16 products
inside each): 80 u together, sp = 80 u sum_d |q_d k_d|.  The score's factors
round 6 times, the exponential is off by 2 units and its argument by u of
itself: P of row i is off by less than
    E_i = 2 max_j sp_ij scale + (6 max_j |S_ij| + 6 |lse_i| + 300 + Tk / 32) u
relative to itself (the row's sum: 64 terms in a chain per tile, one per tile
after that).  Sums over keys or rows then add 100 u + (length / 32) u of their
terms, and every operand 2^-40 of its tile's largest magnitude, 2^-38 of the
operand's with the other factor at its largest."""
from __future__ import annotations

import numpy as np

U = 2.0**-24


class Truth:
    """q [B, Tq, Hq, D], k, v [B, Tk, Hk, D] (any float type), lengths [B] or None, grad like q."""

    def __init__(self, q, k, v, scale, lengths=None, grad=None):
        B, Tq, Hq, D = q.shape
        Tk, Hk = k.shape[1:3]
        self.out, self.out_tol = np.zeros(q.shape), np.zeros(q.shape)
        self.lse, self.lse_tol = np.full((B, Hq, Tq), -np.inf), np.zeros((B, Hq, Tq))
        self.dq, self.dq_tol = np.zeros(q.shape), np.zeros(q.shape)
        self.dk, self.dk_tol = np.zeros(k.shape), np.zeros(k.shape)
        self.dv, self.dv_tol = np.zeros(k.shape), np.zeros(k.shape)
        self.dq_terms, self.dk_terms = np.zeros(q.shape), np.zeros(k.shape)
        q, k, v = (x.astype(np.float64) for x in (q, k, v))
        self.s_max = 0.0
        for b in range(B):
            n = Tk if lengths is None else int(min(max(lengths[b], 0), Tk))
            if n == 0:
                continue
            for h in range(Hq):
                j = h // (Hq // Hk)
                self._head(b, h, j, n, q[b, :, h], k[b, :n, j], v[b, :n, j], scale,
                           None if grad is None else grad[b, :, h].astype(np.float64))

    def _head(self, b, h, j, n, q, k, v, scale, g):
        S = scale * q @ k.T
        self.s_max = max(self.s_max, np.abs(S).max(initial=0.0))
        m = S.max(-1, keepdims=True)
        e = np.exp(S - m)
        l = e.sum(-1, keepdims=True)
        P, lse = e / l, (m + np.log(l))[:, 0]
        out = P @ v
        aq, ak, av = np.abs(q), np.abs(k), np.abs(v)
        D = q.shape[1]
        fl = 2.0**-38 * D
        sp = abs(scale) * (80 * U * (aq @ ak.T) + fl * aq.max(initial=0) * ak.max(initial=0))
        E = (2 * sp.max(-1) + (6 * np.abs(S).max(-1) + 6 * np.abs(lse) + 300 + n / 32) * U)[:, None]
        sums = (100 + n / 32) * U
        out_tol = (2 * E + sums) * (P @ av) + 2.0**-38 * av.max()
        self.out[b, :, h], self.out_tol[b, :, h] = out, out_tol
        self.lse[b, h], self.lse_tol[b, h] = lse, 2 * E[:, 0]
        if g is None:
            return
        ag = np.abs(g)
        delta = (g * out).sum(-1, keepdims=True)
        dP = g @ v.T
        dS = P * (dP - delta)
        e_dp = 80 * U * (ag @ av.T) + fl * ag.max(initial=0) * av.max()
        e_delta = (ag * (out_tol + 80 * U * np.abs(out))).sum(-1, keepdims=True)
        # dS is carried in 22 bits under a bound of its row: 2^-38 of that
        reach = np.sqrt((g * g).sum(-1)).max(initial=0) * np.sqrt((v * v).sum(-1)).max() + np.abs(delta).max(initial=0)
        T = P * (E * (np.abs(dP) + np.abs(delta)) + e_dp + e_delta) + 16 * U * np.abs(dS) + 2.0**-38 * reach
        whole = (P * (np.abs(dP) + np.abs(delta))) ** 2
        self.dq_terms[b, :, h] = abs(scale) * np.sqrt(whole @ (k * k))
        self.dk_terms[b, :n, j] = np.hypot(self.dk_terms[b, :n, j], abs(scale) * np.sqrt(whole.T @ (q * q)))
        rows = (100 + len(q) / 32 + n / 32) * U
        self.dq[b, :, h] = scale * dS @ k
        self.dq_tol[b, :, h] = abs(scale) * (T @ (ak + 2.0**-38 * ak.max()) + rows * np.abs(dS) @ ak)
        self.dk[b, :n, j] += scale * dS.T @ q
        self.dk_tol[b, :n, j] += abs(scale) * (T.T @ (aq + 2.0**-38 * aq.max()) + rows * np.abs(dS).T @ aq)
        self.dv[b, :n, j] += P.T @ g
        self.dv_tol[b, :n, j] += (P * E).T @ ag + rows * P.T @ ag + 2.0**-38 * ag.max() * len(q)


def check(got, want, tol, what):
    got = np.asarray(got, np.float64)
    live = np.isfinite(want)
    assert np.array_equal(got[~live], want[~live]), what
    err = np.abs(got[live] - want[live])
    bad = ~(err <= tol[live] + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), bad.size, float(np.max(err / (tol[live] + 1e-37))))


def near(got, want, what, s_max, terms=None):
    """The errors of the elements are independent: in the 2-norm they stay within 32 u of the result, and within 4 u
    more for each unit of the scores, since P = exp(S - lse) takes over what S and lse are rounded by: three times u of
    S, twice u of lse (a score of 60 is off by 60 u from one rounding alone).  A gradient's dS
    is the difference of dP and delta, each rounded before: `terms` are its products with both in full, added as
    independent errors are (with a single key dS is 0, and what is left of both is all there is)."""
    live = np.isfinite(want)
    norm = np.linalg.norm(want[live]) + (0.0 if terms is None else np.linalg.norm(terms))
    far = np.linalg.norm(np.asarray(got, np.float64)[live] - want[live])
    assert far <= (32 + 4 * s_max) * U * norm, (what, far / norm)
