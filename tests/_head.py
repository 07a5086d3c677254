"""The definition of a model's last layer with its loss in 64 bits (cross entropy
against classes, distillation from a teacher's entries), with the bounds that the
tests hold f32 results to.

u = 2^-24.  A product of two operands is off by less than 12 u of itself (two
22-bit parts and the dropped product of the low parts; the CUDA-core path: 1 u).
A sum leaves the tensor core every 256 elements: 48 additions in a chain, each cut
by 2^-23, with 16 products inside each, less than 144 u of its terms; what left is
added in f32, one addition per 256: with the products (160 + n / 64) u for a sum of
n.  Elements are held to 2^-40 of the largest of their row (hidden), of their piece
of the weight, or of all g h: 2^-38 with the other factor at its largest.

A score x of row i is off by sx = ((160 + D / 64) u sum |h w| + 2^-38 D max|h_i|
max|w|) / temperature + 4 u |x|; lse by the largest of those, its own sum (128 terms
in a chain per part, a part per chain of 8 after that: (300 + V / 32) u) and 4 u of
itself.  softmax(x) is off by
    E_i = 2 max_j sx_ij + (8 max_j |x_ij| + 8 |lse_i| + 300 + V / 32) u
relative to itself; the teacher's p by 40 u.  Sums over the vocabulary or the rows
then add (160 + n / 64) u of their terms."""
from __future__ import annotations

import numpy as np

U = 2.0**-24


class Truth:
    """h [N, D], w [V, D], ids and weights of the entries as lists per row (None: masked), share s / V of every
    token, temperature T, g [N] or None."""

    def __init__(self, h, w, entries, share, T, g=None):
        N, D = h.shape
        V = len(w)
        h, w = h.astype(np.float64), w.astype(np.float64)
        self.live = np.array([e is not None for e in entries], bool)
        self.loss, self.loss_tol = np.zeros(N), np.zeros(N)
        self.lse, self.lse_tol = np.zeros(N), np.zeros(N)
        self.dh, self.dh_tol, self.dh_terms = np.zeros((N, D)), np.zeros((N, D)), np.zeros((N, D))
        self.dw, self.dw_tol, self.dw_terms = np.zeros((V, D)), np.zeros((V, D)), np.zeros((V, D))
        self.s_max = 0.0
        self.loss_size = np.zeros(N)
        rows = np.flatnonzero(self.live)
        if len(rows) == 0:
            return
        h = h[rows]
        n = len(rows)
        t = np.full((n, V), share)
        ent, ent_size = np.zeros(n), np.zeros(n)
        for i, r in enumerate(rows):
            for v, p in entries[r]:
                t[i, v] += p
                if T is not None and p > 0:
                    ent[i] += p * np.log(p)
                    ent_size[i] += abs(p * np.log(p))
        temp = 1.0 if T is None else T
        x = h @ w.T / temp
        top = x.max(-1, keepdims=True)
        e = np.exp(x - top)
        l = e.sum(-1, keepdims=True)
        P, lse = e / l, (top + np.log(l))[:, 0]
        ah, aw = np.abs(h), np.abs(w)
        sums = lambda k: (160 + k / 64) * U  # noqa: E731
        sx = (sums(D) * (ah @ aw.T) + 2.0**-38 * D * ah.max(-1, keepdims=True) * aw.max()) / temp + 4 * U * np.abs(x)
        self.s_max = max(np.abs(x).max(), np.abs(lse).max())
        own = (300 + V / 32) * U
        self.lse[rows], self.lse_tol[rows] = lse, sx.max(-1) + own + 4 * U * np.abs(lse)
        size = np.abs(lse) + (t * np.abs(x)).sum(-1) + ent_size
        self.loss[rows] = temp**2 * (ent + (t * (lse[:, None] - x)).sum(-1))
        self.loss_size[rows] = temp**2 * size
        self.loss_tol[rows] = temp**2 * (self.lse_tol[rows] + (t * sx).sum(-1) + (60 * U + own) * size)
        if g is None:
            return
        g = g.astype(np.float64)[rows][:, None] * temp
        E = (2 * sx.max(-1) + (8 * np.abs(x).max(-1) + 8 * np.abs(lse)) * U + own)[:, None]
        dx = g * (P - t)
        err = np.abs(g) * (P * E + 60 * U * t + 8 * U * np.abs(P - t) + 2.0**-38)
        whole = (np.abs(g) * (P + t)) ** 2
        self.dh[rows] = dx @ w
        self.dh_tol[rows] = err @ aw + (sums(V) * np.abs(dx)) @ aw + 2.0**-38 * aw.max() * np.abs(dx).sum(-1, keepdims=True)
        self.dh_terms[rows] = np.sqrt(whole @ (w * w))
        self.dw = dx.T @ h
        gh = np.abs(g) * ah
        self.dw_tol = err.T @ ah + (sums(n) * np.abs(dx)).T @ ah + 2.0**-38 * gh.max() * (P + t).sum(0)[:, None]
        self.dw_terms = np.sqrt(whole.T @ (h * h))


def teacher(ids, z, V, T):
    """Entries of each row from the teacher's ids and logits [N, K]."""
    out = []
    for i in range(len(ids)):
        k = [j for j in range(ids.shape[1]) if 0 <= ids[i, j] < V and z[i, j] != -np.inf]
        if not k:
            out.append(None)
            continue
        a = z[i, k].astype(np.float64) / T
        p = np.exp(a - a.max())
        out.append(list(zip((int(ids[i, j]) for j in k), p / p.sum())))
    return out


def classes(targets, V, smoothing):
    return [[(int(t), 1.0 - smoothing)] if 0 <= t < V else None for t in targets]


def check(got, want, tol, what):
    got = np.asarray(got, np.float64)
    bad = ~(np.abs(got - want) <= tol + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), bad.size, float(np.max(np.abs(got - want) / (tol + 1e-37))))


def near(got, want, what, s_max, terms):
    """The errors of the elements are independent but for a row's lse: in the 2-norm they stay within 32 u, and within 4 u
    more for each unit of the scores (the exponential takes over what x and lse are rounded by: three times u of x, once u
    of lse), of `terms`, the products of softmax and target in full, and of the result."""
    norm = np.linalg.norm(want) + np.linalg.norm(terms)
    far = np.linalg.norm(np.asarray(got, np.float64) - want)
    assert far <= (32 + 4 * s_max) * U * norm + 1e-37, (what, far / norm)
