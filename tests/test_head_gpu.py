"""A model's last layer with its loss (trs_linear_cross_entropy,
trs_linear_distillation and their gradients) through the C ABI, against the
definition in 64 bits; tests/_head.py derives the tolerances."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import _head as ref
from _gpu import to_host
from tensorrs_b200 import abi, device

pytestmark = pytest.mark.gpu

V_ = device.view_of


def cuda(a):
    return torch.from_numpy(np.array(a, order="C")).cuda()


class Case:
    """Inputs of one call on the host and on the GPU.  kind: cross entropy with a smoothing, or distillation with K
    entries at a temperature."""

    def __init__(self, N, V, D, kind, masked=0.0, seed=0, spread=2.0, it=np.int64):
        g = np.random.default_rng(seed + 7 * N + V + 31 * D)
        self.N, self.V, self.D, self.kind = N, V, D, kind
        w = (g.standard_normal((V, D)) * spread / np.sqrt(D)).astype(np.float32)
        target = np.minimum((V ** g.random(N)).astype(np.int64), V) - 1
        h = (g.standard_normal((N, D)) + 1.5 / spread * w[target] * 2).astype(np.float32)
        gone = g.random(N) < masked
        h[gone] = np.nan  # a masked row is not read
        self.g = (g.standard_normal(N) / N).astype(np.float32)
        self.g[gone] = np.inf
        if kind[0] == "ce":
            self.s = kind[1]
            t = np.where(gone, g.choice([-1, -100, V, 2**31 - 1], N), target)
            self.ids, self.z, self.T = t.astype(it), None, None
            self.entries, self.share = ref.classes(t, V, self.s), self.s / V
        else:
            K, self.T = kind[1], kind[2]
            ids = (target[:, None] + np.arange(K) ** 2 * 3) % V  # ids come twice in a small vocabulary
            z = (g.standard_normal((N, K)) * 3).astype(np.float32)
            z[g.random((N, K)) < 0.05] = -np.inf
            ids = np.where(g.random((N, K)) < 0.1, g.choice([-1, V, -(2**31)], (N, K)), ids)
            ids[gone] = -1
            self.ids, self.z, self.share = ids.astype(it), z, 0.0
            self.entries = ref.teacher(ids, z, V, self.T)
        self.h, self.w = h, w
        self.d = {"h": cuda(h), "w": cuda(w), "ids": cuda(self.ids), "g": cuda(self.g)}
        if self.z is not None:
            self.d["z"] = cuda(self.z)

    def truth(self, grad=True):
        live = np.array([e is not None for e in self.entries], bool)
        return ref.Truth(np.where(live[:, None], self.h, 0), self.w, self.entries, self.share, self.T, self.g if grad else None)

    def forward(self, loss=None, lse=None, **over):
        d = {k: V_(v) for k, v in self.d.items()} | over
        loss = torch.full((self.N,), np.nan, device="cuda") if loss is None else loss
        lse = torch.full((self.N,), np.nan, device="cuda") if lse is None else lse
        if self.z is None:
            device.linear_cross_entropy(d["h"], d["w"], d["ids"], loss, lse, smoothing=self.s)
        else:
            device.linear_distillation(d["h"], d["w"], d["ids"], d["z"], self.T, loss, lse)
        return loss, lse

    def backward(self, lse, dh="new", dw="new", **over):
        d = {k: V_(v) for k, v in self.d.items()} | over
        dh = torch.full((self.N, self.D), np.nan, device="cuda") if isinstance(dh, str) else dh
        dw = torch.full((self.V, self.D), np.nan, device="cuda") if isinstance(dw, str) else dw
        if self.z is None:
            device.linear_cross_entropy_backward(d["g"], d["h"], d["w"], d["ids"], V_(lse), dh, dw, smoothing=self.s)
        else:
            device.linear_distillation_backward(d["g"], d["h"], d["w"], d["ids"], d["z"], V_(lse), self.T, dh, dw)
        return dh, dw


def check_all(c, t, loss, lse, dh=None, dw=None):
    what = (c.N, c.V, c.D, c.kind)
    ref.check(to_host(loss).ravel(), t.loss, t.loss_tol, ("loss", what))
    ref.check(to_host(lse).ravel(), t.lse, t.lse_tol, ("lse", what))
    ref.near(to_host(loss).ravel(), t.loss, ("loss", what), t.s_max, t.loss_size)
    ref.near(to_host(lse).ravel(), t.lse, ("lse", what), t.s_max, t.lse)
    if dh is not None:
        ref.check(to_host(dh).reshape(t.dh.shape), t.dh, t.dh_tol, ("dh", what))
        ref.near(to_host(dh).reshape(t.dh.shape), t.dh, ("dh", what), t.s_max, t.dh_terms)
    if dw is not None:
        ref.check(to_host(dw), t.dw, t.dw_tol, ("dw", what))
        ref.near(to_host(dw), t.dw, ("dw", what), t.s_max, t.dw_terms)


CE, SMOOTH = ("ce", 0.0), ("ce", 0.1)
KD1, KD7, KD64 = ("kd", 1, 1.0), ("kd", 7, 2.0), ("kd", 64, 1.5)

SIZES = [
    # single rows and few, small and odd vocabularies and widths
    (1, 1, 1, CE, 0.0), (1, 2, 3, KD7, 0.0), (2, 7, 16, SMOOTH, 0.0), (3, 255, 63, KD1, 0.0), (4, 256, 64, CE, 0.0),
    (5, 257, 65, KD64, 0.0), (8, 1000, 130, SMOOTH, 0.3), (8, 5003, 1024, CE, 0.0), (9, 300, 257, KD7, 0.2),
    (16, 2000, 512, CE, 0.2), (16, 513, 100, KD64, 0.0), (1, 70_001, 32, CE, 0.0), (7, 900, 4100, KD7, 0.0),
    (3, 40, 20_000, SMOOTH, 0.0),
    # many rows: tiles, and sizes one off them
    (17, 100, 20, CE, 0.0), (33, 129, 64, SMOOTH, 0.1), (64, 1000, 128, KD7, 0.0), (127, 255, 63, CE, 0.5),
    (128, 256, 64, SMOOTH, 0.0), (129, 257, 65, KD64, 0.1), (255, 511, 192, CE, 0.0), (256, 512, 256, KD1, 0.0),
    (257, 513, 300, CE, 0.9), (300, 2049, 520, SMOOTH, 0.35), (513, 1025, 1024, KD7, 0.1), (700, 10_007, 521, CE, 0.3),
    (1030, 777, 2049, CE, 0.0), (2000, 5000, 40, KD64, 0.2), (40, 30_000, 72, CE, 0.0), (1, 3, 2, ("ce", 1.0), 0.0),
    (50, 64, 16, ("ce", 1.0), 0.2), (20, 100, 24, ("kd", 1024, 3.0), 0.0), (4096, 33, 17, CE, 0.5),
    # few rows in two blocks, of widths that bulk copies take and do not
    (12, 300, 2800, CE, 0.1), (16, 333, 2701, KD7, 0.0), (11, 1000, 36, SMOOTH, 0.2), (13, 500, 35, KD64, 0.0),
    # nothing but masked rows
    (5, 100, 32, CE, 1.0), (300, 400, 48, KD7, 1.0),
]
NAMES = ["x".join(str(x) for x in s) for s in SIZES]


@pytest.mark.parametrize("size", SIZES, ids=NAMES)
def test_values_and_gradients(size):
    N, V, D, kind, masked = size
    c = Case(N, V, D, kind, masked)
    t = c.truth()
    loss, lse = c.forward()
    dh, dw = c.backward(lse)
    check_all(c, t, loss, lse, dh, dw)
    # the same bits again
    loss2, lse2 = c.forward()
    dh2, dw2 = c.backward(lse)
    for a, b in ((loss, loss2), (lse, lse2), (dh, dh2), (dw, dw2)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N", [3, 200])
@pytest.mark.parametrize("kind", [SMOOTH, KD7], ids=["ce", "kd"])
def test_one_gradient_and_no_lse(kind, N):
    """Either gradient alone is the one of both together; the loss does not need lse."""
    c = Case(N, 600, 96, kind, 0.2)
    loss, lse = c.forward()
    dh, dw = c.backward(lse)
    only_h, none = c.backward(lse, dw=None)
    assert none is None and torch.equal(only_h, dh)
    none, only_w = c.backward(lse, dh=None)
    assert none is None and torch.equal(only_w, dw)
    alone = torch.empty_like(loss)
    d = {k: V_(v) for k, v in c.d.items()}
    if c.z is None:
        device.linear_cross_entropy(d["h"], d["w"], d["ids"], alone, smoothing=c.s)
    else:
        device.linear_distillation(d["h"], d["w"], d["ids"], d["z"], c.T, alone)
    assert torch.equal(alone, loss)


@pytest.mark.parametrize("N", [6, 180])
@pytest.mark.parametrize("kind", [CE, KD7], ids=["ce", "kd"])
def test_gradient_against_differences(kind, N):
    """The change of sum g loss along a step of hidden and weight, by central differences of the definition in 64 bits,
    is <grad, step>."""
    c = Case(N, 120, 24, kind)
    _, lse = c.forward()
    dh, dw = (to_host(x).astype(np.float64) for x in c.backward(lse))
    g = np.random.default_rng(4)
    sh, sw = g.standard_normal(c.h.shape), g.standard_normal(c.w.shape)
    e = 1e-5
    f = []
    for k in (-e, e):
        t = ref.Truth(c.h + k * sh, c.w + k * sw, c.entries, c.share, c.T)
        f.append((c.g.astype(np.float64) * t.loss).sum())
    want = (f[1] - f[0]) / (2 * e)
    t = c.truth()
    tol = (t.dh_tol * np.abs(sh)).sum() + (t.dw_tol * np.abs(sw)).sum()
    # the second-order error e^2 / 6 of the third derivative (scores change by less than 20 a unit), and cancellation
    size = (np.abs(c.g) * np.abs(t.loss)).sum()
    assert abs((dh * sh).sum() + (dw * sw).sum() - want) <= tol + e * e * 20.0**3 * np.abs(c.g).sum() + 1e-15 * size / e


@pytest.mark.parametrize("N", [4, 150])
@pytest.mark.parametrize("layout", ["shifted", "transposed", "reversed", "offset", "broadcast"])
def test_strides(layout, N):
    B, V, D = 2, 333, 72
    T = N // B
    for kind in (SMOOTH, KD7):
        c = Case(N, V, D, kind, 0.2, it=np.int32)
        t = c.truth()
        h3, g2 = c.d["h"].view(B, T, D), c.d["g"].view(B, T)
        i3 = c.d["ids"].view(B, T, -1) if c.z is not None else c.d["ids"].view(B, T)
        z3 = c.d["z"].view(B, T, -1) if c.z is not None else None
        keep = []

        def inside(x, lo=1, hi=1, fill=np.nan):  # x as a slice of something larger along its tokens and its last dimension
            shape = list(x.shape)
            shape[1] += lo + hi
            shape[-1] += 8 if x.ndim > 2 else 0
            if x.dtype in (torch.int32, torch.int64):
                fill = 5
            big = torch.full(shape, fill, dtype=x.dtype, device="cuda")
            s = big[:, lo:lo + x.shape[1]]
            s = s[..., 4:-4] if x.ndim > 2 else s
            s.copy_(x)
            keep.append(big)
            return s

        loss, lse, dh = (torch.zeros((B, T, *e), device="cuda") for e in ((), (), (D,)))
        dw = torch.zeros((V, D), device="cuda")
        w = V_(c.d["w"])
        if layout == "shifted":
            args = {"h": V_(inside(h3, 0, 1)), "ids": V_(inside(i3, 1, 0)), "g": V_(inside(g2))}
            if z3 is not None:
                args["z"] = V_(inside(z3))
            loss, lse, dh = inside(loss, fill=7.0), inside(lse, fill=7.0), inside(dh, fill=7.0)
        elif layout == "transposed":  # [in, out] storage, tokens before batch
            wt = c.d["w"].T.contiguous()
            w = V_(wt.T)
            dw = torch.zeros((D, V), device="cuda").T
            hp, ip, gp = h3.transpose(0, 1).contiguous(), i3.transpose(0, 1).contiguous(), g2.T.contiguous()
            args = {"h": V_(hp.transpose(0, 1)), "ids": V_(ip.transpose(0, 1)), "g": V_(gp.T)}
            if z3 is not None:
                zp = z3.permute(2, 1, 0).contiguous()
                args["z"] = V_(zp.permute(2, 1, 0))
            dh = torch.zeros((T, B, D), device="cuda").transpose(0, 1)
            loss, lse = torch.zeros((T, B), device="cuda").T, torch.zeros((T, B), device="cuda").T
        elif layout == "reversed":
            hr, wr = h3.flip(1).contiguous(), c.d["w"].flip(0).contiguous()
            w = device.view_of(wr, [V, D], [-D, 1], (V - 1) * D)
            args = {"h": device.view_of(hr, [B, T, D], [T * D, -D, 1], (T - 1) * D), "ids": V_(i3), "g": V_(g2)}
            if z3 is not None:
                args["z"] = V_(z3)
        elif layout == "offset":  # rows off a 16-byte boundary
            buf = torch.zeros(N * D + 1, device="cuda")
            buf[1:] = h3.flatten()
            wb = torch.zeros(V * D + 3, device="cuda")
            wb[3:] = c.d["w"].flatten()
            w = V_(wb[3:].view(V, D))
            args = {"h": V_(buf[1:].view(B, T, D)), "ids": V_(i3), "g": V_(g2)}
            if z3 is not None:
                args["z"] = V_(z3)
            dh, dw = torch.zeros(N * D + 1, device="cuda")[1:].view(B, T, D), torch.zeros(V * D + 1, device="cuda")[1:].view(V, D)
        else:  # one gradient for all rows
            one = torch.full((1,), 0.25, device="cuda")
            c.g[:] = 0.25
            t = c.truth()
            args = {"h": V_(h3), "ids": V_(i3), "g": V_(one.expand(B, T))}
            if z3 is not None:
                args["z"] = V_(z3)
        c.forward(loss, lse, w=w, **args)
        c.backward(lse, dh, dw, w=w, **args)
        check_all(c, t, loss, lse, dh, dw)
        if layout == "shifted":  # what lies around the outputs is as it was
            for x in (loss, lse, dh):
                x.fill_(7.0)
            for big in keep[-3:]:
                assert bool((big == 7.0).all())


@pytest.mark.parametrize("N", [4, 130])
def test_range(N):
    """Scores of thousands, gradients of very different sizes among the rows, rows and weights of very different sizes."""
    g = np.random.default_rng(8)
    for kind in (CE, KD7):
        c = Case(N, 400, 64, kind, spread=2.0)
        c.h *= np.float32(300.0)
        c.g = (10.0 ** g.uniform(-20, 3, N)).astype(np.float32)
        c.g[N // 2] = 0
        c.d["h"], c.d["g"] = cuda(c.h), cuda(c.g)
        t = c.truth()
        loss, lse = c.forward()
        check_all(c, t, loss, lse, *c.backward(lse))
        # every row of dh is near its own truth, whatever the others' gradients are
        dh, _ = c.backward(lse)
        for i in range(N):
            ref.near(to_host(dh)[i], t.dh[i], ("row", i), t.s_max, t.dh_terms[i])
        c = Case(N, 400, 64, kind)
        c.h *= (10.0 ** g.uniform(-12, 0, (N, 1))).astype(np.float32)
        c.w *= (10.0 ** g.uniform(-6, 0.5, (400, 1))).astype(np.float32)
        c.h *= np.float32(1e15)
        c.w *= np.float32(1e-15)
        c.d["h"], c.d["w"] = cuda(c.h), cuda(c.w)
        t = c.truth()
        loss, lse = c.forward()
        check_all(c, t, loss, lse, *c.backward(lse))


LARGE = [(("kd", 7, 2.0**-40), 1), (("kd", 7, 2.0**-20), 1), (("kd", 3, 2.0**-10), 1e-5), (CE, 1e6), (CE, 1e9), (SMOOTH, 1e12),
         (("ce", 1.0), 1e30)]


@pytest.mark.parametrize("N", [4, 20, 130])
@pytest.mark.parametrize("kind,size", LARGE)
def test_scores_of_any_size(kind, size, N):
    """Scores whose last bit is worth more than the exponential's whole range."""
    for seed in range(3):
        c = Case(N, 700, 48, kind, 0.2, seed=seed)
        c.h *= np.float32(size)
        c.d["h"] = cuda(c.h)
        t = c.truth()
        loss, lse = c.forward()
        ref.check(to_host(loss), t.loss, t.loss_tol, ("loss", size))
        ref.check(to_host(lse), t.lse, t.lse_tol, ("lse", size))


@pytest.mark.parametrize("N", [4, 12, 20, 130])
@pytest.mark.parametrize("kind,size", LARGE)
def test_gradients_of_scores_of_any_size(kind, size, N):
    """A softmax taken from an lse that is rounded to f32 lies between 0 and 1, also where the rounding leaves nothing
    of it to compare."""
    for seed in range(3):
        c = Case(N, 700, 48, kind, 0.2, seed=seed)
        c.h *= np.float32(size)
        c.d["h"] = cuda(c.h)
        _, lse = c.forward()
        dh, dw = (to_host(x).astype(np.float64) for x in c.backward(lse))
        live = np.array([e is not None for e in c.entries], bool)
        g = np.where(live, np.abs(c.g.astype(np.float64)), 0)[:, None] * (1.0 if c.T is None else c.T)
        h, w = np.where(live[:, None], np.abs(c.h.astype(np.float64)), 0), np.abs(c.w.astype(np.float64))
        # every element of softmax - t lies in [-1, 1]; 2^-10 for all roundings
        assert (np.abs(dh) <= g * w.sum(0) * (1 + 2.0**-10) + 1e-37).all()
        assert (np.abs(dw) <= (g * h).sum(0) * (1 + 2.0**-10) + 1e-37).all()


@pytest.mark.parametrize("N", [4, 130])
def test_infinities_stay_in_their_rows(N):
    for bad in (np.inf, np.nan):
        c = Case(N, 300, 48, CE)
        t = c.truth()
        c.d["h"][2, 5] = bad
        loss, lse = c.forward()
        assert not np.isfinite(to_host(loss)[2])
        for got, want, tol in ((loss, t.loss, t.loss_tol), (lse, t.lse, t.lse_tol)):
            ref.check(np.delete(to_host(got), 2), np.delete(want, 2), np.delete(tol, 2), bad)
        dh, dw = c.backward(lse)
        assert not np.isfinite(to_host(dh)[2]).any()
        ref.check(np.delete(to_host(dh), 2, 0), np.delete(t.dh, 2, 0), np.delete(t.dh_tol, 2, 0), bad)
        assert not np.isfinite(to_host(dw)).all()
        # the row masked: nothing of it is left
        c.d["ids"][2] = -1
        c.entries[2] = None
        t = c.truth()
        loss, lse = c.forward()
        check_all(c, t, loss, lse, *c.backward(lse))


@pytest.mark.parametrize("N", [4, 12, 130])
@pytest.mark.parametrize("kind", [CE, KD1], ids=["ce", "kd"])
def test_gradients_of_improbable_tokens(kind, N):
    """Rows of grad_weight whose tokens no row finds likely.  softmax(x) - t in two fp16 parts under 2^15 is off by half of
    the smallest fp16 number, 2^-25 / 2^15 = 2^-40, where it is below 2^-17; few rows' kernels keep 22 bits of it."""
    V, D = 300, 32
    c = Case(N, V, D, kind)
    # logarithms of the tokens' probabilities from 0 to -31: 2^-45
    c.h[:, 0], c.w[:, 0] = 8.0, -np.linspace(0, 31 / 8, V)
    c.d["h"], c.d["w"] = cuda(c.h), cuda(c.w)
    t = c.truth()
    loss, lse = c.forward()
    dh, dw = c.backward(lse)
    check_all(c, t, loss, lse, dh, dw)
    # dw's bound of tests/_head.py, with 2^-40 (or nothing) in place of its 2^-38 of softmax(x) - t
    h, w, g = c.h.astype(np.float64), c.w.astype(np.float64), np.abs(c.g.astype(np.float64))[:, None]
    g[[e is None for e in c.entries]] = 0  # masked
    x = h @ w.T
    P = np.exp(x - t.lse[:, None])
    target = np.zeros((N, V))
    for i, e in enumerate(c.entries):
        for v, p in e or []:
            target[i, v] += p
    sx = (160 + D / 64) * ref.U * (np.abs(h) @ np.abs(w).T) + 2.0**-38 * D * np.abs(h).max(-1, keepdims=True) * np.abs(w).max()
    sx += 4 * ref.U * np.abs(x)
    E = 2 * sx.max(-1) + (8 * np.abs(x).max(-1) + 8 * np.abs(t.lse) + 300 + V / 32) * ref.U
    err = g * (P * E[:, None] + 60 * ref.U * target + 8 * ref.U * np.abs(P - target))
    if N > 16:
        err = err + g * 2.0**-40
    dx = g * np.abs(P - target)
    tol = err.T @ np.abs(h) + (160 + N / 64) * ref.U * (dx.T @ np.abs(h))
    tol += 2.0**-38 * (g * np.abs(h)).max() * (P + target).sum(0)[:, None]
    ref.check(to_host(dw), t.dw, tol, ("dw", N))
    if N <= 16:  # the least likely ones have a gradient
        assert np.abs(to_host(dw))[-1].max() > 0


@pytest.mark.parametrize("N", [4, 17, 130])
@pytest.mark.parametrize("kind", [CE, KD7], ids=["ce", "kd"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_bad_weight_rows(bad, kind, N):
    """A row of the vocabulary that is no longer a number, wherever it lies and whoever's target it is, shows in the loss
    and lse of every token (f32: 0 inf and inf - inf are NaN), and in no masked one."""
    for V in (300, 10_007):
        c = Case(N, V, 48, kind, 0.2)
        live = np.array([e is not None for e in c.entries], bool)
        for rows in ([0], [V // 2], [V - 1], [0, 1, 2], [0, V // 3, V - 1]):
            w = c.d["w"].clone()
            w[rows, 7] = bad
            loss, lse = (to_host(x) for x in c.forward(w=V_(w)))
            assert not np.isfinite(loss[live]).any() and not np.isfinite(lse[live]).any(), (V, rows)
            assert not loss[~live].any() and not lse[~live].any()
        w = torch.full_like(c.d["w"], bad)  # nothing else
        loss, lse = (to_host(x) for x in c.forward(w=V_(w)))
        assert not np.isfinite(loss[live]).any() and not np.isfinite(lse[live]).any()


@pytest.mark.parametrize("N", [4, 130])
@pytest.mark.parametrize("temperature", [0.5, 2.0**-10, 3.0])
@pytest.mark.parametrize("low", [-np.finfo(np.float32).max, -1e30])
def test_lowest_teacher_logits(low, temperature, N):
    """Entries masked by a logit far below the others have no share, also where its quotient by the temperature is no f32;
    where a row has no others they share alike."""
    c = Case(N, 300, 48, ("kd", 9, temperature))
    c.z[:, 2::3] = low
    c.z[1, :] = low
    c.z[3, 1:] = low
    c.entries = ref.teacher(c.ids, c.z, 300, temperature)
    c.d["z"] = cuda(c.z)
    t = c.truth()
    loss, lse = c.forward()
    assert np.isfinite(to_host(loss)).all()
    check_all(c, t, loss, lse, *c.backward(lse))


def test_large_vocabulary():
    """140000 tokens, and the weight as a view past 2^31 elements."""
    N, V, D = 300, 140_000, 64
    c = Case(N, V, D, SMOOTH, 0.1)
    t = c.truth()
    loss, lse = c.forward()
    check_all(c, t, loss, lse, *c.backward(lse))
    pitch = 1 << 15  # 140000 rows of 32768 floats: offsets past 2^32
    big = torch.zeros((V, pitch), device="cuda")
    big[:, 64:64 + D] = c.d["w"]
    loss2, lse2 = c.forward(w=V_(big[:, 64:64 + D]))
    assert torch.equal(loss, loss2) and torch.equal(lse, lse2)


def test_pieces_of_the_vocabulary():
    """A weight that either direction takes in several pieces, the last one not whole; the definition in 64 bits on the
    GPU, in the 2-norm."""
    N, V, D = 300, 40_100, 4000
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn((V, D), generator=g, device="cuda") * (2 / D**0.5)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    h = torch.randn((N, D), generator=g, device="cuda") + w[t]
    gl = torch.rand((N,), generator=g, device="cuda")
    loss, lse = torch.empty((N,), device="cuda"), torch.empty((N,), device="cuda")
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    device.linear_cross_entropy(V_(h), V_(w), V_(t), loss, lse)
    device.linear_cross_entropy_backward(V_(gl), V_(h), V_(w), V_(t), V_(lse), dh, dw)
    x = h.double() @ w.double().T
    want_lse = torch.logsumexp(x, -1)
    p = torch.exp(x - want_lse[:, None])
    s_max = float(torch.maximum(x.abs().max(), want_lse.abs().max()))
    here = torch.arange(N, device="cuda")
    want = want_lse - x[here, t]
    both = p.clone()
    both[here, t] += 1
    both *= gl.double()[:, None]
    p[here, t] -= 1
    p *= gl.double()[:, None]
    ref.near(to_host(lse), to_host(want_lse), "lse", s_max, to_host(want_lse))
    ref.near(to_host(loss), to_host(want), "loss", s_max, to_host(want_lse))
    ref.near(to_host(dh), to_host(p @ w.double()), "dh", s_max, to_host(((both * both) @ w.double().square()).sqrt()))
    ref.near(to_host(dw), to_host(p.T @ h.double()), "dw", s_max, to_host(((both * both).T @ h.double().square()).sqrt()))


def test_streams_and_graphs():
    """Two streams at once, a captured step replayed on new inputs, graphs that run at the same time."""
    cases = [Case(150, 700, 80, KD7, 0.1, seed=s) for s in (1, 2)] + [Case(6, 700, 80, SMOOTH, 0.1, seed=3)]
    want = []
    for c in cases:
        loss, lse = c.forward()
        want.append((loss, lse, *c.backward(lse)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for st, c in zip(streams, cases):
            with torch.cuda.stream(st):
                loss, lse = c.forward()
                got.append((loss, lse, *c.backward(lse)))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [], []
    for c in cases:
        out = [torch.empty_like(x) for x in want[0][:2]] if c.N == 150 else [torch.empty((6,), device="cuda") for _ in range(2)]
        out += [torch.empty((c.N, 80), device="cuda"), torch.empty((700, 80), device="cuda")]
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            c.forward(out[0], out[1])
            c.backward(out[1], out[2], out[3])
        graphs.append(gr)
        outs.append(out)
    for _ in range(3):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for k in ("h", "w", "ids", "g", "z"):
        cases[0].d[k].copy_(cases[1].d[k])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs[0], want[1]))


def test_threads_on_one_stream():
    """Host threads that issue whole steps on one stream, in whatever order: bit for bit the results of one thread.  The
    vocabulary leaves SMs free, so that kernels of both can run at once."""
    import threading

    cases = [Case(200, 900, 320, KD7, 0.1, seed=1), Case(150, 700, 200, SMOOTH, 0.2, seed=2), Case(6, 700, 80, KD7, 0.1, seed=3)]
    want = []
    for c in cases:
        loss, lse = c.forward()
        want.append((loss, lse, *c.backward(lse)))
    torch.cuda.synchronize()
    steps, stream = 60, torch.cuda.Stream()
    got = [[[torch.full_like(x, np.nan) for x in w] for _ in range(steps)] for w in want]
    torch.cuda.synchronize()
    start, failed = threading.Barrier(len(cases)), []

    def work(c, outs):
        try:
            with torch.cuda.stream(stream):
                start.wait(60)
                for loss, lse, dh, dw in outs:
                    c.forward(loss, lse)
                    c.backward(lse, dh, dw)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, got)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for w, outs in zip(want, got):
        for i, out in enumerate(outs):
            for k, (a, b) in enumerate(zip(out, w)):
                assert torch.equal(a, b), (i, k)


@pytest.mark.parametrize("N", [4, 30, 150, 700])
@pytest.mark.parametrize("kind", [SMOOTH, KD7], ids=["ce", "kd"])
def test_a_weight_from_the_call_before(kind, N):
    """Each call's weight is what the call before it has just written: bit for bit the results of calls one at a time."""
    c = Case(N, 5000, 192, kind, masked=0.2)
    runs = []
    for wait in (True, False):
        w = V_(c.d["w"])
        shapes = [(N,), (N,), (N, c.D), (c.V, c.D)] * 6  # all there before the first call: nothing runs between the calls
        out = [torch.full(s, np.nan, device="cuda") for s in shapes]
        for i in range(0, len(out), 4):
            c.forward(*out[i : i + 2], w=w)
            if wait:
                torch.cuda.synchronize()
            c.backward(out[i + 1], *out[i + 2 : i + 4], w=w)
            if wait:
                torch.cuda.synchronize()
            w = V_(out[i + 3])
        runs.append([to_host(x) for x in out])
    for i, (a, b) in enumerate(zip(*runs)):
        np.testing.assert_array_equal(a, b, err_msg=f"result {i}")


def test_a_step_of_a_tied_model():
    """Embedding, the last layer on the same table, both gradients added up, one Adam step: a model of one table, against
    the same steps in 64 bits."""
    g = np.random.default_rng(3)
    B, T, V, D = 4, 60, 500, 64
    ids = g.integers(0, V, (B, T + 1))
    ids[1, 40:] = -100
    table = (g.standard_normal((V, D)) * 0.5).astype(np.float32)
    dt, di = cuda(table), cuda(ids)
    x = torch.empty((B, T, D), device="cuda")
    device.embedding(V_(dt), V_(di[:, :-1]), np.sqrt(D), x)
    loss, lse = torch.empty((B, T), device="cuda"), torch.empty((B, T), device="cuda")
    targets = V_(di[:, 1:])
    device.linear_cross_entropy(V_(x), V_(dt), targets, loss, lse)
    count = (ids[:, 1:] >= 0).sum()
    gl = torch.full((1, 1), 1.0 / count, device="cuda").expand(B, T)
    dx, gt = torch.empty_like(x), torch.empty_like(dt)
    device.linear_cross_entropy_backward(V_(gl), V_(x), V_(dt), targets, V_(lse), dx, gt)
    device.embedding_backward(V_(dx), V_(di[:, :-1]), np.sqrt(D), gt, accumulate=True)
    # the definition, one stage at a time on what the calls before it gave
    xs, tok = to_host(x).reshape(-1, D), ids[:, 1:].ravel()
    t = ref.Truth(xs, table, ref.classes(tok, V, 0.0), 0.0, None, np.full(B * T, np.float32(1.0 / count)))
    ref.check(to_host(loss).ravel(), t.loss, t.loss_tol, "loss")
    ref.check(to_host(dx).reshape(-1, D), t.dh, t.dh_tol, "dx")
    src = ids[:, :-1].ravel()
    want, size = t.dw.copy(), np.abs(t.dw)
    d64 = to_host(dx).reshape(-1, D).astype(np.float64) * np.sqrt(D)
    np.add.at(want, src[src >= 0], d64[src >= 0])
    np.add.at(size, src[src >= 0], np.abs(d64[src >= 0]))
    ref.check(to_host(gt), want, t.dw_tol + 4 * ref.U * size, "the table's gradient")
    m, v = torch.zeros_like(dt), torch.zeros_like(dt)
    grad = to_host(gt).astype(np.float64)
    device.adam_step(dt, gt, m, v, 1e-2, 1)
    step = 1e-2 * grad / (np.abs(grad) + 1e-8)
    assert np.abs(to_host(dt) - (table - step)).max() <= 1e-2 * 2.0**-18 + 2.0**-23 * np.abs(table).max()


def test_no_tokens():
    """Without tokens the gradient of the weight is zero."""
    dw = torch.full((50, 8), np.nan, device="cuda")
    z = torch.empty((0, 8), device="cuda")
    e, w, ids = torch.empty((0,), device="cuda"), torch.ones((50, 8), device="cuda"), torch.empty((0,), dtype=torch.int64, device="cuda")
    device.linear_cross_entropy_backward(V_(e), V_(z), V_(w), V_(ids), V_(e), torch.empty_like(z), dw)
    assert not bool(to_host(dw).any())


def test_no_async_error():
    import ctypes

    code = ctypes.c_int32(-1)
    assert abi.load().trs_async_error(ctypes.byref(code)) == abi.OK and code.value == 0
