"""trs_cross_attention and its gradient through the C ABI against the
definition in 64 bits (tests/_cross.py holds the bounds and their reasons)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _cross import Truth, check, near
from _gpu import to_host

pytestmark = pytest.mark.gpu


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def draw(B, Tq, Tk, Hq, Hk, D, seed=0, grad=True):
    g = np.random.default_rng(seed)
    f = np.float32
    return (g.standard_normal((B, Tq, Hq, D)).astype(f), g.standard_normal((B, Tk, Hk, D)).astype(f),
            g.standard_normal((B, Tk, Hk, D)).astype(f), g.standard_normal((B, Tq, Hq, D)).astype(f) if grad else None)


def forward(q, k, v, scale, n=None, lse=True):
    from tensorrs_b200 import device
    V = device.view_of
    out = torch.full(q.shape, float("nan"), device="cuda")
    ls = torch.full((q.shape[0], q.shape[2], q.shape[1]), float("nan"), device="cuda") if lse else None
    device.cross_attention(V(q), V(k), V(v), scale, out, lse=ls, key_lengths=V(n) if n is not None else None)
    return out, ls


def backward(g, q, k, v, out, lse, scale, n=None):
    from tensorrs_b200 import device
    V = device.view_of
    dq, dk, dv = (torch.full(x.shape, float("nan"), device="cuda") for x in (q, k, v))
    device.cross_attention_backward(V(g), V(q), V(k), V(v), V(out), V(lse), scale, dq, dk, dv,
                                    key_lengths=V(n) if n is not None else None)
    return dq, dk, dv


def both(q, k, v, g, scale, lengths=None, dev=None, norm=True):
    """Forward and backward of host arrays (`dev`: device tensors holding the same values) against the truth."""
    tq, tk, tv, tg = dev or (cuda(q), cuda(k), cuda(v), cuda(g))
    n = None if lengths is None else cuda(lengths)
    out, lse = forward(tq, tk, tv, scale, n)
    t = Truth(q, k, v, scale, lengths, g)
    check(to_host(out), t.out, t.out_tol, "out")
    check(to_host(lse), t.lse, t.lse_tol, "lse")
    dq, dk, dv = backward(tg, tq, tk, tv, out, lse, scale, n)
    for name, got, want, tol, terms in (("dq", dq, t.dq, t.dq_tol, t.dq_terms), ("dk", dk, t.dk, t.dk_tol, t.dk_terms),
                                        ("dv", dv, t.dv, t.dv_tol, None)):
        check(to_host(got), want, tol, name)
        if norm:
            near(to_host(got), want, name, t.s_max, terms)
    if norm:
        near(to_host(out), t.out, "out", t.s_max)
    return out, lse, dq, dk, dv


# B, Tq, Tk, Hq, Hk, D
SIZES = [
    (1, 128, 128, 1, 1, 64), (1, 1, 1, 1, 1, 64), (2, 1, 7, 3, 3, 64), (1, 3, 300, 4, 2, 64), (2, 17, 130, 2, 2, 64),
    (1, 130, 129, 2, 1, 64), (1, 257, 65, 1, 1, 64), (2, 100, 300, 4, 4, 33), (1, 33, 5, 6, 2, 16), (3, 20, 1, 2, 1, 64),
    (1, 64, 64, 1, 1, 128), (1, 128, 63, 2, 2, 128), (2, 130, 129, 2, 1, 128), (1, 300, 200, 1, 1, 80), (1, 40, 333, 7, 1, 96),
    (1, 19, 257, 1, 1, 7), (1, 5, 70, 2, 2, 160), (1, 20, 33, 2, 1, 256), (1, 1, 1, 1, 1, 1), (1, 16, 2, 1, 1, 130),
    (1, 1, 1500, 8, 1, 64), (1, 2, 1000, 8, 1, 128), (2, 512, 512, 2, 2, 64), (1, 513, 260, 2, 1, 100),
    (1, 300, 300, 1, 1, 96), (1, 300, 300, 1, 1, 97), (1, 40, 2000, 1, 1, 72), (1, 1500, 40, 1, 1, 96), (2, 200, 150, 3, 1, 65),
    (2, 1, 500, 7, 1, 32), (1, 2, 300, 8, 2, 24), (2, 1, 700, 2, 2, 32), (1, 1, 64, 4, 1, 17),
]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_64_bits(size):
    q, k, v, g = draw(*size, seed=sum(size))
    both(q, k, v, g, size[-1] ** -0.5)


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
@pytest.mark.parametrize("size,lengths", [
    ((4, 130, 200, 2, 2, 64), [0, 1, 200, 65]), ((4, 40, 300, 4, 2, 128), [128, 0, 63, 300]),
    ((4, 2, 300, 4, 2, 64), [0, 1, 300, 257]), ((3, 5, 70, 2, 1, 200), [70, 0, 33]), ((3, 64, 128, 1, 1, 64), [-5, 1000, 64]),
    ((2, 300, 100, 1, 1, 80), [0, 0]), ((5, 300, 700, 6, 2, 64), [700, 0, 3, 128, 513]),
    ((6, 200, 900, 4, 4, 128), [0, 900, 0, 1, 449, 0]), ((40, 20, 70, 1, 1, 64), [(7 * i) % 71 for i in range(40)]),
], ids=str)
def test_key_lengths_and_what_lies_behind_them(size, lengths, dtype):
    q, k, v, g = draw(*size, seed=3)
    n = np.array(lengths, dtype)
    for b, m in enumerate(lengths):  # never read
        for x in (k, v):
            x[b, max(m, 0):] = np.nan if b % 2 else np.inf
    out, lse, dq, dk, dv = both(q, k, v, g, 0.125, n)
    for b, m in enumerate(lengths):
        if m <= 0:
            assert (out[b] == 0).all() and (lse[b] == -np.inf).all() and (dq[b] == 0).all()
        assert (dk[b, max(m, 0):] == 0).all() and (dv[b, max(m, 0):] == 0).all()


@pytest.mark.parametrize("size", [(1, 64, 5000, 1, 1, 64), (1, 30, 3000, 2, 1, 128), (1, 3000, 64, 1, 1, 64),
                                  (1, 2, 9000, 2, 2, 64), (1, 1100, 300, 1, 1, 128)], ids=str)
def test_long_walks_split_over_the_sms(size):
    q, k, v, g = draw(*size, seed=5)
    both(q, k, v, g, 0.2, np.array([size[2] - 3]))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.5])
@pytest.mark.parametrize("size", [(1, 50, 90, 2, 1, 64), (1, 3, 90, 2, 1, 64)], ids=str)
def test_scales(size, scale):
    q, k, v, g = draw(*size, seed=6)
    both(q, k, v, g, scale, norm=scale != 0.0)


def test_strides():
    g = np.random.default_rng(8)
    # q from one projection's output, k and v halves of another's, rows that start off 16 bytes
    for pad in (0, 1):
        qkv = g.standard_normal((2, 70, 6, 64 + pad)).astype(np.float32)
        kv = g.standard_normal((2, 90, 2, 2, 64 + pad)).astype(np.float32)
        go = g.standard_normal((2, 70, 4, 64)).astype(np.float32)
        tq, tkv = cuda(qkv)[:, :, 1:5, pad:], cuda(kv)[..., pad:]
        both(qkv[:, :, 1:5, pad:], kv[:, :, 0, :, pad:], kv[:, :, 1, :, pad:], go, 0.125,
             dev=(tq, tkv[:, :, 0], tkv[:, :, 1], cuda(go)))
    # [B, H, T, D] storage, and D as the slow dimension
    q, k, v, go = draw(2, 40, 50, 2, 2, 32, seed=9)
    perm = [cuda(x.transpose(0, 2, 1, 3)).permute(0, 2, 1, 3) for x in (q, k, v, go)]
    both(q, k, v, go, 0.2, dev=perm)
    slow = [cuda(x.transpose(3, 0, 1, 2)).permute(1, 2, 3, 0) for x in (q, k, v, go)]
    both(q, k, v, go, 0.2, dev=slow)
    # the same with few query rows (CUDA cores)
    q1, g1 = q[:, :3], go[:, :3]
    both(q1, k, v, g1, 0.2, dev=(perm[0][:, :3], perm[1], perm[2], perm[3][:, :3]))
    both(q1, k, v, g1, 0.2, dev=(slow[0][:, :3], slow[1], slow[2], slow[3][:, :3]))
    # one head broadcast to all as an input
    one = cuda(k[:, :, :1]).expand(2, 50, 2, 32)
    kk = np.broadcast_to(k[:, :, :1], k.shape)
    both(q, kk, v, go, 0.2, dev=(cuda(q), one, cuda(v), cuda(go)))


def test_outputs_through_strides_leave_the_rest():
    from tensorrs_b200 import device
    V = device.view_of
    q, k, v, g = draw(2, 40, 50, 2, 1, 48, seed=10)
    tq, tk, tv, tg = map(cuda, (q, k, v, g))
    t = Truth(q, k, v, 0.2, None, g)
    ob = torch.full((2, 40, 3, 50), 7.0, device="cuda")
    lb = torch.full((2, 2, 41), 7.0, device="cuda")
    out, lse = ob[:, :, :2, 1:49], lb[:, :, :40]
    device.cross_attention(V(tq), V(tk), V(tv), 0.2, out, lse=lse)
    check(to_host(out), t.out, t.out_tol, "out")
    check(to_host(lse), t.lse, t.lse_tol, "lse")
    gkv = torch.full((2, 51, 2, 1, 48), 7.0, device="cuda")  # dk and dv as halves of one buffer
    dq = torch.full((2, 2, 40, 48), 7.0, device="cuda").permute(0, 2, 1, 3)
    device.cross_attention_backward(V(tg), V(tq), V(tk), V(tv), V(out), V(lse), 0.2, dq, gkv[:, :50, 0], gkv[:, :50, 1])
    check(to_host(dq), t.dq, t.dq_tol, "dq")
    check(to_host(gkv[:, :50, 0]), t.dk, t.dk_tol, "dk")
    check(to_host(gkv[:, :50, 1]), t.dv, t.dv_tol, "dv")
    assert (ob[:, :, 2] == 7).all() and (ob[..., 0] == 7).all() and (ob[..., 49] == 7).all()
    assert (lb[:, :, 40] == 7).all() and (gkv[:, 50] == 7).all()


@pytest.mark.parametrize("size", [(1, 130, 200, 1, 1, 64), (1, 40, 100, 1, 1, 128), (1, 4, 100, 1, 1, 64)], ids=str)
@pytest.mark.parametrize("qs,vs,gs", [(1e-18, 1e18, 1e-15), (1e15, 1e-20, 1e12), (1e-30, 1e30, 1e-30)])
def test_magnitudes(size, qs, vs, gs):
    """Operands far from 1 (the scores stay of order 1): the parts are placed by a power of two of each tile."""
    q, k, v, g = draw(*size, seed=11)
    f = np.float32
    both(q * f(qs), k * f(1 / qs), v * f(vs), g * f(gs), 0.125)


def test_rows_of_uneven_magnitude():
    """Neighbouring tokens differ by 10^6: the bound allows 2^-38 of a tile's largest, the small rows still come out."""
    q, k, v, g = draw(1, 150, 200, 1, 1, 64, seed=12)
    v[:, ::7] *= np.float32(1e-6)
    g[:, ::5] *= np.float32(1e-6)
    k[:, ::3] *= np.float32(1e-3)
    both(q, k, v, g, 0.125)


@pytest.mark.parametrize("what", ["q", "k"])
def test_the_low_part_of_small_elements_counts(what):
    """One row 2^20 larger than its tile's others.  The others' parts are then off by 2^-40 of the largest, 2^-20 of
    themselves, which needs the subnormal numbers of fp16 (without them 2^-28 of the largest, 2^-8).  The scale makes
    up for the size: a score of D = 64 independent errors of 2^-40 2^20 |q k| is off by 2^-20 * 8 * 4, the weights by
    twice that and the 2-norm of the result by less than 2^-13."""
    q, k, v, g = draw(1, 130, 100, 1, 1, 64, seed=17)
    x = {"q": q, "k": k}[what]
    x *= np.float32(2.0**-20)
    x[0, 0] *= np.float32(2.0**20)
    scale = 0.125 * 2.0**20
    out, lse = forward(cuda(q), cuda(k), cuda(v), scale)
    t = Truth(q, k, v, scale)
    got, want = to_host(out)[0, 1:], t.out[0, 1:]
    if what == "k":  # the large key takes or loses all weight: rows where it lost
        lost = np.abs(want - v[0, 0]).max((1, 2)) > 1e-3
        got, want = got[lost], want[lost]
    assert len(want) > 20 and np.linalg.norm(got - want) <= 2.0**-13 * np.linalg.norm(want)


def test_peaked_rows():
    """Scores of hundreds: one key takes nearly all of the weight."""
    q, k, v, g = draw(1, 140, 180, 1, 1, 64, seed=13)
    both(q * np.float32(20), k, v, g, 1.0, norm=False)


@pytest.mark.parametrize("size", [(1, 130, 90, 2, 1, 64), (1, 3, 90, 2, 1, 64), (1, 20, 40, 1, 1, 160)], ids=str)
def test_special_values_propagate(size):
    q, k, v, g = draw(*size, seed=14)
    scale = size[-1] ** -0.5
    for where, value in (("q", np.nan), ("q", np.inf), ("k", np.nan), ("v", np.nan), ("v", np.inf)):
        x = {"q": q.copy(), "k": k.copy(), "v": v.copy()}
        x[where][0, 2, 0, 1] = value
        out, lse = forward(cuda(x["q"]), cuda(x["k"]), cuda(x["v"]), scale)
        got = to_host(out)
        t = Truth(q, k, v, scale)
        if where == "q":  # this row alone; an infinite score takes no defined weight
            assert np.isnan(got[0, 2, 0]).any() or value == np.inf
            got[0, 2, 0] = t.out[0, 2, 0]
            check(got, t.out, t.out_tol, where)
        elif where == "k":
            assert np.isnan(got[0, :, : size[3] // size[4]]).all()
        else:
            bad = np.isnan(got) if np.isnan(value) else np.isinf(got)
            want = np.zeros(got.shape, bool)
            want[..., 1] = True
            assert np.array_equal(bad, want)
        dq, dk, dv = backward(cuda(g), cuda(x["q"]), cuda(x["k"]), cuda(x["v"]), out, lse, scale)
        if where == "q" and np.isnan(value):
            assert np.isnan(to_host(dq)[0, 2, 0]).all() and np.isfinite(to_host(dq)[0, 1]).all()
    # a row whose scores are all -inf counts as empty
    qi, ki = np.abs(q), np.abs(k)
    qi[0, 1, 0, 0], ki[..., 0] = -np.inf, 1.0
    out, lse = forward(cuda(qi), cuda(ki), cuda(v), scale)
    assert (out[0, 1, 0] == 0).all() and lse[0, 0, 1] == -np.inf


@pytest.mark.parametrize("Tq,Tk", [(0, 5), (5, 0)])
def test_no_queries_or_no_keys(Tq, Tk):
    q, k, v, g = draw(2, Tq, Tk, 2, 1, 16)
    t = tuple(map(cuda, (q, k, v, g)))
    out, lse = forward(*t[:3], 1.0)
    assert (out == 0).all() and (lse == -np.inf).all()
    for x in backward(t[3], *t[:3], out, lse, 1.0):
        assert (x == 0).all()


def test_gradients_against_differences():
    """Central differences of the f64 definition along random directions against the f32 gradient: h = 2^-10 of a
    direction of norm 1, off by h^2 of a third derivative of order 1, and the gradient by 32 u of its norm."""
    q, k, v, g = draw(1, 20, 33, 2, 1, 64, seed=15)
    out, lse, *grads = both(q, k, v, g, 0.125)
    r = np.random.default_rng(1)
    for i, d in enumerate(grads):
        x = [a.astype(np.float64) for a in (q, k, v)]
        w = r.standard_normal(x[i].shape)
        w /= np.linalg.norm(w)
        h = 2.0**-10
        loss = []
        for s in (h, -h):
            y = list(x)
            y[i] = x[i] + s * w
            loss.append((Truth(*y, 0.125).out * g).sum())
        want = (loss[0] - loss[1]) / (2 * h)
        d = to_host(d).astype(np.float64)
        assert abs((d * w).sum() - want) <= 1e-5 * max(1.0, np.linalg.norm(d)), i


def test_streams_graphs_and_repeats_give_the_same_bits():
    q, k, v, g = (cuda(x) for x in draw(3, 150, 200, 4, 2, 64, seed=16))
    q1 = q[:, :2].contiguous()
    n = torch.tensor([200, 0, 77], device="cuda")

    def call():
        out, lse = forward(q, k, v, 0.125, n)
        return [out, lse, *backward(g, q, k, v, out, lse, 0.125, n), *forward(q1, k, v, 0.125, n)]

    first = call()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = call()
    third = call()  # at the same time on another stream
    torch.cuda.synchronize()
    outs, graphs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(call())
        graphs.append(gr)
    for gr in graphs + graphs[::-1]:
        gr.replay()
    torch.cuda.synchronize()
    for o in (second, third, *outs):
        for a, b in zip(first, o):
            assert torch.equal(a, b)


@pytest.mark.parametrize("size,lengths", [((6, 700, 900, 8, 8, 64), [900, 0, 3, 129, 900, 500]),
                                          ((5, 500, 700, 8, 4, 128), [1, 700, 0, 64, 650])], ids=str)
def test_more_items_than_sms_of_ragged_length(size, lengths):
    q, k, v, g = draw(*size, seed=19)
    n = np.array(lengths, np.int32)
    first = both(q, k, v, g, 0.125, n)
    q, k, v, g, n = (cuda(x) for x in (q, k, v, g, n))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, lse = forward(q, k, v, 0.125, n)
        again = (out, lse, *backward(g, q, k, v, out, lse, 0.125, n))
    for _ in range(3):
        for x in again:
            x.fill_(float("nan"))
        gr.replay()
        for x, y in zip(first, again):
            assert torch.equal(x, y)


def test_kernels_never_gave_up_waiting():
    import ctypes
    from tensorrs_b200 import abi
    code = ctypes.c_int32()
    assert abi.load().trs_async_error(ctypes.byref(code)) == abi.OK and code.value == 0
