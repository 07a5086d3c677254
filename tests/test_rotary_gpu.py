"""trs_rotary, trs_head_norm_rotary and their gradients through the C ABI,
against the definition in 80 bits.

Tolerances, u half a unit of the element type (2^-24, 2^-53), relative to
|a| + |b| of the element's pair (`reach`):
  rotation: the f32 turns are off by 2^-25 of half a turn, pi u / 2 of angle;
  sincospif (at most 2 units = 4 u), the magnitude's product (u) and the
  rotation's own product, fma and store (2 u) make less than 9 u.
  norm: a chain of at most 32 fused squares and 5 folds (37 u), halved by the
  root, division, root and two products of 4 roundings: 23 u more, 32 u.
  gradient of x: both of these in each of two terms, the mean's own chain of
  64 products and 5 folds: 9 + 23 + 37 + 23 < 96 u of the terms' sum.
  gradient of gamma: f64 sums of products off by 9 + 23 u each: 36 u.
The f64 path takes sincos of the same product: the same counts with u = 2^-53.
Positions reach 5e6, where the f64 product p f is off by 2^-53 5e6 < 2^-30
of an angle: below u for f32; for f64 both sides take the rounded product."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import _rotary as ref
from _gpu import empty, to_host

pytestmark = pytest.mark.gpu

U = {np.dtype(np.float32): 2.0**-24, np.dtype(np.float64): 2.0**-53}


def check(got, want, tol, what):
    got = got.astype(ref.LD)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want) / np.maximum(tol, 1e-300))))


def cuda(a):
    return torch.from_numpy(np.array(a, order="C")).cuda()


# B, T, Hq, Hk, D, R, dtype
SIZES = [
    (1, 1, 1, 1, 2, 2, "f4"), (2, 3, 4, 2, 64, 64, "f4"), (1, 5, 7, 1, 128, 64, "f4"), (3, 37, 5, 3, 80, 80, "f4"),
    (2, 9, 3, 2, 96, 32, "f4"), (2, 9, 3, 2, 10, 6, "f4"), (1, 4, 2, 2, 7, 2, "f4"), (1, 3, 2, 1, 512, 512, "f4"),
    (1, 3, 2, 1, 510, 250, "f4"), (2, 300, 20, 4, 64, 64, "f4"), (1, 2, 9, 2, 72, 24, "f4"), (1, 6, 2, 2, 130, 66, "f4"),
    (2, 5, 3, 1, 64, 32, "f8"), (1, 3, 2, 2, 11, 4, "f8"), (1, 2, 2, 1, 512, 256, "f8"), (1, 2, 2, 1, 511, 500, "f8"),
    (700, 1, 8, 8, 32, 32, "f4"),
]


def data(B, T, Hq, Hk, D, dt, seed):
    g = np.random.default_rng(seed)
    qkv = g.standard_normal((B, T, Hq + 2 * Hk, D)).astype(dt)
    t = torch.from_numpy(qkv).cuda()
    return qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], t[:, :, :Hq], t[:, :, Hq:Hq + Hk], g


def positions(B, T, g, kind):
    if kind == "i64":
        return g.integers(0, 5_000_000, (B, T))
    if kind == "i32":
        return g.integers(-1000, 100_000, (B, T)).astype(np.int32)
    return np.broadcast_to(np.arange(T, dtype=np.int64), (B, T))  # one row for all


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("kind", ["i64", "i32", "row"])
def test_rotary_and_its_gradient(size, layout, kind):
    from tensorrs_b200 import device
    B, T, Hq, Hk, D, R, dt = size
    q, k, tq, tk, g = data(B, T, Hq, Hk, D, dt, 1)
    pos, fr = positions(B, T, g, kind), ref.frequencies(R // 2)
    tp = cuda(pos[0]) if kind == "row" else cuda(pos)
    tf = cuda(fr)
    qo, ko = empty(q.shape, dt), empty(k.shape, dt)
    u = U[np.dtype(dt)]
    for m in (1.0, 1.25):
        device.rotary(device.view_of(tq), device.view_of(tk), device.view_of(tp), device.view_of(tf), qo, ko,
                      layout=layout, magnitude=m)
        for x, y in ((q, qo), (k, ko)):
            check(to_host(y), ref.rotate(x, pos, fr, layout, m), 9 * u * ref.reach(x, fr, layout, m), "forward")
        device.rotary_backward(device.view_of(tq), device.view_of(tk), device.view_of(tp), device.view_of(tf), qo, ko,
                               layout=layout, magnitude=m)
        for x, y in ((q, qo), (k, ko)):
            check(to_host(y), ref.rotate(x, pos, fr, layout, m, inverse=True), 9 * u * ref.reach(x, fr, layout, m), "back")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_head_norm_rotary_and_its_gradients(size, layout):
    from tensorrs_b200 import device
    B, T, Hq, Hk, D, R, dt = size
    q, k, tq, tk, g = data(B, T, Hq, Hk, D, dt, 2)
    pos, fr, eps, m = positions(B, T, g, "i64"), ref.frequencies(R // 2), 1e-6, 1.25
    gq, gk = (g.uniform(0.5, 1.5, D).astype(dt) for _ in range(2))
    dq, dk = g.standard_normal(q.shape).astype(dt), g.standard_normal(k.shape).astype(dt)
    V = device.view_of
    vq, vk, vgq, vgk = V(tq), V(tk), V(tgq := cuda(gq)), V(tgk := cuda(gk))
    vp, vf = V(tp := cuda(pos)), V(tf := cuda(fr))
    qo, ko, xq, xk = empty(q.shape, dt), empty(k.shape, dt), empty(q.shape, dt), empty(k.shape, dt)
    aq, ak = empty([D], dt), empty([D], dt)
    device.head_norm_rotary(vq, vk, vgq, vgk, eps, vp, vf, qo, ko, layout=layout, magnitude=m)
    device.head_norm_rotary_backward(V(tdq := cuda(dq)), V(tdk := cuda(dk)), vq, vk, vgq, vgk, eps, vp, vf, xq, xk, aq, ak,
                                     layout=layout, magnitude=m)
    u = U[np.dtype(dt)]
    for x, ga, dy, y, dx, dga in ((q, gq, dq, qo, xq, aq), (k, gk, dk, ko, xk, ak)):
        n, _ = ref.norm(x, eps)
        check(to_host(y), ref.norm_rotate(x, ga, eps, pos, fr, layout, m), 32 * u * ref.reach(n * ga, fr, layout, m), "y")
        want, wga = ref.norm_rotate_backward(dy, x, ga, eps, pos, fr, layout, m)
        rx, rg = ref.norm_backward_reach(dy, x, ga, eps, fr, layout, m)
        check(to_host(dx), want, 96 * u * rx, "dx")
        check(to_host(dga), wga, 36 * u * rg, "dgamma")
    del tgq, tgk, tp, tf, tdq, tdk


def test_gradients_against_differences():
    """f64, step h = 2^-17: the difference is off by h^2/6 of a third derivative of order 1 and by 2^-53/h."""
    from tensorrs_b200 import device
    V = device.view_of
    g = np.random.default_rng(5)
    x = cuda(g.standard_normal((1, 3, 2, 16)))
    ga = cuda(g.uniform(0.5, 1.5, 16))
    w = cuda(g.standard_normal((1, 3, 2, 16)))
    pos, fr = cuda(np.array([[0, 7, 1234]])), cuda(ref.frequencies(6))

    def loss(x, ga):
        y = torch.empty_like(x)
        device.head_norm_rotary(V(x), None, V(ga), None, 1e-5, V(pos), V(fr), y, None, layout="interleaved", magnitude=1.1)
        return float((y * w).sum())

    dx, dga = torch.empty_like(x), torch.empty_like(ga)
    device.head_norm_rotary_backward(V(w), None, V(x), None, V(ga), None, 1e-5, V(pos), V(fr), dx, None, dga, None,
                                     layout="interleaved", magnitude=1.1)
    h = 2.0**-17
    for t, d in ((x, dx), (ga, dga)):
        flat, df = t.reshape(-1), d.reshape(-1)
        for i in range(0, flat.numel(), 5):
            keep = float(flat[i])
            flat[i] = keep + h
            up = loss(x, ga)
            flat[i] = keep - h
            down = loss(x, ga)
            flat[i] = keep
            assert abs((up - down) / (2 * h) - float(df[i])) < 1e-7


@pytest.mark.parametrize("kind", ["nan", "inf"])
def test_special_values_stay_in_their_row(kind):
    """A NaN or infinity reaches its own row and pair alone; a row of zeros gives zeros."""
    from tensorrs_b200 import device
    V = device.view_of
    x = torch.randn(1, 4, 2, 64, device="cuda")
    bad = x.clone()
    bad[0, 1, 0, 3] = float(kind)
    bad[0, 2, 1] = 0
    pos, fr = torch.arange(4, device="cuda"), cuda(ref.frequencies(32))
    one = torch.ones(64, device="cuda")
    outs = []
    for t in (x, bad):
        y, n = torch.empty_like(t), torch.empty_like(t)
        device.rotary(V(t), None, V(pos), V(fr), y, None)
        device.head_norm_rotary(V(t), None, V(one), None, 1e-6, V(pos), V(fr), n, None)
        outs.append((y.cpu(), n.cpu()))
    (y0, n0), (y1, n1) = outs
    diff = (y1 != y0) | y1.isnan()
    diff[0, 2, 1] = False
    assert diff.sum() == 2 and diff[0, 1, 0, 3] and diff[0, 1, 0, 35]
    assert (n1[0, 2, 1] == 0).all() and (y1[0, 2, 1] == 0).all()
    same = torch.ones(1, 4, 2, dtype=torch.bool)
    same[0, 1, 0] = same[0, 2, 1] = False
    assert torch.equal(n1[same], n0[same])


def test_in_place_strides_and_no_keys():
    from tensorrs_b200 import device
    V = device.view_of
    g = np.random.default_rng(3)
    h = g.standard_normal((2, 6, 12, 64)).astype(np.float32)  # 6 q heads, 3 k heads, 3 v heads
    pos, fr = g.integers(0, 99, (2, 6)), ref.frequencies(32)
    tp, tf = cuda(pos), cuda(fr)
    buf = cuda(h)
    q, k = buf[:, :, :6], buf[:, :, 6:9]
    device.rotary(V(q), V(k), V(tp), V(tf), q, k)  # in place, inside one projection's output
    got = to_host(buf)
    for sl in (slice(0, 6), slice(6, 9)):
        check(got[:, :, sl], ref.rotate(h[:, :, sl], pos, fr, "half"), 9 * 2.0**-24 * ref.reach(h[:, :, sl], fr, "half"), sl)
    assert np.array_equal(got[:, :, 9:], h[:, :, 9:])
    # [B, H, T, D] storage seen as [B, T, H, D], reversed tokens, an element stride of 2, unaligned rows
    st = cuda(g.standard_normal((2, 3, 6, 64)).astype(np.float32))
    x = st.permute(0, 2, 1, 3)
    y = empty(x.shape, np.float32)
    device.rotary(V(x), None, V(tp), V(tf), y, None, layout="interleaved")
    xh = to_host(st).transpose(0, 2, 1, 3)
    check(to_host(y), ref.rotate(xh, pos, fr, "interleaved"), 9 * 2.0**-24 * ref.reach(xh, fr, "interleaved"), "permuted")
    flat = cuda(g.standard_normal(2 * 6 * 129 * 3).astype(np.float32))
    shape, strides, off = [2, 6, 3, 64], [6 * 129 * 3, -129 * 3, 129, 2], 5 * 129 * 3 + 1
    y = torch.full((2, 6, 3, 65), 7.0, device="cuda")
    device.head_norm_rotary(device.view_of(flat, shape, strides, off), None, None, None, 1e-6, V(tp), V(tf), y[..., :64], None)
    xh = np.lib.stride_tricks.as_strided(to_host(flat)[off:], shape, [4 * s for s in strides])
    n, _ = ref.norm(xh, 1e-6)
    got = to_host(y)
    check(got[..., :64], ref.norm_rotate(xh, np.ones(64), 1e-6, pos, fr, "half"), 32 * 2.0**-24 * ref.reach(n, fr, "half"), "odd")
    assert (got[..., 64] == 7.0).all()


def test_empty_batches_and_zero_gradients():
    from tensorrs_b200 import device
    V = device.view_of
    x = torch.empty(0, 3, 2, 16, device="cuda")
    pos, fr, ga = torch.zeros(3, dtype=torch.int64, device="cuda"), cuda(ref.frequencies(8)), torch.ones(16, device="cuda")
    device.rotary(V(x), V(x), V(pos), V(fr), torch.empty_like(x), torch.empty_like(x))
    dga = torch.full((16,), 3.0, device="cuda")
    device.head_norm_rotary_backward(V(x), None, V(x), None, V(ga), None, 1e-6, V(pos), V(fr), torch.empty_like(x), None, dga, None)
    assert (dga == 0).all()
    # queries without keys' heads: the keys' gradient is zero
    q, k = torch.randn(1, 3, 2, 16, device="cuda"), torch.empty(1, 3, 0, 16, device="cuda")
    dgq, dgk = torch.full((16,), 3.0, device="cuda"), torch.full((16,), 3.0, device="cuda")
    device.head_norm_rotary_backward(V(q), V(k), V(q), V(k), V(ga), V(ga), 1e-6, V(pos), V(fr), torch.empty_like(q),
                                     torch.empty_like(k), dgq, dgk)
    assert (dgk == 0).all() and (dgq != 0).any()


def test_streams_graphs_and_repeats_give_the_same_bits():
    from tensorrs_b200 import device
    V = device.view_of
    g = torch.Generator(device="cuda").manual_seed(1)
    q, dq = (torch.randn(2, 513, 8, 64, device="cuda", generator=g) for _ in range(2))
    k, dk = (torch.randn(2, 513, 2, 64, device="cuda", generator=g) for _ in range(2))
    gq, gk = torch.rand(64, device="cuda"), torch.rand(64, device="cuda")
    pos, fr = torch.arange(513, device="cuda"), cuda(ref.frequencies(32))

    def outs():
        return [torch.full_like(t, float("nan")) for t in (q, k, gq, gk)]

    def call(o):
        device.head_norm_rotary_backward(V(dq), V(dk), V(q), V(k), V(gq), V(gk), 1e-6, V(pos), V(fr), *o)

    first = outs()
    call(first)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = outs()
        call(second)
    s.synchronize()
    third, fourth = outs(), outs()
    torch.cuda.synchronize()
    graphs = []
    for o in (third, fourth):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call(o)
        graphs.append(gr)
    for gr in graphs + graphs[::-1]:
        gr.replay()
    torch.cuda.synchronize()
    for o in (second, third, fourth):
        for a, b in zip(first, o):
            assert torch.equal(a, b)


# scaling, factor, low, high, context
@pytest.mark.parametrize("case", [("none", 1, 1, 32, 0), ("linear", 4, 1, 32, 0), ("base", 8, 1, 32, 0),
                                  ("bands", 8, 1, 4, 8192), ("ramp", 16, 1, 32, 4096)], ids=lambda c: c[0])
@pytest.mark.parametrize("n", [1, 2, 32, 64, 256])
def test_frequencies(case, n):
    """pow and log are off by 2 units, the mix's difference of nearly equal terms is relative to its bounds: 2^-44 of a
    frequency covers both."""
    from tensorrs_b200 import device
    scaling, factor, low, high, context = case
    out = empty([n], np.float64)
    device.rotary_frequencies(out, 10000.0, scaling, factor, low, high, context)
    i = np.arange(n, dtype=ref.LD)
    f = ref.LD(10000.0) ** (-i / n)
    if scaling == "linear":
        f = f / factor
    elif scaling == "base":
        grow = ref.LD(factor) ** (ref.LD(n) / (n - 1)) if n > 1 else ref.LD(factor)
        f = (10000.0 * grow) ** (-i / n)
        assert n == 1 or abs(f[-1] / (ref.LD(10000.0) ** (-i[-1] / n)) - ref.LD(1) / factor) < 1e-15
    elif scaling == "bands":
        keep = np.clip((context * f / (2 * ref.LD(np.pi)) - low) / (high - low), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    elif scaling == "ramp":
        at = [n * np.log(context / (r * 2 * ref.LD(np.pi))) / np.log(ref.LD(10000.0)) for r in (high, low)]
        first, last = max(np.floor(at[0]), 0), min(np.ceil(at[1]), 2 * n - 1)
        keep = 1 - np.clip((i - first) / ((last - first) or ref.LD(0.001)), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    assert np.all(np.abs(to_host(out) - f) <= 2.0**-44 * f)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions_of_any_size(layout):
    """The f64 product p f is an angle like any other: its turns are taken off without losing what the f32 rotation can
    hold (below 2^53 the positions themselves are exact)."""
    from tensorrs_b200 import device
    V = device.view_of
    g = np.random.default_rng(7)
    x, fr = g.standard_normal((1, 60, 2, 64)).astype(np.float32), ref.frequencies(32)
    pos = np.concatenate([2**g.integers(30, 53, 30) - g.integers(0, 1000, 30), -(2**g.integers(30, 53, 30))])[None]
    y = empty(x.shape, np.float32)
    device.rotary(V(tx := cuda(x)), None, V(tp := cuda(pos)), V(tf := cuda(fr)), y, None, layout=layout)
    check(to_host(y), ref.rotate(x, pos, fr, layout), 9 * 2.0**-24 * ref.reach(x, fr, layout), "far")
    del tx, tp, tf
