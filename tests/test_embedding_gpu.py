"""trs_embedding and trs_embedding_backward through the C ABI, against the
definition in 64 bits.

Tolerances, u half a unit of the element type (2^-24, 2^-53):
  lookup: the scale is rounded to the element type (u) and the product rounds
  (u): 2 u of the result, and u^2.
  gradient: the sum is taken in f64 (n additions of 2^-53 of the terms) with
  one product and one rounding to the element type: u of the result and
  (n + 4) 2^-53 of the terms (with accumulate, of what was there too)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _gpu import to_host
from tensorrs_b200 import abi, device

pytestmark = pytest.mark.gpu

U = {"f4": 2.0**-24, "f8": 2.0**-53}
TORCH = {"f4": torch.float32, "f8": torch.float64}


def tokens(g, N, V, kind):
    """Ids of a text: a few make up most of it; some lie outside [0, V)."""
    if kind == "one":
        return np.full(N, V - 1)
    if kind == "none":
        return np.where(g.random(N) < 0.5, -1, V + g.integers(0, 5, N))
    ids = np.minimum((V ** g.random(N)).astype(np.int64), V) - 1
    ids = g.permutation(V)[ids] if V < 1 << 20 else ids
    return np.where(g.random(N) < 0.1, g.choice([-1, -100, V, 2**31 - 1], N), ids)


def truth_lookup(table, ids, scale):
    V = len(table)
    there = (ids >= 0) & (ids < V)
    out = np.zeros((ids.size, table.shape[1]))
    out[there.ravel()] = table[ids[there]].astype(np.float64) * scale
    return out.reshape(*ids.shape, -1)


def truth_grad(grad, ids, scale, V, before=None):
    """The gradient and the sum of its terms' magnitudes."""
    D = grad.shape[-1]
    there = (ids >= 0) & (ids < V)
    g = grad.reshape(-1, D).astype(np.float64)[there.ravel()] * scale
    want, terms = np.zeros((V, D)), np.zeros((V, D))
    np.add.at(want, ids[there], g)
    np.add.at(terms, ids[there], np.abs(g))
    if before is not None:
        want, terms = want + before, terms + np.abs(before)
    return want, terms


def lookup(table, ids, scale, out):
    device.embedding(device.view_of(table), device.view_of(ids), scale, out)
    return to_host(out)


def check(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want) / np.maximum(tol, 1e-300))))


# batch (0: ids of rank 1), tokens, V, D, dtype, kind of ids, id type
SIZES = [
    (0, 1, 1, 1, "f4", "text", "i8"), (0, 1, 7, 4, "f4", "one", "i4"), (2, 1, 300, 64, "f4", "text", "i8"),
    (0, 31, 2, 16, "f4", "text", "i8"), (0, 32, 511, 20, "f4", "one", "i4"), (0, 33, 512, 20, "f4", "one", "i8"),
    (3, 65, 513, 7, "f4", "text", "i4"), (1, 4095, 1000, 12, "f8", "text", "i8"), (1, 4096, 3, 9, "f8", "one", "i8"),
    (2, 2049, 70001, 36, "f4", "text", "i8"), (3, 3333, 300_000, 8, "f4", "text", "i4"), (5, 77, 4000, 1031, "f4", "text", "i8"),
    (2, 500, 900, 2048, "f4", "text", "i8"), (1, 257, 40, 514, "f8", "text", "i8"), (4, 100, 50, 24, "f4", "none", "i8"),
    (2, 9000, 20, 40, "f4", "text", "i8"), (0, 100, 300_000, 8, "f4", "text", "i8"), (1, 4097, 600, 33, "f4", "one", "i4"),
    (0, 40_000, 9, 16, "f4", "one", "i8"),
]
NAMES = ["x".join(str(x) for x in s) for s in SIZES]


@pytest.mark.parametrize("size", SIZES, ids=NAMES)
def test_lookup(size):
    B, T, V, D, dt, kind, it = size
    g = np.random.default_rng(V + D)
    ids = tokens(g, max(B, 1) * T, V, kind).reshape((B, T) if B else (T,)).astype(it)
    table = g.standard_normal((V, D)).astype(dt)
    out = torch.full((*ids.shape, D), np.nan, dtype=TORCH[dt], device="cuda")
    for scale in (1.0, np.sqrt(D) + 0.1):
        got = lookup(torch.from_numpy(table).cuda(), torch.from_numpy(ids).cuda(), scale, out)
        want = truth_lookup(table, ids.astype(np.int64), scale)
        check(got, want, (2 * U[dt] + U[dt] ** 2) * np.abs(want) if scale != 1.0 else 0 * want, size)


@pytest.mark.parametrize("D", [24, 7])
@pytest.mark.parametrize("scale,size", [(1e-50, 1e30), (1e45, 1e-30), (-1e-40, 1e20), (2.0**-149, 1e25), (2.0**128, 1e-10)])
def test_lookup_scales_beyond_f32(scale, size, D):
    """A scale that f32 does not hold in full, with products that it does: one rounding of f64's product."""
    g = np.random.default_rng(D)
    table, ids = (g.standard_normal((40, D)) * size).astype("f4"), tokens(g, 70, 40, "text")
    out = torch.full((70, D), np.nan, device="cuda")
    got = lookup(torch.from_numpy(table).cuda(), torch.from_numpy(ids).cuda(), scale, out)
    want = truth_lookup(table, ids, scale)
    check(got, want, (U["f4"] + 2.0**-52) * np.abs(want), (scale, size))


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=NAMES)
def test_gradient(size, accumulate):
    B, T, V, D, dt, kind, it = size
    g = np.random.default_rng(V * 3 + D)
    ids = tokens(g, max(B, 1) * T, V, kind).reshape((B, T) if B else (T,)).astype(it)
    grad = g.standard_normal((*ids.shape, D)).astype(dt)
    grad[(ids < 0) | (ids >= V)] = np.nan  # what is not looked up is not read
    scale = 1.7
    before = g.standard_normal((V, D)).astype(dt)
    seen = np.zeros(V, bool)
    seen[ids[(ids >= 0) & (ids < V)]] = True
    before[~seen] = np.nan  # nor are the rows that no token looked up touched
    want, terms = truth_grad(grad, ids.astype(np.int64), scale, V, before if accumulate else None)
    res, gt, it = [], torch.from_numpy(grad).cuda(), torch.from_numpy(ids).cuda()
    for _ in range(2):
        out = torch.from_numpy(before.copy()).cuda()
        device.embedding_backward(device.view_of(gt), device.view_of(it), scale, out, accumulate=accumulate)
        res.append(to_host(out))
    got = res[0]
    assert np.array_equal(got, res[1], equal_nan=True)
    if accumulate:
        assert np.isnan(got[~seen]).all()
        got, want, terms = got[seen], want[seen], terms[seen]
    n = np.bincount(ids[(ids >= 0) & (ids < V)].astype(np.int64), minlength=1).max(initial=0)
    check(got, want, U[dt] * np.abs(want) + (n + 4) * 2.0**-53 * terms, size)


def test_gradient_against_differences():
    """<grad_table, step> is the change of <grad_out, out> along the step, which is linear in the table."""
    g = np.random.default_rng(5)
    V, D, ids = 50, 24, g.integers(-1, 50, (3, 40))
    table, step, grad = (torch.from_numpy(g.standard_normal(s)).cuda() for s in ((V, D), (V, D), (3, 40, D)))
    idt = torch.from_numpy(ids).cuda()
    out = [torch.empty((3, 40, D), dtype=torch.float64, device="cuda") for _ in range(2)]
    device.embedding(device.view_of(table), device.view_of(idt), 0.5, out[0])
    device.embedding(device.view_of(table + step), device.view_of(idt), 0.5, out[1])
    gt = torch.empty_like(table)
    device.embedding_backward(device.view_of(grad), device.view_of(idt), 0.5, gt)
    a, b = float((gt * step).sum()), float((grad * (out[1] - out[0])).sum())
    # products of magnitude 1 with values off by 2^-51: 120 * 24 of them
    assert abs(a - b) <= 2880 * 8 * 2.0**-50


@pytest.mark.parametrize("dt", ["f4", "f8"])
@pytest.mark.parametrize("layout", ["transposed", "reversed", "slices", "offset"])
def test_strides(layout, dt):
    g = np.random.default_rng(11)
    B, T, V, D = 3, 50, 60, 24
    ids = tokens(g, B * T, V, "text").reshape(B, T)
    table, grad = g.standard_normal((V, D)).astype(dt), g.standard_normal((B, T, D)).astype(dt)
    tt, gt, it = torch.from_numpy(table).cuda(), torch.from_numpy(grad).cuda(), torch.from_numpy(ids).cuda()
    guard = None
    if layout == "transposed":  # [in, out] storage, tokens before batch
        buf = torch.zeros((D, V), dtype=TORCH[dt], device="cuda")
        buf.copy_(tt.T)
        tv, tout = device.view_of(buf.T), lambda: torch.zeros((D, V), dtype=TORCH[dt], device="cuda").T
        gp, ip = gt.permute(1, 0, 2).contiguous(), it.T.contiguous()
        gv, iv = device.view_of(gp.permute(1, 0, 2)), device.view_of(ip.T)
        rows = torch.zeros((T, B, D), dtype=TORCH[dt], device="cuda").permute(1, 0, 2)
    elif layout == "reversed":
        rt, rg, ri = tt.flip(1).contiguous(), gt.flip(1).contiguous(), it.flip(0).contiguous()
        tv = device.view_of(rt, [V, D], [D, -1], D - 1)
        gv = device.view_of(rg, [B, T, D], [T * D, -D, 1], (T - 1) * D)
        iv = device.view_of(ri, [B, T], [-T, 1], (B - 1) * T)
        tout, rows = lambda: torch.zeros_like(tt), torch.zeros((B, T, D), dtype=TORCH[dt], device="cuda")
    elif layout == "slices":  # a sequence shifted by one, inside a wider row
        wide = torch.full((B, T + 1, D + 8), np.nan, dtype=TORCH[dt], device="cuda")
        wide[:, :-1, 4:-4] = gt
        gv = device.view_of(wide[:, :-1, 4:-4])
        iw = torch.full((B, T + 3), V - 1, device="cuda")
        iw[:, 3:] = it
        iv, tv = device.view_of(iw[:, 3:]), device.view_of(tt)
        tout = lambda: torch.zeros((V, D + 8), dtype=TORCH[dt], device="cuda")[:, 4:-4]  # noqa: E731
        guard = torch.full((B, T + 2, D + 8), 7.0, dtype=TORCH[dt], device="cuda")
        rows = guard[:, 1:-1, 4:-4]
    else:  # rows that begin off a 16-byte boundary
        buf = torch.zeros(V * D + 1, dtype=TORCH[dt], device="cuda")
        buf[1:] = tt.flatten()
        tv, gv, iv = device.view_of(buf[1:].view(V, D)), device.view_of(gt), device.view_of(it)
        tout = lambda: torch.zeros(V * D + 1, dtype=TORCH[dt], device="cuda")[1:].view(V, D)  # noqa: E731
        rows = torch.zeros((B, T, D), dtype=TORCH[dt], device="cuda")
    device.embedding(tv, iv, 3.0, rows)
    want = truth_lookup(table, ids, 3.0)
    check(to_host(rows), want, 2 * U[dt] * np.abs(want), layout)
    if guard is not None:
        rows.fill_(7.0)
        assert bool((guard == 7.0).all())
    out = tout()
    device.embedding_backward(gv, iv, 3.0, out)
    want, terms = truth_grad(grad, ids, 3.0, V)
    check(to_host(out), want, U[dt] * np.abs(want) + (B * T + 4) * 2.0**-53 * terms, layout)
    if layout == "slices":
        whole = out._base if out._base is not None else out
        assert float(whole[:, :4].abs().max()) == 0 and float(whole[:, -4:].abs().max()) == 0


def test_offsets_past_32_bits():
    V, D = 70_000, 32_768
    table = torch.zeros((V, D), device="cuda")
    table[-1] = torch.arange(D, device="cuda")
    ids = torch.tensor([[V - 1, 0, V - 1]], device="cuda")
    out = torch.empty((1, 3, D), device="cuda")
    device.embedding(device.view_of(table), device.view_of(ids), 2.0, out)
    assert torch.equal(out[0, 0], 2 * table[-1]) and torch.equal(out[0, 2], out[0, 0]) and not bool(out[0, 1].any())
    table.fill_(1.0)
    device.embedding_backward(device.view_of(out), device.view_of(ids), 1.0, table)
    assert torch.equal(table[-1], 2 * out[0, 0])
    assert not bool(table[:-1].any())


def test_streams_and_graphs():
    """Calls on two streams at once, and a captured forward and backward replayed on new inputs."""
    g = torch.Generator(device="cuda").manual_seed(1)
    V, D, N = 5000, 256, 6000
    args = []
    for _ in range(2):
        args.append((torch.randint(-1, V, (N,), generator=g, device="cuda"),
                     torch.randn((N, D), generator=g, device="cuda"), torch.empty((V, D), device="cuda")))
    want = []
    for ids, grad, out in args:
        device.embedding_backward(device.view_of(grad), device.view_of(ids), 1.0, out)
        want.append(out.clone())
        out.fill_(np.nan)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(5):
        for st, (ids, grad, out) in zip(streams, args):
            with torch.cuda.stream(st):
                device.embedding_backward(device.view_of(grad), device.view_of(ids), 1.0, out)
    torch.cuda.synchronize()
    for (_, _, out), w in zip(args, want):
        assert torch.equal(out, w)
    ids, grad, out = args[0]
    rows = torch.empty((N, D), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        device.embedding(device.view_of(grad), device.view_of(ids), 1.0, rows)
        device.embedding_backward(device.view_of(rows), device.view_of(ids), 1.0, out)
    for src in (1, 0):
        ids.copy_(args[src][0].clone())
        graph.replay()
        graph.replay()
        ok = (ids >= 0)
        assert torch.equal(rows, torch.where(ok[:, None], grad[ids.clamp(min=0)], 0.0))
        torch.testing.assert_close(out.double(), torch.zeros((V, D), device="cuda", dtype=torch.float64).index_add_(
            0, ids[ok], rows[ok].double()), rtol=2.0**-23, atol=1e-9)


def test_other_device_type_refused():
    ids, out = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.empty((3, 4), device="cuda")
    with pytest.raises(ValueError):
        device.embedding(device.view_of(out), device.view_of(ids), 1.0, out.cpu())
    table = torch.zeros((4, 5), device="cuda")
    with pytest.raises(abi.TrsError):
        device.embedding(device.view_of(table), device.view_of(ids), 1.0, out)
