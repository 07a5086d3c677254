"""What trs_cross_attention and its gradient refuse, before any GPU call."""
from __future__ import annotations

import ctypes

import pytest

BASE = 1 << 24


def view(trs, shape, dtype=None, at=0, strides=None, **kw):
    return trs.make_view(BASE + (at << 24), trs.F32 if dtype is None else dtype, shape, strides, **kw)


def good(trs):
    q, k = [2, 5, 4, 16], [2, 7, 2, 16]
    return {"q": view(trs, q, at=0), "k": view(trs, k, at=1), "v": view(trs, k, at=2), "n": view(trs, [2], trs.I64, 3),
            "scale": 1.0, "out": view(trs, q, at=4), "lse": view(trs, [2, 4, 5], at=5), "g": view(trs, q, at=6),
            "dq": view(trs, q, at=7), "dk": view(trs, k, at=8), "dv": view(trs, k, at=9)}


def ref(v):
    return ctypes.byref(v) if v is not None else None


def forward(trs, a):
    return trs.check(trs.load().trs_cross_attention(ref(a["q"]), ref(a["k"]), ref(a["v"]), ref(a["n"]), a["scale"],
                                                    ref(a["out"]), ref(a["lse"]), None))


def backward(trs, a):
    return trs.check(trs.load().trs_cross_attention_backward(
        ref(a["g"]), ref(a["q"]), ref(a["k"]), ref(a["v"]), ref(a["n"]), ref(a["out"]), ref(a["lse"]), a["scale"],
        ref(a["dq"]), ref(a["dk"]), ref(a["dv"]), None))


Q, K = [2, 5, 4, 16], [2, 7, 2, 16]
BOTH = [
    ("null q", lambda t, a: a.update(q=None), "ERR_ARG"),
    ("null output", lambda t, a: a.update(out=None), "ERR_ARG"),
    ("rank", lambda t, a: a.update(k=view(t, [2, 14, 16], at=1)), "ERR_SHAPE"),
    ("f64", lambda t, a: a.update(q=view(t, Q, t.F64)), "ERR_DTYPE"),
    ("v shape", lambda t, a: a.update(v=view(t, [2, 6, 2, 16], at=2)), "ERR_SHAPE"),
    ("output shape", lambda t, a: a.update(out=view(t, [2, 5, 4, 8], at=4)), "ERR_SHAPE"),
    ("batch", lambda t, a: a.update(k=view(t, [3, 7, 2, 16], at=1), v=view(t, [3, 7, 2, 16], at=2),
                                    dk=view(t, [3, 7, 2, 16], at=8), dv=view(t, [3, 7, 2, 16], at=9)), "ERR_SHAPE"),
    ("heads", lambda t, a: a.update(k=view(t, [2, 7, 3, 16], at=1), v=view(t, [2, 7, 3, 16], at=2),
                                    dk=view(t, [2, 7, 3, 16], at=8), dv=view(t, [2, 7, 3, 16], at=9)), "ERR_SHAPE"),
    ("no key heads", lambda t, a: a.update(k=view(t, [2, 7, 0, 16], at=1), v=view(t, [2, 7, 0, 16], at=2),
                                           dk=view(t, [2, 7, 0, 16], at=8), dv=view(t, [2, 7, 0, 16], at=9)), "ERR_SHAPE"),
    ("head size", lambda t, a: a.update(**{x: view(t, [1, 1, 1, 260], at=i) for i, x in
                                           ((0, "q"), (1, "k"), (2, "v"), (4, "out"), (6, "g"), (7, "dq"), (8, "dk"), (9, "dv"))}),
     "ERR_SHAPE"),
    ("empty head", lambda t, a: a.update(**{x: view(t, [1, 1, 1, 0], at=i) for i, x in
                                            ((0, "q"), (1, "k"), (2, "v"), (4, "out"), (6, "g"), (7, "dq"), (8, "dk"), (9, "dv"))}),
     "ERR_SHAPE"),
    ("scale", lambda t, a: a.update(scale=float("inf")), "ERR_ARG"),
    ("scale beyond f32", lambda t, a: a.update(scale=1e300), "ERR_ARG"),
    ("lse shape", lambda t, a: a.update(lse=view(t, [2, 5, 4], at=5)), "ERR_SHAPE"),
    ("lse type", lambda t, a: a.update(lse=view(t, [2, 4, 5], t.F64, 5)), "ERR_DTYPE"),
    ("lengths type", lambda t, a: a.update(n=view(t, [2], t.F32, 3)), "ERR_DTYPE"),
    ("lengths shape", lambda t, a: a.update(n=view(t, [3], t.I64, 3)), "ERR_SHAPE"),
    ("outside its storage", lambda t, a: a.update(v=view(t, K, at=2, storage_len=10)), "ERR_VIEW"),
]
FORWARD = [
    ("output over q", lambda t, a: a.update(out=view(t, Q, at=0)), "ERR_ALIAS"),
    ("output over v", lambda t, a: a.update(out=view(t, Q, at=2)), "ERR_ALIAS"),
    ("output over the lengths", lambda t, a: a.update(out=view(t, Q, at=3)), "ERR_ALIAS"),
    ("lse over the output", lambda t, a: a.update(lse=view(t, [2, 4, 5], at=4)), "ERR_ALIAS"),
    ("colliding output", lambda t, a: a.update(out=view(t, Q, at=4, strides=[0, 64, 16, 1])), "ERR_ALIAS"),
    ("colliding lse", lambda t, a: a.update(lse=view(t, [2, 4, 5], at=5, strides=[20, 5, 0])), "ERR_ALIAS"),
]
BACKWARD = [
    ("null lse", lambda t, a: a.update(lse=None), "ERR_ARG"),
    ("null gradient", lambda t, a: a.update(g=None), "ERR_ARG"),
    ("null dk", lambda t, a: a.update(dk=None), "ERR_ARG"),
    ("gradient shape", lambda t, a: a.update(g=view(t, K, at=6)), "ERR_SHAPE"),
    ("dq shape", lambda t, a: a.update(dq=view(t, K, at=7)), "ERR_SHAPE"),
    ("dv shape", lambda t, a: a.update(dv=view(t, Q, at=9)), "ERR_SHAPE"),
    ("dk type", lambda t, a: a.update(dk=view(t, K, t.F64, 8)), "ERR_DTYPE"),
    ("dq over q", lambda t, a: a.update(dq=view(t, Q, at=0)), "ERR_ALIAS"),
    ("dq over the output", lambda t, a: a.update(dq=view(t, Q, at=4)), "ERR_ALIAS"),
    ("dk over dv", lambda t, a: a.update(dk=view(t, K, at=9)), "ERR_ALIAS"),
    ("dq over the gradient", lambda t, a: a.update(dq=view(t, Q, at=6)), "ERR_ALIAS"),
    ("colliding dk", lambda t, a: a.update(dk=view(t, K, at=8, strides=[224, 32, 0, 1])), "ERR_ALIAS"),
]
CASES = [(f, *c) for f in (forward, backward) for c in BOTH] + [(forward, *c) for c in FORWARD] + [(backward, *c) for c in BACKWARD]


@pytest.mark.parametrize("call,what,change,status", CASES, ids=[f"{c[0].__name__} {c[1]}" for c in CASES])
def test_refusals(trs, call, what, change, status):
    a = good(trs)
    change(trs, a)
    with pytest.raises(trs.TrsError) as e:
        call(trs, a)
    assert e.value.status == getattr(trs, status), e.value
