"""What the last layer's entry points (trs_linear_cross_entropy,
trs_linear_distillation and their gradients) refuse, before any GPU call."""
from __future__ import annotations

import ctypes

import pytest

BASE = 1 << 24


def view(trs, shape, dtype=None, at=0, strides=None, **kw):
    return trs.make_view(BASE + (at << 24), trs.F32 if dtype is None else dtype, shape, strides, **kw)


def good(trs):
    return {"h": view(trs, [2, 5, 16], at=0), "w": view(trs, [11, 16], at=1), "t": view(trs, [2, 5], trs.I64, 2),
            "ids": view(trs, [2, 5, 4], trs.I64, 3), "z": view(trs, [2, 5, 4], at=4), "s": 0.1, "temp": 2.0,
            "loss": view(trs, [2, 5], at=5), "lse": view(trs, [2, 5], at=6), "g": view(trs, [2, 5], at=7),
            "dh": view(trs, [2, 5, 16], at=8), "dw": view(trs, [11, 16], at=9)}


def ref(v):
    return ctypes.byref(v) if v is not None else None


def ce(trs, a):
    return trs.check(trs.load().trs_linear_cross_entropy(ref(a["h"]), ref(a["w"]), ref(a["t"]), a["s"], ref(a["loss"]),
                                                         ref(a["lse"]), None))


def ce_backward(trs, a):
    return trs.check(trs.load().trs_linear_cross_entropy_backward(
        ref(a["g"]), ref(a["h"]), ref(a["w"]), ref(a["t"]), ref(a["lse"]), a["s"], ref(a["dh"]), ref(a["dw"]), None))


def kd(trs, a):
    return trs.check(trs.load().trs_linear_distillation(ref(a["h"]), ref(a["w"]), ref(a["ids"]), ref(a["z"]), a["temp"],
                                                        ref(a["loss"]), ref(a["lse"]), None))


def kd_backward(trs, a):
    return trs.check(trs.load().trs_linear_distillation_backward(
        ref(a["g"]), ref(a["h"]), ref(a["w"]), ref(a["ids"]), ref(a["z"]), ref(a["lse"]), a["temp"], ref(a["dh"]),
        ref(a["dw"]), None))


ALL, FORWARD, BACKWARD = (ce, ce_backward, kd, kd_backward), (ce, kd), (ce_backward, kd_backward)
CASES = [
    (ALL, "null hidden", lambda t, a: a.update(h=None), "ERR_ARG"),
    (ALL, "null weight", lambda t, a: a.update(w=None), "ERR_ARG"),
    ((ce, ce_backward), "null targets", lambda t, a: a.update(t=None), "ERR_ARG"),
    ((kd, kd_backward), "null ids", lambda t, a: a.update(ids=None), "ERR_ARG"),
    ((kd, kd_backward), "null logits", lambda t, a: a.update(z=None), "ERR_ARG"),
    (FORWARD, "null loss", lambda t, a: a.update(loss=None), "ERR_ARG"),
    (BACKWARD, "null lse", lambda t, a: a.update(lse=None), "ERR_ARG"),
    (BACKWARD, "null loss gradient", lambda t, a: a.update(g=None), "ERR_ARG"),
    (BACKWARD, "no gradient asked for", lambda t, a: a.update(dh=None, dw=None), "ERR_ARG"),
    (ALL, "hidden rank 1", lambda t, a: a.update(h=view(t, [16])), "ERR_SHAPE"),
    (ALL, "hidden rank 4", lambda t, a: a.update(h=view(t, [2, 5, 4, 4])), "ERR_SHAPE"),
    (ALL, "weight rank", lambda t, a: a.update(w=view(t, [11, 4, 4], at=1)), "ERR_SHAPE"),
    (ALL, "width", lambda t, a: a.update(w=view(t, [11, 8], at=1)), "ERR_SHAPE"),
    (ALL, "empty vocabulary", lambda t, a: a.update(w=view(t, [0, 16], at=1), dw=view(t, [0, 16], at=9)), "ERR_SHAPE"),
    (ALL, "empty width", lambda t, a: a.update(h=view(t, [2, 5, 0]), w=view(t, [11, 0], at=1), dh=view(t, [2, 5, 0], at=8),
                                               dw=view(t, [11, 0], at=9)), "ERR_SHAPE"),
    ((ce, ce_backward), "targets shape", lambda t, a: a.update(t=view(t, [2, 4], t.I64, 2)), "ERR_SHAPE"),
    ((ce, ce_backward), "targets rank", lambda t, a: a.update(t=view(t, [10], t.I64, 2)), "ERR_SHAPE"),
    ((ce, ce_backward), "float targets", lambda t, a: a.update(t=view(t, [2, 5], t.F32, 2)), "ERR_DTYPE"),
    ((ce, ce_backward), "smoothing above 1", lambda t, a: a.update(s=1.01), "ERR_ARG"),
    ((ce, ce_backward), "smoothing below 0", lambda t, a: a.update(s=-0.1), "ERR_ARG"),
    ((ce, ce_backward), "smoothing NaN", lambda t, a: a.update(s=float("nan")), "ERR_ARG"),
    ((kd, kd_backward), "float ids", lambda t, a: a.update(ids=view(t, [2, 5, 4], t.F64, 3)), "ERR_DTYPE"),
    ((kd, kd_backward), "f64 logits", lambda t, a: a.update(z=view(t, [2, 5, 4], t.F64, 4)), "ERR_DTYPE"),
    ((kd, kd_backward), "ids and logits", lambda t, a: a.update(z=view(t, [2, 5, 3], at=4)), "ERR_SHAPE"),
    ((kd, kd_backward), "ids rank", lambda t, a: a.update(ids=view(t, [2, 5], t.I64, 3)), "ERR_SHAPE"),
    ((kd, kd_backward), "no entries", lambda t, a: a.update(ids=view(t, [2, 5, 0], t.I64, 3), z=view(t, [2, 5, 0], at=4)), "ERR_SHAPE"),
    ((kd, kd_backward), "too many entries", lambda t, a: a.update(ids=view(t, [2, 5, 1025], t.I64, 3), z=view(t, [2, 5, 1025], at=4)),
     "ERR_SHAPE"),
    ((kd, kd_backward), "temperature 0", lambda t, a: a.update(temp=0.0), "ERR_ARG"),
    ((kd, kd_backward), "temperature below 0", lambda t, a: a.update(temp=-1.0), "ERR_ARG"),
    ((kd, kd_backward), "temperature inf", lambda t, a: a.update(temp=float("inf")), "ERR_ARG"),
    ((kd, kd_backward), "temperature NaN", lambda t, a: a.update(temp=float("nan")), "ERR_ARG"),
    (FORWARD, "loss shape", lambda t, a: a.update(loss=view(t, [10], at=5)), "ERR_SHAPE"),
    (FORWARD, "loss type", lambda t, a: a.update(loss=view(t, [2, 5], t.F64, 5)), "ERR_DTYPE"),
    (ALL, "lse shape", lambda t, a: a.update(lse=view(t, [5, 2], at=6)), "ERR_SHAPE"),
    (ALL, "lse type", lambda t, a: a.update(lse=view(t, [2, 5], t.F64, 6)), "ERR_DTYPE"),
    (ALL, "f64 hidden", lambda t, a: a.update(h=view(t, [2, 5, 16], t.F64)), "ERR_DTYPE"),
    (ALL, "f64 weight", lambda t, a: a.update(w=view(t, [11, 16], t.F64, 1)), "ERR_DTYPE"),
    (BACKWARD, "loss gradient shape", lambda t, a: a.update(g=view(t, [2], at=7)), "ERR_SHAPE"),
    (BACKWARD, "hidden gradient shape", lambda t, a: a.update(dh=view(t, [2, 5, 15], at=8)), "ERR_SHAPE"),
    (BACKWARD, "weight gradient shape", lambda t, a: a.update(dw=view(t, [16, 11], at=9)), "ERR_SHAPE"),
    (BACKWARD, "weight gradient type", lambda t, a: a.update(dw=view(t, [11, 16], t.F64, 9)), "ERR_DTYPE"),
    (ALL, "outside its storage", lambda t, a: a.update(w=view(t, [11, 16], at=1, storage_len=100)), "ERR_VIEW"),
    (FORWARD, "loss over hidden", lambda t, a: a.update(loss=view(t, [2, 5], at=0)), "ERR_ALIAS"),
    (FORWARD, "loss over lse", lambda t, a: a.update(loss=view(t, [2, 5], at=6)), "ERR_ALIAS"),
    (FORWARD, "colliding loss", lambda t, a: a.update(loss=view(t, [2, 5], at=5, strides=[0, 1])), "ERR_ALIAS"),
    (BACKWARD, "gradient over hidden", lambda t, a: a.update(dh=view(t, [2, 5, 16], at=0)), "ERR_ALIAS"),
    (BACKWARD, "gradient over the weight", lambda t, a: a.update(dw=view(t, [11, 16], at=1)), "ERR_ALIAS"),
    (BACKWARD, "gradients over each other", lambda t, a: a.update(dw=view(t, [11, 16], at=8)), "ERR_ALIAS"),
    (BACKWARD, "gradient over lse", lambda t, a: a.update(dh=view(t, [2, 5, 16], at=6)), "ERR_ALIAS"),
    (BACKWARD, "colliding gradient", lambda t, a: a.update(dw=view(t, [11, 16], at=9, strides=[1, 1])), "ERR_ALIAS"),
    (ALL, "too many tokens", lambda t, a: a.update(h=view(t, [1 << 30, 16]), t=view(t, [1 << 30], t.I32, 1 << 14),
                                                   ids=view(t, [1 << 30, 1], t.I32, 1 << 14), z=view(t, [1 << 30, 1], at=1 << 15),
                                                   loss=view(t, [1 << 30], at=1 << 16), lse=view(t, [1 << 30], at=1 << 17),
                                                   g=view(t, [1 << 30], at=1 << 18), dh=None), "ERR_SHAPE"),
    (ALL, "too large a vocabulary", lambda t, a: a.update(w=view(t, [1 << 30, 16], at=1 << 16), dw=None), "ERR_SHAPE"),
]


@pytest.mark.parametrize("call,name,change,status", [(f, n, c, s) for fs, n, c, s in CASES for f in fs],
                         ids=[f"{n}-{f.__name__}" for fs, n, c, s in CASES for f in fs])
def test_refused(trs, call, name, change, status):
    a = good(trs)
    change(trs, a)
    with pytest.raises(trs.TrsError) as e:
        call(trs, a)
    assert e.value.status == getattr(trs, status)


@pytest.mark.parametrize("call", FORWARD)
def test_no_tokens(trs, call):
    """A forward call without tokens launches nothing."""
    a = good(trs)
    a.update(h=view(trs, [0, 16]), t=view(trs, [0], trs.I64, 2), ids=view(trs, [0, 4], trs.I64, 3), z=view(trs, [0, 4], at=4),
             loss=view(trs, [0], at=5), lse=view(trs, [0], at=6))
    assert call(trs, a) == trs.OK
