"""What trs_rotary, trs_head_norm_rotary, their gradients and
trs_rotary_frequencies refuse.  Every refusal comes before any GPU call, so
these run without one."""
from __future__ import annotations

import ctypes

import pytest

BASE = 1 << 24  # a 16-byte aligned fake device address; a refused call never dereferences it


def view(trs, shape, dtype=None, at=0, strides=None, offset=0, **kw):
    return trs.make_view(BASE + (at << 24), trs.F32 if dtype is None else dtype, shape, strides, offset, **kw)


def good(trs):
    return {"q": view(trs, [2, 3, 4, 16], at=0), "k": view(trs, [2, 3, 2, 16], at=1),
            "pos": view(trs, [2, 3], trs.I64, 2), "fr": view(trs, [8], trs.F64, 3), "layout": 0, "m": 1.0,
            "qo": view(trs, [2, 3, 4, 16], at=4), "ko": view(trs, [2, 3, 2, 16], at=5),
            "gq": view(trs, [16], at=6), "gk": view(trs, [16], at=7),
            "dq": view(trs, [2, 3, 4, 16], at=8), "dk": view(trs, [2, 3, 2, 16], at=9),
            "dgq": view(trs, [16], at=10), "dgk": view(trs, [16], at=11)}


def ref(v):
    return ctypes.byref(v) if v is not None else None


def rotary(trs, a):
    return trs.check(trs.load().trs_rotary(ref(a["q"]), ref(a["k"]), ref(a["pos"]), ref(a["fr"]), a["layout"], a["m"],
                                           ref(a["qo"]), ref(a["ko"]), None))


def backward(trs, a):
    return trs.check(trs.load().trs_head_norm_rotary_backward(
        ref(a["dq"]), ref(a["dk"]), ref(a["q"]), ref(a["k"]), ref(a["gq"]), ref(a["gk"]), 1e-6, ref(a["pos"]),
        ref(a["fr"]), a["layout"], a["m"], ref(a["qo"]), ref(a["ko"]), ref(a["dgq"]), ref(a["dgk"]), None))


CASES = [
    ("null q", lambda t, a: a.update(q=None), "ERR_ARG"),
    ("null positions", lambda t, a: a.update(pos=None), "ERR_ARG"),
    ("k without its output", lambda t, a: a.update(ko=None), "ERR_ARG"),
    ("layout", lambda t, a: a.update(layout=2), "ERR_ARG"),
    ("rank 3", lambda t, a: a.update(q=view(t, [6, 4, 16])), "ERR_SHAPE"),
    ("integers", lambda t, a: a.update(q=view(t, [2, 3, 4, 16], t.I32)), "ERR_DTYPE"),
    ("mixed types", lambda t, a: a.update(k=view(t, [2, 3, 2, 16], t.F64, 1)), "ERR_DTYPE"),
    ("output type", lambda t, a: a.update(qo=view(t, [2, 3, 4, 16], t.F64, 4)), "ERR_DTYPE"),
    ("output shape", lambda t, a: a.update(qo=view(t, [2, 3, 4, 8], at=4)), "ERR_SHAPE"),
    ("k tokens", lambda t, a: a.update(k=view(t, [2, 4, 2, 16], at=1), ko=view(t, [2, 4, 2, 16], at=5),
                                       dk=view(t, [2, 4, 2, 16], at=9)), "ERR_SHAPE"),
    ("k head size", lambda t, a: a.update(k=view(t, [2, 3, 2, 8], at=1), ko=view(t, [2, 3, 2, 8], at=5),
                                          dk=view(t, [2, 3, 2, 8], at=9), gk=None, dgk=None), "ERR_SHAPE"),
    ("float positions", lambda t, a: a.update(pos=view(t, [2, 3], t.F32, 2)), "ERR_DTYPE"),
    ("positions shape", lambda t, a: a.update(pos=view(t, [2, 4], t.I64, 2)), "ERR_SHAPE"),
    ("positions batch", lambda t, a: a.update(pos=view(t, [3, 3], t.I64, 2)), "ERR_SHAPE"),
    ("positions rank", lambda t, a: a.update(pos=view(t, [2, 3, 1], t.I64, 2)), "ERR_SHAPE"),
    ("f32 frequencies", lambda t, a: a.update(fr=view(t, [8], t.F32, 3)), "ERR_DTYPE"),
    ("no frequencies", lambda t, a: a.update(fr=view(t, [0], t.F64, 3)), "ERR_SHAPE"),
    ("too many frequencies", lambda t, a: a.update(fr=view(t, [9], t.F64, 3)), "ERR_SHAPE"),
    ("outside its storage", lambda t, a: a.update(q=view(t, [2, 3, 4, 16], storage_len=100)), "ERR_VIEW"),
    ("colliding output", lambda t, a: a.update(qo=view(t, [2, 3, 4, 16], at=4, strides=[192, 64, 0, 1])), "ERR_ALIAS"),
    ("output over another layout of q", lambda t, a: a.update(qo=view(t, [2, 3, 4, 16], strides=[192, 16, 48, 1])), "ERR_ALIAS"),
    ("output over k", lambda t, a: a.update(qo=view(t, [2, 3, 4, 16], at=1)), "ERR_ALIAS"),
    ("outputs over each other", lambda t, a: a.update(ko=view(t, [2, 3, 2, 16], at=4)), "ERR_ALIAS"),
    ("output over the positions", lambda t, a: a.update(qo=view(t, [2, 3, 4, 16], at=2)), "ERR_ALIAS"),
    ("head size", lambda t, a: a.update(q=view(t, [1, 1, 1, 514]), qo=view(t, [1, 1, 1, 514], at=4), k=None, ko=None, dk=None,
                                        dq=view(t, [1, 1, 1, 514], at=8), pos=view(t, [1], t.I64, 2), gq=None, gk=None,
                                        dgq=None, dgk=None), "ERR_SHAPE"),
]


@pytest.mark.parametrize("what,change,status", CASES, ids=[c[0] for c in CASES])
@pytest.mark.parametrize("call", [rotary, backward])
def test_refusals(trs, call, what, change, status):
    a = good(trs)
    change(trs, a)
    with pytest.raises(trs.TrsError) as e:
        call(trs, a)
    assert e.value.status == getattr(trs, status), e.value


@pytest.mark.parametrize("what,change,status", [
    ("gamma size", lambda t, a: a.update(gq=view(t, [8], at=6)), "ERR_SHAPE"),
    ("gamma type", lambda t, a: a.update(gk=view(t, [16], t.F64, 7)), "ERR_DTYPE"),
    ("gamma rank", lambda t, a: a.update(gq=view(t, [1, 16], at=6)), "ERR_SHAPE"),
    ("gamma of no keys", lambda t, a: a.update(k=None, ko=None, dk=None, dgk=None), "ERR_ARG"),
    ("null gradient", lambda t, a: a.update(dq=None), "ERR_ARG"),
    ("gradient shape", lambda t, a: a.update(dk=view(t, [2, 3, 4, 16], at=9)), "ERR_SHAPE"),
    ("gamma gradient over gamma", lambda t, a: a.update(dgq=view(t, [16], at=6)), "ERR_ALIAS"),
    ("colliding gamma gradient", lambda t, a: a.update(dgq=view(t, [16], at=10, strides=[0])), "ERR_ALIAS"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_backward_refusals(trs, what, change, status):
    a = good(trs)
    change(trs, a)
    with pytest.raises(trs.TrsError) as e:
        backward(trs, a)
    assert e.value.status == getattr(trs, status), e.value


@pytest.mark.parametrize("args,status", [
    ((1.0, 0, 1.0, 1, 32, 0), "ERR_ARG"), ((float("nan"), 0, 1.0, 1, 32, 0), "ERR_ARG"), ((1e4, 5, 1.0, 1, 32, 0), "ERR_ARG"),
    ((1e4, 1, 0.0, 1, 32, 0), "ERR_ARG"), ((1e4, 3, 8.0, 4, 4, 8192), "ERR_ARG"), ((1e4, 4, 8.0, 1, 32, 0), "ERR_ARG"),
], ids=str)
def test_frequency_refusals(trs, args, status):
    with pytest.raises(trs.TrsError) as e:
        trs.check(trs.load().trs_rotary_frequencies(*args, ref(view(trs, [8], trs.F64)), None))
    assert e.value.status == getattr(trs, status)


@pytest.mark.parametrize("shape,dtype,status", [([8], "F32", "ERR_DTYPE"), ([2, 4], "F64", "ERR_SHAPE"), ([0], "F64", "ERR_SHAPE"),
                                                ([257], "F64", "ERR_SHAPE")], ids=str)
def test_frequency_view_refusals(trs, shape, dtype, status):
    with pytest.raises(trs.TrsError) as e:
        trs.check(trs.load().trs_rotary_frequencies(1e4, 0, 1.0, 1, 32, 0, ref(view(trs, shape, getattr(trs, dtype))), None))
    assert e.value.status == getattr(trs, status)
