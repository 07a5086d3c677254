"""What trs_embedding and trs_embedding_backward refuse, before any GPU call."""
from __future__ import annotations

import ctypes

import pytest

BASE = 1 << 24  # a 16-byte aligned fake device address; a refused call never dereferences it


def view(trs, shape, dtype=None, at=0, strides=None, **kw):
    return trs.make_view(BASE + (at << 24), trs.F32 if dtype is None else dtype, shape, strides, **kw)


def good(trs):
    return {"table": view(trs, [11, 16], at=0), "ids": view(trs, [2, 5], trs.I64, 1), "rows": view(trs, [2, 5, 16], at=2)}


def ref(v):
    return ctypes.byref(v) if v is not None else None


def forward(trs, a):
    return trs.check(trs.load().trs_embedding(ref(a["table"]), ref(a["ids"]), 1.0, ref(a["rows"]), None))


def backward(trs, a):
    return trs.check(trs.load().trs_embedding_backward(ref(a["rows"]), ref(a["ids"]), 1.0, 0, ref(a["table"]), None))


CASES = [
    ("null table", lambda t, a: a.update(table=None), "ERR_ARG"),
    ("null ids", lambda t, a: a.update(ids=None), "ERR_ARG"),
    ("null rows", lambda t, a: a.update(rows=None), "ERR_ARG"),
    ("null data", lambda t, a: a.update(rows=t.make_view(0, t.F32, [2, 5, 16])), "ERR_ARG"),
    ("table rank", lambda t, a: a.update(table=view(t, [11, 4, 4])), "ERR_SHAPE"),
    ("ids without a dimension", lambda t, a: a.update(ids=view(t, [], t.I64, 1), rows=view(t, [16], at=2)), "ERR_SHAPE"),
    ("ids rank", lambda t, a: a.update(ids=view(t, [2, 5, 1], t.I64, 1)), "ERR_SHAPE"),
    ("rows rank", lambda t, a: a.update(rows=view(t, [10, 16], at=2)), "ERR_SHAPE"),
    ("batch", lambda t, a: a.update(rows=view(t, [3, 5, 16], at=2)), "ERR_SHAPE"),
    ("tokens", lambda t, a: a.update(rows=view(t, [2, 4, 16], at=2)), "ERR_SHAPE"),
    ("width", lambda t, a: a.update(rows=view(t, [2, 5, 8], at=2)), "ERR_SHAPE"),
    ("float ids", lambda t, a: a.update(ids=view(t, [2, 5], t.F32, 1)), "ERR_DTYPE"),
    ("integer table", lambda t, a: a.update(table=view(t, [11, 16], t.I32), rows=view(t, [2, 5, 16], t.I32, 2)), "ERR_DTYPE"),
    ("mixed types", lambda t, a: a.update(rows=view(t, [2, 5, 16], t.F64, 2)), "ERR_DTYPE"),
    ("outside its storage", lambda t, a: a.update(table=view(t, [11, 16], storage_len=100)), "ERR_VIEW"),
    ("rows over the table", lambda t, a: a.update(rows=view(t, [2, 5, 16], at=0)), "ERR_ALIAS"),
    ("rows over the ids", lambda t, a: a.update(ids=view(t, [2, 5], t.I64, 2), table=view(t, [11, 16], at=2)), "ERR_ALIAS"),
    ("too many rows", lambda t, a: a.update(table=view(t, [(1 << 31) - 8192, 16])), "ERR_SHAPE"),
    ("too many tokens", lambda t, a: a.update(ids=view(t, [1 << 16, 1 << 15], t.I64, 1),
                                              rows=view(t, [1 << 16, 1 << 15, 16], at=1000)), "ERR_SHAPE"),
]


@pytest.mark.parametrize("call", [forward, backward])
@pytest.mark.parametrize("name,change,status", CASES, ids=[c[0] for c in CASES])
def test_refused(trs, call, name, change, status):
    a = good(trs)
    change(trs, a)
    with pytest.raises(trs.TrsError) as e:
        call(trs, a)
    assert e.value.status == getattr(trs, status)


def test_colliding_outputs(trs):
    a = good(trs)
    a["rows"] = view(trs, [2, 5, 16], at=2, strides=[80, 0, 1])
    with pytest.raises(trs.TrsError) as e:
        forward(trs, a)
    assert e.value.status == trs.ERR_ALIAS
    a = good(trs)
    a["table"] = view(trs, [11, 16], strides=[8, 1])
    with pytest.raises(trs.TrsError) as e:
        backward(trs, a)
    assert e.value.status == trs.ERR_ALIAS


def test_nothing_to_do(trs):
    """Calls without an element to write launch nothing."""
    a = good(trs)
    a["ids"], a["rows"] = view(trs, [0], trs.I64, 1), view(trs, [0, 16], at=2)
    assert forward(trs, a) == trs.OK
    a["table"] = view(trs, [0, 16])
    assert backward(trs, a) == trs.OK
    a = good(trs)
    a["table"], a["rows"] = view(trs, [11, 0]), view(trs, [2, 5, 0], at=2)
    assert forward(trs, a) == trs.OK and backward(trs, a) == trs.OK
