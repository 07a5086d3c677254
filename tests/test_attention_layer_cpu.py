"""What the attention layer's operators refuse beyond their shapes, before any
GPU call."""
from __future__ import annotations

import ctypes

import pytest
import torch

BASE = 1 << 24


def view(trs, shape, dtype=None, at=0):
    return trs.make_view(BASE + (at << 40), trs.F32 if dtype is None else dtype, shape)


@pytest.mark.parametrize("scale", [2.0**127, -3.0e38, float("inf"), float("nan")])
def test_scales_whose_log2_form_leaves_f32(trs, scale):
    """S is taken in units of log2: the scale times log2 e has to be an f32."""
    q, k, lse = [1, 5, 1, 16], [1, 7, 1, 16], [1, 1, 5]
    v = [view(trs, s, at=i) for i, s in enumerate((q, k, k, q, lse, q, q, k, k))]
    r = [ctypes.byref(x) for x in v]
    lib = trs.load()
    assert lib.trs_cross_attention(r[0], r[1], r[2], None, scale, r[3], r[4], None) == trs.ERR_ARG
    assert lib.trs_cross_attention_backward(r[5], r[0], r[1], r[2], None, r[3], r[4], scale, r[6], r[7], r[8], None) == trs.ERR_ARG


@pytest.mark.parametrize("hq,hk", [(2**31, None), (2**31 - 8, None), (2**30, 2**30), (1, 2**32 + 1)])
def test_more_heads_than_32_bits_count(trs, hq, hk):
    views = {"q": view(trs, [1, 1, hq, 2]), "qo": view(trs, [1, 1, hq, 2], at=1), "pos": view(trs, [1], trs.I64, 2),
             "fr": view(trs, [1], trs.F64, 3)}
    if hk:
        views.update(k=view(trs, [1, 1, hk, 2], at=4), ko=view(trs, [1, 1, hk, 2], at=5))
    r = {n: ctypes.byref(v) for n, v in views.items()}
    k, ko = r.get("k"), r.get("ko")
    lib = trs.load()
    assert lib.trs_rotary(r["q"], k, r["pos"], r["fr"], 0, 1.0, r["qo"], ko, None) == trs.ERR_SHAPE
    assert lib.trs_head_norm_rotary(r["q"], k, None, None, 1e-6, r["pos"], r["fr"], 0, 1.0, r["qo"], ko, None) == trs.ERR_SHAPE


def test_inputs_on_another_device_are_refused(trs, monkeypatch):
    from tensorrs_b200 import device
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)

    def on(where, *args):
        v = view(trs, *args)
        v.device = where
        return v

    x, pos, f, n = (1, 1, 1, 2), on(0, [1], trs.I64), on(0, [1], trs.F64), on(1, [1], trs.I64)
    here, there, out = on(0, x), on(1, x), torch.empty(x)
    calls = [lambda: device.rotary(there, None, pos, f, out, None), lambda: device.rotary(here, there, pos, f, out, out),
             lambda: device.rotary_backward(here, None, n, f, out, None),
             lambda: device.head_norm_rotary(here, None, on(1, [2]), None, 1e-6, pos, f, out, None),
             lambda: device.head_norm_rotary_backward(here, None, there, None, None, None, 1e-6, pos, f, out, None, None, None),
             lambda: device.cross_attention(here, there, here, 1.0, out),
             lambda: device.cross_attention(here, here, here, 1.0, out, key_lengths=n),
             lambda: device.cross_attention_backward(here, here, here, there, here, here, 1.0, out, out, out)]
    for call in calls:
        with pytest.raises(ValueError, match="another device"):
            call()
