"""The operators of an attention layer in the order a layer calls them: the norm
of queries and keys with the rotation (frequencies from
trs_rotary_frequencies), the attention, and the gradients back to the
projection's output and the gammas; against automatic differentiation of the
formulas in 64 bits.

Normed heads have |q| <= 1.5 sqrt(D), so |S| <= 2.25 sqrt(D) = 18; q and k come
out of the norm off by 32 u of themselves (u = 2^-24), which moves a score by
64 * 18 u and a weight by twice that, 2300 u; the other steps add less than
200 u.  2500 u of the 2-norm bounds every result."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _gpu import to_host

pytestmark = pytest.mark.gpu

U = 2.0**-24


def rotate(x, cos, sin, layout):
    n = cos.shape[-1]
    if layout == "half":
        a, b, rest = x[..., :n], x[..., n:2 * n], x[..., 2 * n:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., 2 * n:]], -1)


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hk,D,R,layout", [
    (2, 65, 65, 4, 2, 64, 64, "half"), (3, 40, 100, 6, 3, 64, 32, "interleaved"), (1, 150, 33, 2, 1, 128, 128, "half"),
    (2, 1, 300, 4, 1, 64, 64, "half"), (2, 7, 50, 3, 3, 48, 24, "interleaved"),
])
def test_a_layer_forward_and_backward(B, Tq, Tk, Hq, Hk, D, R, layout):
    from tensorrs_b200 import device
    V = device.view_of
    g = torch.Generator().manual_seed(B + Tq + Tk)
    xq, kv = torch.randn(B, Tq, Hq, D, generator=g), torch.randn(B, Tk, 2, Hk, D, generator=g)
    gq, gk = 0.5 + torch.rand(D, generator=g), 0.5 + torch.rand(D, generator=g)
    w = torch.randn(B, Tq, Hq, D, generator=g)
    n = torch.randint(0, Tk + 1, (B,), generator=g)
    pq, pk = torch.arange(Tq) + Tk, torch.arange(Tk)
    eps, scale, m = 1e-6, D**-0.5, 1.1

    freqs = torch.empty(R // 2, dtype=torch.float64, device="cuda")
    device.rotary_frequencies(freqs, 10000.0, "ramp", 4.0, 1.0, 32.0, 2048.0)
    # the definition, differentiated
    q64, kv64, gq64, gk64 = (t.double().requires_grad_() for t in (xq, kv, gq, gk))
    f = freqs.cpu()

    def prepared(x, gamma, pos):
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gamma
        a = pos.double()[:, None, None] * f
        return rotate(x, torch.cos(a) * m, torch.sin(a) * m, layout)

    qr, kr = prepared(q64, gq64, pq), prepared(kv64[:, :, 0], gk64, pk)
    rep = Hq // Hk
    S = torch.einsum("bthd,bshd->bhts", qr, kr.repeat_interleave(rep, 2)) * scale
    S = S.masked_fill(torch.arange(Tk) >= n[:, None, None, None], -np.inf)
    P = torch.nan_to_num(torch.softmax(S, -1), 0.0)  # a batch without keys
    out64 = torch.einsum("bhts,bshd->bthd", P, kv64[:, :, 1].repeat_interleave(rep, 2))
    want = [out64, *torch.autograd.grad((out64 * w).sum(), [q64, kv64, gq64, gk64])]

    # the layer
    xq, kv, gq, gk, w, n, pq, pk = (t.cuda() for t in (xq, kv, gq, gk, w, n, pq, pk))
    k, v = kv[:, :, 0], kv[:, :, 1]
    vf = V(freqs)
    qr, kr, out = torch.empty_like(xq), torch.empty(k.shape, device="cuda"), torch.empty_like(xq)
    lse = torch.empty(B, Hq, Tq, device="cuda")
    kw = {"layout": layout, "magnitude": m}
    device.head_norm_rotary(V(xq), None, V(gq), None, eps, V(pq), vf, qr, None, **kw)
    device.head_norm_rotary(V(k), None, V(gk), None, eps, V(pk), vf, kr, None, **kw)
    device.cross_attention(V(qr), V(kr), V(v), scale, out, lse=lse, key_lengths=V(n))
    dq, dkv = torch.empty_like(xq), torch.empty_like(kv)
    dgq, dgk = torch.empty_like(gq), torch.empty_like(gk)
    device.cross_attention_backward(V(w), V(qr), V(kr), V(v), V(out), V(lse), scale, dq, dkv[:, :, 0], dkv[:, :, 1],
                                    key_lengths=V(n))
    # in place: the gradients of the rotated heads become those of the projection's output
    device.head_norm_rotary_backward(V(dq), None, V(xq), None, V(gq), None, eps, V(pq), vf, dq, None, dgq, None, **kw)
    dk = dkv[:, :, 0]
    device.head_norm_rotary_backward(V(dk), None, V(k), None, V(gk), None, eps, V(pk), vf, dk, None, dgk, None, **kw)
    for name, got, ref in zip(("out", "dq", "dkv", "dgq", "dgk"), (out, dq, dkv, dgq, dgk), want):
        ref = ref.detach().numpy()
        far = np.linalg.norm(to_host(got).astype(np.float64) - ref)
        assert far <= 2500 * U * np.linalg.norm(ref), (name, far / np.linalg.norm(ref))


def test_generation_agrees_with_the_prompt():
    """Tokens rotated and attended one by one (the single-token kernels) against all of them at once."""
    from tensorrs_b200 import device
    V = device.view_of
    torch.manual_seed(3)
    q, k, v = torch.randn(2, 40, 4, 64, device="cuda"), torch.randn(2, 90, 2, 64, device="cuda"), torch.randn(2, 90, 2, 64, device="cuda")
    freqs = torch.empty(32, dtype=torch.float64, device="cuda")
    device.rotary_frequencies(freqs)
    pos = torch.arange(40, device="cuda")
    whole, qr = torch.empty_like(q), torch.empty_like(q)
    device.rotary(V(q), None, V(pos), V(freqs), qr, None)
    device.cross_attention(V(qr), V(k), V(v), 0.125, whole)
    for t in range(0, 40, 7):
        one, o = torch.empty(2, 1, 4, 64, device="cuda"), torch.empty(2, 1, 4, 64, device="cuda")
        device.rotary(V(q[:, t:t + 1]), None, V(pos[t:t + 1]), V(freqs), one, None)
        assert torch.equal(one, qr[:, t:t + 1])
        device.cross_attention(V(one), V(k), V(v), 0.125, o)
        # both within 32 u + 4 u |S| of the definition, |S| < 8
        assert (o - whole[:, t:t + 1]).norm() <= 128 * U * o.norm()


def test_offsets_past_32_bits():
    """Rows 2^30 elements apart inside one buffer of 8.6 GB: rotation, both attention paths and the gradient."""
    from tensorrs_b200 import device
    V = device.view_of
    step = 2**30
    free, _ = torch.cuda.mem_get_info()
    if free < 20 * 2**30:
        pytest.skip("needs 20 GB of free memory")
    buf = torch.empty(2 * step + 40 * 64, device="cuda")
    far = buf.as_strided((3, 40, 1, 64), (step, 64, 64, 1))
    near = torch.randn(3, 40, 1, 64, device="cuda")
    far.copy_(near)
    freqs, pos = torch.empty(32, dtype=torch.float64, device="cuda"), torch.arange(40, device="cuda")
    device.rotary_frequencies(freqs)
    a, b = torch.empty_like(near), torch.empty_like(near)
    device.rotary(V(far), None, V(pos), V(freqs), a, None)
    device.rotary(V(near), None, V(pos), V(freqs), b, None)
    assert torch.equal(a, b)
    # tokens 2^30 apart as keys: [1, 3, 40, 64] with the batch as tokens
    kf, kn = far.permute(2, 0, 1, 3), near.permute(2, 0, 1, 3)
    for Tq in (1, 33):
        q, g = torch.randn(1, Tq, 40, 64, device="cuda"), torch.randn(1, Tq, 40, 64, device="cuda")
        res = []
        for k in (kf, kn):
            o, lse = torch.empty_like(q), torch.empty(1, 40, Tq, device="cuda")
            device.cross_attention(V(q), V(k), V(k), 0.125, o, lse=lse)
            d = [torch.empty(q.shape, device="cuda"), torch.empty(1, 3, 40, 64, device="cuda"), torch.empty(1, 3, 40, 64, device="cuda")]
            device.cross_attention_backward(V(g), V(q), V(k), V(k), V(o), V(lse), 0.125, *d)
            res.append([o, *d])
        for x, y in zip(*res):
            assert torch.equal(x, y)
    # and as an output
    device.rotary(V(near), None, V(pos), V(freqs), far, None)
    assert torch.equal(far, b)


def test_outputs_on_another_device_are_refused(monkeypatch):
    from tensorrs_b200 import device
    V = device.view_of
    x, pos = torch.randn(1, 1, 1, 2, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    f = torch.ones(1, dtype=torch.float64, device="cuda")
    views, out = (V(x), None, V(pos), V(f)), torch.empty_like(x)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 7)
    with pytest.raises(ValueError, match="another device"):
        device.rotary(*views, out, None)


@pytest.mark.parametrize("where", ["heads", "batch", "tokens", "elements"])
def test_slices_that_share_a_buffer_but_no_element(where):
    """Queries, keys and values interleaved inside one buffer, in any order of its dimensions, rotated in place; the
    gradients of attention written into such a buffer."""
    from tensorrs_b200 import device
    V = device.view_of
    torch.manual_seed(4)
    B, T, H, D = 2, 9, 3, 16
    # the place of the (q, k, v) dimension and how the slice becomes [B, T, H, D]
    shape, cut = {"heads": ((B, T, H, 3, D), lambda x, i: x[:, :, :, i]),
                  "batch": ((B, 3, H, T, D), lambda x, i: x[:, i].transpose(1, 2)),
                  "tokens": ((B, H, T, 3, D), lambda x, i: x[:, :, :, i].transpose(1, 2)),
                  "elements": ((B, T, H, D, 3), lambda x, i: x[..., i])}[where]
    buf = torch.randn(shape, device="cuda")
    q, k, v = (cut(buf, i) for i in range(3))
    w, pos = torch.randn(B, T, H, D, device="cuda"), torch.arange(T, device="cuda")
    freqs = torch.empty(D // 2, dtype=torch.float64, device="cuda")
    device.rotary_frequencies(freqs)
    apart = [torch.empty(B, T, H, D, device="cuda") for _ in range(2)]
    device.rotary(V(q), V(k), V(pos), V(freqs), *apart)
    kept = v.clone()
    device.rotary(V(q), V(k), V(pos), V(freqs), q, k)
    assert torch.equal(q, apart[0]) and torch.equal(k, apart[1]) and torch.equal(v, kept)
    out, lse = torch.empty(B, T, H, D, device="cuda"), torch.empty(B, H, T, device="cuda")
    device.cross_attention(V(q), V(k), V(v), 0.25, out, lse=lse)
    grads = [torch.empty(B, T, H, D, device="cuda") for _ in range(3)]
    device.cross_attention_backward(V(w), V(q), V(k), V(v), V(out), V(lse), 0.25, *grads)
    gbuf = torch.full(shape, float("nan"), device="cuda")
    device.cross_attention_backward(V(w), V(q), V(k), V(v), V(out), V(lse), 0.25, *(cut(gbuf, i) for i in range(3)))
    for i in range(3):
        assert torch.equal(cut(gbuf, i), grads[i])
