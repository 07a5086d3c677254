"""The operators of an attention layer measured next to their plain forms: rotary positions, the per-head norm of
queries and keys with the rotation in the same pass, and the attention of queries to the states of another length.

Every case is one call a program makes (a "train" case the forward and the backward call of one step), on f32 or f64
tensors of the layout [batch, tokens, heads, head size].  `own` False runs the plain form, elementary torch
operations; `own` True runs the calls of this package.
"""
import math

import torch

own = False

DEVICE = "cuda"


# ---- cases --------------------------------------------------------------------


def listed():
    return [
        # one new token of each of 16 sequences that stand far into their contexts: the rotation of a generation step,
        # where the time to issue the call counts
        _rotary("rotary_one_token", 16, 1, 16, 4, 64, 64, "half", "ramp", far=200_000),
        # a prompt of 2 x 4096 tokens, interleaved pairs over the first half of each head, q and k slices of one
        # projection's output
        _rotary("rotary_prompt_part_interleaved", 2, 4096, 32, 8, 128, 64, "interleaved", "none"),
        # the gradient of a training batch whose lengths fit nothing
        _rotary("rotary_backward_odd", 3, 1511, 13, 5, 80, 80, "half", "linear", direction="backward"),
        # the same rotation for a model kept in 64 bits
        _rotary("rotary_f64", 2, 1000, 12, 12, 64, 64, "half", "none", dtype="f64"),
        # norm and rotation of one new token of each of 16 sequences
        _norm("head_norm_one_token", 16, 1, 16, 4, 64, 64, "half", far=200_000),
        # norm and rotation of a prompt
        _norm("head_norm_prompt", 4, 2048, 32, 8, 128, 128, "half"),
        # a training step's forward and backward through norm and rotation
        _norm("head_norm_train", 2, 2048, 16, 4, 64, 64, "interleaved", direction="train"),
        # a step of generation: one query per sequence against encoder states of uneven lengths, one of them empty
        _cross("cross_one_token", 8, 1, 2048, 16, 16, 64, ragged=True),
        # a short prompt against a long document, eight query heads per group of keys
        _cross("cross_long_states", 1, 32, 32768, 32, 4, 128),
        # a decoder's prompt against a padded batch of encoder states
        _cross("cross_prompt", 4, 1024, 1500, 16, 16, 64, ragged=True),
        # a training step, forward and backward, with lengths that end inside every tile
        _cross("cross_train_odd", 3, 333, 777, 8, 2, 80, ragged=True, direction="train"),
        # the largest training step
        _cross("cross_train", 4, 2048, 2048, 16, 16, 64, direction="train"),
    ]


def _rotary(name, B, T, Hq, Hk, D, R, layout, scaling, direction="forward", dtype="f32", far=0):
    return {"name": name, "op": "rotary", "direction": direction, "B": B, "T": T, "Hq": Hq, "Hk": Hk, "D": D, "R": R,
            "layout": layout, "scaling": scaling, "dtype": dtype, "far": far}


def _norm(name, B, T, Hq, Hk, D, R, layout, scaling="none", direction="forward", dtype="f32", far=0):
    return {**_rotary(name, B, T, Hq, Hk, D, R, layout, scaling, direction, dtype, far), "op": "head_norm"}


def _cross(name, B, Tq, Tk, Hq, Hk, D, ragged=False, direction="forward"):
    return {"name": name, "op": "cross", "direction": direction, "B": B, "Tq": Tq, "Tk": Tk, "Hq": Hq, "Hk": Hk,
            "D": D, "ragged": ragged}


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "head_norm", "cross", "cross"])
    if op == "cross":
        direction = rng.choice(["forward", "forward", "train"])
        D = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 128, 128])
        Hk = rng.choice([1, 2, 3, 4, 8, 16])
        Hq = Hk * rng.choice([1, 1, 2, 4, 7])
        B = rng.randint(1, 8)
        Tq = rng.choice([1, _spread(rng, 1, 2048), _spread(rng, 64, 2048)])
        Tk = _spread(rng, 1, 32768)
        most = 4 * 16 * 2048 * 2048 * 64  # the largest listed case's products
        while B * Hq * Tq * Tk * D > most or B * Hq * Tq * Tk > 4 * 16 * 2048 * 2048 or B * Tk * Hk * D > 1 << 26:
            if B > 1:
                B //= 2
            else:
                Tk = max(1, Tk // 2)
                Tq = max(1, Tq - Tq // 4)
        c = _cross("", B, Tq, Tk, Hq, Hk, D, ragged=rng.random() < 0.5, direction=direction)
    else:
        D = rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128, 256])
        R = rng.choice([D, D, D // 2])
        Hk = rng.choice([1, 2, 4, 5, 8])
        Hq = Hk * rng.choice([1, 1, 3, 4])
        B, T = rng.randint(1, 16), rng.choice([1, _spread(rng, 1, 8192), _spread(rng, 64, 8192)])
        while B * T * (Hq + Hk) * D > 2 * 4096 * 40 * 128:
            T = max(1, T // 2)
        make = _rotary if op == "rotary" else _norm
        c = make("", B, T, Hq, Hk, D, R, rng.choice(["half", "interleaved"]),
                 rng.choice(["none", "linear", "ramp"]),
                 direction=rng.choice(["forward", "forward", "backward" if op == "rotary" else "train"]),
                 dtype=rng.choice(["f32", "f32", "f32", "f64"]), far=rng.choice([0, 0, 1000, 500_000]))
    del c["name"]
    return c


# ---- inputs -------------------------------------------------------------------


def _frequencies(c):
    """The table of angles per position (radians), one entry per rotated pair, in 64 bits; and the factor on the
    rotated values."""
    n = c["R"] // 2
    i = torch.arange(n, dtype=torch.float64)
    f = 10000.0 ** (-i / n)
    if c["scaling"] == "linear":
        return (f / 4.0).to(DEVICE), 1.0
    if c["scaling"] == "ramp":  # slow pairs interpolated by 8, fast ones kept, a linear ramp between
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return (f * keep + f / 8.0 * (1 - keep)).to(DEVICE), 0.1 * math.log(8.0) + 1.0
    return f.to(DEVICE), 1.0


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)

    if c["op"] == "cross":
        B, Tq, Tk, Hq, Hk, D = (c[k] for k in ("B", "Tq", "Tk", "Hq", "Hk", "D"))
        s = {"case": c, "scale": 1.0 / math.sqrt(D)}
        s["q"] = normal(B, Tq, Hq, D) * 1.5
        kv = normal(B, Tk, 2, Hk, D)  # keys and values are halves of one projection of the encoder's states
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        s["lengths"] = None
        if c["ragged"]:
            n = torch.randint(Tk // 2, Tk + 1, (B,), generator=g, device=DEVICE)
            if B > 2:
                n[1] = 0
            s["lengths"] = n
        if c["direction"] == "train":
            s["grad"] = normal(B, Tq, Hq, D)
        return s
    B, T, Hq, Hk, D = (c[k] for k in ("B", "T", "Hq", "Hk", "D"))
    dt = torch.float64 if c["dtype"] == "f64" else torch.float32
    qkv = normal(B, T, Hq + 2 * Hk, D, dtype=dt)  # one projection's output: queries, keys, values
    s = {"case": c, "q": qkv[:, :, :Hq], "k": qkv[:, :, Hq:Hq + Hk]}
    start = torch.randint(0, c["far"] + 1, (B, 1), generator=g, device=DEVICE)
    s["positions"] = start + torch.arange(T, device=DEVICE)
    s["freqs"], s["magnitude"] = _frequencies(c)
    if c["op"] == "head_norm":
        s["gq"] = 1.0 + 0.2 * normal(D, dtype=dt)
        s["gk"] = 1.0 + 0.2 * normal(D, dtype=dt)
        s["eps"] = 1e-6
        if c["direction"] == "train":
            s["dq"], s["dk"] = normal(B, T, Hq, D, dtype=dt), normal(B, T, Hk, D, dtype=dt)
    return s


# ---- one pass -------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from tensorrs_b200 import device as trs

    c = s["case"]
    if c["op"] == "cross":
        q, k, v = trs.view_of(s["q"]), trs.view_of(s["k"]), trs.view_of(s["v"])
        n = trs.view_of(s["lengths"]) if s["lengths"] is not None else None
        out = torch.empty_like(s["q"])
        if c["direction"] == "forward":
            return trs.cross_attention(q, k, v, s["scale"], out, key_lengths=n)
        lse = torch.empty((c["B"], c["Hq"], c["Tq"]), device=DEVICE)
        trs.cross_attention(q, k, v, s["scale"], out, lse=lse, key_lengths=n)
        dq, dk, dv = torch.empty_like(out), torch.empty(s["k"].shape, device=DEVICE), torch.empty(s["v"].shape, device=DEVICE)
        trs.cross_attention_backward(trs.view_of(s["grad"]), q, k, v, trs.view_of(out), trs.view_of(lse), s["scale"],
                                     dq, dk, dv, key_lengths=n)
        return out, dq, dk, dv
    q, k = trs.view_of(s["q"]), trs.view_of(s["k"])
    pos, fr = trs.view_of(s["positions"]), trs.view_of(s["freqs"])
    dt = s["q"].dtype
    qo = torch.empty(s["q"].shape, device=DEVICE, dtype=dt)
    ko = torch.empty(s["k"].shape, device=DEVICE, dtype=dt)
    kw = {"layout": c["layout"], "magnitude": s["magnitude"]}
    if c["op"] == "rotary":
        call = trs.rotary if c["direction"] == "forward" else trs.rotary_backward
        call(q, k, pos, fr, qo, ko, **kw)
        return qo, ko
    gq, gk = trs.view_of(s["gq"]), trs.view_of(s["gk"])
    trs.head_norm_rotary(q, k, gq, gk, s["eps"], pos, fr, qo, ko, **kw)
    if c["direction"] == "forward":
        return qo, ko
    dq, dk = torch.empty_like(qo), torch.empty_like(ko)
    dgq, dgk = torch.empty_like(s["gq"]), torch.empty_like(s["gk"])
    trs.head_norm_rotary_backward(trs.view_of(s["dq"]), trs.view_of(s["dk"]), q, k, gq, gk, s["eps"], pos, fr,
                                  dq, dk, dgq, dgk, **kw)
    return qo, ko, dq, dk, dgq, dgk


def _run_plain(s):
    c = s["case"]
    if c["op"] == "cross":
        return _plain_cross(s)
    angle = s["positions"].double()[:, :, None, None] * s["freqs"]
    dt = s["q"].dtype
    cos = (torch.cos(angle) * s["magnitude"]).to(dt)
    sin = (torch.sin(angle) * s["magnitude"]).to(dt)
    if c["op"] == "rotary":
        if c["direction"] == "backward":
            sin = -sin
        return _plain_rotate(c, s["q"], cos, sin), _plain_rotate(c, s["k"], cos, sin)
    nq, rq = _plain_norm(s["q"], s["eps"])
    nk, rk = _plain_norm(s["k"], s["eps"])
    qo, ko = _plain_rotate(c, nq * s["gq"], cos, sin), _plain_rotate(c, nk * s["gk"], cos, sin)
    if c["direction"] == "forward":
        return qo, ko
    dq, dgq = _plain_norm_backward(_plain_rotate(c, s["dq"], cos, -sin), nq, rq, s["gq"])
    dk, dgk = _plain_norm_backward(_plain_rotate(c, s["dk"], cos, -sin), nk, rk, s["gk"])
    return qo, ko, dq, dk, dgq, dgk


def _plain_rotate(c, x, cos, sin):
    R = c["R"]
    if c["layout"] == "half":
        a, b = x[..., :R // 2], x[..., R // 2:R]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., R:]], -1)
    a, b = x[..., 0:R:2], x[..., 1:R:2]
    r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([r, x[..., R:]], -1)


def _plain_norm(x, eps):
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r, r


def _plain_norm_backward(g, n, r, gamma):
    dn = g * gamma
    return r * (dn - n * (dn * n).mean(-1, keepdim=True)), (g * n).sum((0, 1, 2))


def _plain_cross(s):
    c = s["case"]
    B, Tq, Tk, Hq, Hk, D = (c[k] for k in ("B", "Tq", "Tk", "Hq", "Hk", "D"))
    G = Hq // Hk
    q = s["q"].reshape(B, Tq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Tq, D)
    k, v = s["k"].permute(0, 2, 1, 3), s["v"].permute(0, 2, 1, 3)
    sc = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    if s["lengths"] is not None:
        gone = torch.arange(Tk, device=DEVICE) >= s["lengths"][:, None]
        sc = sc.masked_fill(gone[:, None, None, :], -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(sc - m)
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, torch.ones_like(l), l)
    o = torch.matmul(p, v)
    back = lambda x: x.reshape(B, Hk, G, Tq, D).permute(0, 3, 1, 2, 4).reshape(B, Tq, Hq, D)  # noqa: E731
    if c["direction"] == "forward":
        return back(o)
    g = s["grad"].reshape(B, Tq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Tq, D)
    dv = torch.matmul(p.transpose(-1, -2), g)
    dp = torch.matmul(g, v.transpose(-1, -2))
    ds = p * (dp - (g * o).sum(-1, keepdim=True)) * s["scale"]
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q)
    return back(o), back(dq), dk.permute(0, 2, 1, 3).contiguous(), dv.permute(0, 2, 1, 3).contiguous()


# ---- the floor ----------------------------------------------------------------


def work(case):
    c = case
    if c["op"] == "cross":
        B, Tq, Tk, Hq, Hk, D = (c[k] for k in ("B", "Tq", "Tk", "Hq", "Hk", "D"))
        # lengths of a ragged batch are uniform over the upper half, and one sequence of three or more is empty
        keys = B * Tk if not c["ragged"] else 0.75 * Tk * (B - 1 if B > 2 else B)
        qb, kb = 4 * B * Tq * Hq * D, 4 * keys * Hk * D
        if c["direction"] == "forward":
            return {"bytes": int(2 * qb + 2 * kb), "flops": int(4 * Tq * keys * Hq * D)}
        # forward, then q, k, v, out and the gradient again, and three gradients; seven products in all
        return {"bytes": int(2 * qb + 2 * kb + 4 * qb + 2 * kb + 2 * 4 * B * Tk * Hk * D),
                "flops": int(14 * Tq * keys * Hq * D)}
    es = 8 if c["dtype"] == "f64" else 4
    n = c["B"] * c["T"] * (c["Hq"] + c["Hk"]) * c["D"]
    pos = 8 * c["B"] * c["T"] + 4 * c["R"]
    if c["op"] == "rotary":
        return {"bytes": 2 * es * n + pos, "flops": 3 * n}
    if c["direction"] == "forward":
        return {"bytes": 2 * es * n + pos + 2 * es * c["D"], "flops": 7 * n}
    return {"bytes": 5 * es * n + 2 * pos + 6 * es * c["D"], "flops": 24 * n}


# ---- the definition in 64 bits ---------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cross":
        return _exact_cross(case, s)
    c = case
    angle = torch.einsum("bt,f->btf", s["positions"].double(), s["freqs"])
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, :, None]  # magnitude * exp(i angle)

    def rotate(x, turn):
        R = c["R"]
        y = x[..., :R]
        y = y.unflatten(-1, (2, R // 2)).transpose(-1, -2) if c["layout"] == "half" else y.unflatten(-1, (R // 2, 2))
        y = torch.view_as_real(torch.view_as_complex(y.contiguous()) * turn)
        y = (y.transpose(-1, -2) if c["layout"] == "half" else y).flatten(-2)
        return torch.cat((y, x[..., R:]), -1)

    q, k = s["q"].double(), s["k"].double()
    if c["op"] == "rotary":
        t = turn if c["direction"] == "forward" else turn.conj()
        return rotate(q, t), rotate(k, t)
    ins = [q.requires_grad_(), k.requires_grad_(), s["gq"].double().requires_grad_(), s["gk"].double().requires_grad_()]
    outs = [rotate(x / (x.square().mean(-1, keepdim=True) + s["eps"]).sqrt() * g, turn)
            for x, g in ((ins[0], ins[2]), (ins[1], ins[3]))]
    if c["direction"] == "forward":
        return tuple(o.detach() for o in outs)
    return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, ins, [s["dq"].double(), s["dk"].double()])


def _exact_cross(c, s):
    B, Hq, Hk = c["B"], c["Hq"], c["Hk"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    train = c["direction"] == "train"
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    ends = [c["Tk"]] * B if s["lengths"] is None else s["lengths"].tolist()
    for b in range(B):
        n = ends[b]
        if n == 0:
            continue
        for h in range(Hq):
            j = h // (Hq // Hk)
            x = [t.requires_grad_(train) for t in (q[b, :, h].clone(), k[b, :n, j].clone(), v[b, :n, j].clone())]
            o = torch.softmax((x[0] @ x[1].T) * s["scale"], -1) @ x[2]
            out[b, :, h] = o.detach()
            if train:
                a, e, f = torch.autograd.grad(o, x, s["grad"][b, :, h].double())
                dq[b, :, h] = a
                dk[b, :n, j] += e
                dv[b, :n, j] += f
    return (out, dq, dk, dv) if train else out
